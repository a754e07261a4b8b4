"""What the operators for prompts refuse before anything is enqueued, and what they declare; no GPU is used."""
import ctypes as C

import pytest

from paella_b200 import capi
from tests import lm_util as lu

A = 1 << 20      # an address that stands for a buffer: nothing reads it


def norm(**over):
    f = dict(tokens=4, channels=64, dtype=capi.BF16, h_dtype=capi.BF16, scale=1.0, eps=1e-6, x_stride=64, gate_stride=64, residual_stride=64, h_stride=64, y_stride=64, x=A, post_weight=A, gate=A,
             residual=A, h=A, weight=A, y=A)
    return capi.ResidualNormParams(**{**f, **over})


@pytest.mark.parametrize("over", [dict(tokens=-1), dict(channels=0), dict(channels=32769), dict(channels=-1), dict(dtype=3), dict(dtype=-1), dict(h_dtype=capi.F16), dict(dtype=capi.F32), dict(h_dtype=3),
                                  dict(scale=float("inf")), dict(scale=float("nan")), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=None), dict(h=None, y=None), dict(x=A + 1),
                                  dict(gate=A + 1), dict(residual=A + 1), dict(h_dtype=capi.F32, residual=A + 2), dict(h_dtype=capi.F32, h=A + 2), dict(h=A + 1), dict(y=A + 1), dict(post_weight=A + 2),
                                  dict(weight=A + 2), dict(h_stride=0), dict(h_stride=63), dict(y_stride=-63), dict(y_stride=0)])
def test_norm_refusals(over):
    assert lu.refused("residual_norm", norm(**over)).startswith("pb_residual_norm")


@pytest.mark.parametrize("over", [dict(tokens=0, x=None), dict(tokens=1, h_stride=0, y_stride=0), dict(h=None, h_stride=0), dict(y=None, y_stride=0), dict(x_stride=0, gate_stride=0, residual_stride=0),
                                  dict(h_stride=-64), dict(post_weight=None, gate=None, residual=None, weight=None), dict(channels=32768, x_stride=1, h_stride=32768, y_stride=32768)])
def test_norm_takes(over):
    assert lu.info("residual_norm", norm(**over)).num_blocks >= 1


def test_norm_struct_size_and_declared_work():
    assert C.sizeof(capi.ResidualNormParams) == 6 * 4 + 5 * 8 + 7 * 8
    li = lu.info("residual_norm", norm())
    assert li.bytes == 4 * 64 * 2 * 5 + 2 * 4 * 64 and li.threads_per_block >= 32
    assert lu.info("residual_norm", norm(gate_stride=0)).bytes == 4 * 64 * 2 * 4 + 64 * 2 + 2 * 4 * 64
    assert lu.info("residual_norm", norm(tokens=0)).bytes == 0
    L = capi.load()
    assert L.pb_residual_norm_info(None, C.byref(li)) == -2 and L.pb_residual_norm_launch(None, None, 0, None) == -2


def logprobs(**over):
    f = dict(tokens=4, vocab=100, dtype=capi.BF16, top=5, scale=1.0, logits_stride=100, top_stride=5, logits=A, targets=A, logprobs=A, ranks=A, entropy=A, top_ids=A, top_logprobs=A)
    return capi.LogprobsParams(**{**f, **over})


@pytest.mark.parametrize("over", [dict(tokens=-1), dict(vocab=0), dict(vocab=-5), dict(vocab=2 ** 30 + 1), dict(dtype=3), dict(dtype=-1), dict(top=-1), dict(top=33), dict(vocab=4), dict(scale=0.0), dict(scale=-1.0),
                                  dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=2e6), dict(scale=1e-7), dict(logits=None), dict(logits=A + 1), dict(dtype=capi.F32, logits=A + 2), dict(targets=None),
                                  dict(targets=A + 2), dict(logprobs=A + 1), dict(ranks=A + 2), dict(entropy=A + 2), dict(top_ids=A + 2), dict(top_logprobs=A + 3), dict(top=0, top_stride=0), dict(top_stride=4),
                                  dict(top_stride=0), dict(logprobs=None, ranks=None, entropy=None, top_ids=None, top_logprobs=None), dict(targets=None, ranks=None)])
def test_logprobs_refusals(over):
    assert lu.refused("logprobs", logprobs(**over)).startswith("pb_logprobs")


@pytest.mark.parametrize("over", [dict(tokens=0, logits=None), dict(tokens=1, top_stride=0), dict(top=0, top_ids=None, top_logprobs=None, top_stride=0), dict(targets=None, logprobs=None, ranks=None),
                                  dict(top_ids=None), dict(top_stride=-5), dict(logits_stride=0), dict(logits_stride=-100), dict(vocab=5, top=5), dict(scale=1e-6), dict(scale=1e6)])
def test_logprobs_takes(over):
    assert lu.info("logprobs", logprobs(**over)).num_blocks >= 1


def test_logprobs_struct_size_and_declared_work():
    assert C.sizeof(capi.LogprobsParams) == 6 * 4 + 2 * 8 + 7 * 8
    li = lu.info("logprobs", logprobs())
    assert li.bytes == 4 * (100 * 2 + 4 * 4 + 2 * 4 * 5) and li.num_blocks == 4 and li.flops == 6 * 4 * 100
    assert lu.info("logprobs", logprobs(tokens=0)).bytes == 0
    assert lu.info("logprobs", logprobs(vocab=131072)).num_blocks == 32
    L = capi.load()
    assert L.pb_logprobs_info(None, C.byref(li)) == -2 and L.pb_logprobs_launch(None, None, 0, None) == -2


def chunk(**over):
    f = dict(dtype=capi.BF16, batch=4, tokens=40, q_heads=8, kv_heads=2, head_dim=64, page_size=16, max_blocks=8, max_new=20, max_len=128, window=0, scale=0.125, n_pages=40, q_stride=512, q_head_stride=64,
             out_stride=512, out_head_stride=64, page_stride=2048, token_stride=128, head_stride=64, table_stride=8, q=A, out=A, k_cache=A, v_cache=A, block_table=A, starts=A, lens=A, scratch=A,
             scratch_bytes=1 << 40)
    return capi.ChunkAttnParams(**{**f, **over})


@pytest.mark.parametrize("over", [dict(dtype=capi.F32), dict(dtype=3), dict(batch=-1), dict(batch=2 ** 31 - 1), dict(tokens=-1), dict(q_heads=0), dict(kv_heads=0), dict(q_heads=7), dict(q_heads=2 ** 17, kv_heads=1),
                                  dict(head_dim=136), dict(head_dim=12), dict(head_dim=0), dict(page_size=0), dict(page_size=12), dict(page_size=2 ** 25), dict(max_blocks=-1), dict(max_len=129), dict(max_len=-1),
                                  dict(max_len=2 ** 30 + 1, max_blocks=2 ** 30), dict(max_new=-1), dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(n_pages=-1),
                                  dict(n_pages=2 ** 31), dict(n_pages=0), dict(page_stride=2050), dict(page_stride=0), dict(token_stride=4), dict(token_stride=-128), dict(head_stride=63), dict(q_stride=12), dict(q_head_stride=4),
                                  dict(q=A + 8), dict(k_cache=A + 2), dict(v_cache=A + 8), dict(out=A + 1), dict(q=None), dict(out=None), dict(k_cache=None), dict(v_cache=None), dict(block_table=None),
                                  dict(starts=None), dict(lens=None), dict(starts=A + 1), dict(lens=A + 2), dict(block_table=A + 2), dict(out_stride=0), dict(out_stride=63), dict(out_head_stride=-63)])
def test_chunk_refusals(over):
    assert lu.refused("chunk_attn", chunk(**over)).startswith("pb_chunk_attn")


@pytest.mark.parametrize("over", [dict(batch=0, q=None), dict(tokens=0, q=None, out=None), dict(max_new=0, starts=None), dict(max_len=0, k_cache=None, block_table=None, n_pages=0, max_blocks=0), dict(tokens=1, out_stride=0),
                                  dict(q_stride=0), dict(q_stride=-512), dict(out_stride=-512), dict(table_stride=0), dict(window=2 ** 31 - 1), dict(max_new=2 ** 31 - 1), dict(scale=-2e38), dict(max_new=1), dict(max_new=2)])
def test_chunk_takes(over):
    assert lu.info("chunk_attn", chunk(**over)).num_blocks >= 1


def test_chunk_struct_size_and_null_params():
    assert C.sizeof(capi.ChunkAttnParams) == 12 * 4 + 9 * 8 + 9 * 8
    L, li = capi.load(), capi.LaunchInfo()
    assert L.pb_chunk_attn_info(None, C.byref(li)) == -2 and L.pb_chunk_attn_launch(None, None, 0, None) == -2


def test_chunk_starts_of_many_sequences_need_scratch():
    few, many = chunk(batch=256, max_new=1), chunk(batch=257, max_new=1)
    assert lu.info("chunk_attn", few).scratch_bytes == 0
    need = lu.info("chunk_attn", many).scratch_bytes
    assert need >= 4 * 258
    L = capi.load()
    for over in (dict(scratch=None, scratch_bytes=need), dict(scratch=A, scratch_bytes=need - 1), dict(scratch=A + 8, scratch_bytes=need)):
        assert L.pb_chunk_attn_launch(C.byref(chunk(batch=257, max_new=1, **over)), None, 0, None) == -2 and b"scratch" in L.pb_last_error()
