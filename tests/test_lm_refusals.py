"""What the language-model operators refuse before anything is enqueued, and what they declare; no GPU is used."""
import ctypes as C

import pytest

from paella_b200 import capi
from tests import lm_util as lu

A = 1 << 20      # an address that stands for a buffer: nothing reads it


def rope(**over):
    f = dict(dtype=capi.BF16, tokens=4, q_heads=4, kv_heads=2, head_dim=64, rot_dim=64, max_position=16, eps=1e-6, q_stride=256, q_head_stride=64, k_stride=128,
             k_head_stride=64, q_out_stride=256, q_out_head_stride=64, k_out_stride=128, k_out_head_stride=64, q=A, k=A, q_out=A, k_out=A, cos_sin=A, positions=A)
    return capi.QkRopeParams(**{**f, **over})


def append(**over):
    f = dict(dtype=capi.BF16, tokens=4, q_heads=4, kv_heads=2, head_dim=64, rot_dim=64, max_position=16, eps=1e-6, page_size=16, n_pages=4, k_stride=128,
             k_head_stride=64, v_stride=128, v_head_stride=64, page_stride=2048, token_stride=128, head_stride=64, q_stride=256, q_head_stride=64,
             q_out_stride=256, q_out_head_stride=64, k=A, v=A, cos_sin=A, positions=A, slots=A, k_cache=A, v_cache=A, q=A, q_out=A)
    return capi.KvAppendParams(**{**f, **over})


BAD_HEADS = [dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(q_heads=-1), dict(kv_heads=-1), dict(kv_heads=70000), dict(head_dim=0), dict(head_dim=257), dict(rot_dim=63),
             dict(rot_dim=66), dict(rot_dim=-2), dict(max_position=0), dict(cos_sin=None), dict(positions=None), dict(q=None), dict(q_out=None), dict(k=None),
             dict(q=A + 1), dict(k=A + 1), dict(cos_sin=A + 2), dict(positions=A + 2)]


@pytest.mark.parametrize("over", BAD_HEADS + [dict(q_heads=0, kv_heads=0), dict(k_out=None), dict(tokens=2 ** 31 - 1, q_heads=65536, kv_heads=65536)])
def test_rope_refusals(over):
    assert lu.refused("qk_rope", rope(**over)).startswith("pb_qk_rope")


@pytest.mark.parametrize("over", BAD_HEADS + [dict(kv_heads=0), dict(page_size=0), dict(n_pages=-1), dict(n_pages=2 ** 62), dict(v=None), dict(slots=None), dict(slots=A + 4),
                                              dict(k_cache=None), dict(v_cache=None), dict(v_cache=A + 1)])
def test_append_refusals(over):
    assert lu.refused("kv_append", append(**over)).startswith("pb_kv_append")


def test_null_params_are_refused():
    L, li = capi.load(), capi.LaunchInfo()
    for name, kind in (("qk_rope", capi.QkRopeParams), ("kv_append", capi.KvAppendParams)):
        assert getattr(L, f"pb_{name}_info")(None, C.byref(li)) == -2
        assert getattr(L, f"pb_{name}_launch")(None, None, 0, None) == -2


def test_struct_sizes_match_the_header():
    assert C.sizeof(capi.QkRopeParams) == 10 * 4 + 8 * 8 + 8 * 8
    assert C.sizeof(capi.KvAppendParams) == 10 * 4 + 12 * 8 + 11 * 8


def test_declared_work():
    li = lu.info("qk_rope", rope())
    assert li.bytes == 4 * (2 * 2 * 64 * 6 + 4 * 64 + 4) and li.threads_per_block == 256 and li.num_blocks >= 1
    li = lu.info("kv_append", append(tokens=0))
    assert li.bytes == 0 and li.num_blocks == 1


def quantize(**over):
    return capi.Int8QuantizeParams(**{**dict(tokens=4, channels=64, x_dtype=capi.BF16, x_stride=64, q_stride=64, x=A, q=A, scale=A), **over})


def dense(**over):
    return capi.Int8DenseParams(**{**dict(tokens=4, in_channels=64, out_channels=32, y_dtype=capi.BF16, x_stride=64, w_stride=64, y_stride=32, x=A, x_scale=A, w=A, w_scale=A, y=A), **over})


@pytest.mark.parametrize("over", [dict(tokens=-1), dict(channels=0), dict(x_dtype=3), dict(x=None), dict(q=None), dict(scale=None), dict(x=A + 1), dict(scale=A + 2)])
def test_quantize_refusals(over):
    assert lu.refused("int8_quantize", quantize(**over)).startswith("pb_int8_quantize")


@pytest.mark.parametrize("over", [dict(tokens=-1), dict(in_channels=0), dict(out_channels=0), dict(in_channels=131072, x_stride=131072, w_stride=131072), dict(y_dtype=3), dict(act=3), dict(act=-1),
                                  dict(x_stride=72), dict(w_stride=8), dict(x_stride=48), dict(w_stride=48), dict(x=A + 8), dict(w=A + 4), dict(x=None), dict(x_scale=None), dict(w=None),
                                  dict(w_scale=None), dict(y=None), dict(y=A + 1), dict(bias=A + 2), dict(x_scale=A + 1)])
def test_dense_refusals(over):
    assert lu.refused("int8_dense", dense(**over)).startswith("pb_int8_dense")


def test_int8_struct_sizes_and_null_params():
    assert C.sizeof(capi.Int8QuantizeParams) == 4 * 4 + 2 * 8 + 3 * 8 and C.sizeof(capi.Int8DenseParams) == 6 * 4 + 3 * 8 + 6 * 8
    L, li = capi.load(), capi.LaunchInfo()
    for name in ("int8_quantize", "int8_dense"):
        assert getattr(L, f"pb_{name}_info")(None, C.byref(li)) == -2
        assert getattr(L, f"pb_{name}_launch")(None, None, 0, None) == -2


def test_declared_work_of_a_dense_layer():
    li = lu.info("int8_dense", dense(bias=A))
    assert li.flops == 2 * 4 * 64 * 32 and li.bytes == 4 * 64 + 32 * 64 + 4 * 4 + 8 * 32 + 2 * 4 * 32


def attn(**over):
    f = dict(dtype=capi.BF16, batch=4, q_heads=8, kv_heads=2, head_dim=64, page_size=16, max_blocks=4, prefix_len=100, max_own_len=64, scale=0.125, n_pages=40, q_stride=512,
             q_head_stride=64, out_stride=512, out_head_stride=64, page_stride=2048, token_stride=128, head_stride=64, table_stride=4, q=A, out=A, k_cache=A, v_cache=A,
             prefix_pages=A, block_table=A, own_lens=A, scratch=A, scratch_bytes=1 << 40)
    return capi.PrefixAttnParams(**{**f, **over})


@pytest.mark.parametrize("over", [dict(dtype=capi.F32), dict(dtype=3), dict(batch=-1), dict(q_heads=0), dict(kv_heads=0), dict(q_heads=7), dict(head_dim=136), dict(head_dim=12), dict(head_dim=0),
                                  dict(page_size=0), dict(page_size=12), dict(max_blocks=-1), dict(max_own_len=65), dict(max_own_len=-1), dict(prefix_len=-1), dict(scale=float("nan")),
                                  dict(scale=float("inf")), dict(n_pages=-1), dict(n_pages=2 ** 31), dict(page_stride=2050), dict(token_stride=4), dict(head_stride=63), dict(q_stride=12), dict(q_head_stride=4),
                                  dict(q=A + 8), dict(k_cache=A + 2), dict(v_cache=A + 8), dict(out=A + 1), dict(q=None), dict(out=None), dict(k_cache=None), dict(v_cache=None),
                                  dict(prefix_pages=None), dict(block_table=None), dict(own_lens=None), dict(own_lens=A + 2)])
def test_attention_refusals(over):
    assert lu.refused("prefix_attn", attn(**over)).startswith("pb_prefix_attn")


def test_attention_struct_size_and_declared_work():
    assert C.sizeof(capi.PrefixAttnParams) == 10 * 4 + 9 * 8 + 9 * 8
    li = lu.info("prefix_attn", attn())
    assert li.flops == 4 * 64 * 8 * 4 * 164 and li.num_blocks >= 1
    assert lu.info("prefix_attn", attn(prefix_len=0, prefix_pages=None)).num_blocks >= 1
    assert lu.info("prefix_attn", attn(max_own_len=0, block_table=None, own_lens=None, max_blocks=0)).num_blocks >= 1
    L = capi.load()
    assert L.pb_prefix_attn_info(None, C.byref(li)) == -2 and L.pb_prefix_attn_launch(None, None, 0, None) == -2


# sizes whose sums with a tile would pass 32 bits, weights between floats, a scale that is infinite in powers of two
@pytest.mark.parametrize("name,params", [("int8_quantize", quantize(tokens=2 ** 31 - 1)), ("int8_quantize", quantize(channels=2 ** 31 - 1)), ("int8_dense", dense(tokens=2 ** 31 - 1)),
                                         ("int8_dense", dense(out_channels=2 ** 31 - 1)), ("qk_rope", rope(q_weight=A + 2)), ("qk_rope", rope(k_weight=A + 2)),
                                         ("kv_append", append(q_weight=A + 1)), ("kv_append", append(k_weight=A + 2)), ("prefix_attn", attn(scale=3e38)),
                                         ("prefix_attn", attn(scale=-3e38))])
def test_more_refusals(name, params):
    assert lu.refused(name, params).startswith("pb_" + name)


# rows of results that lie over one another, forgotten strides among them; where there is only one row its stride does not matter
@pytest.mark.parametrize("name,params", [("int8_quantize", quantize(q_stride=0)), ("int8_quantize", quantize(q_stride=63)), ("int8_quantize", quantize(q_stride=-63)), ("int8_dense", dense(y_stride=0)),
                                         ("int8_dense", dense(y_stride=31)), ("int8_dense", dense(y_stride=-31)),
                                         ("qk_rope", rope(q_out_stride=0)), ("qk_rope", rope(q_out_head_stride=63)), ("qk_rope", rope(k_out_stride=-63)), ("qk_rope", rope(k_out_head_stride=0)),
                                         ("kv_append", append(page_stride=0)), ("kv_append", append(token_stride=63)), ("kv_append", append(head_stride=0)), ("kv_append", append(q_out_stride=8)),
                                         ("kv_append", append(q_out_head_stride=0)), ("prefix_attn", attn(out_stride=0)), ("prefix_attn", attn(out_stride=63)), ("prefix_attn", attn(out_head_stride=-63))])
def test_rows_of_results_that_overlap_are_refused(name, params):
    assert lu.refused(name, params).startswith("pb_" + name)


@pytest.mark.parametrize("name,params", [("int8_quantize", quantize(tokens=1, q_stride=0)), ("int8_quantize", quantize(q_stride=-64)), ("int8_quantize", quantize(x_stride=0)),
                                         ("int8_dense", dense(tokens=1, y_stride=0)), ("int8_dense", dense(y_stride=-2 ** 63)), ("qk_rope", rope(tokens=1, q_out_stride=0, k_out_stride=0)),
                                         ("qk_rope", rope(kv_heads=1, k_out_head_stride=0)), ("qk_rope", rope(kv_heads=0, k_out_stride=0)), ("qk_rope", rope(q_stride=0, k_head_stride=0)),
                                         ("kv_append", append(n_pages=1, page_stride=0)), ("kv_append", append(page_size=1, token_stride=0)), ("kv_append", append(kv_heads=1, head_stride=0)),
                                         ("kv_append", append(q_heads=0, q_out_stride=0)), ("prefix_attn", attn(batch=1, out_stride=0)), ("prefix_attn", attn(q_heads=1, kv_heads=1, out_head_stride=0))])
def test_strides_of_lone_rows_and_of_inputs_are_free(name, params):
    lu.info(name, params)


def test_attention_declares_what_its_largest_kernel_holds():
    """The last kernel's blocks report, and together they declare the most that any kernel of the launch holds: the prefix's takes whole SMs, with all of their tensor memory."""
    sizes = dict(head_dim=128, page_stride=2 ** 15, token_stride=1024, head_stride=128, q_stride=2 ** 14, out_stride=2 ** 14, q_head_stride=128, out_head_stride=128, n_pages=2 ** 20,
                 page_size=32, max_blocks=32, table_stride=32, max_own_len=512)
    for batch, q_heads, kv_heads, prefix, blocks in ((32, 32, 8, 8192, 144), (1, 8, 1, 130001, 148), (256, 64, 8, 16384, 128)):
        li = lu.info("prefix_attn", attn(batch=batch, q_heads=q_heads, kv_heads=kv_heads, prefix_len=prefix, **sizes))
        assert li.num_blocks * li.threads_per_block >= blocks * 384
        assert li.num_blocks * li.smem_per_block >= blocks * 225 * 1024
        assert li.num_blocks * li.tmem_cols_per_block >= blocks * 512
    # where the sequences' own tokens have more blocks than fit at once, those hold more shared memory than the prefix's, and the join, which reports, less than either
    li = lu.info("prefix_attn", attn(batch=256, q_heads=64, kv_heads=8, prefix_len=16384, **sizes))
    assert li.num_blocks == 2048 and li.smem_per_block >= 64 * 1024 and li.threads_per_block == 128
    li = lu.info("prefix_attn", attn(batch=4, q_heads=32, kv_heads=8, prefix_len=0, **sizes))
    assert li.threads_per_block == 128 and li.tmem_cols_per_block == 0 and li.smem_per_block >= 64 * 1024
