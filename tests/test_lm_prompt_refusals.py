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
