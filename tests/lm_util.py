"""Helpers for the tests of the language-model operators."""
import ctypes as C

import torch

from paella_b200 import capi

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": capi.F32, "bf16": capi.BF16, "f16": capi.F16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}     # the most a rounding is off, relative
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}       # the smallest step near zero


def ptr(t):
    return None if t is None else t.data_ptr()


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def launch(name, p, stream=None, job_id=0, notifier=None):
    L = capi.load()
    st = torch.cuda.current_stream().cuda_stream if stream is None else stream.cuda_stream
    capi.check(getattr(L, f"pb_{name}_launch")(C.byref(p), st, job_id, notifier), f"pb_{name}_launch")


def info(name, p):
    L, li = capi.load(), capi.LaunchInfo()
    capi.check(getattr(L, f"pb_{name}_info")(C.byref(p), C.byref(li)), f"pb_{name}_info")
    return li


def refused(name, p):
    """Both entry points refuse the parameters (no GPU is needed for that); the message."""
    L, li = capi.load(), capi.LaunchInfo()
    assert getattr(L, f"pb_{name}_info")(C.byref(p), C.byref(li)) == -2
    assert getattr(L, f"pb_{name}_launch")(C.byref(p), None, 0, None) == -2
    return L.pb_last_error().decode()


def records(name, p):
    """Launches with a notifier; (blocks started, blocks ended) that its ring reports for the job."""
    L = capi.load()
    ring, nf = C.c_void_p(), C.c_void_p()
    capi.check(L.pb_ring_create(0, 1 << 16, C.byref(ring)), "pb_ring_create")
    capi.check(L.pb_notifier_create_array(ring, 1, C.byref(nf)), "pb_notifier_create_array")
    try:
        launch(name, p, job_id=5, notifier=nf)
        torch.cuda.synchronize()
        buf = (C.c_uint64 * 8192)()
        n = L.pb_ring_poll(ring, buf, 8192)
        started = ended = 0
        for r in buf[:n]:
            assert r >> 32 == 5                                # the job
            num, kind = (r >> 16) & 0xff, r & 0xff
            started += num if kind == 1 else 0
            ended += num if kind == 0 else 0
        return started, ended
    finally:
        L.pb_notifier_free_array(nf)
        L.pb_ring_destroy(ring)

