"""Kernel times by kind: the entry point that callers were built with writes as
many kinds as it always did, the other one all of them."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

FIRST = 11  # kinds of spt_ctx_read_timing


def test_arrays_of_either_size(gpu_ctx):
    import spt
    from test_gpu_attention import Filled, run

    kinds = len(spt.KERNEL_KINDS)
    assert kinds > FIRST and spt.KERNEL_KINDS[FIRST:] == ("kv", "attention")
    gpu_ctx.enable_timing(True)
    try:
        gpu_ctx.read_timing()
        p = Filled(gpu_ctx, 4, 1, 64, 32, [1], [40])
        run(gpu_ctx, p, p.rng.standard_normal((1, 4, 64)).astype("float32"), 0.125)
        got = gpu_ctx.read_timing()
        assert got["kv"][1] == 1 and got["attention"][1] == 1 and got["attention"][0] > 0
        assert gpu_ctx.read_timing()["kv"] == (0.0, 0)
        ms, n = (C.c_double * kinds)(*[-7.0] * kinds), (C.c_int64 * kinds)(*[-7] * kinds)
        assert spt.lib().spt_ctx_read_timing(gpu_ctx.handle, ms, n) == spt.OK
        assert list(ms) == [0.0] * FIRST + [-7.0] * (kinds - FIRST) and list(n) == [0] * FIRST + [-7] * (kinds - FIRST)
    finally:
        gpu_ctx.enable_timing(False)
