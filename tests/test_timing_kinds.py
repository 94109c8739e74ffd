"""How many kinds of kernels a read of their times is asked for (no GPU)."""
import ctypes as C


def test_numbers_of_kinds_that_are_none():
    import spt

    ctx = spt.Context(-1)
    try:
        ms, n = (C.c_double * 64)(), (C.c_int64 * 64)()
        for kinds in (-1, 0, len(spt.KERNEL_KINDS) + 1, 2 ** 31 - 1):
            assert spt.lib().spt_ctx_read_timing_kinds(ctx.handle, ms, n, kinds) == spt.ERR_INVALID
        assert spt.lib().spt_ctx_read_timing_kinds(ctx.handle, ms, n, len(spt.KERNEL_KINDS)) == spt.ERR_DEVICE
        assert spt.lib().spt_ctx_read_timing(ctx.handle, ms, n) == spt.ERR_DEVICE
    finally:
        ctx.close()
