"""What the key/value cache's entry points refuse, on a validation-only
context: every rule of the header, one field wrong at a time; and that a valid
call gets past them (the context has no device)."""
import ctypes as C

import pytest


class Call:
    """A valid set of arguments; addresses are never followed."""

    def __init__(self):
        import spt

        self.cache = spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, 64, 5, 1 << 20)
        self.batch = spt.KVBatch(3, 4, 7, 100, 2, 64, 128, 192)
        self.rope = spt.Rope(150000.0, 32.0, 4096, 32.0, 1.0)
        self.n = 7 * 2 * 64
        self.k, self.v, self.q, self.out = (0x10000000 + i * 0x100000 for i in range(4))
        self.q_len = self.out_len = 7 * 6 * 64
        self.k_len = self.v_len = self.n
        self.sinks, self.scale, self.window, self.q8, self.work, self.work_bytes = None, 0.125, 0, None, None, 0

    def store(self, ctx):
        import spt

        r = lambda s: C.byref(s) if s is not None else None  # noqa: E731
        return spt.lib().spt_kv_store_batch(ctx.handle, r(self.cache), r(self.batch), r(self.rope), self.q, self.q_len, self.out,
                                            self.out_len, self.k, self.k_len, self.v, self.v_len)

    def load(self, ctx):
        import spt

        r = lambda s: C.byref(s) if s is not None else None  # noqa: E731
        return spt.lib().spt_kv_load_batch(ctx.handle, r(self.cache), r(self.batch), self.k, self.k_len, self.v, self.v_len)

    def attend(self, ctx):
        import spt

        r = lambda s: C.byref(s) if s is not None else None  # noqa: E731
        return spt.lib().spt_attention_batch_into(ctx.handle, r(self.cache), r(self.batch), r(self.sinks), self.scale, self.window,
                                                  self.q, self.q_len, self.out, self.out_len, self.q8, self.work, self.work_bytes)


@pytest.fixture(scope="module")
def ctx():
    import spt

    c = spt.Context(-1)
    yield c
    c.close()


ALL = ("store", "load", "attend")


@pytest.mark.parametrize("entry", ALL)
def test_valid_calls_reach_the_device(ctx, entry):
    import spt

    assert getattr(Call(), entry)(ctx) == spt.ERR_DEVICE
    c = Call()  # nothing to do is no error either, but needs a device
    c.batch.n_rows = 0
    c.k_len = c.v_len = c.q_len = c.out_len = 0
    assert getattr(c, entry)(ctx) == spt.ERR_DEVICE


COMMON = {
    "nil cache": lambda c: setattr(c, "cache", None),
    "nil batch": lambda c: setattr(c, "batch", None),
    "type": lambda c: setattr(c.cache, "type", 39),
    "head dim": lambda c: setattr(c.cache, "head_dim", 96),
    "page length": lambda c: setattr(c.cache, "page_len", 48),
    "page length 0": lambda c: setattr(c.cache, "page_len", 0),
    "no heads": lambda c: setattr(c.cache, "n_kv_heads", 0),
    "many heads": lambda c: setattr(c.cache, "n_kv_heads", 1 << 20),
    "no pages": lambda c: setattr(c.cache, "n_pages", 0),
    "pages overflow": lambda c: setattr(c.cache, "n_pages", 1 << 62),
    "bytes": lambda c: setattr(c.cache, "nbytes", c.cache.nbytes - 1),
    "no data": lambda c: setattr(c.cache, "data", None),
    "data alignment": lambda c: setattr(c.cache, "data", (1 << 20) + 8),
    "sequences": lambda c: setattr(c.batch, "n_seqs", -1),
    "many sequences": lambda c: setattr(c.batch, "n_seqs", 65536),
    "rows": lambda c: setattr(c.batch, "n_rows", -1),
    "many rows": lambda c: setattr(c.batch, "n_rows", 1 << 40),
    "rows of the buffers": lambda c: setattr(c.batch, "n_rows", 8),
    "no new": lambda c: setattr(c.batch, "max_new", 0),
    "many new": lambda c: setattr(c.batch, "max_new", (1 << 24) + 1),
    "no length": lambda c: setattr(c.batch, "max_len", 0),
    "long": lambda c: (setattr(c.batch, "max_len", (1 << 30) + 1), setattr(c.batch, "max_pages", 1 << 29)),
    "no page table": lambda c: setattr(c.batch, "max_pages", 0),
    "pages too few": lambda c: setattr(c.batch, "max_len", 129),
    "nil rows": lambda c: setattr(c.batch, "rows_dev", None),
    "nil lengths": lambda c: setattr(c.batch, "lens_dev", None),
    "nil table": lambda c: setattr(c.batch, "pages_dev", None),
    "rows alignment": lambda c: setattr(c.batch, "rows_dev", 66),
}
KV = {
    "nil keys": lambda c: setattr(c, "k", None),
    "nil values": lambda c: setattr(c, "v", None),
    "key alignment": lambda c: setattr(c, "k", c.k + 4),
    "key length": lambda c: setattr(c, "k_len", c.n - 64),
    "value length": lambda c: setattr(c, "v_len", c.n + 64),
    "keys in the cache": lambda c: setattr(c, "k", c.cache.data),
    "values in the cache": lambda c: setattr(c, "v", c.cache.data + 16),
}
STORE = {
    "queries without rope": lambda c: setattr(c, "rope", None),
    "query lengths": lambda c: setattr(c, "out_len", c.q_len - 64),
    "query heads": lambda c: (setattr(c, "q_len", 7 * 5 * 64), setattr(c, "out_len", 7 * 5 * 64)),
    "ragged queries": lambda c: (setattr(c, "q_len", c.q_len + 1), setattr(c, "out_len", c.out_len + 1)),
    "nil queries": lambda c: setattr(c, "q", None),
    "nil rotated": lambda c: setattr(c, "out", None),
    "query alignment": lambda c: setattr(c, "q", c.q + 8),
    "partial overlap": lambda c: setattr(c, "out", c.q + 64),
    "onto the keys": lambda c: setattr(c, "out", c.k),
    "onto the values": lambda c: setattr(c, "out", c.v + 16),
    "into the cache": lambda c: setattr(c, "out", c.cache.data),
    "base 1": lambda c: setattr(c.rope, "base", 1.0),
    "base nan": lambda c: setattr(c.rope, "base", float("nan")),
    "base inf": lambda c: setattr(c.rope, "base", float("inf")),
    "factor": lambda c: setattr(c.rope, "factor", 0.5),
    "factor inf": lambda c: setattr(c.rope, "factor", float("inf")),
    "betas": lambda c: setattr(c.rope, "beta_slow", 32.0),
    "slow 0": lambda c: setattr(c.rope, "beta_slow", 0.0),
    "fast inf": lambda c: setattr(c.rope, "beta_fast", float("inf")),
    "original": lambda c: setattr(c.rope, "original_len", 0),
}
LOAD = {"overlap": lambda c: setattr(c, "v", c.k + 16)}


def _sinks(c, **kw):
    import spt

    c.sinks = spt.Tensor.make("attn_sinks", spt.TYPE_F32, [6], 0x20000000, 24)
    for k, v in kw.items():
        setattr(c.sinks, k, v)


ATTEND = {
    "nil queries": lambda c: setattr(c, "q", None),
    "nil output": lambda c: setattr(c, "out", None),
    "query alignment": lambda c: setattr(c, "q", c.q + 4),
    "output alignment": lambda c: setattr(c, "out", c.out + 4),
    "output length": lambda c: setattr(c, "out_len", c.q_len + 64),
    "heads": lambda c: (setattr(c, "q_len", 7 * 3 * 64), setattr(c, "out_len", 7 * 3 * 64)),
    "ragged": lambda c: (setattr(c, "q_len", c.q_len + 1), setattr(c, "out_len", c.q_len + 1)),
    "in place": lambda c: setattr(c, "out", c.q),
    "output in the cache": lambda c: setattr(c, "out", c.cache.data),
    "window": lambda c: setattr(c, "window", -1),
    "scale 0": lambda c: setattr(c, "scale", 0.0),
    "scale nan": lambda c: setattr(c, "scale", float("nan")),
    "scale inf": lambda c: setattr(c, "scale", float("inf")),
    "sinks type": lambda c: _sinks(c, type=8),
    "sinks bytes": lambda c: _sinks(c, nbytes=28),
    "sinks alignment": lambda c: _sinks(c, data=0x20000002),
    "sinks data": lambda c: _sinks(c, data=None),
    "blocks on the queries": lambda c: setattr(c, "q8", c.q + 2),
    "blocks on the output": lambda c: setattr(c, "q8", c.out + 2),
    "blocks in the cache": lambda c: setattr(c, "q8", c.cache.data + 2),
}


def _entries():
    for entry, sets in (("store", (COMMON, KV, STORE)), ("load", (COMMON, KV, LOAD)), ("attend", (COMMON, ATTEND))):
        for s in sets:
            for what in s:
                yield pytest.param(entry, s[what], id=f"{entry}-{what}")


@pytest.mark.parametrize("entry,change", _entries())
def test_refusals(ctx, entry, change):
    import spt

    c = Call()
    change(c)
    assert getattr(c, entry)(ctx) == spt.ERR_INVALID
    assert spt.lib().spt_last_error()


def test_attention_workspace(ctx):
    """The size entry point: none for a short batch, some where positions are
    split; a smaller, unaligned or overlapping workspace is refused."""
    import spt

    c = Call()
    assert ctx.attention_work_bytes(c.cache, c.batch, 6) == 0
    for heads, window in ((5, 0), (0, 0), (6, -1)):
        with pytest.raises(spt.SptError):
            ctx.attention_work_bytes(c.cache, c.batch, heads, window)
    c.cache = spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, 64, 5, 1 << 44)
    c.batch.max_pages, c.batch.max_len = 4096, 200000
    n = ctx.attention_work_bytes(c.cache, c.batch, 6)
    assert n > 0
    assert ctx.attention_work_bytes(c.cache, c.batch, 6, window=64) == 0
    c.work, c.work_bytes = 0x40000000, n
    assert c.attend(ctx) == spt.ERR_DEVICE
    for work, size in ((0x40000000, n - 1), (0x40000008, n), (c.q, n), (c.out, n), (1 << 44, n)):
        c.work, c.work_bytes = work, size
        assert c.attend(ctx) == spt.ERR_INVALID


def test_sizes(ctx):
    """Cache sizes are the blocks' (18 and 34 bytes a block); sizes that do
    not exist are refused."""
    import spt

    assert spt.KVCache.bytes(spt.TYPE_Q4_0, 8, 64, 128, 8) == 1024 * 8 * 2 * 2 * 18
    assert spt.KVCache.bytes(spt.TYPE_Q8_0, 3, 128, 32, 7) == 7 * 32 * 3 * 2 * 4 * 34
    for bad in ((0, 8, 64, 128, 8), (2, 8, 32, 128, 8), (2, 8, 64, 33, 8), (2, -1, 64, 32, 8), (2, 8, 64, 32, 0)):
        with pytest.raises(spt.SptError):
            spt.KVCache.bytes(*bad)


def test_python_descriptors_check_their_tensors():
    import torch

    import spt

    with pytest.raises(ValueError):
        spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, 64, 5, torch.zeros(100, dtype=torch.uint8))
    i32 = dict(dtype=torch.int32)
    rows, lens, pages = torch.zeros(3, **i32), torch.zeros(2, **i32), torch.zeros(2, 4, **i32)
    spt.KVBatch.make(rows, lens, pages, 1, 1, 1)
    for bad in ((rows.long(), lens, pages), (rows, lens, pages.T.contiguous()), (rows, lens, pages[:, ::2]), (rows[:2], lens, pages)):
        with pytest.raises(ValueError):
            spt.KVBatch.make(*bad, 1, 1, 1)


@pytest.mark.parametrize("array", ("rows_dev", "lens_dev", "pages_dev"))
@pytest.mark.parametrize("entry,what", [("store", "out"), ("store", "cache"), ("load", "k"), ("load", "v"), ("load", "cache"),
                                        ("attend", "out"), ("attend", "q8"), ("attend", "work"), ("attend", "cache")])
def test_the_batch_is_not_written(ctx, entry, what, array):
    """What a call writes may not be the batch's arrays, which it reads."""
    import spt

    c = Call()
    if what == "work":
        c.cache = spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, 64, 5, 1 << 44)
        c.batch.max_pages, c.batch.max_len = 4096, 200000
        c.work, c.work_bytes = 0x40000000, ctx.attention_work_bytes(c.cache, c.batch, 6)
        c.batch.rows_dev, c.batch.lens_dev, c.batch.pages_dev = 0x3000000, 0x4000000, 0x5000000
    assert getattr(c, entry)(ctx) == spt.ERR_DEVICE
    c.q8 = 0x30000000 if what == "q8" else None
    setattr(c.batch, array, (c.cache.data if what == "cache" else getattr(c, what)) + 32)
    assert getattr(c, entry)(ctx) == spt.ERR_INVALID


@pytest.mark.parametrize("what", ("out", "q8", "work"))
def test_sinks_are_not_written(ctx, what):
    import spt

    c = Call()
    c.cache = spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, 64, 5, 1 << 44)
    c.batch.max_pages, c.batch.max_len = 4096, 200000
    c.work, c.work_bytes, c.q8 = 0x40000000, ctx.attention_work_bytes(c.cache, c.batch, 6), 0x30000000
    _sinks(c)
    assert c.attend(ctx) == spt.ERR_DEVICE
    c.sinks.data = getattr(c, what) + 32
    assert c.attend(ctx) == spt.ERR_INVALID


def test_scales_up_to_the_largest(ctx):
    """The scale is taken times log2 e in fp32: refused where that is infinite."""
    import spt

    c = Call()
    c.scale = 2.3e38
    assert c.attend(ctx) == spt.ERR_DEVICE
    c.scale = 2.4e38
    assert c.attend(ctx) == spt.ERR_INVALID


@pytest.mark.parametrize("empty", ("rows", "sequences"))
def test_an_empty_batch_needs_no_workspace(ctx, empty):
    """A workspace sized for the caller's heads is enough for a batch without
    rows, whose buffers say nothing of the heads; an unaligned one is not."""
    import spt

    c = Call()
    c.cache = spt.KVCache.make(spt.TYPE_Q4_0, 8, 64, 64, 5, 1 << 44)
    c.batch.n_seqs, c.batch.max_new, c.batch.max_len, c.batch.max_pages = 4, 16, 4000, 63
    n = ctx.attention_work_bytes(c.cache, c.batch, 64)
    assert n < ctx.attention_work_bytes(c.cache, c.batch, 8)
    c.work, c.work_bytes = 0x40000000, max(16, n)
    if empty == "rows":
        c.batch.n_rows = c.q_len = c.out_len = 0
    else:
        c.batch.n_seqs, c.q_len, c.out_len = 0, 7 * 8 * 64, 7 * 8 * 64
    assert c.attend(ctx) == spt.ERR_DEVICE
    c.work += 8
    assert c.attend(ctx) == spt.ERR_INVALID


def test_views_do_not_pass_for_buffers(ctx):
    """One element expanded, a strided view and too few blocks have as many
    elements as a buffer, or are taken for one; none has the memory."""
    import torch

    import spt

    u8 = dict(dtype=torch.uint8)
    n = spt.KVCache.bytes(spt.TYPE_Q4_0, 2, 64, 64, 5)
    spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, 64, 5, torch.zeros(n, **u8))
    for bad in (torch.zeros(1, **u8).expand(n), torch.zeros(2 * n, **u8)[::2], torch.zeros(n - 1, **u8)):
        with pytest.raises(ValueError):
            spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, 64, 5, bad)
    c = Call()
    c.cache = spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, 64, 5, 1 << 44)
    c.batch.max_pages, c.batch.max_len = 4096, 200000
    q, out = torch.zeros(7, 6, 64), torch.zeros(7, 6, 64)
    blocks, size = q.numel() // 32 * 34, ctx.attention_work_bytes(c.cache, c.batch, 6)
    attend = lambda **kw: ctx.attention_batch_into(c.cache, c.batch, q, out, 0.125, **kw)  # noqa: E731
    assert size % 4 == 0
    for good in (dict(q8=torch.zeros(blocks, **u8)), dict(work=torch.zeros(size, **u8)), dict(work=torch.zeros(size // 4))):
        with pytest.raises(spt.SptError) as e:
            attend(**good)
        assert e.value.code == spt.ERR_DEVICE
    for bad in (dict(q8=torch.zeros(blocks - 1, **u8)), dict(q8=torch.zeros(1, **u8).expand(blocks)),
                dict(work=torch.zeros(1, **u8).expand(size)), dict(work=torch.zeros(2 * size, **u8)[::2])):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(spt.SptError) as e:
        attend(work=torch.zeros(size // 4 - 1))
    assert e.value.code == spt.ERR_INVALID


def test_tensors_of_the_other_four_bytes(ctx):
    """Rows, lengths and pages in fp32, or queries, keys and values in int32,
    are as large as what is expected, and nothing like it."""
    import torch

    import spt

    rows, lens, pages = (torch.zeros(n, dtype=torch.int32) for n in (3, 2, (2, 4)))
    for bad in ((rows.float(), lens, pages), (rows, lens.float(), pages), (rows, lens, pages.float())):
        with pytest.raises(ValueError):
            spt.KVBatch.make(*bad, 1, 1, 1)
    c = Call()
    kv, q = torch.zeros(7, 2, 64), torch.zeros(7, 6, 64)
    calls = (lambda x, y: ctx.kv_load_batch(c.cache, c.batch, x, y), lambda x, y: ctx.kv_store_batch(c.cache, c.batch, x, y),
             lambda x, y: ctx.attention_batch_into(c.cache, c.batch, x, y, 0.125))
    for call, one in zip(calls, (kv, kv, q)):
        other = torch.zeros_like(one)
        with pytest.raises(spt.SptError) as e:
            call(one, other)
        assert e.value.code == spt.ERR_DEVICE
        for bad in ((one.int(), other), (one, other.int())):
            with pytest.raises(ValueError):
                call(*bad)
