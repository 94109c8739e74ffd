"""The quantized key/value cache on the device: what a store writes (rotation,
blocks, marks of values that are not finite), where it writes it, and the
read back, bit for bit against the rule in numpy."""
import numpy as np
import pytest

from kv_reference import YARN, rotate, stored

pytestmark = pytest.mark.gpu


class Paged:
    """A cache of random bytes and a batch of sequences with shuffled pages."""

    def __init__(self, bits, kv, dim, page, new, lens, seed=0, extra_rows=0, spare=2, rows=None):
        import torch

        import spt

        self.rng = rng = np.random.default_rng(seed)
        self.bits, self.kv, self.dim, self.page = bits, kv, dim, page
        n_pages = [-(-x // page) for x in lens]
        self.n_pages = sum(n_pages) + spare
        ids = rng.permutation(self.n_pages)
        table = np.full((len(lens), max(n_pages + [1])), -1, np.int32)
        at = 0
        for i, n in enumerate(n_pages):
            table[i, :n] = ids[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.lens, self.table, self.n_rows = np.asarray(lens, np.int32), table, int(self.starts[-1]) + extra_rows
        typ = spt.TYPE_Q4_0 if bits == 4 else spt.TYPE_Q8_0
        n = spt.KVCache.bytes(typ, kv, dim, page, self.n_pages)
        self.data = torch.from_numpy(rng.integers(0, 256, n, dtype=np.uint8)).cuda()
        self.cache = spt.KVCache.make(typ, kv, dim, page, self.n_pages, self.data)
        self.batch = self.make_batch(self.starts, self.lens, max(list(new) + [1]), max(list(lens) + [1]))

    def make_batch(self, starts, lens, max_new, max_len, n_rows=None, table=None):
        import torch

        import spt

        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()  # noqa: E731
        return spt.KVBatch.make(dev(starts), dev(lens), dev(self.table if table is None else table),
                                self.n_rows if n_rows is None else n_rows, max_new, max_len)

    def positions(self):
        return np.concatenate([np.arange(n - (b - a), n) for a, b, n in zip(self.starts[:-1], self.starts[1:], self.lens)] + [[0]])[:-1]

    def whole(self):
        """(batch, rows) of every position of every sequence."""
        starts = np.concatenate([[0], np.cumsum(self.lens)]).astype(np.int32)
        n = int(starts[-1])
        return self.make_batch(starts, self.lens, max(1, int(self.lens.max())), max(1, int(self.lens.max())), n_rows=n), starts, n

    def load(self, ctx, batch=None, n=None):
        import torch

        if batch is None:
            batch, _, n = self.whole()
        out = [torch.full((n, self.kv, self.dim), 7.0, device="cuda") for _ in range(2)]
        ctx.kv_load_batch(self.cache, batch, *out)
        torch.cuda.synchronize()
        return [x.cpu().numpy() for x in out]


def _cuda(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def same(a, b):
    """Equal as numbers, NaN where NaN (a zero's sign is the scale's)."""
    return np.array_equal(a, b, equal_nan=True)


@pytest.mark.parametrize("bits", (4, 8))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("rope", (None, dict(base=10000.0), YARN), ids=("none", "plain", "yarn"))
@pytest.mark.parametrize("kv,group,page,new,lens", [
    (1, 1, 32, [1], [1]),
    (2, 3, 64, [1], [33]),
    (3, 2, 32, [1, 1, 1, 1], [1, 32, 33, 95]),
    (8, 8, 128, [5, 0, 33, 64], [5, 40, 70, 129]),
    (2, 1, 96, [100], [100]),
    (4, 5, 64, [31, 32, 1], [1000, 32, 64]),
])
def test_store_and_load(gpu_ctx, bits, dim, rope, kv, group, page, new, lens):
    """Rows read back as the rule's values, rotated queries as the 64-bit
    rotation rounded once, and every other position of the cache as it was."""
    import torch

    import spt

    p = Paged(bits, kv, dim, page, new, lens, seed=dim + kv)
    rng, n, pos = p.rng, int(p.starts[-1]), p.positions()
    q = rng.standard_normal((n, kv * group, dim)).astype(np.float32)
    k = (rng.standard_normal((n, kv, dim)) * np.exp(rng.standard_normal((n, kv, 1)))).astype(np.float32)
    v = rng.standard_normal((n, kv, dim)).astype(np.float32)
    before = p.load(gpu_ctx)
    if rope:
        qd = _cuda(q)
        q_out = torch.full_like(qd, 9.0)
        gpu_ctx.kv_store_batch(p.cache, p.batch, _cuda(k), _cuda(v), rope=spt.Rope(**rope), q=qd, q_out=q_out)
        assert same(q_out.cpu().numpy(), rotate(q, pos, rope)) and same(qd.cpu().numpy(), q)
        gpu_ctx.kv_store_batch(p.cache, p.batch, _cuda(k), _cuda(v), rope=spt.Rope(**rope), q=qd, q_out=qd)
        assert torch.equal(qd, q_out)
        k = rotate(k, pos, rope)
    else:
        gpu_ctx.kv_store_batch(p.cache, p.batch, _cuda(k), _cuda(v))
    want = stored(k, v, bits)
    got = p.load(gpu_ctx, p.batch, n)
    assert same(got[0], want[0]) and same(got[1], want[1])
    after = p.load(gpu_ctx)
    starts = np.concatenate([[0], np.cumsum(p.lens)])
    for s in range(len(lens)):
        old, a, b = slice(starts[s], starts[s + 1] - new[s]), p.starts[s], p.starts[s + 1]
        for x, y, w in zip(before, after, want):
            assert same(x[old], y[old])
            assert same(y[starts[s + 1] - new[s]:starts[s + 1]], w[a:b])


def test_pages_of_no_sequence_stay(gpu_ctx):
    """Bytes of pages that no sequence has are not touched."""
    p = Paged(4, 2, 64, 32, [3, 40], [3, 70], spare=5)
    per = p.data.numel() // p.n_pages
    before = p.data.cpu().numpy().reshape(p.n_pages, per)
    n = int(p.starts[-1])
    x = p.rng.standard_normal((n, 2, 64)).astype(np.float32)
    gpu_ctx.kv_store_batch(p.cache, p.batch, _cuda(x), _cuda(x))
    after = p.data.cpu().numpy().reshape(p.n_pages, per)
    free = np.setdiff1d(np.arange(p.n_pages), p.table.ravel())
    assert len(free) >= 5 and np.array_equal(before[free], after[free])
    assert not np.array_equal(before, after)


def _odd_blocks():
    """Rows of 64 that a rule gets wrong first: zeros, equal magnitudes of both
    signs, borders between codes, tiny and huge values."""
    rng = np.random.default_rng(5)
    rows = [np.zeros(64), -np.zeros(64), np.full(64, -8.0), np.tile([3.0, -3.0], 32), np.tile([-3.0, 3.0], 32),
            np.concatenate([np.arange(-8, 8), np.arange(-8, 8) + 0.5, np.arange(-127, -95) + 0.5]),
            np.linspace(-1, 1, 64) * 1e-38, np.linspace(-1, 1, 64) * 1e-42, np.full(64, 1e-45), np.linspace(-7e4, 6e4, 64),
            np.linspace(-1, 1, 64) * 1e30, np.full(64, 3.4e38), np.linspace(-1, 1, 64) * 6e-5, np.linspace(-1, 1, 64) * 4e-7,
            np.where(np.arange(64) == 40, 1000.0, rng.standard_normal(64))]
    return np.asarray(rows).astype(np.float32)


@pytest.mark.parametrize("bits", (4, 8))
def test_blocks_of_odd_values(gpu_ctx, bits):
    x = _odd_blocks()[:, None, :]
    n = len(x)
    p = Paged(bits, 1, 64, 32, [n], [n])
    gpu_ctx.kv_store_batch(p.cache, p.batch, _cuda(x), _cuda(x[::-1]))
    got, want = p.load(gpu_ctx, p.batch, n), stored(x, x[::-1], bits)
    assert np.isfinite(got[0]).all() and np.abs(got[0]).max() <= 65504
    assert same(got[0], want[0]) and same(got[1], want[1])


@pytest.mark.parametrize("bits", (4, 8))
@pytest.mark.parametrize("bad", (np.nan, np.inf, -np.inf))
def test_values_that_are_not_finite(gpu_ctx, bits, bad):
    """One of them anywhere in a head's key or value: its key reads NaN, its
    value 0; other heads and rows are as without it."""
    rng = np.random.default_rng(2)
    k, v = (rng.standard_normal((6, 3, 128)).astype(np.float32) for _ in range(2))
    k[1, 0, 0], k[2, 1, 127], v[3, 2, 31], v[4, 0, 100] = bad, bad, bad, bad
    p = Paged(bits, 3, 128, 32, [6], [40])
    gpu_ctx.kv_store_batch(p.cache, p.batch, _cuda(k), _cuda(v))
    got, want = p.load(gpu_ctx, p.batch, 6), stored(k, v, bits)
    assert same(got[0], want[0]) and same(got[1], want[1])
    for r, h in ((1, 0), (2, 1), (3, 2), (4, 0)):
        assert np.isnan(got[0][r, h]).all() and not got[1][r, h].any()
    assert np.isnan(got[0]).sum() == 4 * 128


def test_far_positions(gpu_ctx):
    """Positions near 2^20 and 2^30 keep their angles (a page table that names
    one page for all of the far ones)."""
    import torch

    import spt

    for pos in ((1 << 20) + 5, (1 << 30) - 1):
        page = 1 << 20
        table = np.zeros((1, -(-(pos + 1) // page)), np.int32)
        n = spt.KVCache.bytes(spt.TYPE_Q8_0, 1, 64, page, 1)
        data = torch.zeros(n, dtype=torch.uint8, device="cuda")
        cache = spt.KVCache.make(spt.TYPE_Q8_0, 1, 64, page, 1, data)
        batch = spt.KVBatch.make(_cuda(np.array([0, 3], np.int32)), _cuda(np.array([pos + 1], np.int32)), _cuda(table), 3, 3, pos + 1)
        rng = np.random.default_rng(1)
        q, k, v = (rng.standard_normal((3, h, 64)).astype(np.float32) for h in (4, 1, 1))
        qd = _cuda(q)
        gpu_ctx.kv_store_batch(cache, batch, _cuda(k), _cuda(v), rope=spt.Rope(**YARN), q=qd, q_out=qd)
        at = np.arange(pos - 2, pos + 1)
        # the angle pos * f is rounded to 2^-53 of itself on both sides, with an f that may differ by 2^-52 of itself
        tol = 2.0 ** -24 + 4 * 2.0 ** -53 * pos
        assert np.abs(qd.cpu().numpy() - rotate(q, at, YARN)).max() <= 8 * tol
        kk, vv = torch.empty(3, 1, 64, device="cuda"), torch.empty(3, 1, 64, device="cuda")
        gpu_ctx.kv_load_batch(cache, batch, kk, vv)
        want = stored(rotate(k, at, YARN), v, 8)
        step = np.abs(rotate(k, at, YARN)).max() / 127
        assert np.abs(kk.cpu().numpy() - want[0]).max() <= 1.001 * step  # a code next to a border
        assert same(vv.cpu().numpy(), want[1])


def test_what_a_batch_says_is_not_trusted(gpu_ctx):
    """Pages that are none, rows outside the buffers, more rows than positions,
    sequences longer than declared: nothing out of place is written, and it
    reads as NaN."""
    import torch

    p = Paged(4, 2, 64, 32, [4, 4, 4, 4], [64, 40, 2, 36], extra_rows=3)
    n = p.n_rows
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((n, 2, 64)).astype(np.float32) for _ in range(2))
    kd, vd = _cuda(k), _cuda(v)
    table = p.table.copy()
    table[0, 1], table[1, 1] = -3, p.n_pages  # the pages of the new rows
    before = p.data.clone()

    def call(starts, lens, max_new, max_len, table, rows=n):
        b = p.make_batch(starts, lens, max_new, max_len, n_rows=rows, table=table)
        gpu_ctx.kv_store_batch(p.cache, b, kd[:rows], vd[:rows])
        out = [torch.full((rows, 2, 64), 7.0, device="cuda") for _ in range(2)]
        gpu_ctx.kv_load_batch(p.cache, b, *out)
        return [x.cpu().numpy() for x in out]

    got = call(p.starts, p.lens, 4, 64, table)
    want = stored(k, v, 4)
    for g, w in zip(got, want):
        assert np.isnan(g[:8]).all()                       # no page
        assert np.isnan(g[8:10]).all()                     # before the first position
        assert same(g[10:16], w[10:16])                    # sequence 2's two positions, sequence 3
        assert (g[16:] == 7.0).all()                       # rows of no sequence
    per = p.data.numel() // p.n_pages
    changed = (p.data != before).reshape(p.n_pages, per).any(1).nonzero().ravel().tolist()
    assert sorted(changed) == sorted([p.table[2, 0], p.table[3, 1]])

    for starts, lens, max_new, max_len in (
            ([0, 4, 8, 12, 16], [64, 40, 2, 65], 4, 64),       # longer than declared
            ([0, 4, 8, 12, 16], [64, 40, 2, 2 ** 31 - 1], 4, 64),
            ([0, 1, 2, 3, 19], [64, 40, 2, 36], 4, 64),        # more rows than declared
            ([0, 1, 2, 3, 2 ** 31 - 1], [64, 40, 2, 36], 4, 64)):
        p.data.copy_(before)
        got = call(starts, lens, max_new, max_len, np.full_like(table, table[3, 1]))
        a = starts[3]
        assert np.isnan(got[0][a:a + 4]).all() and np.isnan(got[1][a:a + 4]).all()
        assert (got[0][a + 4:] == 7.0).all()
    # rows outside the buffers, running backwards, negative
    for starts in ([-5, -2, 1, 0, 40], [30, 20, 10, 5, 2], [-(2 ** 31), 2 ** 31 - 1, -1, 2 ** 31 - 1, -7]):
        call(starts, [8, 8, 8, 8], 4, 64, p.table)
    call(p.starts, [-5, 0, -(2 ** 31), 0], 4, 64, p.table)


def test_other_stream(gpu_ctx):
    """A context on a stream of its own, beside work on torch's current one."""
    import torch

    import spt

    stream = torch.cuda.Stream()
    ctx = spt.Context(0, stream.cuda_stream)
    try:
        p = Paged(8, 2, 64, 32, [50], [50])
        x = p.rng.standard_normal((50, 2, 64)).astype(np.float32)
        xd = _cuda(x)
        torch.cuda.synchronize()
        ctx.kv_store_batch(p.cache, p.batch, xd, xd)
        out = [torch.empty(50, 2, 64, device="cuda") for _ in range(2)]
        ctx.kv_load_batch(p.cache, p.batch, *out)
        ctx.synchronize()
        want = stored(x, x, 8)
        assert same(out[0].cpu().numpy(), want[0]) and same(out[1].cpu().numpy(), want[1])
    finally:
        ctx.close()


def test_cancel_flag(gpu_ctx):
    import spt

    p = Paged(4, 1, 64, 32, [1], [1])
    x = _cuda(np.ones((1, 1, 64), np.float32))
    before = p.data.clone()
    flag = np.array([1], np.int32)
    gpu_ctx.set_cancel_flag(flag)
    try:
        for call in (lambda: gpu_ctx.kv_store_batch(p.cache, p.batch, x, x), lambda: gpu_ctx.kv_load_batch(p.cache, p.batch, x, x.clone())):
            with pytest.raises(spt.SptError) as e:
                call()
            assert e.value.code == spt.ERR_CANCELED
    finally:
        gpu_ctx.set_cancel_flag(None)
    assert bool((p.data == before).all())
