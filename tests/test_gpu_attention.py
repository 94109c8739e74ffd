"""Attention over the quantized cache on the device, against the formula in 64
bits on the values that the cache holds, at the sizes, masks and memory where
it can go wrong; and the layer's attention as its operators run together."""
import numpy as np
import pytest

from kv_reference import YARN, attend, rotate, stored
from test_gpu_kv_cache import Paged, _cuda, same

pytestmark = pytest.mark.gpu


class Filled(Paged):
    """A cache whose sequences hold random keys and values; k, v: what they read back as."""

    def __init__(self, ctx, bits, kv, dim, page, new, lens, seed=0, peak=2.0, **kw):
        super().__init__(bits, kv, dim, page, new, lens, seed=seed, **kw)
        self.data.fill_(0xFF)  # NaN scales wherever nothing is stored
        b, starts, n = self.whole()
        k = (self.rng.standard_normal((n, kv, dim)) * peak).astype(np.float32)
        v = self.rng.standard_normal((n, kv, dim)).astype(np.float32)
        ctx.kv_store_batch(self.cache, b, _cuda(k), _cuda(v))
        k, v = stored(k, v, bits)
        self.k = [k[a:b] for a, b in zip(starts[:-1], starts[1:])]
        self.v = [v[a:b] for a, b in zip(starts[:-1], starts[1:])]

    def want(self, q, scale, window=0, sinks=None):
        out, tol = np.full(q.shape, 9.0), np.zeros(q.shape)
        for s, (a, b) in enumerate(zip(self.starts[:-1], self.starts[1:])):
            out[a:b], tol[a:b] = attend(q[a:b], self.k[s], self.v[s], self.lens[s] - (b - a), scale, window, sinks)
        return out, tol


def run(ctx, p, q, scale, window=0, sinks=None, batch=None, q8=False, work=False, typ=None):
    import torch

    import spt

    qd = _cuda(q)
    out = torch.full_like(qd, 9.0)
    blocks = torch.full((q.size // 32 * 34,), 0xAA, dtype=torch.uint8, device="cuda") if q8 else None
    sk = None
    if sinks is not None:
        sd = _cuda(np.asarray(sinks, np.float32))
        sd = sd if typ is None else sd.to(typ)
        code = {4: spt.TYPE_F32, 2: spt.TYPE_F16 if sd.dtype == torch.float16 else spt.TYPE_BF16}[sd.element_size()]
        sk = spt.Tensor.make("attn_sinks", code, [len(sinks)], sd.data_ptr(), sd.numel() * sd.element_size())
    w = None
    if work:
        n = ctx.attention_work_bytes(p.cache, batch or p.batch, q.shape[1], window)
        w = torch.full((max(16, n),), 0xFF, dtype=torch.uint8, device="cuda")
    ctx.attention_batch_into(p.cache, batch or p.batch, qd, out, scale, window=window, sinks=sk, q8=blocks, work=w)
    torch.cuda.synchronize()
    return (out.cpu().numpy(), blocks) if q8 else out.cpu().numpy()


def check(got, want, tol):
    assert np.isfinite(got).all()
    far = np.abs(got - want)
    assert (far <= tol).all(), f"off by {far.max():.3g}, {(far / np.maximum(tol, 1e-30)).max():.3g} of what it may"
    # roundings are independent: over all outputs they come nowhere near their sum
    norm = np.linalg.norm(want)
    if want.size >= 256 and norm:
        assert np.linalg.norm(got - want) <= 1e-5 * norm


@pytest.mark.parametrize("bits", (4, 8))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("kv,group,page,new,lens,window,sinks", [
    (1, 1, 32, [1], [1], 0, False),
    (1, 1, 32, [1], [1], 1, True),
    (2, 8, 32, [1], [31], 0, True),
    (2, 8, 32, [1], [32], 0, False),
    (2, 8, 64, [1], [33], 0, True),
    (2, 8, 64, [1, 1, 1], [65, 400, 7], 0, True),
    (2, 8, 32, [1, 1, 1], [65, 400, 7], 128, True),
    (1, 3, 32, [1, 1], [500, 33], 33, False),
    (2, 5, 96, [2, 1, 4], [96, 97, 95], 0, True),
    (1, 16, 32, [3], [70], 0, False),
    (1, 17, 32, [3], [70], 40, True),
    (2, 8, 64, [32], [32], 0, True),
    (2, 8, 64, [33], [100], 0, True),
    (1, 8, 32, [70], [70], 16, False),
    (1, 8, 32, [70, 5, 0, 64], [70, 300, 9, 64], 1, True),
    (2, 4, 128, [129, 40], [129, 300], 100, True),
    (1, 1, 32, [200], [200], 0, False),
    (1, 40, 32, [17], [49], 0, True),
])
def test_against_the_formula(gpu_ctx, bits, dim, kv, group, page, new, lens, window, sinks):
    p = Filled(gpu_ctx, bits, kv, dim, page, new, lens, seed=group, peak=6.0 / np.sqrt(dim) * 2)
    q = p.rng.standard_normal((p.n_rows, kv * group, dim)).astype(np.float32)
    sk = (p.rng.standard_normal(kv * group) * 2).astype(np.float32) if sinks else None
    scale = dim ** -0.5
    got = run(gpu_ctx, p, q, scale, window, sk)
    check(got, *p.want(q, scale, window, sk))
    assert np.array_equal(got, run(gpu_ctx, p, q, scale, window, sk, work=True))


@pytest.mark.parametrize("bits,dim,kv,group,new,lens,window", [
    (4, 64, 1, 8, [1], [20001], 0),
    (8, 128, 1, 5, [1], [9000], 0),
    (4, 64, 2, 8, [1, 2, 1], [5000, 3000, 17], 0),
    (4, 128, 1, 4, [40], [6000], 0),
    (8, 64, 1, 8, [33], [7000], 5000),
    (4, 64, 1, 8, [150, 3], [4000, 2001], 0),
])
def test_long_sequences(gpu_ctx, bits, dim, kv, group, new, lens, window):
    """Positions split over workgroups; the same with and without a workspace
    of the caller's, and twice."""
    p = Filled(gpu_ctx, bits, kv, dim, 64, new, lens, seed=3)
    q = p.rng.standard_normal((p.n_rows, kv * group, dim)).astype(np.float32) * 1.5
    sk = p.rng.standard_normal(kv * group).astype(np.float32)
    # (the last case's row tiles fill the compute units whole)
    assert (gpu_ctx.attention_work_bytes(p.cache, p.batch, kv * group, window) > 0) == (max(new) < 150)
    got = run(gpu_ctx, p, q, dim ** -0.5, window, sk)
    check(got, *p.want(q, dim ** -0.5, window, sk))
    for work in (True, False):
        assert np.array_equal(got, run(gpu_ctx, p, q, dim ** -0.5, window, sk, work=work))


@pytest.mark.parametrize("bits,dim,kv,group,new,bound", [
    (4, 64, 4, 8, 1, 20000), (8, 128, 4, 5, 1, 20000), (4, 128, 2, 8, 3, 9000), (8, 64, 2, 16, 2, 9000), (4, 64, 1, 3, 1, 64000)])
def test_shares_of_unequal_sequences(gpu_ctx, bits, dim, kv, group, new, bound):
    """33 sequences, most short or of nothing, for which the bounds allow far more: shares that
    begin and end in units, whole units, several a share."""
    lens = [3000, 1700, 0, 640] + [new + 7 * i for i in range(29)]
    news = [new, new, 0] + [new] * 30
    p = Filled(gpu_ctx, bits, kv, dim, 32, news, lens, seed=bits)
    table = np.full((33, -(-bound // 32)), -1, np.int32)
    table[:, :p.table.shape[1]] = p.table
    q = p.rng.standard_normal((p.n_rows, kv * group, dim)).astype(np.float32)
    sk = p.rng.standard_normal(kv * group).astype(np.float32)
    b = p.make_batch(p.starts, p.lens, new, bound, table=table)
    assert gpu_ctx.attention_work_bytes(p.cache, b, kv * group) > 0
    got = run(gpu_ctx, p, q, dim ** -0.5, 0, sk, batch=b)
    check(got, *p.want(q, dim ** -0.5, 0, sk))
    for work in (True, False):
        assert np.array_equal(got, run(gpu_ctx, p, q, dim ** -0.5, 0, sk, batch=b, work=work))


@pytest.mark.parametrize("bits,new", [(4, [64]), (8, [3, 64])])
def test_shares_of_many_rows(gpu_ctx, bits, new):
    """128 rows at a time of few heads of 128, for which the bounds allow far more positions."""
    kv, group, bound = 4, 16, 32000
    lens = [700, 100][:len(new)]
    p = Filled(gpu_ctx, bits, kv, 128, 32, new, lens, seed=bits, peak=12.0 / np.sqrt(128))
    table = np.full((len(new), -(-bound // 32)), -1, np.int32)
    table[:, :p.table.shape[1]] = p.table
    q = p.rng.standard_normal((p.n_rows, kv * group, 128)).astype(np.float32)
    sk = p.rng.standard_normal(kv * group).astype(np.float32)
    b = p.make_batch(p.starts, p.lens, 64, bound, table=table)
    n = gpu_ctx.attention_work_bytes(p.cache, b, kv * group)
    assert n > 0
    got = run(gpu_ctx, p, q, 128 ** -0.5, 0, sk, batch=b)
    check(got, *p.want(q, 128 ** -0.5, 0, sk))
    assert np.array_equal(got, run(gpu_ctx, p, q, 128 ** -0.5, 0, sk, batch=b, work=True))


@pytest.mark.parametrize("bits,dim,group,new,window", [(4, 64, 4, 1, 0), (8, 64, 5, 3, 40), (4, 128, 3, 5, 0), (8, 128, 8, 1, 33)])
def test_more_units_than_fit_at_once(gpu_ctx, bits, dim, group, new, window):
    """Many heads and sequences: workgroups of fewer waves."""
    kv = 130
    p = Filled(gpu_ctx, bits, kv, dim, 32, [new, 0, new, new, new], [new, 40, 33, 161, 70], seed=group, peak=12.0 / np.sqrt(dim), extra_rows=1)
    q = p.rng.standard_normal((p.n_rows, kv * group, dim)).astype(np.float32)
    sk = (p.rng.standard_normal(kv * group) * 2).astype(np.float32)
    got = run(gpu_ctx, p, q, dim ** -0.5, window, sk)
    check(got, *p.want(q, dim ** -0.5, window, sk))
    assert (got[-1] == 9.0).all()
    table = p.table.copy()
    table[3, 4] = -1  # positions 128 .. 159
    got2 = run(gpu_ctx, p, q, dim ** -0.5, window, sk, batch=p.make_batch(p.starts, p.lens, new, 161, table=table))
    bad = np.zeros(p.n_rows, bool)
    bad[2 * new:3 * new] = True
    assert np.isnan(got2[bad]).all() and np.array_equal(got2[~bad], got[~bad])


@pytest.mark.parametrize("new", (1, 3))
@pytest.mark.parametrize("bound", (6000, 400000))
def test_parts_that_cannot_see(gpu_ctx, new, bound):
    """Sequences cut into parts, by their own and by equal shares: a page that is none in one
    part makes the row NaN, sequences of nothing and too long ones are as when whole."""
    lens = [5000, 0, 2600, 40]
    p = Filled(gpu_ctx, 4, 1, 64, 32, [new, 0, new, new], lens, seed=4)
    table = np.full((4, -(-bound // 32)), -1, np.int32)
    table[:, :p.table.shape[1]] = p.table
    q = p.rng.standard_normal((p.n_rows, 8, 64)).astype(np.float32)
    want, tol = p.want(q, 0.125)
    starts = np.array([0, new, 2 * new, 3 * new, 3 * new], np.int32)
    for page in (0, 80, 5000 // 32):  # the first, one within, the last
        t = table[[0, 2, 3, 1]].copy()
        t[0, page] = p.n_pages
        got = run(gpu_ctx, p, q, 0.125, batch=p.make_batch(starts, [5000, 2600, 40, 0], new, bound, table=t))
        bad = np.arange(5000 - new, 5000) >= 32 * page
        assert np.isnan(got[:new][bad]).all()
        good = np.concatenate([~bad, np.ones(2 * new, bool)])
        assert (np.abs(got - want) <= tol)[good].all()
    t = table[[0, 2, 3, 1]]
    got = run(gpu_ctx, p, q, 0.125, batch=p.make_batch(starts, [bound + 1, -5, 40, bound], new, bound, table=t))
    assert np.isnan(got[:new]).all() and (got[new:2 * new] == 0).all()
    assert (np.abs(got - want) <= tol)[2 * new:].all()


# Many rows a head, 128 at a time: a workgroup a row tile where there are many, shares of few long ones.
MANY = [
    (4, 64, 64, 4, [140, 133], [140, 300], 0, True),
    (8, 64, 130, 4, [130, 0], [130, 9], 37, False),
    (4, 128, 64, 3, [86, 171], [90, 171], 0, False),
    (8, 128, 32, 16, [49, 50, 17, 1], [49, 177, 17, 260], 20, True),
    (8, 128, 16, 16, [65], [65], 0, True),
    (4, 64, 1, 17, [31, 40], [3333, 40], 0, True),
    (8, 128, 1, 8, [65], [4000], 0, False),
    (8, 64, 1, 8, [65, 1], [4000, 5000], 3500, True),
]


@pytest.mark.parametrize("bits,dim,kv,group,new,lens,window,sinks", MANY)
def test_many_rows(gpu_ctx, bits, dim, kv, group, new, lens, window, sinks):
    p = Filled(gpu_ctx, bits, kv, dim, 32, new, lens, seed=kv, peak=12.0 / np.sqrt(dim), extra_rows=1)
    q = p.rng.standard_normal((p.n_rows, kv * group, dim)).astype(np.float32)
    sk = (p.rng.standard_normal(kv * group) * 2).astype(np.float32) if sinks else None
    got, blocks = run(gpu_ctx, p, q, dim ** -0.5, window, sk, q8=True)
    check(got, *p.want(q, dim ** -0.5, window, sk))
    assert (got[-1] == 9.0).all()
    import torch

    n = sum(new) * kv * group * dim
    blk = torch.empty(n // 32 * 34, dtype=torch.uint8, device="cuda")
    gpu_ctx.quantize_q8_0(_cuda(got[:sum(new)]), blk)
    assert torch.equal(blocks[:blk.numel()], blk) and bool((blocks[blk.numel():] == 0xAA).all())


def test_many_rows_that_cannot_see(gpu_ctx):
    """Marked keys, pages that are none and rows before the first position, 128 rows at a time."""
    kv, new = 130, 67
    p = Filled(gpu_ctx, 4, kv, 64, 32, [new, new], [100, 40])
    b, starts, n = p.whole()
    k, v = (p.rng.standard_normal((n, kv, 64)).astype(np.float32) for _ in range(2))
    k[50, 3, 1] = np.nan
    gpu_ctx.kv_store_batch(p.cache, b, _cuda(k), _cuda(v))
    ks, vs = stored(k, v, 4)
    p.k, p.v = [ks[:100], ks[100:]], [vs[:100], vs[100:]]
    q = p.rng.standard_normal((2 * new, kv * 8, 64)).astype(np.float32)
    table = p.table.copy()
    table[0, 2] = -1  # positions 64 .. 95
    got = run(gpu_ctx, p, q, 0.125, batch=p.make_batch(p.starts, p.lens, new, 100, table=table))
    pos = np.arange(100 - new, 100)
    bad = np.repeat((pos >= 64)[:, None], kv * 8, 1)
    bad[pos >= 50, 24:32] = True
    assert np.array_equal(np.isnan(got[:new]).all(-1), bad) and np.array_equal(np.isnan(got[:new]).any(-1), bad)
    want, tol = p.want(q, 0.125)
    assert (np.abs(got[:new] - want[:new])[~bad] <= tol[:new][~bad]).all()
    assert (got[new:2 * new - 40] == 0).all()
    assert (np.abs(got[new:] - want[new:]) <= tol[new:]).all()


@pytest.mark.parametrize("bits,kv,new,window,length", [(4, 1, 1, 20, 90), (8, 1, 4, 20, 90), (4, 1, 40, 9, 90), (4, 130, 129, 5, 200), (8, 2, 129, 3100, 4000)])
def test_only_the_window_was_stored(gpu_ctx, bits, kv, new, window, length):
    """Positions that no row sees hold anything (scales of NaN), in the same
    tiles as those that rows see: before the window and behind the end."""
    p = Paged(bits, kv, 64, 64, [new], [length], seed=2)
    p.data.fill_(0xFF)
    n = min(length, new + window - 1)
    k, v = (p.rng.standard_normal((n, kv, 64)).astype(np.float32) for _ in range(2))
    gpu_ctx.kv_store_batch(p.cache, p.make_batch([0, n], [length], n, length, n_rows=n), _cuda(k), _cuda(v))
    ks, vs = stored(k, v, bits)
    full = np.zeros((length, kv, 64), np.float32), np.zeros((length, kv, 64), np.float32)
    full[0][length - n:], full[1][length - n:] = ks, vs
    q = p.rng.standard_normal((new, kv * 4, 64)).astype(np.float32)
    check(run(gpu_ctx, p, q, 0.125, window), *attend(q, *full, length - new, 0.125, window))


def test_rows_of_a_batch_are_independent(gpu_ctx):
    """A sequence's rows have the same bits alone and beside others."""
    p = Filled(gpu_ctx, 4, 2, 64, 32, [3, 50, 1], [40, 50, 333], seed=8)
    q = p.rng.standard_normal((p.n_rows, 16, 64)).astype(np.float32)
    got = run(gpu_ctx, p, q, 0.125)
    lens, starts = p.lens.copy(), p.starts.copy()
    for s in range(3):
        only = lens.copy()
        rows = np.zeros(4, np.int32)
        rows[:s + 1], rows[s + 1:] = starts[s], starts[s + 1]
        b = p.make_batch(rows, only, 50, 333)
        alone = run(gpu_ctx, p, q, 0.125, batch=b)
        assert np.array_equal(alone[starts[s]:starts[s + 1]], got[starts[s]:starts[s + 1]])
        rest = np.ones(p.n_rows, bool)
        rest[starts[s]:starts[s + 1]] = False
        assert (alone[rest] == 9.0).all()


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
def test_sinks_of_16_bits(gpu_ctx, dtype):
    import torch

    p = Filled(gpu_ctx, 4, 1, 64, 32, [2], [50])
    q = p.rng.standard_normal((2, 7, 64)).astype(np.float32)
    sk = torch.from_numpy(p.rng.standard_normal(7).astype(np.float32)).to(getattr(torch, dtype))
    check(run(gpu_ctx, p, q, 0.125, 0, sk.float().numpy(), typ=sk.dtype), *p.want(q, 0.125, 0, sk.float().numpy()))


@pytest.mark.parametrize("new", (1, 40))
def test_sinks_at_the_ends(gpu_ctx, new):
    """A sink of -inf counts nothing, one far above every score takes all, one
    at the type's lowest is as none."""
    p = Filled(gpu_ctx, 8, 1, 64, 32, [new], [60])
    q = p.rng.standard_normal((new, 4, 64)).astype(np.float32)
    none = run(gpu_ctx, p, q, 0.125)
    got = run(gpu_ctx, p, q, 0.125, 0, [-np.inf, np.finfo(np.float32).min, 200.0, 1e30])
    # with and without a sink of weight 0 the division is the same
    assert np.array_equal(got[:, :2], none[:, :2])
    assert np.abs(got[:, 2]).max() < 1e-30 and (got[:, 3] == 0).all()
    assert np.isnan(run(gpu_ctx, p, q, 0.125, 0, [np.nan, 0.0, 0.0, 0.0])[:, 0]).all()


@pytest.mark.parametrize("new", (1, 40))
@pytest.mark.parametrize("factor", (1e-30, 1e-3, 1e3, 1e18))
def test_queries_of_any_size(gpu_ctx, new, factor):
    """Tiny queries attend evenly, huge ones to the largest score alone."""
    p = Filled(gpu_ctx, 4, 1, 64, 32, [new], [100])
    q = (p.rng.standard_normal((new, 8, 64)) * factor).astype(np.float32)
    got = run(gpu_ctx, p, q, 0.125)
    want, tol = p.want(q, 0.125)
    if factor <= 1:
        check(got, want, tol)
    else:  # two scores further apart than rounding: the weights are 0 and 1
        clear = np.zeros(q.shape[:2], bool)
        for i in range(new):
            s = np.sort(np.einsum("hd,jd->hj", q[i].astype(np.float64), p.k[0][:101 - new + i, 0].astype(np.float64)) * 0.125, axis=1)
            clear[i] = s[:, -1] - s[:, -2] > 100 + 1e-4 * np.abs(s).max()
        assert clear.mean() > 0.2 and np.isfinite(got).all()
        assert np.abs(got - want)[clear].max() <= 2.0 ** -22 * np.abs(want[clear]).max()


@pytest.mark.parametrize("new", (1, 40))
@pytest.mark.parametrize("bits,size", [(4, 3e4), (8, 6e4), (4, 2e-6), (8, 1e-5), (4, 1e-3)])
def test_values_of_any_size(gpu_ctx, new, bits, size):
    """Values near the ends of the scales' range are weighed at the same accuracy."""
    p = Filled(gpu_ctx, bits, 1, 64, 32, [new], [90])
    b, _, n = p.whole()
    k = p.rng.standard_normal((n, 1, 64)).astype(np.float32)
    v = (p.rng.uniform(-1, 1, (n, 1, 64)) * size).astype(np.float32)
    gpu_ctx.kv_store_batch(p.cache, b, _cuda(k), _cuda(v))
    p.k[0], p.v[0] = stored(k, v, bits)
    q = p.rng.standard_normal((new, 8, 64)).astype(np.float32)
    check(run(gpu_ctx, p, q, 0.125), *p.want(q, 0.125))


@pytest.mark.parametrize("new", (1, 3, 40))
@pytest.mark.parametrize("window", (0, 20))
def test_keys_and_values_that_are_not_finite(gpu_ctx, new, window):
    """Rows that see a marked position are NaN, the others as without it."""
    p = Filled(gpu_ctx, 4, 2, 64, 32, [new], [100])
    b, _, n = p.whole()
    k, v = (p.rng.standard_normal((n, 2, 64)).astype(np.float32) for _ in range(2))
    at = [100 - new // 2 - 1, 70, 3]
    k[at[0], 0, 5], v[at[1], 1, 60], k[at[2], 1, 0] = np.nan, np.inf, -np.inf
    gpu_ctx.kv_store_batch(p.cache, b, _cuda(k), _cuda(v))
    p.k[0], p.v[0] = stored(k, v, 4)
    q = p.rng.standard_normal((new, 6, 64)).astype(np.float32)
    got = run(gpu_ctx, p, q, 0.125, window)
    pos = np.arange(100 - new, 100)
    sees = lambda j: (pos >= j) & (pos - j < (window or 1000))  # noqa: E731
    bad = np.stack([sees(at[0])] * 3 + [sees(at[1]) | sees(at[2])] * 3, 1)
    assert np.array_equal(np.isnan(got).any(-1), bad) and np.array_equal(np.isnan(got).all(-1), bad)
    want, tol = p.want(q, 0.125, window)
    good = ~bad
    assert (np.abs(got - want)[good] <= tol[good]).all()


@pytest.mark.parametrize("new", (1, 40))
def test_queries_that_are_not_finite(gpu_ctx, new):
    p = Filled(gpu_ctx, 4, 1, 64, 32, [new], [50])
    q = p.rng.standard_normal((new, 4, 64)).astype(np.float32)
    want, tol = p.want(q, 0.125)
    q[0, 1, 7], q[new - 1, 2, 63] = np.nan, np.inf
    got = run(gpu_ctx, p, q, 0.125)
    bad = np.zeros((new, 4), bool)
    bad[0, 1] = bad[new - 1, 2] = True
    assert np.isnan(got[bad]).all()
    assert (np.abs(got - want)[~bad] <= tol[~bad]).all()


@pytest.mark.parametrize("new", (4, 40))
def test_what_a_batch_says_is_not_trusted(gpu_ctx, new):
    """Sequences of more rows than positions, of nothing, too long, with pages
    that are none: zeros where nothing is seen, NaN where it cannot be."""
    p = Filled(gpu_ctx, 4, 1, 64, 32, [new] * 4, [100, 70, 64, 90], extra_rows=2)
    q = p.rng.standard_normal((p.n_rows, 8, 64)).astype(np.float32)
    want, tol = p.want(q, 0.125)
    part = lambda x, s: x[s * new:(s + 1) * new]  # noqa: E731

    table = p.table.copy()
    table[0, 0], table[1, 1], table[3, 2] = -1, p.n_pages, 2 ** 31 - 1
    got = run(gpu_ctx, p, q, 0.125, batch=p.make_batch(p.starts, p.lens, new, 100, table=table))
    first = 70 - new
    sees = np.arange(first, 70) >= 32
    assert np.isnan(part(got, 0)).all() and np.isnan(part(got, 1)[sees]).all()
    assert (np.abs(part(got, 1) - part(want, 1))[~sees] <= part(tol, 1)[~sees]).all()
    assert (np.abs(part(got, 2) - part(want, 2)) <= part(tol, 2)).all()
    assert np.array_equal(np.isnan(part(got, 3)).all((1, 2)), np.arange(90 - new, 90) >= 64)
    assert (got[4 * new:] == 9.0).all()
    # freed pages before a window are never looked at
    got = run(gpu_ctx, p, q, 0.125, 5, batch=p.make_batch(p.starts, p.lens, new, 100, table=table))
    w, t = p.want(q, 0.125, 5)
    assert (np.abs(part(got, 0) - part(w, 0)) <= part(t, 0)).all() or new == 40

    for lens, max_len in (([0, -3, 2, 90], 100), ([101, 2 ** 31 - 1, 64, 90], 100)):
        got = run(gpu_ctx, p, q, 0.125, batch=p.make_batch(p.starts, lens, new, max_len))
        for s in range(3):
            if lens[s] > max_len:
                assert np.isnan(part(got, s)).all()
            elif lens[s] <= 2:
                assert (part(got, s)[:new - max(0, lens[s])] == 0).all() and np.isfinite(part(got, s)).all()
        assert (np.abs(part(got, 3) - part(want, 3)) <= part(tol, 3)).all()
        assert (got[4 * new:] == 9.0).all()
    # more rows than declared: the declared ones are NaN, the others untouched
    got = run(gpu_ctx, p, q, 0.125, batch=p.make_batch([0, 1, 2, 3, 4 * new], p.lens, 3, 100))
    assert np.isnan(got[3:6]).all() and (got[6:] == 9.0).all()
    for starts in ([-5, -2, 1, 0, 400], [30, 20, 10, 5, 2], [-(2 ** 31), 2 ** 31 - 1, -1, 2 ** 31 - 1, -7]):
        run(gpu_ctx, p, q, 0.125, batch=p.make_batch(starts, p.lens, new, 100))


@pytest.mark.parametrize("dim,new", [(64, 1), (128, 5), (64, 40)])
def test_blocks_of_the_output(gpu_ctx, dim, new):
    """q8: the blocks that spt_quantize_q8_0 makes of the output, byte for
    byte; those of rows of no sequence are left as they were."""
    import torch

    p = Filled(gpu_ctx, 4, 2, dim, 32, [new, new], [50, 3000], extra_rows=1)
    q = p.rng.standard_normal((p.n_rows, 6, dim)).astype(np.float32)
    got, blocks = run(gpu_ctx, p, q, dim ** -0.5, q8=True)
    assert np.array_equal(got, run(gpu_ctx, p, q, dim ** -0.5))
    n = 2 * new * 6 * dim
    want = torch.empty(n // 32 * 34, dtype=torch.uint8, device="cuda")
    gpu_ctx.quantize_q8_0(_cuda(got[:2 * new]), want)
    assert torch.equal(blocks[:want.numel()], want) and bool((blocks[want.numel():] == 0xAA).all())


def test_no_rows(gpu_ctx):
    import torch

    import spt

    p = Filled(gpu_ctx, 4, 1, 64, 32, [0, 0], [5, 40], extra_rows=3)
    q = p.rng.standard_normal((3, 2, 64)).astype(np.float32)
    assert (run(gpu_ctx, p, q, 0.125) == 9.0).all()
    empty = torch.empty(0, 2, 64, device="cuda")
    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    b = spt.KVBatch.make(z[:1], z[:0], z[:0].reshape(0, 1), 0, 1, 1)
    with pytest.raises(spt.SptError):  # nil arrays
        gpu_ctx.attention_batch_into(p.cache, b, empty, empty, 0.125)
    b = spt.KVBatch.make(z[:2], z[:1], torch.from_numpy(p.table[:1]).cuda(), 0, 1, 1)
    gpu_ctx.attention_batch_into(p.cache, b, empty, empty, 0.125)
    gpu_ctx.kv_store_batch(p.cache, b, empty, empty)
    gpu_ctx.kv_load_batch(p.cache, b, empty, empty)


def test_far_into_a_large_cache(gpu_ctx):
    """Pages that begin beyond 2^32 bytes."""
    import torch

    import spt

    page, n_pages = 4096, 7400  # 4.4 GB
    n = spt.KVCache.bytes(spt.TYPE_Q4_0, 2, 64, page, n_pages)
    assert n > 1 << 32
    data = torch.empty(n, dtype=torch.uint8, device="cuda")
    p = Filled(gpu_ctx, 4, 2, 64, 4096, [3], [5000])
    cache = spt.KVCache.make(spt.TYPE_Q4_0, 2, 64, page, n_pages, data)
    per = n // n_pages
    for i, to in enumerate((n_pages - 1, n_pages - 3)):
        src = int(p.table[0, i])
        data[to * per:(to + 1) * per] = p.data[src * per:(src + 1) * per]
    q = p.rng.standard_normal((3, 16, 64)).astype(np.float32)
    want = run(gpu_ctx, p, q, 0.125)
    batch = p.make_batch(p.starts, p.lens, 3, 5000, table=np.array([[n_pages - 1, n_pages - 3]], np.int32))
    p.cache = cache
    assert np.array_equal(run(gpu_ctx, p, q, 0.125, batch=batch), want)
    x = _cuda(p.rng.standard_normal((3, 2, 64)).astype(np.float32))
    gpu_ctx.kv_store_batch(cache, batch, x, x)
    k, v = p.load(gpu_ctx, batch, 3)
    want = stored(x.cpu().numpy(), x.cpu().numpy(), 4)
    assert same(k, want[0]) and same(v, want[1])


@pytest.mark.parametrize("new,lens", [([1, 1], [40, 4000]), ([64, 3], [64, 300])])
def test_in_a_graph(new, lens):
    """Store and attention captured with a workspace of their own, replayed
    with other lengths, pages and rows in the batch's arrays, with eager calls
    that grow the context's arena between the replays."""
    import torch

    import spt

    stream = torch.cuda.Stream()
    ctx = spt.Context(0, stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            p = Filled(ctx, 4, 2, 64, 32, new, lens, seed=5)
            other = Filled(ctx, 4, 2, 64, 32, [2], [9000], seed=6)
            n = p.n_rows
            q, k, v = (_cuda(p.rng.standard_normal((n, h, 64)).astype(np.float32)) for h in (8, 2, 2))
            qr, out = torch.empty_like(q), torch.empty_like(q)
            work = torch.empty(max(16, ctx.attention_work_bytes(p.cache, p.batch, 8)), dtype=torch.uint8, device="cuda")
            rope = spt.Rope(**YARN)

            def step(o, w):
                ctx.kv_store_batch(p.cache, p.batch, k, v, rope=rope, q=q, q_out=qr)
                ctx.attention_batch_into(p.cache, p.batch, qr, o, 0.125, work=w)

            step(out, work)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(out, work)
            rows_dev, lens_dev, pages_dev = p.batch._keep
            for i in range(4):
                for x in (q, k, v):
                    x.normal_()
                lens_dev.copy_(torch.tensor([max(b, x - 7 * i) for b, x in zip(new, lens)]))
                out.fill_(9.0)
                graph.replay()
                stream.synchronize()
                got = out.clone()
                step(out, None)
                stream.synchronize()
                assert torch.equal(got, out)
                run(ctx, other, other.rng.standard_normal((2, 8 * (i + 1), 64)).astype(np.float32), 0.125)
                stream.synchronize()
            del graph
    finally:
        ctx.close()


def test_a_captured_call_without_a_workspace():
    """Refused where it needs one (the arena may move before a replay), and
    the capture goes on; taken where it needs none."""
    import torch

    import spt

    stream = torch.cuda.Stream()
    ctx = spt.Context(0, stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            p, short = (Filled(ctx, 4, 2, 64, 32, [1], [n], seed=n) for n in (9000, 50))
            q = _cuda(p.rng.standard_normal((1, 16, 64)).astype(np.float32))
            assert ctx.attention_work_bytes(p.cache, p.batch, 16) > 0 == ctx.attention_work_bytes(short.cache, short.batch, 16)
            out, eager = torch.full_like(q, 9.0), torch.empty_like(q)
            ctx.attention_batch_into(p.cache, p.batch, q, eager, 0.125)  # the arena is large enough
            ctx.attention_batch_into(short.cache, short.batch, q, eager, 0.125)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                with pytest.raises(spt.SptError) as e:
                    ctx.attention_batch_into(p.cache, p.batch, q, out, 0.125)
                assert e.value.code == spt.ERR_INVALID
                ctx.attention_batch_into(short.cache, short.batch, q, out, 0.125)
            for _ in range(3):
                out.fill_(9.0)
                graph.replay()
                stream.synchronize()
                assert torch.equal(out, eager)
            del graph
    finally:
        ctx.close()


def test_two_contexts_at_once():
    """Calls on two streams at once, each with its own context's arena."""
    import torch

    import spt

    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [spt.Context(0, s.cuda_stream) for s in streams]
    try:
        ps = [Filled(c, 4, 2, 64, 32, [2], [n], seed=n) for c, n in zip(ctxs, (8000, 5000))]
        qs = [_cuda(p.rng.standard_normal((2, 16, 64)).astype(np.float32)) for p in ps]
        outs = [[torch.empty_like(q) for _ in range(5)] for q in qs]
        for p in ps:
            _cuda(np.zeros(1))
        torch.cuda.synchronize()
        alone = []
        for c, p, q in zip(ctxs, ps, qs):
            o = torch.empty_like(q)
            c.attention_batch_into(p.cache, p.batch, q, o, 0.125)
            c.synchronize()
            alone.append(o)
        for i in range(5):
            for c, p, q, o in zip(ctxs, ps, qs, outs):
                c.attention_batch_into(p.cache, p.batch, q, o[i], 0.125)
        torch.cuda.synchronize()
        assert all(torch.equal(x, a) for o, a in zip(outs, alone) for x in o)
    finally:
        for c in ctxs:
            c.close()


def test_a_prompt_at_once_and_by_tokens(gpu_ctx):
    """A prompt stored and attended at once, in chunks and token by token:
    the same cache, and outputs that differ by rounding."""
    import torch

    import spt

    n, kv, heads = 75, 2, 16
    rng = np.random.default_rng(4)
    q, k, v = (rng.standard_normal((n, h, 64)).astype(np.float32) for h in (heads, kv, kv))
    pos = np.arange(n)
    qr, kr = rotate(q, pos, YARN), rotate(k, pos, YARN)
    ks, vs = stored(kr, v, 4)
    want, tol = attend(qr, ks, vs, 0, 0.125, 50)
    bytes_ = []
    for steps in ([n], [32, 32, 11], [1] * n):
        p = Paged(4, kv, 64, 32, [n], [n], seed=1)
        p.data.zero_()
        got = np.zeros(q.shape, np.float32)
        at = 0
        for m in steps:
            b = p.make_batch([0, m], [at + m], m, n, n_rows=m)
            qd = _cuda(q[at:at + m])
            gpu_ctx.kv_store_batch(p.cache, b, _cuda(k[at:at + m]), _cuda(v[at:at + m]), rope=spt.Rope(**YARN), q=qd, q_out=qd)
            out = torch.empty_like(qd)
            gpu_ctx.attention_batch_into(p.cache, b, qd, out, 0.125, window=50)
            got[at:at + m] = out.cpu().numpy()
            at += m
        check(got, want, tol)
        bytes_.append(p.data.cpu().numpy())
    assert np.array_equal(bytes_[0], bytes_[1]) and np.array_equal(bytes_[0], bytes_[2])


@pytest.mark.parametrize("tokens,before", [(1, 200), (7, 33), (40, 0)])
def test_attention_block(gpu_ctx, O, tokens, before):
    """RMSNorm with Q8_0, Q/K/V, rotation and store, attention with Q8_0, and
    the output projection with its residual, all on the device: each stage
    against its plain form on the stage before, the last as the projection
    of the Q8_0 of the formula's output."""
    import torch

    import spt
    from helpers import assert_close

    rng = np.random.default_rng(tokens)
    hidden, heads, kv, dim = 256, 8, 2, 64

    def weight(rows, cols):
        q = rng.integers(0, 256, (rows, cols // 32, 16), dtype=np.uint8)
        d = (rng.uniform(0.5, 1.5, (rows, cols // 32, 1)) * 0.02).astype(np.float16).view(np.uint8)
        raw = np.ascontiguousarray(np.concatenate([d, q], -1))
        lo, hi = (q & 15).astype(np.float64) - 8, (q >> 4).astype(np.float64) - 8
        dense = np.concatenate([lo, hi], -1) * d.view(np.float16).astype(np.float64)
        dev = torch.from_numpy(raw.ravel()).cuda()
        return spt.Tensor.make("w", spt.TYPE_Q4_0, [cols, rows], dev.data_ptr(), dev.numel()), dense.reshape(rows, cols), dev

    ws = [weight(r, hidden) for r in (heads * dim, kv * dim, kv * dim)]
    wo = weight(hidden, heads * dim)
    norm = torch.ones(hidden, device="cuda")
    nw = spt.Tensor.make("norm", spt.TYPE_F32, [hidden], norm.data_ptr(), 4 * hidden)
    p = Filled(gpu_ctx, 4, kv, dim, 32, [tokens], [before + tokens], seed=1)
    x = _cuda(rng.standard_normal((tokens, hidden)).astype(np.float32))
    x0 = x.cpu().numpy().astype(np.float64)
    y, xq = torch.empty_like(x), torch.empty(x.numel() // 32 * 34, dtype=torch.uint8, device="cuda")
    q, k, v = (torch.empty(tokens, h, dim, device="cuda") for h in (heads, kv, kv))
    out, oq = torch.empty_like(q), torch.empty(q.numel() // 32 * 34, dtype=torch.uint8, device="cuda")
    o = torch.empty_like(x)
    sinks = _cuda(rng.standard_normal(heads).astype(np.float32))
    sk = spt.Tensor.make("attn_sinks", spt.TYPE_F32, [heads], sinks.data_ptr(), 4 * heads)

    gpu_ctx.rmsnorm_batch_into(nw, x, y, tokens, 1e-5, q8=xq)
    gpu_ctx.mul_q40_qkv_batch_into([w[0] for w in ws], None, None, [q, k, v], tokens, xq=xq, x_len=x.numel())
    q0, k0, v0 = (t.cpu().numpy() for t in (q, k, v))
    gpu_ctx.kv_store_batch(p.cache, p.batch, k, v, rope=spt.Rope(**YARN), q=q, q_out=q)
    gpu_ctx.attention_batch_into(p.cache, p.batch, q, out, dim ** -0.5, window=128, sinks=sk, q8=oq)
    gpu_ctx.mul_q40_batch_q8_into(wo[0], None, oq, o, tokens, resid=x)
    torch.cuda.synchronize()

    def dequant(blocks, n):
        b = blocks.cpu().numpy().reshape(-1, 34)
        return (b[:, 2:].view(np.int8) * np.ascontiguousarray(b[:, :2]).view(np.float16).astype(np.float64)).reshape(n, -1)

    xn = dequant(xq, tokens)
    for got, w in zip((q0, k0, v0), ws):
        assert_close(got.reshape(tokens, -1), (xn @ w[1].T).astype(np.float32), what="projection")
    pos = np.arange(before, before + tokens)
    qr = rotate(q0, pos, YARN)
    assert same(q.cpu().numpy(), qr)
    ks, vs = stored(rotate(k0, pos, YARN), v0, 4)
    p.k[0][before:], p.v[0][before:] = ks, vs
    check(out.cpu().numpy(), *attend(qr, p.k[0], p.v[0], before, dim ** -0.5, 128, sinks.cpu().numpy()))
    want = dequant(oq, tokens) @ wo[1].T
    assert_close(o.cpu().numpy(), want.astype(np.float32), what="output projection")
    assert_close(x.cpu().numpy(), (x0 + want).astype(np.float32), what="residual")
