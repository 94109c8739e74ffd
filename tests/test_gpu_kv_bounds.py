"""Batches whose arrays claim rows that are not there: nothing behind the
buffers and no row of no sequence is written, by any of the paths."""
import numpy as np
import pytest

from kv_reference import attend, stored
from test_gpu_attention import Filled, run
from test_gpu_kv_cache import Paged, _cuda, same

pytestmark = pytest.mark.gpu

LOW, HIGH = -2 ** 31, 2 ** 31 - 1


def _starts(n):
    return [[HIGH, LOW, LOW, HIGH, LOW], [n - 1, LOW, 5, LOW + 5, n], [n, LOW, n - 1, LOW + n - 2, LOW], [0, 5, LOW, 5, LOW + 1],
            [LOW, HIGH, LOW, HIGH, HIGH], [-5, -2, 1, 0, 40], [30, 20, 10, 5, 2], [LOW, HIGH, -1, HIGH, -7], [HIGH] * 5, [LOW] * 5]


def _claimed(starts, n, max_new):
    rows = np.zeros(n, bool)
    for lo, hi in zip(starts[:-1], starts[1:]):
        lo = max(0, lo)
        rows[lo:max(lo, min(hi, n, lo + max_new))] = True
    return rows


class Guarded:
    """A buffer of n rows with as many more behind it as a call could reach."""

    def __init__(self, n, behind, row, fill, dtype):
        import torch

        self.all = torch.full((n + behind, row), fill, dtype=dtype, device="cuda")
        self.n, self.fill, self.rows = n, fill, self.all[:n]

    def check(self, claimed):
        got = self.all.cpu().numpy()
        assert (got[self.n:] == self.fill).all(), "written behind the buffer"
        assert (got[:self.n][~claimed] == self.fill).all(), "a row of no sequence was written"


@pytest.mark.parametrize("bits,dim", [(4, 64), (8, 128)])
def test_load_and_store(gpu_ctx, bits, dim):
    import torch

    new, n = 40, 35
    p = Paged(bits, 2, dim, 32, [new], [90])
    before = p.data.clone()
    src = _cuda(p.rng.standard_normal((n, 2 * dim)).astype(np.float32))
    for starts in _starts(n):
        for lens in ([8, 8, 8, 8], [HIGH, 0, LOW, 90]):
            b = p.make_batch(starts, lens, new, 90, n_rows=n, table=np.repeat(p.table, 4, 0))
            k, v = (Guarded(n, 2 * new, 2 * dim, 7.0, torch.float32) for _ in range(2))
            gpu_ctx.kv_load_batch(p.cache, b, k.rows, v.rows)
            k.check(_claimed(starts, n, new))
            v.check(_claimed(starts, n, new))
            gpu_ctx.kv_store_batch(p.cache, b, src, src)
            if all(hi <= lo for lo, hi in zip(starts[:-1], starts[1:])):
                assert torch.equal(p.data, before)
            p.data.copy_(before)


# rows of a key/value head by 8, by 16 and by 128; whole and in parts
@pytest.mark.parametrize("bits,dim,kv,group,new,bound", [
    (4, 64, 1, 2, 4, 100), (4, 64, 1, 2, 4, 9000), (8, 128, 1, 4, 40, 100), (4, 64, 130, 8, 67, 100), (8, 128, 64, 8, 67, 100)])
def test_attention(gpu_ctx, bits, dim, kv, group, new, bound):
    import torch

    n = 33
    p = Filled(gpu_ctx, bits, kv, dim, 32, [new], [90])
    table = np.full((4, -(-bound // 32)), -1, np.int32)
    table[:, :p.table.shape[1]] = p.table
    q = _cuda(p.rng.standard_normal((n, kv * group, dim)).astype(np.float32))
    row = kv * group * dim
    for starts in _starts(n):
        for lens in ([8, 8, 8, 8], [HIGH, 0, LOW, 90]):
            b = p.make_batch(starts, lens, new, bound, n_rows=n, table=table)
            out = Guarded(n, 2 * new, row, 9.0, torch.float32)
            blocks = Guarded(n, 2 * new, row // 32 * 34, 0xAA, torch.uint8)
            gpu_ctx.attention_batch_into(p.cache, b, q, out.rows, dim ** -0.5, q8=blocks.rows)
            torch.cuda.synchronize()
            claimed = _claimed(starts, n, new)
            out.check(claimed)
            blocks.check(claimed)


@pytest.mark.parametrize("bits,kv,group,new", [(4, 1, 2, 8), (8, 2, 8, 12), (4, 130, 8, 67)])
def test_rows_cut_by_the_buffers_keep_their_positions(gpu_ctx, bits, kv, group, new):
    """The first sequence begins before the buffers, the last ends behind them:
    their rows that are there are at the positions that they have in whole ones.
    Positions of the others, never stored, hold marks that no row sees."""
    import torch

    cut, lens = new // 2, [90, new + 3, 81]
    p = Paged(bits, kv, 64, 32, [new] * 3, lens, seed=2)
    p.data.fill_(0xFF)
    b, starts, n = p.whole()
    k, v = (p.rng.standard_normal((n, kv, 64)).astype(np.float32) for _ in range(2))
    # what was in the cache before: all but the new rows of the first and last
    shifted = [x.copy() for x in (k, v)]
    for x, y in zip((k, v), shifted):
        for s in (0, 2):
            m = lens[s] - new
            y[starts[s + 1] - m:starts[s + 1]] = x[starts[s]:starts[s] + m]  # last rows are the last positions
    old = p.make_batch(starts, [lens[0] - new, lens[1], lens[2] - new], 90, 90, n_rows=n)
    gpu_ctx.kv_store_batch(p.cache, old, _cuda(shifted[0]), _cuda(shifted[1]))

    rows = 3 * new - 2 * cut
    first, last = -cut, rows + cut  # rows_dev of the batch whose buffers lack cut rows at both ends
    batch = p.make_batch([first, first + new, first + 2 * new, last], lens, new, 90, n_rows=rows)
    pick = np.concatenate([np.arange(starts[s + 1] - new, starts[s + 1]) for s in range(3)])[cut:3 * new - cut]
    gpu_ctx.kv_store_batch(p.cache, batch, _cuda(k[pick]), _cuda(v[pick]))
    got = p.load(gpu_ctx, batch, rows)
    want = stored(k, v, bits)
    assert same(got[0], want[0][pick]) and same(got[1], want[1][pick])
    whole = p.load(gpu_ctx)
    there = np.ones(n, bool)
    there[starts[1] - new:starts[1] - new + cut] = False  # the first sequence's rows before the buffers
    there[n - cut:] = False
    assert same(whole[0][there], want[0][there]) and np.isnan(whole[0][~there]).all()

    # attention: the last sequence's rows see nothing that is not there
    q = p.rng.standard_normal((rows, kv * group, 64)).astype(np.float32)
    out = torch.full((rows, kv * group, 64), 9.0, device="cuda")
    gpu_ctx.attention_batch_into(p.cache, batch, _cuda(q), out, 0.125)
    out = out.cpu().numpy()
    assert np.isnan(out[:new - cut]).all()  # the first's see the positions before theirs, which are marked
    for s, a, m in ((1, new - cut, new), (2, 2 * new - cut, new - cut)):
        w, tol = attend(q[a:a + m], want[0][starts[s]:starts[s + 1]], want[1][starts[s]:starts[s + 1]], lens[s] - new, 0.125)
        assert (np.abs(out[a:a + m] - w) <= tol).all()


def test_rows_of_two_sequences_are_one_of_them(gpu_ctx):
    """Long rows that two sequences claim hold the results of either: sums on
    their way are no mixture, though they are kept in the output."""
    import torch

    kv, new = 130, 67
    p = Filled(gpu_ctx, 4, kv, 64, 32, [new, 0, new], [2500, 1, 2300], seed=1)
    q = _cuda(p.rng.standard_normal((new, kv * 8, 64)).astype(np.float32))

    def rows_of(starts):
        b = p.make_batch(starts, [2500, 0, 2300], new, 2500, n_rows=new)
        out = torch.full((new, kv * 8, 64), 9.0, device="cuda")
        gpu_ctx.attention_batch_into(p.cache, b, q, out, 0.125)
        torch.cuda.synchronize()
        return out

    first, last = rows_of([0, new, 0, 0]), rows_of([0, 0, 0, new])
    both = rows_of([0, new, 0, new])
    near = lambda a, b: (a - b).abs() <= 1e-5 * b.abs() + 1e-6  # noqa: E731
    assert bool((near(both, first) | near(both, last)).all())
    assert not bool(near(first, last).all())


@pytest.mark.parametrize("new", (4, 40))
def test_freed_pages_before_a_window_are_never_looked_at(gpu_ctx, new):
    """Pages whose positions no row sees are none: rows are as with them."""
    p = Filled(gpu_ctx, 4, 1, 64, 32, [new, new], [100, 90])
    q = p.rng.standard_normal((2 * new, 8, 64)).astype(np.float32)
    table = p.table.copy()
    table[0, 0], table[1, 0] = -1, p.n_pages  # positions 0 .. 31; rows see 56 on and 46 on at least
    got = [run(gpu_ctx, p, q, 0.125, 5, batch=p.make_batch(p.starts, p.lens, new, 100, table=t)) for t in (p.table, table)]
    want, tol = p.want(q, 0.125, 5)
    assert (np.abs(got[1] - want) <= tol).all() and np.array_equal(*got)
