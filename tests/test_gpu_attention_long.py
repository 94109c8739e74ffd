"""Attention over many positions against the formula in 64 bits, where what a
sum has already decides how much of the rest it keeps: one position far above
all others, even weights, values of one sign.  The bounds do not grow with the
positions."""
import math

import numpy as np
import pytest

from test_gpu_kv_cache import Paged

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32
# log2 of the first position's weight over each other one, a head each
GAPS = (0.0, 12.0, 20.0, 24.0, 25.0, 27.0, 30.0, 32.0)


class Shared(Paged):
    """seqs sequences that read the same n positions.  A key's element 0 is 1
    at the first position and 0 at all others, its element 1 normal; values are
    within 0.5 and 1.5."""

    def __init__(self, ctx, bits, kv, dim, seqs, new, n):
        import torch

        super().__init__(bits, kv, dim, 256, [n], [n], seed=dim + kv)
        g = torch.Generator(device="cuda").manual_seed(n)
        k = torch.zeros(n, kv, dim, device="cuda")
        k[0, :, 0] = 1.0
        # (a block of its own, so that its scale is not the first element's)
        k[:, :, 32] = torch.randn(n, kv, generator=g, device="cuda")
        v = 0.5 + torch.rand(n, kv, dim, generator=g, device="cuda")
        ctx.kv_store_batch(self.cache, self.batch, k, v)
        ctx.kv_load_batch(self.cache, self.batch, k, v)
        self.k, self.v, self.n = k, v, n
        self.many = self.make_batch(np.arange(seqs + 1) * new, [n] * seqs, new, n, n_rows=seqs * new, table=np.repeat(self.table, seqs, 0))


# by 8, 16 and 128 rows; whole, in parts and in shares
@pytest.mark.parametrize("bits,dim,kv,group,new,seqs,n", [
    (4, 64, 8, 8, 1, 1, 131077), (8, 64, 8, 8, 1, 64, 40003), (4, 64, 8, 8, 1, 130, 9001), (8, 128, 8, 8, 1, 64, 40003),
    (4, 128, 8, 8, 1, 40, 9001), (8, 64, 8, 8, 2, 64, 40003), (4, 128, 4, 8, 2, 20, 40003),
    (4, 64, 8, 8, 16, 150, 40003), (8, 64, 1, 8, 2048, 9, 131077), (8, 128, 8, 8, 16, 48, 40003), (4, 128, 2, 8, 16, 2, 131077)])
@pytest.mark.parametrize("spread", (0.0, 1.0))
def test_sums_keep_what_is_small(gpu_ctx, bits, dim, kv, group, new, seqs, n, spread):
    """The bound, of the sum of p |v|, in U.

    A score is (by construction) the sum of at most two products; it is off by the
    scale's rounding, the query's (times the scale, and 2^-22 in its two halves) and
    five roundings of sums and the key's scale, 11 U of the largest score, and the
    exponent's argument by U of its size, which is at most that and 16.  That
    counts in the weights of numerator and denominator.  The exponential is off by
    2^-22 in either (8), a weight's two halves by 2^-22 (4), or by 2^-32 of the
    largest among the 2,048 positions that are summed together (8 times its value,
    which is at most 3 times another: 24).  Among those, a tile is three products of 32
    onto the running sum; the matrix instruction cuts each of the 32 at 2^-26 of the
    largest of them and the sum, and rounds twice: 3 * (8 + 2) a tile, 1920 for
    64.  The weights are added in 67 steps (and 10 over lanes and waves).  What
    has been summed up is scaled and added at most 64 times, in numerator and
    denominator: 192 each.  The end rounds 4 times.

    That is the worst case, every cut and rounding on the same side.  Over all outputs
    they come nowhere near it: the norm is held to 1e-5."""
    import torch

    p = Shared(gpu_ctx, bits, kv, dim, seqs, new, n)
    scale = 0.125
    q = torch.zeros(seqs * new, kv, group, dim, device="cuda")
    gaps = torch.tensor([GAPS[h % len(GAPS)] for h in range(group)], device="cuda")
    one = float(p.k[0, 0, 0])
    q[..., 0] = gaps * math.log(2) / scale / one
    q[..., 32] = spread / scale
    q = q.reshape(seqs * new, kv * group, dim)
    out = torch.full_like(q, 9.0)
    gpu_ctx.attention_batch_into(p.cache, p.many, q, out, scale)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all())
    c = (8 + 4 + 24 + 1920 + 77 + 2 * 192 + 4) * U
    far2 = want2 = 0.0
    for s in {0, seqs // 2, seqs - 1}:
        for i in {0, new // 2, new - 1}:
            row, see = s * new + i, n - new + i + 1
            for h in range(kv):
                qq = q[row, h * group:(h + 1) * group].double()
                kk, vv = p.k[:see, h].double(), p.v[:see, h].double()
                x = qq[:, :1] * kk[:, 0][None] + qq[:, 32:33] * kk[:, 32][None]
                x = x * scale
                w = torch.exp(x - x.amax(1, keepdim=True))
                mass = torch.matmul(w, vv) / w.sum(1, keepdim=True)  # all values are positive
                size = x.abs().amax(1, keepdim=True)
                tol = (c + 2 * (size * 12 * U + 16 * math.log(2) * U)) * mass
                far = (out[row, h * group:(h + 1) * group].double() - mass).abs()
                far2 += float((far ** 2).sum())
                want2 += float((mass ** 2).sum())
                at = (far / tol).amax(1).argmax().item()
                assert bool((far <= tol).all()), f"head of gap {GAPS[at % len(GAPS)]}: off by {float((far / mass)[at].max()):.3g}, {float((far / tol).max()):.3g} of what it may"
    assert far2 <= 1e-10 * want2, f"norm off by {(far2 / want2) ** 0.5:.3g}"


@pytest.mark.parametrize("bits,dim,kv,group,new,seqs,n", [
    (8, 64, 8, 8, 1, 64, 40003), (4, 64, 8, 8, 1, 130, 9001), (8, 64, 8, 8, 2, 64, 40003), (4, 64, 8, 8, 16, 150, 12003), (8, 128, 8, 8, 16, 48, 12003)])
def test_marks_stay_over_kept_sums(gpu_ctx, bits, dim, kv, group, new, seqs, n):
    """A page that is none, at the beginning, within and at the end of a row
    that is summed up in several sums, makes it NaN; other sequences are as before."""
    import torch

    p = Shared(gpu_ctx, bits, kv, dim, seqs, new, n)
    q = torch.randn(seqs * new, kv * group, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    whole = torch.full_like(q, 9.0)
    gpu_ctx.attention_batch_into(p.cache, p.many, q, whole, 0.125)
    table = np.repeat(p.table, seqs, 0)
    bad = {0: 0, seqs // 2: p.table.shape[1] // 2, seqs - 1: p.table.shape[1] - 1}
    for s, page in bad.items():
        table[s, page] = p.n_pages
    out = torch.full_like(q, 9.0)
    gpu_ctx.attention_batch_into(p.cache, p.make_batch(np.arange(seqs + 1) * new, [n] * seqs, new, n, n_rows=seqs * new, table=table), q, out, 0.125)
    torch.cuda.synchronize()
    lost = torch.zeros(seqs * new, dtype=torch.bool, device="cuda")
    for s in bad:
        lost[s * new:(s + 1) * new] = True
    assert bool(torch.isfinite(whole).all()) and bool(torch.isnan(out[lost]).all())
    assert torch.equal(out[~lost], whole[~lost])
