// spt_attn.hip -- attention of a batch's rows over the quantized cache:
// o = sum_j p_j v_j, p = softmax over the seen positions j of scale * q . k_j
// with a head's sink logit in the denominator; grouped heads, causal, with
// an optional window.
//
// Products run on the fp16 MFMA at fp32's accuracy.  A stored value c d (at
// most 8-bit c, 11-bit d) is exactly the sum of two fp16 numbers: hi =
// fp16(c d), lo = c d - hi (a multiple of 2^-24, like d; one packed multiply
// and one packed FMA for two values).  A query row is scaled by a power of
// two and split the same way (22 bits), and so are the weights p.  Of the four
// products of halves the three larger are added in fp32; the dropped lo * lo is
// below 2^-22 of the product.
//
// k_attn_split, rows 16 at a time (a column of the MFMA each; the group's
// heads of one or more tokens): a wave takes tiles of 32 positions in turn
// and makes their operands in its registers, scores of a tile are its D
// registers, and those are the B operand of the product with the values.  The
// running maximum is one number a row, raised only when a score passes it by
// kSlack (weights up to 2^kSlack fit fp16 beside the scale), so most tiles need
// no exchange between lanes and no rescaling.  The waves' parts meet in LDS;
// where the rows are few, splits of the positions meet in k_attn_merge.
#include <algorithm>

#include "spt_kernels.h"
#include "spt_kv.h"

namespace spt {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kAttnRows = 16;           // rows of a row tile
constexpr int kWaves = 4;
constexpr float kNoMax = -3.0e38f;  // the running maximum before any score
constexpr float kSlack = 8.0f;      // log2 of the largest weight
constexpr float kLift = 5.0f;       // weights are held times 2^kLift (at most 2^13)

union Half8 {
    half8v v;
    half2v h[4];
};

__device__ inline half2v pk(uint32_t w) { return __builtin_bit_cast(half2v, w); }

// Codes of eight positions or dims as fp16 pairs.  Q4_0: w's low nibbles (or
// high) of bytes 0 and 2, then 1 and 3, into the low mantissa bits of 1024
// (or 16 places higher, 64 + n after the multiply by 1/16).
__device__ inline half2v q4_low(uint32_t w) { return pk((w & 0x000F000Fu) | 0x64006400u) + (half2v)(_Float16)-1032.0f; }
__device__ inline half2v q4_high(uint32_t w) {
    return __builtin_elementwise_fma(pk((w & 0x00F000F0u) | 0x64006400u), (half2v)(_Float16)0.0625f, (half2v)(_Float16)-72.0f);
}
__device__ inline half2v q8_pair(uint32_t w, int upper) {
    return pk(__builtin_amdgcn_perm(0x64646464u, w, upper ? 0x04030402u : 0x04010400u)) + (half2v)(_Float16)-1152.0f;
}

// The codes' values, split.
__device__ inline void split_values(const half2v (&c)[4], const half2v (&d)[4], Half8 &hi, Half8 &lo) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        hi.h[i] = c[i] * d[i];
        lo.h[i] = __builtin_elementwise_fma(c[i], d[i], -hi.h[i]);
    }
}

__device__ inline f32x4 mfma(const Half8 &a, const Half8 &b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
}

// A lane's raw bytes of a tile.
template <int BITS, int NB>
struct RawTile {
    static constexpr int kUnits = BITS == 4 ? NB / 2 : NB;
    u32x4 k[kUnits], v[kUnits];
    uint32_t ks[NB];      // key scales [t][b], two fp16 a word
    u32x4 vs[NB];         // value scales of 8 positions

    __device__ inline void load_keys(const uint8_t *tile, int lane) {
        using T = KvTile<BITS, NB>;
#pragma unroll
        for (int u = 0; u < kUnits; u++) k[u] = *reinterpret_cast<const u32x4 *>(tile + (u * 64 + lane) * 16);
#pragma unroll
        for (int i = 0; i < NB; i += 2) {
            const uint2 x = *reinterpret_cast<const uint2 *>(tile + T::kScales + (lane & 15) * 4 * NB + i * 4);
            ks[i] = x.x;
            ks[i + 1] = x.y;
        }
    }
    __device__ inline void load_values(const uint8_t *tile, int lane) {
        using T = KvTile<BITS, NB>;
#pragma unroll
        for (int u = 0; u < kUnits; u++) v[u] = *reinterpret_cast<const u32x4 *>(tile + T::kValues + (u * 64 + lane) * 16);
#pragma unroll
        for (int b = 0; b < NB; b++) vs[b] = *reinterpret_cast<const u32x4 *>(tile + T::kValues + T::kScales + b * 64 + (lane >> 4) * 16);
    }
    // Key operand of tile half t, block b.
    __device__ inline void keys(int t, int b, Half8 &hi, Half8 &lo) const {
        half2v c[4], d[4];
        if (BITS == 4) {
            const uint32_t w = k[b >> 1][t * 2 + (b & 1)], x = w >> 8;
            c[0] = q4_low(w);
            c[1] = q4_high(w);
            c[2] = q4_low(x);
            c[3] = q4_high(x);
        } else {
            const u32x4 &u = k[(b >> 1) * 2 + t];
            const uint32_t w0 = u[(b & 1) * 2], w1 = u[(b & 1) * 2 + 1];
            c[0] = q8_pair(w0, 0);
            c[1] = q8_pair(w0, 1);
            c[2] = q8_pair(w1, 0);
            c[3] = q8_pair(w1, 1);
        }
        const half2v s = pk(ks[(t * NB + b) >> 1]);
        const half2v dd = (b & 1) ? half2v{s[1], s[1]} : half2v{s[0], s[0]};
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = dd;
        split_values(c, d, hi, lo);
    }
    // Value operand of block b, dims 16 h .. 16 h + 15.
    __device__ inline void values(int b, int h, Half8 &hi, Half8 &lo) const {
        half2v c[4], d[4];
        if (BITS == 4) {
            const uint32_t w0 = v[b >> 1][(b & 1) * 2], w1 = v[b >> 1][(b & 1) * 2 + 1];
            c[0] = h ? q4_high(w0) : q4_low(w0);
            c[1] = h ? q4_high(w0 >> 8) : q4_low(w0 >> 8);
            c[2] = h ? q4_high(w1) : q4_low(w1);
            c[3] = h ? q4_high(w1 >> 8) : q4_low(w1 >> 8);
        } else {
            const uint32_t w0 = v[b][h * 2], w1 = v[b][h * 2 + 1];
            c[0] = q8_pair(w0, 0);
            c[1] = q8_pair(w0, 1);
            c[2] = q8_pair(w1, 0);
            c[3] = q8_pair(w1, 1);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = pk(vs[b][i]);
        split_values(c, d, hi, lo);
    }
    // Positions from `left` on (of the lane's eight, at 8 g) are beyond the
    // sequence: whatever is there counts as zero.
    __device__ inline void clear_values(int left) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) vs[b][i] = left <= 2 * i ? 0u : left == 2 * i + 1 ? vs[b][i] & 0xFFFFu : vs[b][i];
    }
};

// What a row tile's rows see: positions [0, ..] of the first and the last row,
// and the tiles that hold any of them.
struct RowSpan {
    int i_first, i_last;  // tokens
    int t_lo, t_hi;       // tiles
};

__device__ inline RowSpan row_span(const AttnArgs &a, const KvSeq &sq, int rt) {
    RowSpan r;
    const int rows = sq.n * a.group;
    r.i_first = rt * kAttnRows / a.group;
    r.i_last = (min(rows, rt * kAttnRows + kAttnRows) - 1) / a.group;
    const int last = sq.first + r.i_last;
    const int lo = a.window ? max(0, sq.first + r.i_first - a.window + 1) : 0;
    r.t_lo = lo / kKvTile;
    r.t_hi = last < 0 ? r.t_lo : last / kKvTile + 1;
    return r;
}

__device__ inline int active_splits(const AttnArgs &a, const RowSpan &r) {
    return max(1, (r.t_hi - r.t_lo + a.split_tiles - 1) / a.split_tiles);
}

// Sink, division and stores of a row's block of 32 (an element a lane of a
// half-wave): o / l with the row's maximum m.
__device__ inline void store_row(const AttnArgs &a, int head, int64_t row, int b, int nb, float o, float l, float m, int lane, bool ok) {
    float f = 1.0f;
    if (a.sinks) {
        const float sink = bias_at(a.sinks, a.sink_type, (uint64_t)head) * 1.44269504088896341f;
        const float top = fmaxf(m, sink);
        f = __builtin_amdgcn_exp2f(m - top);
        l = l * f + __builtin_amdgcn_exp2f(sink - top);
    }
    const float v = l == 0.0f ? 0.0f : o * f / l;
    const int64_t blk = (row * a.heads + head) * nb + b;
    if (ok) a.out[blk * 32 + (lane & 31)] = v;
    if (a.q8) {
        uint16_t dh;
        const int q = q8_quantize_half(v, lane, &dh);
        if (ok) write_q8_lane(q, dh, lane & 31, (size_t)blk, nullptr, nullptr, nullptr, a.q8);
    }
}

template <int BITS, int NB>
__global__ __launch_bounds__(64 * kWaves) void k_attn_split(AttnArgs a) {
    using T = KvTile<BITS, NB>;
    constexpr int kDim = 32 * NB;
    __shared__ float so[kWaves][kAttnRows][kDim + 4];
    __shared__ float sm[kWaves][kAttnRows], sl[kWaves][kAttnRows];
    const int seq = blockIdx.y;
    const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
    const int kvh = unit % a.kv.kv_heads, rt = unit / a.kv.kv_heads;
    const KvSeq sq = kv_seq(a.kv, seq);
    const int rows = sq.n * a.group;
    if (rt * kAttnRows >= rows) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    RowSpan sp = row_span(a, sq, rt);
    if (!sq.ok) sp.t_lo = sp.t_hi = 0;
    if (split >= active_splits(a, sp)) return;

    // the row of this lane's column
    const int flat = rt * kAttnRows + col;
    const bool row_ok = flat < rows;
    const int tok = row_ok ? flat / a.group : sp.i_last, hd = kvh * a.group + (row_ok ? flat % a.group : 0);
    const int pos = sq.first + tok;                    // last position that it sees
    const int from = a.window ? pos - a.window : -1;   // it sees those after this one

    Half8 qh[NB], ql[NB];
    float mul;
    {
        float x[NB][8], top = 0.0f;
        const float *src = a.q + ((int64_t)(sq.r0 + tok) * a.heads + hd) * kDim + 8 * g;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const float4 u = *reinterpret_cast<const float4 *>(src + 32 * b), w = *reinterpret_cast<const float4 *>(src + 32 * b + 4);
            x[b][0] = u.x, x[b][1] = u.y, x[b][2] = u.z, x[b][3] = u.w;
            x[b][4] = w.x, x[b][5] = w.y, x[b][6] = w.z, x[b][7] = w.w;
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, __builtin_fabsf(x[b][i]));
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int e = __builtin_amdgcn_frexp_expf(top);
        mul = __builtin_ldexpf(a.scale, e - 13);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = __builtin_ldexpf(x[b][i], 13 - e);
                qh[b].v[i] = (_Float16)y;
                ql[b].v[i] = (_Float16)(y - (float)qh[b].v[i]);
            }
    }

    f32x4 o[NB][2];
#pragma unroll
    for (int b = 0; b < NB; b++) o[b][0] = o[b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = kNoMax, l = sq.ok ? 0.0f : __builtin_nanf("");
    const int t_end = min(sp.t_hi, sp.t_lo + (split + 1) * a.split_tiles);
    for (int t = sp.t_lo + split * a.split_tiles + wave; t < t_end; t += kWaves) {
        const int p0 = t * kKvTile;
        const uint8_t *tile = kv_tile(a.kv, seq, kvh, t, T::kBytes);
        if (!tile) {
            if (p0 <= pos && p0 + kKvTile - 1 > from) l = __builtin_nanf("");
            continue;
        }
        RawTile<BITS, NB> raw;
        raw.load_keys(tile, lane);
        raw.load_values(tile, lane);
        f32x4 s[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                Half8 kh, kl;
                raw.keys(h, b, kh, kl);
                s[h] = mfma(kh, qh[b], s[h]);
                s[h] = mfma(kh, ql[b], s[h]);
                s[h] = mfma(kl, qh[b], s[h]);
            }
        }
        float x[8], top = -__builtin_inff();
        const bool whole = p0 + kKvTile - 1 <= sq.first + sp.i_first && (!a.window || p0 > sq.first + sp.i_last - a.window);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = s[j >> 2][j & 3] * mul;
        if (!whole) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int p = p0 + 8 * g + j;
                x[j] = p <= pos && p > from ? x[j] : -__builtin_inff();
            }
            if (p0 + kKvTile > sq.len) raw.clear_values(sq.len - p0 - 8 * g);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, x[j]);
        if (__any(top > m + kSlack)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float nm = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - nm);
            m = nm;
            l *= f;
#pragma unroll
            for (int b = 0; b < NB; b++) o[b][0] *= f, o[b][1] *= f;
        }
        Half8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float w = __builtin_amdgcn_exp2f(x[j] - (m - kLift));
            l += w;
            ph.v[j] = (_Float16)w;
            pl.v[j] = (_Float16)(w - (float)ph.v[j]);
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                Half8 vh, vl;
                raw.values(b, h, vh, vl);
                o[b][h] = mfma(vh, ph, o[b][h]);
                o[b][h] = mfma(vh, pl, o[b][h]);
                o[b][h] = mfma(vl, ph, o[b][h]);
            }
    }

    // the waves' parts, on the largest maximum
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) sm[wave][col] = m, sl[wave][col] = l;
    __syncthreads();
    float top = sm[0][col];
#pragma unroll
    for (int w = 1; w < kWaves; w++) top = fmaxf(top, sm[w][col]);
    const float f = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int h = 0; h < 2; h++) *reinterpret_cast<f32x4 *>(&so[wave][col][32 * b + 16 * h + 4 * g]) = o[b][h] * f;
    __syncthreads();
    // a half-wave takes a block of a row
    for (int u = wave * 2 + (lane >> 5); u < kAttnRows * NB; u += 2 * kWaves) {
        const int r = u / NB, b = u % NB, d = 32 * b + (lane & 31);
        float mx = sm[0][r], sum = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; w++) mx = fmaxf(mx, sm[w][r]);
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            den += sl[w][r] * __builtin_amdgcn_exp2f(sm[w][r] - mx);
            sum += so[w][r][d];
        }
        const int fr = rt * kAttnRows + r;
        const bool ok = fr < rows;
        if (a.splits == 1) {
            // the weights are 2^kLift too large on both sides; the sink is not
            store_row(a, kvh * a.group + fr % a.group, sq.r0 + fr / a.group, b, NB, sum, den, mx - kLift, lane, ok);
        } else if (ok) {
            float *part = a.part + (((int64_t)seq * a.row_tiles * a.kv.kv_heads + unit) * a.splits + split) * kAttnRows * (kDim + 2);
            part[r * (kDim + 2) + 2 + d] = sum;
            if (d == 0) part[r * (kDim + 2)] = mx - kLift, part[r * (kDim + 2) + 1] = den;
        }
    }
}

// The splits of a row tile: a wave takes rows in turn, a half-wave a block.
template <int NB>
__global__ __launch_bounds__(256) void k_attn_merge(AttnArgs a) {
    constexpr int kDim = 32 * NB;
    const int seq = blockIdx.y, unit = blockIdx.x, kvh = unit % a.kv.kv_heads, rt = unit / a.kv.kv_heads;
    const KvSeq sq = kv_seq(a.kv, seq);
    const int rows = sq.n * a.group;
    if (rt * kAttnRows >= rows) return;
    RowSpan sp = row_span(a, sq, rt);
    if (!sq.ok) sp.t_lo = sp.t_hi = 0;
    const int n = active_splits(a, sp), lane = threadIdx.x & 63;
    const float *base = a.part + ((int64_t)seq * a.row_tiles * a.kv.kv_heads + unit) * a.splits * kAttnRows * (kDim + 2);
    for (int u = threadIdx.x >> 5; u < kAttnRows * NB; u += 8) {
        const int r = u / NB, b = u % NB, fr = rt * kAttnRows + r;
        const bool ok = fr < rows;
        float m = kNoMax, l = 0.0f, o = 0.0f;
        for (int i = 0; ok && i < n; i++) {
            const float *p = base + ((int64_t)i * kAttnRows + r) * (kDim + 2);
            const float pm = p[0], top = fmaxf(m, pm), f = __builtin_amdgcn_exp2f(m - top), w = __builtin_amdgcn_exp2f(pm - top);
            l = l * f + p[1] * w;
            o = o * f + p[2 + 32 * b + (lane & 31)] * w;
            m = top;
        }
        store_row(a, kvh * a.group + fr % a.group, sq.r0 + fr / a.group, b, NB, o, l, m, lane, ok);
    }
}

}  // namespace

AttnPlan attn_plan(int nb, int kv_heads, int group, int n_seqs, int max_new, int max_len, int window, int n_cu) {
    AttnPlan p;
    p.row_tiles = (int)(((int64_t)max_new * group + kAttnRows - 1) / kAttnRows);
    const int64_t units = (int64_t)n_seqs * kv_heads * p.row_tiles;
    // the tiles of the longest row tile: a window of positions before its first
    // row's, and the rows' own
    const int own = (kAttnRows - 1) / group + 1;
    const int64_t seen = window ? std::min<int64_t>(max_len, (int64_t)window + own) : max_len;
    const int64_t tiles = seen / kKvTile + 2;
    const int64_t want = std::max<int64_t>(1, (int64_t)n_cu * 4 / units);
    const int64_t per = std::max<int64_t>(8, (tiles + want - 1) / want);
    p.splits = (int)((tiles + per - 1) / per);
    p.split_tiles = (int)per;
    p.work_bytes = p.splits > 1 ? (uint64_t)units * p.splits * kAttnRows * (32 * nb + 2) * 4 : 0;
    return p;
}

hipError_t launch_attn(hipStream_t s, int bits, int nb, const AttnArgs &a) {
    const dim3 grid(a.kv.kv_heads * a.row_tiles * a.splits, a.kv.n_seqs);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(64 * kWaves), 0, s, a); };
    if (bits == 4)
        nb == 2 ? go(k_attn_split<4, 2>) : go(k_attn_split<4, 4>);
    else
        nb == 2 ? go(k_attn_split<8, 2>) : go(k_attn_split<8, 4>);
    return hipGetLastError();
}

hipError_t launch_attn_merge(hipStream_t s, int nb, const AttnArgs &a) {
    const dim3 grid(a.kv.kv_heads * a.row_tiles, a.kv.n_seqs);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a); };
    nb == 2 ? go(k_attn_merge<2>) : go(k_attn_merge<4>);
    return hipGetLastError();
}

}  // namespace spt
