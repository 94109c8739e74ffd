// spt_attn.hip -- attention of a batch's rows over the quantized cache:
// o = sum_j p_j v_j, p = softmax over the seen positions j of scale * q . k_j
// with a head's sink logit in the denominator; grouped heads, causal, with
// an optional window.
//
// Products run on the fp16 MFMA at fp32's accuracy.  A query row is scaled by
// a power of two and held as the sum of two fp16 numbers, hi and lo (22 bits);
// keys enter as their codes, exact in fp16, and a block's scale multiplies its
// sum.  Weights p are split like queries.  A stored value c d (at most 8-bit c,
// 11-bit d) is exactly hi + lo, hi = fp16(c d), lo = c d - hi (a multiple of
// 2^-24, like d; one packed multiply and one packed FMA for two values); of the
// four products of halves the three larger are added in fp32, the dropped
// lo * lo being below 2^-22 of the product.  (Scaling the weights by each
// block's d instead takes as many instructions, and leaves fp16's range.)
//
// Few rows (attend: 8 or 16 of a key/value head at a time, a column of the MFMA
// each or two): the workgroup's waves take tiles of 32 positions in turn and
// make their operands in registers; a tile's scores are its D registers, and
// those are the B operand of the product with the values.  Many rows
// (attend_many: 128 at a time): operands are made once a workgroup in LDS.  The
// running maximum is one number a row, raised only when a score passes it by
// kSlack (weights up to 2^kSlack fit fp16 beside the lift), so most tiles need
// no exchange between lanes and no rescaling.
//
// Long rows: fp32 sums of thousands of terms lose small ones behind a large one (one
// position 2^24 above 131,071 even others: 1.9e-3 of the output, nearly all of it in the
// sum of the weights), the MFMA cuts each product at 2^-26 of the sum that it is
// added to, and a weight below 2^-25 is 0 in fp16.  So a wave sums up at most 32 tiles
// (few rows, kept in LDS) or 64 (many, kept in the output's rows: LDS has no place
// beside the operands) with a maximum of their own, and joins these sums in fp32;
// a tile's weights are added in pairs.  Off by at most 7e-6 of sum p |v| there and for other
// gaps up to 2^32 (2,000 to 131,077 positions, values of one sign; evenly weighted ones
// 1e-6).  Price: none for few rows (64 ragged tokens up to 8,192 51.6 us, as one sum
// 51.2); for many none up to 64 tiles, which have kernels without the joins, beyond
// 3 % (a prompt of 8,192: 1,386, 1,350) to 7 % (heads of 128, 4,096 tokens over 8,192:
// 1,479, 1,386).  A tile's sum made from 0 and added took 13 % more and was off by
// 4e-6.
//
// What bounds it: the vector instructions that unpack values and form weights,
// and the MFMAs, which overlap with them in part only (16 MFMAs and 64 FMAs of
// two waves on a SIMD, one wave each: 463 cycles, 319 and 322 alone); compute units
// left idle where units are unequal or few (64 ragged tokens up to 8,192: busy 62 %
// of the time, vector instructions 48 %).  One token over 1,048,576 positions of 8 heads
// of 64 (604 MB): 129 us and 5 us to join the parts, 4.5 TB/s, vector instructions 70 %;
// over 131,071, 22 and 5 us.  A prompt of 2,048 tokens, 64 heads (34 GFLOP, 2.5 times
// that with the halves): 103 us (the same inputs again and again, 112 with others from
// pass to pass); of 8,192, 1.41 ms (970 TFLOP/s of MFMA; compute units busy 95 %,
// vector instructions 69 %, MFMA 41 %).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "spt_kernels.h"
#include "spt_kv.h"

namespace spt {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8;      // of a workgroup (few rows)
constexpr int kHalfWaves = 4;  // of one of many
// Launches, by what the batch's bounds allow (us; heads 64 on 8 of 64, Q4_0):
//   rows of a key/value head: up to 8, two columns a row (a token of 64 ragged
//   sequences up to 8,192: 59, a column a row 70); more, 16 or 128 at a time (many_rows).
//   8 or 16 rows, units (a row tile of a sequence and head) for at most half of the compute
//   units: each cut into equal parts, a workgroup a part and one a compute unit, and a
//   second launch that joins them; a workgroup a unit where the parts would save fewer
//   tiles than that costs, about kSplitTiles / nb (1 sequence of 1,000: 8.2 whole, 10.3 in
//   parts, of 2,000: 11.5, 10.2, of 4,000: 17.9, 11.0; 8 ragged ones up to 6,000: 24.7,
//   16.4, heads of 128 in Q8_0: 38.3, 22.4).  Where two workgroups fit a compute unit
//   and parts pass kLongPart tiles: twice as many parts of one sequence (600,000: 82, 88);
//   of several, shares (4 of 4 tokens up to 32,000: 36.6, parts 42; up to 10,000: 24.4, 20.4).
//   More units: a workgroup a unit, of half the waves where units are more than
//   fit at once (a token of 128 ragged sequences up to 300: 10.6, eight waves 13.7, up to
//   5,000: 58.9, 59.0; heads of 128, of 34 up to 2,000: 28.5, 34.1, of 64: 29.6, 36.9; of
//   32, which fit: 20.7, 19.6; in Q8_0, 17 of 40 heads on 8: up to 4,000 33.9, shares 36.6,
//   up to 5,003 40.3, 40.6, and beyond in shares).
//   That up to kWideTiles position tiles, in proportion to the
//   units while they do not fill the compute units (a token of 64 ragged sequences up to
//   4,096: 31, shares 40; up to 16,384: 104, 97); beyond, equal shares of all tiles
//   and a second launch.
constexpr int kSplitTiles = 140, kLongPart = 160, kWideTiles = 300;
constexpr int kAttnEntries = 1024;  // (sequence, row tile)s that a workgroup of the shares sums up
constexpr float kNoMax = -3.0e38f;  // the running maximum before any score
constexpr float kSlack = 8.0f;      // log2 of the largest weight
constexpr float kLift = 7.0f;       // weights are held times 2^kLift (at most 2^15)
// Position tiles that a wave sums up together (few rows, many).
constexpr int kFewChunk = 32, kManyChunk = 64;

union Half8 {
    half8v v;
    half2v h[4];
};

__device__ inline half2v pk(uint32_t w) { return __builtin_bit_cast(half2v, w); }

// Constants that the compiler does not see through: with them it makes one
// v_and_or_b32 of the mask and the or, and one mixed-precision FMA of a
// conversion and a product or sum, where it would fold known ones apart.
struct Opaque {
    uint32_t low = 0x000F000Fu, high = 0x00F000F0u, k1024 = 0x64006400u;
    float zero = 0.0f, minus = -1.0f;
    __device__ inline Opaque() {
        asm("" : "+s"(low));
        asm("" : "+s"(high));
        asm("" : "+v"(k1024));
        asm("" : "+v"(zero));
        asm("" : "+v"(minus));
    }
};

// Codes as fp16 pairs.  Q4_0: the low (or high) nibbles of bytes 0 and 2 into the
// low mantissa bits of 1024 (or four places higher: 64 + n after the multiply by
// 1/16).
__device__ inline half2v q4_low(const Opaque &o, uint32_t w) { return pk((w & o.low) | o.k1024) + (half2v)(_Float16)-1032.0f; }
__device__ inline half2v q4_high(const Opaque &o, uint32_t w) {
    return __builtin_elementwise_fma(pk((w & o.high) | o.k1024), (half2v)(_Float16)0.0625f, (half2v)(_Float16)-72.0f);
}
__device__ inline half2v q8_pair(uint32_t w, int upper) {
    return pk(__builtin_amdgcn_perm(0x64646464u, w, upper ? 0x04030402u : 0x04010400u)) + (half2v)(_Float16)-1152.0f;
}

// The key operand of a Q4_0 word, and the value operand of two (dims 16 h on).
__device__ inline void q4_key(const Opaque &o, uint32_t w, Half8 &c) {
    const uint32_t x = w >> 8;
    c.h[0] = q4_low(o, w);
    c.h[1] = q4_high(o, w);
    c.h[2] = q4_low(o, x);
    c.h[3] = q4_high(o, x);
}
__device__ inline void q4_value(const Opaque &o, uint32_t w0, uint32_t w1, int h, Half8 &c) {
    const uint32_t x0 = w0 >> 8, x1 = w1 >> 8;
    c.h[0] = h ? q4_high(o, w0) : q4_low(o, w0);
    c.h[1] = h ? q4_high(o, x0) : q4_low(o, x0);
    c.h[2] = h ? q4_high(o, w1) : q4_low(o, w1);
    c.h[3] = h ? q4_high(o, x1) : q4_low(o, x1);
}
// Either operand of two Q8_0 words.
__device__ inline void q8_codes(uint32_t w0, uint32_t w1, Half8 &c) {
    c.h[0] = q8_pair(w0, 0);
    c.h[1] = q8_pair(w0, 1);
    c.h[2] = q8_pair(w1, 0);
    c.h[3] = q8_pair(w1, 1);
}

// The codes' values, split; d: the scales of eight positions.
__device__ inline void split_values(const Half8 &c, const u32x4 &d, Half8 &hi, Half8 &lo) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        hi.h[i] = c.h[i] * pk(d[i]);
        lo.h[i] = __builtin_elementwise_fma(c.h[i], pk(d[i]), -hi.h[i]);
    }
}

// The scales of eight positions, 0 outside [first, left): what is there belongs
// to no row, and may be anything (a weight of 0 times NaN would be NaN).
__device__ inline void clear_scales(u32x4 &d, int first, int left) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t keep = (2 * i >= first && 2 * i < left ? 0xFFFFu : 0u) | (2 * i + 1 >= first && 2 * i + 1 < left ? 0xFFFF0000u : 0u);
        d[i] &= keep;
    }
}
__device__ inline u32x4 load16(rsrc_t tile, int lane_at, int at) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(tile, lane_at, at, 0));
}

__device__ inline f32x4 mfma(const Half8 &a, const Half8 &b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
}

// Two fp32 numbers as hi + lo: hi rounded toward zero, lo what that leaves
// (x - hi, rounded once).
__device__ inline void split_pair(const Opaque &o, float x, float y, half2v &hi, half2v &lo) {
    hi = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(x, y));
    lo[0] = (_Float16)__builtin_fmaf((float)hi[0], o.minus, x);
    lo[1] = (_Float16)__builtin_fmaf((float)hi[1], o.minus, y);
}

// A lane's raw bytes of a tile.
template <int BITS, int NB>
struct RawTile {
    static constexpr int kUnits = BITS == 4 ? NB / 2 : NB;
    u32x4 k[kUnits], v[kUnits];
    u32x4 ks[NB];         // key scales of positions 8 g + i + 4 t: [i][t][b]
    u32x4 vs[NB];         // value scales of 8 positions

    // From a tile's descriptor: of no bytes where there is no tile, and then all is 0.
    __device__ inline void load(rsrc_t tile, int lane) {
        using T = KvTile<BITS, NB>;
        const int l16 = lane * 16, g16 = (lane >> 4) * 16;
#pragma unroll
        for (int u = 0; u < kUnits; u++) k[u] = load16(tile, l16, u * 1024);
#pragma unroll
        for (int i = 0; i < NB; i++) ks[i] = load16(tile, g16 * NB, T::kScales + i * 16);
#pragma unroll
        for (int u = 0; u < kUnits; u++) v[u] = load16(tile, l16, T::kValues + u * 1024);
#pragma unroll
        for (int b = 0; b < NB; b++) vs[b] = load16(tile, g16, T::kValues + T::kScales + b * 64);
    }
    // Key operand of tile half t, block b: the codes.
    __device__ inline void keys(const Opaque &o, int t, int b, Half8 &c) const {
        if (BITS == 4) {
            q4_key(o, k[b >> 1][t * 2 + (b & 1)], c);
        } else {
            const u32x4 &u = k[(b >> 1) * 2 + t];
            q8_codes(u[(b & 1) * 2], u[(b & 1) * 2 + 1], c);
        }
    }
    // s times the scale of position 8 g + 4 t + i, block b, plus c.
    __device__ inline float scaled(float s, int t, int i, int b, float c) const {
        const int h = (i * 2 + t) * NB + b;
        return __builtin_fmaf(s, (float)pk(ks[h >> 3][h >> 1 & 3])[h & 1], c);
    }
    // Value operand of block b, dims 16 h .. 16 h + 15.
    __device__ inline void values(const Opaque &o, int b, int h, Half8 &hi, Half8 &lo) const {
        Half8 c;
        if (BITS == 4)
            q4_value(o, v[b >> 1][(b & 1) * 2], v[b >> 1][(b & 1) * 2 + 1], h, c);
        else
            q8_codes(v[b][h * 2], v[b][h * 2 + 1], c);
        split_values(c, vs[b], hi, lo);
    }
    // Only positions [first, left) of the lane's eight are any row's.
    __device__ inline void clear_values(int first, int left) {
#pragma unroll
        for (int b = 0; b < NB; b++) clear_scales(vs[b], first, left);
    }
};

// Whether a tile is loaded while another is taken, and the waves a SIMD that
// registers have to leave room for.
template <int BITS, int NB, int ROWS>
constexpr bool kAhead = NB == 4 || (BITS == 4 && ROWS == 8);
template <int NB>
constexpr int kMinWaves = NB == 2 ? 4 : 2;

// A unit of work: a row tile (8, 16 or kManyRows rows) of a sequence and a
// key/value head.  Its rows
// are tokens [i_first, i_last]; the tiles [t_lo, t_hi) hold what they see, of
// which p_lo is the first position.
struct Unit {
    KvSeq sq;
    int rows, i_first, i_last, p_lo, t_lo, t_hi;
    __device__ inline int tiles() const { return max(1, t_hi - t_lo); }  // one that sees nothing is written too
};

// Row tile rt of a sequence; rows is 0 where it has none.
template <int ROWS>
__device__ inline Unit unit_of(const AttnArgs &a, const KvSeq &sq, int rt) {
    Unit u;
    u.sq = sq;
    u.rows = min(ROWS, u.sq.n * a.group - rt * ROWS);
    if (u.rows <= 0) {
        u.rows = u.i_first = u.i_last = u.p_lo = u.t_lo = u.t_hi = 0;
        return u;
    }
    u.i_first = rt * ROWS / a.group;
    u.i_last = (rt * ROWS + u.rows - 1) / a.group;
    const int last = u.sq.first + u.i_last;
    u.p_lo = a.window ? max(0, u.sq.first + u.i_first - a.window + 1) : 0;
    u.t_lo = u.p_lo / kKvTile;
    u.t_hi = last < 0 ? u.t_lo : last / kKvTile + 1;
    if (!u.sq.ok) u.t_lo = u.t_hi = 0;
    return u;
}

// The places of tiles t, t + step, .. of a sequence and head, in scalar
// registers; a page past the table is none.
struct TileWalk {
    struct Place {
        int page, tile;
    };
    KvConst table;
    uint32_t page_bytes, head_bytes, n_pages;
    int tile_bytes, page_tiles, max_pages, at, tile, at_step, tile_step;

    __device__ inline TileWalk(const KvArgs &a, int seq, int head, int t, int step, int bytes) {
        table = kv_const(a.pages) + (int64_t)seq * a.max_pages;
        page_tiles = a.page_tiles;
        tile_bytes = bytes;
        head_bytes = (uint32_t)head * page_tiles * bytes;
        page_bytes = (uint32_t)a.kv_heads * page_tiles * bytes;
        n_pages = (uint32_t)a.n_pages;
        max_pages = a.max_pages;
        at = kv_page_of(a, t, &tile);
        at_step = kv_page_of(a, step, &tile_step);
    }
    __device__ inline Place next() {
        const Place p{at < max_pages ? table[at] : -1, tile};
        at += at_step;
        tile += tile_step;
        if (tile >= page_tiles) tile -= page_tiles, at++;
        return p;
    }
    __device__ inline bool ok(const Place &p) const { return (uint32_t)p.page < n_pages; }
    __device__ inline uint64_t offset(const Place &p) const {
        return (uint64_t)(uint32_t)p.page * page_bytes + (head_bytes + (uint32_t)(p.tile * tile_bytes));
    }
};

// The descriptors of tiles t, t + 1, .. of a sequence and head; the table is
// read a page ahead.
struct TileRun {
    KvConst table;
    const uint8_t *data;
    uint64_t at;  // of the next tile, from data
    uint32_t page_bytes, head_bytes, n_pages;
    int next_page, next_at, max_pages, page_tiles, left, bytes;

    __device__ inline TileRun(const KvArgs &a, int seq, int head, int t, int tile_bytes) {
        table = kv_const(a.pages) + (int64_t)seq * a.max_pages;
        data = a.data;
        page_tiles = a.page_tiles;
        head_bytes = (uint32_t)head * page_tiles * tile_bytes;
        page_bytes = (uint32_t)a.kv_heads * page_tiles * tile_bytes;
        n_pages = (uint32_t)a.n_pages;
        max_pages = a.max_pages;
        int tile;
        next_at = kv_page_of(a, t, &tile);
        next_page = next_at < max_pages ? table[next_at] : -1;
        open(tile_bytes);
        at += (uint32_t)(tile * tile_bytes);
        left -= tile;
    }
    __device__ inline void open(int tile_bytes) {
        at = (uint64_t)(uint32_t)next_page * page_bytes + head_bytes;
        bytes = (uint32_t)next_page < n_pages ? tile_bytes : 0;
        left = page_tiles;
        next_at++;
        next_page = next_at < max_pages ? table[next_at] : -1;
    }
    // bytes: 0 where there is no page
    __device__ inline rsrc_t next(int tile_bytes, int *tile_here) {
        if (left == 0) open(tile_bytes);
        *tile_here = bytes;
        const rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(data + at), (short)0, bytes, kRsrcWord3);
        at += (uint32_t)tile_bytes;
        left--;
        return r;
    }
};

// The workspace: each unit's first and last part, each part's (maximum, sum)
// of its rows, and its rows' partial outputs.
struct AttnWork {
    int2 *units;
    float2 *tops;  // [part][unit_rows]
    float *outs;   // [part][unit_rows][dim]
};
__device__ inline AttnWork attn_work(const AttnArgs &a) {
    const int64_t units = (int64_t)a.kv.n_seqs * a.row_tiles * a.kv.kv_heads;
    AttnWork w;
    w.units = reinterpret_cast<int2 *>(a.work);
    w.tops = reinterpret_cast<float2 *>(w.units + (units + 1) / 2 * 2);  // outputs are stored by 16 bytes
    w.outs = reinterpret_cast<float *>(w.tops + (a.groups + units) * a.unit_rows);
    return w;
}

// A head's sink logit (times log2 e; -inf: none).
__device__ inline float sink_of(const AttnArgs &a, int head) {
    return a.sinks ? bias_at(a.sinks, a.sink_type, (uint64_t)head) * 1.44269504088896341f : -__builtin_inff();
}

// What a row's sum of weighted values is multiplied by: one over the sum l of
// its weights (held times 2^-m) and the sink's.  A row that sees nothing is 0.
__device__ inline float row_scale(float l, float m, float sink) {
    const float top = fmaxf(m, sink), f = __builtin_amdgcn_exp2f(m - top);
    l = l * f + __builtin_amdgcn_exp2f(sink - top);
    return l == 0.0f ? 0.0f : f / l;
}

// A row's block of 32 (an element a lane of a half-wave) as output and Q8_0.
__device__ inline void store_block(const AttnArgs &a, int head, int64_t row, int b, int nb, float v, int lane, bool ok) {
    const int64_t blk = (row * a.heads + head) * nb + b;
    if (ok) a.out[blk * 32 + (lane & 31)] = v;
    if (a.q8) {
        uint16_t dh;
        const int q = q8_quantize_half(v, lane, &dh);
        if (ok) write_q8_lane(q, dh, lane & 31, (size_t)blk, nullptr, nullptr, nullptr, a.q8);
    }
}

// A block of 32 as Q8_0 by four lanes: lane i of them has elements 8 i on.  The
// arithmetic of q8_quantize_half (a NaN's bits are above every number's).  (Five
// prompts of up to 1,021 with a window: 52 us, 78 with an element a lane, 48 without blocks.)
__device__ inline void store_q8_quad(const float *v, int i, uint8_t *to) {
    float x[8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = v[j], m = max(m, __float_as_uint(__builtin_fabsf(x[j])));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
    const float d = m > 0x7F800000u ? __builtin_nanf("") : __uint_as_float(m) / 127.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    struct __attribute__((packed, aligned(2))) Codes {
        uint32_t w[2];
    } codes = {};
#pragma unroll
    for (int j = 0; j < 8; j++) codes.w[j >> 2] |= (uint32_t)(q8_code(x[j] * id) & 255) << (8 * (j & 3));
    if (!to) return;
    if (i == 0) *reinterpret_cast<uint16_t *>(to) = f32_to_f16_bits(d);
    *reinterpret_cast<Codes *>(to + 2 + 8 * i) = codes;
}

// A row of queries as the B operand, times the softmax scale, hi and lo; the
// products are scores (times log2 e) divided by mul.
template <int NB>
struct Query {
    Half8 hi[NB], lo[NB];
    float mul;
    __device__ inline void load(const AttnArgs &a, int64_t row, int head, int g) {
        float x[NB][8], top = 0.0f;
        const float *src = a.q + (row * a.heads + head) * 32 * NB + 8 * g;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const float4 u = *reinterpret_cast<const float4 *>(src + 32 * b), w = *reinterpret_cast<const float4 *>(src + 32 * b + 4);
            x[b][0] = u.x, x[b][1] = u.y, x[b][2] = u.z, x[b][3] = u.w;
            x[b][4] = w.x, x[b][5] = w.y, x[b][6] = w.z, x[b][7] = w.w;
#pragma unroll
            for (int i = 0; i < 8; i++) x[b][i] *= a.scale;
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, __builtin_fabsf(x[b][i]));
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        // mul is a power of two, so that scores times it are exact: the largest
        // minus the maximum is 0 however large they are.  (Not so small that it
        // is 0: it multiplies the -inf of hidden positions.)
        const int e = max(-100, __builtin_amdgcn_frexp_expf(top));
        mul = __builtin_ldexpf(1.0f, e - 13);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = __builtin_ldexpf(x[b][i], 13 - e);
                hi[b].v[i] = (_Float16)y;
                lo[b].v[i] = (_Float16)(y - (float)hi[b].v[i]);
            }
    }
};

template <int NB, int WAVES>
struct AttnLds {
    float o[WAVES][16][32 * NB + 4];  // by column
    float m[WAVES][16], l[WAVES][16], sink[16];
};

// The value of lane ^ 8, of each row of 16 lanes.
__device__ inline float other8(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xF, 0xF, false));
}
__device__ inline half2v other8(half2v x) {
    return pk((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__builtin_bit_cast(uint32_t, x), 0x128, 0xF, 0xF, false));
}

// Tiles [t_begin, t_end) of a unit by the workgroup; the result is the unit's
// own (part < 0), or that part of it.
//
// ROWS 16: a row a column.  ROWS 8 (up to eight rows, a token of eight heads
// for instance): columns c and c + 8 are a row's, one multiplied by the hi half of
// the query or the weights and the other by the lo half, which takes a half
// to two thirds of the MFMAs.  The two lanes add their halves of a score
// and take half of the tile's positions each through the softmax.
template <int BITS, int NB, int ROWS, int WAVES>
__device__ __attribute__((always_inline)) inline void attend(const AttnArgs &a, const Unit &un, int seq, int rt, int kvh, int t_begin, int t_end,
                                                             int64_t part, AttnLds<NB, WAVES> &lds) {
    using T = KvTile<BITS, NB>;
    constexpr int kDim = 32 * NB;
    const KvSeq &sq = un.sq;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int t = t_begin + wave;
    TileWalk walk(a.kv, seq, kvh, t, WAVES, T::kBytes);
    // Loads are issued on every path: the compiler waits for all of them where
    // paths join.
    auto load = [&](RawTile<BITS, NB> &raw, const TileWalk::Place &p) __attribute__((always_inline)) {
        raw.load(__builtin_amdgcn_make_buffer_rsrc(a.kv.data + walk.offset(p), (short)0, walk.ok(p) ? T::kBytes : 0, kRsrcWord3), lane);
    };
    RawTile<BITS, NB> even;
    TileWalk::Place p0 = walk.next(), p1 = walk.next();
    load(even, p0);

    // the row of this lane's column
    constexpr bool kPack = ROWS == 8;
    const bool upper = kPack && col >= 8;
    const int flat = rt * ROWS + col % ROWS;
    const bool row_ok = col % ROWS < un.rows;
    const int tok = row_ok ? flat / a.group : un.i_last, hd = kvh * a.group + (row_ok ? flat % a.group : 0);
    const int pos = sq.first + tok;                   // last position that it sees
    const int from = a.window ? pos - a.window : -1;  // it sees those after this one

    Query<NB> q;
    const float sink = sink_of(a, hd);
    q.load(a, sq.r0 + tok, hd, g);
    if (kPack) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) q.hi[b].h[i] = upper ? q.lo[b].h[i] : q.hi[b].h[i];
    }

    const Opaque oc;
    f32x4 o[NB][2];
#pragma unroll
    for (int b = 0; b < NB; b++) o[b][0] = o[b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = kNoMax, l = sq.ok ? 0.0f : __builtin_nanf("");
    // A tile's part, from its bytes in registers.
    auto take = [&](RawTile<BITS, NB> &raw, const TileWalk::Place &at) __attribute__((always_inline)) {
        const int p0 = t * kKvTile;
        if (!walk.ok(at)) {
            if (p0 <= pos && p0 + kKvTile - 1 > from) l = __builtin_nanf("");
            return;
        }
        float x[8] = {}, top = -__builtin_inff();
        const bool whole = p0 + kKvTile - 1 <= sq.first + un.i_first && (!a.window || p0 > sq.first + un.i_last - a.window);
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                Half8 c;
                raw.keys(oc, h, b, c);
                f32x4 s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (!kPack) s = mfma(c, q.lo[b], s);
                s = mfma(c, q.hi[b], s);
#pragma unroll
                for (int i = 0; i < 4; i++) x[4 * h + i] = raw.scaled(s[i], h, i, b, b ? x[4 * h + i] : oc.zero);
            }
        }
        // the lane's positions begin here, x[0 .. kMine) are theirs
        constexpr int kMine = kPack ? 4 : 8;
        const int mine = p0 + 8 * g + (upper ? 4 : 0);
        if (kPack) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float keep = upper ? x[4 + i] : x[i], give = upper ? x[i] : x[4 + i];
                x[i] = keep + other8(give);
            }
        }
        if (!whole) {
            asm volatile("");  // a branch: the whole tiles, nearly all, do without
#pragma unroll
            for (int j = 0; j < kMine; j++) {
                const int p = mine + j;
                x[j] = p <= pos && p > from ? x[j] : -__builtin_inff();
            }
            raw.clear_values(un.p_lo - p0 - 8 * g, sq.end - p0 - 8 * g);
        }
#pragma unroll
        for (int j = 0; j < kMine; j++) top = fmaxf(top, x[j]);
        top *= q.mul;
        if (__any(top > m + kSlack)) {
            if (kPack) top = fmaxf(top, other8(top));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float nm = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - nm);
            m = nm;
            l *= f;
#pragma unroll
            for (int b = 0; b < NB; b++) o[b][0] *= f, o[b][1] *= f;
        }
        Half8 ph, pl;
        const float back = kLift - m;
        float sums[kMine / 2];
#pragma unroll
        for (int j = 0; j < kMine; j += 2) {
            const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], q.mul, back)), w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j + 1], q.mul, back));
            sums[j >> 1] = w0 + w1;
            split_pair(oc, w0, w1, ph.h[j >> 1], pl.h[j >> 1]);
        }
        l += kPack ? sums[0] + sums[1] : (sums[0] + sums[1]) + (sums[kMine / 2 - 2] + sums[kMine / 2 - 1]);
        if (kPack) {
            // the hi column's weights of all positions, and the lo column's
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const half2v got = other8(upper ? ph.h[i] : pl.h[i]);
                ph.h[2 + i] = upper ? pl.h[i] : got;
                ph.h[i] = upper ? got : ph.h[i];
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                Half8 vh, vl;
                raw.values(oc, b, h, vh, vl);
                o[b][h] = mfma(vh, ph, o[b][h]);
                if (!kPack) o[b][h] = mfma(vh, pl, o[b][h]);
                o[b][h] = mfma(vl, ph, o[b][h]);
            }
    };
    // What is summed up goes to this wave's place in LDS, and sums and maximum
    // begin anew.
    bool kept = false;
    int left = kFewChunk;
    auto join = [&]() __attribute__((always_inline)) {
        if (kPack) l += other8(l);
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (!kept) return;
        const float top = fmaxf(m, lds.m[wave][col]), f = __builtin_amdgcn_exp2f(m - top), fk = __builtin_amdgcn_exp2f(lds.m[wave][col] - top);
        m = top;
        l = l * f + lds.l[wave][col] * fk;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) o[b][h] = o[b][h] * f + *reinterpret_cast<const f32x4 *>(&lds.o[wave][col][32 * b + 16 * h + 4 * g]) * fk;
    };
    auto keep = [&]() __attribute__((always_inline)) {
        asm volatile("");  // a branch
        join();
        // (every lane reads back what it wrote itself)
        lds.m[wave][col] = m, lds.l[wave][col] = l;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                *reinterpret_cast<f32x4 *>(&lds.o[wave][col][32 * b + 16 * h + 4 * g]) = o[b][h];
                o[b][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        m = kNoMax, l = 0.0f;
        kept = true;
        left = kFewChunk;
    };
    if (kAhead<BITS, NB, ROWS>) {
        // two tiles in registers, one being loaded while the other is taken
        RawTile<BITS, NB> odd;
        while (t < t_end) {
            if (left <= 0) keep();
            left -= 2;
            load(odd, p1);
            const TileWalk::Place p2 = walk.next();
            take(even, p0);
            t += WAVES;
            if (t >= t_end) break;
            load(even, p2);
            const TileWalk::Place p3 = walk.next();
            take(odd, p1);
            t += WAVES;
            p0 = p2;
            p1 = p3;
        }
    } else {
        for (; t < t_end; t += WAVES) {
            if (left == 0) keep();
            left--;
            take(even, p0);
            p0 = p1;
            p1 = walk.next();
            load(even, p0);
        }
    }

    // the waves' parts, on the largest maximum
    join();
    if (g == 0) lds.m[wave][col] = m, lds.l[wave][col] = l, lds.sink[col] = sink;
    __syncthreads();
    float top = lds.m[0][col];
#pragma unroll
    for (int w = 1; w < WAVES; w++) top = fmaxf(top, lds.m[w][col]);
    const float f = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int h = 0; h < 2; h++) *reinterpret_cast<f32x4 *>(&lds.o[wave][col][32 * b + 16 * h + 4 * g]) = o[b][h] * f;
    __syncthreads();
    // a half-wave takes a block of a row
    for (int u = wave * 2 + (lane >> 5); u < ROWS * NB; u += 2 * WAVES) {
        const int r = u / NB, b = u % NB, d = 32 * b + (lane & 31);
        float mx = lds.m[0][r], sum = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 1; w < WAVES; w++) mx = fmaxf(mx, lds.m[w][r]);
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            den += lds.l[w][r] * __builtin_amdgcn_exp2f(lds.m[w][r] - mx);
            sum += lds.o[w][r][d];
            if (kPack) sum += lds.o[w][r + 8][d];
        }
        mx -= kLift;  // weights are 2^kLift too large, the sink is not
        const int fr = rt * ROWS + r;
        const bool ok = r < un.rows;
        if (part < 0) {
            store_block(a, kvh * a.group + fr % a.group, sq.r0 + fr / a.group, b, NB, sum * row_scale(den, mx, lds.sink[r]), lane, ok);
        } else if (ok) {
            const AttnWork w = attn_work(a);
            w.outs[(part * ROWS + r) * kDim + d] = sum;
            if (d == 0) w.tops[part * ROWS + r] = make_float2(mx, den);
        }
    }
}

// A workgroup a unit.
template <int BITS, int NB, int ROWS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, kMinWaves<NB>) void k_attn_units(AttnArgs a) {
    __shared__ AttnLds<NB, WAVES> lds;
    const int kvh = blockIdx.x % a.kv.kv_heads, rt = blockIdx.x / a.kv.kv_heads, seq = blockIdx.y;
    const Unit u = unit_of<ROWS>(a, kv_seq(a.kv, seq), rt);
    if (u.rows) attend<BITS, NB, ROWS, WAVES>(a, u, seq, rt, kvh, u.t_lo, u.t_hi, -1, lds);
}

// A workgroup a part of a unit: split_tiles of its position tiles (all, where
// it has no more).
template <int BITS, int NB, int ROWS>
__global__ __launch_bounds__(64 * kWaves, kMinWaves<NB>) void k_attn_parts(AttnArgs a) {
    __shared__ AttnLds<NB, kWaves> lds;
    const int kvh = blockIdx.x % a.kv.kv_heads, x = blockIdx.x / a.kv.kv_heads, rt = x % a.row_tiles, split = x / a.row_tiles, seq = blockIdx.y;
    const Unit u = unit_of<ROWS>(a, kv_seq(a.kv, seq), rt);
    const int t0 = u.t_lo + split * a.split_tiles, n = (u.tiles() + a.split_tiles - 1) / a.split_tiles;
    if (u.rows == 0 || split >= n) return;
    const int64_t unit = ((int64_t)seq * a.row_tiles + rt) * a.kv.kv_heads + kvh, first = unit * (a.splits - 1);
    // the part of number x is at x + unit
    if (split == 0 && threadIdx.x == 0) attn_work(a).units[unit] = n == 1 ? make_int2(0, 0) : make_int2((int)first, (int)first + n - 1);
    attend<BITS, NB, ROWS, kWaves>(a, u, seq, rt, kvh, t0, min(u.t_hi, t0 + a.split_tiles), n == 1 ? -1 : first + unit + split, lds);
}

// Rows many at a time: a workgroup's 4 waves have 32 rows each (two columns of
// the MFMA), and share the tiles' operands, made once a workgroup in LDS: key
// codes, and values as hi and lo.  While one tile is taken from one buffer, the
// next is made in the other and the bytes of the one after it are on their
// way.  Each wave makes a quarter of a tile: a unit is a key or value operand of
// one MFMA, 1 KB or twice 1 KB.
constexpr int kManyWaves = 4, kManyRows = 32 * kManyWaves;

template <int NB>
struct ManyLds {
    struct Buffer {
        Half8 k[2 * NB][64];     // [t][b][lane]
        Half8 v[2 * NB][2][64];  // [b][h][hi, lo][lane]
        u32x4 ks[4 * NB];        // scales as they are stored
    };
    union {
        Buffer buf[2];
        float o[kManyWaves][16][32 * NB + 4];
    };
    float2 kept[2][kManyWaves][16];  // maximum and sum of what is kept
};

// Whether the batch's rows fall somewhere: only then can a row be two sequences'.
__device__ inline bool rows_fall(const KvArgs &a) {
    int fall = 0;
    for (int s = threadIdx.x; s < a.n_seqs; s += 64 * kManyWaves) fall |= a.rows[s + 1] < a.rows[s];
    return __syncthreads_or(fall) != 0;
}

// A wave's part of a tile: NB units of keys (waves 0 and 1) or values (2 and 3).
template <int BITS, int NB>
struct ManyPart {
    static constexpr int kHalf = kManyWaves / 2, kUnits = 2 * NB / kHalf;  // waves for keys, units of each
    uint2 c[kUnits];
    u32x4 d[kUnits];  // values: scales of eight positions; keys: all scales, by the first lanes
    bool ok;

    static __device__ inline uint2 load8(rsrc_t tile, int lane_at, int at) {
        return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(tile, lane_at, at, 0));
    }
    __device__ inline void load(rsrc_t tile, bool page_ok, int wave, int lane) {
        using T = KvTile<BITS, NB>;
        ok = page_ok;
#pragma unroll
        for (int j = 0; j < kUnits; j++) {
            const int u = wave % kHalf * kUnits + j;
            if (wave < kHalf) {
                const int t = u / NB, b = u % NB;
                if (BITS == 4)
                    c[j].x = __builtin_amdgcn_raw_buffer_load_b32(tile, lane * 16, (b >> 1) * 1024 + t * 8 + (b & 1) * 4, 0);
                else
                    c[j] = load8(tile, lane * 16, ((b >> 1) * 2 + t) * 1024 + (b & 1) * 8);
                if (j == 0) d[j] = load16(tile, (lane & (4 * NB - 1)) * 16, T::kScales);
            } else {
                const int b = u >> 1, h = u & 1;
                c[j] = BITS == 4 ? load8(tile, lane * 16, T::kValues + (b >> 1) * 1024 + (b & 1) * 8)
                                 : load8(tile, lane * 16, T::kValues + b * 1024 + h * 8);
                d[j] = load16(tile, (lane >> 4) * 16, T::kValues + T::kScales + b * 64);
            }
        }
    }
    // Positions [first, left) of the tile are some row's.
    __device__ inline void make(const Opaque &o, typename ManyLds<NB>::Buffer &buf, int first, int left, int wave, int lane) {
#pragma unroll
        for (int j = 0; j < kUnits; j++) {
            const int u = wave % kHalf * kUnits + j;
            if (wave < kHalf) {
                Half8 k;
                if (BITS == 4)
                    q4_key(o, c[j].x, k);
                else
                    q8_codes(c[j].x, c[j].y, k);
                buf.k[u][lane] = k;
                // no page: the scores are NaN
                if (u == 0 && lane < 4 * NB) buf.ks[lane] = ok ? d[j] : u32x4{0x7E007E00u, 0x7E007E00u, 0x7E007E00u, 0x7E007E00u};
            } else {
                Half8 v, hi, lo;
                if (BITS == 4) {
                    const int down = 4 * (u & 1);  // the upper nibbles moved to the lower's place
                    q4_value(o, c[j].x >> down, c[j].y >> down, 0, v);
                } else {
                    q8_codes(c[j].x, c[j].y, v);
                }
                if (first > 0 || left < kKvTile) {
                    asm volatile("");  // a branch: few tiles are an end
                    clear_scales(d[j], first - 8 * (lane >> 4), left - 8 * (lane >> 4));
                }
                split_values(v, d[j], hi, lo);
                buf.v[u][0][lane] = hi;
                buf.v[u][1][lane] = lo;
            }
        }
    }
};

template <int BITS, int NB, bool CHUNKS>
__device__ __attribute__((always_inline)) inline void attend_many(const AttnArgs &a, const Unit &un, int seq, int rt, int kvh, int t_begin,
                                                                  int t_end, int64_t part, ManyLds<NB> &lds) {
    using T = KvTile<BITS, NB>;
    constexpr int kDim = 32 * NB;
    const KvSeq &sq = un.sq;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // tiles that are summed up together: all of them where another sequence may
    // claim the rows too, which then hold one of the two results and no mixture
    int chunk = kManyChunk;
    if (CHUNKS && part < 0 && t_end - t_begin > kManyChunk && rows_fall(a.kv)) chunk = INT_MAX - 1;
    TileRun run(a.kv, seq, kvh, t_begin, T::kBytes);
    ManyPart<BITS, NB> raw;
    auto load = [&]() __attribute__((always_inline)) {
        int bytes;
        const rsrc_t tile = run.next(T::kBytes, &bytes);
        raw.load(tile, bytes != 0, wave, lane);
    };
    load();

    // this wave's rows: two columns' rows a lane
    const int row0 = rt * kManyRows + wave * 32, rows = un.rows - wave * 32;
    const int i0 = row0 / a.group, i1 = (row0 + min(rows, 32) - 1) / a.group;  // its tokens
    const int pos0 = sq.first + i0, pos1 = sq.first + i1;
    int pos[2], from[2];
    float sink[2];
    Query<NB> q[2];
    f32x4 o[2][NB][2];
    float m[2] = {kNoMax, kNoMax}, l[2];
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const int r = 16 * c + col;
        const bool ok = r < rows;
        const int tok = ok ? (row0 + r) / a.group : un.i_last, hd = kvh * a.group + (ok ? (row0 + r) % a.group : 0);
        pos[c] = sq.first + tok;
        from[c] = a.window ? pos[c] - a.window : -1;
        sink[c] = sink_of(a, hd);
        q[c].load(a, sq.r0 + tok, hd, g);
        l[c] = sq.ok ? 0.0f : __builtin_nanf("");
#pragma unroll
        for (int b = 0; b < NB; b++) o[c][b][0] = o[c][b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const Opaque oc;

    // The tiles that any of this wave's rows sees (the others are made for the
    // other waves), and those of them that all its rows see whole.
    const int w_begin = a.window ? max(0, pos0 - a.window + 1) / kKvTile : 0;
    const int w_end = rows <= 0 || pos1 < 0 ? 0 : pos1 / kKvTile + 1;
    const int whole_begin = a.window ? (max(0, pos1 - a.window + 1) + kKvTile - 1) / kKvTile : 0;
    const int whole_end = (max(-1, pos0) + 1) / kKvTile;
    auto take = [&](const typename ManyLds<NB>::Buffer &buf, int t) __attribute__((always_inline)) {
        if (t < w_begin || t >= w_end) return;
        const int p0 = t * kKvTile;
        u32x4 ks[NB];
#pragma unroll
        for (int i = 0; i < NB; i++) ks[i] = buf.ks[g * NB + i];
        float x[2][8];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const Half8 k = buf.k[h * NB + b][lane];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    f32x4 s = mfma(k, q[c].lo[b], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                    s = mfma(k, q[c].hi[b], s);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int n = (i * 2 + h) * NB + b;
                        x[c][4 * h + i] = __builtin_fmaf(s[i], (float)pk(ks[n >> 3][n >> 1 & 3])[n & 1], b ? x[c][4 * h + i] : oc.zero);
                    }
                }
            }
        if (t < whole_begin || t >= whole_end) {
            asm volatile("");
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int p = p0 + 8 * g + j;
                    x[c][j] = p <= pos[c] && p > from[c] ? x[c][j] : -__builtin_inff();
                }
        }
        float top[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            top[c] = x[c][0];
#pragma unroll
            for (int j = 1; j < 8; j++) top[c] = fmaxf(top[c], x[c][j]);
            top[c] *= q[c].mul;
        }
        if (__any(top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                top[c] = fmaxf(top[c], __shfl_xor(top[c], 16));
                top[c] = fmaxf(top[c], __shfl_xor(top[c], 32));
                const float nm = fmaxf(m[c], top[c]), f = __builtin_amdgcn_exp2f(m[c] - nm);
                m[c] = nm;
                l[c] *= f;
#pragma unroll
                for (int b = 0; b < NB; b++) o[c][b][0] *= f, o[c][b][1] *= f;
            }
        }
        Half8 ph[2], pl[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const float back = kLift - m[c];
            float sums[4];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[c][j], q[c].mul, back));
                const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[c][j + 1], q[c].mul, back));
                sums[j >> 1] = w0 + w1;
                split_pair(oc, w0, w1, ph[c].h[j >> 1], pl[c].h[j >> 1]);
            }
            l[c] += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const Half8 vh = buf.v[b * 2 + h][0][lane], vl = buf.v[b * 2 + h][1][lane];
#pragma unroll
                for (int c = 0; c < 2; c++) o[c][b][h] = mfma(vh, ph[c], o[c][b][h]);
#pragma unroll
                for (int c = 0; c < 2; c++) o[c][b][h] = mfma(vh, pl[c], o[c][b][h]);
#pragma unroll
                for (int c = 0; c < 2; c++) o[c][b][h] = mfma(vl, ph[c], o[c][b][h]);
            }
    };

    // What is summed up goes to the row's own place in the output (the part's, in
    // the workspace), and sums and maximum begin anew: registers and LDS hold no
    // second output.  (Opaque: the loop would carry what the address takes.)
    bool kept = false;
    auto kept_at = [&](int c) __attribute__((always_inline)) {
        int first = row0;
        asm volatile("" : "+s"(first));
        const int fr = first + 16 * c + col;
        const int64_t place = part < 0 ? (int64_t)(sq.r0 + fr / a.group) * a.heads + kvh * a.group + fr % a.group : part * kManyRows + fr - rt * kManyRows;
        return (part < 0 ? a.out : attn_work(a).outs) + place * kDim + 4 * g;
    };
    auto join = [&](int c) __attribute__((always_inline)) {
        l[c] += __shfl_xor(l[c], 16);
        l[c] += __shfl_xor(l[c], 32);
        if (!kept) return;
        const float2 was = lds.kept[c][wave][col];
        const float top = fmaxf(m[c], was.x), f = __builtin_amdgcn_exp2f(m[c] - top), fk = __builtin_amdgcn_exp2f(was.x - top);
        m[c] = top;
        l[c] = l[c] * f + was.y * fk;
        const float *from = kept_at(c);
        if (16 * c + col < rows) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) o[c][b][h] = o[c][b][h] * f + *reinterpret_cast<const f32x4 *>(from + 32 * b + 16 * h) * fk;
        }
    };
    auto keep = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            join(c);
            // (every lane reads back what it wrote itself)
            lds.kept[c][wave][col] = make_float2(m[c], l[c]);
            float *to = kept_at(c);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (16 * c + col < rows) *reinterpret_cast<f32x4 *>(to + 32 * b + 16 * h) = o[c][b][h];
                    o[c][b][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            m[c] = kNoMax, l[c] = 0.0f;
        }
        kept = true;
    };

    raw.make(oc, lds.buf[0], un.p_lo - t_begin * kKvTile, sq.end - t_begin * kKvTile, wave, lane);
    load();
    lds_barrier();
    auto step = [&](int t, int now) __attribute__((always_inline)) {
        raw.make(oc, lds.buf[now ^ 1], un.p_lo - (t + 1) * kKvTile, sq.end - (t + 1) * kKvTile, wave, lane);
        load();
        take(lds.buf[now], t);
        lds_barrier();
    };
    for (int t = t_begin, left = chunk; t < t_end; t += 2, left -= 2) {
        if (CHUNKS && left == 0) {
            asm volatile("");  // a branch
            keep();
            left = chunk;
        }
        step(t, 0);
        if (t + 1 < t_end) step(t + 1, 1);
    }

#pragma unroll
    for (int c = 0; c < 2; c++) {
        join(c);
        m[c] -= kLift;  // weights are 2^kLift too large, the sink is not
        const AttnWork w = attn_work(a);
        const int64_t at = part * kManyRows + wave * 32 + 16 * c;  // the part's rows
        const float f = part < 0 ? row_scale(l[c], m[c], sink[c]) : 1.0f;
        if (part >= 0 && g == 0 && 16 * c + col < rows) w.tops[at + col] = make_float2(m[c], l[c]);
        // through LDS, so that a row's output is stored by consecutive lanes
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) *reinterpret_cast<f32x4 *>(&lds.o[wave][col][32 * b + 16 * h + 4 * g]) = o[c][b][h] * f;
        lds_barrier();
        // the output's row of this lane's column, to be had from lane r for row r
        const int fr = row0 + 16 * c + col;
        const int64_t place = part < 0 ? (int64_t)(sq.r0 + fr / a.group) * a.heads + kvh * a.group + fr % a.group : at + col;
        float *const outs = part < 0 ? a.out : w.outs;
        constexpr int kQuads = kDim / 4;
#pragma unroll
        for (int i = 0; i < 16 * kQuads; i += 64) {
            const int u = i + lane, r = u / kQuads, d = u % kQuads * 4;
            const int64_t to = __shfl(place, r);
            if (16 * c + r < rows) *reinterpret_cast<f32x4 *>(outs + to * kDim + d) = *reinterpret_cast<const f32x4 *>(&lds.o[wave][r][d]);
        }
        if (a.q8 && part < 0) {
            // four lanes a block, the blocks of 16 / NB rows at a time
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const int blk = i * 16 + (lane >> 2), r = blk / NB, b = blk % NB;
                const int64_t to = __shfl(place, r);
                store_q8_quad(&lds.o[wave][r][32 * b + 8 * (lane & 3)], lane & 3, 16 * c + r < rows ? a.q8 + (to * NB + b) * 34 : nullptr);
            }
        }
        lds_barrier();
    }
}

// A workgroup a unit, the last row tiles first: the causal ones with the most
// tiles, so that the short ones even out the end.  Heads of 64 at three waves a
// SIMD (a prompt of 2,048: 101 us, at two 124).  CHUNKS: rows of more than
// kManyChunk tiles.
template <int BITS, int NB, bool CHUNKS>
__global__ __launch_bounds__(64 * kManyWaves, NB == 2 ? 3 : 2) void k_attn_many(AttnArgs a) {
    __shared__ ManyLds<NB> lds;
    const int kvh = blockIdx.x % a.kv.kv_heads, seq = blockIdx.y;
    const KvSeq sq = kv_seq(a.kv, seq);
    const int rt = (sq.n * a.group + kManyRows - 1) / kManyRows - 1 - (int)(blockIdx.x / a.kv.kv_heads);
    if (rt < 0) return;
    const Unit u = unit_of<kManyRows>(a, sq, rt);
    attend_many<BITS, NB, CHUNKS>(a, u, seq, rt, kvh, u.t_lo, u.t_hi, -1, lds);
}

// All units' tiles in a row, cut into equal shares, one a workgroup: however
// unequal the sequences are, the workgroups end together.  A unit counts
// kUnitCost tiles more than it has, for its beginning and end.  Every workgroup
// sums up the units by itself.  The parts of a unit that several workgroups
// share are numbered (workgroup + unit): along the row each part begins a new
// workgroup or a new unit.
constexpr int kUnitCost = 16, kManyCost = 2;
template <int BITS, int NB, int ROWS>
__global__ __launch_bounds__(64 * (ROWS == kManyRows ? kManyWaves : kWaves), ROWS == kManyRows ? 2 : kMinWaves<NB>) void k_attn_shares(AttnArgs a) {
    constexpr bool MANY = ROWS == kManyRows;
    constexpr int kCost = MANY ? kManyCost : kUnitCost;
    constexpr int kGroupWaves = MANY ? kManyWaves : kWaves, kThreads = 64 * kGroupWaves, kEach = kAttnEntries / kThreads;
    __shared__ std::conditional_t<MANY, ManyLds<NB>, AttnLds<NB, kWaves>> lds;
    __shared__ int before[kAttnEntries + 1];  // cost of a head before each (sequence, row tile)
    __shared__ int wave_sum[kGroupWaves];
    const int entries = a.kv.n_seqs * a.row_tiles, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int n[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const int e = tid * kEach + i;
        n[i] = 0;
        if (e < entries) {
            const int q = e / a.row_tiles;
            const Unit u = unit_of<ROWS>(a, kv_seq(a.kv, a.kv.rows[q], a.kv.rows[q + 1], a.kv.lens[q]), e % a.row_tiles);
            n[i] = u.rows ? u.tiles() + kCost : 0;
        }
        sum += n[i];
    }
    int scan = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int x = __shfl_up(scan, d);
        if (lane >= d) scan += x;
    }
    if (lane == 63) wave_sum[wave] = scan;
    __syncthreads();
    int at = scan - sum, total = 0;
#pragma unroll
    for (int w = 0; w < kGroupWaves; w++) {
        if (w < wave) at += wave_sum[w];
        total += wave_sum[w];
    }
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        before[tid * kEach + i] = at;
        at += n[i];
    }
    if (tid == kThreads - 1) before[kAttnEntries] = at;
    __syncthreads();
    const int64_t all = (int64_t)__builtin_amdgcn_readfirstlane(total) * a.kv.kv_heads;
    // fewer workgroups where they would have less than a unit's cost
    const int64_t groups = min((int64_t)a.groups, max((int64_t)1, all / kCost)), b = blockIdx.x;
    if (b >= groups) return;
    const int64_t end = (b + 1) * all / groups;
    int64_t x = b * all / groups;
    // the entry of x: the last with before[e] * kv_heads <= x
    int e = 0;
    if (x < end) {
        int lo = 0, hi = entries;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((int64_t)before[mid] * a.kv.kv_heads <= x) lo = mid; else hi = mid;
        }
        e = lo;
    }
    while (x < end) {
        e = __builtin_amdgcn_readfirstlane(e);
        const int64_t first = (int64_t)__builtin_amdgcn_readfirstlane(before[e]) * a.kv.kv_heads;
        const int cost = __builtin_amdgcn_readfirstlane(before[e + 1] - before[e]);
        const int kvh = cost ? __builtin_amdgcn_readfirstlane((int)((x - first) / cost)) : a.kv.kv_heads;
        if (kvh >= a.kv.kv_heads) {
            e++;
            continue;
        }
        const int64_t u0 = first + (int64_t)kvh * cost, u1 = u0 + cost, stop = min(end, u1);
        // its tiles begin after its cost; a share that ends there has none
        const int64_t tile0 = u0 + kCost;
        if (stop > tile0) {
            const int seq = e / a.row_tiles, rt = e % a.row_tiles;
            const Unit u = unit_of<ROWS>(a, kv_seq(a.kv, seq), rt);
            const int64_t unit = (int64_t)e * a.kv.kv_heads + kvh;
            const bool begins = x <= tile0, alone = begins && stop == u1;
            // the last workgroup whose share begins before u1
            if (begins && tid == 0) attn_work(a).units[unit] = alone ? make_int2(0, 0) : make_int2((int)b, (int)((u1 * groups - 1) / all));
            const int t0 = u.t_lo + (int)(max(x, tile0) - tile0), t1 = min(u.t_hi, u.t_lo + (int)(stop - tile0));
            const int64_t part = alone ? -1 : b + unit;
            if constexpr (MANY)
                attend_many<BITS, NB, true>(a, u, seq, rt, kvh, t0, t1, part, lds);
            else
                attend<BITS, NB, ROWS, kWaves>(a, u, seq, rt, kvh, t0, t1, part, lds);
            __syncthreads();
        }
        x = stop;
    }
}

// The parts of units that workgroups shared: kMergeThreads take `rows` rows at
// a time, the threads left over share a row's parts.
constexpr int kMergeThreads = 512;
template <int NB>
__global__ __launch_bounds__(kMergeThreads) void k_attn_merge(AttnArgs a, int rows) {
    constexpr int kDim = 32 * NB;
    __shared__ float sum[kMergeThreads];
    const AttnWork w = attn_work(a);
    const int chunks = a.unit_rows / rows, chunk = blockIdx.x % chunks;
    const int64_t unit = blockIdx.x / chunks;
    const int e = (int)(unit / a.kv.kv_heads), kvh = (int)(unit % a.kv.kv_heads), seq = e / a.row_tiles, rt = e % a.row_tiles;
    const KvSeq sq = kv_seq(a.kv, seq);
    const int n_rows = min(a.unit_rows, sq.n * a.group - rt * a.unit_rows);
    const int2 wg = w.units[unit];  // (read beside the sequence; of no unit where it has no rows)
    if (chunk * rows >= n_rows) return;
    const int n = wg.y - wg.x + 1;
    if (n <= 1) return;
    const int tid = threadIdx.x, lane = tid & 63, d = tid % kDim, groups = kMergeThreads / kDim / rows;
    const int gr = tid / kDim % groups, r = min(chunk * rows + tid / kDim / groups, n_rows - 1);
    const float2 *top = w.tops + (wg.x + unit) * a.unit_rows + r;
    const float *out = w.outs + ((wg.x + unit) * a.unit_rows + r) * kDim + d;
    float m = kNoMax, l = 0.0f, o = 0.0f;
    for (int i = lane; i < n; i += 64) m = fmaxf(m, top[i * a.unit_rows].x);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    for (int i = lane; i < n; i += 64) {
        const float2 t = top[i * a.unit_rows];
        l += t.y * __builtin_amdgcn_exp2f(t.x - m);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
#pragma unroll 8
    for (int i = gr; i < n; i += groups) o += out[(int64_t)i * a.unit_rows * kDim] * __builtin_amdgcn_exp2f(top[i * a.unit_rows].x - m);
    if (groups > 1) {
        sum[tid] = o;
        __syncthreads();
        if (gr) return;
        for (int i = 1; i < groups; i++) o += sum[tid + i * kDim];
    }
    const int fr = rt * a.unit_rows + r;
    const int head = kvh * a.group + fr % a.group;
    store_block(a, head, sq.r0 + fr / a.group, d / 32, NB, o * row_scale(l, m, sink_of(a, head)), lane,
                chunk * rows + tid / kDim / groups < n_rows);
}

}  // namespace

static uint64_t work_bytes(int64_t units, const AttnPlan &p, int nb) {
    return (uint64_t)(units + 1) / 2 * 16 + (uint64_t)(units + p.groups) * p.unit_rows * (8 + 128 * nb);
}

// Whether 128 rows at a time take less than 16: us of either, for units of `tiles`
// position tiles at most, of which they have `seen` (without those behind a
// prompt's own rows, half of them of several sequences, which are rarely all as long
// as the bounds allow).  Units of 16 rows end evenly; those of 128 last, and where
// they are few the compute units wait for the longest.  Measured (16 rows at a time, 128;
// Q4_0, heads of 64): 128 tokens over 2,000 positions 22, 38; a prompt of 1,000: 50, 49,
// of 2,000: 139, 99; 8 ragged ones up to 100: 18, 13, of 100 tokens over up to 4,000: 103,
// 194; 32 of 80 over up to 800: 82, 73; window 128, 400 tokens: 17, 14, 200: 11, 15.
// Q8_0, heads of 128, 200 tokens over 8,000: 112, 125, over 32,000: 604, 384 (tiles
// behind the caches, and then shares).
static bool many_rows(int nb, int64_t units16, int64_t units128, int64_t tiles, int64_t own, int n_seqs, int n_cu) {
    const double seen = double(std::max<int64_t>(1, tiles - own)) * (n_seqs > 1 ? 0.5 : 1.0), slots = 2.0 * n_cu;
    const bool is_long = nb == 4 && tiles > 256;
    const double few = 6.0 + (nb == 2 ? 1.0 : is_long ? 2.6 : 2.0) * units16 * (2.0 + 0.2 * seen) / slots;
    const double scale = nb == 2 ? 1.0 : 1.6, whole = 5.0 + scale * (1.1 * tiles + units128 * (3.0 + 0.6 * seen) / slots);
    return whole < few || (is_long && 18.0 + scale * 1.9 * seen * units128 / slots < few);
}

AttnPlan attn_plan(int nb, int kv_heads, int group, int n_seqs, int max_new, int max_len, int window, int n_cu) {
    AttnPlan p{};
    const int64_t rows = (int64_t)max_new * group;
    // the position tiles of a unit of so many rows: a window before its first
    // row's, and the rows' own
    auto tiles_of = [&](int unit_rows) {
        const int64_t own = (unit_rows - 1) / group + 1;
        return (window ? std::min<int64_t>(max_len, window + own) : max_len) / kKvTile + 2;
    };
    auto units_of = [&](int unit_rows) { return (int64_t)n_seqs * kv_heads * ((rows + unit_rows - 1) / unit_rows); };
    p.unit_rows = rows <= 8 ? 8 : many_rows(nb, units_of(16), units_of(kManyRows), tiles_of(kManyRows), window ? 0 : std::min(max_new, max_len) / 64, n_seqs, n_cu) ? kManyRows : 16;
    const bool many = p.unit_rows == kManyRows;
    p.chunks = (window ? tiles_of(p.unit_rows) : (max_len + kKvTile - 1) / kKvTile) > kManyChunk;
    p.row_tiles = (int)((rows + p.unit_rows - 1) / p.unit_rows);
    const int64_t entries = (int64_t)n_seqs * p.row_tiles, units = entries * kv_heads, tiles = tiles_of(p.unit_rows);
    p.waves = many ? kManyWaves : kWaves;
    // workgroups at once
    const int64_t resident = (int64_t)n_cu * 4 * (many || nb == 4 ? 2 : kMinWaves<2>) / (many ? kManyWaves : kWaves);
    const int64_t cost = many ? kManyCost : kUnitCost;
    const bool long_parts = tiles * units > (int64_t)kLongPart * n_cu && resident > n_cu;
    if (!many && 2 * units <= n_cu && !(long_parts && n_seqs > 1)) {
        const int64_t splits = std::min<int64_t>((long_parts ? resident : n_cu) / units, tiles / kWaves);
        if (splits < 2 || tiles * (splits - 1) * nb <= kSplitTiles * splits) return p;
        p.split_tiles = (int)((tiles + splits - 1) / splits);
        p.splits = (int)((tiles + p.split_tiles - 1) / p.split_tiles);
        p.groups = (int)(units * (p.splits - 1));
        p.work_bytes = work_bytes(units, p, nb);
        return p;
    }
    // 128 rows at a time, us: 1.25 a tile one workgroup a unit, about 18 and 2 a tile of a
    // workgroup's share in shares (768 tokens 39, 65; 128 over 8,192: 320, 80); heads of 64
    // are taken by 16 where shares would be faster
    const bool direct = many ? nb == 2 || 5 * tiles * resident <= 72 * resident + 8 * units * tiles : tiles <= std::min<int64_t>(kWideTiles, kWideTiles * units / n_cu);
    // (the shares' sums are 32 bits, their merge a workgroup a unit at least)
    if (!direct && entries <= kAttnEntries && units <= (1 << 18) && entries * (tiles + cost) <= INT_MAX) {
        p.groups = (int)std::min<int64_t>(resident, std::max<int64_t>(1, units * (tiles + cost) / cost));
        p.work_bytes = work_bytes(units, p, nb);
    } else if (!many && units > resident) {
        p.waves = kHalfWaves;
    }
    return p;
}

hipError_t launch_attn(hipStream_t s, int bits, int nb, const AttnArgs &a) {
    const bool many = a.unit_rows == kManyRows;
    const dim3 grid = a.splits ? dim3(a.kv.kv_heads * a.row_tiles * a.splits, a.kv.n_seqs) : a.groups ? dim3(a.groups) : dim3(a.kv.kv_heads * a.row_tiles, a.kv.n_seqs);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(64 * a.waves), 0, s, a); };
    auto pick = [&](auto q4_2, auto q4_4, auto q8_2, auto q8_4) {
        if (bits == 4)
            nb == 2 ? go(q4_2) : go(q4_4);
        else
            nb == 2 ? go(q8_2) : go(q8_4);
    };
#define SPT_PICK(kernel, ...) pick(kernel<4, 2, ##__VA_ARGS__>, kernel<4, 4, ##__VA_ARGS__>, kernel<8, 2, ##__VA_ARGS__>, kernel<8, 4, ##__VA_ARGS__>)
    if (a.splits)
        a.unit_rows == 8 ? SPT_PICK(k_attn_parts, 8) : SPT_PICK(k_attn_parts, 16);
    else if (a.groups)
        many && bits == 4 ? go(k_attn_shares<4, 4, kManyRows>)  // (only heads of 128 come here)
        : many            ? go(k_attn_shares<8, 4, kManyRows>)
        : a.unit_rows == 8 ? SPT_PICK(k_attn_shares, 8) : SPT_PICK(k_attn_shares, 16);
    else if (many)
        a.chunks ? SPT_PICK(k_attn_many, true) : SPT_PICK(k_attn_many, false);
    else if (a.waves == kWaves)
        a.unit_rows == 8 ? SPT_PICK(k_attn_units, 8, kWaves) : SPT_PICK(k_attn_units, 16, kWaves);
    else
        a.unit_rows == 8 ? SPT_PICK(k_attn_units, 8, kHalfWaves) : SPT_PICK(k_attn_units, 16, kHalfWaves);
#undef SPT_PICK
    return hipGetLastError();
}

hipError_t launch_attn_merge(hipStream_t s, int nb, const AttnArgs &a) {
    const int64_t units = (int64_t)a.kv.n_seqs * a.row_tiles * a.kv.kv_heads;
    // a row a workgroup while the rows are few, else as many as fill it
    const int rows = units * a.unit_rows <= 512 ? 1 : kMergeThreads / (32 * nb);
    const dim3 grid(units * (a.unit_rows / rows));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kMergeThreads), 0, s, a, rows); };
    nb == 2 ? go(k_attn_merge<2>) : go(k_attn_merge<4>);
    return hipGetLastError();
}

}  // namespace spt
