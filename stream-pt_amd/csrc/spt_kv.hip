// spt_kv.hip -- writing the key/value cache (rotary embedding of queries and
// keys, Q4_0 / Q8_0 blocks of keys and values) and reading it back.
//
// Rotation: the angle of position p and pair i is p * freq[i] in 64 bits,
// reduced by multiples of pi/2 there, and x1 cos - x2 sin, x2 cos + x1 sin
// are formed in 64 bits and rounded once, so a far position loses nothing
// and a value next to a border between two codes falls on the side that the
// formula says.  Quantization is GGML's rule in 32 bits: Q4_0 d = m / -8 with m
// the element of the largest magnitude (the first of equals), code
// min(15, floor(x / d + 8.5)); Q8_0 the rule of spt_quantize_q8_0.  |d| is
// capped so that every stored value is a finite fp16 number (8188 and 515.5:
// 65,504 / 8 and / 127), which the attention kernels' fp16 operands rely on.
// An infinity or NaN in a row's key or value makes the key's scales NaN and the
// value's 0: whoever attends to that position gets NaN, no one else.
#include <algorithm>

#include "spt_kv.h"
#include "spt_kernels.h"

namespace spt {

namespace {

constexpr int kStoreRows = 4;  // rows of a workgroup

// sin and cos of a >= 0 (or of either sign): n = a / (pi/2) rounded, r = a - n
// pi/2 with pi/2 in two parts (each product exact in the FMA; n < 2^31), then
// the Taylor series to r^15 and r^16 on |r| <= pi/4 (the next terms are below
// 5e-17).
__device__ inline void sincos_f64(double a, double *s, double *c) {
    const double n = __builtin_rint(a * 0.63661977236758134308);
    double r = __builtin_fma(-n, 1.57079632679489655800, a);
    r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double p = -1.0 / 1307674368000.0;
    p = __builtin_fma(p, z, 1.0 / 6227020800.0);
    p = __builtin_fma(p, z, -1.0 / 39916800.0);
    p = __builtin_fma(p, z, 1.0 / 362880.0);
    p = __builtin_fma(p, z, -1.0 / 5040.0);
    p = __builtin_fma(p, z, 1.0 / 120.0);
    p = __builtin_fma(p, z, -1.0 / 6.0);
    const double sn = __builtin_fma(p * z, r, r);
    double q = 1.0 / 20922789888000.0;
    q = __builtin_fma(q, z, -1.0 / 87178291200.0);
    q = __builtin_fma(q, z, 1.0 / 479001600.0);
    q = __builtin_fma(q, z, -1.0 / 3628800.0);
    q = __builtin_fma(q, z, 1.0 / 40320.0);
    q = __builtin_fma(q, z, -1.0 / 720.0);
    q = __builtin_fma(q, z, 1.0 / 24.0);
    q = __builtin_fma(q, z, -0.5);
    const double cs = __builtin_fma(q, z, 1.0);
    const int k = (int)n & 3;
    const double u = (k & 1) ? cs : sn, v = (k & 1) ? sn : cs;
    *s = (k & 2) ? -u : u;
    *c = (k == 1 || k == 2) ? -v : v;
}

// A half-wave's block, an element a lane: the code and the stored scale.
__device__ inline int q4_quantize_half(float v, int lane, uint16_t *dbits) {
    const uint32_t a = __float_as_uint(__builtin_fabsf(v));
    const uint64_t eq = __ballot(a == max32_bits(a));
    const int first = __builtin_ctz((uint32_t)(lane < 32 ? eq : eq >> 32));
    const float m = __shfl(v, (lane & 32) + first);
    const float d = fminf(fmaxf(m / -8.0f, -8188.0f), 8188.0f);
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    *dbits = f32_to_f16_bits(d);
    const float r = __builtin_floorf(v * id + 8.5f);
    return r != r ? 8 : (int)fminf(fmaxf(r, 0.0f), 15.0f);
}

__device__ inline int q8_quantize_capped(float v, uint16_t *dbits) {
    const float m = __uint_as_float(max32_bits(__float_as_uint(__builtin_fabsf(v))));
    const float d = fminf(m / 127.0f, 515.5f);
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    *dbits = f32_to_f16_bits(d);
    const float r = __builtin_roundf(v * id);
    return r != r ? 0 : (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

// Keys (VALUES false) or values of one position and head, lane l of the wave
// holding elements l, 64 + l, ..
template <int BITS, int NB, bool VALUES>
__device__ inline void store_blocks(uint8_t *tile, int p, const float (&x)[NB / 2], int lane, bool bad) {
    using T = KvTile<BITS, NB>;
    const int e = lane & 31;
#pragma unroll
    for (int i = 0; i < NB / 2; i++) {
        const int b = 2 * i + (lane >> 5);
        uint16_t d;
        int c;
        if (BITS == 4)
            c = q4_quantize_half(bad ? 0.0f : x[i], lane, &d);
        else
            c = q8_quantize_capped(bad ? 0.0f : x[i], &d) + 128;
        if (bad && !VALUES) d = 0x7e00u;
        if (e == 0) *reinterpret_cast<uint16_t *>(tile + (VALUES ? T::value_scale(p, b) : T::key_scale(p, b))) = d;
        if (BITS == 8) {
            tile[VALUES ? T::value_code(p, b, e) : T::key_code(p, b, e)] = (uint8_t)c;
        } else if (VALUES) {
            const int o = __builtin_amdgcn_ds_swizzle(c, 0x401F);  // lane ^ 16
            if (e < 16) tile[T::value_code(p, b, e)] = (uint8_t)(c | o << 4);
        } else {
            // the word of eight dims, by ORs within eight lanes
            uint32_t w = (uint32_t)c << (4 * ((e & 1) * 4 + ((e & 7) >> 1)));
            w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xF, 0xF, false);
            w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x4E, 0xF, 0xF, false);
            w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x141, 0xF, 0xF, false);
            if ((e & 7) == 0) *reinterpret_cast<uint32_t *>(tile + T::key_code(p, b, e)) = w;
        }
    }
}

// Rows [4 x, 4 x + 4) of sequence y, heads of part z: angles of the rows into
// LDS, then query pairs by threads and keys and values by waves.
template <int BITS, int NB>
__global__ __launch_bounds__(256) void k_kv_store(KvStoreArgs a, RopeTable rope) {
    constexpr int kDim = 32 * NB, kPairs = kDim / 2;
    __shared__ double cs[kStoreRows][kPairs], sn[kStoreRows][kPairs];
    const KvSeq sq = kv_seq(a.kv, blockIdx.y);
    const int i0 = blockIdx.x * kStoreRows, n = min(kStoreRows, sq.n - i0);
    if (!sq.ok || n <= 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.z;
    if (a.rotate) {
        for (int u = tid; u < n * kPairs; u += 256) {
            const int r = u / kPairs, i = u % kPairs;
            double s, c;
            sincos_f64((double)(sq.first + i0 + r) * rope.freq[i], &s, &c);
            cs[r][i] = c * rope.mscale;
            sn[r][i] = s * rope.mscale;
        }
        __syncthreads();
    }
    if (a.q) {
        const int h0 = (int)((int64_t)a.heads * part / a.parts), nh = (int)((int64_t)a.heads * (part + 1) / a.parts) - h0;
        constexpr int kQuads = kPairs / 4;
#pragma unroll 4
        for (int u = tid; u < n * nh * kQuads; u += 256) {
            const int i = u % kQuads * 4, h = u / kQuads % nh, r = u / (kQuads * nh);
            const int64_t at = ((int64_t)(sq.r0 + i0 + r) * a.heads + h0 + h) * kDim + i;
            const float4 x = *reinterpret_cast<const float4 *>(a.q + at), y = *reinterpret_cast<const float4 *>(a.q + at + kPairs);
            float4 ox, oy;
            auto turn = [&](float xi, float yi, float &o, float &p, int j) {
                const double c = cs[r][i + j], s = sn[r][i + j];
                o = (float)((double)xi * c - (double)yi * s);
                p = (float)((double)yi * c + (double)xi * s);
            };
            turn(x.x, y.x, ox.x, oy.x, 0);
            turn(x.y, y.y, ox.y, oy.y, 1);
            turn(x.z, y.z, ox.z, oy.z, 2);
            turn(x.w, y.w, ox.w, oy.w, 3);
            *reinterpret_cast<float4 *>(a.q_out + at) = ox;
            *reinterpret_cast<float4 *>(a.q_out + at + kPairs) = oy;
        }
    }
    const int h0 = a.kv.kv_heads * part / a.parts, nh = a.kv.kv_heads * (part + 1) / a.parts - h0;
    for (int u = wave; u < n * nh; u += 4) {
        const int r = u / nh, h = h0 + u % nh, pos = sq.first + i0 + r;
        if (pos < 0) continue;
        uint8_t *tile = kv_tile(a.kv, blockIdx.y, h, pos / kKvTile, KvTile<BITS, NB>::kBytes);
        if (!tile) continue;
        const int64_t at = ((int64_t)(sq.r0 + i0 + r) * a.kv.kv_heads + h) * kDim;
        float k[NB / 2], v[NB / 2];
        bool odd = false;
#pragma unroll
        for (int i = 0; i < NB / 2; i++) {
            const int d = 64 * i + lane;
            k[i] = a.k[at + d];
            v[i] = a.v[at + d];
            if (a.rotate) {
                const bool lower = d < kPairs;
                const double o = a.k[at + (lower ? d + kPairs : d - kPairs)], c = cs[r][d % kPairs], s = sn[r][d % kPairs];
                k[i] = lower ? (float)((double)k[i] * c - o * s) : (float)((double)k[i] * c + o * s);
            }
            odd |= !(__builtin_fabsf(k[i]) < __builtin_inff()) || !(__builtin_fabsf(v[i]) < __builtin_inff());
        }
        odd = __any(odd);
        store_blocks<BITS, NB, false>(tile, pos % kKvTile, k, lane, odd);
        store_blocks<BITS, NB, true>(tile, pos % kKvTile, v, lane, odd);
    }
}

// A tile of a sequence and head through LDS: 16-byte loads of the tile, 16-byte
// stores of the rows that it holds.
template <int BITS, int NB>
__global__ __launch_bounds__(256) void k_kv_load(KvLoadArgs a) {
    using T = KvTile<BITS, NB>;
    constexpr int kDim = 32 * NB;
    __shared__ __align__(16) uint8_t img[T::kBytes];
    const KvSeq sq = kv_seq(a.kv, blockIdx.y);
    const int n = sq.n;
    if (n <= 0) return;
    // the tiles of the rows' positions; the rows before position 0 are the first tile's
    const int t = max(0, sq.first) / kKvTile + (int)blockIdx.x;
    const int lo = blockIdx.x == 0 ? 0 : t * kKvTile - sq.first, hi = min(n, (t + 1) * kKvTile - sq.first);
    if (lo >= hi) return;
    const int head = blockIdx.z;
    const uint8_t *tile = sq.ok ? kv_tile(a.kv, blockIdx.y, head, t, T::kBytes) : nullptr;
    if (tile) {
        for (int i = threadIdx.x; i < T::kBytes / 16; i += 256)
            reinterpret_cast<uint4 *>(img)[i] = reinterpret_cast<const uint4 *>(tile)[i];
    }
    __syncthreads();
    constexpr int kQuads = kDim / 4;
    for (int u = threadIdx.x; u < (hi - lo) * kQuads * 2; u += 256) {
        const int qd = u % kQuads, values = u / kQuads & 1, r = lo + u / (2 * kQuads), pos = sq.first + r;
        const int b = qd / 8, e = qd % 8 * 4, p = pos & (kKvTile - 1);
        float o[4];
        const float none = __builtin_nanf("");
        const float d = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(img + (values ? T::value_scale(p, b) : T::key_scale(p, b))));
#pragma unroll
        for (int j = 0; j < 4; j++) {
            int c = img[values ? T::value_code(p, b, e + j) : T::key_code(p, b, e + j)];
            if (BITS == 4)
                c = ((c >> (4 * (values ? T::value_nibble(e + j) : T::key_nibble(e + j)))) & 15) - 8;
            else
                c -= 128;
            o[j] = (tile && pos >= 0) ? (float)c * d : none;
        }
        const int64_t at = ((int64_t)(sq.r0 + r) * a.kv.kv_heads + head) * kDim + qd * 4;
        *reinterpret_cast<float4 *>((values ? a.v : a.k) + at) = make_float4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace

// Few rows are shared by heads among up to kv_heads workgroups, while those
// are fewer than 16 a compute unit (4,099 rows of 64 query and 8 key/value heads
// of 64, the same inputs again: 40.3 us with two a compute unit and rows by eight, 31 us;
// inputs that change: 38).
int kv_store_parts(const KvArgs &a, int n_cu) {
    const int64_t chunks = (int64_t)((a.max_new + kStoreRows - 1) / kStoreRows) * a.n_seqs;
    return (int)std::min<int64_t>(a.kv_heads, std::max<int64_t>(1, 16 * (int64_t)n_cu / chunks));
}

hipError_t launch_kv_store(hipStream_t s, int bits, int nb, const KvStoreArgs &a, const RopeTable &rope) {
    const dim3 grid((a.kv.max_new + kStoreRows - 1) / kStoreRows, a.kv.n_seqs, a.parts);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a, rope); };
    if (bits == 4)
        nb == 2 ? go(k_kv_store<4, 2>) : go(k_kv_store<4, 4>);
    else
        nb == 2 ? go(k_kv_store<8, 2>) : go(k_kv_store<8, 4>);
    return hipGetLastError();
}

hipError_t launch_kv_load(hipStream_t s, int bits, int nb, const KvLoadArgs &a) {
    // n rows touch at most (n - 1 + 31) / 32 + 1 tiles
    const dim3 grid((a.kv.max_new - 1 + kKvTile - 1) / kKvTile + 1, a.kv.n_seqs, a.kv.kv_heads);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a); };
    if (bits == 4)
        nb == 2 ? go(k_kv_load<4, 2>) : go(k_kv_load<4, 4>);
    else
        nb == 2 ? go(k_kv_load<8, 2>) : go(k_kv_load<8, 4>);
    return hipGetLastError();
}

}  // namespace spt
