// spt_kv.h -- layout of the quantized key/value cache and the device helpers
// that its writer, its reader and the attention kernels share.
//
// The cache is pages of page_len positions; a page holds, for each key/value
// head, page_len / 32 tiles.  A tile is 32 positions of one head, contiguous:
// key codes, key scales, value codes, value scales.  Blocks are GGML's (32
// elements of a head's vector, fp16 scale d; Q4_0: value (n - 8) d, Q8_0:
// c d, held as c + 128); only the order of the bytes is this library's: a lane
// of a wavefront takes its operands of the 16x16x32 MFMA by 16-byte loads.
//   keys   A operand, rows = positions, k = dims: a lane (g = lane / 16,
//          r = lane % 16) holds dims 8g .. 8g + 7 of the blocks, for the
//          positions 8 (r / 4) + 4 t + r % 4, t = 0, 1.  A Q4_0 word holds
//          dims 0, 2, 4, 6, 1, 3, 5, 7 of the eight, so that its nibbles 0
//          and 4, 1 and 5, .. become the fp16 pairs of consecutive dims.
//   values A operand transposed, rows = dims, k = positions: a lane holds
//          positions 8g .. 8g + 7 of dims r and r + 16 of a block (the two
//          nibbles of a Q4_0 byte).  A Q4_0 word's bytes are positions 0, 2,
//          1, 3 of four.
// So the row 4g + i of the product of keys and queries (tile half t) is the
// position 8g + 4t + i, and its D registers are the B operand of the product
// with the values as they stand: no exchange between lanes.
// Every byte belongs to one position: a position is written without reading.
#pragma once

#include "spt_device.h"
#include "spt_kv_seq.h"

namespace spt {

constexpr int kKvTile = 32;  // positions of a tile

// bytes of a tile of heads of nb blocks of 32, codes of `bits` bits
constexpr int kv_codes(int bits, int nb) { return 128 * bits * nb; }
constexpr int kv_half(int bits, int nb) { return kv_codes(bits, nb) + 64 * nb; }
constexpr int kv_tile_bytes(int bits, int nb) { return 2 * kv_half(bits, nb); }

template <int BITS, int NB>
struct KvTile {
    static constexpr int kScales = kv_codes(BITS, NB);
    static constexpr int kValues = kv_half(BITS, NB);
    static constexpr int kBytes = kv_tile_bytes(BITS, NB);
    // byte (and nibble) of a code; p = position in the tile, b = block, e = element
    static __device__ inline int key_code(int p, int b, int e) {
        const int r = (p >> 3) * 4 + (p & 3), t = (p >> 2) & 1, l = (e >> 3) * 16 + r;
        if (BITS == 4) return ((b >> 1) * 64 + l) * 16 + t * 8 + (b & 1) * 4 + ((e & 1) * 2 + ((e & 7) >> 2));
        return (((b >> 1) * 2 + t) * 64 + l) * 16 + (b & 1) * 8 + (e & 7);
    }
    static __device__ inline int key_nibble(int e) { return (e >> 1) & 1; }
    static __device__ inline int key_scale(int p, int b) {
        const int r = (p >> 3) * 4 + (p & 3), t = (p >> 2) & 1;
        return kScales + ((r * 2 + t) * NB + b) * 2;
    }
    static __device__ inline int value_code(int p, int b, int e) {
        const int l = (p >> 3) * 16 + (e & 15);
        if (BITS == 4)
            return kValues + ((b >> 1) * 64 + l) * 16 + (b & 1) * 8 + ((p >> 2) & 1) * 4 + (p & 1) * 2 + ((p >> 1) & 1);
        return kValues + (b * 64 + l) * 16 + (e >> 4) * 8 + (p & 7);
    }
    static __device__ inline int value_nibble(int e) { return e >> 4; }
    static __device__ inline int value_scale(int p, int b) { return kValues + kScales + (b * 32 + p) * 2; }
};

// The batch and cache as the kernels take them.
struct KvArgs {
    uint8_t *data;
    int kv_heads;
    int page_tiles;  // tiles of a page
    uint32_t page_inv;  // 2^32 / page_tiles rounded up (its low 32 bits; 0: one tile)
    int n_pages;
    int n_seqs;
    int max_new;
    int n_rows;
    int max_len;
    int max_pages;
    const int32_t *rows;
    const int32_t *lens;
    const int32_t *pages;
};

__device__ inline KvSeq kv_seq(const KvArgs &a, int lo, int hi, int len) {
    return kv_seq_of(lo, hi, len, a.n_rows, a.max_len, a.max_new);
}

// The batch's arrays, which no kernel here writes, as constant memory: a
// uniform index is then a scalar load, also after the kernel's own stores.
typedef const int32_t __attribute__((address_space(4))) *KvConst;
__device__ inline KvConst kv_const(const int32_t *p) { return (KvConst)(uintptr_t)p; }

// Sequence s, the same for all lanes.
__device__ inline KvSeq kv_seq(const KvArgs &a, int s) {
    return kv_seq(a, kv_const(a.rows)[s], kv_const(a.rows)[s + 1], kv_const(a.lens)[s]);
}

// Tile t >= 0 of a sequence: the page of its table, and the tile of that.
__device__ inline int kv_page_of(const KvArgs &a, int t, int *tile) {
    // t / page_tiles: the product is at most one too large (t < 2^32)
    int at = a.page_inv ? (int)__umulhi((uint32_t)t, a.page_inv) : t;
    if (at * a.page_tiles > t) at--;
    *tile = t - at * a.page_tiles;
    return at;
}

// Tile t of a sequence and head, null where its page is none of the cache's.
__device__ inline uint8_t *kv_tile(const KvArgs &a, int s, int head, int t, int tile_bytes) {
    int tile;
    const int at = kv_page_of(a, t, &tile);
    if (at >= a.max_pages) return nullptr;
    const int page = a.pages[(int64_t)s * a.max_pages + at];
    if (page < 0 || page >= a.n_pages) return nullptr;
    return a.data + (((int64_t)page * a.kv_heads + head) * a.page_tiles + tile) * tile_bytes;
}

// Rotation of pairs (i, i + dim / 2): freq[i] radians a position, cos and sin
// scaled by mscale.
struct RopeTable {
    double freq[64];
    double mscale;
};

struct KvStoreArgs {
    KvArgs kv;
    const float *k, *v;
    const float *q;  // null: none (set only with rotate)
    float *q_out;
    int heads;
    int rotate;
    int parts;  // workgroups that share a chunk of rows, by heads
};
// Parts that fill n_cu compute units.
int kv_store_parts(const KvArgs &a, int n_cu);
hipError_t launch_kv_store(hipStream_t s, int bits, int nb, const KvStoreArgs &a, const RopeTable &rope);

struct KvLoadArgs {
    KvArgs kv;
    float *k, *v;
};
hipError_t launch_kv_load(hipStream_t s, int bits, int nb, const KvLoadArgs &a);

// Attention of the batch's rows (spt_attn.hip).
struct AttnArgs {
    KvArgs kv;
    const float *q;
    float *out;
    uint8_t *q8;  // null, or GGML Q8_0 blocks of out
    const void *sinks;
    int sink_type;
    int heads;
    int group;      // heads / kv_heads
    float scale;    // of a score, times log2 e
    int window;     // 0: none
    int unit_rows;  // rows of a row tile
    int row_tiles;  // row tiles of a sequence and key/value head
    int groups;     // parts in the workspace beyond one a unit: of equal shares, their
                    // workgroups; 0: a workgroup a unit, no workspace
    int waves;        // of a workgroup
    bool chunks;      // 128 rows at a time: more tiles than are summed up together
    int splits;       // most parts of a unit, a workgroup each; 0: equal shares
    int split_tiles;  // position tiles of such a part
    void *work;
};
// What a call launches, and the workspace that takes.
struct AttnPlan {
    int unit_rows, row_tiles, waves, groups, splits, split_tiles;
    bool chunks;
    uint64_t work_bytes;
};
AttnPlan attn_plan(int nb, int kv_heads, int group, int n_seqs, int max_new, int max_len, int window, int n_cu);
hipError_t launch_attn(hipStream_t s, int bits, int nb, const AttnArgs &a);
// After launch_attn, where groups > 0.
hipError_t launch_attn_merge(hipStream_t s, int nb, const AttnArgs &a);

}  // namespace spt
