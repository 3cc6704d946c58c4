// What the packed-attention kernels share: the problem, and how a block finds its sequence and its rows.
//
// Queries are read as PACKED ROWS of one key head: row r of a sequence is token r / group, query head
// kv_head * group + r % group. A tile of M rows holds floor(M / group) tokens, so the heads that share a key head
// share its tiles, one key is read once for all of them, and their gradients of k and v add up inside a tile.
//
// The host knows the number of tokens and sequences, not where they lie. A block's tile index is turned into a
// sequence and a place in it with the monotone map  first(b) = offsets[b] / per_tile + b : sequence b owns the
// indexes first(b) .. first(b + 1) - 1, which are never fewer than its tiles (floor(x + n) - floor(x) + 1 >=
// ceil(n) for lengths in tiles); an index past its tiles has nothing to do. So a launch needs no list of tiles, no
// copy to the host and no maximum length. With few sequences the indexes are dealt out heaviest tile first instead
// (find_place): blocks start in order, and a long tile that starts last is waited for by the whole GPU.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace fmd {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRowTile = 128;  // packed rows, or keys, of a tile on the tensor cores

struct Attn {
    const void* q;      // [rows, hq, dim]
    const void* k;      // [keys, hk, dim]
    const void* v;
    void* out;          // [rows, hq, dim] contiguous (forward) / read by the backward pass
    float* lse;         // [rows, hq]
    const void* g;      // gradient of out
    const float* delta; // [rows, hq]: sum_d g out - the gradient of lse
    void* dq;           // [rows, hq, dim] contiguous
    void* dk;           // [keys, hk, dim] contiguous
    void* dv;
    float* part;        // [splits, rows, hq, dim]: outputs, or gradients of q, of the splits of the keys (workspace)
    float* part_lse;    // [splits, rows, hq]
    float* part_dk;     // [splits, keys, hk, dim]: gradients of the splits of the rows (workspace)
    float* part_dv;
    const int64_t* offsets;      // [batch + 1] tokens
    const int64_t* key_offsets;  // [batch + 1]
    const int64_t* key_counts;   // [batch] or null: the whole slot
    int32_t* flags;
    int64_t rows, keys;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, g_row, g_head;
    float scale;
    int32_t batch, hq, hk, group, dim, causal;
    int32_t lse_gradient;  // backward: lse has a gradient too
};

// The sequence of one block: its tokens [row0, row0 + rows), its keys [key0, key0 + keys), of a slot of `slot` rows.
struct Span {
    int64_t row0, key0;
    int64_t rows, keys, slot;
};

inline int64_t tile_bound(int64_t tokens, int64_t batch, int64_t per_tile) { return tokens / per_tile + batch; }

// The last b in [0, batch) with offsets[b] / per_tile + b <= index. All 32 lanes of a warp; every lane gets it.
__device__ __forceinline__ int find_sequence(const int64_t* offsets, int batch, int64_t per_tile, int64_t index) {
    const int lane = threadIdx.x & 31;
    int low = 0, count = batch;  // the answer lies in [low, low + count)
    while (count > 1) {
        const int step = (count + 31) / 32;
        const int b = low + lane * step;
        const bool fits = lane * step < count && offsets[b] / per_tile + b <= index;
        const unsigned votes = __ballot_sync(0xffffffffu, fits) | 1u;
        const int last = 31 - __clz(votes);
        low += last * step;
        count = min(step, count - last * step);
    }
    return low;
}

// The span of sequence b, held inside the arrays whatever the offsets say (bad ones raise FMD_FLAG_INDEX_RANGE).
__device__ __forceinline__ Span load_span(const Attn& a, int b) {
    const int64_t r0 = a.offsets[b], r1 = a.offsets[b + 1], k0 = a.key_offsets[b], k1 = a.key_offsets[b + 1];
    Span s;
    s.row0 = min(max(r0, int64_t(0)), a.rows);
    s.rows = min(max(r1, s.row0), a.rows) - s.row0;
    s.key0 = min(max(k0, int64_t(0)), a.keys);
    s.slot = min(max(k1, s.key0), a.keys) - s.key0;
    int64_t n = s.slot;
    bool bad = r0 != s.row0 || r1 != s.row0 + s.rows || k0 != s.key0 || k1 != s.key0 + s.slot;
    if (a.key_counts != nullptr) {
        n = a.key_counts[b];
        bad = bad || n < 0 || n > s.slot;
        n = min(max(n, int64_t(0)), s.slot);
    }
    // packed rows no sequence holds would stay unwritten: the offsets have to cover them all
    bad = bad || (b == 0 && (r0 != 0 || k0 != 0)) || (b == a.batch - 1 && (r1 != a.rows || k1 != a.keys));
    if (bad) raise_flag(a.flags, FMD_FLAG_INDEX_RANGE);
    s.keys = n;
    return s;
}

// Sequences that a warp sorts by, one a lane. With more of them the blocks are many and even out by themselves, and the
// longer search cost more than it gave (64 sequences of 135 rows: dk and dv 66 -> 75 us).
constexpr int kSorted = 32;

// Looks at sequence b, where there are more than a warp sorts (else every block looks at all): a search among offsets
// that fall may pass a sequence by. The forward kernels do this (they have a block for every sequence at least), and the
// backward pass does it beside its row sums: in both gradient kernels too it took 2 % of 64 sequences of 135.
__device__ __forceinline__ void check_sequence(const Attn& a, int64_t b) {
    if (a.batch > kSorted && b < a.batch) load_span(a, int(b));
}

// Tiles of a sequence whose work is at least `level` units, all of them for level 0. KEYS: tiles of `per` keys, their
// work the tokens that see the first one, the heavy ones at the front; else tiles of `per` tokens, their work the keys
// that the last one sees, the heavy ones at the end.
template <bool KEYS>
__device__ __forceinline__ int tiles_of(const Span& s, bool causal, int per, int unit, int level) {
    const int rows = int(s.rows), keys = int(s.keys);
    const int all = ((KEYS ? int(s.slot) : rows) + per - 1) / per;
    if (level == 0) return all;
    const int least = (level - 1) * unit + 1;
    if (keys < least && !KEYS) return 0;
    if (KEYS) {
        if (rows < least || keys == 0) return 0;
        return causal ? (keys < least ? 0 : (keys - least) / per + 1) : (keys + per - 1) / per;
    }
    const int token = least - keys + rows;  // tokens up to here see fewer keys
    return !causal || token <= 0 ? all : all - (token + per - 1) / per + 1;
}

// A block's sequence and its tile in it (from its first row or key); b < 0: nothing to do.
struct Place {
    int b, tile;
};

// The index-th tile, heaviest first where there are at most kSorted sequences. All 32 lanes of a warp.
template <bool KEYS>
__device__ __forceinline__ Place find_place(const Attn& a, int per, int index, int places) {
    const int lane = threadIdx.x & 31;
    if (a.batch > kSorted) {
        const int64_t* offsets = KEYS ? a.key_offsets : a.offsets;
        if (!KEYS) index = places - 1 - index;  // a causal sequence's last rows see the most
        const int b = find_sequence(offsets, a.batch, per, index);
        const int64_t tile = index - (offsets[b] / per + b);
        const Span s = load_span(a, b);
        return tile < 0 || tile * per >= (KEYS ? s.slot : s.rows) ? Place{-1, 0} : Place{b, int(tile)};
    }
    const int unit = KEYS ? kRowTile / a.group : kRowTile;
    const Span s = lane < a.batch ? load_span(a, lane) : Span{};
    auto mine = [&](int level) { return tiles_of<KEYS>(s, a.causal, per, unit, level); };
    auto count = [&](int level) { return int(__reduce_add_sync(0xffffffffu, unsigned(mine(level)))); };
    if (index >= count(0)) return Place{-1, 0};
    // the highest level with more than `index` tiles
    int low = 0, high = int(__reduce_max_sync(0xffffffffu, unsigned((KEYS ? s.rows : s.keys) / unit + 1)));
    while (low < high) {
        const int mid = (low + high + 1) / 2;
        if (count(mid) > index) low = mid;
        else high = mid - 1;
    }
    // the rank among the tiles of this very level, which go by sequence
    const int here = mine(low), above = mine(low + 1);
    int before = here - above;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    before -= here - above;
    const int rank = index - int(__reduce_add_sync(0xffffffffu, unsigned(above)));
    const int b = __ffs(__ballot_sync(0xffffffffu, rank >= before && rank < before + here - above)) - 1;
    const int first = KEYS ? above : mine(0) - here;
    return Place{b, __shfl_sync(0xffffffffu, first + rank - before, b)};
}

// The same for a whole block: its first warp looks, all get the answer. Blocks count through the key heads first, so
// that the order holds for all heads together; `head` is the block's. CHECK: the offsets have not been looked at before.
template <bool KEYS, bool CHECK = false>
__device__ __forceinline__ Place block_place(const Attn& a, int per, int* head) {
    __shared__ Place place;
    const int index = int(blockIdx.x / unsigned(a.hk));
    *head = int(blockIdx.x - unsigned(index) * unsigned(a.hk));
    if (threadIdx.x < 32) {
        const Place p = find_place<KEYS>(a, per, index, int(gridDim.x / unsigned(a.hk)));
        if (threadIdx.x == 0) place = p;
    } else if (CHECK && threadIdx.x == 32 && *head == 0 && blockIdx.z == 0) {
        check_sequence(a, index);
    }
    __syncthreads();
    return place;
}

// Keys that token t (of the span) sees: all, or with causal those up to its place counted from the end.
__device__ __forceinline__ int64_t seen(const Span& s, bool causal, int64_t t) {
    return causal ? min(max(t + 1 + s.keys - s.rows, int64_t(0)), s.keys) : s.keys;
}

// Whether the scores of a row that sees `keys` keys have a gradient: the softmax of one score is 1 whatever the score, and
// p (dp - delta) would leave the rounding of two equal numbers' difference.
__device__ __forceinline__ bool scores_count(const Attn& a, int64_t keys) { return keys > 1 || a.lse_gradient; }

// Splits of the axis that blocks walk along, for `blocks` places and `tiles` blocks of `length` steps each: the number
// that ends first when a block takes two steps' time besides its own and adding up the splits as much again. Where the
// blocks fill the places four times over they are not split.
inline int split_count(int64_t tiles, int64_t length, int blocks) {
    if (tiles == 0 || tiles >= 4 * int64_t(blocks)) return 1;
    int best = 1;
    int64_t least = INT64_MAX;
    for (int64_t splits = 1; splits <= 64 && (splits == 1 || 2 * splits <= length); ++splits) {
        const int64_t rounds = (tiles * splits + blocks - 1) / blocks;
        const int64_t time = rounds * ((length + splits - 1) / splits + 2) + (splits > 1 ? 2 : 0);
        if (time < least) {
            least = time;
            best = int(splits);
        }
    }
    return best;
}

// Of the keys, for tiles of `per_tile` tokens. The host goes by the mean length of a sequence's slot: the lengths are on
// the device.
inline int key_splits(const Attn& a, int per_tile, int blocks, int tile) {
    if (a.batch == 0) return 1;
    return split_count(tile_bound(a.rows, a.batch, per_tile) * a.hk, (a.keys / a.batch + tile - 1) / tile, blocks);
}

// Of the rows, for tiles of `tile` keys that walk over tiles of `per_tile` tokens.
inline int row_splits(const Attn& a, int per_tile, int blocks, int tile) {
    if (a.batch == 0) return 1;
    return split_count(tile_bound(a.keys, a.batch, tile) * a.hk, (a.rows / a.batch + per_tile - 1) / per_tile, blocks);
}

// Blocks along z of the two gradient kernels; more than one: each writes its part in FP32.
struct BackwardSplits {
    int queries, keys;
};

// bfloat16
int attention_splits_mma(const Attn& a);
fmd_status attention_forward_mma(const Attn& a, int splits, cudaStream_t s);
fmd_status attention_backward_mma(const Attn& a, BackwardSplits splits, cudaStream_t s);
// float32, dim up to 64: by planes of bfloat16 in a workspace
size_t attention_planes_bytes(const Attn& a, bool backward);
fmd_status attention_forward_planes(const Attn& a, int splits, void* planes, cudaStream_t s);
fmd_status attention_backward_planes(const Attn& a, BackwardSplits splits, void* planes, cudaStream_t s);
// float32, wider heads
fmd_status attention_forward_simt(const Attn& a, int splits, cudaStream_t s);
fmd_status attention_backward_simt(const Attn& a, BackwardSplits splits, cudaStream_t s);

}  // namespace fmd
