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
// copy to the host and no maximum length.
#pragma once

#include <cuda_bf16.h>
#include <float.h>

#include "common.cuh"

namespace fmd {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
    float* part;        // [splits, rows, hq, dim] and
    float* part_lse;    // [splits, rows, hq]: the splits of the keys, workspace
    const int64_t* offsets;      // [batch + 1] tokens
    const int64_t* key_offsets;  // [batch + 1]
    const int64_t* key_counts;   // [batch] or null: the whole slot
    int32_t* flags;
    int64_t rows, keys;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, g_row, g_head;
    float scale;
    int32_t batch, hq, hk, group, dim, causal;
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
    if (bad && (threadIdx.x & 31) == 0) raise_flag(a.flags, FMD_FLAG_INDEX_RANGE);
    s.keys = n;
    return s;
}

// Keys that token t (of the span) sees: all, or with causal those up to its place counted from the end.
__device__ __forceinline__ int64_t seen(const Span& s, bool causal, int64_t t) {
    return causal ? min(max(t + 1 + s.keys - s.rows, int64_t(0)), s.keys) : s.keys;
}

// Splits of the keys in the forward pass, where the tiles of `per_tile` tokens do not fill `blocks` places: the host
// goes by the mean length of a sequence's slot (the lengths are on the device), and a split has `least` keys at least.
inline int key_splits(const Attn& a, int per_tile, int blocks, int least) {
    const int64_t tiles = tile_bound(a.rows, a.batch, per_tile) * a.hk;
    if (tiles == 0 || a.batch == 0) return 1;
    int64_t splits = blocks / tiles;
    const int64_t most = a.keys / a.batch / least;
    if (splits > most) splits = most;
    return splits < 1 ? 1 : splits > 64 ? 64 : int(splits);
}

// bfloat16
int attention_splits_mma(const Attn& a);
fmd_status attention_forward_mma(const Attn& a, int splits, cudaStream_t s);
fmd_status attention_backward_mma(const Attn& a, cudaStream_t s);
// float32, dim up to 64: by planes of bfloat16 in a workspace
size_t attention_planes_bytes(const Attn& a, bool backward);
fmd_status attention_forward_planes(const Attn& a, int splits, void* planes, cudaStream_t s);
fmd_status attention_backward_planes(const Attn& a, void* planes, cudaStream_t s);
// float32, wider heads
fmd_status attention_forward_simt(const Attn& a, int splits, cudaStream_t s);
fmd_status attention_backward_simt(const Attn& a, cudaStream_t s);

}  // namespace fmd
