// What the kernels of decay attention share: one recurrence that serves the outputs and all three gradients.
//
//   S_t = l S_{t-1} + b_t c_t^T,  out_t = a_t S_t                           with l = e^{log_decay} of the head
//       = sum_{s <= t} l^{t-s} (a_t . b_s) c_s + l^{t+1} a_t S_0
//
//   out: (a, b, c) = (q, k, v);   dq: (g, v, k) with S_0^T;   and from the last row to the first (LATER)
//   dv:  (k, q, g);               dk: (v, g, q)               with the gradient of the last state in S_0's place
//
// Rows are taken in chunks: inside a chunk pair by pair, what lies before it through the matrix. A sequence is cut into
// segments that run side by side: what each adds to the matrix is summed up first (states), carried from segment to
// segment (carry), and every segment then starts from its own (rows). A sequence of one segment needs the last step only.
//
// Going backwards the matrix is taken one decay further, R = l (sum of what lies behind), because the last state's
// gradient reaches the last row with no decay: a chunk of n rows reads it times l^{i + 1 - later} at its i-th row and
// leaves l^n R + sum_j l^{n - 1 - j + later} b_j c_j^T, i and j counted in the direction of the walk.
//
// Where a factor of the scale belongs: `near` to pairs of one chunk, `add` to what enters the matrix, `far` to what is read.
#pragma once

#include <cuda_bf16.h>

#include "packed_attention.cuh"

namespace fmd {

struct Decay {
    const void *a, *b, *c;       // [rows, heads, dim]
    void* out;                   // [rows, heads, dim] contiguous, or null
    const float* log_decay;      // [heads]
    const int64_t* offsets;      // [batch + 1]
    const float* start;          // [batch, heads, dim, dim]: S_0, or null for zeros
    float* states;               // [segments, heads, dim, dim]: what a segment adds, then what it starts from
    float* after;                // [batch, heads, dim, dim]: the matrix behind the last row, or null
    int32_t* flags;
    int64_t rows;
    int64_t a_row, a_head, b_row, b_head, c_row, c_head;
    int64_t length;              // rows of a segment; kWhole: a segment is a sequence
    float near, add, far;
    int32_t batch, heads, dim, later;
    int32_t transposed;          // start and after: indexed [c][b] for [b][c]
};

// Up to three of them, of the same rows, that run side by side.
struct Decays {
    Decay d[3];
    int32_t count;
};

constexpr int64_t kWhole = int64_t(1) << 40;  // a segment that holds any sequence

// Places for segments (tiles of `length` rows): some may have nothing to do.
__host__ __device__ inline int64_t decay_segments(const Decay& d) {
    return d.length >= kWhole ? d.batch : d.rows / d.length + d.batch;
}

// The place of one block: rows [row0, row0 + rows) of a sequence that has `all`, its number among the segments.
struct Stretch {
    int b;
    int64_t row0, rows, index;
};

// Segment `index` of the map that counts them by sequence (as tiles of `length` rows); rows == 0: nothing to do. All 32
// lanes of a warp. Offsets that do not start at 0, fall or end elsewhere than at the last row raise FMD_FLAG_INDEX_RANGE.
__device__ __forceinline__ Stretch stretch_of(const Decay& d, int64_t index) {
    int b;
    if (d.length >= kWhole && d.batch <= 32) {  // the longest first: the GPU waits for the block that ends last
        const int lane = threadIdx.x & 31;
        const int64_t mine = lane < d.batch ? d.offsets[lane + 1] - d.offsets[lane] : -1;
        int rank = 0;
        for (int i = 0; i < d.batch; ++i) {
            const int64_t other = __shfl_sync(0xffffffffu, mine, i);
            rank += other > mine || (other == mine && i < lane);
        }
        b = __ffs(__ballot_sync(0xffffffffu, lane < d.batch && rank == index)) - 1;
    } else {
        b = find_sequence(d.offsets, d.batch, d.length, index);
    }
    const int64_t r0 = d.offsets[b], r1 = d.offsets[b + 1];
    const int64_t lo = min(max(r0, int64_t(0)), d.rows), hi = min(max(r1, lo), d.rows);
    const int64_t from = d.length >= kWhole ? 0 : (index - (r0 / d.length + b)) * d.length, n = hi - lo;
    Stretch s{b, lo, 0, index};
    if (from < 0 || from >= n) return s;
    s.rows = min(d.length, n - from);
    s.row0 = d.later ? hi - from - s.rows : lo + from;
    return s;
}

// The matrix that a stretch starts from, or null for zeros.
__device__ __forceinline__ const float* start_of(const Decay& d, const Stretch& s, int head) {
    const int64_t size = int64_t(d.dim) * d.dim;
    if (d.length < kWhole) return d.states + (s.index * d.heads + head) * size;
    return d.start != nullptr ? d.start + (int64_t(s.b) * d.heads + head) * size : nullptr;
}

// Looks at sequence b's offsets.
__device__ __forceinline__ void check_offsets(const Decay& d, int64_t b) {
    const int64_t r0 = d.offsets[b], r1 = d.offsets[b + 1];
    if (r0 < 0 || r1 < r0 || r1 > d.rows || (b == 0 && r0 != 0) || (b == d.batch - 1 && r1 != d.rows))
        raise_flag(d.flags, FMD_FLAG_INDEX_RANGE);
}

// l^n; a logarithm above zero counts as zero, and nothing of -inf is left after a row. NaN stays NaN.
__device__ __forceinline__ float log2_decay(const Decay& d, int head) {
    const float log = d.log_decay[head];
    return (log != log ? log : fmaxf(fminf(log, 0.0f), -1.0e4f)) * kLog2e;
}

// What the segments add to the matrix (whole sequences: the matrix behind them, in `after`), and the rows; early: behind
// another kernel of the same call, which they may overlap until they need its results. bfloat16:
fmd_status decay_states_mma(const Decays& d, bool early, cudaStream_t s);
fmd_status decay_rows_mma(const Decays& d, bool early, cudaStream_t s);
// float32: a, b and c are three planes of bfloat16, [3][rows][heads][dim]
fmd_status decay_states_planes(const Decays& d, bool early, cudaStream_t s);
fmd_status decay_rows_planes(const Decays& d, bool early, cudaStream_t s);

}  // namespace fmd
