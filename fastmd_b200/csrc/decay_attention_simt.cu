// Decay attention in float32 for heads of more than 64 values, on the FP32 cores.
//
// A block of 256 threads walks over the chunks of 64 rows of one segment and head; the chunk's rows of a, b and c and the
// matrix lie in shared memory in FP32, padded to DP columns. A thread owns pieces of 4 x 4 pairs, of 4 rows x DP / 16
// values of the output, and of DP / 16 x DP / 16 of the matrix, which it also keeps in registers. Bound by the FP32 cores and
// the shared memory that feeds them, a block an SM: 64 sequences of 100 to 500 rows, 8 heads of 128, forward and backward,
// 2,700 us (heads of 64 by planes 360); one of 20,000 rows, 16 heads of 128, forward, 1,850.

#include "decay_attention.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 256, kChunk = 64, kDim = 128;

template <int DP>
struct Tiles {
    static constexpr int kLd = DP + 4;
    static constexpr size_t kStates = size_t(2 * kChunk * kLd + kChunk) * 4;
    static constexpr size_t kRows = size_t(3 * kChunk * kLd + DP * kLd + kChunk * (kChunk + 4) + kChunk) * 4;
};

// `count` rows from `row0` on, zeros behind them and behind dim.
template <int DP>
__device__ __forceinline__ void load_rows(float* to, const void* from, int64_t row0, int64_t row, int64_t offset, int count,
                                          int dim) {
    for (int i = threadIdx.x; i < kChunk * DP / 4; i += kThreads) {
        const int r = i / (DP / 4), c = i % (DP / 4) * 4;
        float4 v = f4_zero();
        if (r < count && c < dim) {
            v = ldg4(static_cast<const float*>(from) + (row0 + r) * row + offset + c);
        }
        st4(to + r * Tiles<DP>::kLd + c, v);
    }
}

template <int PER>
__device__ __forceinline__ void load_piece(const float* p, float (&v)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; i += (PER < 4 ? 2 : 4)) {
        if constexpr (PER < 4) {
            const float2 x = *reinterpret_cast<const float2*>(p + i);
            v[i] = x.x;
            v[i + 1] = x.y;
        } else {
            const float4 x = *reinterpret_cast<const float4*>(p + i);
            v[i] = x.x;
            v[i + 1] = x.y;
            v[i + 2] = x.z;
            v[i + 3] = x.w;
        }
    }
}

// state += sum_j w_j b_j c_j^T over the chunk, the piece of rows ty PER .. and columns tx PER ..
template <int DP>
__device__ __forceinline__ void add_outer(const float* b, const float* c, const float* weight, int count, int ty, int tx,
                                          float (&state)[DP / 16][DP / 16]) {
    constexpr int kPer = DP / 16, kLd = Tiles<DP>::kLd;
#pragma unroll 2
    for (int j = 0; j < count; ++j) {
        float x[kPer], y[kPer];
        load_piece<kPer>(b + j * kLd + ty * kPer, x);
        load_piece<kPer>(c + j * kLd + tx * kPer, y);
        const float w = weight[j];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            x[i] *= w;
#pragma unroll
            for (int e = 0; e < kPer; ++e) state[i][e] = fmaf(x[i], y[e], state[i][e]);
        }
    }
}

// The rows of the next chunk of a stretch: `done` rows lie behind the walk.
__device__ __forceinline__ int64_t chunk_row(const Decay& d, const Stretch& s, int64_t done, int count) {
    return d.later ? s.row0 + s.rows - done - count : s.row0 + done;
}

__global__ void __launch_bounds__(kThreads) states_kernel(const __grid_constant__ Decays all) {
    constexpr int DP = kDim;
    const Decay& d = all.d[blockIdx.x % unsigned(all.count)];
    const int64_t place = blockIdx.x / unsigned(all.count);
    constexpr int kPer = DP / 16, kLd = Tiles<DP>::kLd;
    extern __shared__ float smem[];
    float *b = smem, *c = b + kChunk * kLd, *weight = c + kChunk * kLd;
    const int head = int(place % d.heads);
    const Stretch s = stretch_of(d, place / d.heads);
    const bool whole = d.length >= kWhole;
    if (s.rows == 0 && !whole) return;
    const float l2 = log2_decay(d, head);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const float* start = whole ? start_of(d, s, head) : nullptr;
    float state[kPer][kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) state[i][e] = start_at(d, start, ty * kPer + i, tx * kPer + e);
    for (int64_t done = 0; done < s.rows; done += kChunk) {
        const int count = int(min(int64_t(kChunk), s.rows - done));
        const int64_t row = chunk_row(d, s, done, count);
        __syncthreads();
        load_rows<DP>(b, d.b, row, d.b_row, head * d.b_head, count, d.dim);
        load_rows<DP>(c, d.c, row, d.c_row, head * d.c_head, count, d.dim);
        if (threadIdx.x < kChunk) {
            const int j = threadIdx.x;
            weight[j] = j < count ? d.add * exp2f(float(d.later ? j + 1 : count - 1 - j) * l2) : 0.0f;
        }
        __syncthreads();
        const float keep = exp2f(float(count) * l2);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int e = 0; e < kPer; ++e) state[i][e] *= keep;
        add_outer<DP>(b, c, weight, count, ty, tx, state);
    }
    float* out = (whole ? d.after + int64_t(s.b) * d.heads * d.dim * d.dim : d.states + s.index * d.heads * d.dim * d.dim) +
                 int64_t(head) * d.dim * d.dim;
    const bool turn = whole && d.transposed;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int r = ty * kPer + i, col = tx * kPer + e;
            if (r < d.dim && col < d.dim) out[turn ? col * d.dim + r : r * d.dim + col] = state[i][e];
        }
}

__global__ void __launch_bounds__(kThreads) rows_kernel(const __grid_constant__ Decays all) {
    constexpr int DP = kDim;
    const Decay& d = all.d[blockIdx.x % unsigned(all.count)];
    const int64_t place = blockIdx.x / unsigned(all.count);
    constexpr int kPer = DP / 16, kLd = Tiles<DP>::kLd, kPairs = kChunk + 4;
    extern __shared__ float smem[];
    float *a = smem, *b = a + kChunk * kLd, *c = b + kChunk * kLd, *matrix = c + kChunk * kLd, *pairs = matrix + DP * kLd,
          *weight = pairs + kChunk * kPairs;
    const int head = int(place % d.heads);
    const int64_t index = place / d.heads;
    if (head == 0 && threadIdx.x == 32 && index < d.batch) check_offsets(d, index);
    const Stretch s = stretch_of(d, index);
    if (s.rows == 0) return;
    const float l2 = log2_decay(d, head);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const float* start = start_of(d, s, head);
    float state[kPer][kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            state[i][e] = start_at(d, start, ty * kPer + i, tx * kPer + e);
            matrix[(ty * kPer + i) * kLd + tx * kPer + e] = state[i][e];
        }
    for (int64_t done = 0; done < s.rows; done += kChunk) {
        const int count = int(min(int64_t(kChunk), s.rows - done));
        const int64_t row = chunk_row(d, s, done, count);
        __syncthreads();
        load_rows<DP>(a, d.a, row, d.a_row, head * d.a_head, count, d.dim);
        load_rows<DP>(b, d.b, row, d.b_row, head * d.b_head, count, d.dim);
        load_rows<DP>(c, d.c, row, d.c_row, head * d.c_head, count, d.dim);
        if (threadIdx.x < kChunk) {
            const int j = threadIdx.x;
            weight[j] = j < count ? d.add * exp2f(float(d.later ? j + 1 : count - 1 - j) * l2) : 0.0f;
        }
        __syncthreads();
        float dot[4][4] = {};
#pragma unroll 2
        for (int x = 0; x < DP; x += 4) {
            float4 p[4], q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * kLd + x);
                q[i] = *reinterpret_cast<const float4*>(b + (tx + 16 * i) * kLd + x);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    dot[i][j] = fmaf(p[i].x, q[j].x, dot[i][j]);
                    dot[i][j] = fmaf(p[i].y, q[j].y, dot[i][j]);
                    dot[i][j] = fmaf(p[i].z, q[j].z, dot[i][j]);
                    dot[i][j] = fmaf(p[i].w, q[j].w, dot[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = ty + 16 * i, u = tx + 16 * j, gap = d.later ? u - t : t - u;
                pairs[t * kPairs + u] = gap >= 0 && u < count ? d.near * dot[i][j] * exp2f(float(gap) * l2) : 0.0f;
            }
        __syncthreads();
        float far[4][kPer] = {}, near[4][kPer] = {};
#pragma unroll 2
        for (int x = 0; x < DP; ++x) {
            float y[kPer];
            load_piece<kPer>(matrix + x * kLd + tx * kPer, y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = a[(ty + 16 * i) * kLd + x];
#pragma unroll
                for (int e = 0; e < kPer; ++e) far[i][e] = fmaf(p, y[e], far[i][e]);
            }
        }
#pragma unroll 2
        for (int j = 0; j < count; ++j) {
            float y[kPer];
            load_piece<kPer>(c + j * kLd + tx * kPer, y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = pairs[(ty + 16 * i) * kPairs + j];
#pragma unroll
                for (int e = 0; e < kPer; ++e) near[i][e] = fmaf(p, y[e], near[i][e]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = ty + 16 * i;
            if (t >= count) continue;
            const float reach = d.far * exp2f(float(d.later ? count - 1 - t : t + 1) * l2);
            float* out = static_cast<float*>(d.out) + ((row + t) * d.heads + head) * d.dim;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                if (tx * kPer + e < d.dim) out[tx * kPer + e] = fmaf(reach, far[i][e], near[i][e]);
            }
        }
        const float keep = exp2f(float(count) * l2);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int e = 0; e < kPer; ++e) state[i][e] *= keep;
        add_outer<DP>(b, c, weight, count, ty, tx, state);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int e = 0; e < kPer; ++e) matrix[(ty * kPer + i) * kLd + tx * kPer + e] = state[i][e];
    }
}

fmd_status launch(const Decays& d, bool states, cudaStream_t s) {
    const size_t bytes = states ? Tiles<kDim>::kStates : Tiles<kDim>::kRows;
    const void* kernel = states ? (const void*)states_kernel : (const void*)rows_kernel;
    const fmd_status st = grant_dynamic_smem(kernel, bytes, true);
    if (st != FMD_OK) return st;
    const unsigned blocks = unsigned(decay_segments(d.d[0]) * d.d[0].heads * d.count);
    if (states) states_kernel<<<blocks, kThreads, bytes, s>>>(d);
    else rows_kernel<<<blocks, kThreads, bytes, s>>>(d);
    return check_launch();
}

}  // namespace

fmd_status decay_states_simt(const Decays& d, cudaStream_t s) { return launch(d, true, s); }

fmd_status decay_rows_simt(const Decays& d, cudaStream_t s) { return launch(d, false, s); }

}  // namespace fmd
