// RMS norm of each query and key head with the rotation of its position, one pass over the data, and the
// backward pass of both.
//
//   n = sqrt(sum_d x_d^2 / D + eps),  y_d = w_d x_d / n                 (weights given; else y = x)
//   pair p of the first R values, (a, b) = (y_p, y_{p + R/2}) or, interleaved, (y_{2p}, y_{2p+1}):
//       (a', b') = (a c - b s, b c + a s),  c = cos[pos, p], s = sin[pos, p];  the rest passes
//   backward: gy = the gradient turned by -angle;  u = x / n;  dw = sum gy u (all rows and heads);
//       h = w gy;  dx = (h - u mean_d(h u)) / n
//
// Everything is computed in FP32 and rounded once, as the value is stored.
//
// What bounds it: memory. A head is D / V lanes of one 16-byte load each (V = 8 bfloat16 or 4 float32 values;
// 4 bfloat16 where a rotated half does not divide by 8), the lanes padded to a power of two for the sums, so
// a warp takes 32 / P heads at a time. The partner of a value in the half layout is the same value of another
// lane (one shuffle); interleaved partners share a lane. A warp's unit is one row and kHeads heads per lane
// group, all of the queries or all of the keys: the row's cos and sin are read once per unit, into registers,
// and the loads of all its heads are in flight together. The backward pass keeps the weights' gradients in
// registers over a persistent grid, sums a block's warps in shared memory in warp order and the blocks'
// partial sums in block order in a second kernel: no atomics, the same bits every time.

#include <cuda_bf16.h>

#include "common.cuh"

namespace fmd {
namespace {

constexpr int kHeads = 4;     // heads per lane group and unit: their loads are in flight together
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 128;

struct Side {
    const void* x;    // [rows, heads, D], strides row and head
    const void* g;    // gradient of the output, strides grow and ghead (backward)
    void* y;          // output (or the input's gradient), contiguous
    const void* w;    // [D] or null
    int64_t row, head, grow, ghead;
    int32_t heads, units;  // units of kHeads heads per lane group
};

struct Args {
    Side side[2];
    const int64_t* positions;
    const float* cos;
    const float* sin;
    float* partial;     // [blocks][2][D] weight gradients (backward) or null
    int32_t* flags;
    int64_t rows, table;
    float eps, inv_dim;
    int32_t dim, rot, interleaved, w_float;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float& o, float v) { o = v; }
__device__ __forceinline__ void from_float(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }

template <typename T, int V>
__device__ __forceinline__ void load_weight(const Args& a, const Side& s, int c0, bool active, float (&w)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w[j] = 0.0f;
        if (s.w != nullptr && active)
            w[j] = a.w_float ? static_cast<const float*>(s.w)[c0 + j] : to_float(static_cast<const T*>(s.w)[c0 + j]);
    }
}

// Turns the lane's V values by the row's angle (sign -1: back). `there` marks the lanes inside the rotated part.
template <int V>
__device__ __forceinline__ void turn(float (&y)[V], const float (&c)[V], const float (&s)[V], int partner, bool first,
                                     bool there, bool interleaved, float sign) {
    if (interleaved) {
        if (there) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float p = y[j], q = y[j + 1], t = sign * s[j / 2];
                y[j] = p * c[j / 2] - q * t;
                y[j + 1] = q * c[j / 2] + p * t;
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float other = __shfl_sync(0xffffffffu, y[j], partner);
        const float t = sign * (first ? -s[j] : s[j]);
        if (there) y[j] = y[j] * c[j] + other * t;
    }
}


template <typename T, int V, bool BACKWARD>
__global__ void __launch_bounds__(kThreads) head_rotary_kernel(const Args a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lanes = a.dim / V;
    int span = 1;
    while (span < lanes) span <<= 1;
    const int groups = 32 / span, group = lane / span, sub = lane % span;
    const bool active = sub < lanes;
    const int c0 = sub * V;
    const int half = a.rot / 2;
    const bool inter = a.interleaved != 0;
    const bool there = active && c0 < a.rot;
    const bool first = c0 < half;
    const int partner = inter || !there ? lane : (first ? lane + half / V : lane - half / V);
    const int t0 = inter ? c0 / 2 : (first ? c0 : c0 - half);
    const int units = a.side[0].units + a.side[1].units;
    const int64_t total = a.rows * units;

    float dw[2][V];
#pragma unroll
    for (int j = 0; j < V; ++j) dw[0][j] = dw[1][j] = 0.0f;

    for (int64_t u = int64_t(blockIdx.x) * kWarps + warp; u < total; u += int64_t(gridDim.x) * kWarps) {
        const int64_t row = u / units;
        int unit = int(u - row * units);
        const int which = unit >= a.side[0].units;
        const Side& s = a.side[which];
        if (which) unit -= a.side[0].units;
        const int head0 = unit * kHeads * groups + group;

        Pack<T, V> x[kHeads], g[kHeads];
        const bool need_x = !BACKWARD || s.w != nullptr;
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = head0 + i * groups;
            if (active && h < s.heads) {
                if (need_x)
                    x[i] = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(s.x) + row * s.row +
                                                                h * s.head + c0);
                if (BACKWARD)
                    g[i] = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(s.g) + row * s.grow +
                                                                h * s.ghead + c0);
            }
        }
        const int64_t pos = a.positions[row];
        const bool known = pos >= 0 && pos < a.table;
        if (!known && lane == 0) raise_flag(a.flags, FMD_FLAG_INDEX_RANGE);
        float c[V], sn[V], w[V];
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = sn[j] = 0.0f;
        if (there && known) {
            const float* cr = a.cos + pos * half + t0;
            const float* sr = a.sin + pos * half + t0;
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < (inter ? V / 2 : V)) {
                    c[j] = __ldg(cr + j);
                    sn[j] = __ldg(sr + j);
                }
        }
        load_weight<T, V>(a, s, c0, active, w);

#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = head0 + i * groups;
            const bool mine = active && h < s.heads;
            float v[V], n = 1.0f;
            if (need_x) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[j] = mine ? to_float(x[i].v[j]) : 0.0f;
                    sum += v[j] * v[j];
                }
                if (s.w != nullptr) {
                    for (int o = span / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    n = rsqrtf(sum * a.inv_dim + a.eps);
                }
            }
            float y[V];
            if (!BACKWARD) {
#pragma unroll
                for (int j = 0; j < V; ++j) y[j] = s.w != nullptr ? v[j] * n * w[j] : v[j];
                turn<V>(y, c, sn, partner, first, there, inter, 1.0f);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) y[j] = mine ? to_float(g[i].v[j]) : 0.0f;
                turn<V>(y, c, sn, partner, first, there, inter, -1.0f);
                if (s.w != nullptr) {
                    float dot = 0.0f;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        v[j] *= n;  // u
                        const float t = y[j] * v[j];
                        if (which) dw[1][j] += t;
                        else dw[0][j] += t;
                        y[j] *= w[j];
                        dot += y[j] * v[j];
                    }
                    for (int o = span / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                    dot *= a.inv_dim;
#pragma unroll
                    for (int j = 0; j < V; ++j) y[j] = n * (y[j] - v[j] * dot);
                }
            }
            if (mine) {
                Pack<T, V> o;
#pragma unroll
                for (int j = 0; j < V; ++j) from_float(o.v[j], y[j]);
                *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(s.y) + (row * s.heads + h) * a.dim + c0) = o;
            }
        }
    }

    if (BACKWARD && a.partial != nullptr) {
        __shared__ float sums[kWarps][2][kMaxDim];
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float t = dw[side][j];
                for (int o = 16; o >= span; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
                if (group == 0 && active) sums[warp][side][c0 + j] = t;
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * a.dim; i += kThreads) {
            const int side = i / a.dim, col = i - side * a.dim;
            float t = 0.0f;
            for (int k = 0; k < kWarps; ++k) t += sums[k][side][col];
            a.partial[(int64_t(blockIdx.x) * 2 + side) * a.dim + col] = t;
        }
    }
}

// dw[side][col] = the blocks' partial sums in a fixed order: warp w of a block of 8 adds blocks w, w + 8, ..,
// then the warps are added in order. One block per 32 columns.
template <typename W>
__global__ void __launch_bounds__(kThreads) weight_sum_kernel(const float* partial, int blocks, int dim, W* dq, W* dk) {
    __shared__ float sums[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + lane;
    float t = 0.0f;
    if (i < 2 * dim)
        for (int b = warp; b < blocks; b += kWarps) t += partial[int64_t(b) * 2 * dim + i];
    sums[warp][lane] = t;
    __syncthreads();
    if (warp == 0 && i < 2 * dim) {
        float r = 0.0f;
        for (int k = 0; k < kWarps; ++k) r += sums[k][lane];
        if (i < dim) {
            if (dq != nullptr) from_float(dq[i], r);
        } else if (dk != nullptr) {
            from_float(dk[i - dim], r);
        }
    }
}

constexpr int kBackwardBlocks = kNumSMs * 4;

template <typename T, int V>
fmd_status launch(const Args& a, bool backward, int grid, cudaStream_t s) {
    if (backward) head_rotary_kernel<T, V, true><<<grid, kThreads, 0, s>>>(a);
    else head_rotary_kernel<T, V, false><<<grid, kThreads, 0, s>>>(a);
    return check_launch();
}

bool vector_rows(const void* p, int64_t row, int64_t head, int size) {
    return aligned16(p) && (row * size) % 16 == 0 && (head * size) % 16 == 0;
}

}  // namespace
}  // namespace fmd

using namespace fmd;

extern "C" {

fmd_status fmd_head_rotary_workspace_bytes(int32_t dim, size_t* bytes) {
    if (bytes == nullptr || dim < 8 || dim > kMaxDim || dim % 8) return FMD_ERR_INVALID_ARGUMENT;
    *bytes = size_t(kBackwardBlocks) * 2 * dim * sizeof(float);
    return FMD_OK;
}

fmd_status fmd_head_rotary(const fmd_head_rotary_side* sides, int32_t type, int32_t weight_type, int64_t rows,
                           int32_t dim, int32_t rot, int32_t interleaved, float eps, const int64_t* positions,
                           const float* cos, const float* sin, int64_t table, int32_t backward, void* workspace,
                           size_t workspace_bytes, int32_t* flags, void* stream) {
    if (sides == nullptr || rows < 0 || dim < 8 || dim > kMaxDim || dim % 8 || rot < 8 || rot > dim || rot % 8 ||
        table < 0 || (type != FMD_F32 && type != FMD_BF16) || (weight_type != type && weight_type != FMD_F32))
        return FMD_ERR_INVALID_ARGUMENT;
    const bool norm = sides[0].w != nullptr || sides[1].w != nullptr;
    const int size = type == FMD_F32 ? 4 : 2;
    const int v = type == FMD_F32 ? 4 : (interleaved || rot % 16 == 0) ? 8 : 4;
    int span = 1;
    while (span * v < dim) span <<= 1;
    const int per_unit = 32 / span * kHeads;
    Args a{};
    bool any = false;
    for (int i = 0; i < 2; ++i) {
        const fmd_head_rotary_side& q = sides[i];
        if (q.heads < 0) return FMD_ERR_INVALID_ARGUMENT;
        any = any || q.heads > 0;
        if (rows > 0 && q.heads > 0) {
            if (q.y == nullptr || (!backward && q.x == nullptr) ||
                (backward && (q.g == nullptr || (q.w != nullptr && q.x == nullptr))))
                return FMD_ERR_INVALID_ARGUMENT;
            if (!aligned16(q.y) || (q.x != nullptr && !vector_rows(q.x, q.row_stride, q.head_stride, size)) ||
                (backward && !vector_rows(q.g, q.g_row_stride, q.g_head_stride, size)))
                return FMD_ERR_UNSUPPORTED;
        }
        a.side[i] = Side{q.x, q.g, q.y, q.w, q.row_stride, q.head_stride, q.g_row_stride, q.g_head_stride, q.heads,
                         (q.heads + per_unit - 1) / per_unit};
    }
    const bool weights = backward && norm;
    if (weights) {
        size_t need = 0;
        fmd_head_rotary_workspace_bytes(dim, &need);
        if (workspace == nullptr || workspace_bytes < need) return FMD_ERR_WORKSPACE;
    }
    const int64_t units = rows * (a.side[0].units + a.side[1].units);
    if (rows > 0 && any && (positions == nullptr || (table > 0 && (cos == nullptr || sin == nullptr))))
        return FMD_ERR_INVALID_ARGUMENT;
    a.positions = positions;
    a.cos = cos;
    a.sin = sin;
    a.partial = weights ? static_cast<float*>(workspace) : nullptr;
    a.flags = flags;
    a.rows = rows;
    a.table = table;
    a.eps = eps;
    a.inv_dim = 1.0f / float(dim);
    a.dim = dim;
    a.rot = rot;
    a.interleaved = interleaved != 0;
    a.w_float = weight_type == FMD_F32;
    const cudaStream_t s = as_stream(stream);
    int64_t blocks = (units + kWarps - 1) / kWarps;
    if (backward && blocks > kBackwardBlocks) blocks = kBackwardBlocks;
    if (blocks > INT32_MAX) return FMD_ERR_UNSUPPORTED;
    if (blocks > 0) {
        fmd_status st;
        if (type == FMD_F32) st = launch<float, 4>(a, backward, int(blocks), s);
        else if (v == 8) st = launch<__nv_bfloat16, 8>(a, backward, int(blocks), s);
        else st = launch<__nv_bfloat16, 4>(a, backward, int(blocks), s);
        if (st != FMD_OK) return st;
    }
    if (weights) {
        const int grid = (2 * dim + 31) / 32;
        if (weight_type == FMD_F32)
            weight_sum_kernel<float><<<grid, kThreads, 0, s>>>(a.partial, int(blocks), dim,
                                                               static_cast<float*>(sides[0].dw),
                                                               static_cast<float*>(sides[1].dw));
        else
            weight_sum_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a.partial, int(blocks), dim,
                                                                       static_cast<__nv_bfloat16*>(sides[0].dw),
                                                                       static_cast<__nv_bfloat16*>(sides[1].dw));
        return check_launch();
    }
    return FMD_OK;
}

}  // extern "C"
