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
// What bounds it: memory, then the issue of instructions (about ten per value), so a lane does as little else as it
// can. It holds two quads of a head, four whole pairs: (x_p .. x_{p+3}, x_{p+R/2} ..) or, interleaved, eight values
// side by side, so that no pair crosses lanes and the lane needs four cosines and four sines; lanes behind the turned
// part hold eight values and turn by (1, 0). A head is D / 8 lanes, padded to a power of two for the sums; the lane
// groups of a warp take the heads of one row, or of several rows where a row has fewer. A warp keeps its heads (all
// of the queries or all of the keys) and walks over the rows: weights and addresses are set up once, the next
// position is loaded a row ahead, and the loads of all its heads are in flight together. The weights' gradients stay
// in registers over the walk; a block adds its warps in warp order, a second kernel the blocks in block order: no
// atomics, the same bits every time.
//
// Measured: 32,000 rows of 16 + 4 heads of 128, bfloat16: forward 83 us (3.9 TB/s), backward 139 us (3.5 TB/s) of
// the 50 and 75 us that the bytes take at the copy rate of 6.55 TB/s; what is left is latency (a third of the warps
// fit, issue slots 57 and 48 % busy). 10,007 rows of 24 heads of 96 without a norm: 16 us (5.9 TB/s).

#include <cuda_bf16.h>

#include "common.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 128, kMaxHeads = 1024;

struct Side {
    const void* x;    // [rows, heads, D], strides row and head
    const void* g;    // gradient of the output, strides grow and ghead (backward)
    void* y;          // output (or the input's gradient), contiguous
    const void* w;    // [D] or null
    int64_t row, head, grow, ghead;
    int32_t heads;
    int32_t across;   // heads of a row that a warp's lane groups take at a time (a power of two)
    int32_t units;    // warps that share a row
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
    int32_t dim, rot, w_float;
};

// A lane's two quads as they are in memory, kept packed until they are used; then as four pairs of neighbours.
template <typename T>
struct Raw;

template <>
struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p, int gap) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + gap);
    }
    __device__ __forceinline__ void zero() { a = b = f4_zero(); }
    __device__ __forceinline__ void get(float2 (&v)[4]) const {
        v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w);
        v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
    }
    static __device__ __forceinline__ void put(float* p, int gap, const float2 (&v)[4]) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        *reinterpret_cast<float4*>(p + gap) = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
};

template <>
struct Raw<__nv_bfloat16> {
    uint2 a, b;
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int gap) {
        if (gap == 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(p);
            a = make_uint2(w.x, w.y), b = make_uint2(w.z, w.w);
        } else {
            a = *reinterpret_cast<const uint2*>(p);
            b = *reinterpret_cast<const uint2*>(p + gap);
        }
    }
    __device__ __forceinline__ void zero() { a = b = make_uint2(0, 0); }
    __device__ __forceinline__ void get(float2 (&v)[4]) const {
        v[0] = unpack_bf16(a.x), v[1] = unpack_bf16(a.y), v[2] = unpack_bf16(b.x), v[3] = unpack_bf16(b.y);
    }
    static __device__ __forceinline__ void put(__nv_bfloat16* p, int gap, const float2 (&v)[4]) {
        const uint2 a = make_uint2(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y));
        const uint2 b = make_uint2(pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
        if (gap == 4) {
            *reinterpret_cast<uint4*>(p) = make_uint4(a.x, a.y, b.x, b.y);
        } else {
            *reinterpret_cast<uint2*>(p) = a;
            *reinterpret_cast<uint2*>(p + gap) = b;
        }
    }
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float& o, float v) { o = v; }
__device__ __forceinline__ void from_float(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Turns the lane's four pairs: c and s hold the four cosines and sines, two and two (s negated to turn back).
template <bool INTER>
__device__ __forceinline__ void turn(float2 (&v)[4], const float2 (&c)[2], const float2 (&s)[2]) {
    if (INTER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float ci = i & 1 ? c[i / 2].y : c[i / 2].x, si = i & 1 ? s[i / 2].y : s[i / 2].x;
            v[i] = fma2(v[i], both(ci), mul2(make_float2(v[i].y, v[i].x), make_float2(-si, si)));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 a = v[i], b = v[i + 2];
            v[i] = fma2(a, c[i], mul2(b, make_float2(-s[i].x, -s[i].y)));
            v[i + 2] = fma2(b, c[i], mul2(a, s[i]));
        }
    }
}

// The sum of the pairwise products of a lane, over the lanes of a head.
__device__ __forceinline__ float dot(const float2 (&a)[4], const float2 (&b)[4], int span) {
    float2 t = mul2(a[0], b[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) t = fma2(a[i], b[i], t);
    float sum = t.x + t.y;
    for (int o = span / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// Blocks of an SM by the registers they need: the backward pass holds twice the loads and the weights' sums, a norm the
// weights. (Four blocks with a norm, or three in the backward pass, spill: 32,000 rows forward 80 us -> 95.)
template <bool NORM, bool BACKWARD>
constexpr int kResident = BACKWARD ? 2 : NORM ? 3 : 4;

// HEADS: heads of a lane group and row whose loads are in flight together.
template <typename T, bool INTER, bool NORM, bool BACKWARD, int HEADS>
__global__ void __launch_bounds__(kThreads, kResident<NORM, BACKWARD>) head_rotary_kernel(const Args a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lanes = a.dim / 8;
    int span = 1;
    while (span < lanes) span <<= 1;
    const int groups = 32 / span, group = lane / span, sub = lane % span;
    const bool active = sub < lanes;
    const int half = a.rot / 2;
    const bool turned = 8 * sub < a.rot;
    const int qa = !INTER && turned ? 4 * sub : 8 * sub, gap = !INTER && turned ? half : 4;  // the second quad

    // this warp's heads: unit `u` of the row's units
    const int units = a.side[0].units + a.side[1].units;
    const int64_t walker = int64_t(blockIdx.x) * kWarps + warp;
    const int64_t walkers = int64_t(gridDim.x) * kWarps / units;  // warps with the same unit
    const int64_t start = walker / units;
    int u = int(walker - start * units);
    const int which = u >= a.side[0].units;
    const Side s = a.side[which];
    if (which) u -= a.side[0].units;
    const int across = s.across, rows_at_once = groups / across;
    const int head0 = u * HEADS * across + group % across;
    const int64_t row_step = walkers * rows_at_once;

    float2 w[4], dw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        dw[j] = both(0.0f);
        w[j] = both(1.0f);
        if (NORM && s.w != nullptr && active) {
            const int at = qa + (j < 2 ? 2 * j : gap + 2 * j - 4);
            if (a.w_float) w[j] = make_float2(static_cast<const float*>(s.w)[at], static_cast<const float*>(s.w)[at + 1]);
            else w[j] = make_float2(to_float(static_cast<const T*>(s.w)[at]), to_float(static_cast<const T*>(s.w)[at + 1]));
        }
    }
    const bool norm = NORM && s.w != nullptr;
    // addresses are set up once and move by the walk's step
    int64_t row = start * rows_at_once + group / across;
    const T* x = static_cast<const T*>(s.x) + row * s.row + head0 * s.head + qa;
    const T* g = static_cast<const T*>(s.g) + row * s.grow + head0 * s.ghead + qa;
    T* y = static_cast<T*>(s.y) + (row * s.heads + head0) * a.dim + qa;
    const int64_t x_step = row_step * s.row, g_step = row_step * s.grow, y_step = row_step * s.heads * a.dim;
    const int64_t x_head = across * s.head, g_head = across * s.ghead;
    const int y_head = across * a.dim;
    int64_t next = start < walkers && row < a.rows ? a.positions[row] : 0;
    // the loop's bound is the warp's first row: its lanes stay together for the shuffles
    for (int64_t base = start < walkers ? row - group / across : a.rows; base < a.rows; base += row_step) {
        const bool here = active && row < a.rows;
        Raw<T> xs[HEADS], gs[HEADS];
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            const bool mine = here && head0 + i * across < s.heads;
            if (!BACKWARD || norm) {
                if (mine) xs[i].load(x + i * x_head, gap);
                else xs[i].zero();
            }
            if (BACKWARD) {
                if (mine) gs[i].load(g + i * g_head, gap);
                else gs[i].zero();
            }
        }
        const int64_t pos = next;
        if (row + row_step < a.rows) next = a.positions[row + row_step];
        const bool known = pos >= 0 && pos < a.table;
        if (!known && row < a.rows && sub == 0) raise_flag(a.flags, FMD_FLAG_INDEX_RANGE);
        float2 c[2] = {both(1.0f), both(1.0f)}, sn[2] = {both(0.0f), both(0.0f)};
        if (turned && here) {
            float4 cf = f4_zero(), sf = f4_zero();
            if (known) {
                cf = ldg4(a.cos + pos * half + 4 * sub);
                sf = ldg4(a.sin + pos * half + 4 * sub);
            }
            const float sign = BACKWARD ? -1.0f : 1.0f;
            c[0] = make_float2(cf.x, cf.y), c[1] = make_float2(cf.z, cf.w);
            sn[0] = make_float2(sign * sf.x, sign * sf.y), sn[1] = make_float2(sign * sf.z, sign * sf.w);
        }
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            if (u * HEADS * across + i * across >= s.heads) break;  // the same for the whole warp
            const bool mine = here && head0 + i * across < s.heads;
            float2 v[4], o[4];
            float n = 1.0f;
            if (!BACKWARD || norm) xs[i].get(v);
            if (norm) {
                n = rsqrtf(dot(v, v, span) * a.inv_dim + a.eps);
                if (BACKWARD && !mine) n = 0.0f;  // with eps = 0 it is infinite there, and zeros times it no numbers
            }
            if (!BACKWARD) {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = norm ? mul2(v[j], mul2(both(n), w[j])) : v[j];
                turn<INTER>(o, c, sn);
            } else {
                gs[i].get(o);
                turn<INTER>(o, c, sn);
                if (norm) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[j] = mul2(v[j], both(n));  // u; zero, as its gradient, in lanes without a head
                        dw[j] = fma2(o[j], v[j], dw[j]);
                        o[j] = mul2(o[j], w[j]);
                    }
                    const float mean = -dot(o, v, span) * a.inv_dim;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = mul2(both(n), fma2(v[j], both(mean), o[j]));
                }
            }
            if (mine) Raw<T>::put(y + i * y_head, gap, o);
        }
        row += row_step;
        x += x_step;
        g += g_step;
        y += y_step;
    }

    if (BACKWARD && NORM && a.partial != nullptr) {
        __shared__ float sums[kWarps][kMaxDim];
        __shared__ int side_of[kWarps];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float t = j & 1 ? dw[j / 2].y : dw[j / 2].x;
            for (int o = 16; o >= span; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (group == 0 && active) sums[warp][qa + (j < 4 ? j : gap + j - 4)] = t;
        }
        if (lane == 0) side_of[warp] = which;
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * a.dim; i += kThreads) {
            const int side = i / a.dim, col = i - side * a.dim;
            float t = 0.0f;
            for (int k = 0; k < kWarps; ++k) t += side_of[k] == side ? sums[k][col] : 0.0f;
            a.partial[int64_t(blockIdx.x) * 2 * a.dim + i] = t;
        }
    }
}

// dw[side][col] = the blocks' partial sums in a fixed order: warp w of 32 adds blocks w, w + 32, .., then the warps
// are added in order. One block per 32 columns.
template <typename W>
__global__ void __launch_bounds__(1024) weight_sum_kernel(const float* partial, int blocks, int dim, W* dq, W* dk) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + lane;
    float t = 0.0f;
    if (i < 2 * dim) {
#pragma unroll 8
        for (int b = warp; b < blocks; b += 32) t += partial[int64_t(b) * 2 * dim + i];
    }
    sums[warp][lane] = t;
    __syncthreads();
    if (warp == 0 && i < 2 * dim) {
        float r = 0.0f;
        for (int k = 0; k < 32; ++k) r += sums[k][lane];
        if (i < dim) {
            if (dq != nullptr) from_float(dq[i], r);
        } else if (dk != nullptr) {
            from_float(dk[i - dim], r);
        }
    }
}

// Heads per lane group whose loads are in flight together: 16 bytes of each in 16 bits, 32 in 32.
template <typename T, bool BACKWARD>
constexpr int kHeadsOf = sizeof(T) == 2 && !BACKWARD ? 4 : 2;

template <typename T, bool INTER, bool NORM, bool BACKWARD>
fmd_status launch(Args& a, int* blocks, cudaStream_t s) {
    constexpr int H = kHeadsOf<T, BACKWARD>;
    int span = 1;
    while (span * 8 < a.dim) span <<= 1;
    const int groups = 32 / span;
    int rows_at_once = groups;  // of the side that takes the fewest: its warps walk the furthest
    for (Side& q : a.side) {
        q.across = 1;
        while (q.across < groups && q.across < q.heads) q.across <<= 1;
        q.units = (q.heads + H * q.across - 1) / (H * q.across);
        if (q.heads > 0 && groups / q.across < rows_at_once) rows_at_once = groups / q.across;
    }
    const int units = a.side[0].units + a.side[1].units;
    *blocks = 0;
    if (a.rows == 0 || units == 0) return FMD_OK;
    // all blocks resident, and a warp at least for every unit: kMaxHeads heads are fewer units than the grid's warps
    const int64_t wanted = ((a.rows + rows_at_once - 1) / rows_at_once * units + kWarps - 1) / kWarps;
    const int most = kNumSMs * kResident<NORM, BACKWARD>;
    *blocks = int(wanted < most ? wanted : most);
    head_rotary_kernel<T, INTER, NORM, BACKWARD, H><<<*blocks, kThreads, 0, s>>>(a);
    return check_launch();
}

template <typename T>
fmd_status launch(Args& a, bool inter, bool norm, bool backward, int* blocks, cudaStream_t s) {
    if (backward) {
        if (inter) return norm ? launch<T, true, true, true>(a, blocks, s) : launch<T, true, false, true>(a, blocks, s);
        return norm ? launch<T, false, true, true>(a, blocks, s) : launch<T, false, false, true>(a, blocks, s);
    }
    if (inter) return norm ? launch<T, true, true, false>(a, blocks, s) : launch<T, true, false, false>(a, blocks, s);
    return norm ? launch<T, false, true, false>(a, blocks, s) : launch<T, false, false, false>(a, blocks, s);
}

}  // namespace
}  // namespace fmd

using namespace fmd;

extern "C" {

fmd_status fmd_head_rotary_workspace_bytes(int32_t dim, size_t* bytes) {
    if (bytes == nullptr || dim < 8 || dim > kMaxDim || dim % 8) return FMD_ERR_INVALID_ARGUMENT;
    *bytes = size_t(kNumSMs * kResident<true, true>) * 2 * dim * sizeof(float);
    return FMD_OK;
}

fmd_status fmd_head_rotary(const fmd_head_rotary_side* sides, int32_t type, int32_t weight_type, int64_t rows,
                           int32_t dim, int32_t rot, int32_t interleaved, float eps, const int64_t* positions,
                           const float* cos, const float* sin, int64_t table, int32_t backward, void* workspace,
                           size_t workspace_bytes, int32_t* flags, void* stream) {
    if (sides == nullptr || rows < 0 || dim < 8 || dim > kMaxDim || dim % 8 || rot < 8 || rot > dim || rot % 8 ||
        table < 0 || (type != FMD_F32 && type != FMD_BF16) || (weight_type != type && weight_type != FMD_F32) ||
        !(eps >= 0.0f && eps <= 1.0e38f))
        return FMD_ERR_INVALID_ARGUMENT;
    const bool norm = sides[0].w != nullptr || sides[1].w != nullptr;
    const int size = type == FMD_F32 ? 4 : 2;
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
            if (q.heads > kMaxHeads || !aligned16(q.y) || (q.x != nullptr && !vector_rows(q.x, q.row_stride, q.head_stride, size)) ||
                (backward && !vector_rows(q.g, q.g_row_stride, q.g_head_stride, size)))
                return FMD_ERR_UNSUPPORTED;
        }
        a.side[i] = Side{q.x, q.g, q.y, q.w, q.row_stride, q.head_stride, q.g_row_stride, q.g_head_stride, q.heads, 1, 0};
    }
    const bool weights = backward && norm;
    if (weights) {
        size_t need = 0;
        fmd_head_rotary_workspace_bytes(dim, &need);
        if (workspace == nullptr || workspace_bytes < need) return FMD_ERR_WORKSPACE;
    }
    if (rows > 0 && any && (positions == nullptr || (table > 0 && (cos == nullptr || sin == nullptr))))
        return FMD_ERR_INVALID_ARGUMENT;
    if (rows > 0 && any && (!aligned16(cos) || !aligned16(sin))) return FMD_ERR_UNSUPPORTED;
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
    a.w_float = weight_type == FMD_F32;
    const cudaStream_t s = as_stream(stream);
    int blocks = 0;
    const fmd_status st = type == FMD_F32 ? launch<float>(a, interleaved != 0, norm, backward != 0, &blocks, s)
                                          : launch<__nv_bfloat16>(a, interleaved != 0, norm, backward != 0, &blocks, s);
    if (st != FMD_OK) return st;
    if (weights) {
        const int grid = (2 * dim + 31) / 32;
        if (weight_type == FMD_F32)
            weight_sum_kernel<float><<<grid, 1024, 0, s>>>(a.partial, blocks, dim,
                                                           static_cast<float*>(sides[0].dw),
                                                           static_cast<float*>(sides[1].dw));
        else
            weight_sum_kernel<__nv_bfloat16><<<grid, 1024, 0, s>>>(a.partial, blocks, dim,
                                                                   static_cast<__nv_bfloat16*>(sides[0].dw),
                                                                   static_cast<__nv_bfloat16*>(sides[1].dw));
        return check_launch();
    }
    return FMD_OK;
}

}  // extern "C"
