// Packed attention in float32 on the FP32 cores, for heads of more than 64 values: forward, and the gradients of q and
// of k and v. (Smaller heads take the tensor cores, in three planes. Those kernels hold their tiles in full width; for wider
// heads the forward pass would have to keep q's planes in TMEM and stream keys by 64, the gradients to work on half a head at
// a time. That is not built.)
//
//   forward   s = scale q k^T (log2 units), running maximum m and sum l per row over key tiles:
//             o = (o 2^(m - m') + 2^(s - m') v),  l likewise;  out = o / l,  lse = m + log l
//   backward  p = exp(scale q k^T - lse),  dp = g v^T,  ds = p (dp - delta);
//             dq = scale ds k   (one kernel, a block per tile of queries)
//             dv = p^T g, dk = scale ds^T q   (one kernel, a block per tile of keys, over all rows that see it)
//
// Tiles of 64 rows x 64 keys in row-major shared memory, 256 threads, a 4 x 4 (rows ty + 16 i, columns tx + 16 j)
// piece of every product each. A block owns its output rows and adds in one order: no atomics, the same bits every
// time. Bound by the FP32 cores and shared memory: per four values of the inner axis a thread reads 8 vectors for 64
// products (2 x 4 pieces for 512 threads, two products an instruction: 20 % slower). One sequence of 3,000 rows, 4 heads
// of 128, forward and backward: 3.0 ms, 21 TFLOP/s of the cores' 70.

#include "packed_attention.cuh"

namespace fmd {
namespace {

constexpr int kM = 64, kN = 64, kThreads = 256, kDim = 128;

// rows [0, count) of src (row stride ld, dim values) into dst [64][kDim + 4], zeros elsewhere
template <typename RowOf>
__device__ __forceinline__ void load_tile(float* dst, const float* src, int count, int dim, RowOf row_of) {
#pragma unroll
    for (int i = threadIdx.x; i < 64 * kDim / 4; i += kThreads) {
        const int r = i / (kDim / 4), c = i % (kDim / 4) * 4;
        st4(dst + r * (kDim + 4) + c, r < count && c < dim ? ldg4(src + row_of(r) + c) : f4_zero());
    }
}

// acc[i][j] += sum_d a[ty + 16 i][d] b[tx + 16 j][d]
__device__ __forceinline__ void dots(const float* a, const float* b, int ty, int tx, float (&acc)[4][4]) {
#pragma unroll 4
    for (int d = 0; d < kDim; d += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * (kDim + 4) + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * (kDim + 4) + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
                acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
                acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
                acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
            }
    }
}

// column c of a thread's kDim / 16
__device__ __forceinline__ int column(int tx, int c) { return 4 * tx + 64 * (c / 4) + c % 4; }

// acc[i][c] += sum_n p[ty + 16 i][n] b[n][column(tx, c)] over the 64 rows of b
__device__ __forceinline__ void weigh(const float* p, const float* b, int ty, int tx, float (&acc)[4][kDim / 16]) {
#pragma unroll 2
    for (int n = 0; n < 64; n += 4) {
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(p + (ty + 16 * i) * (64 + 4) + n);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int c = 0; c < kDim / 64; ++c) {
                const float4 y = *reinterpret_cast<const float4*>(b + (n + u) * (kDim + 4) + 4 * tx + 64 * c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = u == 0 ? x[i].x : u == 1 ? x[i].y : u == 2 ? x[i].z : x[i].w;
                    acc[i][4 * c] = fmaf(w, y.x, acc[i][4 * c]);
                    acc[i][4 * c + 1] = fmaf(w, y.y, acc[i][4 * c + 1]);
                    acc[i][4 * c + 2] = fmaf(w, y.z, acc[i][4 * c + 2]);
                    acc[i][4 * c + 3] = fmaf(w, y.w, acc[i][4 * c + 3]);
                }
            }
        }
    }
}

__device__ __forceinline__ float sum16(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float max16(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Where a packed row of the tile lies; token0: the tile's first token (of the sequence).
struct Rows {
    int64_t row0;
    int group, head0, hq;
    __device__ int64_t at(int r, int64_t row_stride, int64_t head_stride) const {
        return (row0 + r / group) * row_stride + int64_t(head0 + r % group) * head_stride;
    }
    __device__ int64_t flat(int r) const { return (row0 + r / group) * hq + head0 + r % group; }
};

template <bool SPLIT>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Attn a) {
    extern __shared__ float smem[];
    float* qs = smem;
    float* ks = qs + 64 * (kDim + 4);
    float* vs = ks + 64 * (kDim + 4);
    float* ps = vs + 64 * (kDim + 4);
    const int per_tile = kM / a.group;
    int head;
    const Place place = block_place<false, true>(a, per_tile, &head);
    if (place.b < 0) return;
    const Span s = load_span(a, place.b);
    const int64_t token0 = int64_t(place.tile) * per_tile;
    const int tokens = int(min(int64_t(per_tile), s.rows - token0)), rows = tokens * a.group;
    const Rows at{s.row0 + token0, a.group, head * a.group, a.hq};
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float* kp = static_cast<const float*>(a.k) + s.key0 * a.k_row + head * a.k_head;
    const float* vp = static_cast<const float*>(a.v) + s.key0 * a.v_row + head * a.v_head;
    load_tile(qs, static_cast<const float*>(a.q), rows, a.dim,
                     [&](int r) { return at.at(r, a.q_row, a.q_head); });
    int64_t limit[4];
    float m[4], l[4], o[4][kDim / 16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i;
        limit[i] = r < rows ? seen(s, a.causal, token0 + r / a.group) : 0;
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < kDim / 16; ++c) o[i][c] = 0.0f;
    }
    int64_t end = seen(s, a.causal, token0 + tokens - 1), from = 0;
    if (SPLIT) {  // a range of the key tiles
        const int64_t share = (((end + kN - 1) / kN + gridDim.z - 1) / gridDim.z) * kN;
        from = min(end, blockIdx.z * share);
        end = min(end, from + share);
    }
    const float scale = a.scale * kLog2e;
    for (int64_t n0 = from; n0 < end; n0 += kN) {
        const int n = int(min(int64_t(kN), end - n0));
        __syncthreads();
        load_tile(ks, kp + n0 * a.k_row, n, a.dim, [&](int r) { return r * a.k_row; });
        load_tile(vs, vp + n0 * a.v_row, n, a.dim, [&](int r) { return r * a.v_row; });
        __syncthreads();
        float x[4][4] = {};
        dots(qs, ks, ty, tx, x);
        float keep[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i][j] = n0 + tx + 16 * j < limit[i] ? x[i][j] * scale : -INFINITY;
                top = fmaxf(top, x[i][j]);
            }
            top = fmaxf(m[i], max16(top));
            const float base = top == -INFINITY ? 0.0f : top;  // a row with nothing yet: exp2(-inf) stays 0
            keep[i] = exp2f(m[i] - base);
            m[i] = top;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(x[i][j] - base);
                sum += p;
                ps[(ty + 16 * i) * (64 + 4) + tx + 16 * j] = p;
            }
            l[i] = l[i] * keep[i] + sum16(sum);
        }
        __syncthreads();
        // a tile's sum starts from zero: n keys are n / 64 + 64 additions in a row, not n
        float tile[4][kDim / 16] = {};
        weigh(ps, vs, ty, tx, tile);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < kDim / 16; ++c) o[i][c] = fmaf(o[i][c], keep[i], tile[i][c]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i;
        if (r >= rows) continue;
        const float inv = l[i] > 0.0f ? 1.0f / l[i] : (l[i] == 0.0f ? 0.0f : l[i]);
        const int64_t flat = at.flat(r) + (SPLIT ? int64_t(blockIdx.z) * a.rows * a.hq : 0);
        float* out = (SPLIT ? a.part : static_cast<float*>(a.out)) + flat * a.dim;
#pragma unroll
        for (int c = 0; c < kDim / 16; ++c) {
            const int col = column(tx, c);
            if (col < a.dim) out[col] = o[i][c] * inv;
        }
        float* lse = SPLIT ? a.part_lse : a.lse;
        if (lse != nullptr && tx == 0) lse[flat] = l[i] == 0.0f ? -INFINITY : m[i] * kLn2 + logf(l[i]);
    }
}

// p and ds of one 4 x 4 piece: rows ty + 16 i of the first operand, columns tx + 16 j of the second
__device__ __forceinline__ float weight_of(float dot, float scale, float lse2, bool there) {
    return there ? exp2f(dot * scale - lse2) : 0.0f;
}

__global__ void __launch_bounds__(kThreads) query_gradient_kernel(const Attn a) {
    extern __shared__ float smem[];
    float* qs = smem;
    float* gs = qs + 64 * (kDim + 4);
    float* ks = gs + 64 * (kDim + 4);
    float* vs = ks + 64 * (kDim + 4);
    float* ds = vs + 64 * (kDim + 4);
    const int per_tile = kM / a.group;
    int head;
    const Place place = block_place<false>(a, per_tile, &head);
    if (place.b < 0) return;
    const Span s = load_span(a, place.b);
    const int64_t token0 = int64_t(place.tile) * per_tile;
    const int tokens = int(min(int64_t(per_tile), s.rows - token0)), rows = tokens * a.group;
    const Rows at{s.row0 + token0, a.group, head * a.group, a.hq};
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float* kp = static_cast<const float*>(a.k) + s.key0 * a.k_row + head * a.k_head;
    const float* vp = static_cast<const float*>(a.v) + s.key0 * a.v_row + head * a.v_head;
    load_tile(qs, static_cast<const float*>(a.q), rows, a.dim,
                     [&](int r) { return at.at(r, a.q_row, a.q_head); });
    load_tile(gs, static_cast<const float*>(a.g), rows, a.dim,
                     [&](int r) { return at.at(r, a.g_row, a.g_head); });
    int64_t limit[4];
    float lse2[4], delta[4], dq[4][kDim / 16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i;
        lse2[i] = r < rows ? a.lse[at.flat(r)] * kLog2e : -INFINITY;
        limit[i] = lse2[i] != -INFINITY ? seen(s, a.causal, token0 + r / a.group) : 0;  // an empty row has no share
        if (!scores_count(a, limit[i])) limit[i] = 0;
        delta[i] = r < rows ? a.delta[at.flat(r)] : 0.0f;
#pragma unroll
        for (int c = 0; c < kDim / 16; ++c) dq[i][c] = 0.0f;
    }
    int64_t end = seen(s, a.causal, token0 + tokens - 1), from = 0;
    if (gridDim.z > 1) {  // a range of the key tiles
        const int64_t share = (((end + kN - 1) / kN + gridDim.z - 1) / gridDim.z) * kN;
        from = min(end, blockIdx.z * share);
        end = min(end, from + share);
    }
    const float scale = a.scale * kLog2e;
    for (int64_t n0 = from; n0 < end; n0 += kN) {
        const int n = int(min(int64_t(kN), end - n0));
        __syncthreads();
        load_tile(ks, kp + n0 * a.k_row, n, a.dim, [&](int r) { return r * a.k_row; });
        load_tile(vs, vp + n0 * a.v_row, n, a.dim, [&](int r) { return r * a.v_row; });
        __syncthreads();
        float x[4][4] = {}, y[4][4] = {};
        dots(qs, ks, ty, tx, x);
        dots(gs, vs, ty, tx, y);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool there = n0 + tx + 16 * j < limit[i];
                const float p = weight_of(x[i][j], scale, lse2[i], there);
                ds[(ty + 16 * i) * (64 + 4) + tx + 16 * j] = there ? p * (y[i][j] - delta[i]) : 0.0f;
            }
        __syncthreads();
        weigh(ds, ks, ty, tx, dq);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i;
        if (r >= rows) continue;
        float* out = gridDim.z > 1 ? a.part + int64_t(blockIdx.z) * a.rows * a.hq * a.dim : static_cast<float*>(a.dq);
        out += at.flat(r) * a.dim;
#pragma unroll
        for (int c = 0; c < kDim / 16; ++c) {
            const int col = column(tx, c);
            if (col < a.dim) out[col] = dq[i][c] * a.scale;
        }
    }
}

__global__ void __launch_bounds__(kThreads) key_gradient_kernel(const Attn a) {
    extern __shared__ float smem[];
    float* ks = smem;
    float* vs = ks + 64 * (kDim + 4);
    float* qs = vs + 64 * (kDim + 4);
    float* gs = qs + 64 * (kDim + 4);
    float* ps = gs + 64 * (kDim + 4);
    float* ds = ps + 64 * (64 + 4);
    __shared__ float lse2[64], delta[64];
    __shared__ int64_t limit[64];
    int head;
    const Place place = block_place<true>(a, kN, &head);
    if (place.b < 0) return;
    const Span s = load_span(a, place.b);
    const int64_t n0 = int64_t(place.tile) * kN;
    const int n = int(max(int64_t(0), min(int64_t(kN), s.keys - n0)));
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    load_tile(ks, static_cast<const float*>(a.k) + (s.key0 + n0) * a.k_row + head * a.k_head, n, a.dim,
                     [&](int r) { return r * a.k_row; });
    load_tile(vs, static_cast<const float*>(a.v) + (s.key0 + n0) * a.v_row + head * a.v_head, n, a.dim,
                     [&](int r) { return r * a.v_row; });
    float dk[4][kDim / 16] = {}, dv[4][kDim / 16] = {};
    const int per_tile = kM / a.group;
    const float scale = a.scale * kLog2e;
    // tiles of rows from the one that holds the first token that sees key n0
    int64_t tile = a.causal ? max(int64_t(0), n0 + s.rows - s.keys) / per_tile : 0;
    int64_t tiles = n > 0 ? (s.rows + per_tile - 1) / per_tile : tile;
    if (gridDim.z > 1) {  // a range of them
        const int64_t share = (max(int64_t(0), tiles - tile) + gridDim.z - 1) / gridDim.z;
        tile += blockIdx.z * share;
        tiles = min(tiles, tile + share);
    }
    for (; tile < tiles; ++tile) {
        const int64_t token0 = tile * per_tile;
        const int tokens = int(min(int64_t(per_tile), s.rows - token0)), rows = tokens * a.group;
        const Rows at{s.row0 + token0, a.group, head * a.group, a.hq};
        __syncthreads();
        load_tile(qs, static_cast<const float*>(a.q), rows, a.dim,
                         [&](int r) { return at.at(r, a.q_row, a.q_head); });
        load_tile(gs, static_cast<const float*>(a.g), rows, a.dim,
                         [&](int r) { return at.at(r, a.g_row, a.g_head); });
        if (threadIdx.x < 64) {
            const int r = threadIdx.x;
            lse2[r] = r < rows ? a.lse[at.flat(r)] * kLog2e : -INFINITY;
            limit[r] = lse2[r] != -INFINITY ? seen(s, a.causal, token0 + r / a.group) : 0;
            delta[r] = r < rows ? a.delta[at.flat(r)] : 0.0f;
        }
        __syncthreads();
        float x[4][4] = {}, y[4][4] = {};
        dots(ks, qs, ty, tx, x);
        dots(vs, gs, ty, tx, y);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = ty + 16 * i, r = tx + 16 * j;
                const bool there = key < n && n0 + key < limit[r];
                const float p = weight_of(x[i][j], scale, lse2[r], there);
                ps[key * (64 + 4) + r] = p;
                ds[key * (64 + 4) + r] = there ? p * (y[i][j] - delta[r]) : 0.0f;
            }
        __syncthreads();
        weigh(ps, gs, ty, tx, dv);
        weigh(ds, qs, ty, tx, dk);
    }
    const int64_t part = int64_t(blockIdx.z) * a.keys * a.hk * a.dim;
    float* dk_out = gridDim.z > 1 ? a.part_dk + part : static_cast<float*>(a.dk);
    float* dv_out = gridDim.z > 1 ? a.part_dv + part : static_cast<float*>(a.dv);
    // every row of the slot is written: keys that no query may see have zero gradients
    const int out_rows = int(min(int64_t(kN), s.slot - n0));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int key = ty + 16 * i;
        if (key >= out_rows) continue;
        const int64_t flat = ((s.key0 + n0 + key) * a.hk + head) * a.dim;
#pragma unroll
        for (int c = 0; c < kDim / 16; ++c) {
            const int col = column(tx, c);
            if (col < a.dim) {
                dk_out[flat + col] = scores_count(a, s.keys) ? dk[i][c] * a.scale : 0.0f;
                dv_out[flat + col] = dv[i][c];
            }
        }
    }
}

}  // namespace

fmd_status attention_forward_simt(const Attn& a, int splits, cudaStream_t s) {
    const size_t bytes = size_t(3 * 64 * (kDim + 4) + 64 * 68) * sizeof(float);
    const void* kernel = splits > 1 ? (const void*)forward_kernel<true> : (const void*)forward_kernel<false>;
    const fmd_status st = grant_dynamic_smem(kernel, bytes);
    if (st != FMD_OK) return st;
    const dim3 grid(unsigned(tile_bound(a.rows, a.batch, kM / a.group) * a.hk), 1, unsigned(splits));
    if (splits > 1) forward_kernel<true><<<grid, kThreads, bytes, s>>>(a);
    else forward_kernel<false><<<grid, kThreads, bytes, s>>>(a);
    return check_launch();
}

fmd_status attention_backward_simt(const Attn& a, BackwardSplits splits, cudaStream_t s) {
    const size_t bytes = size_t(4 * 64 * (kDim + 4) + 2 * 64 * 68) * sizeof(float);
    fmd_status st = grant_dynamic_smem((const void*)query_gradient_kernel, bytes);
    if (st == FMD_OK) st = grant_dynamic_smem((const void*)key_gradient_kernel, bytes);
    if (st != FMD_OK) return st;
    if (a.dq != nullptr && a.rows > 0) {
        const dim3 grid(unsigned(tile_bound(a.rows, a.batch, kM / a.group) * a.hk), 1, unsigned(splits.queries));
        query_gradient_kernel<<<grid, kThreads, bytes, s>>>(a);
        if ((st = check_launch()) != FMD_OK) return st;
    }
    if (a.dk != nullptr && a.keys > 0) {
        const dim3 grid(unsigned(tile_bound(a.keys, a.batch, kN) * a.hk), 1, unsigned(splits.keys));
        key_gradient_kernel<<<grid, kThreads, bytes, s>>>(a);
        st = check_launch();
    }
    return st;
}

}  // namespace fmd
