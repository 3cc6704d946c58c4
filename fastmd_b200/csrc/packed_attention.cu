// C entry points of packed attention: argument checks, the choice of kernels, and the row sums that the backward
// pass starts from.

#include <cfloat>

#include "packed_attention.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float attn_float(float v) { return v; }
__device__ __forceinline__ float attn_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ void store4(float* p, float4 v) { st4(p, v); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// out and lse of the splits of the keys together: out = sum_z exp(lse_z - lse) out_z. Many splits of few rows: a block
// per row, 32 threads of four values each, times eight that share the splits (their loads are what the time goes to).
template <typename T>
__global__ void __launch_bounds__(kThreads) join_kernel(const Attn a, int splits) {
    constexpr int kParts = kThreads / 32;
    __shared__ float4 sums[kParts][32];
    __shared__ float weights[kParts];
    const int quad = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t row = blockIdx.x, all = a.rows * a.hq;
    float top = -INFINITY, sum = 0.0f;
    for (int z = quad; z < splits; z += 32) top = fmaxf(top, a.part_lse[z * all + row]);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    const float base = top == -INFINITY ? 0.0f : top;
    float4 o = f4_zero();
#pragma unroll 4
    for (int z = part; z < splits; z += kParts) {
        const float lse = a.part_lse[z * all + row];
        if (lse == -INFINITY) continue;  // a split without keys of this row wrote nothing else
        const float w = exp2f((lse - base) * kLog2e);
        sum += w;
        if (quad * 4 < a.dim) {
            const float4 v = *reinterpret_cast<const float4*>(a.part + (z * all + row) * a.dim + quad * 4);
            o = make_float4(fmaf(w, v.x, o.x), fmaf(w, v.y, o.y), fmaf(w, v.z, o.z), fmaf(w, v.w, o.w));
        }
    }
    sums[part][quad] = o;
    if (quad == 0) weights[part] = sum;
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int i = 1; i < kParts; ++i) {
        o = f4_add(o, sums[i][quad]);
        sum += weights[i];
    }
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
    if (quad * 4 < a.dim)
        store4(static_cast<T*>(a.out) + row * a.dim + quad * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    if (quad == 0 && a.lse != nullptr) a.lse[row] = sum == 0.0f ? -INFINITY : top + logf(sum);
}

// The same for few splits of many rows: a thread per row and four values.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_few_kernel(const Attn a, int splits) {
    const int quads = a.dim / 4;
    const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x, all = a.rows * a.hq, row = i / quads;
    const int quad = int(i - row * quads);
    if (row >= all) return;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll 4
    for (int z = 0; z < splits; ++z) top = fmaxf(top, a.part_lse[z * all + row]);
    const float base = top == -INFINITY ? 0.0f : top;
    float4 o = f4_zero();
#pragma unroll 4
    for (int z = 0; z < splits; ++z) {
        const float lse = a.part_lse[z * all + row];
        if (lse == -INFINITY) continue;
        const float w = exp2f((lse - base) * kLog2e);
        const float4 v = *reinterpret_cast<const float4*>(a.part + (z * all + row) * a.dim + quad * 4);
        sum += w;
        o = make_float4(fmaf(w, v.x, o.x), fmaf(w, v.y, o.y), fmaf(w, v.z, o.z), fmaf(w, v.w, o.w));
    }
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
    store4(static_cast<T*>(a.out) + row * a.dim + quad * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    if (quad == 0 && a.lse != nullptr) a.lse[row] = sum == 0.0f ? -INFINITY : top + logf(sum);
}

// A block per row where its eight parts have enough splits each for the rows that an SM has to take, about 128 rows a
// split at the most; else a thread per four values. us of the whole call, by blocks and by threads:
//   rows    64, splits 14: 18.4, 22.0     128,  8: 17.8, 19.5     512,  2: 38.6, 39.0     512, 32: 24.0, 33.8
//   rows 1,024, splits  4: 22.2, 20.8   1,024,  7: 26.9, 27.0   1,024, 10: 23.4, 24.4   1,024, 32: 26.7, 33.9
//   rows 2,048, splits  6: 34.1, 31.0   2,048, 14: 43.7, 42.2   1,536, 18: 36.2, 38.2   4,224,  4: 51.7, 42.7
template <typename T>
fmd_status join(const Attn& a, int splits, cudaStream_t s) {
    const int64_t all = a.rows * a.hq;
    const bool many = all <= 128 * int64_t(splits);
    const int64_t blocks = many ? all : (all * (a.dim / 4) + kThreads - 1) / kThreads;
    if (blocks > INT32_MAX) return FMD_ERR_UNSUPPORTED;
    if (many) join_kernel<T><<<unsigned(blocks), kThreads, 0, s>>>(a, splits);
    else join_few_kernel<T><<<unsigned(blocks), kThreads, 0, s>>>(a, splits);
    return check_launch();
}

// out[i] = the sum of the splits' parts, four values a thread; y: a second pair of arrays.
template <typename T>
__global__ void __launch_bounds__(kThreads) add_kernel(const float* part0, const float* part1, T* out0, T* out1,
                                                       int64_t values, int splits) {
    const float* part = blockIdx.y ? part1 : part0;
    T* out = blockIdx.y ? out1 : out0;
    const int64_t i = (int64_t(blockIdx.x) * kThreads + threadIdx.x) * 4;
    if (i >= values) return;
    float4 sum = f4_zero();
#pragma unroll 4
    for (int z = 0; z < splits; ++z) sum = f4_add(sum, *reinterpret_cast<const float4*>(part + z * values + i));
    store4(out + i, sum);
}

template <typename T>
fmd_status add(const float* part0, const float* part1, void* out0, void* out1, int64_t values, int splits,
               cudaStream_t s) {
    const int64_t blocks = (values / 4 + kThreads - 1) / kThreads;
    if (blocks > INT32_MAX) return FMD_ERR_UNSUPPORTED;
    add_kernel<T><<<dim3(unsigned(blocks), out1 != nullptr ? 2 : 1), kThreads, 0, s>>>(
        part0, part1, static_cast<T*>(out0), static_cast<T*>(out1), values, splits);
    return check_launch();
}

template <typename T, int N>
__device__ __forceinline__ void load_floats(const T* p, float (&v)[N]) {
    T x[N];
    *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = attn_float(x[j]);
}

// delta[row] = sum_d g out - (gradient of lse): 8 lanes per packed row, 16-byte loads.
template <typename T>
__global__ void __launch_bounds__(kThreads) delta_kernel(const Attn a, const float* glse, float* delta) {
    constexpr int kV = 16 / sizeof(T);
    const int64_t i = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / 8;
    const int lane = threadIdx.x & 7;
    float sum = 0.0f;
    if (i < a.rows * a.hq) {
        const int64_t row = i / a.hq;
        const int head = int(i - row * a.hq);
        const T* g = static_cast<const T*>(a.g) + row * a.g_row + head * a.g_head;
        const T* o = static_cast<const T*>(a.out) + i * a.dim;
        for (int c = lane * kV; c < a.dim; c += 8 * kV) {
            float x[kV], y[kV];
            load_floats(g + c, x);
            load_floats(o + c, y);
#pragma unroll
            for (int j = 0; j < kV; ++j) sum = fmaf(x[j], y[j], sum);
        }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (i < a.rows * a.hq && lane == 0) delta[i] = glse != nullptr ? sum - glse[i] : sum;
    for (int64_t b = int64_t(blockIdx.x) * kThreads + threadIdx.x; b < a.batch; b += int64_t(gridDim.x) * kThreads)
        check_sequence(a, b);
}

// Packed rows of 16 bits that see at most kFewKeys keys take delta = sum_j p_j dp_j - (gradient of lse) instead. The stored
// out carries two roundings (of p for p v, of the sum), and ds = p (dp - delta) takes delta's error along the mean key: for n
// keys about n^-1/2 of the rounding of the result, which for few keys is more than all else (dq and dk of causal sequences of
// one to three rows had 2.4 times the error of rounding them alone, now 1.0; from 17 keys on it is 1.2 times at most). Takes
// 3 us for 64 sequences of 135 rows, 8 us for 16 causal ones of up to 2,000.
// blockIdx.x: the sequence. A warp per packed row, two lanes per key, so that all its loads are in flight together.
constexpr int kFewKeys = 16;

__global__ void __launch_bounds__(kThreads) few_delta_kernel(const Attn a, const float* glse, float* delta) {
    const Span s = load_span(a, blockIdx.x);
    // the first token that sees a key, and how many see kFewKeys at most
    const int64_t first = a.causal ? max(int64_t(0), s.rows - s.keys) : 0;
    const int64_t tokens = a.causal ? min(s.rows, s.rows - s.keys + kFewKeys) - first : s.keys <= kFewKeys ? s.rows : 0;
    const int lane = threadIdx.x & 31, key = lane / 2, half = lane % 2;
    const __nv_bfloat16 *qs = static_cast<const __nv_bfloat16*>(a.q), *gs = static_cast<const __nv_bfloat16*>(a.g);
    const __nv_bfloat16 *ks = static_cast<const __nv_bfloat16*>(a.k), *vs = static_cast<const __nv_bfloat16*>(a.v);
    for (int64_t r = int64_t(blockIdx.y) * (kThreads / 32) + threadIdx.x / 32; r < tokens * a.hq;
         r += int64_t(gridDim.y) * (kThreads / 32)) {
        const int64_t token = first + r / a.hq, row = s.row0 + token;
        const int head = int(r % a.hq), n = int(seen(s, a.causal, token));
        const float lse = a.lse[row * a.hq + head];
        float score = 0.0f, dp = 0.0f;
        if (key < n) {
            const __nv_bfloat16 *q = qs + row * a.q_row + head * a.q_head, *g = gs + row * a.g_row + head * a.g_head;
            const __nv_bfloat16* k = ks + (s.key0 + key) * a.k_row + head / a.group * a.k_head;
            const __nv_bfloat16* v = vs + (s.key0 + key) * a.v_row + head / a.group * a.v_head;
#pragma unroll 4
            for (int c = half * 8; c < a.dim; c += 16) {
                float x[8], y[8];
                load_floats(q + c, x);
                load_floats(k + c, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) score = fmaf(x[e], y[e], score);
                load_floats(g + c, x);
                load_floats(v + c, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) dp = fmaf(x[e], y[e], dp);
            }
        }
        score += __shfl_xor_sync(0xffffffffu, score, 1);
        dp += __shfl_xor_sync(0xffffffffu, dp, 1);
        float sum = key < n && lse != -INFINITY ? exp2f((score * a.scale - lse) * kLog2e) * dp : 0.0f;
#pragma unroll
        for (int o = 2; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) delta[row * a.hq + head] = glse != nullptr ? sum - glse[row * a.hq + head] : sum;
    }
}

fmd_status check(const fmd_attention& q, Attn& a) {
    if ((q.type != FMD_F32 && q.type != FMD_BF16) || q.rows < 0 || q.keys < 0 || q.batch < 0 || q.heads < 1 ||
        q.key_heads < 1 || q.heads % q.key_heads || q.heads / q.key_heads > 64 || q.dim < 8 || q.dim > 128 ||
        q.dim % 8 || !(q.scale >= 0.0f && q.scale <= 1.0e38f) || (q.batch > 0 && (q.offsets == nullptr || q.key_offsets == nullptr)) ||
        (q.batch == 0 && (q.rows > 0 || q.keys > 0)) || (q.rows > 0 && q.q == nullptr) ||
        (q.keys > 0 && (q.k == nullptr || q.v == nullptr)))
        return FMD_ERR_INVALID_ARGUMENT;
    const int size = q.type == FMD_F32 ? 4 : 2;
    if ((q.rows > 0 && !vector_rows(q.q, q.q_row, q.q_head, size)) ||
        (q.keys > 0 && (!vector_rows(q.k, q.k_row, q.k_head, size) || !vector_rows(q.v, q.v_row, q.v_head, size))) ||
        q.rows > (1 << 29) || q.keys > (1 << 29) || q.batch > (1 << 24) ||
        // a block per tile (of 64 rows at least) and key head
        tile_bound(q.rows, q.batch, 64 / (q.heads / q.key_heads)) > INT32_MAX / q.key_heads ||
        tile_bound(q.keys, q.batch, 64) > INT32_MAX / q.key_heads)
        return FMD_ERR_UNSUPPORTED;
    a = Attn{};
    a.q = q.q;
    a.k = q.k;
    a.v = q.v;
    a.offsets = q.offsets;
    a.key_offsets = q.key_offsets;
    a.key_counts = q.key_counts;
    a.rows = q.rows;
    a.keys = q.keys;
    a.q_row = q.q_row;
    a.q_head = q.q_head;
    a.k_row = q.k_row;
    a.k_head = q.k_head;
    a.v_row = q.v_row;
    a.v_head = q.v_head;
    // The smallest normal number stands for 0: a masked score is -inf before it is scaled, and -inf * 0 is not a number.
    a.scale = fmaxf(q.scale, FLT_MIN);
    a.batch = q.batch;
    a.hq = q.heads;
    a.hk = q.key_heads;
    a.group = q.heads / q.key_heads;
    a.dim = q.dim;
    a.causal = q.causal != 0;
    return FMD_OK;
}

// float32 heads of up to this many values go through planes on the tensor cores, wider ones stay on the FP32 cores, whose
// kernels are also right for every size. Forward, us by planes and on the FP32 cores: 64 slots of 2,000 keys, 2 key heads of
// 64, one new row of 8 heads each 104 and 393, 32 rows 109 and 785, 128 rows 232 and 2,573. All rows of k and v are split,
// filled or not, since the host knows no count: with a tenth filled 73 and 44 for one row, 113 and 245 for 128.
constexpr int kPlanesDim = 64;

// How the forward pass runs, from the sizes alone: its splits of the keys, and its workspace: planes, then the splits.
struct Plan {
    int splits;
    size_t planes, bytes;
};

Plan plan(const Attn& a, int type) {
    Plan p{1, 0, 0};
    if (a.rows == 0) return p;
    const bool planes = type == FMD_F32 && a.dim <= kPlanesDim;
    // one block an SM by its shared memory, or two
    if (type == FMD_BF16) p.splits = attention_splits_mma(a);
    else p.splits = key_splits(a, (planes ? 128 : 64) / a.group, kNumSMs, planes ? 128 : 64);
    if (planes) p.planes = attention_planes_bytes(a, false);
    p.bytes = p.planes + (p.splits > 1 ? size_t(p.splits) * a.rows * a.hq * (a.dim + 1) * sizeof(float) : 0);
    return p;
}

size_t delta_bytes(const Attn& a) { return (size_t(a.rows) * a.hq * sizeof(float) + 15) & ~size_t(15); }

// How the backward pass runs, and its workspace: delta, planes, then the splits' parts.
struct BackwardPlan {
    BackwardSplits splits;
    size_t delta, planes, dq, dkv, bytes;
};

BackwardPlan backward_plan(const Attn& a, int type, bool dq, bool dkv) {
    BackwardPlan p{{1, 1}, delta_bytes(a), 0, 0, 0, 0};
    const bool planes = type == FMD_F32 && a.dim <= kPlanesDim;
    if (planes) p.planes = attention_planes_bytes(a, true);
    const int own = type == FMD_BF16 || planes ? 128 : 64, stream = type == FMD_BF16 ? 128 : 64;  // rows of the tiles
    if (dq) p.splits.queries = key_splits(a, own / a.group, kNumSMs, stream);
    if (dkv) p.splits.keys = row_splits(a, stream / a.group, kNumSMs, own);
    if (p.splits.queries > 1) p.dq = size_t(p.splits.queries) * a.rows * a.hq * a.dim * sizeof(float);
    if (p.splits.keys > 1) p.dkv = size_t(p.splits.keys) * a.keys * a.hk * a.dim * sizeof(float);
    p.bytes = p.delta + p.planes + p.dq + 2 * p.dkv;
    return p;
}

}  // namespace
}  // namespace fmd

using namespace fmd;

extern "C" {

fmd_status fmd_packed_attention_workspace_bytes(const fmd_attention* problem, int32_t backward, size_t* bytes) {
    Attn a;
    if (problem == nullptr || bytes == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const fmd_status st = check(*problem, a);
    if (st == FMD_OK) *bytes = backward ? backward_plan(a, problem->type, true, true).bytes : plan(a, problem->type).bytes;
    return st;
}

fmd_status fmd_packed_attention(const fmd_attention* problem, void* out, float* lse, void* workspace,
                                size_t workspace_bytes, int32_t* flags, void* stream) {
    Attn a;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check(*problem, a);
    if (st != FMD_OK) return st;
    if (a.rows == 0) return FMD_OK;
    if (out == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    if (!aligned16(out)) return FMD_ERR_UNSUPPORTED;
    const Plan p = plan(a, problem->type);
    if (workspace_bytes < p.bytes || (p.bytes > 0 && workspace == nullptr)) return FMD_ERR_WORKSPACE;
    if (!aligned16(workspace)) return FMD_ERR_UNSUPPORTED;
    a.out = out;
    a.lse = lse;
    a.flags = flags;
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.planes);
    a.part_lse = a.part + int64_t(p.splits) * a.rows * a.hq * a.dim;
    const cudaStream_t s = as_stream(stream);
    if (problem->type == FMD_BF16) st = attention_forward_mma(a, p.splits, s);
    else if (a.dim <= kPlanesDim) st = attention_forward_planes(a, p.splits, workspace, s);
    else st = attention_forward_simt(a, p.splits, s);
    if (st != FMD_OK || p.splits == 1) return st;
    return problem->type == FMD_BF16 ? join<__nv_bfloat16>(a, p.splits, s) : join<float>(a, p.splits, s);
}

fmd_status fmd_packed_attention_bwd(const fmd_attention* problem, const void* out, const float* lse, const void* g,
                                    int64_t g_row, int64_t g_head, const float* glse, void* dq, void* dk, void* dv,
                                    void* workspace, size_t workspace_bytes, int32_t* flags, void* stream) {
    Attn a;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check(*problem, a);
    if (st != FMD_OK) return st;
    if ((dk == nullptr) != (dv == nullptr)) return FMD_ERR_INVALID_ARGUMENT;
    if (a.rows > 0 && (out == nullptr || lse == nullptr || g == nullptr)) return FMD_ERR_INVALID_ARGUMENT;
    const BackwardPlan p = backward_plan(a, problem->type, dq != nullptr, dk != nullptr);
    if (workspace_bytes < p.bytes || (p.bytes > 0 && workspace == nullptr)) return FMD_ERR_WORKSPACE;
    if ((a.rows > 0 && (!vector_rows(g, g_row, g_head, problem->type == FMD_F32 ? 4 : 2) || !aligned16(out))) ||
        !aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !aligned16(workspace))
        return FMD_ERR_UNSUPPORTED;
    float* delta = static_cast<float*>(workspace);
    a.out = const_cast<void*>(out);
    a.lse = const_cast<float*>(lse);
    a.g = g;
    a.g_row = g_row;
    a.g_head = g_head;
    a.delta = delta;
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.flags = flags;
    a.lse_gradient = glse != nullptr;
    const cudaStream_t s = as_stream(stream);
    if (a.rows > 0) {
        const int64_t blocks = (a.rows * a.hq * 8 + kThreads - 1) / kThreads;
        if (blocks > INT32_MAX) return FMD_ERR_UNSUPPORTED;
        if (problem->type == FMD_F32) delta_kernel<float><<<unsigned(blocks), kThreads, 0, s>>>(a, glse, delta);
        else delta_kernel<__nv_bfloat16><<<unsigned(blocks), kThreads, 0, s>>>(a, glse, delta);
        if ((st = check_launch()) != FMD_OK) return st;
        if (problem->type == FMD_BF16) {
            // by the mean sequence: eight packed rows a block, or eight blocks an SM that walk on
            const int64_t mean = a.rows / a.batch + 1, most = 8 * kNumSMs / a.batch + 1;
            const int64_t each = ((a.causal && mean > kFewKeys ? kFewKeys : mean) * a.hq + 7) / 8;
            few_delta_kernel<<<dim3(unsigned(a.batch), unsigned(each < most ? each : most)), kThreads, 0, s>>>(a, glse, delta);
            if ((st = check_launch()) != FMD_OK) return st;
        }
    }
    char* at = static_cast<char*>(workspace) + p.delta;
    a.part = reinterpret_cast<float*>(at + p.planes);
    a.part_dk = reinterpret_cast<float*>(at + p.planes + p.dq);
    a.part_dv = reinterpret_cast<float*>(at + p.planes + p.dq + p.dkv);
    if (problem->type == FMD_BF16) st = attention_backward_mma(a, p.splits, s);
    else if (a.dim <= kPlanesDim) st = attention_backward_planes(a, p.splits, at, s);
    else st = attention_backward_simt(a, p.splits, s);
    const int64_t q_values = a.rows * a.hq * a.dim, k_values = a.keys * a.hk * a.dim;
    const bool bf16 = problem->type == FMD_BF16;
    if (st == FMD_OK && p.splits.queries > 1 && q_values > 0)
        st = bf16 ? add<__nv_bfloat16>(a.part, nullptr, dq, nullptr, q_values, p.splits.queries, s)
                  : add<float>(a.part, nullptr, dq, nullptr, q_values, p.splits.queries, s);
    if (st == FMD_OK && p.splits.keys > 1 && k_values > 0)
        st = bf16 ? add<__nv_bfloat16>(a.part_dk, a.part_dv, dk, dv, k_values, p.splits.keys, s)
                  : add<float>(a.part_dk, a.part_dv, dk, dv, k_values, p.splits.keys, s);
    return st;
}

}  // extern "C"
