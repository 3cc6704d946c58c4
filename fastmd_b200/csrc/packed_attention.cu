// C entry points of packed attention: argument checks, the choice of kernels, and the row sums that the backward
// pass starts from.

#include "packed_attention.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 256;

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
            T x[kV], y[kV];
            *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(g + c);
            *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(o + c);
#pragma unroll
            for (int j = 0; j < kV; ++j) sum = fmaf(attn_float(x[j]), attn_float(y[j]), sum);
        }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (i < a.rows * a.hq && lane == 0) delta[i] = glse != nullptr ? sum - glse[i] : sum;
}

bool rows16(const void* p, int64_t row, int64_t head, int size) {
    return aligned16(p) && (row * size) % 16 == 0 && (head * size) % 16 == 0;
}

fmd_status check(const fmd_attention& q, Attn& a) {
    if ((q.type != FMD_F32 && q.type != FMD_BF16) || q.rows < 0 || q.keys < 0 || q.batch < 0 || q.heads < 1 ||
        q.key_heads < 1 || q.heads % q.key_heads || q.heads / q.key_heads > 64 || q.dim < 8 || q.dim > 128 ||
        q.dim % 8 || (q.batch > 0 && (q.offsets == nullptr || q.key_offsets == nullptr)) ||
        (q.batch == 0 && (q.rows > 0 || q.keys > 0)) || (q.rows > 0 && q.q == nullptr) ||
        (q.keys > 0 && (q.k == nullptr || q.v == nullptr)))
        return FMD_ERR_INVALID_ARGUMENT;
    const int size = q.type == FMD_F32 ? 4 : 2;
    if ((q.rows > 0 && !rows16(q.q, q.q_row, q.q_head, size)) ||
        (q.keys > 0 && (!rows16(q.k, q.k_row, q.k_head, size) || !rows16(q.v, q.v_row, q.v_head, size))) ||
        q.key_heads > 65535 || q.rows > INT32_MAX || q.keys > INT32_MAX || q.batch > (1 << 24))
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
    a.scale = q.scale;
    a.batch = q.batch;
    a.hq = q.heads;
    a.hk = q.key_heads;
    a.group = q.heads / q.key_heads;
    a.dim = q.dim;
    a.causal = q.causal != 0;
    return FMD_OK;
}

size_t workspace_bytes(const Attn& a, int type) {
    const int splits = type == FMD_BF16 ? attention_splits(a) : 1;
    return splits > 1 ? size_t(splits) * a.rows * a.hq * (a.dim + 1) * sizeof(float) : 0;
}

}  // namespace
}  // namespace fmd

using namespace fmd;

extern "C" {

fmd_status fmd_packed_attention_workspace_bytes(const fmd_attention* problem, size_t* bytes) {
    Attn a;
    if (problem == nullptr || bytes == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const fmd_status st = check(*problem, a);
    if (st == FMD_OK) *bytes = workspace_bytes(a, problem->type);
    return st;
}

fmd_status fmd_packed_attention(const fmd_attention* problem, void* out, float* lse, void* workspace,
                                size_t workspace_size, int32_t* flags, void* stream) {
    Attn a;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check(*problem, a);
    if (st != FMD_OK) return st;
    if (a.rows == 0) return FMD_OK;
    if (out == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    if (!aligned16(out)) return FMD_ERR_UNSUPPORTED;
    if (workspace_size < workspace_bytes(a, problem->type)) return FMD_ERR_WORKSPACE;
    if (!aligned16(workspace)) return FMD_ERR_UNSUPPORTED;
    a.out = out;
    a.lse = lse;
    a.flags = flags;
    if (problem->type == FMD_BF16) {
        a.part = static_cast<float*>(workspace);
        a.part_lse = a.part + int64_t(attention_splits(a)) * a.rows * a.hq * a.dim;
    }
    if (problem->type == FMD_BF16) return attention_forward_mma(a, as_stream(stream));
    return attention_forward_simt(a, problem->type, as_stream(stream));
}

fmd_status fmd_packed_attention_bwd(const fmd_attention* problem, const void* out, const float* lse, const void* g,
                                    int64_t g_row, int64_t g_head, const float* glse, float* delta, void* dq, void* dk,
                                    void* dv, int32_t* flags, void* stream) {
    Attn a;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check(*problem, a);
    if (st != FMD_OK) return st;
    if ((dk == nullptr) != (dv == nullptr)) return FMD_ERR_INVALID_ARGUMENT;
    if (a.rows > 0 && (out == nullptr || lse == nullptr || g == nullptr || delta == nullptr))
        return FMD_ERR_INVALID_ARGUMENT;
    if ((a.rows > 0 && (!rows16(g, g_row, g_head, problem->type == FMD_F32 ? 4 : 2) || !aligned16(out))) ||
        !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
        return FMD_ERR_UNSUPPORTED;
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
    const cudaStream_t s = as_stream(stream);
    if (a.rows > 0) {
        const int64_t blocks = (a.rows * a.hq * 8 + kThreads - 1) / kThreads;
        if (blocks > INT32_MAX) return FMD_ERR_UNSUPPORTED;
        if (problem->type == FMD_F32) delta_kernel<float><<<unsigned(blocks), kThreads, 0, s>>>(a, glse, delta);
        else delta_kernel<__nv_bfloat16><<<unsigned(blocks), kThreads, 0, s>>>(a, glse, delta);
        if ((st = check_launch()) != FMD_OK) return st;
    }
    return problem->type == FMD_BF16 ? attention_backward_mma(a, s) : attention_backward_simt(a, problem->type, s);
}

}  // extern "C"
