// C entry points of decay attention: argument checks, the cut into segments, what is carried from segment to segment, and
// the recurrence for single rows.

#include "decay_attention.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 256;

// From what each segment adds to what it starts from, in place, and the matrix behind the last row. A block per sequence,
// head and 1,024 of the matrix's values (four a thread), which it takes through the segments one after the other; the next
// ones are loaded ahead.
__global__ void __launch_bounds__(kThreads) carry_kernel(const Decay d) {
    constexpr int kAhead = 8;
    const int b = blockIdx.x / d.heads, head = blockIdx.x % d.heads;
    const int size = d.dim * d.dim, at = (blockIdx.y * kThreads + threadIdx.x) * 4;
    const float l2 = log2_decay(d, head);
    if (head == 0 && blockIdx.y == 0 && threadIdx.x == 0) check_offsets(d, b);
    if (at >= size) return;
    const int64_t r0 = d.offsets[b], lo = min(max(r0, int64_t(0)), d.rows), hi = min(max(d.offsets[b + 1], lo), d.rows);
    const int64_t n = hi - lo, most = decay_segments(d);
    // bad offsets do not lead out of the array
    const int64_t first = min(max(r0 / d.length + b, int64_t(0)), most);
    const int64_t count = min((n + d.length - 1) / d.length, most - first);
    const int64_t mine = (int64_t(b) * d.heads + head) * size;
    const int row = at / d.dim, col = at - row * d.dim;
    float4 state = f4_zero();
    if (d.start != nullptr) {
        if (d.transposed) {
            const float* p = d.start + mine + int64_t(col) * d.dim + row;
            state = make_float4(p[0], p[d.dim], p[2 * d.dim], p[3 * d.dim]);
        } else {
            state = ldg4(d.start + mine + at);
        }
    }
    const float whole = exp2f(float(d.length) * l2);
    float* p = d.states + (first * d.heads + head) * size + at;
    const int64_t step = int64_t(d.heads) * size;
    for (int64_t i = 0; i < count; i += kAhead) {
        float4 added[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e)
            if (i + e < count) added[e] = *reinterpret_cast<const float4*>(p + (i + e) * step);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            if (i + e >= count) break;
            const int64_t rows = min(d.length, n - (i + e) * d.length);
            const float keep = rows == d.length ? whole : exp2f(float(rows) * l2);
            st4(p + (i + e) * step, state);
            state = make_float4(fmaf(keep, state.x, added[e].x), fmaf(keep, state.y, added[e].y),
                                fmaf(keep, state.z, added[e].z), fmaf(keep, state.w, added[e].w));
        }
    }
    if (d.after == nullptr) return;
    if (d.transposed) {
        float* q = d.after + mine + int64_t(col) * d.dim + row;
        q[0] = state.x, q[d.dim] = state.y, q[2 * d.dim] = state.z, q[3 * d.dim] = state.w;
    } else {
        st4(d.after + mine + at, state);
    }
}

__device__ __forceinline__ float read(const float* p) { return *p; }
__device__ __forceinline__ float read(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void write(float* p, float v) { *p = v; }
__device__ __forceinline__ void write(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One row of every sequence: S = l S + k v^T in place, out = scale q S. A block per row and head; dim / 4 threads side by
// side hold four columns each, the others further rows of the matrix. Bound by the state, which is read and written once.
template <typename T>
__global__ void __launch_bounds__(kThreads) step_kernel(const Decay d, float* state) {
    __shared__ float q[128], k[128], v[128];
    __shared__ float4 sums[kThreads];
    const int64_t b = blockIdx.x / unsigned(d.heads);
    const int head = int(blockIdx.x - b * d.heads), dim = d.dim, quads = dim / 4;
    for (int i = threadIdx.x; i < dim; i += kThreads) {
        q[i] = read(static_cast<const T*>(d.a) + b * d.a_row + head * d.a_head + i);
        k[i] = read(static_cast<const T*>(d.b) + b * d.b_row + head * d.b_head + i);
        v[i] = read(static_cast<const T*>(d.c) + b * d.c_row + head * d.c_head + i);
    }
    const float keep = exp2f(log2_decay(d, head));
    const int quad = threadIdx.x % quads, first = threadIdx.x / quads, rows = kThreads / quads;
    float4* s = reinterpret_cast<float4*>(state + (b * d.heads + head) * int64_t(dim) * dim) + quad;
    __syncthreads();
    float4 sum = f4_zero();
    const float4 mine = *reinterpret_cast<const float4*>(v + 4 * quad);
    if (first < rows) {
#pragma unroll 8
        for (int r = first; r < dim; r += rows) {
            float4 x = s[r * quads];
            const float w = k[r], u = q[r];
            x = make_float4(fmaf(keep, x.x, w * mine.x), fmaf(keep, x.y, w * mine.y), fmaf(keep, x.z, w * mine.z),
                            fmaf(keep, x.w, w * mine.w));
            s[r * quads] = x;
            sum = make_float4(fmaf(u, x.x, sum.x), fmaf(u, x.y, sum.y), fmaf(u, x.z, sum.z), fmaf(u, x.w, sum.w));
        }
    }
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x >= dim) return;
    const float* all = reinterpret_cast<const float*>(sums);
    float out = 0.0f;
    for (int r = 0; r < rows; ++r) out += all[r * dim + threadIdx.x];
    write(static_cast<T*>(d.out) + (b * d.heads + head) * dim + threadIdx.x, d.far * out);
}

fmd_status check(const fmd_decay& p, Decay& d, bool rows_aligned) {
    if ((p.type != FMD_F32 && p.type != FMD_BF16) || p.rows < 0 || p.batch < 0 || p.heads < 1 || p.dim < 8 || p.dim > 128 ||
        p.dim % 8 || !(p.scale >= 0.0f && p.scale <= 1.0e38f) || p.log_decay == nullptr ||
        (p.rows > 0 && (p.q == nullptr || p.k == nullptr || p.v == nullptr)))
        return FMD_ERR_INVALID_ARGUMENT;
    const int size = p.type == FMD_F32 ? 4 : 2;
    if (p.rows > (1 << 29) || p.batch > (1 << 24) || p.heads > 1024 ||
        (rows_aligned && p.rows > 0 &&
         (!vector_rows(p.q, p.q_row, p.q_head, size) || !vector_rows(p.k, p.k_row, p.k_head, size) ||
          !vector_rows(p.v, p.v_row, p.v_head, size))))
        return FMD_ERR_UNSUPPORTED;
    d = Decay{};
    d.log_decay = p.log_decay;
    d.offsets = p.offsets;
    d.rows = p.rows;
    d.batch = p.batch;
    d.heads = p.heads;
    d.dim = p.dim;
    return FMD_OK;
}

// The sequences' form of the checks.
fmd_status check_rows(const fmd_decay& p, Decay& d) {
    const fmd_status st = check(p, d, true);
    if (st != FMD_OK) return st;
    if ((p.batch > 0 && p.offsets == nullptr) || (p.batch == 0 && p.rows > 0)) return FMD_ERR_INVALID_ARGUMENT;
    return FMD_OK;
}

// Rows of a segment: whole sequences where these are blocks enough for the GPU or short; else so many that there are
// about two blocks an SM.
int64_t segment_length(const Decay& d) {
    if (d.batch == 0) return kWhole;
    const int64_t blocks = int64_t(d.batch) * d.heads, mean = d.rows / d.batch;
    if (blocks >= 2 * kNumSMs || mean <= 512) return kWhole;
    const int64_t want = (2 * kNumSMs + d.heads - 1) / d.heads;  // segments of all sequences together
    int64_t length = (d.rows / want + 127) / 128 * 128;
    return length < 256 ? 256 : length;
}

size_t matrices(const Decay& d, int64_t n) { return size_t(n) * d.heads * d.dim * d.dim * sizeof(float); }

// One pass of the recurrence: with segments, or where the last matrix is wanted, what the segments add comes first.
fmd_status mix(Decay d, bool bf16, void* workspace, cudaStream_t s) {
    d.length = segment_length(d);
    const bool carried = d.length < kWhole || d.after != nullptr;
    const int64_t segments = decay_segments(d);
    if (segments * d.heads > INT32_MAX) return FMD_ERR_UNSUPPORTED;
    fmd_status st = FMD_OK;
    if (carried && d.batch > 0) {
        d.states = static_cast<float*>(workspace);
        if (d.rows > 0) st = bf16 ? decay_states_mma(d, s) : decay_states_simt(d, s);
        if (st != FMD_OK) return st;
        const int64_t blocks = int64_t(d.batch) * d.heads;
        if (blocks > INT32_MAX) return FMD_ERR_UNSUPPORTED;
        carry_kernel<<<dim3(unsigned(blocks), unsigned((d.dim * d.dim + 4 * kThreads - 1) / (4 * kThreads))), kThreads, 0,
                       s>>>(d);
        if ((st = check_launch()) != FMD_OK) return st;
    }
    if (d.rows == 0 || d.out == nullptr) return FMD_OK;
    return bf16 ? decay_rows_mma(d, carried, s) : decay_rows_simt(d, carried, s);
}

size_t mix_bytes(Decay d, bool after) {
    d.length = segment_length(d);
    return d.length < kWhole || after ? matrices(d, decay_segments(d)) : 0;
}

}  // namespace

}  // namespace fmd

using namespace fmd;

extern "C" {

fmd_status fmd_decay_attention_workspace_bytes(const fmd_decay* problem, int32_t after, size_t* bytes) {
    Decay d;
    if (problem == nullptr || bytes == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const fmd_status st = check_rows(*problem, d);
    if (st == FMD_OK) *bytes = mix_bytes(d, after != 0);
    return st;
}

fmd_status fmd_decay_attention(const fmd_decay* problem, const float* state, void* out, float* after, void* workspace,
                               size_t workspace_bytes, int32_t* flags, void* stream) {
    Decay d;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const fmd_status st = check_rows(*problem, d);
    if (st != FMD_OK) return st;
    const fmd_decay& p = *problem;
    if (p.rows > 0 && out == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const size_t need = mix_bytes(d, after != nullptr);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return FMD_ERR_WORKSPACE;
    if (!aligned16(out) || !aligned16(state) || !aligned16(after) || !aligned16(workspace)) return FMD_ERR_UNSUPPORTED;
    d.a = p.q, d.b = p.k, d.c = p.v, d.out = out;
    d.a_row = p.q_row, d.a_head = p.q_head, d.b_row = p.k_row, d.b_head = p.k_head, d.c_row = p.v_row, d.c_head = p.v_head;
    d.start = state;
    d.after = after;
    d.flags = flags;
    d.near = d.far = p.scale;
    d.add = 1.0f;
    return mix(d, p.type == FMD_BF16, workspace, as_stream(stream));
}

fmd_status fmd_decay_attention_bwd(const fmd_decay* problem, const float* state, const void* g, int64_t g_row,
                                   int64_t g_head, const float* gafter, void* dq, void* dk, void* dv, float* dstate,
                                   void* workspace, size_t workspace_bytes, int32_t* flags, void* stream) {
    Decay d;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check_rows(*problem, d);
    if (st != FMD_OK) return st;
    const fmd_decay& p = *problem;
    const bool bf16 = p.type == FMD_BF16;
    if (p.rows > 0 && g == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const size_t need = mix_bytes(d, dstate != nullptr);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return FMD_ERR_WORKSPACE;
    if (!aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !aligned16(state) || !aligned16(gafter) ||
        !aligned16(dstate) || !aligned16(workspace) || (p.rows > 0 && !vector_rows(g, g_row, g_head, bf16 ? 2 : 4)))
        return FMD_ERR_UNSUPPORTED;
    const cudaStream_t s = as_stream(stream);
    d.flags = flags;
    d.near = p.scale;
    if (dq != nullptr) {
        Decay m = d;
        m.a = g, m.b = p.v, m.c = p.k, m.out = dq;
        m.a_row = g_row, m.a_head = g_head, m.b_row = p.v_row, m.b_head = p.v_head, m.c_row = p.k_row, m.c_head = p.k_head;
        m.start = state;
        m.transposed = 1;
        m.add = 1.0f;
        m.far = p.scale;
        if ((st = mix(m, bf16, workspace, s)) != FMD_OK) return st;
    }
    d.later = 1;
    d.add = p.scale;
    d.far = 1.0f;
    d.start = gafter;
    if (dk != nullptr) {
        Decay m = d;
        m.a = p.v, m.b = g, m.c = p.q, m.out = dk;
        m.a_row = p.v_row, m.a_head = p.v_head, m.b_row = g_row, m.b_head = g_head, m.c_row = p.q_row, m.c_head = p.q_head;
        m.transposed = 1;
        if ((st = mix(m, bf16, workspace, s)) != FMD_OK) return st;
    }
    if (dv != nullptr || dstate != nullptr) {
        Decay m = d;
        m.a = p.k, m.b = p.q, m.c = g, m.out = dv;
        m.a_row = p.k_row, m.a_head = p.k_head, m.b_row = p.q_row, m.b_head = p.q_head, m.c_row = g_row, m.c_head = g_head;
        m.after = dstate;
        if ((st = mix(m, bf16, workspace, s)) != FMD_OK) return st;
    }
    return FMD_OK;
}

fmd_status fmd_decay_attention_step(const fmd_decay* problem, float* state, void* out, void* stream) {
    Decay d;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const fmd_status st = check(*problem, d, false);
    if (st != FMD_OK || problem->rows == 0) return st;
    const fmd_decay& p = *problem;
    if (out == nullptr || state == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    if (!aligned16(state) || p.rows * p.heads > INT32_MAX) return FMD_ERR_UNSUPPORTED;
    d.a = p.q, d.b = p.k, d.c = p.v, d.out = out;
    d.a_row = p.q_row, d.a_head = p.q_head, d.b_row = p.k_row, d.b_head = p.k_head, d.c_row = p.v_row, d.c_head = p.v_head;
    d.far = p.scale;
    const unsigned blocks = unsigned(p.rows * p.heads);
    if (p.type == FMD_BF16) step_kernel<__nv_bfloat16><<<blocks, kThreads, 0, as_stream(stream)>>>(d, state);
    else step_kernel<float><<<blocks, kThreads, 0, as_stream(stream)>>>(d, state);
    return check_launch();
}

}  // extern "C"
