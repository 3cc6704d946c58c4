// C entry points of decay attention: argument checks, the cut into segments, what is carried from segment to segment, and
// the recurrence row by row, for single rows and for sequences of a few.

#include "decay_attention.cuh"
#include "tensor_cores.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 256;

// From what each segment adds to what it starts from, in place, and the matrix behind the last row. A block per sequence,
// head and 1,024 of the matrix's values (four a thread), which it takes through the segments one after the other, sixteen
// loaded at a time: bound by the latency of a few of these loads (8 us for 9 segments of 16 heads of 128).
__global__ void __launch_bounds__(kThreads) carry_kernel(const __grid_constant__ Decays all) {
    constexpr int kAhead = 16;
    dependents_may_start();
    wait_for_the_kernel_ahead();
    const Decay& d = all.d[blockIdx.z];
    const int b = blockIdx.x / d.heads, head = blockIdx.x % d.heads;
    const int size = d.dim * d.dim, at = (blockIdx.y * kThreads + threadIdx.x) * 4;
    const float l2 = log2_decay(d, head);
    if (head == 0 && blockIdx.y == 0 && threadIdx.x == 0) check_offsets(d, b);
    if (at >= size) return;
    const int64_t r0 = d.offsets[b], lo = min(max(r0, int64_t(0)), d.rows), hi = min(max(d.offsets[b + 1], lo), d.rows);
    const int64_t n = hi - lo, most = decay_segments(d);
    // bad offsets do not lead out of the array
    const int64_t first = min(max(r0 / d.length + b, int64_t(0)), most);
    const int count = int(min((n + d.length - 1) / d.length, most - first));
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
    const float whole = exp2f(float(d.length) * l2), last = exp2f(float(n - (count - 1) * d.length) * l2);
    float* p = d.states + (first * d.heads + head) * size + at;
    const int64_t step = int64_t(d.heads) * size;
    for (int i = 0; i < count; i += kAhead) {
        float4 added[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e)
            if (i + e < count) added[e] = *reinterpret_cast<const float4*>(p + (i + e) * step);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            if (i + e >= count) break;
            const float keep = i + e + 1 < count ? whole : last;
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

// float32 [rows, heads, dim] as three planes [3][rows][heads][dim] of bfloat16, up to four arrays (blockIdx.y). Bound by
// memory: three arrays, 118 MB in and 177 MB out, take 43 us with the last ones left in L2.
struct SplitArgs {
    const float* x[4];
    __nv_bfloat16* to[4];
    int64_t row[4], head[4];
    int64_t rows;
    int32_t heads, dim;
};

__global__ void __launch_bounds__(kThreads) split_kernel(const SplitArgs a) {
    dependents_may_start();
    const int t = blockIdx.y, per = a.dim / 8;
    const int64_t heads = a.rows * a.heads, all = heads * per;
    for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < all; i += int64_t(gridDim.x) * kThreads) {
        const int64_t r = i / per, row = r / a.heads;
        const float* x = a.x[t] + row * a.row[t] + (r - row * a.heads) * a.head[t] + (i - r * per) * 8;
        const float4 p = ldg4(x), q = ldg4(x + 4);
        float v[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
        uint4* to = reinterpret_cast<uint4*>(a.to[t]) + i;
        to[0] = first_plane8(v);
        to[all] = next_plane8(v);
        to[2 * all] = next_plane8(v);
    }
}

__device__ __forceinline__ float read(const float* p) { return *p; }
__device__ __forceinline__ float read(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void write(float* p, float v) { *p = v; }
__device__ __forceinline__ void write(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One row of every sequence: S = l S + k v^T in place, out = scale q S. A block per row and head; dim / 4 threads side by
// side hold four columns each, the others further rows of the matrix. Bound by the state, which is read and written once:
// 1.08 GB of 512 rows, 16 heads of 128, in 186 us, 5.8 TB/s.
template <typename T>
__global__ void __launch_bounds__(kThreads) step_kernel(const Decay d, float* state) {
    __shared__ alignas(16) float q[128], k[128], v[128];
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

__device__ __forceinline__ float4 read4(const float* p) { return ldg4(p); }
__device__ __forceinline__ float4 read4(const __nv_bfloat16* p) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    const float2 x = unpack_bf16(w.x), y = unpack_bf16(w.y);
    return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ void write4(float* p, float4 v) { st4(p, v); }
__device__ __forceinline__ void write4(__nv_bfloat16* p, float4 v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// Sequences of a few rows, row by row: the step above, with the matrix in registers from the first row to the last and in either
// direction. A block per sequence, head, pass and 32 columns of the matrix (which do not see each other); a thread holds four
// columns of every 32nd row. It takes four rows at a time, whose sums over the matrix's rows are joined together.
template <typename T>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(const __grid_constant__ Decays all) {
    constexpr int kRows = 4, kQuads = 8, kGroups = kThreads / kQuads, kMost = 128 / kGroups;
    __shared__ alignas(16) float2 ab[kRows][128];
    __shared__ float4 c[kRows][kQuads], sums[kThreads / 32][kRows][kQuads];
    const Decay& d = all.d[blockIdx.x % unsigned(all.count)];
    const int dim = d.dim, quads = dim / 4, parts = (quads + kQuads - 1) / kQuads;
    const unsigned place = blockIdx.x / unsigned(all.count), whose = place / unsigned(parts);
    const int head = int(whose % unsigned(d.heads)), seq = int(whose / unsigned(d.heads));
    const int quad0 = int(place % unsigned(parts)) * kQuads;
    if (head == 0 && quad0 == 0 && threadIdx.x == 0) check_offsets(d, seq);
    const int64_t lo = min(max(d.offsets[seq], int64_t(0)), d.rows), hi = min(max(d.offsets[seq + 1], lo), d.rows), n = hi - lo;
    const int x = int(threadIdx.x), quad = x % kQuads, group = x / kQuads;
    const bool here = quad0 + quad < quads;
    const float keep = exp2f(log2_decay(d, head));
    // who brings what of the next four rows: four warps a and b, a fifth c
    const bool brings_ab = x < 128 && x % 32 < quads, brings_c = x >= 128 && x < 160 && here;
    const int row_of = brings_c ? x / kQuads % kRows : x / 32;
    auto row_at = [&](int64_t i) { return d.later ? hi - 1 - i : lo + i; };
    float4 next[2] = {};
    auto fetch = [&](int64_t i) {
        if (i + row_of >= n) return;
        const int64_t t = row_at(i + row_of);
        if (brings_ab) {
            next[0] = read4(static_cast<const T*>(d.a) + t * d.a_row + head * d.a_head + x % 32 * 4);
            next[1] = read4(static_cast<const T*>(d.b) + t * d.b_row + head * d.b_head + x % 32 * 4);
        } else if (brings_c) {
            next[0] = read4(static_cast<const T*>(d.c) + t * d.c_row + head * d.c_head + (quad0 + quad) * 4);
        }
    };
    fetch(0);
    // value (r, col) of a given matrix lies at r * down + col * right
    const int64_t mine = (int64_t(seq) * d.heads + head) * dim * dim;
    const int down = d.transposed ? 1 : dim, right = d.transposed ? dim : 1;
    float4 s[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int r = group + i * kGroups;
        s[i] = f4_zero();
        if (d.start != nullptr && here && r < dim) {
            const float* p = d.start + mine + r * down + 4 * (quad0 + quad) * right;
            s[i] = d.transposed ? make_float4(p[0], p[dim], p[2 * dim], p[3 * dim]) : ldg4(p);
        }
    }
    for (int64_t i = 0; i < n; i += kRows) {
        if (brings_ab) {
            const float4 p = next[0], q = next[1];
            float2* to = &ab[row_of][x % 32 * 4];
            to[0] = make_float2(p.x, d.add * q.x), to[1] = make_float2(p.y, d.add * q.y);
            to[2] = make_float2(p.z, d.add * q.z), to[3] = make_float2(p.w, d.add * q.w);
        } else if (brings_c) {
            c[row_of][quad] = next[0];
        }
        __syncthreads();
        fetch(i + kRows);
        const int rows = int(min(int64_t(kRows), n - i));
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            if (j >= rows) break;
            const float w = d.later && i + j == 0 ? 1.0f : keep;
            const float4 y = c[j][quad];
            float4 sum = f4_zero();
#pragma unroll
            for (int m = 0; m < kMost; ++m) {
                const int r = group + m * kGroups;
                if (r >= dim) break;
                const float2 u = ab[j][r];
                s[m] = make_float4(fmaf(w, s[m].x, u.y * y.x), fmaf(w, s[m].y, u.y * y.y), fmaf(w, s[m].z, u.y * y.z),
                                   fmaf(w, s[m].w, u.y * y.w));
                sum = make_float4(fmaf(u.x, s[m].x, sum.x), fmaf(u.x, s[m].y, sum.y), fmaf(u.x, s[m].z, sum.z),
                                  fmaf(u.x, s[m].w, sum.w));
            }
#pragma unroll
            for (int e = kQuads; e < 32; e *= 2)
                sum = f4_add(sum, make_float4(__shfl_xor_sync(0xffffffffu, sum.x, e), __shfl_xor_sync(0xffffffffu, sum.y, e),
                                              __shfl_xor_sync(0xffffffffu, sum.z, e), __shfl_xor_sync(0xffffffffu, sum.w, e)));
            if (x % 32 < kQuads) sums[x / 32][j][quad] = sum;
        }
        __syncthreads();
        const int j = x / kQuads;
        if (d.out == nullptr || !here || j >= rows) continue;
        float4 out = f4_zero();
#pragma unroll
        for (int g = 0; g < kThreads / 32; ++g) out = f4_add(out, sums[g][j][quad]);
        write4(static_cast<T*>(d.out) + (row_at(i + j) * d.heads + head) * dim + 4 * (quad0 + quad),
               make_float4(d.far * out.x, d.far * out.y, d.far * out.z, d.far * out.w));
    }
    if (d.after == nullptr || !here) return;
    const float w = d.later && n > 0 ? keep : 1.0f;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int r = group + i * kGroups;
        if (r >= dim) break;
        float* p = d.after + mine + r * down + 4 * (quad0 + quad) * right;
        const float4 v = make_float4(w * s[i].x, w * s[i].y, w * s[i].z, w * s[i].w);
        if (d.transposed) p[0] = v.x, p[dim] = v.y, p[2 * dim] = v.z, p[3 * dim] = v.w;
        else st4(p, v);
    }
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

// Whether the sequences are taken row by row: up to 16 rows each on average, in float32 32. us row by row and by chunks, 23
// sequences with states, 32 heads: heads of 128 in bfloat16, 1 row 25 and 134, 16 rows 64 and 137, 33 rows 115 and 142, with
// gradients 237 and 377, 435 and 386; in float32 1 row 25 and 348, 33 rows 106 and 386, with gradients 411 and 1,220; heads of 64
// in bfloat16 28 and 71 (16 rows), 48 and 73 (33). Four sequences, 8 heads: 23 and 27 (16 rows, bfloat16), 22 and 34 (33,
// float32), what the host needs. All rows may be one sequence's, which then takes 0.2 to 0.3 us a row, without a bound but theirs:
// 500 rows 156 and 43 (32 heads of 128, bfloat16), 7,681 beside 511 single ones 1,960 (8 heads of 64; by itself 38).
bool few_rows(const Decay& d, int type) { return d.rows <= (type == FMD_F32 ? 32 : 16) * int64_t(d.batch); }

fmd_status run_few(const Decays& all, int type, cudaStream_t s) {
    const Decay& d = all.d[0];
    if (all.count == 0 || d.batch == 0) return FMD_OK;
    const int64_t blocks = int64_t(d.batch) * d.heads * all.count * ((d.dim + 31) / 32);
    if (blocks > INT32_MAX) return FMD_ERR_UNSUPPORTED;
    if (type == FMD_BF16) few_rows_kernel<__nv_bfloat16><<<unsigned(blocks), kThreads, 0, s>>>(all);
    else few_rows_kernel<float><<<unsigned(blocks), kThreads, 0, s>>>(all);
    return check_launch();
}

// Rows of a segment: whole sequences where these are blocks enough for the GPU or short, both on average; else so many that the
// segments fill it once (the sequences' last ones are half a segment long on average). Segments cost a second look at two of the
// three inputs and two more launches. A long sequence among short ones is walked by its heads' blocks alone: 30,000 rows beside
// 63 of 50, 8 heads of 64, take 485 us in bfloat16 and 1,190 in float32, by themselves 61 and 199.
int64_t segment_length(const Decay& d, bool planes) {
    const int64_t heads = d.heads * (planes && d.dim > 64 ? 2 : 1);  // blocks for a sequence
    if (d.rows / d.batch <= 512 || 10 * d.batch * heads >= 6 * kNumSMs) return kWhole;
    const int64_t want = 2 * kNumSMs / heads - d.batch;  // twice the segments, less the sequences' last ones
    const int64_t length = (2 * d.rows / (want > 1 ? want : 1) + 127) / 128 * 128;
    return length < 256 ? 256 : length;
}

size_t matrices(const Decay& d, int64_t n) { return size_t(n) * d.heads * d.dim * d.dim * sizeof(float); }

size_t plane_bytes(const Decay& d) { return (size_t(d.rows) * d.heads * d.dim * 6 + 255) / 256 * 256; }

// Planes of `arrays` inputs (float32), and what the segments of `passes` passes add.
size_t workspace_of(Decay d, int type, int arrays, int passes) {
    if (few_rows(d, type)) return 0;
    const bool planes = type == FMD_F32;
    d.length = segment_length(d, planes);
    return (planes ? arrays * plane_bytes(d) : 0) + (d.length < kWhole ? passes * matrices(d, decay_segments(d)) : 0);
}

// The inputs as the kernels read them: in float32 their planes, which `split` makes.
struct Input {
    const void* data;
    int64_t row, head;
};

// The planes of `inputs`, the first `made` of which are there already, at `made_at`: the workspace holds those of the others.
fmd_status make_planes(const Decay& d, Input* inputs, int count, int made, const void* made_at, char*& workspace,
                       cudaStream_t s) {
    SplitArgs a{};
    a.rows = d.rows;
    a.heads = d.heads;
    a.dim = d.dim;
    for (int i = 0; i < count; ++i) {
        if (i >= made) {
            a.x[i - made] = static_cast<const float*>(inputs[i].data);
            a.row[i - made] = inputs[i].row;
            a.head[i - made] = inputs[i].head;
            a.to[i - made] = reinterpret_cast<__nv_bfloat16*>(workspace);
        }
        const void* at = i < made ? static_cast<const char*>(made_at) + i * plane_bytes(d) : workspace;
        inputs[i] = Input{at, int64_t(d.heads) * d.dim, d.dim};
        if (i >= made) workspace += plane_bytes(d);
    }
    const dim3 grid(unsigned(grid_for(d.rows * d.heads * (d.dim / 8), kThreads)), unsigned(count - made));
    split_kernel<<<grid, kThreads, 0, s>>>(a);
    return check_launch();
}

void read_from(Decay& d, const Input& a, const Input& b, const Input& c) {
    d.a = a.data, d.a_row = a.row, d.a_head = a.head;
    d.b = b.data, d.b_row = b.row, d.b_head = b.head;
    d.c = c.data, d.c_row = c.row, d.c_head = c.head;
}

fmd_status run_states(const Decays& d, bool planes, bool early, cudaStream_t s) {
    return planes ? decay_states_planes(d, early, s) : decay_states_mma(d, early, s);
}

// Passes of the recurrence over the same rows, side by side: with segments what these add comes first.
fmd_status mix(Decays all, bool planes, char* workspace, cudaStream_t s) {
    const Decay& d = all.d[0];
    if (all.count == 0) return FMD_OK;
    const int64_t length = segment_length(d, planes);
    for (int i = 0; i < all.count; ++i) all.d[i].length = length;
    const int64_t segments = decay_segments(d);
    if (4 * segments * d.heads * all.count > INT32_MAX || int64_t(d.batch) * d.heads > INT32_MAX) return FMD_ERR_UNSUPPORTED;
    fmd_status st = FMD_OK;
    bool early = planes;  // behind the kernel that makes them
    if (length < kWhole) {
        for (int i = 0; i < all.count; ++i) {
            all.d[i].states = reinterpret_cast<float*>(workspace);
            workspace += matrices(d, segments);
        }
        if ((st = run_states(all, planes, early, s)) != FMD_OK) return st;
        const dim3 grid(unsigned(d.batch) * d.heads, unsigned((d.dim * d.dim + 4 * kThreads - 1) / (4 * kThreads)),
                        unsigned(all.count));
        if ((st = launch_early(carry_kernel, grid, kThreads, 0, s, all)) != FMD_OK) return st;
        early = true;
    } else {
        Decays ends{};  // those whose last matrix is asked for
        for (int i = 0; i < all.count; ++i)
            if (all.d[i].after != nullptr) ends.d[ends.count++] = all.d[i];
        if (ends.count > 0 && (st = run_states(ends, planes, early, s)) != FMD_OK) return st;
        early = early || ends.count > 0;
    }
    Decays rows{};
    for (int i = 0; i < all.count; ++i)
        if (all.d[i].out != nullptr) rows.d[rows.count++] = all.d[i];
    if (rows.count == 0) return FMD_OK;
    return planes ? decay_rows_planes(rows, early, s) : decay_rows_mma(rows, early, s);
}

}  // namespace

}  // namespace fmd

using namespace fmd;

extern "C" {

fmd_status fmd_decay_attention_workspace_bytes(const fmd_decay* problem, int32_t backward, size_t* bytes) {
    Decay d;
    if (problem == nullptr || bytes == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const fmd_status st = check_rows(*problem, d);
    if (st == FMD_OK) *bytes = workspace_of(d, problem->type, backward == 2 ? 1 : backward ? 4 : 3, backward ? 3 : 1);
    return st;
}

fmd_status fmd_decay_attention(const fmd_decay* problem, const float* state, void* out, float* after, void* workspace,
                               size_t workspace_bytes, int32_t* flags, void* stream) {
    Decay d;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check_rows(*problem, d);
    if (st != FMD_OK) return st;
    const fmd_decay& p = *problem;
    if (p.rows > 0 && out == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const size_t need = workspace_of(d, p.type, 3, 1);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return FMD_ERR_WORKSPACE;
    if (!aligned16(out) || !aligned16(state) || !aligned16(after) || !aligned16(workspace)) return FMD_ERR_UNSUPPORTED;
    const cudaStream_t s = as_stream(stream);
    const bool few = few_rows(d, p.type), planes = p.type == FMD_F32 && !few;
    char* at = static_cast<char*>(workspace);
    Input in[3] = {{p.q, p.q_row, p.q_head}, {p.k, p.k_row, p.k_head}, {p.v, p.v_row, p.v_head}};
    if (planes && (st = make_planes(d, in, 3, 0, nullptr, at, s)) != FMD_OK) return st;
    read_from(d, in[0], in[1], in[2]);
    d.out = out;
    d.start = state;
    d.after = after;
    d.flags = flags;
    d.near = d.far = p.scale;
    d.add = 1.0f;
    return few ? run_few(Decays{{d}, 1}, p.type, s) : mix(Decays{{d}, 1}, planes, at, s);
}

fmd_status fmd_decay_attention_bwd(const fmd_decay* problem, const float* state, const void* forward, const void* g,
                                   int64_t g_row, int64_t g_head, const float* gafter, void* dq, void* dk, void* dv,
                                   float* dstate, void* workspace, size_t workspace_bytes, int32_t* flags, void* stream) {
    Decay d;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check_rows(*problem, d);
    if (st != FMD_OK) return st;
    const fmd_decay& p = *problem;
    if (p.rows > 0 && g == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const size_t need = workspace_of(d, p.type, forward != nullptr ? 1 : 4, 3);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return FMD_ERR_WORKSPACE;
    if (!aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !aligned16(state) || !aligned16(gafter) ||
        !aligned16(dstate) || !aligned16(workspace) || !aligned16(forward) ||
        (p.rows > 0 && !vector_rows(g, g_row, g_head, p.type == FMD_BF16 ? 2 : 4)))
        return FMD_ERR_UNSUPPORTED;
    const cudaStream_t s = as_stream(stream);
    const bool few = few_rows(d, p.type), planes = p.type == FMD_F32 && !few;
    char* at = static_cast<char*>(workspace);
    Input in[4] = {{p.q, p.q_row, p.q_head}, {p.k, p.k_row, p.k_head}, {p.v, p.v_row, p.v_head}, {g, g_row, g_head}};
    if (planes && (st = make_planes(d, in, 4, forward != nullptr ? 3 : 0, forward, at, s)) != FMD_OK) return st;
    const Input &q = in[0], &k = in[1], &v = in[2], &go = in[3];
    d.flags = flags;
    d.near = p.scale;
    Decays all{};
    if (dk != nullptr || dv != nullptr || dstate != nullptr) {  // from the last row to the first
        Decay m = d;
        m.later = 1;
        m.add = p.scale;
        m.far = 1.0f;
        m.start = gafter;
        if (dv != nullptr || dstate != nullptr) {
            read_from(m, k, q, go);
            m.out = dv;
            m.after = dstate;
            all.d[all.count++] = m;
        }
        if (dk != nullptr) {
            read_from(m, v, go, q);
            m.out = dk;
            m.after = nullptr;
            m.transposed = 1;
            all.d[all.count++] = m;
        }
    }
    if (dq != nullptr) {
        Decay m = d;
        read_from(m, go, v, k);
        m.out = dq;
        m.start = state;
        m.transposed = 1;
        m.add = 1.0f;
        m.far = p.scale;
        all.d[all.count++] = m;
    }
    return few ? run_few(all, p.type, s) : mix(all, planes, at, s);
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
