// Decay attention in bfloat16 on the tensor cores.
//
// A block walks over the chunks of 128 rows of one segment and head. Of a chunk (rows t, u of it, l the decay):
//   pairs   s = a b^T;  p_tu = near l^{t-u} s_tu for u <= t, in bfloat16 back into TMEM;  near part  n = p c
//   far     f = a S with the matrix S of what lies before, in shared memory as two planes of bfloat16 (16 bits)
//   out_t = n_t + far l^{t+1} f_t
//   matrix  b'_u = l^{count-1-u} b_u in bfloat16, in place of b;  S = l^count S + b'^T c, in FP32 in registers
// (going backwards: the decays counted from the other end, decay_attention.cuh). p and b' are rounded once each, which costs
// an output about as much as its own rounding: 1.4 of it in all. One plane of S would cost as much again.
//
// states_kernel does the last line alone, for what a segment adds to the matrix; with three planes of b' where the matrix
// itself is a result, so that it is exact to FP32.
//
//   warp 8       TMA: a, b, c of one chunk after the other through a ring of slots
//   warp 9       one thread issues the products: s, f | (p, b' ready) b'^T c, p c | s of the next chunk, (S ready) f
//   warps 0-7    thread = row of the chunk and half of the pairs or columns; for the matrix its row, and half of its columns
// What lies in TMEM: s and p in its place (each thread overwrites what it has read), n, and f with b'^T c in its place.
//
// Rows of a tile that lie behind a chunk's end belong to others: their pairs are zeros, b' is zero there, and c is set to
// zero, whatever their values.
//
// Every wait is bounded: on expiry the block raises FMD_FLAG_WAIT_TIMEOUT, waits (bounded) for its copies and products in
// flight, frees its TMEM and returns.

#include "decay_attention.cuh"
#include "packed_attention_mma.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 320, kWorkers = 256;  // the workers first: a warp's part of TMEM goes by its number

// KS: steps of 16 of a head, rounded up.
template <int KS>
struct Shape {
    static constexpr int kDim = 16 * KS;
    static constexpr int kPanels = (KS + 3) / 4;
    static constexpr uint32_t kTileBytes = kPanels * kPanelBytes;
};

template <int KS>
struct RowsShape : Shape<KS> {
    using S = Shape<KS>;
    static constexpr uint32_t kMatrixPanel = S::kDim * 128;  // kDim rows x 64 columns
    static constexpr uint32_t kMatrixPlane = S::kPanels * kMatrixPanel;
    static constexpr int kSlots = 5;
    // one panel: b' is read as 128 columns of which 64 exist, so as much again follows the last slot
    static constexpr size_t kBytes =
        kSlots * S::kTileBytes + (2 * kMatrixPlane > kPanelBytes ? 2 * kMatrixPlane : kPanelBytes) + 1024;
    static constexpr uint32_t kTmem = KS <= 4 ? 256 : 512;
    static constexpr uint32_t kNear = 128, kFar = 128 + S::kDim;  // columns; the pairs at 0
};

// PLANES: of b'.
template <int KS, int PLANES>
struct StatesShape : Shape<KS> {
    using S = Shape<KS>;
    static constexpr int kSlots = PLANES == 1 ? 6 : 4;
    static constexpr size_t kBytes = kSlots * S::kTileBytes + (PLANES - 1) * S::kTileBytes + kPanelBytes + 1024;
    static constexpr uint32_t kTmem = KS <= 4 ? 64 : 128;
};

template <int SLOTS>
struct Ctrl {
    Ring<SLOTS> ring;
    uint64_t pairs, ready, added, out, matrix;
    uint64_t drain;
    uint32_t tmem;
    int32_t abort;
};

struct Maps {
    CUtensorMap a, b, c;
};

// D (+)= A^T B over `steps` steps of 16 rows of both: the columns of A are the product's M index.
__device__ __forceinline__ void product_columns(uint32_t d, uint32_t a, uint32_t b, int steps, uint32_t idesc, bool add) {
    const uint32_t ad = columns_desc(a), bd = columns_desc(b);
    for (int k = 0; k < steps; ++k)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 u, v;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 u, {%1, %3};\n\t"
            "mov.b64 v, {%2, %3};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], u, v, %4, p;\n\t}" ::"r"(d),
            "r"(ad + k * 128), "r"(bd + k * 128), "r"(kDescHigh), "r"(idesc), "r"(uint32_t(add || k > 0))
            : "memory");
}

// D (+)= A B: the rows of A the product's M index, those of B (panels `panel` bytes apart) its inner index.
template <int KS>
__device__ __forceinline__ void product_matrix(uint32_t d, uint32_t a, uint32_t b, uint32_t panel, uint32_t idesc, bool add) {
    const uint32_t ad = rows_desc(a), bd = ((b & 0x3FFFFu) >> 4) | ((panel >> 4) << 16);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        const uint32_t off = uint32_t(k / 4) * kPanelStep + uint32_t(k % 4) * 2;
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 u, v;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 u, {%1, %3};\n\t"
            "mov.b64 v, {%2, %3};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], u, v, %4, p;\n\t}" ::"r"(d),
            "r"(ad + off), "r"(bd + k * 128), "r"(kDescHigh), "r"(idesc), "r"(uint32_t(add || k > 0))
            : "memory");
    }
}

// Row r of a tile times `weight` as PLANES planes (the first in its place, the others `more` apart from there on): the
// eights of a row in an order that keeps the banks apart; the swizzle moves eights within their row only.
template <int KS, int PLANES>
__device__ __forceinline__ void weigh_row(unsigned char* tile, unsigned char* more, int r, int half, float weight, bool real) {
    constexpr int kEights = KS <= 4 ? 4 : 8;  // of a row and panel that this half takes
    unsigned char* row = tile + (KS <= 4 ? 0 : half * kPanelBytes) + r * 128;
#pragma unroll
    for (int i = 0; i < kEights; ++i) {
        const int at = (((KS <= 4 ? 4 * half : 0) + i) ^ (r & 7)) * 16;
        uint4* p = reinterpret_cast<uint4*>(row + at);
        float v[8];
        uint32_t w[4] = {0, 0, 0, 0};
        if (real) {
            const uint4 x = *p;
            const float2 y[4] = {unpack_bf16(x.x), unpack_bf16(x.y), unpack_bf16(x.z), unpack_bf16(x.w)};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = y[e].x * weight;
                v[2 * e + 1] = y[e].y * weight;
            }
            next_plane<4>(v, w);
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int q = 1; q < PLANES; ++q) {
            if (real) next_plane<4>(v, w);
            *reinterpret_cast<uint4*>(more + size_t(q - 1) * Shape<KS>::kTileBytes + (KS <= 4 ? 0 : half * kPanelBytes) +
                                      r * 128 + at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// The decay of row j of a chunk of `count` as it enters the matrix.
__device__ __forceinline__ float weight_of(const Decay& d, int j, int count, float l2) {
    return d.add * ex2(float(d.later ? j + 1 : count - 1 - j) * l2);
}

// Columns [0, N) that follow `col0` of the thread's row of the matrix: FP32 in `state`, as two planes in shared memory.
template <int KS, int N>
__device__ __forceinline__ void store_matrix(unsigned char* to, int r, int col0, const float (&state)[N]) {
    using S = RowsShape<KS>;
#pragma unroll
    for (int i = 0; i < N; i += 8) {
        float v[8];
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = state[i + e];
        const int eight = (col0 + i) / 8;
        unsigned char* p = to + (eight / 8) * S::kMatrixPanel + r * 128 + ((eight % 8) ^ (r & 7)) * 16;
        next_plane<4>(v, w);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
        *reinterpret_cast<uint4*>(p + S::kMatrixPlane) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// state = keep state + N columns of TMEM.
template <int N>
__device__ __forceinline__ void add_columns(uint32_t at, float keep, float (&state)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 16) {
        float x[16];
        tmem_load16(at + i, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) state[i + e] = fmaf(keep, state[i + e], x[e]);
    }
}

template <int SLOTS>
__device__ __forceinline__ void open_block(Ctrl<SLOTS>& ctl) {
    if (threadIdx.x == 0) {
        init_ring(ctl.ring);
        mbar_init(&ctl.pairs, 1);
        mbar_init(&ctl.ready, kWorkers / 32);
        mbar_init(&ctl.added, 1);
        mbar_init(&ctl.out, 1);
        mbar_init(&ctl.matrix, kWorkers / 32);
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
}

// The copies of a walk, tile i by load(i, slot, barrier); then until their slots are released, or have landed.
template <int SLOTS, typename Load>
__device__ __forceinline__ void feed_tiles(Ctrl<SLOTS>& ctl, volatile int32_t* abort, int count, uint32_t bytes, Load load) {
    int slot = 0, armed = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < count; ++i) {
        if (!mbar_wait(&ctl.ring.empty[slot], phase ^ 1u, abort)) {
            ok = false;
            break;
        }
        mbar_expect_tx(&ctl.ring.full[slot], bytes);
        load(i, slot, &ctl.ring.full[slot]);
        armed = i + 1;
        if (++slot == SLOTS) {
            slot = 0;
            phase ^= 1u;
        }
    }
    for (int i = max(0, armed - SLOTS); i < armed; ++i) {
        const uint32_t parity = uint32_t(i / SLOTS) & 1u;
        if (ok) ok = mbar_wait(&ctl.ring.empty[i % SLOTS], parity, abort);
        if (!ok) mbar_wait(&ctl.ring.full[i % SLOTS], parity, abort, true);
    }
}

__device__ __forceinline__ bool worker_wait(uint64_t* bar, uint32_t parity, volatile int32_t* abort) {
    const bool got = mbar_wait(bar, parity, abort);
    if (__all_sync(0xffffffffu, got)) return true;  // uniform in the warp: TMEM access is .sync.aligned
    *abort = 1;
    return false;
}

// The stretch of this block, found by its first warp.
__device__ __forceinline__ Stretch block_stretch(const Decay& d, int64_t index) {
    __shared__ Stretch place;
    if (threadIdx.x < 32) {
        const Stretch s = stretch_of(d, index);
        if (threadIdx.x == 0) place = s;
    }
    __syncthreads();
    return place;
}

template <int KS>
__global__ void __launch_bounds__(kThreads, KS <= 4 ? 2 : 1) rows_kernel(const __grid_constant__ Maps maps, const Decay d,
                                                                         const bool carried) {
    using S = RowsShape<KS>;
    constexpr int kHalf = 8 * KS;  // columns of a half
    extern __shared__ unsigned char raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* matrix = ring + S::kSlots * S::kTileBytes;
    __shared__ Ctrl<S::kSlots> ctl;
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = int(blockIdx.x % unsigned(d.heads));
    const int64_t index = blockIdx.x / unsigned(d.heads);

    if (head == 0 && threadIdx.x == 256 && index < d.batch) check_offsets(d, index);
    const Stretch s = block_stretch(d, index);
    if (s.rows == 0) return;
    const int chunks = int((s.rows + kTile - 1) / kTile);
    open_block(ctl);
    if (warp == 9) tmem_alloc<S::kTmem>(&ctl.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    auto rows_of = [&](int i) { return int(min(int64_t(kTile), s.rows - int64_t(i) * kTile)); };
    auto first_of = [&](int i) {
        return d.later ? s.row0 + s.rows - int64_t(i) * kTile - rows_of(i) : s.row0 + int64_t(i) * kTile;
    };

    if (warp == 8) {
        if (lane == 0)
            feed_tiles(ctl, abort, 3 * chunks, S::kTileBytes, [&](int i, int slot, uint64_t* bar) {
                const int chunk = i / 3, what = i - 3 * chunk, row = int(first_of(chunk));
                const CUtensorMap* map = what == 0 ? &maps.a : what == 1 ? &maps.b : &maps.c;
                for (int p = 0; p < S::kPanels; ++p)
                    tma_load_4d(su32(ring + slot * S::kTileBytes + p * kPanelBytes), map, bar, p * 64, 0, head, row);
            });
    } else if (warp == 9) {
        const uint32_t base = uniform(tmem), first_slot = uniform(su32(ring)), planes = uniform(su32(matrix));
        const int count = uniform(chunks), last = uniform(rows_of(chunks - 1));
        const uint32_t pairs_desc = bf16_idesc(kTile, false), out_desc = bf16_idesc(S::kDim, true),
                       add_desc = out_desc | 1u << 15;
        auto slot = [&](int i) { return first_slot + uint32_t(i % S::kSlots) * S::kTileBytes; };
        bool ok = true, issued = false;
        auto pairs = [&](int i) {  // over the pairs of the chunk before, whose product has been issued
            ok = ok && landed(ctl.ring, 3 * i, abort) && landed(ctl.ring, 3 * i + 1, abort);
            if (!ok) return;
            tc_fence_after();
            if (elect_one()) product_rows<KS>(base, slot(3 * i), slot(3 * i + 1), pairs_desc);
            issued = true;
        };
        pairs(0);
        for (int i = 0; i < count && ok; ++i) {
            ok = warp_wait(&ctl.matrix, uint32_t(i) & 1u, abort);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                product_matrix<KS>(base + S::kFar, slot(3 * i), planes + S::kMatrixPlane, S::kMatrixPanel, out_desc, false);
                product_matrix<KS>(base + S::kFar, slot(3 * i), planes, S::kMatrixPanel, out_desc, true);
                tc_commit(&ctl.pairs);
                tc_commit(&ctl.ring.empty[(3 * i) % S::kSlots]);
            }
            ok = landed(ctl.ring, 3 * i + 2, abort) && warp_wait(&ctl.ready, uint32_t(i) & 1u, abort);
            if (!ok) break;
            tc_fence_after();
            const int steps = ((i + 1 == count ? last : kTile) + 15) / 16;
            if (elect_one()) {
                product_columns(base + S::kFar, slot(3 * i + 1), slot(3 * i + 2), steps, add_desc, false);
                tc_commit(&ctl.added);
                tc_commit(&ctl.ring.empty[(3 * i + 1) % S::kSlots]);
                product_weights<8, 4, 64>(base + S::kNear, base, slot(3 * i + 2), steps, out_desc, false);
                tc_commit(&ctl.out);
                tc_commit(&ctl.ring.empty[(3 * i + 2) % S::kSlots]);
            }
            if (i + 1 < count) pairs(i + 1);
        }
        if (!ok && issued) {  // the products in flight end before TMEM is freed
            if (elect_one()) tc_commit(&ctl.drain);
            warp_wait(&ctl.drain, 0, abort, true);
        }
    } else {
        const int half = warp >> 2, r = threadIdx.x & 127, col0 = half * kHalf;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t at_pairs = tmem + lanes + uint32_t(half) * 64u, at_near = tmem + lanes + S::kNear + col0,
                       at_far = tmem + lanes + S::kFar + col0;
        const float l2 = log2_decay(d, head), way = d.later ? -1.0f : 1.0f;
        float state[kHalf];
        {
            const float* start = carried ? d.states + (index * d.heads + head) * d.dim * d.dim
                                 : d.start != nullptr ? d.start + (int64_t(s.b) * d.heads + head) * d.dim * d.dim : nullptr;
            const bool turn = !carried && d.transposed;
#pragma unroll
            for (int i = 0; i < kHalf; ++i) {
                const int col = col0 + i;
                state[i] = start != nullptr && r < d.dim && col < d.dim ? start[turn ? col * d.dim + r : r * d.dim + col] : 0.0f;
            }
        }
        const bool holds = r < S::kDim;
        if (holds) store_matrix<KS>(matrix, r, col0, state);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        warp_arrive(&ctl.matrix);
        for (int i = 0; i < chunks; ++i) {
            const int count = rows_of(i);
            const uint32_t parity = uint32_t(i) & 1u;
            if (!worker_wait(&ctl.pairs, parity, abort)) break;
            tc_fence_after();
            const float t = way * float(r - 64 * half);
#pragma unroll
            for (int ch = 0; ch < 64; ch += 32) {
                float x[32];
                uint32_t p[16];
                tmem_load32(at_pairs + ch, x);
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float gap = fmaf(float(ch + e), -way, t);
                    const float w = ex2(gap * l2) * d.near;
                    x[e] = gap >= 0.0f && ch + e < count - 64 * half ? x[e] * w : 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
                tmem_store16(at_pairs + ch / 2, p);
            }
            float far[kHalf];
#pragma unroll
            for (int e = 0; e < kHalf; e += 16) tmem_load16(at_far + e, reinterpret_cast<float(&)[16]>(far[e]));
            const int tile_b = 3 * i + 1, tile_c = 3 * i + 2;
            if (!worker_wait(&ctl.ring.full[tile_b % S::kSlots], uint32_t(tile_b / S::kSlots) & 1u, abort)) break;
            weigh_row<KS, 1>(ring + (tile_b % S::kSlots) * S::kTileBytes, nullptr, r, half,
                             r < count ? weight_of(d, r, count, l2) : 0.0f, r < count);
            if (count < kTile) {
                if (!worker_wait(&ctl.ring.full[tile_c % S::kSlots], uint32_t(tile_c / S::kSlots) & 1u, abort)) break;
                zero_rows(ring + (tile_c % S::kSlots) * S::kTileBytes, S::kPanels, kPanelBytes, count, (count + 15) & ~15,
                          threadIdx.x, kWorkers);
            }
            tmem_wait_st();
            tc_fence_before();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(&ctl.ready);
            if (!worker_wait(&ctl.added, parity, abort)) break;
            tc_fence_after();
            add_columns(at_far, ex2(float(count) * l2), state);
            if (i + 1 < chunks) {
                if (holds) store_matrix<KS>(matrix, r, col0, state);
                tc_fence_before();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                warp_arrive(&ctl.matrix);
            }
            if (!worker_wait(&ctl.out, parity, abort)) break;
            tc_fence_after();
            const float reach = d.far * ex2(float(d.later ? count - 1 - r : r + 1) * l2);
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(d.out) + ((first_of(i) + r) * d.heads + head) * d.dim + col0;
#pragma unroll
            for (int e = 0; e < kHalf; e += 16) {
                float x[16];
                tmem_load16(at_near + e, x);
                if (r >= count) continue;
                uint32_t w[8];
#pragma unroll
                for (int o = 0; o < 8; ++o)
                    w[o] = pack_bf16(fmaf(reach, far[e + 2 * o], x[2 * o]), fmaf(reach, far[e + 2 * o + 1], x[2 * o + 1]));
                if (col0 + e < d.dim) *reinterpret_cast<uint4*>(out + e) = make_uint4(w[0], w[1], w[2], w[3]);
                if (col0 + e + 8 < d.dim) *reinterpret_cast<uint4*>(out + e + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_free<S::kTmem>(tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(d.flags, FMD_FLAG_WAIT_TIMEOUT);
}

template <int KS, int PLANES>
__global__ void __launch_bounds__(kThreads, 1) states_kernel(const __grid_constant__ Maps maps, const Decay d) {
    using S = StatesShape<KS, PLANES>;
    constexpr int kHalf = 8 * KS;
    extern __shared__ unsigned char raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* more = ring + S::kSlots * S::kTileBytes;
    __shared__ Ctrl<S::kSlots> ctl;
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = int(blockIdx.x % unsigned(d.heads));
    const int64_t index = blockIdx.x / unsigned(d.heads);

    const Stretch s = block_stretch(d, index);
    if (s.rows == 0) return;
    const int chunks = int((s.rows + kTile - 1) / kTile);
    open_block(ctl);
    if (warp == 9) tmem_alloc<S::kTmem>(&ctl.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    auto rows_of = [&](int i) { return int(min(int64_t(kTile), s.rows - int64_t(i) * kTile)); };
    auto first_of = [&](int i) {
        return d.later ? s.row0 + s.rows - int64_t(i) * kTile - rows_of(i) : s.row0 + int64_t(i) * kTile;
    };

    if (warp == 8) {
        if (lane == 0)
            feed_tiles(ctl, abort, 2 * chunks, S::kTileBytes, [&](int i, int slot, uint64_t* bar) {
                for (int p = 0; p < S::kPanels; ++p)
                    tma_load_4d(su32(ring + slot * S::kTileBytes + p * kPanelBytes), i & 1 ? &maps.c : &maps.b, bar, p * 64, 0,
                                head, int(first_of(i >> 1)));
            });
    } else if (warp == 9) {
        const uint32_t base = uniform(tmem), first_slot = uniform(su32(ring)), planes = uniform(su32(more));
        const int count = uniform(chunks), last = uniform(rows_of(chunks - 1));
        const uint32_t desc = bf16_idesc(S::kDim, true) | 1u << 15;
        auto slot = [&](int i) { return first_slot + uint32_t(i % S::kSlots) * S::kTileBytes; };
        bool ok = true, issued = false;
        for (int i = 0; i < count && ok; ++i) {
            ok = landed(ctl.ring, 2 * i, abort) && landed(ctl.ring, 2 * i + 1, abort) &&
                 warp_wait(&ctl.ready, uint32_t(i) & 1u, abort);
            if (!ok) break;
            tc_fence_after();
            const int steps = ((i + 1 == count ? last : kTile) + 15) / 16;
            if (elect_one()) {
#pragma unroll
                for (int p = PLANES - 1; p > 0; --p)
                    product_columns(base, planes + (p - 1) * S::kTileBytes, slot(2 * i + 1), steps, desc, p < PLANES - 1);
                product_columns(base, slot(2 * i), slot(2 * i + 1), steps, desc, PLANES > 1);
                tc_commit(&ctl.added);
                tc_commit(&ctl.ring.empty[(2 * i) % S::kSlots]);
                tc_commit(&ctl.ring.empty[(2 * i + 1) % S::kSlots]);
            }
            issued = true;
        }
        if (!ok && issued) {
            if (elect_one()) tc_commit(&ctl.drain);
            warp_wait(&ctl.drain, 0, abort, true);
        }
    } else {
        const int half = warp >> 2, r = threadIdx.x & 127, col0 = half * kHalf;
        const uint32_t at = tmem + (uint32_t((warp & 3) * 32) << 16) + col0;
        const float l2 = log2_decay(d, head);
        float state[kHalf] = {};
        bool ok = true;
        for (int i = 0; i < chunks; ++i) {
            const int count = rows_of(i), tile_b = 2 * i, tile_c = 2 * i + 1;
            ok = worker_wait(&ctl.ring.full[tile_b % S::kSlots], uint32_t(tile_b / S::kSlots) & 1u, abort);
            if (!ok) break;
            weigh_row<KS, PLANES>(ring + (tile_b % S::kSlots) * S::kTileBytes, more, r, half,
                                  r < count ? weight_of(d, r, count, l2) : 0.0f, r < count);
            if (count < kTile) {
                ok = worker_wait(&ctl.ring.full[tile_c % S::kSlots], uint32_t(tile_c / S::kSlots) & 1u, abort);
                if (!ok) break;
                zero_rows(ring + (tile_c % S::kSlots) * S::kTileBytes, S::kPanels, kPanelBytes, count, (count + 15) & ~15,
                          threadIdx.x, kWorkers);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(&ctl.ready);
            ok = worker_wait(&ctl.added, uint32_t(i) & 1u, abort);
            if (!ok) break;
            tc_fence_after();
            add_columns(at, ex2(float(count) * l2), state);
            tc_fence_before();
        }
        if (ok && r < d.dim) {
            float* out = d.states + ((index * d.heads + head) * d.dim + r) * d.dim + col0;
#pragma unroll
            for (int i = 0; i < kHalf; i += 4)
                if (col0 + i < d.dim) st4(out + i, make_float4(state[i], state[i + 1], state[i + 2], state[i + 3]));
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_free<S::kTmem>(tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(d.flags, FMD_FLAG_WAIT_TIMEOUT);
}

fmd_status encode(Maps& maps, const Decay& d, bool rows) {
    const DriverCalls& drv = driver_calls();
    if (drv.encode == nullptr || drv.ctx_get_current == nullptr)
        return record_error_text(FMD_ERR_CUDA, "driver entry point cuTensorMapEncodeTiled unavailable", 0);
    fmd_status st = bind_context(drv);
    if (st == FMD_OK && rows) st = encode_packed(drv, &maps.a, d.a, d.rows, d.heads, 1, d.dim, d.a_row, d.a_head, kTile);
    if (st == FMD_OK) st = encode_packed(drv, &maps.b, d.b, d.rows, d.heads, 1, d.dim, d.b_row, d.b_head, kTile);
    if (st == FMD_OK) st = encode_packed(drv, &maps.c, d.c, d.rows, d.heads, 1, d.dim, d.c_row, d.c_head, kTile);
    return st;
}

template <int KS>
fmd_status launch_rows(const Maps& maps, const Decay& d, bool carried, cudaStream_t s) {
    constexpr size_t bytes = RowsShape<KS>::kBytes;
    const fmd_status st = grant_dynamic_smem((const void*)rows_kernel<KS>, bytes, true);
    if (st != FMD_OK) return st;
    rows_kernel<KS><<<unsigned(decay_segments(d) * d.heads), kThreads, bytes, s>>>(maps, d, carried);
    return check_launch();
}

template <int KS, int PLANES>
fmd_status launch_states(const Maps& maps, const Decay& d, cudaStream_t s) {
    constexpr size_t bytes = StatesShape<KS, PLANES>::kBytes;
    const fmd_status st = grant_dynamic_smem((const void*)states_kernel<KS, PLANES>, bytes, true);
    if (st != FMD_OK) return st;
    states_kernel<KS, PLANES><<<unsigned(decay_segments(d) * d.heads), kThreads, bytes, s>>>(maps, d);
    return check_launch();
}

template <int KS>
fmd_status launch_states(const Maps& maps, const Decay& d, cudaStream_t s) {
    return d.after != nullptr ? launch_states<KS, 3>(maps, d, s) : launch_states<KS, 1>(maps, d, s);
}

}  // namespace

fmd_status decay_states_mma(const Decay& d, cudaStream_t s) {
    Maps maps{};
    const fmd_status st = encode(maps, d, false);
    if (st != FMD_OK) return st;
    return d.dim <= 32 ? launch_states<2>(maps, d, s) : d.dim <= 64 ? launch_states<4>(maps, d, s)
         : d.dim <= 96 ? launch_states<6>(maps, d, s) : launch_states<8>(maps, d, s);
}

fmd_status decay_rows_mma(const Decay& d, bool carried, cudaStream_t s) {
    Maps maps{};
    const fmd_status st = encode(maps, d, true);
    if (st != FMD_OK) return st;
    return d.dim <= 32 ? launch_rows<2>(maps, d, carried, s) : d.dim <= 64 ? launch_rows<4>(maps, d, carried, s)
         : d.dim <= 96 ? launch_rows<6>(maps, d, carried, s) : launch_rows<8>(maps, d, carried, s);
}

}  // namespace fmd
