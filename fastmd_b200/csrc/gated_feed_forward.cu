// Gated feed-forward block and its backward pass, as products on the tensor cores with the rest of the block in them.
//
//   a = x Wg^T, b = x Wu^T, h = act(a) b, y = h Wd^T              x [rows, width], Wg, Wu [hidden, width], Wd [out, hidden]
//   dh = g Wd;  da = dh (b act'(a)), db = dh act(a)
//   dx = da Wg + db Wu;  dWg = da^T x, dWu = db^T x, dWd = g^T h
//
// Five products, each a kernel of the one form below; they differ in how operands lie and in what follows the sums. us and
// TFLOP/s of 32,000 x 1,024 x 4,096 in bfloat16, forward and backward (1,816 in all, 1,330 TFLOP/s):
//   up       x [Wg; Wu]^T: a tile's columns are half a's and half b's, so that h follows where the sums are; where a backward
//            pass follows, b act'(a) and act(a) are kept too                                          416 us, 1,290 TFLOP/s
//   down     h Wd^T                                                                                   181 us, 1,490
//   hidden   g Wd, times what was kept: da and db; 1.1 GB of memory, 170 us by itself                 304 us,   880
//   input    [da, db] [Wg; Wu]: one sum over both                                                     347 us, 1,550
//   weights  da^T x, db^T x, g^T h: three problems of one launch                                      546 us, 1,480
// Many rows are bound by the tensor cores (up and hidden by what follows the sums: waits for memory, 16 warps an SM), a few by
// the weights' bytes: up of 8 x 4,096 x 11,000 takes 36 us, 5.0 TB/s.
//
// Roundings: h, da and db are operands of further products and are stored in bfloat16; each costs the result as much as its
// own last rounding, 1.4 of it in all. What the gradients are multiplied by is kept in 11 bits, beside the largest of a row's 16
// units (Args), which costs next to nothing; as bfloat16 it would cost as much again.
//
// float32: every operand is three planes of bfloat16 (x = x0 + x1 + x2, 24 bits) and a product is the six of its planes
// that count: x0 w0 apart from the five small ones, because the tensor cores cut off what does not fit as they add. For the
// same reason sums are taken out of TMEM and added up in registers every kSegment steps of 64.
//
// A block walks over tiles of 128 x bn: one warp loads operands by TMA through a ring of slots (64 values of the inner index
// each), one thread of another issues the products, 8 or 16 take the sums from one of two accumulators in TMEM while the
// other one is filled: thread = row and part of the columns.
//
// Pairs of blocks: where a launch has enough tiles, the two SMs of a cluster work on 256 x 256 together, each with its own 128
// rows of A and half of B's columns, since one block's tile of 128 x 256 takes 48 KB a step of 512 cycles of products and an
// SM gets about 64 bytes a cycle (1,230 TFLOP/s). The first block of the pair issues the products of both; copies of both
// arrive on its barriers, its commits on both blocks'.
//
// Every wait is bounded: on expiry the block raises FMD_FLAG_WAIT_TIMEOUT, waits (bounded) for its copies and products in
// flight, frees its TMEM and returns.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tensor_cores.cuh"

namespace fmd {
namespace {

constexpr int kM = 128, kK = 64;
constexpr uint32_t kTileA = kM * kK * 2, kPanel = 64 * kK * 2;  // bytes of an operand's tile, of 64 columns of it
constexpr int kMostSlots = 12;
constexpr int kSegment = 2;

enum Kind { kUp, kDown, kHidden, kInput, kWeights };

// Warps that take the sums: sixteen where much follows them, which eight did not get through in the time of a tile's products
// (up of 32,000 x 1,024 x 4,096 with its factors 718 us, hidden 923); hidden in float32 has six times the products, and needs
// the registers.
template <int KIND, int P>
struct Shape {
    static constexpr int kWarps = KIND == kUp || (P == 1 && KIND == kHidden) ? 16 : 8;
    static constexpr int kThreads = 64 + 32 * kWarps;  // the takers first: a warp's part of TMEM goes by its number
    static constexpr size_t kScratch = kWarps == 16 ? 2048 : 4096;  // of each of these warps
    static constexpr size_t kRing = 224 * 1024 - kWarps * kScratch;
    static constexpr size_t kBytes = 225 * 1024;
};

// One product [m, n] of a launch; `out` null (kinds with one): not asked for, its tiles are passed over.
struct Problem {
    void* out;
    int64_t m, n;
    int32_t a, b;  // maps
    int32_t a_panels, b_panels;  // whether the operands' maps go by panels of 64 columns
    int32_t m_tiles, n_tiles;
};

struct Args {
    Problem problem[3];
    int32_t problems;
    int32_t tiles, whole, splits;  // tiles of all problems; those from `whole` on are shared out along the inner index
    float* part;                   // [tiles - whole][splits][128][bn]: the shares' sums
    int32_t tile_m;                // rows of a tile: 128, of a pair 256
    int32_t steps, turn;  // of 64 along the inner index; from step `turn` on the second pair of maps (kInput)
    int32_t bn, slots, act;
    int32_t tile_a;  // bytes of A's tile in a slot
    // h, da and db in panels of 64 hidden units, [planes][panels][rows][64]: a warp's store and a tile's copy are each in one
    // piece of memory. The last panel is filled up with zeros.
    __nv_bfloat16 *h, *da, *db;
    int64_t plane;  // values of a plane
    int32_t panels;
    // What the gradients are multiplied by, b act'(a) and act(a), as the threads hold it: blocks of 32 rows x 16 units,
    // [unit / 16][row / 32][piece of 16 bytes][row % 32]. FP32; in 16 bits float16 times a power of two of each row's 16
    // units, whose inverse is `unit` [unit / 16][row] (11 bits, for values over 2^-29 of the largest of the 16, fewer below and
    // none under 2^-39, where a unit adds next to nothing to what its neighbours do: a rounding to bfloat16 would cost the
    // gradients as much as their own, and FP32 the kernels that wait for memory a fifth)
    void *slope, *level;
    float2* unit;
    int32_t blocks;  // of 32 rows
    int32_t* flags;
};

struct Maps {
    CUtensorMap a[3], b[3];
};

struct Ctrl {
    uint64_t full[kMostSlots], empty[kMostSlots];
    uint64_t sums[2], taken[2];
    uint64_t drain;
    uint32_t tmem;
    int32_t abort;
};

__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[16]) { tmem_load16(at, v); }
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[32]) { tmem_load32(at, v); }
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[64]) { tmem_load64(at, v); }

#define FMD_MMA2(GROUP)                                                                                            \
    asm volatile(                                                                                                  \
        "{\n\t.reg .pred p;\n\t.reg .b32 x, y;\n\t.reg .b64 u, v, w, z;\n\t"                                         \
        "setp.ne.b32 p, %5, 0;\n\tadd.u32 x, %1, %6;\n\tadd.u32 y, %2, %7;\n\t"                                     \
        "mov.b64 u, {%1, %3};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 w, {x, %3};\n\tmov.b64 z, {y, %3};\n\t"             \
        "tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], u, v, %4, p;\n\t"                                         \
        "tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], w, z, %4, 1;\n\t}" ::"r"(d),                              \
        "r"(a), "r"(b), "r"(kDescHigh), "r"(idesc), "r"(add), "n"(ASTEP), "n"(BSTEP)                               \
        : "memory")

// Two steps of 16 of D (+)= A B^T; ASTEP, BSTEP: how far a step is, in descriptor units. PAIR: of both blocks' rows.
template <bool PAIR, int ASTEP, int BSTEP>
__device__ __forceinline__ void mma2(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    if constexpr (PAIR) FMD_MMA2("2");
    else FMD_MMA2("1");
}

// What a single block does by itself and a pair together.
template <bool PAIR>
struct Group {
    __device__ static uint32_t rank() {
        uint32_t r = 0;
        if (PAIR) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
        return r;
    }
    // the first block's copy of a barrier
    __device__ static uint32_t first(uint64_t* bar) {
        uint32_t a = su32(bar);
        if (PAIR) asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(a));
        return a;
    }
    __device__ static void sync() {
        __syncwarp();
        if (PAIR)
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else
            __syncthreads();
    }
    __device__ static void load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
        if (PAIR)
            asm volatile(
                "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
                "{%2, %3, %4, %5}], [%6];" ::"r"(dst),
                "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                : "memory");
        else
            asm volatile(
                "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
                "%5}], [%6];" ::"r"(dst),
                "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                : "memory");
    }
    // all products so far: an arrival on the barrier, in both blocks
    __device__ static void commit(uint64_t* bar) {
        if (PAIR)
            asm volatile(
                "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                    su32(bar)),
                "h"(uint16_t(3))
                : "memory");
        else
            tc_commit(bar);
    }
    // a warp's arrival on the first block's barrier
    __device__ static void arrive(uint64_t* bar) {
        __syncwarp();
        if ((threadIdx.x & 31) != 0) return;
        if (PAIR)
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(first(bar)) : "memory");
        else
            mbar_arrive(bar);
    }
    __device__ static void alloc(uint32_t* address) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(address)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc<512>(address);
        }
    }
    __device__ static void free(uint32_t address) {
        if (PAIR) {
            __syncwarp();
            tc_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(address) : "memory");
        } else {
            tmem_free<512>(address);
        }
    }
};

// The place of a block's turn: its problem, rows and columns, the steps of its share of the inner index, and which of the
// shares it is (part: its place among them; -1: a whole tile).
struct Place {
    int problem, m, n, part, from, to;
};

__device__ __forceinline__ int turns_of(const Args& g) { return g.whole + (g.tiles - g.whole) * g.splits; }

__device__ __forceinline__ Place place_of(const Args& g, int t) {
    Place p;
    p.problem = 0;
    p.part = -1;
    p.from = 0;
    p.to = g.steps;
    if (t >= g.whole && g.splits > 1) {
        const int shared = g.tiles - g.whole, split = (t - g.whole) / shared, share = (g.steps + g.splits - 1) / g.splits;
        t -= split * shared;
        p.part = (t - g.whole) * g.splits + split;
        p.from = min(g.steps, split * share);
        p.to = min(g.steps, p.from + share);
    }
    while (p.problem + 1 < g.problems) {
        const int here = g.problem[p.problem].m_tiles * g.problem[p.problem].n_tiles;
        if (t < here) break;
        t -= here;
        ++p.problem;
    }
    const Problem& q = g.problem[p.problem];
    p.m = t / q.n_tiles;
    p.n = t - p.m * q.n_tiles;
    return p;
}

// Whether anybody wants the problem.
template <int KIND>
__device__ __forceinline__ bool wanted(const Problem& q) {
    return KIND != kWeights || q.out != nullptr;
}

__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The normal distribution's share below a, with density = e^{-a a / 2}: a tail is density t Q(t), t = 1 / (1 + 0.24 |a|), with
// Q of degree 7 fitted to the smallest RELATIVE error over all of t (Lawson's reweighted least squares on 4,001 points), so
// that the far tail, which is act(a) / a itself, keeps its bits: 8 10^-7 with FP32's roundings, and below zero the density's
// own (2^-17 at a = -9, where its exponent is 58). A fit with a small absolute error is off by 1.5 % there. Half of up's
// instructions were the library's erfc (10,007 x 264 x 1,000: 47 -> 34 us).
__device__ __forceinline__ float normal_share(float a, float density) {
    const float t = rcp(fmaf(fabsf(a), 0.24f, 1.0f));
    float sum = fmaf(-0.0529904664f, t, 0.152788535f);
    sum = fmaf(sum, t, -0.0656932741f);
    sum = fmaf(sum, t, 0.118379958f);
    sum = fmaf(sum, t, 0.0634018555f);
    sum = fmaf(sum, t, 0.0928374827f);
    sum = fmaf(sum, t, 0.0955223069f);
    sum = fmaf(sum, t, 0.0957537889f);
    const float tail = density * t * sum;
    return a < 0.0f ? tail : 1.0f - tail;
}

// act(a) and act'(a). EXACT: to FP32's last bits; else, for results in 16 bits, to 2^-20 or so. Of themselves, that is, but far
// below zero, where both keep what the rounding of e^{-a a / 2}'s or e^a's exponent leaves (2^-17 at a = -9).
template <bool EXACT>
__device__ __forceinline__ void activate(int act, float a, float& value, float& slope) {
    // held where a factor of 0 stands for the limit, so that an infinity gives its limit too
    const float low = fmaxf(a, -1.0e18f), held = fminf(low, 1.0e18f);
    if (act == FMD_FEED_SILU) {
        const float turn = EXACT ? 1.0f / (1.0f + expf(-a)) : rcp(1.0f + ex2(-1.4426950408889634f * a));
        value = low * turn;
        slope = fmaf(held * turn, 1.0f - turn, turn);
    } else {
        const float density = EXACT ? expf(-0.5f * a * a) : ex2(-0.7213475204444817f * a * a);
        const float share = EXACT ? 0.5f * erfcf(-0.7071067811865476f * a) : normal_share(a, density);
        value = low * share;
        slope = fmaf(held, 0.3989422804014327f * density, share);
    }
}

__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }

// The power of two that takes 16 values to float16's upper range, and those values; `unit`: its inverse.
__device__ __forceinline__ void pack_halves(const float* v, uint4 (&w)[2], float& unit) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(v[i]));
    int e = int(__float_as_uint(most) >> 23);
    if (e == 255) {  // of the finite ones
        most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(v[i]) < __int_as_float(0x7f800000) ? fabsf(v[i]) : 0.0f);
        e = int(__float_as_uint(most) >> 23);
    }
    const int shift = min(127 + 14 - e, 100);  // the largest becomes 2^14 .. 2^15
    const float up = __uint_as_float(uint32_t(127 + shift) << 23);
    unit = __uint_as_float(uint32_t(127 - shift) << 23);
    uint32_t* p = reinterpret_cast<uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i] * up, v[2 * i + 1] * up);
        p[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
}

__device__ __forceinline__ float2 unpack_half(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

__device__ __forceinline__ uint4 as_piece(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}

// N values a row as P planes, `plane` values apart. The values are used up.
template <int P, int N>
__device__ __forceinline__ void put_planes(unsigned char* scratch, float* v, __nv_bfloat16* to, int64_t row, int64_t plane,
                                           int rows, int columns) {
    uint4 w[N / 8];
#pragma unroll
    for (int q = 0; q < P; ++q) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i)
            w[i] = P == 1 ? pack8(v + 8 * i) : q == 0 ? first_plane8(v + 8 * i) : next_plane8(v + 8 * i);
        put_rows<N / 8>(scratch, w, to + q * plane, row * 2, rows, (columns + 7) / 8);
    }
}

// N values a row in FP32, as far as `columns` (rounded up to a multiple of 4).
template <int N>
__device__ __forceinline__ void put_floats(unsigned char* scratch, const float* v, float* to, int64_t row, int rows,
                                           int columns) {
    uint4 w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = as_piece(v + 4 * i);
    put_rows<N / 4>(scratch, w, to, row * 4, rows, (columns + 3) / 4);
}

// N columns of a result's rows, `columns` of which exist. Rows start at multiples of 16 bytes (`vector`), else in 16 bits at
// words where they are of even length, or anywhere.
template <int N, typename T>
__device__ __forceinline__ void put_result(unsigned char* scratch, const float (&v)[N], T* to, int64_t row, int rows, int columns,
                                           bool vector) {
    const int lane = threadIdx.x & 31;
    if (columns <= 0) return;
    if (vector) {
        if constexpr (sizeof(T) == 2) {
            uint4 w[N / 8];
#pragma unroll
            for (int i = 0; i < N / 8; ++i) w[i] = pack8(v + 8 * i);
            put_rows<N / 8>(scratch, w, to, row * 2, rows, columns / 8);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 32)
                if (columns > i) put_floats<32>(scratch, v + i, to + i, row, rows, columns - i);
        }
        return;
    }
#pragma unroll
    for (int part = 0; part < N; part += 32) {  // a row of 33 words: lanes side by side in a row or in a column
        float* cells = reinterpret_cast<float*>(scratch);
#pragma unroll
        for (int turn = 0; turn < 32; turn += 16) {
            __syncwarp();
            if (lane >= turn && lane < turn + 16)
#pragma unroll
                for (int i = 0; i < 32; ++i) cells[(lane - turn) * 33 + i] = v[part + i];
            __syncwarp();
            if (sizeof(T) == 2 && row % 2 == 0) {  // two rows at a time
                const int c = lane % 16 * 2;
                for (int r = lane / 16; r < 16 && turn + r < rows; r += 2)
                    if (part + c < columns)
                        *reinterpret_cast<uint32_t*>(to + (turn + r) * row + part + c) =
                            pack_bf16(cells[r * 33 + c], cells[r * 33 + c + 1]);
                continue;
            }
            for (int r = 0; r < 16 && turn + r < rows; ++r)
                if (part + lane < columns) store1(to + (turn + r) * row + part + lane, cells[r * 33 + lane]);
        }
    }
}

// W: columns of the sums that a warp takes at a time (kUp: half of them a's, half b's).
template <int KIND, int P, int W, bool PAIR>
__global__ void __launch_bounds__(Shape<KIND, P>::kThreads, 1) feed_kernel(const __grid_constant__ Maps maps, const Args g) {
    using S = Shape<KIND, P>;
    using G = Group<PAIR>;
    constexpr bool kColumnsA = KIND == kWeights, kColumnsB = KIND == kHidden || KIND == kInput || KIND == kWeights;
    extern __shared__ unsigned char raw[];
    const uint32_t ring = (su32(raw) + 1023u) & ~1023u;
    __shared__ Ctrl ctl;
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = G::rank();
    const int first_turn = PAIR ? int(blockIdx.x) / 2 : int(blockIdx.x), turns = PAIR ? int(gridDim.x) / 2 : int(gridDim.x);
    const int columns = PAIR ? g.bn / 2 : g.bn;  // of B in this block
    const uint32_t tile_b = uint32_t(columns) * 128u, tile_a = g.tile_a, slot_bytes = P * (tile_a + tile_b);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kMostSlots; ++i) {
            mbar_init(&ctl.full[i], 1);
            mbar_init(&ctl.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl.sums[i], 1);
            mbar_init(&ctl.taken[i], PAIR ? 2 * S::kWarps : S::kWarps);
        }
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == S::kWarps + 1) G::alloc(&ctl.tmem);
    tc_fence_before();
    G::sync();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    dependents_may_start();  // with this block's TMEM in hand: they take theirs and hold it until this kernel ends
    // down in 16 bits: its weights were there before the kernel ahead, so that the first of them come while that one ends
    constexpr bool kAhead = KIND == kDown && P == 1 && !PAIR;
    int ahead = 0;
    if (kAhead && warp == S::kWarps && lane == 0 && first_turn < turns_of(g)) {
        const Place p = place_of(g, first_turn);
        const bool pb = g.problem[0].b_panels != 0;
        for (; ahead < min(g.slots, p.to - p.from); ++ahead) {
            const int k = p.from + ahead;
            mbar_expect_tx(&ctl.full[ahead], slot_bytes);
            G::load(ring + uint32_t(ahead) * slot_bytes, &maps.b[0], su32(&ctl.full[ahead]), pb ? 0 : k * kK, p.n * g.bn,
                    pb ? k : 0, 0);
        }
    }
    wait_for_the_kernel_ahead();

    if (warp == S::kWarps) {
        if (lane == 0) {
            const uint32_t first_full = G::first(ctl.full);
            int slot = 0;
            uint32_t phase = 0, armed = 0;  // armed: slots with a copy that nobody may have waited for
            bool ok = true;
            for (int t = first_turn; t < turns_of(g) && ok; t += turns) {
                const Place p = place_of(g, t);
                const Problem& q = g.problem[p.problem];
                if (!wanted<KIND>(q)) continue;
                const int m0 = p.m * g.tile_m + int(rank) * kM, n0 = p.n * (KIND == kUp ? g.bn / 2 : g.bn) +
                                                                     (PAIR && KIND != kUp ? int(rank) * columns : 0);
                const bool pa = q.a_panels != 0, pb = q.b_panels != 0;
                for (int half = 0; half < (KIND == kInput ? 2 : 1) && ok; ++half) {  // kInput: da and gate, db and up
                    const int base = half * g.turn, from = max(p.from, base);
                    const int to = KIND == kInput && half == 0 ? min(p.to, g.turn) : p.to;
                    const CUtensorMap *ma = &maps.a[half > 0 ? 1 : q.a], *mb = &maps.b[half > 0 ? 1 : q.b];
                    const CUtensorMap* up = &maps.b[KIND == kUp && PAIR ? rank : 1];
                    for (int step = from; step < to; ++step) {
                        if (!mbar_wait(&ctl.empty[slot], phase ^ 1u, abort)) {
                            ok = false;
                            break;
                        }
                        const uint32_t bar = first_full + uint32_t(slot) * 8u;
                        const bool given = kAhead && ahead > 0;  // B is there, or on its way
                        if (given) --ahead;
                        else if (!PAIR || rank == 0) mbar_expect_tx(&ctl.full[slot], PAIR ? 2 * slot_bytes : slot_bytes);
                        armed |= 1u << slot;
                        const uint32_t at = ring + uint32_t(slot) * slot_bytes;
                        const int k = step - base, k0 = k * kK;
#pragma unroll
                        for (int i = 0; i < P; ++i) {
                            const uint32_t a = at + P * tile_b + uint32_t(i) * tile_a, b = at + uint32_t(i) * tile_b;
                            if (kColumnsA) {
                                if (pa) {
                                    G::load(a, ma, bar, 0, k0, m0 / 64, i);
                                } else {
                                    G::load(a, ma, bar, m0, k0, 0, i);
                                    G::load(a + kPanel, ma, bar, m0 + 64, k0, 0, i);
                                }
                            } else {
                                G::load(a, ma, bar, pa ? 0 : k0, m0, pa ? k : 0, i);
                            }
                            if (KIND == kUp && PAIR) {
                                G::load(b, up, bar, pb ? 0 : k0, n0, pb ? k : 0, i);
                            } else if (KIND == kUp) {
                                G::load(b, mb, bar, pb ? 0 : k0, n0, pb ? k : 0, i);
                                G::load(b + tile_b / 2, up, bar, pb ? 0 : k0, n0, pb ? k : 0, i);
                            } else if (kColumnsB) {
                                if (pb)
                                    G::load(b, mb, bar, 0, k0, n0 / 64, i);
                                else
                                    for (int c = 0; c < columns / 64; ++c)
                                        G::load(b + c * kPanel, mb, bar, n0 + 64 * c, k0, 0, i);
                            } else if (!given) {
                                G::load(b, mb, bar, pb ? 0 : k0, n0, pb ? k : 0, i);
                            }
                        }
                        if (++slot == g.slots) {
                            slot = 0;
                            phase ^= 1u;
                        }
                    }
                }
            }
            // the block ends after the copies in flight and, where all went well, after the products that read them
            for (int i = 0; i < g.slots; ++i) {
                const uint32_t uses = phase + (i < slot ? 1u : 0u);  // parity of the number of uses of slot i
                if (!(armed >> i & 1u)) continue;
                if (ok) ok = mbar_wait(&ctl.empty[i], (uses ^ 1u) & 1u, abort);
                if (!ok && rank == 0) mbar_wait(&ctl.full[i], (uses ^ 1u) & 1u, abort, true);
            }
            // copies whose barrier the other block has not armed or does not look at, or that came ahead of a step not taken
            if (!ok && (PAIR || ahead > 0))
                for (const unsigned long long t0 = global_ns(); global_ns() - t0 < 1000000ull;) {
                }
        }
    } else if (warp > S::kWarps && rank == 0) {
        const uint32_t base = uniform(tmem), first = uniform(ring), bytes = uniform(slot_bytes), b_bytes = uniform(tile_b),
                       a_bytes = uniform(tile_a);
        const int slots = uniform(g.slots), bn = uniform(g.bn);
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (kColumnsA ? 1u << 15 : 0u) |
                               (kColumnsB ? 1u << 16 : 0u) | (uint32_t(bn >> 3) << 17) |
                               (uint32_t((PAIR ? 2 * kM : kM) >> 4) << 24);
        constexpr int kStepA = kColumnsA ? 128 : 2, kStepB = kColumnsB ? 128 : 2;
        auto desc = [](uint32_t at, bool columns) {
            return ((at & 0x3FFFFu) >> 4) | (columns ? (kPanel >> 4) << 16 : 1u << 16);
        };
        int slot = 0, unit = 0;
        uint32_t phase = 0;
        bool ok = true, issued = false;
        for (int t = first_turn; t < turns_of(g) && ok; t += turns) {
            const Place p = place_of(g, t);
            if (!wanted<KIND>(g.problem[p.problem])) continue;
            const int from = uniform(p.from), to = uniform(p.to);
            for (int start = from; start < to && ok; ++unit) {
                const int end = P == 1 ? to : min(to, start + kSegment);
                const uint32_t d = base + uint32_t(unit & 1) * 256u;
                ok = warp_wait(&ctl.taken[unit & 1], (uint32_t(unit >> 1) & 1u) ^ 1u, abort);
                for (int step = start; step < end && ok; ++step) {
                    ok = warp_wait(&ctl.full[slot], phase, abort);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t at = first + uint32_t(slot) * bytes;
                    if (elect_one()) {
                        const uint32_t a = desc(at + P * b_bytes, kColumnsA), b = desc(at, kColumnsB);
                        const bool add = step > start;
                        if (P == 1) {
                            mma2<PAIR, kStepA, kStepB>(d, a, b, idesc, add);
                            mma2<PAIR, kStepA, kStepB>(d, a + 2 * kStepA, b + 2 * kStepB, idesc, true);
                        } else {  // the small products first, into sums of their own
                            constexpr int kPa[6] = {2, 1, 0, 1, 0, 0}, kPb[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
                            for (int i = 0; i < 6; ++i) {
                                const uint32_t x = a + kPa[i] * (a_bytes >> 4), y = b + kPb[i] * (b_bytes >> 4);
                                const uint32_t to_sum = i < 5 ? d + 128 : d;
                                mma2<PAIR, kStepA, kStepB>(to_sum, x, y, idesc, add || (i > 0 && i < 5));
                                mma2<PAIR, kStepA, kStepB>(to_sum, x + 2 * kStepA, y + 2 * kStepB, idesc, true);
                            }
                        }
                        G::commit(&ctl.empty[slot]);
                        if (step + 1 == end) G::commit(&ctl.sums[unit & 1]);
                    }
                    issued = true;
                    if (++slot == slots) {
                        slot = 0;
                        phase ^= 1u;
                    }
                }
                start = end;
            }
        }
        if (!ok && issued) {  // the products in flight end before TMEM is freed
            if (elect_one()) G::commit(&ctl.drain);
            warp_wait(&ctl.drain, 0, abort, true);
        }
    } else if (warp < S::kWarps) {
        using T = typename std::conditional<P == 1, __nv_bfloat16, float>::type;
        constexpr int kGroups = S::kWarps / 4, kStep = KIND == kUp ? W / 2 : W;  // kStep: columns of the result a unit
        const int group = warp >> 2, units = g.bn / W;
        unsigned char* scratch = raw + (ring - su32(raw)) + S::kRing + warp * S::kScratch;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        int unit = 0;
        bool ok = true;
        auto wait = [&]() {  // uniform in the warp: TMEM access is .sync.aligned
            const bool got = mbar_wait(&ctl.sums[unit & 1], uint32_t(unit >> 1) & 1u, abort);
            if (!__all_sync(0xffffffffu, got)) {
                *abort = 1;
                return false;
            }
            tc_fence_after();
            return true;
        };
        auto done = [&]() {
            tc_fence_before();
            G::arrive(&ctl.taken[unit & 1]);
            ++unit;
        };
        // the block of 32 rows from row0 on and 16 hidden units from col on, this lane's first piece
        constexpr int kPieces = P == 1 ? 2 : 4;
        auto block_at = [&](int64_t row0, int64_t col) { return ((col / 16 * g.blocks + row0 / 32) * kPieces) * 32 + lane; };
        auto panel_at = [&](int64_t row0, int64_t col, int64_t rows) { return (col / 64 * rows + row0) * 64 + col % 64; };
        // kHidden: factors of 32 columns, those of the next ones on their way while the last ones are stored
        uint4 slopes[2 * kPieces], levels[P == 1 ? 2 * kPieces : 1];
        float2 unit_of[2];
        auto fetch = [&](const void* factor, int64_t row0, int64_t col, int64_t n, uint4* to) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4* p = static_cast<const uint4*>(factor) + block_at(row0, col + 16 * i);
                const bool here = col + 16 * i < n;
#pragma unroll
                for (int e = 0; e < kPieces; ++e) to[i * kPieces + e] = here ? __ldg(p + 32 * e) : make_uint4(0, 0, 0, 0);
            }
        };
        auto fetch_both = [&](int64_t row0, int64_t col, int64_t n) {
            fetch(g.slope, row0, col, n, slopes);
            fetch(g.level, row0, col, n, levels);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                unit_of[i] = col + 16 * i < n ? __ldg(g.unit + (col / 16 + i) * g.blocks * 32 + row0 + lane)
                                              : make_float2(0.0f, 0.0f);
        };
        // float32: one factor after the other
        auto spread = [&](const Problem& q, int64_t row0, int rows, int64_t col, int64_t after, const float* v) {
            __nv_bfloat16* const to[2] = {g.da, g.db};
            const int columns = col < g.panels * 64 ? 32 : 0;
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                float x[32];
                const float* f = reinterpret_cast<const float*>(slopes);
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = f[i] * v[i];
                if (o == 0) fetch(g.level, row0, col, rows > 0 ? q.n : 0, slopes);
                else fetch(g.slope, row0, after, rows > 0 ? q.n : 0, slopes);
                put_planes<P, 32>(scratch, x, to[o] + panel_at(row0, col, q.m), 64, g.plane, rows, columns);
            }
        };
        // What follows the W sums of column `col` and on (kUp: of the hidden units).
        auto finish = [&](const Problem& q, const Place& p, int64_t row0, int rows, int64_t col, float(&v)[W]) {
            if constexpr (KIND == kUp) {
                constexpr int kH = W / 2;
                const int columns = col < g.panels * 64 ? kH : 0;
                uint4 first[kH / 8];
                float h[P == 3 ? kH : 8];
#pragma unroll
                for (int i = 0; i < kH; ++i) {
                    float level, slope;
                    activate<P == 3>(g.act, v[i], level, slope);
                    h[P == 3 ? i : i % 8] = level * v[kH + i];
                    v[i] = level;
                    v[kH + i] *= slope;
                    if (P == 1 && i % 8 == 7) first[i / 8] = pack8(h);
                }
                const int64_t at = panel_at(row0, col, q.m);
                if constexpr (P == 1)
                    put_rows<kH / 8>(scratch, first, g.h + at, 128, rows, columns / 8);
                else
                    put_planes<P, kH>(scratch, h, g.h + at, 64, g.plane, rows, columns);
                if (g.slope != nullptr && col < q.n && rows > 0) {
                    uint4 *slope = static_cast<uint4*>(g.slope) + block_at(row0, col),
                          *level = static_cast<uint4*>(g.level) + block_at(row0, col);
                    if constexpr (P == 1) {
                        uint4 w[2];
                        float2 unit;
                        pack_halves(v + kH, w, unit.x);
                        slope[0] = w[0], slope[32] = w[1];
                        pack_halves(v, w, unit.y);
                        level[0] = w[0], level[32] = w[1];
                        g.unit[col / 16 * g.blocks * 32 + row0 + lane] = unit;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            slope[32 * i] = as_piece(v + kH + 4 * i);
                            level[32 * i] = as_piece(v + 4 * i);
                        }
                    }
                }
            } else if constexpr (KIND != kHidden) {
                const int columns = int(max(int64_t(0), min(int64_t(W), q.n - col)));
                if (p.part >= 0)
                    put_result<W>(scratch, v,
                                  g.part + (int64_t(p.part) * g.tile_m + rank * kM + (warp & 3) * 32) * g.bn +
                                      (col - int64_t(p.n) * g.bn),
                                  g.bn, rows, W, true);
                else
                    put_result<W>(scratch, v, static_cast<T*>(q.out) + row0 * q.n + col, q.n, rows, columns, q.n % 8 == 0);
            }
        };
        for (int t = first_turn; t < turns_of(g) && ok; t += turns) {
            const Place p = place_of(g, t);
            const Problem& q = g.problem[p.problem];
            if (!wanted<KIND>(q)) continue;
            const int64_t row0 = int64_t(p.m) * g.tile_m + rank * kM + (warp & 3) * 32,
                          n0 = int64_t(p.n) * (KIND == kUp ? g.bn / 2 : g.bn);
            const int rows = int(max(int64_t(0), min(int64_t(32), q.m - row0)));
            if constexpr (KIND == kHidden) {
                if constexpr (P == 1) {
                    if (group < units) fetch_both(row0, n0 + group * kStep, rows > 0 ? q.n : 0);
                } else {
                    fetch(g.slope, row0, n0 + group * kStep, rows > 0 ? q.n : 0, slopes);
                }
            }
            if (KIND == kUp && p.n + 1 == q.n_tiles)  // what the last tile leaves of the last panel
                for (int64_t col = n0 + g.bn / 2 + group * 16; col < g.panels * 64; col += kGroups * 16) {
                    float v[16] = {};
                    put_planes<P, 16>(scratch, v, g.h + panel_at(row0, col, q.m), 64, g.plane, rows, 16);
                }
            if (p.from >= p.to) {  // a split without a share: sums of zero
                float v[W] = {};
                for (int u = group; u < units; u += kGroups) finish(q, p, row0, rows, n0 + u * kStep, v);
                continue;
            }
            if constexpr (P == 1) {
                if (!(ok = wait())) break;
                const uint32_t at = tmem + lanes + uint32_t(unit & 1) * 256u;
                if (group >= units) done();
                for (int u = group; u < units; u += kGroups) {
                    const bool last = u + kGroups >= units;
                    if constexpr (KIND == kHidden) {
                        const int64_t col = n0 + u * 32;
                        const int columns = col < g.panels * 64 ? 32 : 0;
                        uint4 da[4], db[4];
                        const uint32_t *s = reinterpret_cast<const uint32_t*>(slopes),
                                       *l = reinterpret_cast<const uint32_t*>(levels);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float v[16], x[16], y[16];
                            tmem_load16(at + u * 32 + j * 16, v);
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                const float2 f = unpack_half(s[j * 8 + i / 2]), h = unpack_half(l[j * 8 + i / 2]);
                                x[i] = v[i] * (f.x * unit_of[j].x), x[i + 1] = v[i + 1] * (f.y * unit_of[j].x);
                                y[i] = v[i] * (h.x * unit_of[j].y), y[i + 1] = v[i + 1] * (h.y * unit_of[j].y);
                            }
                            da[2 * j] = pack8(x), da[2 * j + 1] = pack8(x + 8);
                            db[2 * j] = pack8(y), db[2 * j + 1] = pack8(y + 8);
                        }
                        if (last) done();
                        else fetch_both(row0, col + kGroups * 32, rows > 0 ? q.n : 0);
                        const int64_t to = panel_at(row0, col, q.m);
                        put_rows<4>(scratch, da, g.da + to, 128, rows, columns / 8);
                        put_rows<4>(scratch, db, g.db + to, 128, rows, columns / 8);
                    } else {
                        float v[W];
                        if constexpr (KIND == kUp) {
                            tmem_load(at + u * kStep, reinterpret_cast<float(&)[W / 2]>(v[0]));
                            tmem_load(at + g.bn / 2 + u * kStep, reinterpret_cast<float(&)[W / 2]>(v[W / 2]));
                        } else {
                            tmem_load(at + u * kStep, v);
                        }
                        if (last) done();
                        finish(q, p, row0, rows, n0 + u * kStep, v);
                    }
                }
            } else {
                constexpr int kUnits = 128 / W / kGroups > 0 ? 128 / W / kGroups : 1;  // at most: bn is up to 128
                float sum[kUnits][W] = {};
                for (int start = p.from; start < p.to; start += kSegment) {
                    if (!(ok = wait())) break;
                    const uint32_t at = tmem + lanes + uint32_t(unit & 1) * 256u;
#pragma unroll
                    for (int u = 0; u < kUnits; ++u) {
                        if (KIND != kHidden && group + u * kGroups >= units) break;
#pragma unroll
                        for (int j = 0; j < W; j += 16) {
                            const int col = (group + u * kGroups) * kStep +
                                            (KIND == kUp && j >= W / 2 ? g.bn / 2 + j - W / 2 : j);
                            float big[16], small[16];
                            tmem_load16(at + col, big);
                            tmem_load16(at + 128 + col, small);
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum[u][j + i] += big[i] + small[i];
                        }
                    }
                    done();
                }
                if (!ok) break;
#pragma unroll
                for (int u = 0; u < kUnits; ++u) {
                    if (KIND != kHidden && group + u * kGroups >= units) break;
                    const int64_t col = n0 + (group + u * kGroups) * kStep;
                    if constexpr (KIND == kHidden)
                        spread(q, row0, rows, col, u + 1 < kUnits ? col + kGroups * kStep : q.n, sum[u]);
                    else
                        finish(q, p, row0, rows, col, sum[u]);
                }
            }
        }
    }

    tc_fence_before();
    G::sync();
    if (warp == S::kWarps + 1) G::free(tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(g.flags, FMD_FLAG_WAIT_TIMEOUT);
}

// ------------------------------------------------------------------- few rows in float32

// A few rows in float32 without planes, whose making moves four times the weights' bytes: on the FP32 cores. A block takes R
// rows of x and J rows of weights (GATED: J / 2 units, their gate and up rows) through the inner index in chunks of 256, which
// lie in shared memory, one in use and one on its way; each of its eight warps takes 32 of a chunk, all R x J sums, a lane
// 4 x C of them (C = J R / 128): 4 + C vectors of shared memory for 16 C products. The warps' sums are added up at the end.
// 33 rows of 512 x 1,365: 13.7 and 13.5 us, of which reading the weights, 8.4 MB, would be one each: start, end, and chunks
// that wait for memory by turns.
constexpr int kFewThreads = 256, kFewChunk = 256, kFewLd = kFewChunk + 4;

struct Few {
    const float *x, *w0, *w1;  // w1: up
    float* out;
    int64_t x_row, w0_row, w1_row, out_row;
    int32_t rows, inner, units, act;
    bool vector_x, vector_w;  // rows start at multiples of 16 bytes, and the inner size is one of four values
};

template <int R, int J>
struct FewShape {
    static constexpr int kRowGroups = R / 4, kColumnGroups = 32 / kRowGroups, kC = J / kColumnGroups;
    static constexpr int kStage = (R + J) * kFewLd;  // values of a chunk
    static constexpr size_t kChunks = size_t(2) * kStage * 4, kSums = size_t(8) * R * J * 4;
    static constexpr size_t kBytes = kChunks > kSums ? kChunks : kSums;
};

// Four bytes, or sixteen, to shared memory; zeros where there are none.
__device__ __forceinline__ void copy4(float* to, const float* from, bool here) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(su32(to)), "l"(from), "r"(here ? 4 : 0) : "memory");
}

__device__ __forceinline__ void copy16(float* to, const float* from, bool here) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(su32(to)), "l"(from), "r"(here ? 16 : 0) : "memory");
}

// A chunk of `count` rows, row r at row_of(r): sixteen bytes a thread where rows start at multiples of them.
template <typename RowOf>
__device__ __forceinline__ void copy_rows(float* to, int count, int k0, int inner, bool vector, RowOf row_of) {
    if (vector) {
        const int k = k0 + int(threadIdx.x) % 64 * 4;
        const bool here = k < inner;
#pragma unroll 4
        for (int r = int(threadIdx.x) / 64; r < count; r += 4)
            copy16(to + r * kFewLd + int(threadIdx.x) % 64 * 4, row_of(r) + (here ? k : 0), here);
    } else {
        const int k = k0 + int(threadIdx.x);
        const bool here = k < inner;
#pragma unroll 8
        for (int r = 0; r < count; ++r) copy4(to + r * kFewLd + threadIdx.x, row_of(r) + (here ? k : 0), here);
    }
}

template <int R, int J, bool GATED>
__global__ void __launch_bounds__(kFewThreads) few_kernel(const Few f) {
    using S = FewShape<R, J>;
    constexpr int kUnits = GATED ? J / 2 : J;
    extern __shared__ __align__(16) float few_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rg = lane % S::kRowGroups, cg = lane / S::kRowGroups;
    const int unit0 = int(blockIdx.x) * kUnits, row0 = int(blockIdx.y) * R, chunks = (f.inner + kFewChunk - 1) / kFewChunk;
    const int rows = min(R, f.rows - row0);
    auto load = [&](int chunk) {
        float *x = few_smem + chunk % 2 * S::kStage, *w = x + R * kFewLd;
        copy_rows(w, J, chunk * kFewChunk, f.inner, f.vector_w, [&](int j) {
            const int unit = min(unit0 + j % kUnits, f.units - 1);  // units behind the last one are computed and dropped
            return GATED && j >= kUnits ? f.w1 + unit * f.w1_row : f.w0 + unit * f.w0_row;
        });
        copy_rows(x, rows, chunk * kFewChunk, f.inner, f.vector_x, [&](int r) { return f.x + (row0 + r) * f.x_row; });
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float acc[4][S::kC] = {};
    load(0);
    for (int chunk = 0; chunk < chunks; ++chunk) {
        if (chunk + 1 < chunks) {
            load(chunk + 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        const float *x = few_smem + chunk % 2 * S::kStage, *w = x + R * kFewLd;
#pragma unroll 2
        for (int e = 0; e < 32; e += 4) {
            float4 a[4], b[S::kC];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a[i] = *reinterpret_cast<const float4*>(x + (rg + S::kRowGroups * i) * kFewLd + warp * 32 + e);
#pragma unroll
            for (int c = 0; c < S::kC; ++c)
                b[c] = *reinterpret_cast<const float4*>(w + (cg + S::kColumnGroups * c) * kFewLd + warp * 32 + e);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < S::kC; ++c) {
                    acc[i][c] = fmaf(a[i].x, b[c].x, acc[i][c]);
                    acc[i][c] = fmaf(a[i].y, b[c].y, acc[i][c]);
                    acc[i][c] = fmaf(a[i].z, b[c].z, acc[i][c]);
                    acc[i][c] = fmaf(a[i].w, b[c].w, acc[i][c]);
                }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < S::kC; ++c)
            few_smem[(warp * R + rg + S::kRowGroups * i) * J + cg + S::kColumnGroups * c] = acc[i][c];
    __syncthreads();
    for (int i = threadIdx.x; i < R * kUnits; i += kFewThreads) {
        const int r = i / kUnits, u = i % kUnits, unit = unit0 + u;
        if (row0 + r >= f.rows || unit >= f.units) continue;
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            a += few_smem[(q * R + r) * J + u];
            if (GATED) b += few_smem[(q * R + r) * J + kUnits + u];
        }
        if (GATED) {
            float level, slope;
            activate<true>(f.act, a, level, slope);
            a = level * b;
        }
        f.out[(row0 + r) * f.out_row + unit] = a;
    }
}

template <int R, int J, bool GATED>
fmd_status launch_few(const Few& f, cudaStream_t s) {
    constexpr size_t bytes = FewShape<R, J>::kBytes;
    const fmd_status st = grant_dynamic_smem((const void*)few_kernel<R, J, GATED>, bytes);
    if (st != FMD_OK) return st;
    const int units = GATED ? J / 2 : J;
    few_kernel<R, J, GATED><<<dim3(unsigned((f.units + units - 1) / units), unsigned((f.rows + R - 1) / R)), kFewThreads, bytes,
                             s>>>(f);
    return check_launch();
}

// As many rows of weights a block, of sixteen at most, as leave a block for every SM.
template <int R, bool GATED>
fmd_status launch_few(const Few& f, cudaStream_t s) {
    const int64_t rows = int64_t(f.units) * (GATED ? 2 : 1);
    if (rows >= 16 * kNumSMs) return launch_few<R, 16, GATED>(f, s);
    if constexpr (R >= 32)
        if (rows < 8 * kNumSMs) return launch_few<R, 4, GATED>(f, s);
    return launch_few<R, 8, GATED>(f, s);
}

template <bool GATED>
fmd_status launch_few(const Few& f, cudaStream_t s) {
    return f.rows <= 16 ? launch_few<16, GATED>(f, s) : launch_few<32, GATED>(f, s);
}

// ------------------------------------------------------------------- planes and sums of splits

// float32 [rows, columns] as three planes [3][rows][row] of bfloat16, up to four arrays (blockIdx.y).
struct SplitArgs {
    const float* x[4];
    __nv_bfloat16* to[4];
    int64_t rows[4], from_row[4], row[4];
    int32_t columns[4];
};

__global__ void __launch_bounds__(256) split_kernel(const SplitArgs a) {
    dependents_may_start();
    const int t = blockIdx.y, per = int(a.row[t] / 8), n = a.columns[t];
    const int64_t all = a.rows[t] * per, plane = a.rows[t] * a.row[t];
    const bool vector = a.from_row[t] % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x[t]) & 15u) == 0;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / per;
        const int c = int(i - row * per) * 8;
        const float* x = a.x[t] + row * a.from_row[t] + c;
        float v[8];
        if (vector && c + 8 <= n) {
            const float4 p = ldg4(x), q = ldg4(x + 4);
            v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w, v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < n ? x[e] : 0.0f;
        }
        uint4* to = reinterpret_cast<uint4*>(a.to[t] + row * a.row[t] + c);
        to[0] = first_plane8(v);
        to[plane / 8] = next_plane8(v);
        to[plane / 4] = next_plane8(v);
    }
}

// Matrices of 16-bit values with any strides, up to four (blockIdx.y), as rows that TMA reads: `row` values apart, a multiple
// of 8, with zeros behind their columns. 27,341 rows of 1,812: 49 us, 4.1 TB/s.
struct PadArgs {
    fmd_padded x[4];
};

__global__ void __launch_bounds__(256) pad_kernel(const PadArgs a) {
    const fmd_padded& x = a.x[blockIdx.y];
    const int per = int(x.to_row / 8);
    const int64_t all = x.rows * per;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / per;
        const int c = int(i - row * per) * 8;
        const uint16_t* from = static_cast<const uint16_t*>(x.from) + row * x.from_row + c * x.from_column;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = c + e < x.columns ? __ldg(from + e * x.from_column) : 0u;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(x.to) + row * x.to_row + c) =
            make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
}

// The tiles that were shared out: the sums of their shares, in their order. blockIdx.y: the tile; a thread per four columns.
template <typename T>
__global__ void __launch_bounds__(256) add_kernel(const Args g) {
    dependents_may_start();
    wait_for_the_kernel_ahead();
    const Place p = place_of(g, g.whole + int(blockIdx.y));
    const Problem& q = g.problem[p.problem];
    if (q.out == nullptr) return;
    const int per = g.bn / 4, at = int(blockIdx.x) * 256 + int(threadIdx.x), row = at / per, col = (at - row * per) * 4;
    if (row >= g.tile_m) return;
    const float* part = g.part + (int64_t(blockIdx.y) * g.splits * g.tile_m + row) * g.bn + col;
    float4 sum = f4_zero();
#pragma unroll 4
    for (int z = 0; z < g.splits; ++z) sum = f4_add(sum, *reinterpret_cast<const float4*>(part + int64_t(z) * g.tile_m * g.bn));
    const int64_t m = int64_t(p.m) * g.tile_m + row, n = int64_t(p.n) * g.bn + col;
    if (m >= q.m) return;
    T* out = static_cast<T*>(q.out) + m * q.n + n;
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
    if (q.n % 4 == 0 && n < q.n) {
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
        else
            st4(out, sum);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < q.n) store1(out + e, v[e]);
    }
}

// ------------------------------------------------------------------- host

// A matrix of bfloat16 as TMA reads it: `planes` of [rows, columns] with rows `row` apart, or (panels > 0) in panels of 64
// columns, [planes][panels][rows][64].
struct Matrix {
    const void* data;
    int64_t rows, columns, row;
    int planes, panels;
    // Read panel by panel, so that one copy takes several: any matrix of whole panels. Else a copy is at most 64 columns,
    // and what lies behind the last column is filled with zeros.
    bool by_panels() const { return panels > 0 || columns % 64 == 0; }
};

fmd_status encode(CUtensorMap* map, const Matrix& x, int box_rows, int box_panels) {
    const DriverCalls& drv = driver_calls();
    const int64_t row = x.panels > 0 ? 64 : x.rows == 1 ? (x.columns + 7) / 8 * 8 : x.row;
    const int64_t panel = x.panels > 0 ? 64 * x.rows : 64, count = x.panels > 0 ? x.panels : x.columns / 64;
    const bool panels = x.by_panels();
    const cuuint64_t dims[4] = {cuuint64_t(panels ? 64 : x.columns), cuuint64_t(x.rows), cuuint64_t(panels ? count : 1),
                                cuuint64_t(x.planes)};
    const cuuint64_t strides[3] = {cuuint64_t(row) * 2, cuuint64_t(panels ? panel : row * x.rows) * 2,
                                   cuuint64_t(x.panels > 0 ? panel * count : row * x.rows) * 2};
    const cuuint32_t box[4] = {64, cuuint32_t(box_rows), cuuint32_t(panels ? box_panels : 1), 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = drv.encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(x.data), dims, strides, box,
                                  step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FMD_OK : record_error_text(FMD_ERR_CUDA, "cuTensorMapEncodeTiled failed, CUresult", r);
}

int64_t round_up(int64_t v, int64_t unit) { return (v + unit - 1) / unit * unit; }

// Rows up to which float32 goes without planes where no backward pass follows: two blocks of 32 where the weights are small,
// else one. us on the FP32 cores and by planes, width x hidden: 256 x 512, 32 rows 10 and 22, 64 rows 11 and 22; 512 x 1,365,
// 32 rows 19 and 29, 64 rows 31 and 29 (with two launches less); 1,024 x 4,096, 16 rows 38 and 62, 32 rows 64 and 61, 64 rows
// 125 and 61; 4,096 x 11,000, 1 row 217 and 440, 32 rows 363 and 439, 64 rows 707 and 449.
int64_t few_limit(int64_t width, int64_t hidden) { return width * hidden <= (1 << 20) ? 64 : 32; }

// How a launch runs: rows (256: pairs of blocks) and columns of a tile, the tiles that are not shared out, shares of the
// others along the inner index.
struct Plan {
    int tile_m, bn, tiles, whole, splits;
    size_t bytes() const { return splits > 1 ? size_t(tiles - whole) * splits * tile_m * bn * sizeof(float) : 0; }
};

// The time of a launch in steps of 128 x 256 x 64, about 0.4 us each: rounds of blocks, each its tile's steps and, besides,
// about six for its start and end. Narrower tiles wait for their operands and barriers all the same (steps of 64 columns:
// 0.39 us, of 256: 0.45); a pair's step of 256 x 256 takes 0.75 of one. Tiles are shared out along the inner index where that
// ends sooner: all of them, or those of the last round, which do not fill the GPU; the shares' sums are written and read
// again. unit: bn is a multiple of it (panels of 64 columns where the rows of B are the inner index; else any 32, so that few
// rows' weights are read by all SMs alike).
Plan plan(const int64_t* m, const int64_t* n, int problems, int64_t steps, int planes, int unit, bool can_split) {
    Plan best{kM, 128, 0, 0, 1};
    double least = 1e300;
    auto look = [&](int tile_m, int bn) {
        int64_t tiles = 0;
        for (int i = 0; i < problems; ++i) tiles += ((m[i] + tile_m - 1) / tile_m) * ((n[i] + bn - 1) / bn);
        const int64_t places = kNumSMs * kM / tile_m;
        const double step = planes == 3 ? 1.0 + 4.0 * bn / 256.0 : tile_m > kM ? 0.75 : 0.7 + 0.3 * bn / 256.0;
        for (int full = 0; full < (can_split && tiles > places ? 2 : 1); ++full) {
            const int64_t whole = full ? tiles / places * places : 0, rest = tiles - whole;
            const double before = whole / places * (steps * step + 6.0);
            // shares beyond four rounds of blocks even nothing out any more
            for (int splits = 1; splits <= (can_split ? 64 : 1) &&
                                 (splits == 1 || (4 * splits <= steps && rest * (splits - 1) < 4 * places)); ++splits) {
                const int64_t rounds = (rest * splits + places - 1) / places;
                const double moved = (2.0 * splits + 1.0) * rest * tile_m * bn * 4.0;
                const double sums = splits > 1 ? 10.0 + moved / 6.5e6 / 0.4 : 0.0;
                const double time = before + rounds * (((steps + splits - 1) / splits) * step + 6.0) + sums;
                if (time < least) {
                    least = time;
                    best = Plan{tile_m, bn, int(tiles), int(splits > 1 ? whole : tiles), splits};
                }
            }
        }
    };
    for (int bn = unit; bn <= (planes == 1 ? 256 : 128); bn += unit) look(kM, bn);
    int64_t most = 0;
    for (int i = 0; i < problems; ++i) most = m[i] > most ? m[i] : most;
    if (planes == 1 && most > kM) look(2 * kM, 256);
    return best;
}

struct Sizes {
    int64_t rows, width, hidden, out;
    int planes;  // 3: float32
    int64_t hidden_row, width_row, out_row;  // of planes of what is given
    int panels, blocks;                      // of h, da and db; of 32 rows, of the factors
    size_t values() const { return size_t(rows) * panels * 64; }
};

// early: behind another kernel of the same call, which it may overlap. Not for pairs of blocks: placed as SMs become free they
// took 4 % longer over many tiles (feed_frames_bf16 2018 -> 2095 us), and few are left to gain.
template <int KIND, int P, int W, bool PAIR>
fmd_status launch(const Maps& maps, Args& g, bool early, cudaStream_t s) {
    using S = Shape<KIND, P>;
    const fmd_status st = grant_dynamic_smem((const void*)feed_kernel<KIND, P, W, PAIR>, S::kBytes, true);
    if (st != FMD_OK) return st;
    const int slots = int(S::kRing / (P * (g.tile_a + (PAIR ? g.bn / 2 : g.bn) * 128)));
    g.slots = slots < kMostSlots ? slots : kMostSlots;
    const int64_t turns = g.whole + int64_t(g.tiles - g.whole) * g.splits, places = PAIR ? kNumSMs / 2 : kNumSMs;
    const unsigned blocks = unsigned((turns < places ? turns : places) * (PAIR ? 2 : 1));
    cudaLaunchAttribute attributes[2]{};
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(unsigned(S::kThreads));
    config.dynamicSmemBytes = S::kBytes;
    config.stream = s;
    config.attrs = attributes;
    if (early && !PAIR) {
        attributes[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (PAIR) {
        attributes[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attributes[config.numAttrs++].val.clusterDim = {2, 1, 1};
    }
    const cudaError_t err = cudaLaunchKernelEx(&config, feed_kernel<KIND, P, W, PAIR>, maps, g);
    return err == cudaSuccess ? check_launch() : record_cuda_error(err);
}

template <int KIND>
fmd_status run(int planes, const Matrix* a, const Matrix* b, int operands, Args& g, const Plan& p, bool early, cudaStream_t s) {
    Maps maps{};
    const bool columns_a = KIND == kWeights, columns_b = KIND == kHidden || KIND == kInput || KIND == kWeights;
    // Few rows: the slots hold these alone, so that more of the weights are on their way (up of 8 rows, 4,096 x 11,000:
    // 57 -> 36 us). The products read on to 128 rows, into what follows in shared memory, for rows of the result that
    // nobody takes.
    const int rows = g.problem[0].m < kM ? int(round_up(g.problem[0].m, 8)) : kM;
    g.tile_a = columns_a ? int(kTileA) : rows * kK * 2;
    for (int i = 0; i < operands; ++i) {
        fmd_status st = FMD_OK;
        if (a[i].data != nullptr) st = encode(&maps.a[i], a[i], columns_a ? kK : rows, columns_a ? kM / 64 : 1);
        if (st == FMD_OK && b[i].data != nullptr)
            st = encode(&maps.b[i], b[i], columns_b ? kK : KIND == kUp || p.tile_m > kM ? p.bn / 2 : p.bn,
                        columns_b ? (p.tile_m > kM ? p.bn / 2 : p.bn) / 64 : 1);
        if (st != FMD_OK) return st;
    }
    g.tile_m = p.tile_m;
    g.bn = p.bn;
    g.tiles = p.tiles;
    g.whole = p.whole;
    g.splits = p.splits;
    for (int i = 0; i < g.problems; ++i) {
        Problem& q = g.problem[i];
        const int columns = KIND == kUp ? p.bn / 2 : p.bn;
        q.a_panels = a[q.a].by_panels();
        q.b_panels = b[q.b].by_panels();
        q.m_tiles = int((q.m + p.tile_m - 1) / p.tile_m);
        q.n_tiles = int((q.n + columns - 1) / columns);
    }
    constexpr int kWide = KIND == kUp || KIND == kHidden ? 32 : 64;
    const fmd_status st = planes == 3       ? launch<KIND, 3, 32, false>(maps, g, early, s)
                          : p.tile_m > kM   ? launch<KIND, 1, kWide, true>(maps, g, early, s)
                          : g.bn == 256     ? launch<KIND, 1, kWide, false>(maps, g, early, s)
                                            : launch<KIND, 1, 32, false>(maps, g, early, s);
    if (st != FMD_OK || p.splits == 1) return st;
    const dim3 grid(unsigned((p.tile_m * p.bn / 4 + 255) / 256), unsigned(p.tiles - p.whole));
    return launch_early(planes == 1 ? add_kernel<__nv_bfloat16> : add_kernel<float>, grid, 256, 0, s, g);
}

int64_t steps_of(int64_t k) { return (k + kK - 1) / kK; }

Plan down_plan(const Sizes& z) { return plan(&z.rows, &z.out, 1, steps_of(z.hidden), z.planes, 32, true); }
Plan input_plan(const Sizes& z) { return plan(&z.rows, &z.width, 1, 2 * steps_of(z.hidden), z.planes, 64, true); }
Plan weights_plan(const Sizes& z) {
    const int64_t m[3] = {z.hidden, z.hidden, z.out}, n[3] = {z.width, z.width, z.hidden};
    return plan(m, n, 3, steps_of(z.rows), z.planes, 64, true);
}

// Arrays in one buffer, each at a multiple of 256 bytes.
struct Layout {
    size_t bytes = 0;
    size_t take(size_t n) {
        const size_t at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    }
};

// What the forward pass keeps for the backward pass: h, the factors, and in float32 the planes of what it was given.
struct Kept {
    size_t h, slope, level, unit, x, gate, up, down, bytes;
};

Kept kept_layout(const Sizes& z, bool factors) {
    Layout at;
    Kept k{};
    k.h = at.take(z.values() * z.planes * 2);
    if (factors) {
        const size_t blocks = size_t(z.blocks) * ((z.hidden + 15) / 16);  // of 32 rows x 16 units
        k.slope = at.take(blocks * 512 * (z.planes == 3 ? 4 : 2));
        k.level = at.take(blocks * 512 * (z.planes == 3 ? 4 : 2));
        if (z.planes == 1) k.unit = at.take(blocks * 32 * sizeof(float2));
    }
    if (z.planes == 3) {
        k.x = at.take(size_t(z.rows) * z.width_row * 6);
        k.gate = at.take(size_t(z.hidden) * z.width_row * 6);
        k.up = at.take(size_t(z.hidden) * z.width_row * 6);
        k.down = at.take(size_t(z.out) * z.hidden_row * 6);
    }
    k.bytes = at.bytes;
    return k;
}

// The backward pass's workspace: da, db, the planes of g, and sums of splits (of one product at a time).
struct Scratch {
    size_t da, db, g, part, bytes;
};

Scratch scratch_layout(const Sizes& z) {
    Layout at;
    Scratch k{};
    const size_t hidden = z.values() * z.planes * 2;
    k.da = at.take(hidden);
    k.db = at.take(hidden);
    if (z.planes == 3) k.g = at.take(size_t(z.rows) * z.out_row * 6);
    const size_t weights = weights_plan(z).bytes(), input = input_plan(z).bytes();
    k.part = at.take(weights > input ? weights : input);
    k.bytes = at.bytes;
    return k;
}

fmd_status check(const fmd_feed_forward& f, Sizes& z) {
    if ((f.type != FMD_F32 && f.type != FMD_BF16) || (f.activation != FMD_FEED_SILU && f.activation != FMD_FEED_GELU) ||
        f.rows < 0 || f.width < 1 || f.hidden < 1 || f.out < 1 || (f.rows > 0 && f.x == nullptr) || f.gate == nullptr ||
        f.up == nullptr || f.down == nullptr || (f.rows > 1 && f.x_row < f.width) ||
        (f.hidden > 1 && (f.gate_row < f.width || f.up_row < f.width)) || (f.out > 1 && f.down_row < f.hidden))
        return FMD_ERR_INVALID_ARGUMENT;
    if (f.rows > (1 << 28) || f.width > (1 << 20) || f.hidden > (1 << 20) || f.out > (1 << 20)) return FMD_ERR_UNSUPPORTED;
    if (f.type == FMD_BF16 &&
        ((f.rows > 0 && !vector_rows(f.x, f.rows > 1 ? f.x_row : 0, 0, 2)) ||
         !vector_rows(f.gate, f.hidden > 1 ? f.gate_row : 0, 0, 2) || !vector_rows(f.up, f.hidden > 1 ? f.up_row : 0, 0, 2) ||
         !vector_rows(f.down, f.out > 1 ? f.down_row : 0, 0, 2)))
        return FMD_ERR_UNSUPPORTED;
    z = Sizes{f.rows, f.width, f.hidden, f.out, f.type == FMD_F32 ? 3 : 1, round_up(f.hidden, 8), round_up(f.width, 8),
              round_up(f.out, 8), int((f.hidden + 63) / 64), int((f.rows + 31) / 32)};
    // tiles are counted in 32 bits
    if (((z.rows + 127) / 128) * ((z.hidden + 63) / 64 + (z.width + 63) / 64 + (z.out + 63) / 64) * 64 > INT32_MAX)
        return FMD_ERR_UNSUPPORTED;
    return FMD_OK;
}

// A few rows: h alone, by rows.
bool few_rows(const Sizes& z, bool keep) {
    return z.planes == 3 && !keep && z.rows > 0 && z.rows <= few_limit(z.width, z.hidden);
}

size_t few_bytes(const Sizes& z) { return (size_t(z.rows) * round_up(z.hidden, 4) * sizeof(float) + 255) / 256 * 256; }

fmd_status run_few(const fmd_feed_forward& f, float* h, float* y, cudaStream_t s) {
    const float *x = static_cast<const float*>(f.x), *gate = static_cast<const float*>(f.gate),
                *up = static_cast<const float*>(f.up), *down = static_cast<const float*>(f.down);
    auto whole = [](const float* p, int64_t row, int64_t inner) { return inner % 4 == 0 && row % 4 == 0 && aligned16(p); };
    const int64_t h_row = round_up(f.hidden, 4);
    const fmd_status st = launch_few<true>(
        Few{x, gate, up, h, f.x_row, f.gate_row, f.up_row, h_row, int32_t(f.rows), f.width, f.hidden, f.activation,
            whole(x, f.rows > 1 ? f.x_row : 0, f.width), whole(gate, f.gate_row, f.width) && whole(up, f.up_row, f.width)}, s);
    if (st != FMD_OK) return st;
    return launch_few<false>(Few{h, down, nullptr, y, h_row, f.down_row, 0, f.out, int32_t(f.rows), f.hidden, f.out, 0,
                                 f.hidden % 4 == 0, whole(down, f.down_row, f.hidden)}, s);
}

fmd_status ready() {
    const DriverCalls& drv = driver_calls();
    if (drv.encode == nullptr || drv.ctx_get_current == nullptr)
        return record_error_text(FMD_ERR_CUDA, "driver entry point cuTensorMapEncodeTiled unavailable", 0);
    return bind_context(drv);
}

void add_split(SplitArgs& a, int& count, const void* x, void* to, int64_t rows, int64_t columns, int64_t from_row,
               int64_t row) {
    a.x[count] = static_cast<const float*>(x);
    a.to[count] = static_cast<__nv_bfloat16*>(to);
    a.rows[count] = rows;
    a.columns[count] = int32_t(columns);
    a.from_row[count] = from_row;
    a.row[count++] = row;
}

fmd_status split(const SplitArgs& a, int count, cudaStream_t s) {
    int64_t most = 0;
    for (int i = 0; i < count; ++i) most = a.rows[i] * (a.row[i] / 8) > most ? a.rows[i] * (a.row[i] / 8) : most;
    split_kernel<<<dim3(unsigned(grid_for(most, 256)), unsigned(count)), 256, 0, s>>>(a);
    return check_launch();
}

// x and the weights as the products read them.
struct Inputs {
    Matrix x, gate, up, down;
};

Inputs inputs_of(const fmd_feed_forward& f, const Sizes& z, const Kept& k, char* kept) {
    if (z.planes == 1)
        return Inputs{{f.x, z.rows, z.width, f.x_row, 1, 0}, {f.gate, z.hidden, z.width, f.gate_row, 1, 0},
                      {f.up, z.hidden, z.width, f.up_row, 1, 0}, {f.down, z.out, z.hidden, f.down_row, 1, 0}};
    return Inputs{{kept + k.x, z.rows, z.width, z.width_row, 3, 0}, {kept + k.gate, z.hidden, z.width, z.width_row, 3, 0},
                  {kept + k.up, z.hidden, z.width, z.width_row, 3, 0}, {kept + k.down, z.out, z.hidden, z.hidden_row, 3, 0}};
}

}  // namespace
}  // namespace fmd

using namespace fmd;

extern "C" {

fmd_status fmd_gated_feed_forward_bytes(const fmd_feed_forward* problem, int32_t keep, size_t* kept, size_t* forward,
                                        size_t* backward) {
    Sizes z;
    if (problem == nullptr || kept == nullptr || forward == nullptr || backward == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    const fmd_status st = check(*problem, z);
    if (st != FMD_OK) return st;
    const bool few = few_rows(z, keep);
    *kept = few ? few_bytes(z) : z.rows > 0 ? kept_layout(z, keep != 0).bytes : 0;
    *forward = few || z.rows == 0 ? 0 : down_plan(z).bytes();
    *backward = z.rows > 0 && keep ? scratch_layout(z).bytes : 0;
    return FMD_OK;
}

fmd_status fmd_pad_rows(const fmd_padded* x, int32_t count, void* stream) {
    if (x == nullptr || count < 1 || count > 4) return FMD_ERR_INVALID_ARGUMENT;
    PadArgs a{};
    int64_t most = 0;
    for (int i = 0; i < count; ++i) {
        if (x[i].rows < 0 || x[i].columns < 1 || x[i].columns > (1 << 20) || x[i].to_row < x[i].columns || x[i].to_row % 8 != 0 ||
            (x[i].rows > 0 && (x[i].from == nullptr || x[i].to == nullptr)))
            return FMD_ERR_INVALID_ARGUMENT;
        if (!aligned16(x[i].to) || x[i].to_row > (1 << 24) || x[i].rows > (1 << 28)) return FMD_ERR_UNSUPPORTED;
        a.x[i] = x[i];
        most = x[i].rows * (x[i].to_row / 8) > most ? x[i].rows * (x[i].to_row / 8) : most;
    }
    if (most == 0) return FMD_OK;
    pad_kernel<<<dim3(unsigned(grid_for(most, 256)), unsigned(count)), 256, 0, as_stream(stream)>>>(a);
    return check_launch();
}

fmd_status fmd_gated_feed_forward(const fmd_feed_forward* problem, void* y, int32_t keep, void* kept, size_t kept_bytes,
                                  void* workspace, size_t workspace_bytes, int32_t* flags, void* stream) {
    Sizes z;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check(*problem, z);
    if (st != FMD_OK || z.rows == 0) return st;
    if (y == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    if (few_rows(z, keep)) {
        if (kept == nullptr || kept_bytes < few_bytes(z)) return FMD_ERR_WORKSPACE;
        if (!aligned16(y) || !aligned16(kept)) return FMD_ERR_UNSUPPORTED;
        return run_few(*problem, static_cast<float*>(kept), static_cast<float*>(y), as_stream(stream));
    }
    const Kept k = kept_layout(z, keep != 0);
    const Plan down = down_plan(z);
    if (kept_bytes < k.bytes || kept == nullptr || workspace_bytes < down.bytes() ||
        (down.splits > 1 && workspace == nullptr))
        return FMD_ERR_WORKSPACE;
    if (!aligned16(y) || !aligned16(kept) || !aligned16(workspace)) return FMD_ERR_UNSUPPORTED;
    if ((st = ready()) != FMD_OK) return st;
    const cudaStream_t s = as_stream(stream);
    char* at = static_cast<char*>(kept);
    const fmd_feed_forward& f = *problem;
    const Inputs in = inputs_of(f, z, k, at);
    if (z.planes == 3) {
        SplitArgs a{};
        int count = 0;
        add_split(a, count, f.x, at + k.x, z.rows, z.width, f.x_row, z.width_row);
        add_split(a, count, f.gate, at + k.gate, z.hidden, z.width, f.gate_row, z.width_row);
        add_split(a, count, f.up, at + k.up, z.hidden, z.width, f.up_row, z.width_row);
        add_split(a, count, f.down, at + k.down, z.out, z.hidden, f.down_row, z.hidden_row);
        if ((st = split(a, count, s)) != FMD_OK) return st;
    }
    Args g{};
    g.problems = 1;
    g.flags = flags;
    g.act = f.activation;
    g.h = reinterpret_cast<__nv_bfloat16*>(at + k.h);
    g.plane = int64_t(z.values());
    g.panels = z.panels;
    g.blocks = z.blocks;
    if (keep) {
        g.slope = at + k.slope;
        g.level = at + k.level;
        g.unit = reinterpret_cast<float2*>(at + k.unit);
    }
    g.problem[0].m = z.rows;
    g.problem[0].n = z.hidden;
    g.steps = int(steps_of(z.width));
    {
        const Matrix a[2] = {in.x, {}}, b[2] = {in.gate, in.up};
        const int64_t twice = 2 * z.hidden;  // two columns of sums for one of h
        if ((st = run<kUp>(z.planes, a, b, 2, g, plan(&z.rows, &twice, 1, g.steps, z.planes, 32, false),
                           z.planes == 3, s)) != FMD_OK) return st;
    }
    g.problem[0].n = z.out;
    g.problem[0].out = y;
    g.part = static_cast<float*>(workspace);
    g.steps = int(steps_of(z.hidden));
    const Matrix h{at + k.h, z.rows, z.hidden, 64, z.planes, z.panels};
    return run<kDown>(z.planes, &h, &in.down, 1, g, down, true, s);
}

fmd_status fmd_gated_feed_forward_bwd(const fmd_feed_forward* problem, void* kept, size_t kept_bytes, const void* g,
                                      int64_t g_row, void* dx, void* dgate, void* dup, void* ddown, void* workspace,
                                      size_t workspace_bytes, int32_t* flags, void* stream) {
    Sizes z;
    if (problem == nullptr) return FMD_ERR_INVALID_ARGUMENT;
    fmd_status st = check(*problem, z);
    if (st != FMD_OK) return st;
    const fmd_feed_forward& f = *problem;
    const cudaStream_t s = as_stream(stream);
    const int size = z.planes == 1 ? 2 : 4;
    if (z.rows == 0) {  // nothing was summed
        void* const out[3] = {dgate, dup, ddown};
        const int64_t values[3] = {z.hidden * z.width, z.hidden * z.width, z.out * z.hidden};
        for (int i = 0; i < 3; ++i) {
            if (out[i] == nullptr) continue;
            const cudaError_t err = cudaMemsetAsync(out[i], 0, size_t(values[i]) * size, s);
            if (err != cudaSuccess) return record_cuda_error(err);
        }
        return FMD_OK;
    }
    const Kept k = kept_layout(z, true);
    const Scratch w = scratch_layout(z);
    if (g == nullptr || (z.rows > 1 && g_row < z.out)) return FMD_ERR_INVALID_ARGUMENT;
    if (kept == nullptr || kept_bytes < k.bytes || workspace == nullptr || workspace_bytes < w.bytes)
        return FMD_ERR_WORKSPACE;
    if (!aligned16(kept) || !aligned16(workspace) || !aligned16(dx) || !aligned16(dgate) || !aligned16(dup) ||
        !aligned16(ddown) || (z.planes == 1 && !vector_rows(g, z.rows > 1 ? g_row : 0, 0, 2)))
        return FMD_ERR_UNSUPPORTED;
    if ((st = ready()) != FMD_OK) return st;
    char *at = static_cast<char*>(kept), *own = static_cast<char*>(workspace);
    const Inputs in = inputs_of(f, z, k, at);
    Matrix gm{g, z.rows, z.out, g_row, 1, 0};
    if (z.planes == 3) {
        SplitArgs a{};
        int count = 0;
        add_split(a, count, g, own + w.g, z.rows, z.out, g_row, z.out_row);
        if ((st = split(a, count, s)) != FMD_OK) return st;
        gm = Matrix{own + w.g, z.rows, z.out, z.out_row, 3, 0};
    }
    Args args{};
    args.flags = flags;
    args.plane = int64_t(z.values());
    args.panels = z.panels;
    args.blocks = z.blocks;
    args.slope = at + k.slope;
    args.level = at + k.level;
    args.unit = reinterpret_cast<float2*>(at + k.unit);
    args.da = reinterpret_cast<__nv_bfloat16*>(own + w.da);
    args.db = reinterpret_cast<__nv_bfloat16*>(own + w.db);
    args.part = reinterpret_cast<float*>(own + w.part);
    const bool hidden = dx != nullptr || dgate != nullptr || dup != nullptr;
    if (hidden) {
        args.problems = 1;
        args.problem[0].m = z.rows;
        args.problem[0].n = z.hidden;
        args.steps = int(steps_of(z.out));
        st = run<kHidden>(z.planes, &gm, &in.down, 1, args,
                          plan(&z.rows, &z.hidden, 1, args.steps, z.planes, z.planes == 1 ? 64 : 128, false), z.planes == 3, s);
        if (st != FMD_OK) return st;
    }
    const Matrix da{own + w.da, z.rows, z.hidden, 64, z.planes, z.panels};
    const Matrix db{own + w.db, z.rows, z.hidden, 64, z.planes, z.panels};
    if (dx != nullptr) {
        args.problems = 1;
        args.problem[0].n = z.width;
        args.problem[0].out = dx;
        args.turn = int(steps_of(z.hidden));
        args.steps = 2 * args.turn;
        const Matrix a[2] = {da, db}, b[2] = {in.gate, in.up};
        if ((st = run<kInput>(z.planes, a, b, 2, args, input_plan(z), true, s)) != FMD_OK) return st;
    }
    // the products of the weights' gradients that are asked for
    const Plan p = weights_plan(z);
    const Matrix h{at + k.h, z.rows, z.hidden, 64, z.planes, z.panels};
    const Matrix a[3] = {da, db, gm}, b[3] = {in.x, in.x, h};
    void* const out[3] = {dgate, dup, ddown};
    // all three have their places whichever are asked for, so that each has the same bits
    args.problems = 3;
    for (int i = 0; i < 3; ++i) {
        Problem& q = args.problem[i];
        q = Problem{};
        q.out = out[i];
        q.m = i < 2 ? z.hidden : z.out;
        q.n = i < 2 ? z.width : z.hidden;
        q.a = q.b = i;
    }
    args.steps = int(steps_of(z.rows));
    if (dgate == nullptr && dup == nullptr && ddown == nullptr) return FMD_OK;
    return run<kWeights>(z.planes, a, b, 3, args, p, z.planes == 3 || hidden, s);
}

}  // extern "C"
