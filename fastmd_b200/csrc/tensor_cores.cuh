// The tensor-core pieces that all kernels on bfloat16 operands share: TMA loads, the warp that issues products, TMEM access,
// rings of tiles, planes of float32.
#pragma once

#include "sm100.cuh"

namespace fmd {

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                            int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(su32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}

// The products are issued by one thread of a warp whose lanes all walk through the same waits: only there, with every
// operand the same in all lanes, does the compiler keep descriptors and addresses in uniform registers. Under a branch
// on the lane each product took about 115 cycles to issue, twice what the tensor cores need for it.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// mbar_wait by a whole warp: true when every lane has seen the phase complete.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int32_t* abort,
                                          bool ignore_abort = false) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, ignore_abort));
}

// One arrival for a warp, after all its lanes have come this far (32 arrivals on one barrier go one by one).
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// The upper halves of the two descriptors (the lower ones hold the address and the leading offset, in 16 bytes):
// groups of 8 rows 1024 bytes apart, descriptor version 1, 128-byte swizzle.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);

// An operand whose rows are the product's M or N index: a step of 16 along the row is 32 bytes (+ 2).
__device__ __forceinline__ uint32_t rows_desc(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | (1u << 16); }

#define FMD_TMEM_R32                                                                                              \
    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, " \
    "%23, %24, %25, %26, %27, %28, %29, %30, %31}"

// 32 consecutive TMEM columns of this thread's lane. The load writes its registers asynchronously: the wait belongs
// to the same statement, so that nothing between the two can copy or reuse them.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " FMD_TMEM_R32 ", [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                   "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]),
                   "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]),
                   "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]),
                   "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
                 : "r"(addr)
                 : "memory");
}

#define FMD_TMEM_R64 \
    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, " \
    "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, " \
    "%42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, " \
    "%62, %63}"

// 64 columns, in the same way
__device__ __forceinline__ void tmem_load64(uint32_t addr, float (&v)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 " FMD_TMEM_R64 ", [%64];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
          "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]),
          "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
          "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]), "=f"(v[32]), "=f"(v[33]), "=f"(v[34]),
          "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]),
          "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]), "=f"(v[48]),
          "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
          "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]),
          "=f"(v[63])
        : "r"(addr)
        : "memory");
}

#define FMD_TMEM_R128 \
    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, " \
    "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, " \
    "%42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, " \
    "%62, %63, %64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, %80, %81, " \
    "%82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, %96, %97, %98, %99, %100, " \
    "%101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, %112, %113, %114, %115, %116, " \
    "%117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}"

// 128 columns, in the same way
__device__ __forceinline__ void tmem_load128(uint32_t addr, float (&v)[128]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x128.b32 " FMD_TMEM_R128 ", [%128];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
          "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]),
          "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
          "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]), "=f"(v[32]), "=f"(v[33]), "=f"(v[34]),
          "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]),
          "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]), "=f"(v[48]),
          "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
          "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]),
          "=f"(v[63]), "=f"(v[64]), "=f"(v[65]), "=f"(v[66]), "=f"(v[67]), "=f"(v[68]), "=f"(v[69]),
          "=f"(v[70]), "=f"(v[71]), "=f"(v[72]), "=f"(v[73]), "=f"(v[74]), "=f"(v[75]), "=f"(v[76]),
          "=f"(v[77]), "=f"(v[78]), "=f"(v[79]), "=f"(v[80]), "=f"(v[81]), "=f"(v[82]), "=f"(v[83]),
          "=f"(v[84]), "=f"(v[85]), "=f"(v[86]), "=f"(v[87]), "=f"(v[88]), "=f"(v[89]), "=f"(v[90]),
          "=f"(v[91]), "=f"(v[92]), "=f"(v[93]), "=f"(v[94]), "=f"(v[95]), "=f"(v[96]), "=f"(v[97]),
          "=f"(v[98]), "=f"(v[99]), "=f"(v[100]), "=f"(v[101]), "=f"(v[102]), "=f"(v[103]),
          "=f"(v[104]), "=f"(v[105]), "=f"(v[106]), "=f"(v[107]), "=f"(v[108]), "=f"(v[109]),
          "=f"(v[110]), "=f"(v[111]), "=f"(v[112]), "=f"(v[113]), "=f"(v[114]), "=f"(v[115]),
          "=f"(v[116]), "=f"(v[117]), "=f"(v[118]), "=f"(v[119]), "=f"(v[120]), "=f"(v[121]),
          "=f"(v[122]), "=f"(v[123]), "=f"(v[124]), "=f"(v[125]), "=f"(v[126]), "=f"(v[127])
        : "r"(addr)
        : "memory");
}

// 16 columns, in the same way
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(addr)
        : "memory");
}

// 8 columns, in the same way
__device__ __forceinline__ void tmem_load8(uint32_t addr, float (&v)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
        : "r"(addr)
        : "memory");
}

// 16 columns: 32 bfloat16 of this thread's lane
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
        : "memory");
}

// 8 columns: 16 bfloat16 of this thread's lane
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The largest of N values: four chains, not one of N dependent steps.
template <int N>
__device__ __forceinline__ float largest(const float (&x)[N]) {
    float t[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int i = 4; i < N; ++i) t[i & 3] = fmaxf(t[i & 3], x[i]);
    return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
}

// The next plane of 2 N values, two neighbours in a word; the values become what is left (exactly).
template <int N>
__device__ __forceinline__ void next_plane(float* y, uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        w[i] = pack_bf16(y[2 * i], y[2 * i + 1]);
        const float2 part = unpack_bf16(w[i]);
        const float2 left = add2(make_float2(y[2 * i], y[2 * i + 1]), make_float2(-part.x, -part.y));
        y[2 * i] = left.x;
        y[2 * i + 1] = left.y;
    }
}

constexpr float kMostBf16 = 3.38953139e38f;  // the largest finite one

__device__ __forceinline__ uint4 pack8(const float* v) {
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

// Eight values' first plane; `v` becomes what is left of them. Held to the largest bfloat16: finite values stay finite.
__device__ __forceinline__ uint4 first_plane8(float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = pack_bf16(fminf(fmaxf(v[2 * i], -kMostBf16), kMostBf16), fminf(fmaxf(v[2 * i + 1], -kMostBf16), kMostBf16));
        const float2 part = unpack_bf16(w[i]);
        v[2 * i] -= part.x;
        v[2 * i + 1] -= part.y;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 next_plane8(float* v) {
    uint32_t w[4];
    next_plane<4>(v, w);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A thread holds a row of a result, memory wants rows side by side: what a warp stores or loads goes through shared memory of
// its own (32 rows), W pieces of 16 bytes a row, so that W lanes reach into one row. The pieces of a row are turned by the
// row's number, which keeps the banks apart both ways.
template <int W>
__device__ __forceinline__ uint4* piece_at(unsigned char* scratch, int row, int piece) {
    constexpr int kShift = W == 8 ? 0 : W == 4 ? 1 : 2;
    return reinterpret_cast<uint4*>(scratch + (row * W + (piece ^ (row >> kShift & (W - 1)))) * 16);
}

// From a row a lane to W lanes a row: piece i becomes piece lane % W of row i (32 / W) + lane / W.
template <int W>
__device__ __forceinline__ void turn_pieces(unsigned char* scratch, uint4 (&w)[W]) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < W; ++i) *piece_at<W>(scratch, lane, i) = w[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = *piece_at<W>(scratch, i * (32 / W) + lane / W, lane % W);
}

// Turned pieces: the first `pieces` of each of the first `rows` rows to `to` and on, rows `stride` bytes apart.
template <int W>
__device__ __forceinline__ void store_pieces(const uint4 (&w)[W], void* to, int64_t stride, int rows, int pieces) {
    const int lane = threadIdx.x & 31, left = lane % W < pieces ? rows - lane / W : 0;
    char* p = static_cast<char*>(to) + (lane / W) * stride + (lane % W) * 16;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (i * (32 / W) < left) *reinterpret_cast<uint4*>(p) = w[i];
        p += (32 / W) * stride;
    }
}

template <int W>
__device__ __forceinline__ void put_rows(unsigned char* scratch, uint4 (&w)[W], void* to, int64_t stride, int rows, int pieces) {
    turn_pieces<W>(scratch, w);
    store_pieces<W>(w, to, stride, rows, pieces);
}

// Zeros rows [first, last) of `panels` panels that lie `stride` bytes apart (the swizzle keeps a row's 128 bytes in
// place), by `count` threads; then visible to the tensor cores after the barrier that follows.
__device__ __forceinline__ void zero_rows(unsigned char* tile, int panels, uint32_t stride, int first, int last,
                                          int thread, int count) {
    const int per = (last - first) * 8;
    for (int i = thread; i < per * panels; i += count) {
        const int p = i / per, w = i - p * per;
        *reinterpret_cast<uint4*>(tile + p * stride + first * 128 + w * 16) = make_uint4(0, 0, 0, 0);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// A ring of shared-memory slots that TMA fills in order.
template <int SLOTS>
struct Ring {
    uint64_t full[SLOTS], empty[SLOTS];
};

template <int SLOTS>
__device__ __forceinline__ void init_ring(Ring<SLOTS>& ring) {
    for (int i = 0; i < SLOTS; ++i) {
        mbar_init(&ring.full[i], 1);
        mbar_init(&ring.empty[i], 1);
    }
}

// The producer (one thread): `count` tiles of `bytes` each, tile i by load(i, slot, barrier). `own`: the barrier of
// the copies that the caller has started before.
template <int SLOTS, typename Load>
__device__ __forceinline__ void feed(Ring<SLOTS>& ring, uint64_t* own, volatile int32_t* abort, int count,
                                     uint32_t bytes, Load load) {
    int slot = 0, armed = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < count; ++i) {
        if (!mbar_wait(&ring.empty[slot], phase ^ 1u, abort)) {
            ok = false;
            break;
        }
        mbar_expect_tx(&ring.full[slot], bytes);
        load(i, slot, &ring.full[slot]);
        armed = i + 1;
        if (++slot == SLOTS) {
            slot = 0;
            phase ^= 1u;
        }
    }
    if (!ok) {  // the copies in flight land before the block ends
        mbar_wait(own, 0, abort, true);
        for (int i = max(0, armed - SLOTS); i < armed; ++i)
            mbar_wait(&ring.full[i % SLOTS], uint32_t(i / SLOTS) & 1u, abort, true);
    } else {  // the last slots' releases land before the block ends
        for (int i = 0; i < SLOTS && mbar_wait(&ring.empty[slot], phase ^ 1u, abort); ++i)
            if (++slot == SLOTS) {
                slot = 0;
                phase ^= 1u;
            }
    }
}

// Waits (a whole warp) for tile i; only for a warp that takes the tiles of each slot in order.
template <int SLOTS>
__device__ __forceinline__ bool landed(Ring<SLOTS>& ring, int i, volatile int32_t* abort) {
    return warp_wait(&ring.full[i % SLOTS], uint32_t(i / SLOTS) & 1u, abort);
}

// The block's TMEM: COLUMNS of it, by one whole warp; the address through shared memory.
template <int COLUMNS>
__device__ __forceinline__ void tmem_alloc(uint32_t* address) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(address)), "n"(COLUMNS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

template <int COLUMNS>
__device__ __forceinline__ void tmem_free(uint32_t address) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "n"(COLUMNS) : "memory");
}

__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;"); }

// Waits for the kernel ahead, whose results are to be seen; every block of a kernel launched early comes here, so that its end
// is also the end of all before it.
__device__ __forceinline__ void wait_for_the_kernel_ahead() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------------- host

// Launches `kernel` so that it may start before the one ahead of it in the stream is complete.
template <typename... Params, typename... Given>
fmd_status launch_early(void (*kernel)(Params...), dim3 grid, int threads, size_t bytes, cudaStream_t s, Given... given) {
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(unsigned(threads));
    config.dynamicSmemBytes = bytes;
    config.stream = s;
    config.attrs = &early;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, Params(given)...);
    return err == cudaSuccess ? check_launch() : record_cuda_error(err);
}

}  // namespace fmd
