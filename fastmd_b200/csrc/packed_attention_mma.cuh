// The tensor-core pieces that the attention kernels share, bfloat16 ones and those in planes of float32: operand tiles, descriptors, products, TMEM access.
//
// An operand tile is 128 rows of up to 128 values as panels of 64 values: panel p holds 128 rows of 128 bytes, in the
// 128-byte swizzle that TMA writes. The same tile serves as a K-major operand (the product runs over its 64-value
// rows: scores) and, read the other way, as an MN-major one (the product runs over its rows: weights times values).
#pragma once

#include "packed_attention.cuh"
#include "tensor_cores.cuh"

namespace fmd {

constexpr int kTile = kRowTile;                      // the M of every product
constexpr uint32_t kPanelBytes = kTile * 128;        // 128 rows x 64 bfloat16
constexpr uint32_t kPanelStep = kPanelBytes >> 4;    // in descriptor units of 16 bytes

// An operand whose rows are the product's inner index and whose 64-value panels are its N index (leading offset: the
// next panel): a step of 16 rows is 2048 bytes (+ 128).
__device__ __forceinline__ uint32_t columns_desc(uint32_t saddr) {
    return ((saddr & 0x3FFFFu) >> 4) | (kPanelStep << 16);
}

// Instruction descriptor of kind::f16: FP32 accumulator, bfloat16 operands, M = 128, N; B transposed when its rows
// are the inner index.
__device__ __forceinline__ uint32_t bf16_idesc(int n, bool b_columns) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_columns ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) |
           (uint32_t(kTile >> 4) << 24);
}

// Two steps of 16 of D [128, n] (+)= A B^T along the rows of both operands, as one statement without branches.
__device__ __forceinline__ void mma_rows2(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 x, y;\n\t.reg .b64 u, v, w, z;\n\t"
        "setp.ne.b32 p, %5, 0;\n\tadd.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\t"
        "mov.b64 u, {%1, %3};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 w, {x, %3};\n\tmov.b64 z, {y, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], u, v, %4, p;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], w, z, %4, 1;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(kDescHigh), "r"(idesc), "r"(add)
        : "memory");
}

// One step of 16 of D [128, n] (+)= P B with P in TMEM (8 columns a step), the rows of B the inner index.
__device__ __forceinline__ void mma_weights(uint32_t d, uint32_t p, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 v;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 v, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], v, %4, p;\n\t}" ::"r"(d),
        "r"(p), "r"(b), "r"(kDescHigh), "r"(idesc), "r"(add)
        : "memory");
}

// D [128, n] (+)= A B^T over KS steps of 16 along the rows of both tiles.
template <int KS>
__device__ __forceinline__ void product_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add = false) {
    const uint32_t ad = rows_desc(a), bd = rows_desc(b);
#pragma unroll
    for (int k = 0; k < KS; k += 2) {
        const uint32_t off = uint32_t(k / 4) * kPanelStep + uint32_t(k % 4) * 2;
        mma_rows2(d, ad + off, bd + off, idesc, add || k > 0);
    }
}

// D [128, n] (+)= P B over `steps` (at most STEPS) steps of 16 rows of B, P [128, 16 steps] bfloat16 in TMEM: groups of
// GROUP steps, kNext columns apart.
template <int STEPS, int GROUP, uint32_t kNext>
__device__ __forceinline__ void product_weights(uint32_t d, uint32_t p, uint32_t b, int steps, uint32_t idesc,
                                                bool add) {
    const uint32_t bd = columns_desc(b);
    if (steps == STEPS) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
            mma_weights(d, p + 8 * (k % GROUP) + (k / GROUP) * kNext, bd + k * 128, idesc, add || k > 0);
    } else {
        for (int k = 0; k < steps; ++k)
            mma_weights(d, p + 8 * (k % GROUP) + (k / GROUP) * kNext, bd + k * 128, idesc, add || k > 0);
    }
}

// The kernel of the keys' gradients follows that of the queries' without depending on it: it is launched so that its
// blocks start as soon as every block of the first has (dependents_may_start), and fill the SMs that the first one's
// end leaves idle. Its last block waits for the first kernel before it ends (wait_for_previous), so that what follows in
// the stream finds both complete.
__device__ __forceinline__ void wait_for_previous() {
    if (blockIdx.x == gridDim.x - 1 && blockIdx.z == gridDim.z - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------------- host

// Packed rows: x [rows, key_heads, group, dim], a box of `tokens` tokens x group heads x 64 values.
fmd_status encode_packed(const DriverCalls& drv, CUtensorMap* map, const void* x, int64_t rows, int hk, int group,
                         int dim, int64_t row, int64_t head, int tokens);

}  // namespace fmd
