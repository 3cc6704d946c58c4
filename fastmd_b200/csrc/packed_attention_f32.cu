// Packed attention in float32 on the tensor cores, for heads of up to 64 values: forward and gradients.
//
// A float32 number is the sum of three bfloat16 ones, x = h + m + l (8 bits of the significand each; the differences
// are exact; an infinity has no such sum, and its products are no numbers). A product of two numbers is then nine
// products of which six matter, largest last:
//   x y ~ l h' + h l' + m m' + m h' + h m' + h h'          (what is left out is below 2^-24 of x y)
// so each FP32 product is six bfloat16 ones with FP32 sums: at the tensor cores' rate about five times what the FP32
// cores could do. q, k, v (and g) are split once by a small kernel into three planes in memory; the weights p and ds
// are split by the threads that compute them, into TMEM. The tensor cores' FP32 sums do not round to nearest, which
// over thousands of keys would show: every product starts from zero, covers one tile, and the sum over tiles (with
// the softmax's rescaling) is kept in registers.
//
// The forward pass is a block per 128 packed rows and key tiles of 128, the gradients as for bfloat16 (queries: a
// block per 128 packed rows; keys: a block per 128 keys) with streamed tiles of 64. There the block's own planes are in
// TMEM: a product of 64 columns takes 32 cycles so and 48 with both operands in shared memory, and shared memory holds
// four stages. Roles of the warps, masks and bounded waits are those of the bfloat16 kernels. 256 workers: two threads
// per lane, each half of the columns. Order of the products:
//   forward  S0 S1 | [p j] o(j), S(j+2)
//   queries  S0 dP0 | S(j+1) dP(j+1), [ds j] dq(j)
//   keys     S0 dP0 | [p j] dv(j), S(j+1), [ds j] dk(j), dP(j+1)

//
// Measured: one sequence of 5,000 rows, 4 heads of 64: forward 160 us (tensor cores 59 % busy: 6 x 25.6 GFLOP as
// bfloat16), queries' gradients 260 us, keys' 360 us (50 and 47 %), five splits each; the error against 64 bits is
// 5e-7 where plain FP32 operations have 1.4e-6.

#include "packed_attention_mma.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 384;
constexpr int kWorkers = 256;
constexpr uint32_t kHalfPanel = kPanelBytes / 2;  // 64 rows
// the plane (0: h, 1: m, 2: l) of each factor in the six products, the smallest first
__device__ constexpr int kPlaneA[6] = {2, 0, 1, 1, 0, 0};
__device__ constexpr int kPlaneB[6] = {0, 2, 1, 0, 1, 0};

struct Maps {
    CUtensorMap q, g, k, v;
};

// the planes in memory, for the rows that a block keeps
struct Own {
    const __nv_bfloat16 *q, *g, *k, *v;
};

// N columns of TMEM (16 or 32) added to a sum in registers, which is then scaled.
template <int N>
__device__ __forceinline__ void drain(uint32_t addr, float (&sum)[N], float keep) {
    float o[N];
    if constexpr (N == 32) tmem_load32(addr, o);
    else tmem_load16(addr, o);
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = (sum[i] + o[i]) * keep;
}

template <int N>
__device__ __forceinline__ void store_values(float* out, const float (&v)[N], float factor, int col0, int dim) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
        if (col0 + i < dim)
            *reinterpret_cast<float4*>(out + col0 + i) =
                make_float4(v[i] * factor, v[i + 1] * factor, v[i + 2] * factor, v[i + 3] * factor);
}

// D [128, n] = the six products of two operands of three planes, along their rows.
template <int KS>
__device__ __forceinline__ void product6(uint32_t d, uint32_t a, uint32_t b, uint32_t b_plane, uint32_t idesc) {
#pragma unroll
    for (int i = 0; i < 6; ++i)
        product_rows<KS>(d, a + kPlaneA[i] * kPanelBytes, b + kPlaneB[i] * b_plane, idesc, i > 0);
}

// The same with the first operand's planes in TMEM (8 KS columns each) and a streamed tile of 64 rows.
template <int KS>
__device__ __forceinline__ void product6_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const uint32_t bd = rows_desc(b + kPlaneB[i] * kHalfPanel);
#pragma unroll
        for (int k = 0; k < KS; ++k)
            mma_weights(d, a + 8u * (kPlaneA[i] * KS + k), bd + 2 * k, idesc, i > 0 || k > 0);
    }
}

// D [128, n] = the six products of weights over a tile's 64 columns (planes h and m at w, 16 columns each of every 32
// that they replace; l at low, 16 columns of every kLow) and a streamed tile.
template <uint32_t kLow>
__device__ __forceinline__ void weigh6(uint32_t d, uint32_t w, uint32_t low, uint32_t b, int steps, uint32_t idesc) {
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const uint32_t at = b + kPlaneB[i] * kHalfPanel;
        if (kPlaneA[i] == 2) product_weights<4, 2, kLow>(d, low, at, steps, idesc, i > 0);
        else product_weights<4, 2, 32>(d, w + 16u * kPlaneA[i], at, steps, idesc, i > 0);
    }
}

// ---------------------------------------------------------------- planes

struct SplitArgs {
    const float* x[4];
    __nv_bfloat16* planes[4];  // [3][rows][heads][dim]
    int64_t rows[4], row[4], head[4];
    int32_t heads[4];
    int32_t dim;
};

constexpr float kBf16Max = 3.38953139e38f;  // (2 - 2^-7) 2^127

// 8 values a thread
__global__ void __launch_bounds__(256) split_kernel(const SplitArgs a) {
    const int t = blockIdx.y, per = a.dim / 8;
    const int64_t heads = a.heads[t], all = a.rows[t] * heads * per;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i / per, row = r / heads;
        const int c = int(i - r * per) * 8;
        const float* x = a.x[t] + row * a.row[t] + (r - row * heads) * a.head[t] + c;
        const float4 p = ldg4(x), q = ldg4(x + 4);
        float v[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
        uint4* out = reinterpret_cast<uint4*>(a.planes[t] + r * a.dim + c);
        const int64_t plane = a.rows[t] * heads * a.dim / 8;
        uint32_t w[4];
        // the first plane is held to the largest bfloat16: beyond it finite numbers would round to an infinity, and what
        // it leaves of them (2^120 at most) is exact all the same
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = pack_bf16(fminf(fmaxf(v[2 * j], -kBf16Max), kBf16Max),
                             fminf(fmaxf(v[2 * j + 1], -kBf16Max), kBf16Max));
            const float2 part = unpack_bf16(w[j]);
            v[2 * j] -= part.x;
            v[2 * j + 1] -= part.y;
        }
        out[0] = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int i = 1; i < 3; ++i) {
            next_plane<4>(v, w);
            out[i * plane] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// ---------------------------------------------------------------- forward

constexpr int kSlots = 3;
constexpr uint32_t kTile3 = 3 * kPanelBytes;  // a tile of 128 rows: three planes
constexpr size_t kForwardBytes = size_t(1 + kSlots) * kTile3 + 1024;

struct ForwardCtrl {
    uint64_t own;
    Ring<kSlots> ring;
    // two barriers for weights and outputs by turns: the workers may be done with the next tile's weights before the
    // issuing warp, which waits for v to land first, has looked at this one's, and a phase that is run over is never seen
    uint64_t scores[2], weights[2], swap, out[2];
    uint64_t tail_here, tail, drain;
    uint32_t tmem;
    int32_t abort;
};

template <int KS, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) forward_kernel(const __grid_constant__ Maps maps, const Attn a) {
    constexpr int kDim = 16 * KS, kMine = kDim / 2;  // output columns, and those of one half
    constexpr uint32_t kL = 256, kO = 384;           // TMEM columns, two buffers each: scores, p's lowest plane, output
    extern __shared__ unsigned char raw[];
    unsigned char* own = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = own + kTile3;
    __shared__ ForwardCtrl ctl;
    __shared__ float maxima[2][2][kTile], sums[2][kTile];
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int per_tile = kTile / a.group;
    int head;
    const Place place = block_place<false, true>(a, per_tile, &head);
    if (place.b < 0) return;
    const Span s = load_span(a, place.b);
    const int64_t token0 = int64_t(place.tile) * per_tile;
    const int tokens = int(min(int64_t(per_tile), s.rows - token0));
    int end = int(seen(s, a.causal, token0 + tokens - 1)), tiles = (end + kTile - 1) / kTile, from = 0;
    if (SPLIT) {  // a range of the key tiles; from here on everything counts from its first key
        const int share = (tiles + int(gridDim.z) - 1) / int(gridDim.z);
        from = min(tiles, int(blockIdx.z) * share) * kTile;
        end = max(0, min(end, min(tiles, int(blockIdx.z + 1) * share) * kTile) - from);
        tiles = (end + kTile - 1) / kTile;
        if (tiles == 0) {
            for (int r = threadIdx.x; r < tokens * a.group; r += blockDim.x)
                a.part_lse[(int64_t(blockIdx.z) * a.rows + s.row0 + token0 + r / a.group) * a.hq + head * a.group +
                           r % a.group] = -INFINITY;
            return;
        }
    }
    const int keys = int(s.keys) - from;
    const bool tail = tiles > 0 && keys < tiles * kTile;

    if (threadIdx.x == 0) {
        mbar_init(&ctl.own, 1);
        init_ring(ctl.ring);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl.scores[i], 1);
            mbar_init(&ctl.weights[i], kWorkers / 32);
            mbar_init(&ctl.out[i], 1);
        }
        mbar_init(&ctl.swap, kWorkers / 32);
        mbar_init(&ctl.tail_here, 1);
        mbar_init(&ctl.tail, 64);
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<512>(&ctl.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;

    if (warp == 0) {
        if (lane == 0 && tiles > 0) {
            mbar_expect_tx(&ctl.own, 3u * 128u * uint32_t(per_tile * a.group));
            for (int p = 0; p < 3; ++p)
                tma_load_4d(su32(own + p * kPanelBytes), &maps.q, &ctl.own, 0, 0, head,
                            int(p * a.rows + s.row0 + token0));
            feed(ctl.ring, &ctl.own, abort, 2 * tiles, kTile3, [&](int i, int slot, uint64_t* bar) {
                const bool last = i == 2 * tiles - 1, v = last || (i > 0 && i % 2 == 0);
                const int j = last ? tiles - 1 : v ? i / 2 - 1 : (i + 1) / 2;
                for (int p = 0; p < 3; ++p)
                    tma_load_4d(su32(ring + slot * kTile3 + p * kPanelBytes), v ? &maps.v : &maps.k, bar, 0, 0, head,
                                int(p * a.keys + s.key0) + from + j * kTile);
            });
        }
    } else if (warp == 1) {
        if (tiles > 0) {
            const uint32_t base = uniform(tmem), own_at = uniform(su32(own)), first_slot = uniform(su32(ring));
            const uint32_t o_desc = bf16_idesc(kDim, true);
            const int count = uniform(tiles), last_key = uniform(end);
            const bool zeroed = uniform(int(tail));
            // two key tiles ahead of the values: k0 k1 v0 k2 v1 .. k(n-1) v(n-2) v(n-1)
            auto key_at = [&](int j) { return j > 0 ? 2 * j - 1 : 0; };
            auto value_at = [&](int j) { return j + 1 < count ? 2 * j + 2 : 2 * j + 1; };
            auto slot = [&](int i) { return first_slot + uint32_t(i % kSlots) * kTile3; };
            auto width = [&](int j) { return min(kTile, (last_key - j * kTile + 15) & ~15); };
            bool ok = warp_wait(&ctl.own, 0, abort), issued = false;
            auto scores = [&](int j) {
                ok = ok && landed(ctl.ring, key_at(j), abort);
                if (!ok) return;
                tc_fence_after();
                const uint32_t desc = bf16_idesc(width(j), false);
                if (elect_one()) {
                    product6<KS>(base + uint32_t(j & 1) * 128u, own_at, slot(key_at(j)), kPanelBytes, desc);
                    tc_commit(&ctl.scores[j & 1]);
                    tc_commit(&ctl.ring.empty[key_at(j) % kSlots]);
                }
                issued = true;
            };
            scores(0);
            if (count > 1) scores(1);
            for (int j = 0; j < count && ok; ++j) {
                ok = landed(ctl.ring, value_at(j), abort);
                if (ok && zeroed && j == count - 1) {
                    if (elect_one()) mbar_arrive(&ctl.tail_here);
                    ok = warp_wait(&ctl.tail, 0, abort);
                }
                ok = ok && warp_wait(&ctl.weights[j & 1], uint32_t(j >> 1) & 1u, abort);
                if (!ok) break;
                tc_fence_after();
                const uint32_t odd = uint32_t(j & 1);
                const uint32_t o = base + kO + odd * 64u, p = base + odd * 128u, low = base + kL + odd * 64u;
                const int steps = width(j) / 16;
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < 6; ++i) {
                        const uint32_t at = slot(value_at(j)) + kPlaneB[i] * kPanelBytes;
                        if (kPlaneA[i] == 2) product_weights<8, 4, 32>(o, low, at, steps, o_desc, i > 0);
                        else product_weights<8, 4, 64>(o, p + 32u * kPlaneA[i], at, steps, o_desc, i > 0);
                    }
                    tc_commit(&ctl.out[j & 1]);
                    tc_commit(&ctl.ring.empty[value_at(j) % kSlots]);
                }
                if (j + 2 < count) scores(j + 2);  // over this tile's weights, behind the product that reads them
            }
            if (!ok && issued) {
                if (elect_one()) tc_commit(&ctl.drain);
                warp_wait(&ctl.drain, 0, abort, true);
            }
        }
    } else if (warp < 4) {
        if (tail && mbar_wait(&ctl.tail_here, 0, abort)) {
            const int first = keys - (tiles - 1) * kTile;
            zero_rows(ring + ((2 * tiles - 1) % kSlots) * kTile3, 3, kPanelBytes, first, (first + 15) & ~15,
                      threadIdx.x - 64, 64);
            mbar_arrive(&ctl.tail);
        }
    } else {
        const int half = (warp - 4) >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const int token = r / a.group;
        const bool real = token < tokens;
        const int limit = real ? min(max(int(seen(s, a.causal, token0 + token)) - from, 0), end) : 0;
        const float c = a.scale * kLog2e;
        const uint32_t at_o = tmem + lanes + kO + uint32_t(half * kMine);
        float m = -INFINITY, l = 0.0f, o[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) o[i] = 0.0f;
        bool ok = true;
        auto all = [&](bool got) {  // uniform in the warp: TMEM access is .sync.aligned
            ok = __all_sync(0xffffffffu, got);
            if (!ok) *abort = 1;
            tc_fence_after();
            return ok;
        };
        for (int j = 0; j < tiles; ++j) {
            if (!all(mbar_wait(&ctl.scores[j & 1], uint32_t(j >> 1) & 1u, abort))) break;
            const uint32_t at_s = tmem + lanes + uint32_t(j & 1) * 128u + uint32_t(half) * 64u;
            const int columns = end - j * kTile - 64 * half, mine = limit - j * kTile - 64 * half;
            float x[64];
            tmem_load64(at_s, x);  // columns behind the products' width hold anything: no row sees them
#pragma unroll
            for (int i = 0; i < 64; ++i) x[i] = i < mine ? x[i] : -INFINITY;
            float top = largest(x);
            // the row's maximum over both halves
            maxima[j & 1][half][r] = top;
            warp_arrive(&ctl.swap);
            if (!all(mbar_wait(&ctl.swap, uint32_t(j) & 1u, abort))) break;
            top = fmaxf(m, fmaxf(top, maxima[j & 1][1 - half][r]) * c);
            const float base = top == -INFINITY ? 0.0f : top;
            const float keep = ex2(m - base);
            m = top;
            const float2 c2 = make_float2(c, c), base2 = make_float2(-base, -base);
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
                const float2 y = fma2(make_float2(x[i], x[i + 1]), c2, base2);
                x[i] = ex2(y.x);
                x[i + 1] = ex2(y.y);
                sum[(i / 2) & 1] = add2(sum[(i / 2) & 1], make_float2(x[i], x[i + 1]));
            }
            l = l * keep + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
            const uint32_t at_l = tmem + lanes + kL + uint32_t(j & 1) * 64u + uint32_t(half) * 32u;
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                if (32 * ch < columns) {
                    uint32_t w[16];
                    next_plane<16>(x + 32 * ch, w);
                    tmem_store16(at_s + ch * 16, w);
                    next_plane<16>(x + 32 * ch, w);
                    tmem_store16(at_s + 32 + ch * 16, w);
                    next_plane<16>(x + 32 * ch, w);
                    tmem_store16(at_l + ch * 16, w);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.weights[j & 1]);
            if (j > 0) {  // the last tile's output, against the old maximum, while this one's products run
                if (!all(mbar_wait(&ctl.out[(j - 1) & 1], uint32_t((j - 1) >> 1) & 1u, abort))) break;
                drain<kMine>(at_o + uint32_t((j - 1) & 1) * 64u, o, keep);
            }
        }
        if (ok && tiles > 0) {
            sums[half][r] = l;
            warp_arrive(&ctl.swap);
            if (all(mbar_wait(&ctl.out[(tiles - 1) & 1], uint32_t((tiles - 1) >> 1) & 1u, abort) &&
                    mbar_wait(&ctl.swap, uint32_t(tiles) & 1u, abort))) {
                drain<kMine>(at_o + uint32_t((tiles - 1) & 1) * 64u, o, 1.0f);
                l = sums[0][r] + sums[1][r];
            }
        }
        if (ok && real) {
            int64_t flat = (s.row0 + token0 + token) * a.hq + head * a.group + r % a.group;
            const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
            const float lse = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
            if (SPLIT) flat += int64_t(blockIdx.z) * a.rows * a.hq;
            if (limit == 0) {
#pragma unroll
                for (int i = 0; i < kMine; ++i) o[i] = 0.0f;
            }
            store_values<kMine>((SPLIT ? a.part : static_cast<float*>(a.out)) + flat * a.dim, o, inv, half * kMine, a.dim);
            if (half == 0 && SPLIT) a.part_lse[flat] = lse;
            if (half == 0 && !SPLIT && a.lse != nullptr) a.lse[flat] = lse;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free<512>(tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(a.flags, FMD_FLAG_WAIT_TIMEOUT);
}

// --------------------------------------------------------------- gradients

constexpr int kStream = 64;                     // rows of a streamed tile
constexpr int kStreamSlots = 8;
constexpr uint32_t kSlot3 = 3 * kHalfPanel;
constexpr size_t kBackwardBytes = kStreamSlots * size_t(kSlot3) + 1024;

struct BackwardCtrl {
    uint64_t own;                // the block's own planes are in TMEM
    Ring<kStreamSlots> ring;
    uint64_t scores[2], dp[2];   // products done
    uint64_t p, ds;              // written by the workers
    uint64_t out;
    uint64_t stats[2], read[2];  // keys: lse and delta of a tile in shared memory; read by all worker warps
    uint64_t tail_here, tail, drain;
    uint32_t tmem;
    int32_t abort;
};

__device__ __forceinline__ void open_block(BackwardCtrl& ctl, int warp) {
    if (threadIdx.x == 0) {
        mbar_init(&ctl.own, kWorkers / 32);
        init_ring(ctl.ring);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl.scores[i], 1);
            mbar_init(&ctl.dp[i], 1);
            mbar_init(&ctl.stats[i], 64);
            mbar_init(&ctl.read[i], kWorkers / 32);
        }
        mbar_init(&ctl.p, kWorkers / 32);
        mbar_init(&ctl.ds, kWorkers / 32);
        mbar_init(&ctl.out, 1);
        mbar_init(&ctl.tail_here, 1);
        mbar_init(&ctl.tail, 64);
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<512>(&ctl.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
}

__device__ __forceinline__ void close_block(BackwardCtrl& ctl, int warp, int32_t* flags) {
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free<512>(ctl.tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(flags, FMD_FLAG_WAIT_TIMEOUT);
}

// A worker's row of one tensor: its three planes into TMEM, 8 KS columns each; zeros where there is no row.
template <int KS>
__device__ __forceinline__ void load_own(uint32_t at, const __nv_bfloat16* row, int64_t plane, int dim, bool real) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int c = 0; c < KS; c += 2) {  // 32 values: 16 columns
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (real && 16 * c + 8 * i < dim) v = *reinterpret_cast<const uint4*>(row + p * plane + 16 * c + 8 * i);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
            tmem_store16(at + uint32_t(8 * (p * KS + c)), w);
        }
    }
}

// The three planes of a thread's 32 weights: h and m over the columns it has read, l beside.
__device__ __forceinline__ void store_planes(uint32_t w, uint32_t low, float (&y)[32]) {
    uint32_t plane[16];
    next_plane<16>(y, plane);
    tmem_store16(w, plane);
    next_plane<16>(y, plane);
    tmem_store16(w + 16, plane);
    next_plane<16>(y, plane);
    tmem_store16(low, plane);
}

template <int KS>
__global__ void __launch_bounds__(kThreads, 1)
    query_gradient_kernel(const __grid_constant__ Maps maps, const Attn a, const Own own) {
    constexpr int kDim = 16 * KS, kMine = kDim / 2;
    // TMEM columns: two buffers of scores (then of ds's lowest plane) and of dP (then ds's other planes), dq, q, g
    constexpr uint32_t kDp = 128, kDq = 256, kQ = 320, kG = 416;
    extern __shared__ unsigned char raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    __shared__ BackwardCtrl ctl;
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    dependents_may_start();
    const int per_tile = kTile / a.group;
    int head;
    const Place place = block_place<false>(a, per_tile, &head);
    if (place.b < 0) return;
    const Span s = load_span(a, place.b);
    const int64_t token0 = int64_t(place.tile) * per_tile;
    const int tokens = int(min(int64_t(per_tile), s.rows - token0));
    int end = int(seen(s, a.causal, token0 + tokens - 1)), tiles = (end + kStream - 1) / kStream, from = 0;
    if (gridDim.z > 1) {  // a range of the key tiles; from here on everything counts from its first key
        const int share = (tiles + int(gridDim.z) - 1) / int(gridDim.z);
        from = min(tiles, int(blockIdx.z) * share) * kStream;
        end = max(0, min(end, min(tiles, int(blockIdx.z + 1) * share) * kStream) - from);
        tiles = (end + kStream - 1) / kStream;
    }
    const int keys = int(s.keys) - from;
    const bool tail = tiles > 0 && keys < tiles * kStream;

    open_block(ctl, warp);
    const uint32_t tmem = ctl.tmem;

    if (warp == 0) {
        if (lane == 0 && tiles > 0) {
            feed(ctl.ring, &ctl.own, abort, 2 * tiles, kSlot3, [&](int i, int slot, uint64_t* bar) {
                for (int p = 0; p < 3; ++p)  // k0, v0, k1, v1, ..
                    tma_load_4d(su32(ring + slot * kSlot3 + p * kHalfPanel), i & 1 ? &maps.v : &maps.k, bar, 0, 0, head,
                                int(p * a.keys + s.key0) + from + (i >> 1) * kStream);
            });
        }
    } else if (warp == 1) {
        if (tiles > 0) {
            const uint32_t base = uniform(tmem), first_slot = uniform(su32(ring));
            const uint32_t out_desc = bf16_idesc(kDim, true);
            const int count = uniform(tiles), last_key = uniform(end);
            auto width = [&](int j) { return min(kStream, (last_key - j * kStream + 15) & ~15); };
            const bool zeroed = uniform(int(tail));
            auto slot = [&](int i) { return first_slot + uint32_t(i % kStreamSlots) * kSlot3; };
            bool ok = warp_wait(&ctl.own, 0, abort), issued = false;
            auto both = [&](int j) {  // scores and dP of tile j
                ok = ok && landed(ctl.ring, 2 * j, abort) && landed(ctl.ring, 2 * j + 1, abort);
                if (!ok) return;
                tc_fence_after();
                const uint32_t at = base + uint32_t(j & 1) * kStream, desc = bf16_idesc(width(j), false);
                if (elect_one()) {
                    product6_tmem<KS>(at, base + kQ, slot(2 * j), desc);
                    tc_commit(&ctl.scores[j & 1]);
                    product6_tmem<KS>(at + kDp, base + kG, slot(2 * j + 1), desc);
                    tc_commit(&ctl.dp[j & 1]);
                    tc_commit(&ctl.ring.empty[(2 * j + 1) % kStreamSlots]);
                }
                issued = true;
            };
            both(0);
            for (int j = 0; j < count && ok; ++j) {
                if (j + 1 < count) both(j + 1);
                if (ok && zeroed && j == count - 1) {
                    if (elect_one()) mbar_arrive(&ctl.tail_here);
                    ok = warp_wait(&ctl.tail, 0, abort);
                }
                ok = ok && warp_wait(&ctl.ds, uint32_t(j) & 1u, abort);
                if (!ok) break;
                tc_fence_after();
                const int steps = width(j) / 16;
                const uint32_t odd = uint32_t(j & 1);
                if (elect_one()) {
                    weigh6<32>(base + kDq, base + kDp + odd * kStream, base + odd * kStream, slot(2 * j), steps, out_desc);
                    tc_commit(&ctl.out);
                    tc_commit(&ctl.ring.empty[(2 * j) % kStreamSlots]);
                }
            }
            if (!ok && issued) {
                if (elect_one()) tc_commit(&ctl.drain);
                warp_wait(&ctl.drain, 0, abort, true);
            }
        }
    } else if (warp < 4) {
        if (tail && mbar_wait(&ctl.tail_here, 0, abort)) {
            const int first = keys - (tiles - 1) * kStream;
            zero_rows(ring + ((2 * tiles - 2) % kStreamSlots) * kSlot3, 3, kHalfPanel, first, (first + 15) & ~15,
                      threadIdx.x - 64, 64);
            mbar_arrive(&ctl.tail);
        }
    } else {
        const int half = (warp - 4) >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const int token = r / a.group;
        const bool real = token < tokens;
        const int64_t flat = (s.row0 + token0 + token) * a.hq + head * a.group + r % a.group;
        const float lse = real ? a.lse[flat] : -INFINITY, delta = real ? a.delta[flat] : 0.0f;
        const int64_t keys_seen = seen(s, a.causal, token0 + token);
        const int limit =
            lse != -INFINITY && scores_count(a, keys_seen) ? min(max(int(keys_seen) - from, 0), end) : 0;
        const float base = lse != -INFINITY ? -lse * kLog2e : 0.0f;
        const float2 c2 = make_float2(a.scale * kLog2e, a.scale * kLog2e), base2 = make_float2(base, base);
        const float2 delta2 = make_float2(-delta, -delta);
        const uint32_t at_q = tmem + lanes + kDq + uint32_t(half * kMine);
        float dq[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) dq[i] = 0.0f;
        if (tiles > 0) {  // the first four warps bring q, the others g
            const int64_t plane = a.rows * a.hq * a.dim;
            load_own<KS>(tmem + lanes + (half ? kG : kQ), (half ? own.g : own.q) + flat * a.dim, plane, a.dim, real);
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.own);
        }
        bool ok = true;
        auto all = [&](bool got) {
            ok = __all_sync(0xffffffffu, got);
            if (!ok) *abort = 1;
            tc_fence_after();
            return ok;
        };
        for (int j = 0; j < tiles; ++j) {
            const int mine = limit - j * kStream - 32 * half;
            const bool any = end - j * kStream - 32 * half > 0;
            const uint32_t at = tmem + lanes + uint32_t(j & 1) * kStream + uint32_t(half) * 32u;
            float p[32], x[32];
            if (!all(mbar_wait(&ctl.scores[j & 1], uint32_t(j >> 1) & 1u, abort))) break;
            if (any) {
                tmem_load32(at, p);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 y = fma2(make_float2(p[i], p[i + 1]), c2, base2);
                    p[i] = ex2(y.x);
                    p[i + 1] = ex2(y.y);
                }
            }
            if (!all(mbar_wait(&ctl.dp[j & 1], uint32_t(j >> 1) & 1u, abort))) break;
            if (any) {
                tmem_load32(at + kDp, x);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 y = mul2(add2(make_float2(x[i], x[i + 1]), delta2), make_float2(p[i], p[i + 1]));
                    x[i] = i < mine ? y.x : 0.0f;
                    x[i + 1] = i + 1 < mine ? y.y : 0.0f;
                }
            }
            if (j > 0) {  // the last tile's product is added before this one's starts over
                if (!all(mbar_wait(&ctl.out, uint32_t(j - 1) & 1u, abort))) break;
                drain<kMine>(at_q, dq, 1.0f);
            }
            if (any) store_planes(at + kDp, at, x);
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.ds);
        }
        if (ok && tiles > 0 && all(mbar_wait(&ctl.out, uint32_t(tiles - 1) & 1u, abort)))
            drain<kMine>(at_q, dq, 1.0f);
        float* out = gridDim.z > 1 ? a.part + int64_t(blockIdx.z) * a.rows * a.hq * a.dim : static_cast<float*>(a.dq);
        if (ok && real) store_values<kMine>(out + flat * a.dim, dq, a.scale, half * kMine, a.dim);
    }
    close_block(ctl, warp, a.flags);
}

template <int KS>
__global__ void __launch_bounds__(kThreads, 1) key_gradient_kernel(const __grid_constant__ Maps maps, const Attn a, const Own own) {
    constexpr int kDim = 16 * KS;
    // TMEM columns: scores (then p's planes h and m), dP (then ds's), the lowest planes of p and ds, dv, dk, k, v
    constexpr uint32_t kDp = 64, kPl = 128, kDl = 160, kDv = 192, kDk = 256, kK = 320, kV = 416;
    extern __shared__ unsigned char raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    __shared__ BackwardCtrl ctl;
    // of two tiles: - lse log2 e, - delta and the number of keys that each packed row sees
    __shared__ alignas(16) float lse_of[2][kStream], delta_of[2][kStream];
    __shared__ alignas(16) int limit_of[2][kStream];
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    int head;
    const Place place = block_place<true>(a, kTile, &head);
    if (place.b < 0) {
        wait_for_previous();
        return;
    }
    const Span s = load_span(a, place.b);
    const int64_t key0 = int64_t(place.tile) * kTile;
    const int per_tile = kStream / a.group, full_rows = per_tile * a.group;
    int64_t first = a.causal ? max(int64_t(0), key0 + s.rows - s.keys) / per_tile : 0;
    const int64_t all = (s.rows + per_tile - 1) / per_tile;
    int tiles = key0 < s.keys ? int(max(int64_t(0), all - first)) : 0;
    if (gridDim.z > 1) {  // a range of them
        const int share = (tiles + int(gridDim.z) - 1) / int(gridDim.z), skip = min(tiles, int(blockIdx.z) * share);
        first += skip;
        tiles = min(tiles, skip + share) - skip;
    }
    const int last_rows = tiles > 0 ? int(min(int64_t(per_tile), s.rows - (first + tiles - 1) * per_tile)) * a.group : 0;
    const bool tail = tiles > 0 && last_rows % 16 != 0 && last_rows < full_rows;

    if (full_rows < kStream && warp >= 4)  // rows of the slots that no copy ever writes are inner rows of the products
        for (int i = 0; i < kStreamSlots; ++i)
            zero_rows(ring + i * kSlot3, 3, kHalfPanel, full_rows, kStream, threadIdx.x - 128, kWorkers);
    open_block(ctl, warp);
    const uint32_t tmem = ctl.tmem;

    if (warp == 0) {
        if (lane == 0 && tiles > 0) {
            feed(ctl.ring, &ctl.own, abort, 2 * tiles, 3u * 128u * full_rows, [&](int i, int slot, uint64_t* bar) {
                for (int p = 0; p < 3; ++p)  // q0, g0, q1, g1, ..
                    tma_load_4d(su32(ring + slot * kSlot3 + p * kHalfPanel), i & 1 ? &maps.g : &maps.q, bar, 0, 0, head,
                                int(p * a.rows + s.row0 + (first + (i >> 1)) * per_tile));
            });
        }
    } else if (warp == 1) {
        if (tiles > 0) {
            const uint32_t base = uniform(tmem), first_slot = uniform(su32(ring));
            const uint32_t out_desc = bf16_idesc(kDim, true);
            const int count = uniform(tiles), rows_last = uniform(last_rows), rows_full = uniform(full_rows);
            const bool zeroed = uniform(int(tail));
            auto slot = [&](int i) { return first_slot + uint32_t(i % kStreamSlots) * kSlot3; };
            auto width = [&](int j) { return ((j == count - 1 ? rows_last : rows_full) + 15) & ~15; };
            bool ok = warp_wait(&ctl.own, 0, abort), issued = false;
            auto scores = [&](int j) {
                ok = ok && landed(ctl.ring, 2 * j, abort);
                if (!ok) return;
                tc_fence_after();
                const uint32_t desc = bf16_idesc(width(j), false);
                if (elect_one()) {
                    product6_tmem<KS>(base, base + kK, slot(2 * j), desc);
                    tc_commit(&ctl.scores[0]);
                }
                issued = true;
            };
            auto dp = [&](int j) {
                ok = ok && landed(ctl.ring, 2 * j + 1, abort);
                if (!ok) return;
                tc_fence_after();
                const uint32_t desc = bf16_idesc(width(j), false);
                if (elect_one()) {
                    product6_tmem<KS>(base + kDp, base + kV, slot(2 * j + 1), desc);
                    tc_commit(&ctl.dp[0]);
                }
            };
            scores(0);
            dp(0);
            for (int j = 0; j < count && ok; ++j) {
                const int steps = width(j) / 16;
                if (zeroed && j == count - 1) {
                    if (elect_one()) mbar_arrive(&ctl.tail_here);
                    ok = warp_wait(&ctl.tail, 0, abort);
                }
                ok = ok && warp_wait(&ctl.p, uint32_t(j) & 1u, abort);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    weigh6<16>(base + kDv, base, base + kPl, slot(2 * j + 1), steps, out_desc);
                    tc_commit(&ctl.ring.empty[(2 * j + 1) % kStreamSlots]);
                }
                if (j + 1 < count) scores(j + 1);
                ok = ok && warp_wait(&ctl.ds, uint32_t(j) & 1u, abort);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    weigh6<16>(base + kDk, base + kDp, base + kDl, slot(2 * j), steps, out_desc);
                    if (j + 1 == count) tc_commit(&ctl.out);
                    tc_commit(&ctl.ring.empty[(2 * j) % kStreamSlots]);
                }
                if (j + 1 < count) dp(j + 1);
            }
            if (!ok && issued) {
                if (elect_one()) tc_commit(&ctl.drain);
                warp_wait(&ctl.drain, 0, abort, true);
            }
        }
    } else if (warp < 4) {
        const int r = threadIdx.x - 64;
        bool ok = true;
        for (int j = 0; j < tiles && ok; ++j) {
            if (j >= 2 && !mbar_wait(&ctl.read[j & 1], uint32_t((j >> 1) - 1) & 1u, abort)) {
                ok = false;
                break;
            }
            const int64_t token = (first + j) * per_tile + r / a.group;
            float lse = -INFINITY, delta = 0.0f;
            int limit = 0;
            if (r < full_rows && token < s.rows) {
                const int64_t flat = (s.row0 + token) * a.hq + head * a.group + r % a.group;
                lse = a.lse[flat];
                delta = a.delta[flat];
                limit = int(max(int64_t(0), min(int64_t(kTile), seen(s, a.causal, token) - key0)));
            }
            const bool none = lse == -INFINITY;
            lse_of[j & 1][r] = none ? 0.0f : -lse * kLog2e;
            delta_of[j & 1][r] = -delta;
            limit_of[j & 1][r] = none ? 0 : limit;
            mbar_arrive(&ctl.stats[j & 1]);
        }
        if (tail && ok && mbar_wait(&ctl.tail_here, 0, abort)) {
            for (int i = 2 * tiles - 2; i < 2 * tiles; ++i)
                zero_rows(ring + (i % kStreamSlots) * kSlot3, 3, kHalfPanel, last_rows, (last_rows + 15) & ~15, r, 64);
            mbar_arrive(&ctl.tail);
        }
    } else {
        const int half = (warp - 4) >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const float2 c2 = make_float2(a.scale * kLog2e, a.scale * kLog2e);
        // the first four warps keep the sum of dv, the others that of dk
        const uint32_t at_out = tmem + lanes + (half ? kDk : kDv);
        float out[kDim / 32][32];
#pragma unroll
        for (int i = 0; i < kDim; ++i) out[i / 32][i % 32] = 0.0f;
        if (tiles > 0) {  // the first four warps bring k, the others v
            const int64_t at = ((s.key0 + key0 + r) * a.hk + head) * a.dim, plane = a.keys * a.hk * a.dim;
            load_own<KS>(tmem + lanes + (half ? kV : kK), (half ? own.v : own.k) + at, plane, a.dim, key0 + r < s.keys);
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.own);
        }
        bool ok = true;
        auto all = [&](bool got) {
            ok = __all_sync(0xffffffffu, got);
            if (!ok) *abort = 1;
            tc_fence_after();
            return ok;
        };
        auto drain_all = [&] {
#pragma unroll
            for (int i = 0; i < kDim / 32; ++i) drain<32>(at_out + 32 * i, out[i], 1.0f);
        };
        for (int j = 0; j < tiles; ++j) {
            const int rows = j == tiles - 1 ? last_rows : full_rows;
            const bool any = rows > 32 * half;
            const float* nl = lse_of[j & 1] + 32 * half;
            const float* nd = delta_of[j & 1] + 32 * half;
            const int* lim = limit_of[j & 1] + 32 * half;
            const uint32_t at = tmem + lanes + uint32_t(half) * 32u, low = tmem + lanes + uint32_t(half) * 16u;
            float p[32], x[32];
            if (!all(mbar_wait(&ctl.stats[j & 1], uint32_t(j >> 1) & 1u, abort) &&
                     mbar_wait(&ctl.scores[0], uint32_t(j) & 1u, abort)))
                break;
            if (any) {
                tmem_load32(at, p);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 y = fma2(make_float2(p[i], p[i + 1]), c2, *reinterpret_cast<const float2*>(nl + i));
                    const int2 m = *reinterpret_cast<const int2*>(lim + i);
                    p[i] = x[i] = r < m.x ? ex2(y.x) : 0.0f;
                    p[i + 1] = x[i + 1] = r < m.y ? ex2(y.y) : 0.0f;
                }
                store_planes(at, low + kPl, x);
            }
            // the scores were issued behind the last tile's dv, dP behind its dk: each is complete, and added here
            // before the products that start over
            if (j > 0 && half == 0) drain_all();
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.p);
            if (!all(mbar_wait(&ctl.dp[0], uint32_t(j) & 1u, abort))) break;
            if (any) {
                tmem_load32(at + kDp, x);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 d = *reinterpret_cast<const float2*>(nd + i);
                    const int2 m = *reinterpret_cast<const int2*>(lim + i);
                    const float2 y = mul2(add2(make_float2(x[i], x[i + 1]), d), make_float2(p[i], p[i + 1]));
                    x[i] = r < m.x ? y.x : 0.0f;
                    x[i + 1] = r < m.y ? y.y : 0.0f;
                }
                store_planes(at + kDp, low + kDl, x);
            }
            if (j > 0 && half == 1) drain_all();
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.ds);
            if (lane == 0) mbar_arrive(&ctl.read[j & 1]);
        }
        if (ok && tiles > 0 && all(mbar_wait(&ctl.out, 0, abort))) drain_all();
        if (ok && key0 + r < s.slot) {  // slot rows that are no keys get zeros
            float* row = gridDim.z > 1 ? (half ? a.part_dk : a.part_dv) + int64_t(blockIdx.z) * a.keys * a.hk * a.dim
                                       : static_cast<float*>(half ? a.dk : a.dv);
            row += ((s.key0 + key0 + r) * a.hk + head) * a.dim;
            const bool keep = key0 + r < s.keys && !(half && !scores_count(a, s.keys));
#pragma unroll
            for (int i = 0; i < kDim / 32; ++i) {
                if (!keep) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) out[i][e] = 0.0f;
                }
                store_values<32>(row, out[i], half ? a.scale : 1.0f, 32 * i, a.dim);
            }
        }
    }
    wait_for_previous();
    close_block(ctl, warp, a.flags);
}

// ------------------------------------------------------------------- host

// The planes of up to four tensors, one behind the other in the workspace; their tensor maps' base addresses.
struct Planes {
    SplitArgs args{};
    int count = 0;
    __nv_bfloat16* next;

    explicit Planes(void* workspace) : next(static_cast<__nv_bfloat16*>(workspace)) {}

    const __nv_bfloat16* add(const void* x, int64_t rows, int heads, int64_t row, int64_t head, int dim) {
        __nv_bfloat16* const planes = next;
        args.x[count] = static_cast<const float*>(x);
        args.planes[count] = planes;
        args.rows[count] = rows;
        args.heads[count] = heads;
        args.row[count] = row;
        args.head[count] = head;
        args.dim = dim;
        ++count;
        next += 3 * rows * heads * dim;
        return planes;
    }

    fmd_status launch(cudaStream_t s) const {
        int64_t most = 0;
        for (int i = 0; i < count; ++i) {
            const int64_t n = args.rows[i] * args.heads[i] * (args.dim / 8);
            most = n > most ? n : most;
        }
        if (most == 0) return FMD_OK;
        split_kernel<<<dim3(unsigned(grid_for(most, 256)), unsigned(count)), 256, 0, s>>>(args);
        return check_launch();
    }
};

fmd_status encode_planes(const DriverCalls& drv, CUtensorMap* map, const void* planes, int64_t rows, int hk, int group,
                         int dim, int tokens) {
    return encode_packed(drv, map, planes, 3 * rows, hk, group, dim, int64_t(hk) * group * dim, dim, tokens);
}

template <int KS>
fmd_status launch_forward(const Maps& maps, const Attn& a, int splits, cudaStream_t s) {
    const void* kernel = splits > 1 ? (const void*)forward_kernel<KS, true> : (const void*)forward_kernel<KS, false>;
    const fmd_status st = grant_dynamic_smem(kernel, kForwardBytes, true);
    if (st != FMD_OK) return st;
    const dim3 grid(unsigned(tile_bound(a.rows, a.batch, kTile / a.group) * a.hk), 1, unsigned(splits));
    if (splits > 1) forward_kernel<KS, true><<<grid, kThreads, kForwardBytes, s>>>(maps, a);
    else forward_kernel<KS, false><<<grid, kThreads, kForwardBytes, s>>>(maps, a);
    return check_launch();
}

template <int KS>
fmd_status launch_backward(const Maps& maps, const Attn& a, const Own& own, BackwardSplits splits, cudaStream_t s) {
    fmd_status st = grant_dynamic_smem((const void*)query_gradient_kernel<KS>, kBackwardBytes, true);
    if (st == FMD_OK) st = grant_dynamic_smem((const void*)key_gradient_kernel<KS>, kBackwardBytes, true);
    if (st != FMD_OK) return st;
    if (a.dq != nullptr && a.rows > 0) {
        const dim3 grid(unsigned(tile_bound(a.rows, a.batch, kTile / a.group) * a.hk), 1, unsigned(splits.queries));
        query_gradient_kernel<KS><<<grid, kThreads, kBackwardBytes, s>>>(maps, a, own);
        if ((st = check_launch()) != FMD_OK) return st;
    }
    if (a.dk != nullptr && a.keys > 0) {
        const dim3 grid(unsigned(tile_bound(a.keys, a.batch, kTile) * a.hk), 1, unsigned(splits.keys));
        if (a.dq != nullptr && a.rows > 0)
            return launch_early(key_gradient_kernel<KS>, grid, kThreads, kBackwardBytes, s, maps, a, own);
        key_gradient_kernel<KS><<<grid, kThreads, kBackwardBytes, s>>>(maps, a, own);
        st = check_launch();
    }
    return st;
}

}  // namespace

size_t attention_planes_bytes(const Attn& a, bool backward) {
    const size_t values = size_t(a.rows) * a.hq * (backward ? 2 : 1) + size_t(a.keys) * a.hk * 2;
    return (values * a.dim * 3 * sizeof(__nv_bfloat16) + 15) & ~size_t(15);
}

fmd_status attention_forward_planes(const Attn& a, int splits, void* workspace, cudaStream_t s) {
    const DriverCalls& drv = driver_calls();
    if (drv.encode == nullptr || drv.ctx_get_current == nullptr)
        return record_error_text(FMD_ERR_CUDA, "driver entry point cuTensorMapEncodeTiled unavailable", 0);
    fmd_status st = bind_context(drv);
    Maps maps{};
    Planes planes(workspace);
    if (st == FMD_OK)
        st = encode_planes(drv, &maps.q, planes.add(a.q, a.rows, a.hq, a.q_row, a.q_head, a.dim), a.rows, a.hk, a.group,
                           a.dim, kTile / a.group);
    if (a.keys > 0) {
        if (st == FMD_OK)
            st = encode_planes(drv, &maps.k, planes.add(a.k, a.keys, a.hk, a.k_row, a.k_head, a.dim), a.keys, a.hk, 1,
                               a.dim, kTile);
        if (st == FMD_OK)
            st = encode_planes(drv, &maps.v, planes.add(a.v, a.keys, a.hk, a.v_row, a.v_head, a.dim), a.keys, a.hk, 1,
                               a.dim, kTile);
    }
    if (st == FMD_OK) st = planes.launch(s);
    if (st != FMD_OK) return st;
    return a.dim <= 32 ? launch_forward<2>(maps, a, splits, s) : launch_forward<4>(maps, a, splits, s);
}

fmd_status attention_backward_planes(const Attn& a, BackwardSplits splits, void* workspace, cudaStream_t s) {
    const DriverCalls& drv = driver_calls();
    if (drv.encode == nullptr || drv.ctx_get_current == nullptr)
        return record_error_text(FMD_ERR_CUDA, "driver entry point cuTensorMapEncodeTiled unavailable", 0);
    fmd_status st = bind_context(drv);
    Maps maps{};  // of streamed tiles of 64 rows; a block reads its own rows by itself
    Own own{};
    Planes planes(workspace);
    if (a.rows > 0) {
        const int tokens = kStream / a.group;
        own.q = planes.add(a.q, a.rows, a.hq, a.q_row, a.q_head, a.dim);
        own.g = planes.add(a.g, a.rows, a.hq, a.g_row, a.g_head, a.dim);
        if (st == FMD_OK) st = encode_planes(drv, &maps.q, own.q, a.rows, a.hk, a.group, a.dim, tokens);
        if (st == FMD_OK) st = encode_planes(drv, &maps.g, own.g, a.rows, a.hk, a.group, a.dim, tokens);
    }
    if (a.keys > 0) {
        own.k = planes.add(a.k, a.keys, a.hk, a.k_row, a.k_head, a.dim);
        own.v = planes.add(a.v, a.keys, a.hk, a.v_row, a.v_head, a.dim);
        if (st == FMD_OK) st = encode_planes(drv, &maps.k, own.k, a.keys, a.hk, 1, a.dim, kStream);
        if (st == FMD_OK) st = encode_planes(drv, &maps.v, own.v, a.keys, a.hk, 1, a.dim, kStream);
    }
    if (st == FMD_OK) st = planes.launch(s);
    if (st != FMD_OK) return st;
    return a.dim <= 32 ? launch_backward<2>(maps, a, own, splits, s) : launch_backward<4>(maps, a, own, splits, s);
}

}  // namespace fmd
