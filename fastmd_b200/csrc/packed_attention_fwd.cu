// Packed attention in bfloat16 on the tensor cores: the forward pass.
//
//   s = q k^T;  per row a reference m and a sum l over key tiles of 128:
//   p = 2^(c s - m), c = scale log2 e;  l += sum p;  o += p v;  out = o / l,  lse = ln 2 (m + log2 l)
//
// The same out and lse follow for any reference m, so m follows the row's maximum loosely: it moves (and o and l are
// multiplied by 2^(m_old - m_new)) only when the maximum has grown by more than kSlack, which after the first tile is
// rare. p stays below 2^kSlack, in range for bfloat16 and the FP32 sums.
//
// A block owns NT tiles of 128 packed rows of one key head and walks the key tiles they see:
//   warp 0       TMA: q once, then k and v tiles through a ring of shared-memory slots
//   warp 1       one thread issues the products: S_t = q k^T (both from shared memory, into TMEM), O_t += p v (p from
//                TMEM); for two tiles in turn, so the tensor cores work on one tile while the other is exponentiated
//                (a thread for each tile let their products mix and cost 15 %)
//   warps 2, 3   zero the rows behind the last key (another sequence's or an unused slot's: 0 * NaN must not happen)
//   then 4 warps per tile: thread = row. Scores from TMEM, maximum, exp2, sum, p back over the scores as bfloat16;
//                o rescaled in TMEM when m moves; at the end o / l to memory.
// A score tile is only issued after the product that read the weights at its place, by the same thread, and commits
// cover all products before them: "scores ready" therefore also says that o is at rest. The last key tile's products
// are as narrow as its keys (multiples of 16).
//
// Measured: one causal sequence of 10,000, 16 heads on 2 key heads of 128: 431 us, 950 TFLOP/s of the 1,650 that a
// library product reaches; the tensor cores are 50 % busy and so is the special-function unit (a tile of 128 x 128 takes
// 1,024 cycles of products and 1,024 of exponentials, and 2,300 in all: what remains is the hand-over between the two).
// A cubic on the FMA pipes for a quarter of the exponentials cost 15 % instead of saving. 33 new rows of 8 sequences
// behind up to 5,000 keys, four splits: 43 us; one new row of 3 sequences against 20,000 to 60,000 keys, 24 splits:
// 72 us, 3.4 TB/s (the splits of the longest sequence are what it ends with).
//
// Every wait is bounded: on expiry the block raises FMD_FLAG_WAIT_TIMEOUT, waits (bounded) for its copies and
// products in flight, frees its TMEM and returns.

#include "packed_attention_mma.cuh"

namespace fmd {
namespace {

constexpr float kSlack = 8.0f;

template <int KS, int NT>
struct Shape {
    static constexpr int kDim = 16 * KS;  // of a head, rounded up; TMA fills the rest with zeros
    static constexpr int kPanels = (KS + 3) / 4;
    static constexpr uint32_t kTileBytes = kPanels * kPanelBytes;
    // NT = 1: two blocks share an SM (96 or 80 KB each); NT = 2 (two panels): one block, and the ring deep
    static constexpr int kSlots = NT == 1 && kPanels == 2 ? 2 : 4;
    static constexpr int kThreads = 128 + 128 * NT;
    static constexpr uint32_t kTmem = NT == 1 ? 256 : 512;
    static constexpr uint32_t kO = NT * 128;  // first column of the outputs, behind the score tiles
    static constexpr size_t kBytes = size_t(NT + kSlots) * kTileBytes + 1024 + 256;
};

template <int KS, int NT>
struct Ctrl {
    uint64_t q_full;
    Ring<Shape<KS, NT>::kSlots> ring;
    uint64_t scores[NT], weights[NT], done[NT];
    uint64_t tail_here, tail;  // the last v tile has landed; its rows behind the last key are zeros
    uint64_t drain;
    uint32_t tmem;
    int32_t abort;
};

struct Maps {
    CUtensorMap q, k, v;
};

__device__ __forceinline__ void load_scores(uint32_t addr, float (&x)[64]) { tmem_load64(addr, x); }
__device__ __forceinline__ void load_scores(uint32_t addr, float (&x)[128]) { tmem_load128(addr, x); }

// What a row does not see is as if it were not there.
template <int N>
__device__ __forceinline__ void hide(float (&x)[N], int mine) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < mine ? x[i] : -INFINITY;
}

template <int KS, int NT, bool SPLIT>
__global__ void __launch_bounds__(Shape<KS, NT>::kThreads, NT == 1 ? 2 : 1)
    forward_kernel(const __grid_constant__ Maps maps, const Attn a) {
    using S = Shape<KS, NT>;
    extern __shared__ unsigned char raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = smem + NT * S::kTileBytes;
    __shared__ Ctrl<KS, NT> ctl;
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int per_tile = kTile / a.group, per_block = NT * per_tile;
    int head;
    const Place place = block_place<false, true>(a, per_block, &head);
    if (place.b < 0) return;
    const Span s = load_span(a, place.b);
    const int64_t token0 = int64_t(place.tile) * per_block;
    int tokens[NT], ends[NT], counts[NT];  // tokens of each tile, the keys its last one sees, key tiles
    int last = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        tokens[t] = int(max(int64_t(0), min(int64_t(per_tile), s.rows - token0 - t * per_tile)));
        ends[t] = tokens[t] > 0 ? int(seen(s, a.causal, token0 + t * per_tile + tokens[t] - 1)) : 0;
        counts[t] = (ends[t] + kTile - 1) / kTile;
        last = max(last, counts[t]);
    }
    // a split takes a range of the key tiles; from here on everything counts from its first key
    int from = 0;
    if (SPLIT) {
        const int share = (last + int(gridDim.z) - 1) / int(gridDim.z);
        from = min(last, int(blockIdx.z) * share) * kTile;
        const int to = min(last, int(blockIdx.z + 1) * share) * kTile;
        last = 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            ends[t] = max(0, min(ends[t], to) - from);
            counts[t] = (ends[t] + kTile - 1) / kTile;
            last = max(last, counts[t]);
        }
        if (last == 0) {  // nothing to add: a sum of zero
            for (int r = threadIdx.x; r < tokens[0] * a.group; r += blockDim.x)
                a.part_lse[(int64_t(blockIdx.z) * a.rows + s.row0 + token0 + r / a.group) * a.hq + head * a.group +
                           r % a.group] = -INFINITY;
            return;
        }
    }
    const int keys = int(s.keys) - from;
    // the last key tile read holds rows behind the sequence's last key
    const bool tail = last > 0 && keys < last * kTile;

    if (threadIdx.x == 0) {
        mbar_init(&ctl.q_full, 1);
        init_ring(ctl.ring);
        for (int t = 0; t < NT; ++t) {
            mbar_init(&ctl.scores[t], 1);
            mbar_init(&ctl.weights[t], 4);
            mbar_init(&ctl.done[t], 1);
        }
        mbar_init(&ctl.tail_here, 1);
        mbar_init(&ctl.tail, 64);
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<S::kTmem>(&ctl.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;

    if (warp == 0) {
        if (lane == 0 && last > 0) {
            const uint32_t q_bytes = uint32_t(S::kPanels) * 128u * uint32_t(per_tile * a.group);
            int tiles = 0;
            for (int t = 0; t < NT; ++t) tiles += counts[t] > 0;
            mbar_expect_tx(&ctl.q_full, q_bytes * tiles);
            for (int t = 0; t < NT; ++t)
                if (counts[t] > 0)
                    for (int p = 0; p < S::kPanels; ++p)
                        tma_load_4d(su32(smem + t * S::kTileBytes + p * kPanelBytes), &maps.q, &ctl.q_full, p * 64, 0,
                                    head, int(s.row0 + token0) + t * per_tile);
            feed(ctl.ring, &ctl.q_full, abort, 2 * last, S::kTileBytes, [&](int i, int slot, uint64_t* bar) {
                for (int p = 0; p < S::kPanels; ++p)  // k0, v0, k1, v1, ..
                    tma_load_4d(su32(ring + slot * S::kTileBytes + p * kPanelBytes), i & 1 ? &maps.v : &maps.k, bar,
                                p * 64, 0, head, int(s.key0) + from + (i >> 1) * kTile);
            });
        }
    } else if (warp == 1) {
        if (last > 0) {
            const uint32_t base = uniform(tmem), q_tile = uniform(su32(smem)), first_slot = uniform(su32(ring));
            const uint32_t o_desc = bf16_idesc(S::kDim, true);
            const int tiles = uniform(last);
            const bool zeroed = uniform(int(tail));
            int count[NT], end[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                count[t] = uniform(counts[t]);
                end[t] = uniform(ends[t]);
            }
            auto slot = [&](int i) { return first_slot + uint32_t(i % S::kSlots) * S::kTileBytes; };
            auto width = [&](int t, int j) { return min(kTile, (end[t] - j * kTile + 15) & ~15); };
            bool ok = warp_wait(&ctl.q_full, 0, abort), issued = false;
            auto score = [&](int t, int j) {
                tc_fence_after();
                const uint32_t desc = bf16_idesc(width(t, j), false);
                if (elect_one()) {
                    product_rows<KS>(base + t * 128u, q_tile + t * S::kTileBytes, slot(2 * j), desc);
                    tc_commit(&ctl.scores[t]);
                    if (t == NT - 1 || j >= count[NT - 1]) tc_commit(&ctl.ring.empty[(2 * j) % S::kSlots]);
                }
                issued = true;
            };
            ok = ok && landed(ctl.ring, 0, abort);
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (ok && count[t] > 0) score(t, 0);
            for (int j = 0; j < tiles && ok; ++j) {
                ok = landed(ctl.ring, 2 * j + 1, abort);
                if (ok && zeroed && j == tiles - 1) {
                    if (elect_one()) mbar_arrive(&ctl.tail_here);
                    ok = warp_wait(&ctl.tail, 0, abort);
                }
                bool next = false;  // the next k tile has landed
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (j >= count[t]) continue;
                    ok = ok && warp_wait(&ctl.weights[t], uint32_t(j) & 1u, abort);
                    if (!ok) break;
                    tc_fence_after();
                    const int steps = width(t, j) / 16;
                    if (elect_one()) {
                        product_weights<8, 4, 32>(base + S::kO + uint32_t(t) * S::kDim, base + t * 128u, slot(2 * j + 1),
                                                  steps, o_desc, j > 0);
                        if (j + 1 == count[t]) tc_commit(&ctl.done[t]);
                        if (t == NT - 1 || j >= count[NT - 1]) tc_commit(&ctl.ring.empty[(2 * j + 1) % S::kSlots]);
                    }
                    if (j + 1 >= count[t]) continue;
                    if (!next) ok = landed(ctl.ring, 2 * j + 2, abort);
                    if (!ok) break;
                    next = true;
                    score(t, j + 1);
                }
            }
            if (!ok && issued) {  // the products in flight end before TMEM is freed
                if (elect_one()) tc_commit(&ctl.drain);
                warp_wait(&ctl.drain, 0, abort, true);
            }
        }
    } else if (warp < 4) {
        if (tail && mbar_wait(&ctl.tail_here, 0, abort)) {
            const int first = keys - (last - 1) * kTile;
            zero_rows(ring + ((2 * last - 1) % S::kSlots) * S::kTileBytes, S::kPanels, kPanelBytes, first,
                      (first + 15) & ~15, threadIdx.x - 64, 64);
            mbar_arrive(&ctl.tail);
        }
    } else {
        // ---------------------------------------------------------- softmax: thread = row
        constexpr int kLoad = NT == 2 ? 128 : 64;
        const int t = (warp - 4) >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t at_s = tmem + lanes + t * 128u, at_o = tmem + lanes + S::kO + uint32_t(t) * S::kDim;
        const int token = r / a.group;
        const bool real = token < tokens[t];
        // keys (from the first of the split) that the row sees
        const int limit = real ? min(max(int(seen(s, a.causal, token0 + t * per_tile + token)) - from, 0), ends[t]) : 0;
        const bool idle = !__any_sync(0xffffffffu, limit > 0);  // a warp without rows passes the scores on unread
        const float c = a.scale * kLog2e;
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < counts[t]; ++j) {
            const bool got = mbar_wait(&ctl.scores[t], uint32_t(j) & 1u, abort);
            if (!__all_sync(0xffffffffu, got)) {  // uniform in the warp: TMEM access is .sync.aligned
                *abort = 1;
                ok = false;
                break;
            }
            tc_fence_after();
            if (idle) {
                warp_arrive(&ctl.weights[t]);
                continue;
            }
            const int seen_here = min(kTile, ends[t] - j * kTile);  // columns that some row sees
            const int mine = limit - j * kTile;                     // that this row sees
            const bool masked = __any_sync(0xffffffffu, mine < kTile);
            // the scores stay in registers where a thread may have them all; two blocks an SM read them twice, by halves
            float x[kLoad];
            float top = -INFINITY;
#pragma unroll
            for (int part = 0; part < kTile / kLoad; ++part) {
                if (part * kLoad >= seen_here) break;
                load_scores(at_s + part * kLoad, x);
                if (masked) hide(x, mine - part * kLoad);
                top = fmaxf(top, largest(x));
            }
            top *= c;
            const bool move = top > m + kSlack;  // the first finite maximum always moves: m starts at -inf
            if (__any_sync(0xffffffffu, move)) {
                const float keep = move ? ex2(m - top) : 1.0f;
                if (move) m = top;
                l *= keep;
                if (j > 0) {
#pragma unroll 1
                    for (int ch = 0; ch < S::kDim / 16; ++ch) {
                        float o[16];
                        tmem_load16(at_o + ch * 16, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] *= keep;
                        tmem_store16(at_o + ch * 16, reinterpret_cast<const uint32_t(&)[16]>(o));
                    }
                }
            }
            const float base = m == -INFINITY ? 0.0f : m;
            const float2 c2 = make_float2(c, c), base2 = make_float2(-base, -base);
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int part = 0; part < kTile / kLoad; ++part) {
                if (part * kLoad >= seen_here) break;
                if (kLoad < kTile) {
                    load_scores(at_s + part * kLoad, x);
                    if (masked) hide(x, mine - part * kLoad);
                }
#pragma unroll
                for (int ch = 0; ch < kLoad; ch += 32) {
                    if (part * kLoad + ch >= seen_here) break;
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float2 y = fma2(make_float2(x[ch + i], x[ch + i + 1]), c2, base2);
                        y.x = ex2(y.x);
                        y.y = ex2(y.y);
                        sum[(i / 2) & 1] = add2(sum[(i / 2) & 1], y);
                        p[i / 2] = pack_bf16(y.x, y.y);
                    }
                    tmem_store16(at_s + (part * kLoad + ch) / 2, p);
                }
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.weights[t]);
        }
        if (ok && counts[t] > 0) {
            const bool got = mbar_wait(&ctl.done[t], 0, abort);
            ok = __all_sync(0xffffffffu, got);
            tc_fence_after();
        }
        if (ok && tokens[t] > 0) {
            int64_t flat = (s.row0 + token0 + t * per_tile + token) * a.hq + head * a.group + r % a.group;
            // a row without keys: zeros; a sum that is not a number stays one
            const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
            const float lse = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
            if (SPLIT) flat += int64_t(blockIdx.z) * a.rows * a.hq;
            for (int ch = 0; ch < S::kDim / 32; ++ch) {
                float o[32];
                if (counts[t] > 0) tmem_load32(at_o + ch * 32, o);
                if (!real) continue;
                if (SPLIT) {
                    float* part = a.part + flat * a.dim + ch * 32;
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        if (limit > 0 && ch * 32 + i < a.dim)
                            *reinterpret_cast<float4*>(part + i) =
                                make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
                    continue;
                }
                __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + flat * a.dim + ch * 32;
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (limit > 0)
                        w = make_uint4(pack_bf16(o[i] * inv, o[i + 1] * inv), pack_bf16(o[i + 2] * inv, o[i + 3] * inv),
                                       pack_bf16(o[i + 4] * inv, o[i + 5] * inv), pack_bf16(o[i + 6] * inv, o[i + 7] * inv));
                    if (ch * 32 + i < a.dim) *reinterpret_cast<uint4*>(out + i) = w;
                }
            }
            if (real && SPLIT) a.part_lse[flat] = lse;
            if (real && !SPLIT && a.lse != nullptr) a.lse[flat] = lse;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free<S::kTmem>(tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(a.flags, FMD_FLAG_WAIT_TIMEOUT);
}

template <int KS, int NT, bool SPLIT>
fmd_status launch(const Maps& maps, const Attn& a, int splits, cudaStream_t s) {
    using S = Shape<KS, NT>;
    const fmd_status st = grant_dynamic_smem((const void*)forward_kernel<KS, NT, SPLIT>, S::kBytes, true);
    if (st != FMD_OK) return st;
    const int64_t tiles = tile_bound(a.rows, a.batch, NT * (kTile / a.group));
    forward_kernel<KS, NT, SPLIT>
        <<<dim3(unsigned(tiles * a.hk), 1, unsigned(splits)), S::kThreads, S::kBytes, s>>>(maps, a);
    return check_launch();
}

// Two tiles a block, which read each key tile once, for heads of more than 64 values where that gives every SM a block and a
// mean sequence has eight key tiles; else one tile, two blocks an SM: the one hides what the other takes to start and end.
// us with two tiles and with one, launches back to back until the clocks have settled, heads / key heads x values:
//   1 x 10,000 causal   16/2 x 128: 434, 441    16/2 x 72: 379, 447    16/4 x 64: 364, 349    16/4 x 32: 346, 333
//   8 x 3,000           16/4 x 128: 678, 688    16/4 x 96: 607, 628     8/2 x 64: 312, 282     8/8 x 32: 304, 282
//   24 x 1,024          16/4 x 128: 282, 277    16/4 x 96: 257, 252     8/2 x 64: 128, 113
// (a few launches on a GPU at rest gain less by two: 128 values, 388 and 379, 24 x 1,024 272 and 247). With fewer blocks
// than SMs (1 x 2,500, 8/8 x 128) 54 and 62, causal 54 and 48.
constexpr int kTwoTilesDim = 64;

bool two_tiles(const Attn& a) {
    return a.dim > kTwoTilesDim && a.batch > 0 && tile_bound(a.rows, a.batch, 2 * (kTile / a.group)) * a.hk >= kNumSMs &&
           a.keys / a.batch >= 8 * kTile;
}

template <int KS>
fmd_status launch(const Maps& maps, const Attn& a, int splits, cudaStream_t s) {
    if (splits > 1) return launch<KS, 1, true>(maps, a, splits, s);
    if constexpr (16 * KS > kTwoTilesDim)
        if (two_tiles(a)) return launch<KS, 2, false>(maps, a, 1, s);
    return launch<KS, 1, false>(maps, a, 1, s);
}

}  // namespace

fmd_status encode_packed(const DriverCalls& drv, CUtensorMap* map, const void* x, int64_t rows, int hk, int group,
                         int dim, int64_t row, int64_t head, int tokens) {
    if (hk * group == 1) head = dim;  // the stride of an axis of one is anything
    if (rows == 1) row = head * hk * group;
    const cuuint64_t dims[4] = {cuuint64_t(dim), cuuint64_t(group), cuuint64_t(hk), cuuint64_t(rows)};
    const cuuint64_t strides[3] = {cuuint64_t(head) * 2, cuuint64_t(head) * 2 * group, cuuint64_t(row) * 2};
    const cuuint32_t box[4] = {64, cuuint32_t(group), 1, cuuint32_t(tokens)};
    const cuuint32_t step[4] = {1, 1, 1, 1};
    const CUresult r = drv.encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(x), dims, strides, box,
                                  step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FMD_OK : record_error_text(FMD_ERR_CUDA, "cuTensorMapEncodeTiled failed, CUresult", r);
}

fmd_status attention_forward_mma(const Attn& a, int splits, cudaStream_t s) {
    const DriverCalls& drv = driver_calls();
    if (drv.encode == nullptr || drv.ctx_get_current == nullptr)
        return record_error_text(FMD_ERR_CUDA, "driver entry point cuTensorMapEncodeTiled unavailable", 0);
    fmd_status st = bind_context(drv);
    Maps maps{};
    if (st == FMD_OK)
        st = encode_packed(drv, &maps.q, a.q, a.rows, a.hk, a.group, a.dim, a.q_row, a.q_head, kTile / a.group);
    if (a.keys > 0) {  // without keys nothing is loaded
        if (st == FMD_OK) st = encode_packed(drv, &maps.k, a.k, a.keys, a.hk, 1, a.dim, a.k_row, a.k_head, kTile);
        if (st == FMD_OK) st = encode_packed(drv, &maps.v, a.v, a.keys, a.hk, 1, a.dim, a.v_row, a.v_head, kTile);
    }
    if (st != FMD_OK) return st;
    return a.dim <= 32 ? launch<2>(maps, a, splits, s) : a.dim <= 64 ? launch<4>(maps, a, splits, s)
         : a.dim <= 96 ? launch<6>(maps, a, splits, s) : launch<8>(maps, a, splits, s);
}

int attention_splits_mma(const Attn& a) { return two_tiles(a) ? 1 : key_splits(a, kTile / a.group, 2 * kNumSMs, kTile); }

}  // namespace fmd
