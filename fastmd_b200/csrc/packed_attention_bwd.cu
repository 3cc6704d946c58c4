// Packed attention in bfloat16 on the tensor cores: the gradients of q and of k and v.
//
//   p = exp(scale q k^T - lse),  dp = g v^T,  ds = p (dp - delta)
//   dq = scale ds k;   dv = p^T g,  dk = scale ds^T q
//
// p is rounded to bfloat16 for its product with g, as for that with v in the forward pass: its roundings average out
// to about that of the stored result. Those of ds would count for more, because sums over ds cancel (a row's adds up
// to zero), and took the error of dq and dk to 1.5 times that of rounding the result alone; so ds is kept in two planes,
// ds = h + m of 16 significant bits, at the price of one more product each.
//
// Two kernels, each of which owns the rows it writes and adds in one order, so that the gradients are the same bits on
// every run without atomics; the price is that scores and dp are computed twice (seven products for five). Where the
// blocks do not fill the GPU the axis they walk along is shared out: each part is then written in FP32 and a third kernel
// adds the parts in their order. Both keep one side's tiles in shared memory and stream the other's:
//
//   queries  a block per 128 packed rows: S = q k^T, dP = g v^T, ds over dP in TMEM, dq += ds k
//   keys     a block per 128 keys: S = k q^T and dP = v g^T with the keys in the lanes, so that p and ds are already
//            the transposed operands: p over S, dv += p g; ds over dP, dk += ds q; lse and delta of the columns
//            come through shared memory. The heads of a group are rows of the same tiles: their sum is the product's.
//
//   warp 0       TMA: the block's own tiles once, the others through a ring of shared-memory slots
//   warp 1       one thread issues the products
//   warps 2, 3   rows that must not count (behind a sequence's end) become zeros; keys: lse and delta of each tile
//   warps 4-11   thread = lane; the first four warps columns 0 .. 63, the others 64 .. 127 (each overwrites only
//                columns that it has read itself)
//
// Order of the products (one thread issues them, they run in order; a product that reads a TMEM operand is issued
// before the one that overwrites it):
//   queries  S0 dP0 | S(j+1), [ds j] dq(j), dP(j+1)       S has two buffers: exp2 of tile j + 1 runs during dq(j)
//   keys     S0 dP0 | [p j] dv(j), S(j+1), [ds j] dk(j), dP(j+1)     exp2 of j + 1 runs during dk(j) and dP(j+1)
// Measured: 16 causal trajectories of 100 to 2,000 frames, 16 heads on 4 key heads of 128 (7 products of 9 with the
// second planes, where 5 are the least): queries 264 us, keys 246 us, tensor cores 37 and 55 % busy. The queries' blocks
// are short here (six key tiles), so that starting and ending them is half their time; the keys' blocks are bound by
// their exponentials and planes (3,600 cycles a tile for 2,560 of products). Twice the workers (a quarter of the columns
// each) did not help.
// Every wait is bounded, as in the forward pass.

#include "packed_attention_mma.cuh"

namespace fmd {
namespace {

constexpr int kThreads = 384;
constexpr int kWorkers = 256;

template <int KS, bool KEYS>
struct Shape {
    static constexpr int kDim = 16 * KS;
    static constexpr int kPanels = (KS + 3) / 4;
    static constexpr uint32_t kTileBytes = kPanels * kPanelBytes;
    // as many as fit beside the two tiles that stay (and, for the keys, lse and delta): with five a tile's copy need
    // not wait for the products of the one before
    static constexpr int kSlots = kPanels == 1 ? 8 : KEYS ? 4 : 5;
    static constexpr size_t kBytes = size_t(2 + kSlots) * kTileBytes + 1024 + 256;
};

template <int KS, bool KEYS>
struct Ctrl {
    uint64_t own;  // the two tiles that stay have landed
    Ring<Shape<KS, KEYS>::kSlots> ring;
    uint64_t scores[2], dp;      // products done
    uint64_t p, ds;              // written by the workers
    uint64_t stats[2], read[2];  // keys: lse and delta of a tile in shared memory; read by all worker warps
    uint64_t tail_here, tail;    // the last tiles have landed; their rows behind the end are zeros
    uint64_t done, drain;
    uint32_t tmem;
    int32_t abort;
};

struct Maps {
    CUtensorMap q, g, k, v;
};

template <int KS, bool KEYS>
__device__ __forceinline__ void open_block(Ctrl<KS, KEYS>& ctl, int warp) {
    if (threadIdx.x == 0) {
        mbar_init(&ctl.own, 1);
        init_ring(ctl.ring);
        mbar_init(&ctl.scores[0], 1);
        mbar_init(&ctl.scores[1], 1);
        mbar_init(&ctl.dp, 1);
        mbar_init(&ctl.p, kWorkers / 32);
        mbar_init(&ctl.ds, kWorkers / 32);
        mbar_init(&ctl.stats[0], 64);
        mbar_init(&ctl.stats[1], 64);
        mbar_init(&ctl.read[0], kWorkers / 32);
        mbar_init(&ctl.read[1], kWorkers / 32);
        mbar_init(&ctl.tail_here, 1);
        mbar_init(&ctl.tail, 64);
        mbar_init(&ctl.done, 1);
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<512>(&ctl.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
}

template <int KS, bool KEYS>
__device__ __forceinline__ void close_block(Ctrl<KS, KEYS>& ctl, int warp, int32_t* flags) {
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free<512>(ctl.tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(flags, FMD_FLAG_WAIT_TIMEOUT);
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    st4(p, make_float4(v[0], v[1], v[2], v[3]));
    st4(p + 4, make_float4(v[4], v[5], v[6], v[7]));
}

// Writes 32 FP32 columns of TMEM times `factor` as T, as far as dim goes. loaded (the same in the whole warp):
// the columns hold a result; keep: this row's counts, else it is zeros; real: the row exists.
template <typename T>
__device__ __forceinline__ void store_row(T* out, uint32_t tmem, int col0, int dim, float factor, bool loaded, bool keep,
                                          bool real) {
    float o[32];
    if (loaded) tmem_load32(tmem + col0, o);
    if (!real) return;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = loaded && keep ? o[i + e] * factor : 0.0f;
        if (col0 + i < dim) store8(out + col0 + i, v);
    }
}

// The two planes of ds over the columns of dP that the thread has read: of each 32, 16 and 16.
template <int N>
__device__ __forceinline__ void store_planes(uint32_t at, float (&ds)[N], int chunks) {
#pragma unroll
    for (int ch = 0; ch < N / 32; ++ch) {
        if (ch < chunks) {
            uint32_t w[16];
            next_plane<16>(ds + 32 * ch, w);
            tmem_store16(at + ch * 32, w);
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = pack_bf16(ds[32 * ch + 2 * i], ds[32 * ch + 2 * i + 1]);
            tmem_store16(at + ch * 32 + 16, w);
        }
    }
}

// D (+)= ds B with ds in two planes, 16 columns each of every 32 that they replace: the lower one first.
__device__ __forceinline__ void product_planes(uint32_t d, uint32_t ds, uint32_t b, int steps, uint32_t idesc, bool add) {
    product_weights<8, 2, 32>(d, ds + 16, b, steps, idesc, add);
    product_weights<8, 2, 32>(d, ds, b, steps, idesc, true);
}

// ---------------------------------------------------------------- queries

template <int KS>
__global__ void __launch_bounds__(kThreads, 1)
    query_gradient_kernel(const __grid_constant__ Maps maps, const Attn a) {
    using S = Shape<KS, false>;
    extern __shared__ unsigned char raw[];
    unsigned char* own = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = own + 2 * S::kTileBytes;
    __shared__ Ctrl<KS, false> ctl;
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
    int end = int(seen(s, a.causal, token0 + tokens - 1)), tiles = (end + kTile - 1) / kTile, from = 0;
    if (gridDim.z > 1) {  // a range of the key tiles; from here on everything counts from its first key
        const int share = (tiles + int(gridDim.z) - 1) / int(gridDim.z);
        from = min(tiles, int(blockIdx.z) * share) * kTile;
        end = max(0, min(end, min(tiles, int(blockIdx.z + 1) * share) * kTile) - from);
        tiles = (end + kTile - 1) / kTile;
    }
    const int keys = int(s.keys) - from;
    const bool tail = tiles > 0 && keys < tiles * kTile;
    constexpr uint32_t kDp = 256, kDq = 384;  // TMEM columns: two score buffers, dP, dq

    open_block(ctl, warp);
    const uint32_t tmem = ctl.tmem;

    if (warp == 0) {
        if (lane == 0 && tiles > 0) {
            mbar_expect_tx(&ctl.own, 2u * S::kPanels * 128u * uint32_t(per_tile * a.group));
            for (int p = 0; p < S::kPanels; ++p) {
                tma_load_4d(su32(own + p * kPanelBytes), &maps.q, &ctl.own, p * 64, 0, head, int(s.row0 + token0));
                tma_load_4d(su32(own + S::kTileBytes + p * kPanelBytes), &maps.g, &ctl.own, p * 64, 0, head,
                            int(s.row0 + token0));
            }
            feed(ctl.ring, &ctl.own, abort, 2 * tiles, S::kTileBytes, [&](int i, int slot, uint64_t* bar) {
                for (int p = 0; p < S::kPanels; ++p)  // k0, v0, k1, v1, ..
                    tma_load_4d(su32(ring + slot * S::kTileBytes + p * kPanelBytes), i & 1 ? &maps.v : &maps.k, bar,
                                p * 64, 0, head, int(s.key0) + from + (i >> 1) * kTile);
            });
        }
    } else if (warp == 1) {
        if (tiles > 0) {
            const uint32_t base = uniform(tmem), own_at = uniform(su32(own)), first_slot = uniform(su32(ring));
            const uint32_t out_desc = bf16_idesc(S::kDim, true);
            const int count = uniform(tiles), last_key = uniform(end);
            const bool zeroed = uniform(int(tail));
            auto slot = [&](int i) { return first_slot + uint32_t(i % S::kSlots) * S::kTileBytes; };
            auto width = [&](int j) { return min(kTile, (last_key - j * kTile + 15) & ~15); };
            bool ok = warp_wait(&ctl.own, 0, abort), issued = false;
            auto scores = [&](int j) {  // into buffer j % 2
                ok = ok && landed(ctl.ring, 2 * j, abort);
                if (!ok) return;
                tc_fence_after();
                const uint32_t desc = bf16_idesc(width(j), false);
                if (elect_one()) {
                    product_rows<KS>(base + uint32_t(j & 1) * 128u, own_at, slot(2 * j), desc);
                    tc_commit(&ctl.scores[j & 1]);
                }
                issued = true;
            };
            auto dp = [&](int j) {
                ok = ok && landed(ctl.ring, 2 * j + 1, abort);
                if (!ok) return;
                tc_fence_after();
                const uint32_t desc = bf16_idesc(width(j), false);
                if (elect_one()) {
                    product_rows<KS>(base + kDp, own_at + S::kTileBytes, slot(2 * j + 1), desc);
                    tc_commit(&ctl.dp);
                    tc_commit(&ctl.ring.empty[(2 * j + 1) % S::kSlots]);
                }
            };
            scores(0);
            dp(0);
            for (int j = 0; j < count && ok; ++j) {
                if (j + 1 < count) scores(j + 1);
                if (ok && zeroed && j == count - 1) {
                    if (elect_one()) mbar_arrive(&ctl.tail_here);
                    ok = warp_wait(&ctl.tail, 0, abort);
                }
                ok = ok && warp_wait(&ctl.ds, uint32_t(j) & 1u, abort);
                if (!ok) break;
                tc_fence_after();
                const int steps = width(j) / 16;
                if (elect_one()) {
                    product_planes(base + kDq, base + kDp, slot(2 * j), steps, out_desc, j > 0);
                    if (j + 1 == count) tc_commit(&ctl.done);
                    tc_commit(&ctl.ring.empty[(2 * j) % S::kSlots]);
                }
                if (j + 1 < count) dp(j + 1);
            }
            if (!ok && issued) {
                if (elect_one()) tc_commit(&ctl.drain);
                warp_wait(&ctl.drain, 0, abort, true);
            }
        }
    } else if (warp < 4) {
        if (tail && mbar_wait(&ctl.tail_here, 0, abort)) {  // keys behind the last one: they are the inner index of dq
            const int first = keys - (tiles - 1) * kTile;
            zero_rows(ring + ((2 * tiles - 2) % S::kSlots) * S::kTileBytes, S::kPanels, kPanelBytes, first, (first + 15) & ~15,
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
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            const int columns = end - j * kTile - 64 * half;  // of this half that some row sees
            const int chunks = min(2, max(0, (columns + 31) / 32));
            const int mine = limit - j * kTile - 64 * half;
            const bool masked = __any_sync(0xffffffffu, mine < chunks * 32);
            float p[64];
            bool got = mbar_wait(&ctl.scores[j & 1], uint32_t(j >> 1) & 1u, abort);
            if (!__all_sync(0xffffffffu, got)) {
                *abort = 1;
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t at_s = tmem + lanes + uint32_t(j & 1) * 128u + uint32_t(half) * 64u;
            if (chunks > 0) {
                tmem_load64(at_s, p);
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const float2 y = fma2(make_float2(p[i], p[i + 1]), c2, base2);
                    p[i] = ex2(y.x);
                    p[i + 1] = ex2(y.y);
                }
            }
            got = mbar_wait(&ctl.dp, uint32_t(j) & 1u, abort);
            if (!__all_sync(0xffffffffu, got)) {
                *abort = 1;
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t at_d = tmem + lanes + kDp + uint32_t(half) * 64u;
            if (chunks > 0) {
                float x[64];
                tmem_load64(at_d, x);
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    float2 y = add2(make_float2(x[i], x[i + 1]), delta2);
                    y = mul2(y, make_float2(p[i], p[i + 1]));
                    if (masked) {  // what a row does not see has no share, whatever its values
                        y.x = i < mine ? y.x : 0.0f;
                        y.y = i + 1 < mine ? y.y : 0.0f;
                    }
                    x[i] = y.x;
                    x[i + 1] = y.y;
                }
                store_planes(at_d, x, chunks);
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.ds);
        }
        if (ok && tiles > 0) {
            const bool got = mbar_wait(&ctl.done, 0, abort);
            ok = __all_sync(0xffffffffu, got);
            tc_fence_after();
        }
        if (ok) {
            const int64_t at = flat * a.dim, part = int64_t(blockIdx.z) * a.rows * a.hq * a.dim;
            for (int col = 32 * half; col < S::kDim; col += 64) {
                if (gridDim.z > 1)
                    store_row(a.part + part + at, tmem + lanes + kDq, col, a.dim, a.scale, tiles > 0, true, real);
                else
                    store_row(static_cast<__nv_bfloat16*>(a.dq) + at, tmem + lanes + kDq, col, a.dim, a.scale, tiles > 0,
                              true, real);
            }
        }
    }
    close_block(ctl, warp, a.flags);
}

// ------------------------------------------------------------------- keys

template <int KS>
__global__ void __launch_bounds__(kThreads, 1) key_gradient_kernel(const __grid_constant__ Maps maps, const Attn a) {
    using S = Shape<KS, true>;
    extern __shared__ unsigned char raw[];
    unsigned char* own = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = own + 2 * S::kTileBytes;
    __shared__ Ctrl<KS, true> ctl;
    // of two tiles: - lse log2 e, - delta and the number of keys that each packed row sees
    __shared__ alignas(16) float lse_of[2][kTile], delta_of[2][kTile];
    __shared__ alignas(16) int limit_of[2][kTile];
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
    const int per_tile = kTile / a.group, full_rows = per_tile * a.group;
    // tiles of rows from the one that holds the first token that sees key0
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
    constexpr uint32_t kDp = 128, kDv = 256, kDk = 384;  // TMEM columns, the scores at 0

    if (full_rows < kTile && warp >= 4)  // rows of the slots that no copy ever writes are inner rows of the products
        for (int i = 0; i < S::kSlots; ++i)
            zero_rows(ring + i * S::kTileBytes, S::kPanels, kPanelBytes, full_rows, kTile, threadIdx.x - 128, kWorkers);
    open_block(ctl, warp);
    const uint32_t tmem = ctl.tmem;

    if (warp == 0) {
        if (lane == 0 && tiles > 0) {
            mbar_expect_tx(&ctl.own, 2u * S::kTileBytes);
            for (int p = 0; p < S::kPanels; ++p) {
                tma_load_4d(su32(own + p * kPanelBytes), &maps.k, &ctl.own, p * 64, 0, head, int(s.key0 + key0));
                tma_load_4d(su32(own + S::kTileBytes + p * kPanelBytes), &maps.v, &ctl.own, p * 64, 0, head,
                            int(s.key0 + key0));
            }
            feed(ctl.ring, &ctl.own, abort, 2 * tiles, uint32_t(S::kPanels) * 128u * full_rows,
                 [&](int i, int slot, uint64_t* bar) {
                     for (int p = 0; p < S::kPanels; ++p)  // q0, g0, q1, g1, ..
                         tma_load_4d(su32(ring + slot * S::kTileBytes + p * kPanelBytes), i & 1 ? &maps.g : &maps.q, bar,
                                     p * 64, 0, head, int(s.row0 + (first + (i >> 1)) * per_tile));
                 });
        }
    } else if (warp == 1) {
        if (tiles > 0) {
            const uint32_t base = uniform(tmem), own_at = uniform(su32(own)), first_slot = uniform(su32(ring));
            const uint32_t out_desc = bf16_idesc(S::kDim, true);
            const int count = uniform(tiles), rows_last = uniform(last_rows), rows_full = uniform(full_rows);
            const bool zeroed = uniform(int(tail));
            auto slot = [&](int i) { return first_slot + uint32_t(i % S::kSlots) * S::kTileBytes; };
            auto width = [&](int j) { return ((j == count - 1 ? rows_last : rows_full) + 15) & ~15; };
            bool ok = warp_wait(&ctl.own, 0, abort), issued = false;
            auto scores = [&](int j) {
                ok = ok && landed(ctl.ring, 2 * j, abort);
                if (!ok) return;
                tc_fence_after();
                const uint32_t desc = bf16_idesc(width(j), false);
                if (elect_one()) {
                    product_rows<KS>(base, own_at, slot(2 * j), desc);
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
                    product_rows<KS>(base + kDp, own_at + S::kTileBytes, slot(2 * j + 1), desc);
                    tc_commit(&ctl.dp);
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
                    product_weights<8, 4, 64>(base + kDv, base, slot(2 * j + 1), steps, out_desc, j > 0);
                    tc_commit(&ctl.ring.empty[(2 * j + 1) % S::kSlots]);
                }
                if (j + 1 < count) scores(j + 1);
                ok = ok && warp_wait(&ctl.ds, uint32_t(j) & 1u, abort);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    product_planes(base + kDk, base + kDp, slot(2 * j), steps, out_desc, j > 0);
                    if (j + 1 == count) tc_commit(&ctl.done);
                    tc_commit(&ctl.ring.empty[(2 * j) % S::kSlots]);
                }
                if (j + 1 < count) dp(j + 1);
            }
            if (!ok && issued) {
                if (elect_one()) tc_commit(&ctl.drain);
                warp_wait(&ctl.drain, 0, abort, true);
            }
        }
    } else if (warp < 4) {
        const int thread = threadIdx.x - 64;
        bool ok = true;
        for (int j = 0; j < tiles && ok; ++j) {
            if (j >= 2 && !mbar_wait(&ctl.read[j & 1], uint32_t((j >> 1) - 1) & 1u, abort)) {
                ok = false;
                break;
            }
            const int64_t token0 = (first + j) * per_tile;
            for (int r = thread; r < kTile; r += 64) {
                const int64_t token = token0 + r / a.group;
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
            }
            mbar_arrive(&ctl.stats[j & 1]);
        }
        if (tail && ok && mbar_wait(&ctl.tail_here, 0, abort)) {  // another sequence's rows
            for (int i = 2 * tiles - 2; i < 2 * tiles; ++i)
                zero_rows(ring + (i % S::kSlots) * S::kTileBytes, S::kPanels, kPanelBytes, last_rows,
                          (last_rows + 15) & ~15, thread, 64);
            mbar_arrive(&ctl.tail);
        }
    } else {
        const int half = (warp - 4) >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const float2 c2 = make_float2(a.scale * kLog2e, a.scale * kLog2e);
        const uint32_t at_s = tmem + lanes + uint32_t(half) * 64u, at_d = at_s + kDp;
        const int here = int(min(int64_t(kTile), s.keys - key0));  // keys of this tile
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            const int rows = j == tiles - 1 ? last_rows : full_rows;
            const int chunks = min(2, max(0, (rows - 64 * half + 31) / 32));
            const float* nl = lse_of[j & 1] + 64 * half;
            const float* nd = delta_of[j & 1] + 64 * half;
            const int* lim = limit_of[j & 1] + 64 * half;
            float p[64];
            bool got = mbar_wait(&ctl.stats[j & 1], uint32_t(j >> 1) & 1u, abort) &&
                       mbar_wait(&ctl.scores[0], uint32_t(j) & 1u, abort);
            if (!__all_sync(0xffffffffu, got)) {
                *abort = 1;
                ok = false;
                break;
            }
            tc_fence_after();
            // a column is masked where its row sees fewer keys than the tile has, or is no row at all
            bool masked = false;
            if (lane < 16 * chunks) {
                const int2 w = *reinterpret_cast<const int2*>(lim + 2 * lane);
                masked = w.x < here || w.y < here;
            }
            masked = __any_sync(0xffffffffu, masked);
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                if (ch < chunks) {
                    float x[32];
                    uint32_t w[16];
                    tmem_load32(at_s + ch * 32, x);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 l = *reinterpret_cast<const float2*>(nl + ch * 32 + i);
                        float2 y = fma2(make_float2(x[i], x[i + 1]), c2, l);
                        y.x = ex2(y.x);
                        y.y = ex2(y.y);
                        if (masked) {
                            const int2 m = *reinterpret_cast<const int2*>(lim + ch * 32 + i);
                            y.x = r < m.x ? y.x : 0.0f;
                            y.y = r < m.y ? y.y : 0.0f;
                        }
                        p[ch * 32 + i] = y.x;
                        p[ch * 32 + i + 1] = y.y;
                        w[i / 2] = pack_bf16(y.x, y.y);
                    }
                    tmem_store16(at_s + ch * 16, w);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.p);
            got = mbar_wait(&ctl.dp, uint32_t(j) & 1u, abort);
            if (!__all_sync(0xffffffffu, got)) {
                *abort = 1;
                ok = false;
                break;
            }
            tc_fence_after();
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                if (ch < chunks) {
                    float x[32];
                    tmem_load32(at_d + ch * 32, x);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 d = *reinterpret_cast<const float2*>(nd + ch * 32 + i);
                        float2 y = add2(make_float2(x[i], x[i + 1]), d);
                        y = mul2(y, make_float2(p[ch * 32 + i], p[ch * 32 + i + 1]));
                        if (masked) {  // also where dp is not a number
                            const int2 m = *reinterpret_cast<const int2*>(lim + ch * 32 + i);
                            y.x = r < m.x ? y.x : 0.0f;
                            y.y = r < m.y ? y.y : 0.0f;
                        }
                        x[i] = y.x;
                        x[i + 1] = y.y;
                    }
                    store_planes(at_d + ch * 32, x, 1);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.ds);
            if (lane == 0) mbar_arrive(&ctl.read[j & 1]);
        }
        if (ok && tiles > 0) {
            const bool got = mbar_wait(&ctl.done, 0, abort);
            ok = __all_sync(0xffffffffu, got);
            tc_fence_after();
        }
        if (ok) {
            // the first four warps write dv, the others dk; slot rows that are no keys get zeros
            const int64_t flat = ((s.key0 + key0 + r) * a.hk + head) * a.dim;
            const int64_t part = int64_t(blockIdx.z) * a.keys * a.hk * a.dim;
            const bool real = key0 + r < s.slot;
            const uint32_t from = tmem + lanes + (half ? kDk : kDv);
            const float factor = half ? a.scale : 1.0f;
            const bool keep = r < here && !(half && !scores_count(a, s.keys));
            for (int col = 0; col < S::kDim; col += 32) {
                if (gridDim.z > 1)
                    store_row((half ? a.part_dk : a.part_dv) + part + flat, from, col, a.dim, factor, tiles > 0, keep,
                              real);
                else
                    store_row(static_cast<__nv_bfloat16*>(half ? a.dk : a.dv) + flat, from, col, a.dim, factor, tiles > 0,
                              keep, real);
            }
        }
    }
    wait_for_previous();
    close_block(ctl, warp, a.flags);
}

template <int KS>
fmd_status launch(const Maps& maps, const Attn& a, BackwardSplits splits, cudaStream_t s) {
    constexpr size_t query_bytes = Shape<KS, false>::kBytes, key_bytes = Shape<KS, true>::kBytes;
    fmd_status st = grant_dynamic_smem((const void*)query_gradient_kernel<KS>, query_bytes, true);
    if (st == FMD_OK) st = grant_dynamic_smem((const void*)key_gradient_kernel<KS>, key_bytes, true);
    if (st != FMD_OK) return st;
    if (a.dq != nullptr && a.rows > 0) {
        const int64_t tiles = tile_bound(a.rows, a.batch, kTile / a.group);
        query_gradient_kernel<KS><<<dim3(unsigned(tiles * a.hk), 1, unsigned(splits.queries)), kThreads, query_bytes, s>>>(maps, a);
        if ((st = check_launch()) != FMD_OK) return st;
    }
    if (a.dk != nullptr && a.keys > 0) {
        const dim3 grid(unsigned(tile_bound(a.keys, a.batch, kTile) * a.hk), 1, unsigned(splits.keys));
        if (a.dq != nullptr && a.rows > 0) return launch_early(key_gradient_kernel<KS>, grid, kThreads, key_bytes, s, maps, a);
        key_gradient_kernel<KS><<<grid, kThreads, key_bytes, s>>>(maps, a);
        st = check_launch();
    }
    return st;
}

}  // namespace

fmd_status attention_backward_mma(const Attn& a, BackwardSplits splits, cudaStream_t s) {
    const DriverCalls& drv = driver_calls();
    if (drv.encode == nullptr || drv.ctx_get_current == nullptr)
        return record_error_text(FMD_ERR_CUDA, "driver entry point cuTensorMapEncodeTiled unavailable", 0);
    fmd_status st = bind_context(drv);
    Maps maps{};
    const int tokens = kTile / a.group;
    if (a.rows > 0) {
        if (st == FMD_OK) st = encode_packed(drv, &maps.q, a.q, a.rows, a.hk, a.group, a.dim, a.q_row, a.q_head, tokens);
        if (st == FMD_OK) st = encode_packed(drv, &maps.g, a.g, a.rows, a.hk, a.group, a.dim, a.g_row, a.g_head, tokens);
    }
    if (a.keys > 0) {
        if (st == FMD_OK) st = encode_packed(drv, &maps.k, a.k, a.keys, a.hk, 1, a.dim, a.k_row, a.k_head, kTile);
        if (st == FMD_OK) st = encode_packed(drv, &maps.v, a.v, a.keys, a.hk, 1, a.dim, a.v_row, a.v_head, kTile);
    }
    if (st != FMD_OK) return st;
    return a.dim <= 32 ? launch<2>(maps, a, splits, s) : a.dim <= 64 ? launch<4>(maps, a, splits, s)
         : a.dim <= 96 ? launch<6>(maps, a, splits, s) : launch<8>(maps, a, splits, s);
}

}  // namespace fmd
