// Decay attention on the tensor cores: bfloat16, and float32 as planes of bfloat16.
//
// A block walks over the chunks of 128 rows of one segment and head. Of a chunk (rows t, u of it, l the decay):
//   pairs   s = a b^T;  p_tu = near l^{t-u} s_tu for u <= t, as bfloat16 back into TMEM;  near part  n = p c
//   far     f = a S with the matrix S of what lies before, in shared memory as two planes of bfloat16 (16 bits)
//   out_t = n_t + far l^{t+1} f_t
//   matrix  b'_u = l^{count-1-u} b_u as bfloat16, in place of b;  S = l^count S + b'^T c, in FP32 in registers
// (going backwards: the decays counted from the other end, decay_attention.cuh). p and b' are rounded once each, which costs
// an output about as much as its own rounding: 1.4 of it in all. One plane of S would cost as much again.
//
// float32: a, b, c, p, b' and S are three planes each (24 bits) and a product is the six of its planes that count, the
// small ones first. There is room for heads of up to 64 values. Wider ones go in parts of 64, since the output is linear in the
// pairs: its values fall into two (blocks of their own), a . b into two sums, of which a second launch adds the second to the
// output that the first one left.
//
// states_kernel does the last line alone, for what a segment adds to the matrix or for the matrix behind a sequence; in
// bfloat16 with three planes of b' where the matrix itself is a result, so that it is exact to FP32. There is room for one
// chunk's planes, so a chunk goes by halves: one half's rows are weighed while the other's products run, and its sums are
// taken a chunk later.
//
// Warps, after the workers (16 of them: thread = row of the chunk and a part of the pairs or columns; for the matrix
// its row, and a part of its columns):
//   TMA: a, b, c of one chunk after the other through a ring of slots; the output out of c's slot before that is filled again
//   (the last chunk's rows by the workers themselves)
//   one thread issues the products, each as soon as what it needs is there: f (S of this chunk), b'^T c (b'), n (p), s of the
//   next chunk. What goes from chunk to chunk is S alone: while f runs the workers weigh the pairs.
// What lies in TMEM: s and p in its place (each thread overwrites what it has read), n, f, b'^T c.
//
// Three of four blocks of 32 x 32 pairs lie to one side of the diagonal: nothing is computed above it, and below it a weight
// is the product of one factor of the row and one of the column (a table), l^{t-u} = l^{t-a} l^{a-u}, neither above 1.
//
// Rows of a tile that lie behind a chunk's end belong to others: their pairs are zeros, b' is zero there, and c is set to
// zero, whatever their values.
//
// What bounds it. A chunk among those of all SMs, whole sequences of one length, at 1,965 MHz: a head of 128 in bfloat16 3.5 us,
// with 5.4 TB/s of memory, a float32 head of 64 6.1 us; and a block takes some 6 us besides, for its offsets, TMEM, first copies
// and last output, in which its SM does nothing else (148 blocks of 1, 4 and 16 chunks 9.3, 19.6 and 62.7 us; eight times as many
// of 1 chunk 74). By itself a chunk is bound by the traffic of shared memory, 128 bytes a cycle: in bfloat16 the products'
// operands 2,300 cycles (f, with two planes of S, 1,000), copies in and out 1,000, what the workers read and write 1,300 (b' and
// S 500 each, the output 250), of 5,500 (products alone 2,560); in float32 5,000, 1,400 and 1,200 of about 9,000. Not in this
// account: the registers that heads of 128 spill, 160 bytes stored and 140 read a thread, up to 1,200 cycles were all of them
// in the walk. Measured and not kept: eight workers for the pairs and the output beside eight for the matrix (rows of 50,000 x 16
// heads of 128: 163 -> 200 us), one lane that waits for its warp (163 -> 170).
//
// Every wait is bounded: on expiry the block raises FMD_FLAG_WAIT_TIMEOUT, waits (bounded) for its copies and products in
// flight, frees its TMEM and returns.

#include "decay_attention.cuh"
#include "packed_attention_mma.cuh"

namespace fmd {
namespace {

// KS: steps of 16 of a head, rounded up. P: planes of what is given.
template <int KS, int P>
struct Shape {
    static constexpr int kDim = 16 * KS;
    static constexpr int kPanels = (KS + 3) / 4;
    static constexpr uint32_t kTileBytes = kPanels * kPanelBytes;  // of a plane
    static constexpr uint32_t kSlotBytes = P * kTileBytes;
    // Rows of the product that the matrix is summed up by: 64 are enough for heads of up to 64 values, and read half as much of
    // b'. They lie in the first 16 lanes of each of TMEM's quarters.
    static constexpr int kRows = KS <= 4 ? 64 : 128;
    static constexpr uint32_t kSumDesc = (uint32_t(kRows) >> 4) << 24 | 1u << 15;
    // The row of the matrix that a thread holds, or kDim for none.
    __device__ static int matrix_row() {
        const int quarter = int(threadIdx.x >> 5) & 3, lane = int(threadIdx.x) & 31;
        if (KS > 4) return quarter * 32 + lane < kDim ? quarter * 32 + lane : kDim;
        return lane < 16 && quarter * 16 + lane < kDim ? quarter * 16 + lane : kDim;
    }
};

template <int KS, int P>
struct RowsShape : Shape<KS, P> {
    using S = Shape<KS, P>;
    // Sixteen workers hide each other's waits: two blocks an SM of eight each, which heads of up to 64 values in bfloat16 leave
    // room for, took up to 9 % longer (4 sequences of 3,000 to 8,000 rows, 8 heads of 64, forward and backward: 233 us, 214).
    static constexpr int kGroups = 4, kWorkers = 128 * kGroups, kThreads = kWorkers + 64;
    static constexpr int kColumns = S::kDim / kGroups, kPairs = kTile / kGroups;  // of a thread
    static constexpr int kSize = P == 3 ? 4 : 2, kOutPanels = (S::kDim * kSize + 127) / 128;  // of the output
    static constexpr int kSlots = P == 3 ? 4 : 5;
    static constexpr int kPlanes = P == 3 ? 3 : 2;           // of the matrix
    static constexpr uint32_t kPanel = S::kDim * 128;        // of the matrix: kDim rows x 64 columns
    static constexpr uint32_t kPlane = S::kPanels * kPanel;
    static constexpr uint32_t kMatrix = kPlanes * kPlane;
    static constexpr size_t kBytes = kSlots * S::kSlotBytes + kMatrix + 1024;
    // columns: the pairs at 0, their third plane, n, f, and b'^T c
    static constexpr uint32_t kTmem = 512;
    static constexpr uint32_t kThird = 128, kNear = kThird + (P == 3 ? 64 : 0), kFar = kNear + S::kDim, kSum = kFar + S::kDim;
};

// PLANES: of b'.
template <int KS, int P, int PLANES>
struct StatesShape : Shape<KS, P> {
    using S = Shape<KS, P>;
    static constexpr int kGroups = 4, kWorkers = 128 * kGroups, kThreads = kWorkers + 64;
    static constexpr int kColumns = S::kDim / kGroups;
    static constexpr int kMore = PLANES - P;                 // planes of b' beside the slots
    static constexpr int kSlots = P == 3 || PLANES == 3 ? 4 : 6;
    static constexpr size_t kBytes = kSlots * S::kSlotBytes + kMore * S::kTileBytes + 1024;
    static constexpr uint32_t kTmem = KS <= 2 ? 64 : KS <= 4 ? 128 : 256;  // two sums by turns
};

// stored: of two chunks by turns. Nothing but the time of a copy keeps the workers from finishing the next chunk before the
// warp that copies has looked at the last one; they cannot finish two, since the copies of the second come after that look.
template <int SLOTS>
struct Ctrl {
    Ring<SLOTS> ring;
    uint64_t pairs, far, ready, weights, added, out, matrix, stored[2];
    uint64_t drain;
    uint32_t tmem;
    int32_t abort;
};

// ready, freed: of the halves of a chunk; added, taken: of two sums by turns, since nobody may run a phase of a barrier ahead of
// a wait that has not looked yet.
template <int SLOTS>
struct StatesCtrl {
    Ring<SLOTS> ring;
    uint64_t ready[2], freed[2], added[2], taken[2];
    uint64_t drain;
    uint32_t tmem;
    int32_t abort;
};

struct Maps {
    CUtensorMap a, b, c, out;
};

struct AllMaps {
    Maps m[3];
};

// The planes of a product of two operands of three planes each, the small ones first.
__device__ constexpr int first_plane(int q) { return q == 0 ? 2 : q == 1 || q == 3 ? 1 : 0; }
__device__ constexpr int second_plane(int q) { return q == 2 ? 2 : q == 1 || q == 4 ? 1 : 0; }

__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 u, v;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 u, {%1, %3};\n\t"
        "mov.b64 v, {%2, %3};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], u, v, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(kDescHigh), "r"(idesc), "r"(uint32_t(add))
        : "memory");
}

// D (+)= A^T B over steps [from, to) of 16 rows of both: the columns of A are the product's M index.
__device__ __forceinline__ void product_columns(uint32_t d, uint32_t a, uint32_t b, int from, int to, uint32_t idesc, bool add) {
    const uint32_t ad = columns_desc(a), bd = columns_desc(b);
    for (int k = from; k < to; ++k) mma(d, ad + k * 128, bd + k * 128, idesc, add || k > from);
}

// D (+)= A B: the rows of A the product's M index, those of B (panels `panel` bytes apart) its inner index.
template <int KS>
__device__ __forceinline__ void product_matrix(uint32_t d, uint32_t a, uint32_t b, uint32_t panel, uint32_t idesc, bool add) {
    const uint32_t ad = rows_desc(a), bd = ((b & 0x3FFFFu) >> 4) | ((panel >> 4) << 16);
#pragma unroll
    for (int k = 0; k < KS; ++k)
        mma(d, ad + uint32_t(k / 4) * kPanelStep + uint32_t(k % 4) * 2, bd + k * 128, idesc, add || k > 0);
}

template <int N>
__device__ __forceinline__ void tmem_read(uint32_t at, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i + 16 <= N; i += 16) tmem_load16(at + i, reinterpret_cast<float(&)[16]>(v[i]));
    if constexpr (N % 16 != 0) tmem_load8(at + N / 16 * 16, reinterpret_cast<float(&)[8]>(v[N / 16 * 16]));
}

__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// Two bfloat16 times a weight in two planes, rounded once (but for 2^-18).
__device__ __forceinline__ uint32_t times(uint32_t x, uint32_t high, uint32_t low) {
    uint32_t y;
    asm("{\n\t.reg .b32 t;\n\tmul.rn.bf16x2 t, %1, %3;\n\tfma.rn.bf16x2 %0, %1, %2, t;\n\t}"
        : "=r"(y)
        : "r"(x), "r"(high), "r"(low));
    return y;
}

// Row r of a tile of P planes times `weight` as OUT planes: the first P in place, the others from `more` on. A group takes
// eights that lie side by side, in an order that keeps the banks apart; the swizzle moves eights within a panel's row.
template <int KS, int P, int OUT, int GROUPS>
__device__ __forceinline__ void weigh_row(unsigned char* tile, unsigned char* more, int r, int group, float weight, bool real) {
    using S = Shape<KS, P>;
    constexpr int kEach = 8 * S::kPanels / GROUPS;
    const float2 w2 = twice(real ? weight : 0.0f);
    const uint32_t high = pack_bf16(w2.x, w2.x), low = pack_bf16(w2.x - unpack_bf16(high).x, w2.x - unpack_bf16(high).x);
    uint32_t at[kEach];
    uint4 x[kEach][P];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int eight = group * kEach + i;
        at[i] = uint32_t(eight / 8) * kPanelBytes + uint32_t(r) * 128 + uint32_t(((eight % 8) ^ (r & 7)) * 16);
#pragma unroll
        for (int q = 0; q < P; ++q) {
            x[i][q] = *reinterpret_cast<const uint4*>(tile + q * S::kTileBytes + at[i]);
            if (!real) x[i][q] = make_uint4(0, 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if constexpr (OUT == 1) {
            *reinterpret_cast<uint4*>(tile + at[i]) = make_uint4(times(x[i][0].x, high, low), times(x[i][0].y, high, low),
                                                                 times(x[i][0].z, high, low), times(x[i][0].w, high, low));
        } else {
            float2 v[4];
#pragma unroll
            for (int q = P - 1; q >= 0; --q) {  // exact: the planes are the parts of one FP32 number, the small ones first
                const float2 y[4] = {unpack_bf16(x[i][q].x), unpack_bf16(x[i][q].y), unpack_bf16(x[i][q].z),
                                     unpack_bf16(x[i][q].w)};
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = q == P - 1 ? y[e] : add2(v[e], y[e]);
            }
            float y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = mul2(v[e], w2);
                y[2 * e] = v[e].x;
                y[2 * e + 1] = v[e].y;
            }
#pragma unroll
            for (int q = 0; q < OUT; ++q) {
                const uint4 w = q + 1 == OUT ? pack8(y) : q == 0 && P == 3 ? first_plane8(y) : next_plane8(y);
                *reinterpret_cast<uint4*>((q < P ? tile + q * S::kTileBytes : more + (q - P) * S::kTileBytes) + at[i]) = w;
            }
        }
    }
}

// The thread's row of the matrix, columns from col0 on: as planes in shared memory.
template <int KS, int P, int N>
__device__ __forceinline__ void store_matrix(unsigned char* to, int r, int col0, const float (&state)[N]) {
    using S = RowsShape<KS, P>;
#pragma unroll
    for (int i = 0; i < N; i += 8) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = state[i + e];
        const int eight = (col0 + i) / 8;
        unsigned char* p = to + (eight / 8) * S::kPanel + r * 128 + ((eight % 8) ^ (r & 7)) * 16;
#pragma unroll
        for (int q = 0; q < S::kPlanes; ++q)
            *reinterpret_cast<uint4*>(p + q * S::kPlane) =
                q + 1 == S::kPlanes ? pack8(v) : q == 0 && P == 3 ? first_plane8(v) : next_plane8(v);
    }
}

// state = keep state + N columns of TMEM.
template <int N>
__device__ __forceinline__ void add_columns(uint32_t at, float keep, float (&state)[N]) {
    float x[N];
    tmem_read(at, x);
    const float2 k = twice(keep);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const float2 y = fma2(k, make_float2(state[e], state[e + 1]), make_float2(x[e], x[e + 1]));
        state[e] = y.x;
        state[e + 1] = y.y;
    }
}

template <int SLOTS>
__device__ __forceinline__ void open_block(Ctrl<SLOTS>& ctl, int workers) {
    if (threadIdx.x == 0) {
        init_ring(ctl.ring);
        mbar_init(&ctl.pairs, 1);
        mbar_init(&ctl.far, 1);
        mbar_init(&ctl.ready, uint32_t(workers));
        mbar_init(&ctl.weights, uint32_t(workers));
        mbar_init(&ctl.added, 1);
        mbar_init(&ctl.out, 1);
        mbar_init(&ctl.matrix, uint32_t(workers));
        for (int i = 0; i < 2; ++i) mbar_init(&ctl.stored[i], uint32_t(workers));
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
}

// The copies of a walk, tile i by load(i, slot, barrier); then until their slots are released, or have landed.
template <typename Control, typename Load>
__device__ __forceinline__ void feed_tiles(Control& ctl, volatile int32_t* abort, int count, uint32_t bytes, Load load) {
    constexpr int SLOTS = sizeof(ctl.ring.full) / sizeof(ctl.ring.full[0]);
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

// One tile: P planes of `panels` panels each, rows from `row` on of `all`, the head's values from `first` on.
template <int KS, int P>
__device__ __forceinline__ void load_tile(uint32_t to, const CUtensorMap* map, uint64_t* bar, int head, int64_t row,
                                          int64_t all, int first) {
    using S = Shape<KS, P>;
    for (int q = 0; q < P; ++q)
        for (int p = 0; p < S::kPanels; ++p)
            tma_load_4d(to + q * S::kTileBytes + p * kPanelBytes, map, bar, first + p * 64, 0, head, int(q * all + row));
}

// The values of a head in parts of 64 (float32 heads of more than that): those of c and the output, and those of a and b, which
// each add to the output.
__host__ __device__ constexpr int parts_of(int planes, int dim) { return planes == 3 && dim > 64 ? 2 : 1; }

// Adds a tile of shared memory to memory.
__device__ __forceinline__ void tma_add_4d(const CUtensorMap* map, uint32_t src, int x, int y, int z, int w) {
    asm volatile("cp.reduce.async.bulk.tensor.4d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}

// What store_pieces overwrites next, added to the pieces (FP32).
template <int W>
__device__ __forceinline__ void add_pieces(uint4 (&w)[W], const void* from, int64_t stride, int rows, int pieces) {
    const int lane = threadIdx.x & 31, left = lane % W < pieces ? rows - lane / W : 0;
    const char* p = static_cast<const char*>(from) + (lane / W) * stride + (lane % W) * 16;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (i * (32 / W) < left) {
            const float4 x = *reinterpret_cast<const float4*>(p);
            w[i] = make_uint4(__float_as_uint(__uint_as_float(w[i].x) + x.x), __float_as_uint(__uint_as_float(w[i].y) + x.y),
                              __float_as_uint(__uint_as_float(w[i].z) + x.z), __float_as_uint(__uint_as_float(w[i].w) + x.w));
        }
        p += (32 / W) * stride;
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

// What a stretch starts from: row r of the matrix (dim or more: none), columns from col0 on.
template <int N>
__device__ __forceinline__ void load_start(const Decay& d, const Stretch& s, int head, int r, int col0, float (&state)[N]) {
    const float* from = start_of(d, s, head);
    const bool turn = d.length >= kWhole && d.transposed, here = from != nullptr && r < d.dim;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const int col = col0 + i;
        float4 x = f4_zero();
        if (here && col < d.dim) {
            if (turn) {
                const float* p = from + col * d.dim + r;
                x = make_float4(p[0], p[d.dim], p[2 * d.dim], p[3 * d.dim]);
            } else {
                x = ldg4(from + r * d.dim + col);
            }
        }
        state[i] = x.x, state[i + 1] = x.y, state[i + 2] = x.z, state[i + 3] = x.w;
    }
}

// Chunk i of a stretch: its rows, and the first of them.
struct Walk {
    int row0, rows, chunks, later;
    __device__ __forceinline__ Walk(const Stretch& s, const Decay& d)
        : row0(int(s.row0)), rows(int(s.rows)), chunks((rows + kTile - 1) / kTile), later(d.later) {}
    __device__ __forceinline__ int count(int i) const { return min(kTile, rows - i * kTile); }
    __device__ __forceinline__ int first(int i) const { return later ? row0 + max(0, rows - (i + 1) * kTile) : row0 + i * kTile; }
};

// us: 50,000 rows, 16 heads of 128 in bfloat16, in segments 162 (802 MB, 5.0 TB/s); 16 sequences of 100 to 2,000 rows, 16 heads
// of 128, the output 66 (256 blocks of up to 16 chunks on 148 SMs) and three gradients 178; in float32 64 sequences of 100 to
// 500 rows, 8 heads of 64, 88 and 225, heads of 128 four times that (1,275 with the planes; 2,700 on the FP32 cores).
// part: of a's and b's values.
template <int KS, int P>
__global__ void __launch_bounds__(RowsShape<KS, P>::kThreads, 1)
    rows_kernel(const __grid_constant__ AllMaps all_maps, const __grid_constant__ Decays all, const int part) {
    using S = RowsShape<KS, P>;
    constexpr int kColumns = S::kColumns, kFeeder = S::kWorkers / 32;
    extern __shared__ unsigned char raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* matrix = ring + S::kSlots * S::kSlotBytes;
    __shared__ Ctrl<S::kSlots> ctl;
    // near l^n at 31 + n, zeros before it; and the factors of the columns of a block of 32 pairs: l^{31 - e}, backwards l^e
    __shared__ alignas(16) float powers[64], table[32];
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned which = blockIdx.x % unsigned(all.count), place = blockIdx.x / unsigned(all.count);
    const Decay& d = all.d[which];
    const Maps& maps = all_maps.m[which];
    const unsigned parts = parts_of(P, d.dim);
    const int head = int(place / parts % unsigned(d.heads)), first_in = 64 * part, first_out = 64 * int(place % parts);
    const int64_t index = place / parts / unsigned(d.heads);

    if (threadIdx.x < 32) {
        const float l2 = log2_decay(d, head);
        table[lane] = exp2f(float(d.later ? lane : 31 - lane) * l2);
        if (lane < 31) powers[lane] = 0.0f;
        powers[lane + 31] = d.near * exp2f(float(lane) * l2);
    }
    if (head == 0 && threadIdx.x == 32 && index < d.batch) check_offsets(d, index);
    const Stretch s = block_stretch(d, index);
    if (s.rows == 0) {
        wait_for_the_kernel_ahead();
        return;
    }
    const Walk walk(s, d);
    open_block(ctl, kFeeder);
    if (warp == kFeeder + 1) tmem_alloc<S::kTmem>(&ctl.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    dependents_may_start();  // with this block's TMEM in hand: they take theirs and hold it until this kernel ends
    wait_for_the_kernel_ahead();

    if (warp == kFeeder) {
        if (lane == 0) {
            const int tiles = 3 * walk.chunks;
            uint32_t phases = 0;  // of the slots' releases after a and b
            // tile i's slot is free again: after c's, once the output has left it
            auto released = [&](int i) {
                const int slot = i % S::kSlots, chunk = i / 3;
                if (i % 3 != 2) {
                    const bool got = mbar_wait(&ctl.ring.empty[slot], phases >> slot & 1u, abort);
                    phases ^= 1u << slot;
                    return got;
                }
                if (!mbar_wait(&ctl.stored[chunk & 1], uint32_t(chunk >> 1) & 1u, abort)) return false;
                if (walk.count(chunk) == kTile) {
                    for (int p = 0; p < S::kOutPanels; ++p) {
                        const uint32_t from = su32(ring + slot * S::kSlotBytes + p * kPanelBytes);
                        const int x = first_out + p * (128 / S::kSize);
                        if (x >= d.dim) break;
                        if (P == 3 && part > 0) tma_add_4d(&maps.out, from, x, 0, head, walk.first(chunk));
                        else tma_store_4d(&maps.out, from, x, 0, head, walk.first(chunk));
                    }
                    asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
                }
                return true;
            };
            bool ok = true;
            int armed = 0;
            for (int i = 0; i < tiles && ok; ++i) {
                const int slot = i % S::kSlots, chunk = i / 3, what = i - 3 * chunk;
                if (i >= S::kSlots && !(ok = released(i - S::kSlots))) break;
                mbar_expect_tx(&ctl.ring.full[slot], S::kSlotBytes);
                load_tile<KS, P>(su32(ring + slot * S::kSlotBytes), what == 0 ? &maps.a : what == 1 ? &maps.b : &maps.c,
                                 &ctl.ring.full[slot], head, walk.first(chunk), d.rows, what == 2 ? first_out : first_in);
                armed = i + 1;
            }
            for (int i = max(0, armed - S::kSlots); i < armed; ++i) {
                if (ok) ok = released(i);
                if (!ok) mbar_wait(&ctl.ring.full[i % S::kSlots], uint32_t(i / S::kSlots) & 1u, abort, true);
            }
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    } else if (warp > kFeeder) {
        const uint32_t base = uniform(tmem), first_slot = uniform(su32(ring)), planes = uniform(su32(matrix));
        const int count = uniform(walk.chunks), last = uniform(walk.count(walk.chunks - 1));
        const uint32_t pairs_desc = bf16_idesc(kTile, false), out_desc = bf16_idesc(S::kDim, true),
                       add_desc = (out_desc & 0xFFFFFFu) | S::kSumDesc;
        auto slot = [&](int i) { return first_slot + uint32_t(i % S::kSlots) * S::kSlotBytes; };
        bool ok = true, issued = false;
        auto pairs = [&](int i) {  // over pairs whose product has been issued
            ok = ok && landed(ctl.ring, 3 * i, abort) && landed(ctl.ring, 3 * i + 1, abort);
            if (!ok) return;
            tc_fence_after();
            const uint32_t a = slot(3 * i), b = slot(3 * i + 1);
            if (elect_one()) {
                if (P == 1) {
                    product_rows<KS>(base, a, b, pairs_desc);
                } else {
#pragma unroll
                    for (int q = 0; q < 6; ++q)
                        product_rows<KS>(base, a + first_plane(q) * S::kTileBytes, b + second_plane(q) * S::kTileBytes,
                                         pairs_desc, q > 0);
                }
                tc_commit(&ctl.pairs);
            }
            issued = true;
        };
        pairs(0);
        for (int i = 0; i < count && ok; ++i) {
            ok = warp_wait(&ctl.matrix, uint32_t(i) & 1u, abort);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a = slot(3 * i), b = slot(3 * i + 1), c = slot(3 * i + 2);
            const uint32_t far = base + S::kFar, near = base + S::kNear, sum = base + S::kSum;
            if (elect_one()) {
                if (P == 1) {
                    product_matrix<KS>(far, a, planes + S::kPlane, S::kPanel, out_desc, false);
                    product_matrix<KS>(far, a, planes, S::kPanel, out_desc, true);
                } else {
#pragma unroll
                    for (int q = 0; q < 6; ++q)
                        product_matrix<KS>(far, a + first_plane(q) * S::kTileBytes, planes + second_plane(q) * S::kPlane,
                                           S::kPanel, out_desc, q > 0);
                }
                tc_commit(&ctl.far);
                tc_commit(&ctl.ring.empty[(3 * i) % S::kSlots]);
            }
            ok = landed(ctl.ring, 3 * i + 2, abort) && warp_wait(&ctl.ready, uint32_t(i) & 1u, abort);
            if (!ok) break;
            tc_fence_after();
            const int steps = ((i + 1 == count ? last : kTile) + 15) / 16;
            if (elect_one()) {
#pragma unroll
                for (int q = P == 1 ? 5 : 0; q < 6; ++q)
                    product_columns(sum, b + first_plane(q) * S::kTileBytes, c + second_plane(q) * S::kTileBytes, 0, steps,
                                    add_desc, P != 1 && q > 0);
                tc_commit(&ctl.added);
                tc_commit(&ctl.ring.empty[(3 * i + 1) % S::kSlots]);
            }
            ok = ok && warp_wait(&ctl.weights, uint32_t(i) & 1u, abort);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                if (P == 1) {
                    product_weights<8, S::kPairs / 16, S::kPairs>(near, base, c, steps, out_desc, false);
                } else {
#pragma unroll
                    for (int q = 0; q < 6; ++q) {
                        const uint32_t from = c + second_plane(q) * S::kTileBytes;
                        if (first_plane(q) == 2)
                            product_weights<8, 8, 0>(near, base + S::kThird, from, steps, out_desc, q > 0);
                        else
                            product_weights<8, 2, 32>(near, base + 16 * first_plane(q), from, steps, out_desc, q > 0);
                    }
                }
                tc_commit(&ctl.out);
            }
            if (i + 1 < count) pairs(i + 1);  // not before n: the workers wait for that (5 % slower)
        }
        if (!ok && issued) {  // the products in flight end before TMEM is freed
            if (elect_one()) tc_commit(&ctl.drain);
            warp_wait(&ctl.drain, 0, abort, true);
        }
    } else {
        using T = typename std::conditional<P == 1, __nv_bfloat16, float>::type;
        const int group = warp >> 2, r = threadIdx.x & 127, col0 = group * kColumns, pair0 = group * S::kPairs;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t at_pairs = tmem + lanes + pair0, at_third = tmem + lanes + S::kThird + pair0 / 2;
        const uint32_t at_near = tmem + lanes + S::kNear + col0, at_far = tmem + lanes + S::kFar + col0,
                       at_sum = tmem + lanes + S::kSum + col0;
        const float l2 = log2_decay(d, head);
        auto power = [&](int n) { return P == 1 ? ex2(float(n) * l2) : exp2f(float(n) * l2); };
        const int matrix_row = S::matrix_row();
        const bool holds = matrix_row < S::kDim;
        float state[kColumns];
        load_start(d, s, head, holds ? first_in + matrix_row : d.dim, first_out + col0, state);
        if (holds) store_matrix<KS, P>(matrix, matrix_row, col0, state);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        warp_arrive(&ctl.matrix);
        // the weights of 32 pairs from column `first` on
        auto weigh_pairs = [&](int first, int count, float(&x)[32]) {
            const int beside = (first / 32 - (warp & 3)) * (d.later ? -1 : 1);  // blocks above the diagonal
            if (beside < 0 && first + 32 <= count) {
                const float2 row = twice(d.near * power(d.later ? first - r : r - first - 31));
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(table + e);
                    const float2 u = mul2(make_float2(x[e], x[e + 1]), mul2(row, make_float2(y.x, y.y)));
                    const float2 v = mul2(make_float2(x[e + 2], x[e + 3]), mul2(row, make_float2(y.z, y.w)));
                    x[e] = u.x, x[e + 1] = u.y, x[e + 2] = v.x, x[e + 3] = v.y;
                }
            } else {
                // on the diagonal, or in the last chunk: the pairs of the columns [from, to)
                const int t = r - first, from = d.later ? max(0, t) : 0, to = min(count - first, d.later ? 32 : t + 1);
                const uint32_t seen = to > from ? (to >= 32 ? 0xffffffffu : (1u << to) - 1u) & (0xffffffffu << from) : 0u;
                // every weight is computed and then chosen: a choice of what to compute would be a branch for every pair
                float w[32];
                if (beside == 0) {
                    const float* from_t = powers + 31 + (d.later ? -t : t);
                    const int step = d.later ? 1 : -1;
#pragma unroll
                    for (int e = 0; e < 32; ++e) w[e] = from_t[step * e];
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) w[e] = d.near * power(d.later ? e - t : t - e);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float y = x[e] * w[e];
                    x[e] = seen >> e & 1u ? y : 0.0f;
                }
            }
        };
        auto above = [&](int first) { return d.later ? first / 32 < (warp & 3) : first / 32 > (warp & 3); };
        // of a whole chunk; the last one has its own
        float enters = d.add * power(d.later ? r + 1 : kTile - 1 - r), keep = power(kTile),
              reach = d.far * power(d.later ? kTile - 1 - r : r + 1);
        for (int i = 0; i < walk.chunks; ++i) {
            const int count = walk.count(i);
            if (count < kTile) {
                enters = d.add * power(d.later ? r + 1 : count - 1 - r);
                keep = power(count);
                reach = d.far * power(d.later ? count - 1 - r : r + 1);
            }
            const uint32_t parity = uint32_t(i) & 1u;
            if (!worker_wait(&ctl.pairs, parity, abort)) break;
            const int tile_b = 3 * i + 1, tile_c = 3 * i + 2;
            if (!worker_wait(&ctl.ring.full[tile_b % S::kSlots], uint32_t(tile_b / S::kSlots) & 1u, abort)) break;
            tc_fence_after();
            weigh_row<KS, P, P, S::kGroups>(ring + (tile_b % S::kSlots) * S::kSlotBytes, nullptr, r, group, enters, r < count);
            if (count < kTile) {
                if (!worker_wait(&ctl.ring.full[tile_c % S::kSlots], uint32_t(tile_c / S::kSlots) & 1u, abort)) break;
                zero_rows(ring + (tile_c % S::kSlots) * S::kSlotBytes, P * S::kPanels, kPanelBytes, count, (count + 15) & ~15,
                          threadIdx.x, S::kWorkers);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(&ctl.ready);

#pragma unroll
            for (int ch = 0; ch < S::kPairs; ch += 32) {
                uint32_t p[16];
                const uint32_t at = at_pairs + (P == 1 ? ch / 2 : 0);
                if (above(pair0 + ch)) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) p[e] = 0;
#pragma unroll
                    for (int q = 0; q < P; ++q) tmem_store16(q == 2 ? at_third : at + 16 * q, p);
                    continue;
                }
                float x[32];
                tmem_load32(at_pairs + ch, x);
                weigh_pairs(pair0 + ch, count, x);
#pragma unroll
                for (int q = 0; q < P; ++q) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        const uint4 w = P == 1 ? pack8(x + e) : q == 0 ? first_plane8(x + e) : next_plane8(x + e);
                        p[e / 2] = w.x, p[e / 2 + 1] = w.y, p[e / 2 + 2] = w.z, p[e / 2 + 3] = w.w;
                    }
                    tmem_store16(q == 2 ? at_third : at + 16 * q, p);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&ctl.weights);
            if (!worker_wait(&ctl.added, parity, abort)) break;
            tc_fence_after();
            add_columns(at_sum, keep, state);

            if (!worker_wait(&ctl.far, parity, abort)) break;
            tc_fence_after();
            float far[kColumns];
            tmem_read(at_far, far);
            if (i + 1 < walk.chunks) {
                if (holds) store_matrix<KS, P>(matrix, matrix_row, col0, state);
                tc_fence_before();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                warp_arrive(&ctl.matrix);
            }

            if (!worker_wait(&ctl.out, parity, abort)) break;
            tc_fence_after();
            constexpr int kPieces = kColumns * S::kSize / 16, kWide = kPieces > 2 ? 4 : kPieces;
            uint4 row[kWide] = {};
            const float2 reach2 = twice(reach);
            constexpr int kStep = kColumns % 16 == 0 ? 16 : 8;
#pragma unroll
            for (int e = 0; e < kColumns; e += kStep) {
                float near[kStep];
                tmem_read(at_near + e, near);
#pragma unroll
                for (int o = 0; o < kStep; o += 2) {
                    const float2 y = fma2(reach2, make_float2(far[e + o], far[e + o + 1]), make_float2(near[o], near[o + 1]));
                    near[o] = y.x;
                    near[o + 1] = y.y;
                }
                constexpr int kValues = 16 / int(sizeof(T));  // of a piece
#pragma unroll
                for (int o = 0; o < kStep; o += kValues)
                    row[(e + o) / kValues] = P == 1 ? pack8(near + o)
                                                    : make_uint4(__float_as_uint(near[o]), __float_as_uint(near[o + 1]),
                                                                 __float_as_uint(near[o + 2]), __float_as_uint(near[o + 3]));
            }
            tc_fence_before();
            // by way of c's slot, which nobody reads any more: as TMA stores it, or turned for the workers' own stores. The fence
            // comes before those: it would wait for them.
            unsigned char* slot = ring + (tile_c % S::kSlots) * S::kSlotBytes;
            if (count == kTile) {
#pragma unroll
                for (int e = 0; e < kPieces; ++e) {
                    const int piece = col0 * S::kSize / 16 + e;
                    *reinterpret_cast<uint4*>(slot + (piece / 8) * kPanelBytes + r * 128 + ((piece % 8) ^ (r & 7)) * 16) = row[e];
                }
            } else {
                turn_pieces<kWide>(slot + warp * (kWide * 512), row);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(&ctl.stored[i & 1]);
            if (count < kTile) {
                const int first_row = (warp & 3) * 32, left = min(kColumns, d.dim - first_out - col0) * S::kSize / 16;
                T* out = static_cast<T*>(d.out) + (int64_t(walk.first(i) + first_row) * d.heads + head) * d.dim + first_out +
                         col0;
                if (P == 3 && part > 0)
                    add_pieces<kWide>(row, out, int64_t(d.heads) * d.dim * S::kSize, count - first_row, left);
                store_pieces<kWide>(row, out, int64_t(d.heads) * d.dim * S::kSize, count - first_row, left);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kFeeder + 1) tmem_free<S::kTmem>(tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(d.flags, FMD_FLAG_WAIT_TIMEOUT);
}

// 50,000 rows, 16 heads of 128 in bfloat16, three planes of b': 102 us (410 MB, 4.0 TB/s). A chunk's traffic of shared memory is
// 3,100 cycles, 70 us in all; the rest is the start and the waits for memory of one block an SM.
template <int KS, int P, int PLANES>
__global__ void __launch_bounds__(StatesShape<KS, P, PLANES>::kThreads, 1)
    states_kernel(const __grid_constant__ AllMaps all_maps, const __grid_constant__ Decays all) {
    using S = StatesShape<KS, P, PLANES>;
    constexpr int kColumns = S::kColumns, kFeeder = S::kWorkers / 32;
    extern __shared__ unsigned char raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* more = ring + S::kSlots * S::kSlotBytes;
    __shared__ StatesCtrl<S::kSlots> ctl;
    volatile int32_t* abort = &ctl.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned which = blockIdx.x % unsigned(all.count), place = blockIdx.x / unsigned(all.count);
    const Decay& d = all.d[which];
    const Maps& maps = all_maps.m[which];
    const unsigned parts = parts_of(P, d.dim);
    const int head = int(place / (parts * parts) % unsigned(d.heads)), first_c = 64 * int(place % parts),
              first_b = 64 * int(place / parts % parts);
    const bool whole = d.length >= kWhole;

    const Stretch s = block_stretch(d, place / (parts * parts) / unsigned(d.heads));
    if (s.rows == 0 && !whole) {
        wait_for_the_kernel_ahead();
        return;
    }
    const Walk walk(s, d);
    if (threadIdx.x == 0) {
        init_ring(ctl.ring);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl.ready[i], kFeeder / 2);
            mbar_init(&ctl.freed[i], 1);
            mbar_init(&ctl.added[i], 1);
            mbar_init(&ctl.taken[i], kFeeder);
        }
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kFeeder + 1) tmem_alloc<S::kTmem>(&ctl.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    dependents_may_start();  // with this block's TMEM in hand: they take theirs and hold it until this kernel ends
    wait_for_the_kernel_ahead();

    if (warp == kFeeder) {
        if (lane == 0)
            feed_tiles(ctl, abort, 2 * walk.chunks, S::kSlotBytes, [&](int i, int slot, uint64_t* bar) {
                load_tile<KS, P>(su32(ring + slot * S::kSlotBytes), i & 1 ? &maps.c : &maps.b, bar, head, walk.first(i >> 1),
                                 d.rows, i & 1 ? first_c : first_b);
            });
    } else if (warp > kFeeder) {
        const uint32_t base = uniform(tmem), first_slot = uniform(su32(ring)), planes = uniform(su32(more));
        const int count = uniform(walk.chunks), last = count > 0 ? uniform(walk.count(walk.chunks - 1)) : 0;
        const uint32_t desc = (bf16_idesc(S::kDim, true) & 0xFFFFFFu) | S::kSumDesc;
        auto slot = [&](int i) { return first_slot + uint32_t(i % S::kSlots) * S::kSlotBytes; };
        bool ok = true, issued = false;
        for (int i = 0; i < count && ok; ++i) {
            const uint32_t sum = base + uint32_t(i & 1) * S::kDim, b = slot(2 * i), c = slot(2 * i + 1);
            const int steps = ((i + 1 == count ? last : kTile) + 15) / 16;
            ok = landed(ctl.ring, 2 * i, abort) && landed(ctl.ring, 2 * i + 1, abort);
            if (ok && i > 1) ok = warp_wait(&ctl.taken[i & 1], (uint32_t(i >> 1) & 1u) ^ 1u, abort);
            // the planes' products number `first` to `last`, the large ones the last, over a half's rows
            constexpr int kProducts = P == 1 ? PLANES : 6;
            auto products = [&](int first, int last, int half) {
                const int from = 4 * half, to = min(4 * half + 4, steps);
#pragma unroll
                for (int q = first; q < last; ++q) {
                    const int plane = P == 1 ? PLANES - 1 - q : first_plane(q);
                    product_columns(sum, P == 1 && plane > 0 ? planes + (plane - 1) * S::kTileBytes : b + plane * S::kTileBytes,
                                    c + (P == 1 ? 0 : second_plane(q)) * S::kTileBytes, from, to, desc, half > 0 || q > 0);
                }
            };
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                ok = ok && warp_wait(&ctl.ready[half], uint32_t(i) & 1u, abort);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    // float32: small products that are added to the large one of the half before would be cut off at its last
                    // bits, twenty steps one after the other (the matrix was off by 10 units of 2^-24, and is by 2): both
                    // halves' large ones come last. In bfloat16 eight steps count little (2.1 units both ways; 3 % slower).
                    constexpr int kFirst = P == 1 ? kProducts : kProducts - 1;
                    products(0, kFirst, half);
                    tc_commit(&ctl.freed[half]);
                    if (half > 0) {
                        if (kFirst < kProducts) products(kFirst, kProducts, 0), products(kFirst, kProducts, 1);
                        tc_commit(&ctl.added[i & 1]);
                        tc_commit(&ctl.ring.empty[(2 * i) % S::kSlots]);
                        tc_commit(&ctl.ring.empty[(2 * i + 1) % S::kSlots]);
                    }
                }
                issued = true;
            }
        }
        if (!ok && issued) {
            if (elect_one()) tc_commit(&ctl.drain);
            warp_wait(&ctl.drain, 0, abort, true);
        }
    } else {
        const int group = warp >> 2, r = threadIdx.x & 127, col0 = group * kColumns;
        const uint32_t at = tmem + (uint32_t((warp & 3) * 32) << 16) + col0;
        const float l2 = log2_decay(d, head);
        float state[kColumns];
        const int matrix_row = S::matrix_row() < S::kDim ? first_b + S::matrix_row() : d.dim;  // of the whole head's
        if (whole) {
            load_start(d, s, head, matrix_row, first_c + col0, state);
        } else {
#pragma unroll
            for (int i = 0; i < kColumns; ++i) state[i] = 0.0f;
        }
        const int half = r >> 6;
        bool ok = true;
        auto take = [&](int i) {  // the sums of chunk i
            if (!worker_wait(&ctl.added[i & 1], uint32_t(i >> 1) & 1u, abort)) return false;
            tc_fence_after();
            add_columns(at + uint32_t(i & 1) * S::kDim, exp2f(float(walk.count(i)) * l2), state);
            tc_fence_before();
            warp_arrive(&ctl.taken[i & 1]);
            return true;
        };
        for (int i = 0; i < walk.chunks && ok; ++i) {
            const int count = walk.count(i), tile_b = 2 * i, tile_c = 2 * i + 1;
            ok = worker_wait(&ctl.ring.full[tile_b % S::kSlots], uint32_t(tile_b / S::kSlots) & 1u, abort);
            if (S::kMore > 0 && ok && i > 0) ok = worker_wait(&ctl.freed[half], uint32_t(i - 1) & 1u, abort);
            if (!ok) break;
            const float weight = d.add * exp2f(float(d.later ? r + 1 : count - 1 - r) * l2);
            weigh_row<KS, P, PLANES, S::kGroups>(ring + (tile_b % S::kSlots) * S::kSlotBytes, more, r, group, weight, r < count);
            if (count < kTile) {
                ok = worker_wait(&ctl.ring.full[tile_c % S::kSlots], uint32_t(tile_c / S::kSlots) & 1u, abort);
                if (!ok) break;
                const int first = max(count, 64 * half), end = min((count + 15) & ~15, 64 * half + 64);
                if (first < end)
                    zero_rows(ring + (tile_c % S::kSlots) * S::kSlotBytes, P * S::kPanels, kPanelBytes, first, end,
                              group * 64 + (r & 63), S::kWorkers / 2);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (S::kMore == 0 && i > 0) ok = worker_wait(&ctl.freed[half], uint32_t(i - 1) & 1u, abort);
            if (!ok) break;
            warp_arrive(&ctl.ready[half]);
            if (i > 0) ok = take(i - 1);
        }
        if (ok && walk.chunks > 0) ok = take(walk.chunks - 1);
        if (ok && matrix_row < d.dim) {
            const int64_t size = int64_t(d.dim) * d.dim;
            float* out = whole ? d.after + (int64_t(s.b) * d.heads + head) * size
                               : d.states + (s.index * d.heads + head) * size;
            const bool turn = whole && d.transposed;
#pragma unroll
            for (int i = 0; i < kColumns; i += 4) {
                const int col = first_c + col0 + i;
                if (col >= d.dim) break;
                if (turn) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[(col + e) * d.dim + matrix_row] = state[i + e];
                } else {
                    st4(out + matrix_row * d.dim + col, make_float4(state[i], state[i + 1], state[i + 2], state[i + 3]));
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kFeeder + 1) tmem_free<S::kTmem>(tmem);
    if (threadIdx.x == 0 && ctl.abort) raise_flag(d.flags, FMD_FLAG_WAIT_TIMEOUT);
}

// The output, [rows, heads, dim] contiguous: panels of 128 bytes and 128 rows of a head.
fmd_status encode_out(const DriverCalls& drv, CUtensorMap* map, const Decay& d, bool f32) {
    const cuuint64_t size = f32 ? 4 : 2;
    const cuuint64_t dims[4] = {cuuint64_t(d.dim), 1, cuuint64_t(d.heads), cuuint64_t(d.rows)};
    const cuuint64_t strides[3] = {d.dim * size, d.dim * size, d.heads * d.dim * size};
    const cuuint32_t box[4] = {cuuint32_t(128 / size), 1, 1, cuuint32_t(kTile)}, step[4] = {1, 1, 1, 1};
    const CUresult r = drv.encode(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, d.out, dims,
                                  strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FMD_OK : record_error_text(FMD_ERR_CUDA, "cuTensorMapEncodeTiled failed, CUresult", r);
}

fmd_status encode(AllMaps& maps, const Decays& all, bool rows, int planes) {
    const DriverCalls& drv = driver_calls();
    if (drv.encode == nullptr || drv.ctx_get_current == nullptr)
        return record_error_text(FMD_ERR_CUDA, "driver entry point cuTensorMapEncodeTiled unavailable", 0);
    fmd_status st = bind_context(drv);
    for (int i = 0; i < all.count; ++i) {
        const Decay& d = all.d[i];
        const int64_t n = d.rows * planes;
        if (st == FMD_OK && rows) st = encode_packed(drv, &maps.m[i].a, d.a, n, d.heads, 1, d.dim, d.a_row, d.a_head, kTile);
        if (st == FMD_OK && rows) st = encode_out(drv, &maps.m[i].out, d, planes == 3);
        if (st == FMD_OK) st = encode_packed(drv, &maps.m[i].b, d.b, n, d.heads, 1, d.dim, d.b_row, d.b_head, kTile);
        if (st == FMD_OK) st = encode_packed(drv, &maps.m[i].c, d.c, n, d.heads, 1, d.dim, d.c_row, d.c_head, kTile);
    }
    return st;
}

unsigned blocks_of(const Decays& d, int parts) { return unsigned(decay_segments(d.d[0]) * d.d[0].heads * d.count * parts); }

template <int KS, int P>
fmd_status launch_rows(const AllMaps& maps, const Decays& d, bool early, cudaStream_t s) {
    using S = RowsShape<KS, P>;
    const fmd_status st = grant_dynamic_smem((const void*)rows_kernel<KS, P>, S::kBytes, true);
    if (st != FMD_OK) return st;
    const int parts = parts_of(P, d.d[0].dim);
    const unsigned blocks = blocks_of(d, parts);
    if (early) {
        const fmd_status first = launch_early(rows_kernel<KS, P>, blocks, S::kThreads, S::kBytes, s, maps, d, 0);
        if (first != FMD_OK) return first;
    } else {
        rows_kernel<KS, P><<<blocks, S::kThreads, S::kBytes, s>>>(maps, d, 0);
    }
    return parts > 1 ? launch_early(rows_kernel<KS, P>, blocks, S::kThreads, S::kBytes, s, maps, d, 1) : check_launch();
}

template <int KS, int P, int PLANES>
fmd_status launch_states(const AllMaps& maps, const Decays& d, bool early, cudaStream_t s) {
    using S = StatesShape<KS, P, PLANES>;
    const fmd_status st = grant_dynamic_smem((const void*)states_kernel<KS, P, PLANES>, S::kBytes, true);
    if (st != FMD_OK) return st;
    const int parts = parts_of(P, d.d[0].dim);
    const unsigned blocks = blocks_of(d, parts * parts);
    if (early) return launch_early(states_kernel<KS, P, PLANES>, blocks, S::kThreads, S::kBytes, s, maps, d);
    states_kernel<KS, P, PLANES><<<blocks, S::kThreads, S::kBytes, s>>>(maps, d);
    return check_launch();
}

template <int KS>
fmd_status launch_states(const AllMaps& maps, const Decays& d, bool early, cudaStream_t s) {
    bool after = false;
    for (int i = 0; i < d.count; ++i) after = after || d.d[i].after != nullptr;
    return after ? launch_states<KS, 1, 3>(maps, d, early, s) : launch_states<KS, 1, 1>(maps, d, early, s);
}

}  // namespace

fmd_status decay_states_mma(const Decays& d, bool early, cudaStream_t s) {
    AllMaps maps{};
    const fmd_status st = encode(maps, d, false, 1);
    if (st != FMD_OK) return st;
    const int dim = d.d[0].dim;
    return dim <= 32 ? launch_states<2>(maps, d, early, s) : dim <= 64 ? launch_states<4>(maps, d, early, s)
         : dim <= 96 ? launch_states<6>(maps, d, early, s) : launch_states<8>(maps, d, early, s);
}

fmd_status decay_rows_mma(const Decays& d, bool early, cudaStream_t s) {
    AllMaps maps{};
    const fmd_status st = encode(maps, d, true, 1);
    if (st != FMD_OK) return st;
    const int dim = d.d[0].dim;
    return dim <= 32 ? launch_rows<2, 1>(maps, d, early, s) : dim <= 64 ? launch_rows<4, 1>(maps, d, early, s)
         : dim <= 96 ? launch_rows<6, 1>(maps, d, early, s) : launch_rows<8, 1>(maps, d, early, s);
}

fmd_status decay_states_planes(const Decays& d, bool early, cudaStream_t s) {
    AllMaps maps{};
    const fmd_status st = encode(maps, d, false, 3);
    if (st != FMD_OK) return st;
    return d.d[0].dim <= 32 ? launch_states<2, 3, 3>(maps, d, early, s) : launch_states<4, 3, 3>(maps, d, early, s);
}

fmd_status decay_rows_planes(const Decays& d, bool early, cudaStream_t s) {
    AllMaps maps{};
    const fmd_status st = encode(maps, d, true, 3);
    if (st != FMD_OK) return st;
    return d.d[0].dim <= 32 ? launch_rows<2, 3>(maps, d, early, s) : launch_rows<4, 3>(maps, d, early, s);
}

}  // namespace fmd
