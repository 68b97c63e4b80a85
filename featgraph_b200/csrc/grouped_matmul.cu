// Products grouped by expert (node type, relation): y[p] = W[g(p)] x[row(p)] for the rows p of each group, the same with
// the weight read the other way for the gradient of x, and dW[g] = sum over p of dy[p] x[row(p)]^T.
//
// Bound: the tensor cores where groups have many rows, the weights' bytes where they have few.  The groups' sizes are on
// the device only, so a launch covers every way they can fall: persistent blocks, one an SM, scan the offsets into
// shared memory once (a microsecond) and walk a numbering of 128-row tiles that never span two groups.
//
// Warp 0 of a block loads: 128-byte wide tiles of both operands through TMA into a ring of stages.  Warp 1 issues tcgen05
// products of 128 x BN x 32 bytes into one of two accumulators in tensor memory; both through one thread that elect.sync
// picks (under `lane == 0` a stage cost the issuing thread 570 cycles instead of 400).  Warps 2 to 9 take a finished
// accumulator to the output while the other one fills.
//
// Rows of a tile beyond its group's end belong to the next group (or to nothing): in y they are computed and not
// stored.  In dW they would be terms of the sum, so they are overwritten with zeros in shared memory, in both
// operands - a zero times their infinities or NaN would still be NaN - by a warp of its own as the group's last chunk
// lands (by the warp that issues the products it took them 3000 cycles a tile).
//
// fp32: no tensor-core type holds it, so x and w are each cut into three bf16 parts (x = a + b + c exactly, but for bits below
// 2^-133, bf16's smallest step) and six products of parts are summed, smallest first: a c', b b', c a', a b', b a', a a'.
// a and b are rounded to nearest, so |b| <= 2^-8 |x| and |c| <= 2^-17 |x|, and what is left out, b c', c b' and c c', is below
// 2^-23.9 of a term and of either sign; parts that were cut off instead all had x's sign and left out up to 2^-21, always
// towards zero.  Six bf16 products against one fp32 product on the scalar units.  The tensor cores cut the
// sum off at 24 bits at each step, always towards zero, which adds up: summed through a whole inner axis, 704 x 6
// / 16 steps left dW 5e-6 off, against 1e-6 for a library's fp32 product.  So an accumulator holds the products of one
// chunk of 64 - the five small ones first, then four steps at full size - and the output warps add the chunks in
// registers, rounding to nearest.
//
// Rows that are gathered (slot p reads row order[p] / choices) are first copied into slot order, unless there are few columns
// (rows_gathered): every column tile reads them again, and row-gather TMA loads (tile::gather4, four rows an instruction) move a
// 128-row tile at a fraction of the tile loads' rate.  Measured at 65536 x 2048 x 4096 in bf16: 2767 us with gather loads in
// the ring, 922 us for rows in slot order, the copy about 70 us; dW 8512 against 1241 us.  The same kernel copies an
// operand that TMA cannot read (a row pitch or a start off the 16-byte grid, two strides above 1) and cuts fp32 into parts.
#include <atomic>
#include <climits>
#include <mutex>
#include <type_traits>

#include "rows.cuh"
#include "tcgen05.cuh"

namespace {

using fg::from_f32;
using fg::Pack;
using fg::store_pack;
using fg::to_f32;

constexpr int kTileRows = 128, kChunkBytes = 128, kMaxGroups = 1024, kSuperRows = 16;

__device__ int g_stuck;  // set when a wait ran out; fg_wait_status reads it

struct MmaArgs {
    const int32_t *offsets, *order;
    const float *x_scales, *w_scales;
    void* y;              // output rows, dW, or partial sums of dW
    int64_t m, x_rows;    // slots; rows of x
    int32_t choices, groups, inner, outer;  // inner: the summed axis (y) or x's width (dW); outer: width of y
    int32_t out_type, format;
    bool b_mn, shared_weight;
    int32_t split;        // dW: rows of one partial sum (0: a group's rows in one)
    int32_t units;        // dW: partial sums that there is room for
    // few rows
    const void* x;
    int64_t ldx;
    int32_t stages, held;  // stages of weights; bytes of the rows
    bool vector_rows;      // rows on the 16-byte grid
    bool gather;           // rows fetched from where they lie
};

// 16-bit values, e4m3, fp32 in three bf16 parts; kCut: the weight in parts, the rows as they are, cut on their way
enum Kind { kHalf, kEight, kParts, kCut };

// Parts multiplied in each of the six products, smallest first.
__host__ __device__ constexpr int part_a(int pair) { return (0x001102 >> (4 * pair)) & 3; }
__host__ __device__ constexpr int part_b(int pair) { return (0x010120 >> (4 * pair)) & 3; }

// A stage holds 128 bytes of the summed axis of both operands, of all parts: each is loaded once for its three, two
// or one products (loaded for each product anew, 100003 x 256 x 128 took 66 us against the copy engines' rate).
//
// FEW: at most 32 slots in all.  Their rows, gathered as the block starts, stay in shared memory for all of its tiles (row =
// slot; the products read 128 rows from there on, of which those that are not stored are whatever lies behind), and the
// stages hold weights alone, 256 bytes of the summed axis each: a stage costs the thread that issues its products some 400
// cycles, in which 64 columns x 128 bytes from each of the SMs are less than the memory delivers.
//
// BLOCKS = 2: a pair of blocks computes 256 x BN; each loads 128 rows of the one operand and half the columns of the other,
// and the first one's products read both shared memories (cta_group::2).
template <int BN, Kind KIND, bool FEW, int BLOCKS>
struct Shape {
    static constexpr int kParts = KIND == Kind::kParts || KIND == kCut ? 3 : 1;
    static constexpr int kOwnCols = BN / BLOCKS;
    static constexpr int kA = FEW ? 0 : kTileRows * kChunkBytes, kB = kOwnCols * kChunkBytes;  // bytes of one part
    static constexpr int kDeep = FEW ? 2 : 1;  // 128-byte chunks a stage
    static constexpr int kStageBytes = kParts * (kA + kB) * kDeep;
    static constexpr int kStages = 196608 / kStageBytes < 16 ? 196608 / kStageBytes : 16;  // at most
    static constexpr int kColumns = 2 * BN;
    static constexpr int kOutput = 8 * 2048;  // 2 KB for each output warp
    static constexpr int kRaw = KIND == kCut ? 3 : 0, kRawBytes = kTileRows * 128;  // 32 fp32 values of each row
    static constexpr int kSmem = 1024 + kOutput + kRaw * kRawBytes + (FEW ? 196608 : kStages * kStageBytes);
};

struct Tables {
    uint64_t full[16], empty[16], tail[16], filled[2], drained[2], raw[3], spent[3], rows, last;
    uint32_t tmem;
    int stop;
    int warp_sums[19];
    int sources[32];            // few rows: the row of x behind each slot, or -1
    int start[kMaxGroups + 1];  // first slot of each group
    int tiles[kMaxGroups + 1];  // row tiles (partial sums of dW) before each group
};

// Adds this warp's share of an accumulator - every second 16 of the BN columns - to its sums.
template <int BN>
__device__ __forceinline__ void add_chunk(uint32_t tmem, float (&sums)[BN / 2], int half) {
#pragma unroll
    for (int n = 0; n < BN / 32; n += 2) {
        uint32_t raw[2][16];
#pragma unroll
        for (int u = 0; u < 2; ++u) fg::tmem_load<16>(tmem + (2 * (n + u) + half) * 16, raw[u]);
        fg::tmem_load_wait();
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[(n + u) * 16 + j] = __fadd_rn(sums[(n + u) * 16 + j], __uint_as_float(raw[u][j]));
    }
}

// Takes a warp's 32 rows of an accumulator, from `tmem` on, to the output rows from `out` on (row pitch `width`; rows
// outside [from, rows) and columns >= `left` are not stored): every second 64-byte wide piece of the BN columns, the warp's
// partner takes the others.  A thread holds a row in tensor memory's layout, so the pieces go through the warp's 2 KB of shared memory
// (16-byte cells, XOR-swizzled: no bank conflicts either way) and leave as whole sectors, 4 lanes a row.  Stored
// straight from the threads, 16 bytes in each of 32 rows at a time, or by four warps instead of eight, the output of
// products with a short inner axis keeps the tensor cores waiting.
// `sums` (SUMS): the values are there instead, in the order that add_chunk leaves them.
template <typename O, int BN, bool EIGHT, bool SUMS>
__device__ __forceinline__ void store_rows(uint32_t tmem, bool filled, const float (&sums)[BN / 2], O* out, int64_t width, int from, int rows, int left,
                                           bool vector, uint32_t staging, int half, float scale, const float* column_scales) {
    constexpr int kCols = 64 / sizeof(O), kCells = 16 / sizeof(O);
    const int lane = threadIdx.x & 31;
#pragma unroll (SUMS ? 16 : 1)
    for (int n = 0; n < BN / (2 * kCols); ++n) {
        const int c = (2 * n + half) * kCols, rest = left - c;
        if (rest <= 0) continue;
        uint32_t raw[kCols];
        if (SUMS) {
#pragma unroll
            for (int j = 0; j < kCols; ++j) raw[j] = __float_as_uint(sums[n * kCols + j]);
        } else if (filled) {
            fg::tmem_load<kCols>(tmem + c, raw);
            fg::tmem_load_wait();
        } else {
#pragma unroll
            for (int j = 0; j < kCols; ++j) raw[j] = 0;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            Pack<O, kCells> p;
#pragma unroll
            for (int j = 0; j < kCells; ++j) {
                const int k = q * kCells + j;
                float v = __uint_as_float(raw[k]);
                if (EIGHT) v = __fmul_rn(__fmul_rn(v, scale), k < rest ? column_scales[c + k] : 0.0f);
                p.v[j] = from_f32<O>(v);
            }
            const uint32_t* word = reinterpret_cast<const uint32_t*>(&p);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staging + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)), "r"(word[0]),
                         "r"(word[1]), "r"(word[2]), "r"(word[3])
                         : "memory");
        }
        __syncwarp();
        if (vector) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 2), q = lane & 3;
                Pack<uint32_t, 4> p;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(p.v[0]), "=r"(p.v[1]), "=r"(p.v[2]), "=r"(p.v[3])
                             : "r"(staging + r * 64 + ((q ^ ((r >> 1) & 3)) << 4))
                             : "memory");
                if (r >= from && r < rows && q * kCells < rest) store_pack<uint32_t, 4>(reinterpret_cast<uint32_t*>(out + r * width + c + q * kCells), p);
            }
        } else {
            constexpr int kAtOnce = 32 / kCols;  // rows side by side
            for (int r = lane / kCols; r < min(rows, 32); r += kAtOnce) {
                const int k = lane % kCols;
                const uint32_t at = staging + r * 64 + (((k / kCells) ^ ((r >> 1) & 3)) << 4) + (k % kCells) * sizeof(O);
                O v;
                if constexpr (sizeof(O) == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(*reinterpret_cast<uint32_t*>(&v)) : "r"(at) : "memory");
                else asm volatile("ld.shared.b16 %0, [%1];" : "=h"(*reinterpret_cast<uint16_t*>(&v)) : "r"(at) : "memory");
                if (r >= from && k < rest) out[r * width + c + k] = v;
            }
        }
        __syncwarp();
    }
}

// Few rows: 256 threads gather the slots' rows into shared memory, as a TMA load would lay them: 128-byte chunks of each
// row, `chunk` bytes a chunk of all, 16-byte cells XOR-swizzled, zeros beyond the inner axis and for a slot without a row.
template <bool EIGHT>
__device__ __forceinline__ void hold_rows(const MmaArgs& a, uint32_t held, int chunk, const int* sources, int thread) {
    using V = typename std::conditional<EIGHT, uint8_t, uint16_t>::type;
    constexpr int kPer = 16 / sizeof(V), kAhead = 8;
    const int pieces = (a.inner + kPer * 16 - 1) / (kPer * 16) * 16, all = (int)a.m * pieces;
    for (int first = thread; first < all; first += 256 * kAhead) {
        Pack<V, kPer> p[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = first + u * 256, r = min(i, all - 1) / pieces, k = (i - r * pieces) * kPer, source = sources[r];
            const V* x = static_cast<const V*>(a.x) + (int64_t)max(source, 0) * a.ldx + k;
            const bool in = i < all && source >= 0;
            if (in && a.vector_rows && k + kPer <= a.inner) {
                p[u] = fg::load_pack<V, kPer>(x);
            } else {
#pragma unroll
                for (int j = 0; j < kPer; ++j) p[u].v[j] = in && k + j < a.inner ? x[j] : V(0);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = first + u * 256, r = min(i, all - 1) / pieces, piece = i - r * pieces;
            if (i >= all) break;
            const uint32_t* word = reinterpret_cast<const uint32_t*>(&p[u]);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(held + (piece >> 3) * chunk + r * 128 + (((piece & 7) ^ (r & 7)) << 4)),
                         "r"(word[0]), "r"(word[1]), "r"(word[2]), "r"(word[3])
                         : "memory");
        }
    }
}

// Eight fp32 values in three bf16 parts each: x = a + b + c.  a and b are rounded to nearest by adding half a step of theirs to
// the bits (a carry into the exponent is a rounding up to the next power of two), where conversions to bf16 would run at a
// fraction of the adds' rate; c has 8 bits at most and is exact.  Where one of the eight would round up to an infinity, a is cut
// off instead: b is then up to 2^-7 of x, and the sum still exact.  An infinity's parts have a NaN among them, a NaN's too.
__device__ __forceinline__ void cut_values(const float (&v)[8], Pack<__nv_bfloat16, 8> (&p)[3]) {
    uint32_t part[3][8];
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(v[j]));
    const uint32_t half = most < 0x1.ffp127f ? 0x8000u : 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        part[0][j] = __float_as_uint(v[j]) + half;
        const float rest = __fsub_rn(v[j], __uint_as_float(part[0][j] & 0xffff0000u));
        part[1][j] = __float_as_uint(rest) + 0x8000u;
        part[2][j] = __float_as_uint(__fsub_rn(rest, __uint_as_float(part[1][j] & 0xffff0000u)));
    }
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) reinterpret_cast<uint32_t*>(&p[k])[j] = __byte_perm(part[k][2 * j], part[k][2 * j + 1], 0x7632);
}

// Half `h` of a chunk: 32 fp32 values of 128 rows at `raw` (128 bytes a row, 16-byte cells XOR-swizzled) to that half of the
// three parts' tiles at `stage`, 16 KB each, laid the same way.  256 threads, 8 values each, twice.
__device__ __forceinline__ void cut_rows(uint32_t raw, uint32_t stage, int h, int thread) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int unit = thread + u * 256, r = unit >> 2, q = unit & 3, x = r & 7;
        float v[8];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[4 * e]), "=f"(v[4 * e + 1]), "=f"(v[4 * e + 2]), "=f"(v[4 * e + 3])
                         : "r"(raw + r * 128 + (((2 * q + e) ^ x) << 4))
                         : "memory");
        Pack<__nv_bfloat16, 8> p[3];
        cut_values(v, p);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const uint32_t* word = reinterpret_cast<const uint32_t*>(&p[k]);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + k * kTileRows * kChunkBytes + r * 128 + (((h * 4 + q) ^ x) << 4)),
                         "r"(word[0]), "r"(word[1]), "r"(word[2]), "r"(word[3])
                         : "memory");
        }
    }
}

// A wait of all lanes, with one answer for all of them.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* stop) {
    return __all_sync(0xffffffffu, fg::barrier_wait(bar, parity, stop));
}

template <Kind KIND, bool WGRAD, bool GATHER>
constexpr int kThreads = KIND == kCut ? 608 : GATHER ? 576 : WGRAD ? 352 : 320;

// GATHER: a warp fetches the 128 bytes of each of a tile's rows that a chunk holds, each row from where it lies, and lays
// them as a TMA load would: 16-byte cells, XOR-swizzled, zeros beyond the inner axis and for a slot without a row.
__device__ __forceinline__ void gather_chunk(const MmaArgs& a, uint32_t to, const int* sources, int chunk, int row_bytes, int64_t pitch_bytes) {
    const int lane = threadIdx.x & 31, q = lane & 7, at = chunk * kChunkBytes + q * 16, bytes = max(min(16, row_bytes - at), 0);
#pragma unroll 8
    for (int i = 0; i < 32; ++i) {
        const int r = i * 4 + (lane >> 3), source = sources[r];
        const char* from = static_cast<const char*>(a.x) + (source < 0 || bytes == 0 ? 0 : source * pitch_bytes + at);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + r * kChunkBytes + ((q ^ (r & 7)) << 4)), "l"(from),
                     "r"(source < 0 ? 0 : bytes)
                     : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

template <int BN, Kind KIND, bool WGRAD, bool FEW, int BLOCKS, bool GATHER>
__global__ void __launch_bounds__(kThreads<KIND, WGRAD, GATHER>, 1)
    product_kernel(const MmaArgs a, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b) {
    using S = Shape<BN, KIND, FEW, BLOCKS>;
    constexpr bool EIGHT = KIND == kEight;
    constexpr int kChunk = (EIGHT ? 128 : 64) * S::kDeep;  // values of the summed axis a stage holds
    constexpr int kRows = kTileRows * BLOCKS;
    extern __shared__ uint8_t dynamic[];
    __shared__ Tables t;
    __shared__ int row_sources[GATHER ? 8 * kTileRows : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = BLOCKS == 2 ? (int)fg::cluster_rank() : 0;
    const uint32_t held = (fg::smem_address(dynamic) + 1023u) & ~1023u;  // few rows: they come first
    const uint32_t ring = held + (FEW ? a.held : 0);
    const int stages = FEW ? a.stages : S::kStages;
    const int held_chunk = (int)(a.m + 7) / 8 * 1024;  // few rows: bytes of 128 bytes of each

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            fg::barrier_init(fg::smem_address(&t.full[s]), KIND == kCut ? 8 : GATHER ? 2 : BLOCKS);
            fg::barrier_init(fg::smem_address(&t.tail[s]), 1);
            fg::barrier_init(fg::smem_address(&t.empty[s]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            fg::barrier_init(fg::smem_address(&t.filled[s]), 1);
            fg::barrier_init(fg::smem_address(&t.drained[s]), 8 * BLOCKS);
        }
        for (int s = 0; s < S::kRaw; ++s) {
            fg::barrier_init(fg::smem_address(&t.raw[s]), 1);
            fg::barrier_init(fg::smem_address(&t.spent[s]), 8);
        }
        fg::barrier_init(fg::smem_address(&t.rows), 8);
        fg::barrier_init(fg::smem_address(&t.last), 1);
        fg::barrier_init_fence();
        t.stop = 0;
        if (!FEW && !GATHER) fg::prefetch_map(&map_a);
        fg::prefetch_map(&map_b);
    }
    if (warp == 1) fg::tmem_alloc<BLOCKS>(fg::smem_address(&t.tmem), S::kColumns);

    if (FEW && threadIdx.x < 32 && threadIdx.x < a.m) {
        int r = threadIdx.x;
        if (a.order) {
            const int e = a.order[r];
            r = e >= 0 ? e / a.choices : -1;
        }
        t.sources[threadIdx.x] = r < a.x_rows ? r : -1;
    }

    // groups' first slots and tile counts, scanned: thread i takes groups [i * each, (i + 1) * each).  Lists whose groups overlap
    // can add up to more tiles than 32 bits count: the sums end at INT_MAX, so that the table never falls.
    {
        constexpr int kAll = kThreads<KIND, WGRAD, GATHER>;
        const int each = (a.groups + kAll - 1) / kAll, from = min((int)threadIdx.x * each, a.groups), to = min(from + each, a.groups);
        const int64_t unit = WGRAD ? (a.split ? a.split : (int64_t)INT_MAX) : kRows;
        auto plus = [](int x, int y) { return (int)min((uint32_t)x + (uint32_t)y, (uint32_t)INT_MAX); };
        int own = 0;
        for (int g = from; g < to; ++g) {
            const int64_t b = min((int64_t)max(a.offsets[g], 0), a.m), e = min((int64_t)max(a.offsets[g + 1], 0), a.m);
            const int64_t n = max(e - b, (int64_t)0);
            t.start[g] = (int)b;
            own += (int)(WGRAD ? max((n + unit - 1) / unit, (int64_t)1) : (n + unit - 1) / unit);
        }
        int sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum = plus(sum, v);
        }
        if (lane == 31) t.warp_sums[warp] = sum;
        __syncthreads();
        int before = sum < INT_MAX ? sum - own : sum;
        for (int w = 0; w < warp; ++w) before = plus(before, t.warp_sums[w]);
        for (int g = from; g < to; ++g) {
            const int64_t b = t.start[g], e = min((int64_t)max(a.offsets[g + 1], 0), a.m);
            const int64_t n = max(e - b, (int64_t)0);
            t.tiles[g] = before;
            before = plus(before, (int)(WGRAD ? max((n + unit - 1) / unit, (int64_t)1) : (n + unit - 1) / unit));
        }
        if (threadIdx.x == kAll - 1) {
            t.tiles[a.groups] = before;
            t.start[a.groups] = (int)min((int64_t)max(a.offsets[a.groups], 0), a.m);
        }
    }
    fg::tcgen05_before_sync();
    __syncthreads();
    if (BLOCKS == 2) fg::cluster_sync();  // the other block's barriers are there
    fg::tcgen05_after_sync();

    const int rows_tiles = WGRAD ? (a.outer + kRows - 1) / kRows : 1;
    const int col_tiles = ((WGRAD ? a.inner : a.outer) + BN - 1) / BN;
    const int per_unit = WGRAD ? rows_tiles * col_tiles : col_tiles;  // output tiles for each counted row tile or partial sum
    const int64_t total = (int64_t)t.tiles[a.groups] * per_unit;
    const int64_t start = blockIdx.x / BLOCKS, stride = gridDim.x / BLOCKS;
    const uint32_t tmem = t.tmem;
    volatile int* stop = &t.stop;

    // What output tile `index` is for this block: its group, first row and column, the slots [begin, end) it is about.
    struct Tile {
        int group, unit, row, col;
        int begin, end, chunks;
        __device__ bool ragged() const { return (end - begin) % 16 != 0; }
    };
    int cursor = 0;
    auto locate = [&](int64_t index) {
        Tile w;
        while (index >= (int64_t)t.tiles[cursor + 1] * per_unit) ++cursor;
        const int64_t local = index - (int64_t)t.tiles[cursor] * per_unit;
        const int count = t.tiles[cursor + 1] - t.tiles[cursor];
        const int first = t.start[cursor], stop_at = max(first, (int)min((int64_t)max(a.offsets[cursor + 1], 0), a.m));
        w.group = cursor;
        if (WGRAD) {
            const int part = (int)(local / per_unit), tile = (int)(local - (int64_t)part * per_unit);
            w.unit = (int)min((int64_t)t.tiles[cursor] + part, (int64_t)a.units - 1);  // lists that overlap: wrong sums, no wrong address
            w.row = tile % rows_tiles * kRows + rank * kTileRows;
            w.col = tile / rows_tiles * BN;
            w.begin = a.split ? first + part * a.split : first;
            w.end = a.split ? (int)min((int64_t)w.begin + a.split, (int64_t)stop_at) : stop_at;
            w.chunks = max(w.end - w.begin + kChunk - 1, 0) / kChunk;
        } else {
            // up to 16 row tiles share a column tile's weights while they are in L2, then the next column tile
            const int super = (int)(local / ((int64_t)kSuperRows * col_tiles)), left = min(kSuperRows, count - super * kSuperRows);
            const int rest = (int)(local - (int64_t)super * kSuperRows * col_tiles);
            w.unit = 0;
            w.begin = first + (super * kSuperRows + rest % left) * kRows + rank * kTileRows;
            w.end = min(w.begin + kTileRows, stop_at);
            w.row = 0;
            w.col = rest / left * BN;
            w.chunks = (a.inner + kChunk - 1) / kChunk;
        }
        return w;
    };

    if (warp == 0) {
        if (fg::elect_one()) {
            int s = 0, parity = 1;  // next stage, and the parity that its emptying will have had (a fresh barrier passes for 1)
            int64_t step = 0;       // stages filled so far
            uint32_t tail_now = 0, tail_parity = 0;  // a bit a stage: holds a tail; parity of its next tail
            bool live = true;
            for (int64_t i = start; live && i < total; i += stride) {
                const Tile w = locate(i);
                const int col = w.col + rank * S::kOwnCols;
                // 8 KB blocks of both operands; blocks beyond the last column are not loaded, their products not stored
                auto blocks_a = [&](int row) { return WGRAD ? max(min(2, (a.outer - row + 63) / 64), 0) : 0; };
                auto blocks_b = [&](int at) {
                    return WGRAD || a.b_mn ? max(min(S::kOwnCols / 64, ((WGRAD ? a.inner : a.outer) - at + 63) / 64), 0) : S::kOwnCols / 64;
                };
                const int a_blocks = blocks_a(w.row), b_blocks = blocks_b(col);
                const uint32_t own = ((WGRAD ? a_blocks * 8192 : KIND == kCut || GATHER ? 0 : S::kA) + b_blocks * 8192) * S::kParts * S::kDeep;
                uint32_t bytes = own;
                if (BLOCKS == 2)  // the first block's barrier counts the second one's loads too
                    bytes += ((WGRAD ? blocks_a(w.row + kTileRows) * 8192 : S::kA) + blocks_b(col + S::kOwnCols) * 8192) * S::kParts;
                for (int c = 0; c < w.chunks; ++c, ++step) {
                    const int at_stage = s;
                    // (cut rows: the weights have a barrier of their own, the stage's counts the cutting warps)
                    const uint32_t full = fg::smem_address(KIND == kCut ? &t.tail[s] : &t.full[s]), stage = ring + s * S::kStageBytes;
                    if (!fg::barrier_wait(fg::smem_address(&t.empty[s]), parity, stop)) {
                        live = false;
                        break;
                    }
                    if (++s == stages) s = 0, parity ^= 1;
                    const int k = c * kChunk;
                    if (WGRAD && c == w.chunks - 1 && w.ragged()) {  // goes through the warp that clears it, each block's own
                        const uint32_t bar = fg::smem_address(&t.tail[at_stage]);
                        tail_now |= 1u << at_stage;
                        tail_parity ^= 1u << at_stage;
                        fg::barrier_expect(bar, own);
#pragma unroll
                        for (int p = 0; p < S::kParts; ++p) {
                            const uint32_t at = stage + p * S::kA, bt = stage + S::kParts * S::kA + p * S::kB;
                            const int slot = w.begin + k + p * (int)a.m;
                            for (int q = 0; q < a_blocks; ++q) fg::tma_load_2d<1>(at + q * 8192, &map_a, w.row + q * 64, slot, bar);
                            for (int q = 0; q < b_blocks; ++q) fg::tma_load_2d<1>(bt + q * 8192, &map_b, col + q * 64, slot, bar);
                        }
                        continue;
                    }
                    tail_now &= ~(1u << at_stage);
                    if (rank == 0) {
                        fg::barrier_expect(full, bytes);
                        if (BLOCKS == 2) fg::barrier_arrive(full);  // two arrivals: those of the clearing warps, for a tail
                    }
#pragma unroll
                    for (int p = 0; p < S::kParts; ++p) {
                        const uint32_t at = stage + p * S::kA, bt = stage + S::kParts * S::kA + p * S::kB;
                        if (WGRAD) {  // 64 slots by 64 columns a block
                            const int slot = w.begin + k + p * (int)a.m;
                            for (int q = 0; q < a_blocks; ++q) fg::tma_load_2d<BLOCKS>(at + q * 8192, &map_a, w.row + q * 64, slot, full);
                            for (int q = 0; q < b_blocks; ++q) fg::tma_load_2d<BLOCKS>(bt + q * 8192, &map_b, col + q * 64, slot, full);
                        } else {
                            const int g = a.shared_weight ? p : w.group + p * a.groups;
                            if (!FEW && KIND != kCut && !GATHER) fg::tma_load_2d<BLOCKS>(at, &map_a, k, w.begin + p * (int)a.m, full);
#pragma unroll
                            for (int h = 0; h < S::kDeep; ++h) {
                                const int kh = k + h * (kChunk / S::kDeep);
                                const uint32_t to = bt + h * S::kB;
                                if (!a.b_mn) {
                                    fg::tma_load_3d<BLOCKS>(to, &map_b, kh, col, g, full);
                                } else {
                                    for (int q = 0; q < b_blocks; ++q) fg::tma_load_3d<BLOCKS>(to + q * 8192, &map_b, col + q * 64, kh, g, full);
                                }
                            }
                        }
                    }
                }
            }
            if (BLOCKS == 2)  // the first block's products arrive at both blocks' stages: none may arrive when this one has ended
                for (int q = 0; live && q < stages; ++q) {
                    live = fg::barrier_wait(fg::smem_address(&t.empty[s]), parity, stop);
                    if (++s == stages) s = 0, parity ^= 1;
                }
            if (*stop) {  // no copy may be in flight when the block (or its pair) ends
                for (int64_t q = max(step - stages, (int64_t)0); q < step; ++q) {
                    const int at = (int)(q % stages);
                    if (KIND == kCut) fg::barrier_wait(fg::smem_address(&t.tail[at]), (q / stages) & 1, stop, true);
                    else if (tail_now >> at & 1) fg::barrier_wait(fg::smem_address(&t.tail[at]), ~tail_parity >> at & 1, stop, true);
                    else if (rank == 0) fg::barrier_wait(fg::smem_address(&t.full[at]), (q / stages) & 1, stop, true);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && fg::elect_one()) {
            int s = 0, parity = 0;
            int64_t turn = 0;
            const uint32_t descriptor = fg::product_descriptor(a.format, WGRAD, WGRAD || a.b_mn, kRows, BN);
            const bool b_mn = WGRAD || a.b_mn;
            bool live = !FEW || start >= total || fg::barrier_wait(fg::smem_address(&t.rows), 0, stop);
            for (int64_t i = start; live && i < total; i += stride) {
                const Tile w = locate(i);
                if (w.chunks == 0) continue;  // an empty group's dW: nothing to add up
                for (int c = 0; c < w.chunks; ++c) {
                    const int buffer = (int)(turn & 1);
                    const uint32_t acc = tmem + buffer * BN;
                    if (c == 0 || S::kParts == 3) {  // a fresh accumulator
                        live = turn < 2 || fg::barrier_wait<BLOCKS == 2>(fg::smem_address(&t.drained[buffer]), (turn / 2 - 1) & 1, stop);
                        if (!live) break;
                        fg::tcgen05_after_sync();
                    }
                    const uint32_t stage = ring + s * S::kStageBytes, empty = fg::smem_address(&t.empty[s]);
                    live = fg::barrier_wait<BLOCKS == 2 && WGRAD>(fg::smem_address(&t.full[s]), parity, stop);
                    if (KIND == kCut) live = live && fg::barrier_wait(fg::smem_address(&t.tail[s]), parity, stop);
                    if (++s == stages) s = 0, parity ^= 1;
                    if (!live) break;
                    fg::tcgen05_after_sync();
                    // of a group's last chunk only the steps that have rows of it
                    const int steps = WGRAD && c == w.chunks - 1 ? (w.end - w.begin - c * kChunk + 15) / 16 : 4;
#pragma unroll
                    for (int pair = S::kParts == 3 ? 0 : 5; pair < 6; ++pair) {
                        const uint32_t at = FEW ? held + c * 2 * held_chunk : stage + part_a(pair) * S::kA, bt = stage + S::kParts * S::kA + part_b(pair) * S::kB;
#pragma unroll
                        for (int k = 0; k < 4 * S::kDeep; ++k) {
                            const uint32_t ah = at + k / 4 * held_chunk, bh = bt + k / 4 * S::kB;  // a chunk further from the fifth step on
                            const uint64_t da = WGRAD ? fg::operand_descriptor(at + k * 2048, 8192, 1024) : fg::operand_descriptor(ah + k % 4 * 32, 16, 1024);
                            const uint64_t db = b_mn ? fg::operand_descriptor(bh + k % 4 * 2048, 8192, 1024) : fg::operand_descriptor(bh + k % 4 * 32, 16, 1024);
                            if (!WGRAD || k < steps) fg::product_step<BLOCKS, EIGHT>(acc, da, db, descriptor, (S::kParts == 1 && c > 0) || pair > (S::kParts == 3 ? 0 : 5) || k > 0);
                        }
                    }
                    fg::product_commit<BLOCKS>(empty);
                    if (c == w.chunks - 1 || S::kParts == 3) {
                        fg::product_commit<BLOCKS>(fg::smem_address(&t.filled[buffer]));
                        ++turn;
                    }
                }
            }
            if (*stop) {  // products in flight end before the accumulators are freed
                fg::product_commit<BLOCKS>(fg::smem_address(&t.last));
                fg::barrier_wait(fg::smem_address(&t.last), 0, stop, true);
            }
        }
        __syncwarp();
    } else if (KIND == kCut && warp == 18) {
        if (fg::elect_one()) {  // the rows, half a chunk a load, ahead of the weights' stages
            int raw = 0, parity = 1;
            int64_t loads = 0;
            bool live = true;
            for (int64_t i = start; live && i < total; i += stride) {
                const Tile w = locate(i);
                for (int h = 0; h < 2 * w.chunks; ++h, ++loads) {
                    live = fg::barrier_wait(fg::smem_address(&t.spent[raw]), parity, stop);
                    if (!live) break;
                    const uint32_t bar = fg::smem_address(&t.raw[raw]);
                    fg::barrier_expect(bar, S::kRawBytes);
                    fg::tma_load_2d<1>(ring + S::kStages * S::kStageBytes + raw * S::kRawBytes, &map_a, h * 32, w.begin, bar);
                    if (++raw == S::kRaw) raw = 0, parity ^= 1;
                }
            }
            if (*stop)
                for (int64_t q = max(loads - S::kRaw, (int64_t)0); q < loads; ++q)
                    fg::barrier_wait(fg::smem_address(&t.raw[q % 3]), (q / 3) & 1, stop, true);
        }
        __syncwarp();
    } else if (KIND == kCut && warp >= 10) {
        // x = a + b + c: 8 values a thread and step, from 32 bytes of a raw row to 16 bytes of each part's row
        int s = 0, parity = 1, raw = 0, raw_parity = 0;
        bool live = true;
        for (int64_t i = start; live && i < total; i += stride) {
            const Tile w = locate(i);
            for (int c = 0; live && c < w.chunks; ++c) {
                const uint32_t stage = ring + s * S::kStageBytes;
                live = warp_wait(fg::smem_address(&t.empty[s]), parity, stop);
                for (int h = 0; live && h < 2; ++h) {
                    live = warp_wait(fg::smem_address(&t.raw[raw]), raw_parity, stop);
                    if (!live) break;
                    cut_rows(ring + S::kStages * S::kStageBytes + raw * S::kRawBytes, stage, h, threadIdx.x - 320);
                    __syncwarp();
                    if (lane == 0) fg::barrier_arrive(fg::smem_address(&t.spent[raw]));
                    if (++raw == S::kRaw) raw = 0, raw_parity ^= 1;
                }
                if (!live) break;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) fg::barrier_arrive(fg::smem_address(&t.full[s]));
                if (++s == stages) s = 0, parity ^= 1;
            }
        }
    } else if (GATHER && warp >= 10) {
        // Warps take the chunks in turn, so that as many are on their way as the ring holds - and no more: a warp that is
        // further ahead could take the emptying before the last for the one that it waits for.
        constexpr int kTurns = S::kStages < 8 ? S::kStages : 8;
        const int mine = warp - 10, size = EIGHT ? 1 : 2, row_bytes = a.inner * size;
        const int64_t pitch = a.ldx * size;
        int* sources = row_sources + mine * kTileRows;
        int s = 0, parity = 1, turn = 0;
        bool live = true;
        for (int64_t i = start; mine < kTurns && live && i < total; i += stride) {
            const Tile w = locate(i);
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int slot = w.begin + u * 32 + lane, e = slot < w.end ? a.order[slot] : -1, r = e >= 0 ? e / a.choices : -1;
                sources[u * 32 + lane] = r < a.x_rows ? r : -1;
            }
            __syncwarp();
            for (int c = 0; c < w.chunks; ++c) {
                if (turn == mine) {
                    live = warp_wait(fg::smem_address(&t.empty[s]), parity, stop);
                    if (!live) break;
                    gather_chunk(a, ring + s * S::kStageBytes, sources, c, row_bytes, pitch);
                    if (lane == 0) fg::barrier_arrive(fg::smem_address(&t.full[s]));
                }
                if (++turn == kTurns) turn = 0;
                if (++s == stages) s = 0, parity ^= 1;
            }
        }
    } else if (WGRAD && warp == 10) {
        // In a group's last chunk, the rows that are not its own become zeros, as far as the last step of 16 reaches: 128
        // bytes a row, 64 rows a column block.
        int64_t step = 0;
        uint32_t tail_parity = 0;
        for (int64_t i = start; i < total; i += stride) {
            const Tile w = locate(i);
            step += w.chunks;
            if (w.chunks == 0 || !w.ragged()) continue;
            const int s = (int)((step - 1) % stages), keep = (w.end - w.begin - 1) % kChunk + 1, upto = (keep + 15) / 16 * 16;
            const uint32_t stage = ring + s * S::kStageBytes;
            if (!warp_wait(fg::smem_address(&t.tail[s]), tail_parity >> s & 1, stop)) break;
            tail_parity ^= 1u << s;
            for (int z = keep * 8 + lane; z < upto * 8; z += 32)
#pragma unroll
                for (int q = 0; q < S::kStageBytes / 8192; ++q)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(stage + q * 8192 + z * 16), "r"(0) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (BLOCKS == 2) fg::barrier_arrive_at<true>(fg::smem_address(&t.full[s]), 0);
                else fg::barrier_arrive(fg::smem_address(&t.full[s]));
            }
            __syncwarp();
        }
    } else {
        const int quarter = warp & 3;  // the lanes of tensor memory this warp can read
        const int half = (warp - 2) >> 2;
        const uint32_t staging = ring + stages * S::kStageBytes + S::kRaw * S::kRawBytes + (warp - 2) * 2048;
        if (FEW && start < total) {
            hold_rows<EIGHT>(a, held, held_chunk, t.sources, threadIdx.x - 64);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) fg::barrier_arrive(fg::smem_address(&t.rows));
        }
        const int width = WGRAD ? a.inner : a.outer;
        const int size = a.out_type == FG_F32 ? 4 : 2;
        const bool vector = (int64_t)width * size % 16 == 0 && ((uintptr_t)a.y & 15) == 0;
        int64_t turn = 0;
        for (int64_t i = start; i < total; i += stride) {
            const Tile w = locate(i);
            const int above = quarter * 32;
            // a tile's rows start with its first slot, held ones with slot 0: there, rows of [begin, end) are stored
            const int slot0 = FEW ? 0 : w.begin, from = FEW ? w.begin - above : 0;
            const int rows = (WGRAD ? a.outer - w.row : w.end - slot0) - above;
            const int64_t first = (WGRAD ? (int64_t)(a.split ? w.unit : w.group) * a.outer + w.row : slot0) + above;
            float scale = 0.0f;
            const float* column_scales = nullptr;
            if (EIGHT) {
                const int slot = slot0 + above + lane;
                if (slot >= w.begin && slot < w.end) {
                    const int e = a.order ? a.order[slot] : 0, r = a.order ? e / a.choices : slot;
                    if (e >= 0 && r < a.x_rows) scale = a.x_scales[r];
                }
                column_scales = a.w_scales + (int64_t)w.group * a.outer + w.col;
            }
            const int64_t at = first * width + w.col;
            auto drained = [&](int buffer) {
                fg::tcgen05_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (BLOCKS == 2) fg::barrier_arrive_at<false>(fg::smem_address(&t.drained[buffer]), 0);
                    else fg::barrier_arrive(fg::smem_address(&t.drained[buffer]));
                }
                ++turn;
            };
            float sums[BN / 2];  // fp32: over the chunks
            if constexpr (S::kParts == 3) {
#pragma unroll
                for (int j = 0; j < BN / 2; ++j) sums[j] = 0.0f;
                bool live = true;
                for (int c = 0; c < w.chunks; ++c) {
                    const int buffer = (int)(turn & 1);
                    live = warp_wait(fg::smem_address(&t.filled[buffer]), (turn / 2) & 1, stop);
                    if (!live) break;
                    fg::tcgen05_after_sync();
                    add_chunk<BN>(tmem + ((uint32_t)above << 16) + buffer * BN, sums, half);
                    drained(buffer);
                }
                if (!live) break;
                store_rows<float, BN, false, true>(0, true, sums, static_cast<float*>(a.y) + at, width, from, rows, width - w.col, vector, staging, half, scale,
                                                   column_scales);
            } else {
                const int buffer = (int)(turn & 1);
                if (w.chunks) {
                    if (!warp_wait(fg::smem_address(&t.filled[buffer]), (turn / 2) & 1, stop)) break;
                    fg::tcgen05_after_sync();
                }
                const uint32_t acc = tmem + ((uint32_t)above << 16) + buffer * BN;
                const int left = width - w.col;
                if (a.out_type == FG_F32)
                    store_rows<float, BN, EIGHT, false>(acc, w.chunks > 0, sums, static_cast<float*>(a.y) + at, width, from, rows, left, vector, staging, half,
                                                        scale, column_scales);
                else if (a.out_type == FG_F16)
                    store_rows<__half, BN, EIGHT, false>(acc, w.chunks > 0, sums, static_cast<__half*>(a.y) + at, width, from, rows, left, vector, staging,
                                                         half, scale, column_scales);
                else
                    store_rows<__nv_bfloat16, BN, EIGHT, false>(acc, w.chunks > 0, sums, static_cast<__nv_bfloat16*>(a.y) + at, width, from, rows, left, vector,
                                                                staging, half, scale, column_scales);
                if (w.chunks) drained(buffer);
            }
        }
        if (!WGRAD) {  // rows in no group
            const int64_t from = (int64_t)t.start[a.groups] * a.outer, values = a.m * a.outer;
            for (int64_t i = from + (int64_t)blockIdx.x * 256 + (threadIdx.x - 64); i < values; i += (int64_t)gridDim.x * 256) {
                if (a.out_type == FG_F32) static_cast<float*>(a.y)[i] = 0.0f;
                else static_cast<uint16_t*>(a.y)[i] = 0;
            }
        }
    }
    fg::tcgen05_before_sync();
    __syncthreads();
    if (BLOCKS == 2) fg::cluster_sync();  // nothing of the other block is still to arrive here
    if (warp == 1) fg::tmem_free<BLOCKS>(tmem, S::kColumns);
    if (threadIdx.x == 0 && t.stop) atomicExch(&g_stuck, 1);
}

// ---- few rows ----

// The form for single tokens whose weights the loads cannot take as they are: fp32, or off the 16-byte grid.  At most kFewRows
// slots in all.  Bound: the touched weights' bytes, read once for the rows of a group (up to 8 at a time); the other way
// would be to cut or copy all groups' weights first.  A block takes 64 columns of the j-th group that has rows, holds up
// to 8 of its rows in shared memory, and a warp computes four columns at a time, its lanes side by side along the dense
// inner axis: 16-byte loads, four in flight a lane, each row's values fetched from shared memory once for the four
// columns; 32-bit multiply-adds and a sum across the warp.  4 rows x 2 of 16 experts, 2048 to 4096 in fp32: 49 us (4.1
// TB/s); 16 rows x 2 of 64, 1001 to 1000 in bf16: 34 us, 87 us by a copy of the weights.
constexpr int kFewRows = 32, kFewCols = 64;

template <typename T>
__device__ __forceinline__ void widen(const Pack<T, 16 / sizeof(T)>& p, float (&v)[16 / sizeof(T)]) {
#pragma unroll
    for (int j = 0; j < (int)(16 / sizeof(T)); ++j) v[j] = to_f32<T>(p.v[j]);
}

struct FewArgs {
    const void *x, *w;
    const float *x_scales, *w_scales;
    const int32_t *offsets, *order;
    void* y;
    int64_t ldx, w_group, w_out, x_rows;
    int32_t m, choices, groups, inner, outer, out_type, pitch;  // pitch: values of a row in shared memory
    bool vector, vector_rows;                                   // weights, rows on the 16-byte grid
};

template <typename T, int R>
__device__ __forceinline__ void few_columns(const FewArgs& a, const T* rows, const T* w, int col, int count, int first, int n, const float* scales,
                                            const float* column_scales) {
    constexpr int kPer = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    float acc[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = 0.0f;
    const T* column[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) column[c] = w + (int64_t)(col + min(c, count - 1)) * a.w_out;
#pragma unroll 2
    for (int k = lane * kPer; k < a.inner; k += 32 * kPer) {
        float v[4][kPer];
        if (a.vector && k + kPer <= a.inner) {
            Pack<T, kPer> p[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) p[c] = fg::load_pack<T, kPer>(column[c] + k);
#pragma unroll
            for (int c = 0; c < 4; ++c) widen<T>(p[c], v[c]);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int j = 0; j < kPer; ++j) v[c][j] = k + j < a.inner ? to_f32<T>(column[c][k + j]) : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x[kPer];
            widen<T>(fg::load_pack<T, kPer>(rows + r * a.pitch + k), x);  // zeros beyond the inner axis
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int j = 0; j < kPer; ++j) acc[r][c] = __fmaf_rn(x[j], v[c][j], acc[r][c]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = fg::warp_sum(acc[r][c]);
        if (r >= n) break;
        if (lane < count) {
            float v = lane == 0 ? acc[r][0] : lane == 1 ? acc[r][1] : lane == 2 ? acc[r][2] : acc[r][3];
            if (scales) v = __fmul_rn(__fmul_rn(v, scales[r]), column_scales[col + lane]);
            const int64_t at = (int64_t)(first + r) * a.outer + col + lane;
            if (a.out_type == FG_F32) static_cast<float*>(a.y)[at] = v;
            else if (a.out_type == FG_F16) static_cast<__half*>(a.y)[at] = from_f32<__half>(v);
            else static_cast<__nv_bfloat16*>(a.y)[at] = from_f32<__nv_bfloat16>(v);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) few_rows_kernel(const FewArgs a) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ int offsets[kMaxGroups + 1];
    __shared__ int group;
    __shared__ float scales[8];
    T* rows = reinterpret_cast<T*>(dynamic);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.y, col0 = blockIdx.x * kFewCols;
    for (int g = threadIdx.x; g <= a.groups; g += 256) offsets[g] = min(max(a.offsets[g], 0), a.m);
    if (threadIdx.x == 0) group = -1;
    __syncthreads();
    if (warp == 0) {  // the group of this rank among those with rows
        int before = 0;
        for (int base = 0; base < a.groups; base += 32) {
            const int g = base + lane;
            const bool some = g < a.groups && offsets[g + 1] > offsets[g];
            const unsigned vote = __ballot_sync(0xffffffffu, some);
            if (some && before + __popc(vote & ((1u << lane) - 1u)) == rank) group = g;
            before += __popc(vote);
            if (before > rank) break;
        }
    }
    if (rank == 0) {  // rows in no group
        const int from = offsets[a.groups], cols = min(kFewCols, a.outer - col0);
        for (int i = threadIdx.x; i < (a.m - from) * cols; i += 256) {
            const int64_t at = (int64_t)(from + i / cols) * a.outer + col0 + i % cols;
            if (a.out_type == FG_F32) static_cast<float*>(a.y)[at] = 0.0f;
            else static_cast<uint16_t*>(a.y)[at] = 0;
        }
    }
    __syncthreads();
    if (group < 0) return;
    const int begin = offsets[group], end = offsets[group + 1];
    const T* w = static_cast<const T*>(a.w) + (int64_t)group * a.w_group;
    const float* column_scales = a.w_scales ? a.w_scales + (int64_t)group * a.outer : nullptr;
    for (int first = begin; first < end; first += 8) {
        const int n = min(8, end - first), held = n <= 2 ? n : n <= 4 ? 4 : 8;
        constexpr int kPer = 16 / sizeof(T);
        const int pieces = a.pitch / kPer;
        for (int i = threadIdx.x; i < held * pieces; i += 256) {  // 16 bytes of a row a thread
            const int r = i / pieces, k = (i - r * pieces) * kPer;
            int64_t source = -1;
            if (r < n) {
                source = first + r;
                if (a.order) {
                    const int e = a.order[first + r];
                    source = e >= 0 ? e / a.choices : -1;
                }
                if (source >= a.x_rows) source = -1;
            }
            const T* x = static_cast<const T*>(a.x) + (source < 0 ? 0 : source) * a.ldx + k;
            Pack<T, kPer> p;
            if (source >= 0 && a.vector_rows && k + kPer <= a.inner) {
                p = fg::load_pack<T, kPer>(x);
            } else {
#pragma unroll
                for (int j = 0; j < kPer; ++j) p.v[j] = source >= 0 && k + j < a.inner ? x[j] : T(0.0f);
            }
            store_pack<T, kPer>(rows + r * a.pitch + k, p);
            if (k == 0) scales[r] = a.x_scales && source >= 0 ? a.x_scales[source] : 0.0f;
        }
        __syncthreads();
        for (int c = warp * 4; c < kFewCols && col0 + c < a.outer; c += 32) {
            const int col = col0 + c, count = min(4, a.outer - col);
            const float* sc = a.x_scales ? scales : nullptr;
            if (n == 1) few_columns<T, 1>(a, rows, w, col, count, first, n, sc, column_scales);
            else if (n == 2) few_columns<T, 2>(a, rows, w, col, count, first, n, sc, column_scales);
            else if (n <= 4) few_columns<T, 4>(a, rows, w, col, count, first, n, sc, column_scales);
            else few_columns<T, 8>(a, rows, w, col, count, first, n, sc, column_scales);
        }
        __syncthreads();
    }
}

// dW[g] = its partial sums added in order.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ partial, const int32_t* __restrict__ offsets, int groups, int64_t m,
                                                   int split, int units, int64_t cells, T* __restrict__ dw) {
    __shared__ int first, count;
    const int g = blockIdx.y;  // `units`: partial sums that there are
    if (threadIdx.x == 0) {
        int64_t before = 0, n = 0;
        for (int q = 0; q <= g; ++q) {
            const int64_t b = min((int64_t)max(offsets[q], 0), m), e = min((int64_t)max(offsets[q + 1], 0), m);
            n = max((max(e - b, (int64_t)0) + split - 1) / split, (int64_t)1);
            if (q < g) before += n;
        }
        first = (int)min(before, (int64_t)units - 1);
        count = (int)min(n, (int64_t)units - first);
    }
    __syncthreads();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (int64_t)gridDim.x * 256) {
        float s = partial[(int64_t)first * cells + i];
        int q = 1;
        for (; q + 8 <= count; q += 8) {  // eight loads in flight, added in order
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = partial[(int64_t)(first + q + j) * cells + i];
#pragma unroll
            for (int j = 0; j < 8; ++j) s = __fadd_rn(s, v[j]);
        }
        for (; q < count; ++q) s = __fadd_rn(s, partial[(int64_t)(first + q) * cells + i]);
        dw[(int64_t)g * cells + i] = from_f32<T>(s);
    }
}

// dst[g][r][c], c < pitch, from src at g s0 + r s1 + c s2: the same type, or the three bf16 parts of an fp32 value in
// three consecutive copies.  With an order (one group), row r comes from row order[r] / choices; a slot that names no row
// gets zeros.  16 bytes of output (of each part) a thread and step; 2^shift threads share a row.  Bound: device memory in 16 and
// 32 bits; 8-bit rows are bound by instructions (16384 rows of 4096: 33 us, ALU pipe 67 % busy, DRAM 20 %).
struct PackArgs {
    const void* src;
    void* dst;
    const int32_t* order;
    int64_t s0, s1, s2, groups, rows, source_rows;
    int32_t cols, pitch, choices, shift;
    bool vector;  // 128-bit reads: dense columns, every row on a 16-byte boundary
};
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const PackArgs a) {
    constexpr int kPer = sizeof(T) == 1 ? 16 : 8;
    const int per_row = a.pitch / kPer, threads = 1 << a.shift, mine = threadIdx.x & (threads - 1);
    const int64_t lines = a.groups * a.rows, plane = lines * a.pitch;
    for (int64_t line = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> a.shift; line < lines; line += ((int64_t)gridDim.x * 256) >> a.shift) {
        int64_t g = 0, r = line;
        if (a.groups > 1) g = line / a.rows, r = line - g * a.rows;
        bool in = true;
        if (a.order) {
            const int e = a.order[line];
            r = e / a.choices;
            in = e >= 0 && r < a.source_rows;
        }
        const T* row = static_cast<const T*>(a.src) + (in ? g * a.s0 + r * a.s1 : 0);
        for (int q = mine; q < per_row; q += threads) {
            const int c = q * kPer;
            alignas(16) T v[kPer];
            if (!in) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) v[j] = T(0.0f);
            } else if (a.vector && c + kPer <= a.cols) {
                constexpr int kHalf = 16 / sizeof(T);
#pragma unroll
                for (int j = 0; j < kPer; j += kHalf) *reinterpret_cast<Pack<T, kHalf>*>(v + j) = fg::load_pack<T, kHalf>(row + c + j);
            } else {
#pragma unroll
                for (int j = 0; j < kPer; ++j) v[j] = c + j < a.cols ? row[(int64_t)(c + j) * a.s2] : T(0.0f);
            }
            const int64_t at = line * a.pitch + c;
            if constexpr (sizeof(T) == 4) {
                Pack<__nv_bfloat16, 8> p[3];
                cut_values(v, p);
                for (int k = 0; k < 3; ++k) store_pack<__nv_bfloat16, 8>(static_cast<__nv_bfloat16*>(a.dst) + k * plane + at, p[k]);
            } else {
                Pack<T, kPer> p;
#pragma unroll
                for (int j = 0; j < kPer; ++j) p.v[j] = v[j];
                store_pack<T, kPer>(static_cast<T*>(a.dst) + at, p);
            }
        }
    }
}

// ---- host side ----

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static EncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) == cudaSuccess &&
            found == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(p);
    });
    return fn;
}

// A matrix, or one for each group, as the loads see it: rows of `cols` dense values.
struct Matrix {
    const void* data;
    int64_t cols, rows, groups;    // groups 0: a plain matrix
    int64_t pitch, group_stride;   // in values
    int32_t type;                  // as stored (bf16 for the parts of fp32)
};

int make_map(CUtensorMap* map, const Matrix& m, int box_cols, int box_rows) {
    EncodeFn encode = encoder();
    if (!encode) return fg::fail(FG_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const int size = fg::type_size(m.type);
    const cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)(m.groups ? m.groups : 1)};
    const cuuint64_t strides[2] = {(cuuint64_t)(m.pitch * size), (cuuint64_t)(m.group_stride * size)};
    const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1}, ones[3] = {1, 1, 1};
    const CUtensorMapDataType type = m.type == FG_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : m.type == FG_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : m.type == FG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    auto run = [&] {
        return encode(map, type, m.groups ? 3 : 2, const_cast<void*>(m.data), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult rc = run();
    if (rc == CUDA_ERROR_INVALID_CONTEXT) {  // a host thread's first CUDA call (an autograd thread's): bind the device's context
        int device = 0;
        FG_CUDA_TRY(cudaGetDevice(&device));
        FG_CUDA_TRY(cudaSetDevice(device));
        rc = run();
    }
    if (rc != CUDA_SUCCESS) return fg::fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)rc);
    return FG_OK;
}

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t pitch_of(int64_t cols, int32_t type) { return round_up(cols, type == FG_E4M3 ? 16 : 8); }
// Bytes of the dense copy (three bf16 copies of fp32), on a 256-byte grid.
int64_t packed_bytes(int64_t lines, int64_t cols, int32_t type) {
    return round_up(lines * pitch_of(cols, type) * (type == FG_F32 ? 6 : fg::type_size(type)), 256);
}
bool loadable(const void* p, int64_t pitch, int64_t group_stride, int32_t type) {
    const int size = fg::type_size(type);
    return type != FG_F32 && fg::aligned16(p) && pitch > 0 && pitch * size % 16 == 0 && group_stride * size % 16 == 0 &&
           pitch * size < (1ll << 40) && group_stride * size < (1ll << 40);
}

// Copies [groups][rows][cols] at strides (s0, s1, s2) - or the rows that `order` names - into `*work`, and moves that on.
int pack(const void* src, int64_t s0, int64_t s1, int64_t s2, int64_t groups, int64_t rows, int64_t cols, const int32_t* order, int32_t choices,
         int64_t source_rows, int32_t type, uint8_t** work, cudaStream_t s) {
    const int size = fg::type_size(type), per = type == FG_E4M3 ? 16 : 8;
    PackArgs p{src, *work, order, s0, s1, s2, groups, rows, source_rows, (int32_t)cols, (int32_t)pitch_of(cols, type), choices, 0, false};
    p.vector = s2 == 1 && fg::aligned16(src) && s0 * size % 16 == 0 && s1 * size % 16 == 0;
    while (p.shift < 8 && (1 << p.shift) < p.pitch / per) ++p.shift;
    const int64_t blocks = ((groups * rows << p.shift) + 255) / 256, most = (int64_t)fg::device_props().sm_count * 32;
    if (blocks == 0) return FG_OK;
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    if (type == FG_F32) pack_kernel<float><<<grid, 256, 0, s>>>(p);
    else if (type == FG_F16) pack_kernel<__half><<<grid, 256, 0, s>>>(p);
    else if (type == FG_BF16) pack_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
    else pack_kernel<__nv_fp8_e4m3><<<grid, 256, 0, s>>>(p);
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    *work += packed_bytes(groups * rows, cols, type);
    return FG_OK;
}

// The slots' rows [m, cols] as a loadable matrix: where they lie, or copied.
bool rows_need_copy(const void* p, int64_t ld, const int32_t* order, int32_t type) { return order || !loadable(p, ld, 0, type); }
// fp32 rows that a product takes as they are (kCut): on the 16-byte grid, in slot order, and at most two column tiles, each of
// which cuts them again.  100003 rows, 7 groups: 256 to 128 columns 74 us (72 with the parts cut off instead of rounded), in
// parts beforehand 90; 64 to 64: 20 and 26; but 128 to 256 79 and 74.
bool rows_cut_on_the_way(const void* p, int64_t ld, const int32_t* order, int32_t outer, int32_t type) {
    return type == FG_F32 && !order && outer <= 128 && fg::aligned16(p) && ld % 4 == 0 && ld < (1ll << 38);
}
int rows_matrix(Matrix* out, const void* p, int64_t ld, int64_t source_rows, const int32_t* order, int32_t choices, int64_t m, int64_t cols,
                int32_t type, uint8_t** work, cudaStream_t s) {
    if (!rows_need_copy(p, ld, order, type)) {
        *out = Matrix{p, cols, m, 0, ld, 0, type};
        return FG_OK;
    }
    const int parts = type == FG_F32 ? 3 : 1;
    *out = Matrix{*work, cols, m * parts, 0, pitch_of(cols, type), 0, type == FG_F32 ? FG_BF16 : type};
    return pack(p, 0, ld, 1, 1, m, cols, order, choices, source_rows, type, work, s);
}

// Few fp32 rows (or a weight off the 16-byte grid), a dense inner axis and 8 rows of it in shared memory: the form without
// tiles, which reads the weights as they are.
bool few_rows(int64_t num_rows, const void* w, int64_t w_group, int64_t w_out, int64_t w_in, int32_t inner, int32_t type) {
    return num_rows <= kFewRows && (w_in == 1 || inner == 1) && round_up(inner, 16) * 8 * fg::type_size(type) <= 192 * 1024 &&
           !loadable(w, w_out, w_group, type);
}
// Few rows that stay in shared memory beside 8 stages of weights: their bytes there; 0 where they do not.
int64_t held_bytes(int64_t num_rows, int32_t inner, int32_t type) {
    if (num_rows > kFewRows || type == FG_F32) return 0;
    const int64_t bytes = round_up((int64_t)inner * fg::type_size(type), 2 * kChunkBytes) * round_up(num_rows, 8);
    return bytes <= 64 * 1024 ? bytes : 0;
}
template <typename T>
int launch_few(const FewArgs& a, cudaStream_t s) {
    const int held = a.m < 8 ? (a.m <= 2 ? a.m : a.m <= 4 ? 4 : 8) : 8;
    const size_t smem = (size_t)held * a.pitch * sizeof(T);
    if (smem > 40 * 1024) FG_CUDA_TRY(cudaFuncSetAttribute(few_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    const dim3 grid((a.outer + kFewCols - 1) / kFewCols, a.m < a.groups ? a.m : a.groups);
    few_rows_kernel<T><<<grid, 256, smem, s>>>(a);
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return FG_OK;
}

// Rows that the product gathers itself: 16- or 8-bit ones on the 16-byte grid, many of them for at most 256 columns, where the
// copy in slot order would be much of the work.  16-byte copies by a few warps fill a stage more slowly than TMA does, and
// every column tile (one from some 18000 slots on, up to four below) fetches its rows again.  Gathered / copied first, in bf16:
// 55960 slots, 2160 to 64 50 / 134 us; 32854, 1776 to 208 48 / 79; 65536, 256 to 256 26 / 31; but 65536, 2048 to 4096
// 1230 / 912, and 2000, 1024 to 512 20 / 16.  Several tiles, 4096 to 256: 16384 68 / 86, 12000 64 / 69, 8192 in two groups
// 55 / 50, in sixteen 34 / 46; 1024 to 256: 16384 22 / 23, 12000 22 / 20, 8192 19.5 / 17.4 and 14.4 / 15.5.
bool rows_gathered(const void* p, int64_t ld, const int32_t* order, int64_t m, int32_t outer, int32_t type) {
    return order && outer <= 256 && m >= 8192 && loadable(p, ld, 0, type);
}

// The weight is read as it is stored where its inner or its outer axis is dense (8-bit products want the inner one), or
// copied with that axis dense; a group stride of 0 is one weight for all groups.
struct WeightLayout {
    int64_t count, rows, cols;
    bool b_mn, copy;
    WeightLayout(const void* p, int64_t w_group, int64_t w_out, int64_t w_in, int32_t groups, int32_t inner, int32_t outer, int32_t type) {
        const bool k_dense = w_in == 1 || inner == 1, n_dense = type != FG_E4M3 && (w_out == 1 || outer == 1);
        const bool k_loads = k_dense && loadable(p, w_out, w_group, type), n_loads = n_dense && loadable(p, w_in, w_group, type);
        b_mn = k_loads ? false : n_loads ? true : !k_dense && n_dense;
        copy = !k_loads && !n_loads;
        count = w_group == 0 ? 1 : groups;
        rows = b_mn ? inner : outer;
        cols = b_mn ? outer : inner;
    }
};

template <int BN, Kind KIND, bool WGRAD, bool FEW, int BLOCKS, bool GATHER = false>
int launch_shape(const MmaArgs& a, const CUtensorMap& map_a, const CUtensorMap& map_b, int64_t most_tiles, cudaStream_t s) {
    constexpr int kSmem = Shape<BN, KIND, FEW, BLOCKS>::kSmem;
    const auto kernel = product_kernel<BN, KIND, WGRAD, FEW, BLOCKS, GATHER>;
    cudaLaunchConfig_t config = {};
    config.blockDim = dim3(kThreads<KIND, WGRAD, GATHER>);
    config.dynamicSmemBytes = kSmem;
    config.stream = s;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = BLOCKS, cluster.val.clusterDim.y = 1, cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = BLOCKS == 2 ? 1 : 0;
    static std::atomic<int> resident[fg::kMaxDevices];  // blocks (pairs) that run at once; found once a device, twice does no harm
    const int slot = fg::current_device_slot();
    int most = slot < 0 ? 0 : resident[slot].load();
    if (most == 0) {
        FG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        most = fg::device_props().sm_count;
        if (BLOCKS == 2) {
            config.gridDim = dim3(most / 2 * 2);
            FG_CUDA_TRY(cudaOccupancyMaxActiveClusters(&most, kernel, &config));
            if (most < 1) return fg::fail(FG_ERR_CUDA, "no room for a pair of blocks");
        }
        if (slot >= 0) resident[slot].store(most);
    }
    config.gridDim = dim3((unsigned)(most_tiles < most ? most_tiles : most) * BLOCKS);
    FG_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, a, map_a, map_b));
    fg::count_launches(1);
    return FG_OK;
}
// bn 512 stands for pairs of blocks: 256 x 256 tiles.
template <Kind KIND, bool WGRAD>
int launch(int bn, const MmaArgs& a, const CUtensorMap& map_a, const CUtensorMap& map_b, int64_t most_tiles, cudaStream_t s) {
    if constexpr (KIND == kCut) return launch_shape<64, kCut, false, false, 1>(a, map_a, map_b, most_tiles, s);
    if constexpr (KIND != kParts && KIND != kCut) {
        if constexpr (!WGRAD)
            if (a.held) return launch_shape<64, KIND, false, true, 1>(a, map_a, map_b, most_tiles, s);
        if constexpr (!WGRAD)
            if (a.gather)
                return bn == 256   ? launch_shape<256, KIND, false, false, 1, true>(a, map_a, map_b, most_tiles, s)
                       : bn == 128 ? launch_shape<128, KIND, false, false, 1, true>(a, map_a, map_b, most_tiles, s)
                                   : launch_shape<64, KIND, false, false, 1, true>(a, map_a, map_b, most_tiles, s);
        if (bn == 512) return launch_shape<256, KIND, WGRAD, false, 2>(a, map_a, map_b, most_tiles, s);
        if (bn == 256) return launch_shape<256, KIND, WGRAD, false, 1>(a, map_a, map_b, most_tiles, s);
    }
    if constexpr (KIND != kCut)
        return bn == 128 ? launch_shape<128, KIND, WGRAD, false, 1>(a, map_a, map_b, most_tiles, s)
                         : launch_shape<64, KIND, WGRAD, false, 1>(a, map_a, map_b, most_tiles, s);
}

// Columns of an output tile: the widest whose tiles still give each SM one (and of which two stages of parts fit).
int tile_width(int64_t units, int width, int32_t type) {
    for (int bn = type == FG_F32 ? 128 : 256; bn > 64; bn /= 2)
        if (width > bn / 2 && units * ((width + bn - 1) / bn) >= fg::device_props().sm_count) return bn;
    return 64;
}
// Pairs of blocks (256 x 256 tiles) load a third less for the same products, which is what 128 x 256 tiles wait for, but
// leave more of the last tiles empty: taken where the tiles they add are less than a tenth of all, and give
// each pair two.  20000 x 1024 x 1024 over 5 groups in bf16: 43 us, in pairs 37; 32768 x 4096 x 4096 over 8: 783 and 736.
// Not for fp32, whose accumulators are handed over with every chunk: 100003 x 256 x 128, gradient of x, 71 us, in pairs 97.
// `row_tiles`, `row_pairs`: 128- and 256-row tiles.
bool pairs_pay(int64_t row_tiles, int64_t row_pairs, int width, int32_t type) {
    if (type == FG_F32 || width <= 128) return false;
    const int64_t cols = (width + 255) / 256;
    return row_pairs * cols >= fg::device_props().sm_count && row_pairs * 2 * 10 <= row_tiles * 11;
}

// Rows of one partial sum of dW: 0 (none) where the tiles of all groups already give each SM two, else such that they do.
int64_t split_rows(int64_t m, int32_t groups, int64_t tiles) {
    const int64_t want = 2ll * fg::device_props().sm_count;
    if (groups * tiles >= want || m <= 1024) return 0;
    const int64_t parts = (want + tiles - 1) / tiles;
    int64_t rows = round_up((m + parts - 1) / parts, 64);
    return rows < 512 ? 512 : rows;
}
int64_t wgrad_tiles(int32_t inner, int32_t outer) {
    return (int64_t)((outer + kTileRows - 1) / kTileRows) * ((inner + 127) / 128);
}

int64_t partial_bytes(int64_t m, int32_t groups, int32_t inner, int32_t outer) {
    const int64_t split = split_rows(m, groups, wgrad_tiles(inner, outer));
    return split ? round_up((m / split + groups) * (int64_t)inner * outer * 4, 256) : 0;
}

int check_product(int64_t m, int64_t x_rows, int32_t choices, int32_t groups, int32_t inner, int32_t outer, int32_t type) {
    if (m < 0 || m > INT_MAX - 1024 || x_rows < 0 || x_rows > INT_MAX || choices < 1 || groups < 1 || groups > kMaxGroups || inner < 1 || outer < 1 ||
        inner > INT_MAX - 1024 || outer > INT_MAX - 1024 ||
        (type == FG_F32 && (m > INT_MAX / 4 || x_rows > INT_MAX / 4)))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "bad sizes rows=%lld of %lld choices=%d groups=%d inner=%d outer=%d (groups <= %d)",
                        (long long)m, (long long)x_rows, choices, groups, inner, outer, kMaxGroups);
    return FG_OK;
}

// Bytes of the slots' 32-bit parts of a gathered row's gradient.
int64_t slot_parts_bytes(int64_t m, int32_t inner) { return round_up(m * (int64_t)inner * 4, 256); }

// A launch's sizes and lists, as the entry points get them.
struct Problem {
    const int32_t *offsets, *order;
    int64_t m, x_rows;
    int32_t choices, groups, inner, outer, type;
};

int64_t weight_bytes(const Problem& p, const void* w, int64_t w_group, int64_t w_out, int64_t w_in) {
    const WeightLayout layout(w, w_group, w_out, w_in, p.groups, p.inner, p.outer, p.type);
    return layout.copy ? packed_bytes(layout.count * layout.rows, layout.cols, p.type) : 0;
}

// y = products of the slots' rows; `x` as loads see them, or, where `held`, as they lie (d_x, ldx, by the order).
int run_product(const Problem& p, const Matrix& x, const void* d_x, int64_t ldx, const float* x_scales, const void* d_w, int64_t w_group,
                int64_t w_out, int64_t w_in, const float* w_scales, int64_t held, void* d_y, int32_t out_type, uint8_t** work, cudaStream_t s) {
    const WeightLayout layout(d_w, w_group, w_out, w_in, p.groups, p.inner, p.outer, p.type);
    const bool b_mn = layout.b_mn;
    const int64_t step = b_mn ? w_in : w_out;  // of the weight's rows as stored
    Matrix w;
    if (!layout.copy) {
        w = Matrix{d_w, layout.cols, layout.rows, layout.count, step, w_group ? w_group : layout.rows * step, p.type};
    } else {
        const int64_t pitch = pitch_of(layout.cols, p.type);
        w = Matrix{*work, layout.cols, layout.rows, layout.count * (p.type == FG_F32 ? 3 : 1), pitch, layout.rows * pitch, p.type == FG_F32 ? FG_BF16 : p.type};
        if (int rc = pack(d_w, w_group, step, b_mn ? w_out : w_in, layout.count, layout.rows, layout.cols, nullptr, 1, 0, p.type, work, s)) return rc;
    }
    const int64_t units = p.m / kTileRows + (p.groups < p.m ? p.groups : p.m);
    // half a tile of each group is empty on average
    const int64_t expected = p.m / kTileRows + p.groups / 2, expected_pairs = p.m / (2 * kTileRows) + p.groups / 2;
    const bool cut = p.type == FG_F32 && x.type == FG_F32;  // rows as they are
    const bool gather = !held && rows_gathered(d_x, ldx, p.order, p.m, p.outer, p.type);
    const bool paired = !held && !gather && pairs_pay(expected, expected_pairs, p.outer, p.type);
    const int bn = held || cut ? 64 : paired ? 512 : tile_width(units, p.outer, p.type), chunk = p.type == FG_E4M3 ? 128 : 64;
    CUtensorMap map_x = {}, map_w;
    if (!held && !gather)
        if (int rc = make_map(&map_x, x, cut ? 32 : chunk, kTileRows)) return rc;
    if (int rc = make_map(&map_w, w, chunk, b_mn ? 64 : paired ? 128 : bn)) return rc;
    MmaArgs a{};
    a.offsets = p.offsets, a.order = p.order, a.x_scales = x_scales, a.w_scales = w_scales, a.y = d_y;
    a.m = p.m, a.x_rows = p.x_rows, a.choices = p.choices, a.groups = p.groups, a.inner = p.inner, a.outer = p.outer;
    a.out_type = out_type, a.format = w.type == FG_BF16 ? 1 : 0;
    a.b_mn = b_mn, a.shared_weight = w_group == 0;
    a.x = d_x, a.ldx = ldx, a.held = (int32_t)held, a.vector_rows = fg::aligned16(d_x) && ldx * fg::type_size(p.type) % 16 == 0;
    a.stages = (int32_t)((196608 - held) / 16384), a.gather = gather;
    const int64_t tiles = units * ((p.outer + (paired ? 256 : bn) - 1) / (paired ? 256 : bn));
    return p.type == FG_E4M3  ? launch<kEight, false>(bn, a, map_x, map_w, tiles, s)
           : cut              ? launch<kCut, false>(bn, a, map_x, map_w, tiles, s)
           : p.type == FG_F32 ? launch<kParts, false>(bn, a, map_x, map_w, tiles, s)
                              : launch<kHalf, false>(bn, a, map_x, map_w, tiles, s);
}

// dW = sums over each group's rows of dy x^T; `sums`: partial_bytes() of workspace.
int run_weight_gradient(const Problem& p, const Matrix& x, const Matrix& dy, void* d_dw, float* sums, cudaStream_t s) {
    const int64_t cells = (int64_t)p.inner * p.outer, split = split_rows(p.m, p.groups, wgrad_tiles(p.inner, p.outer));
    CUtensorMap map_x, map_dy;
    if (int rc = make_map(&map_dy, dy, 64, 64)) return rc;
    if (int rc = make_map(&map_x, x, 64, 64)) return rc;
    const int64_t units = split ? p.m / split + p.groups : p.groups, rows_tiles = (p.outer + kTileRows - 1) / kTileRows;
    // in pairs, the columns' waste counts as well as the rows', and a short sum is mostly output: 256 rows a group, 128
    // groups of 2048 x 1408 took 325 us in pairs and 292 without, 1024 rows and more are faster in pairs
    const int64_t singles = units * rows_tiles * ((p.inner + 127) / 128), doubles = units * ((p.outer + 255) / 256) * ((p.inner + 255) / 256);
    const bool paired = p.m >= 768 * units && pairs_pay(singles, doubles * 2, 256, p.type);
    const int bn = paired ? 512 : tile_width(units * rows_tiles, p.inner, p.type);
    MmaArgs a{};
    a.offsets = p.offsets, a.y = split ? static_cast<void*>(sums) : d_dw;
    a.m = p.m, a.x_rows = p.x_rows, a.choices = p.choices, a.groups = p.groups, a.inner = p.inner, a.outer = p.outer;
    a.out_type = split ? FG_F32 : p.type, a.format = dy.type == FG_BF16 ? 1 : 0;
    a.split = (int32_t)split, a.units = (int32_t)units;
    const int64_t tiles = paired ? doubles : units * rows_tiles * ((p.inner + bn - 1) / bn);
    if (int rc = p.type == FG_F32 ? launch<kParts, true>(bn, a, map_dy, map_x, tiles, s) : launch<kHalf, true>(bn, a, map_dy, map_x, tiles, s)) return rc;
    if (!split) return FG_OK;
    const dim3 grid((unsigned)((cells + 255) / 256 < 4096 ? (cells + 255) / 256 : 4096), (unsigned)p.groups);
    if (p.type == FG_F32) join_kernel<float><<<grid, 256, 0, s>>>(sums, p.offsets, p.groups, p.m, (int)split, a.units, cells, static_cast<float*>(d_dw));
    else if (p.type == FG_F16) join_kernel<__half><<<grid, 256, 0, s>>>(sums, p.offsets, p.groups, p.m, (int)split, a.units, cells, static_cast<__half*>(d_dw));
    else join_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(sums, p.offsets, p.groups, p.m, (int)split, a.units, cells, static_cast<__nv_bfloat16*>(d_dw));
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return FG_OK;
}

// The gradient of x, slot by slot, is a product with the weight read the other way.
Problem other_way(const Problem& p) {
    Problem q = p;
    q.order = nullptr, q.choices = 1, q.x_rows = p.m, q.inner = p.outer, q.outer = p.inner;
    return q;
}

}  // namespace

extern "C" {

int fg_wait_status(void* stream) {
    int product = 0, norm = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    FG_CUDA_TRY(cudaMemcpyFromSymbolAsync(&product, g_stuck, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
    if (int rc = fg::norm_stuck(s, &norm)) return rc;
    FG_CUDA_TRY(cudaStreamSynchronize(s));
    return product || norm ? fg::fail(FG_ERR_CUDA, "%s gave up waiting for its own copies", product ? "a grouped product" : "a norm of rows, its gradient or 8-bit form") : FG_OK;
}

int64_t fg_grouped_matmul_workspace(const void* d_x, int64_t ldx, const void* d_w, int64_t w_group, int64_t w_out, int64_t w_in,
                                    const int32_t* d_order, int64_t num_rows, int32_t groups, int32_t inner, int32_t outer, int32_t type) {
    if (num_rows <= 0 || groups < 1 || inner < 1 || outer < 1 || few_rows(num_rows, d_w, w_group, w_out, w_in, inner, type)) return 0;
    const WeightLayout w(d_w, w_group, w_out, w_in, groups, inner, outer, type);
    const bool as_is = held_bytes(num_rows, inner, type) || rows_cut_on_the_way(d_x, ldx ? ldx : inner, d_order, outer, type) ||
                       rows_gathered(d_x, ldx ? ldx : inner, d_order, num_rows, outer, type);
    return (!as_is && rows_need_copy(d_x, ldx ? ldx : inner, d_order, type) ? packed_bytes(num_rows, inner, type) : 0) +
           (w.copy ? packed_bytes(w.count * w.rows, w.cols, type) : 0);
}

int fg_grouped_matmul(const void* d_x, int64_t ldx, const float* d_x_scales, const void* d_w, int64_t w_group, int64_t w_out,
                      int64_t w_in, const float* d_w_scales, const int32_t* d_offsets, const int32_t* d_order, int32_t choices,
                      int64_t x_rows, void* d_y, int64_t num_rows, int32_t groups, int32_t inner, int32_t outer, int32_t type,
                      int32_t out_type, void* d_workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_product(num_rows, x_rows, choices, groups, inner, outer, type)) return rc;
    if (!fg::float_type(type) && type != FG_E4M3) return fg::fail(FG_ERR_INVALID_ARGUMENT, "unknown value type %d", type);
    if (type == FG_E4M3 ? !fg::float_type(out_type) : out_type != type)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "the output is of the inputs' type, or of a wider one for e4m3");
    if (ldx == 0) ldx = inner;
    if (ldx < inner) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= inner=%d", inner);
    if (w_group < 0 || w_out < 0 || w_in < 0) return fg::fail(FG_ERR_INVALID_ARGUMENT, "the weight's strides must be >= 0");
    if (num_rows == 0) return FG_OK;
    if (!d_x || !d_w || !d_offsets || !d_y || (type == FG_E4M3 && (!d_x_scales || !d_w_scales)))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    if (!d_order && x_rows != num_rows) return fg::fail(FG_ERR_INVALID_ARGUMENT, "without an order x has a row for each slot");
    cudaStream_t s = static_cast<cudaStream_t>(stream);

    if (few_rows(num_rows, d_w, w_group, w_out, w_in, inner, type)) {
        const int size = fg::type_size(type);
        FewArgs f{d_x, d_w, type == FG_E4M3 ? d_x_scales : nullptr, type == FG_E4M3 ? d_w_scales : nullptr, d_offsets, d_order, d_y, ldx, w_group, w_out, x_rows,
                  (int32_t)num_rows, choices, groups, inner, outer, out_type, (int32_t)round_up(inner, 16), false, false};
        f.vector_rows = fg::aligned16(d_x) && ldx * size % 16 == 0;
        f.vector = fg::aligned16(d_w) && w_out * size % 16 == 0 && w_group * size % 16 == 0;
        return type == FG_F32   ? launch_few<float>(f, s)
               : type == FG_F16 ? launch_few<__half>(f, s)
               : type == FG_BF16 ? launch_few<__nv_bfloat16>(f, s)
                                 : launch_few<__nv_fp8_e4m3>(f, s);
    }
    const int64_t need = fg_grouped_matmul_workspace(d_x, ldx, d_w, w_group, w_out, w_in, d_order, num_rows, groups, inner, outer, type);
    if (workspace_bytes < need || (need && !d_workspace)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "workspace smaller than fg_grouped_matmul_workspace()");
    if (need && !fg::aligned16(d_workspace)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "the workspace must start on a 16-byte boundary");
    uint8_t* work = static_cast<uint8_t*>(d_workspace);
    const Problem p{d_offsets, d_order, num_rows, x_rows, choices, groups, inner, outer, type};
    Matrix x{};
    const int64_t held = held_bytes(num_rows, inner, type);
    if (rows_cut_on_the_way(d_x, ldx, d_order, outer, type)) x = Matrix{d_x, inner, num_rows, 0, ldx, 0, type};
    else if (!held && !rows_gathered(d_x, ldx, d_order, num_rows, outer, type))
        if (int rc = rows_matrix(&x, d_x, ldx, x_rows, d_order, choices, num_rows, inner, type, &work, s)) return rc;
    return run_product(p, x, d_x, ldx, d_x_scales, d_w, w_group, w_out, w_in, d_w_scales, held, d_y, out_type, &work, s);
}

int64_t fg_grouped_matmul_backward_workspace(const void* d_x, int64_t ldx, const void* d_w, int64_t w_group, int64_t w_out, int64_t w_in,
                                             const int32_t* d_order, const void* d_dy, int64_t lddy, int32_t want_dx, int32_t want_dw,
                                             int64_t num_rows, int32_t groups, int32_t inner, int32_t outer, int32_t type) {
    if (num_rows <= 0 || groups < 1 || inner < 1 || outer < 1) return 0;
    const Problem p{nullptr, d_order, num_rows, 0, 1, groups, inner, outer, type};
    return (rows_need_copy(d_dy, lddy ? lddy : outer, nullptr, type) ? packed_bytes(num_rows, outer, type) : 0) +
           (want_dx ? weight_bytes(other_way(p), d_w, w_group, w_in, w_out) : 0) +
           (want_dx && d_order ? slot_parts_bytes(num_rows, inner) : 0) +
           (want_dw ? partial_bytes(num_rows, groups, inner, outer) : 0) +
           (want_dw && rows_need_copy(d_x, ldx ? ldx : inner, d_order, type) ? packed_bytes(num_rows, inner, type) : 0);
}

int fg_grouped_matmul_backward(const void* d_x, int64_t ldx, const void* d_w, int64_t w_group, int64_t w_out, int64_t w_in,
                               const int32_t* d_offsets, const int32_t* d_order, const int32_t* d_position, int32_t choices, int64_t x_rows,
                               const void* d_dy, int64_t lddy, void* d_dx, void* d_dw, int64_t num_rows, int32_t groups, int32_t inner,
                               int32_t outer, int32_t type, void* d_workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_product(num_rows, x_rows, choices, groups, inner, outer, type)) return rc;
    if (!fg::float_type(type)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "unknown value type %d", type);
    if (ldx == 0) ldx = inner;
    if (lddy == 0) lddy = outer;
    if (ldx < inner || lddy < outer) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= the width");
    if (w_group < 0 || w_out < 0 || w_in < 0) return fg::fail(FG_ERR_INVALID_ARGUMENT, "the weight's strides must be >= 0");
    if (!d_dx && !d_dw) return FG_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (num_rows == 0) {  // no slots: no rows of x either
        if (d_dw) FG_CUDA_TRY(cudaMemsetAsync(d_dw, 0, (size_t)groups * inner * outer * fg::type_size(type), s));
        return FG_OK;
    }
    if (!d_offsets || !d_dy || (d_dw && !d_x) || (d_dx && !d_w) || (d_order && !d_position))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    if (!d_order && x_rows != num_rows) return fg::fail(FG_ERR_INVALID_ARGUMENT, "without an order x has a row for each slot");
    if (d_order && x_rows * choices != num_rows) return fg::fail(FG_ERR_INVALID_ARGUMENT, "the order lists `choices` slots a row of x");
    const int64_t need = fg_grouped_matmul_backward_workspace(d_x, ldx, d_w, w_group, w_out, w_in, d_order, d_dy, lddy, d_dx != nullptr, d_dw != nullptr,
                                                              num_rows, groups, inner, outer, type);
    if (workspace_bytes < need || (need && !d_workspace))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "workspace smaller than fg_grouped_matmul_backward_workspace()");
    if (need && !fg::aligned16(d_workspace)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "the workspace must start on a 16-byte boundary");
    uint8_t* work = static_cast<uint8_t*>(d_workspace);
    const Problem p{d_offsets, d_order, num_rows, x_rows, choices, groups, inner, outer, type};
    // dW needs dy in parts; alone, dx may take it as it is
    Matrix dy;
    if (!d_dw && rows_cut_on_the_way(d_dy, lddy, nullptr, inner, type)) dy = Matrix{d_dy, outer, num_rows, 0, lddy, 0, type};
    else if (int rc = rows_matrix(&dy, d_dy, lddy, num_rows, nullptr, 1, num_rows, outer, type, &work, s)) return rc;
    if (d_dx) {
        // A gathered row's gradient is the sum over its slots.  The slots' parts stay in 32 bits and the sum is rounded once: parts
        // in x's type would add a rounding each, and in fp16 overflow where their sum does not.  One slot a row has nothing
        // to add, so its part is rounded as the product leaves it.
        const int32_t parts_type = choices > 1 ? FG_F32 : type;
        void* parts = d_dx;
        if (d_order) {
            parts = work;
            work += slot_parts_bytes(num_rows, inner);
        }
        if (int rc = run_product(other_way(p), dy, nullptr, 0, nullptr, d_w, w_group, w_in, w_out, nullptr, 0, parts, d_order ? parts_type : type, &work, s))
            return rc;
        if (d_order && parts_type == FG_F32) {
            if (int rc = fg::sum_slots(static_cast<const float*>(parts), d_position, d_dx, x_rows, choices, inner, type, s)) return rc;
        } else if (d_order) {
            if (int rc = fg_combine_rows(parts, 0, nullptr, d_position, d_dx, x_rows, choices, inner, type, stream)) return rc;
        }
    }
    if (!d_dw) return FG_OK;
    float* sums = reinterpret_cast<float*>(work);
    work += partial_bytes(num_rows, groups, inner, outer);
    Matrix x;
    if (int rc = rows_matrix(&x, d_x, ldx, x_rows, d_order, choices, num_rows, inner, type, &work, s)) return rc;
    return run_weight_gradient(p, x, dy, d_dw, sums, s);
}

}  // extern "C"
