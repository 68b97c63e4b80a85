// Root-mean-square norm of rows with the residual's addition, its 8-bit form, and its gradient.
//
//   h = round(x + residual)      y = h * r * w,   r = 1 / sqrt(mean(h^2) + eps)
//   8 bits: s = max|h r w| / 448 (1 where that is 0 in 32 bits),  q = e4m3(h r w / s)
//   dx = dresidual = dh + r (g - (h r) (r / d * sum(g h))),  g = dy w;      dw = sum over rows of dy h r
//   (r^3 would leave the 32-bit range before dx does: without eps at rows of 1e-18)
//
// Bound: device memory - each array is touched once.  TPR threads own a row and hold its E values each in
// registers between the reductions and the output, so a row is read once whatever is computed from it (its sum of
// squares, its largest value, its products with the incoming gradient); a row wider than TPR * E goes to the next
// larger TPR.  The statistics are recomputed from h in the backward pass: h has to be read there in any case, and a
// saved r would be one more array.  All sums are 32-bit; h is rounded to its type before it is normalised, because
// the rounded value is what the following layers add to and what the backward pass reads.
//
// dw: each block adds the rows it walks into registers (a fixed row sequence per block) and writes one partial row;
// a second kernel adds the partial rows in order.  No atomics: the same bits on every run.
#include <climits>

#include "rows.cuh"
#include "tcgen05.cuh"

namespace {

using fg::from_f32;
using fg::load_pack;
using fg::Pack;
using fg::store_pack;
using fg::to_f32;

constexpr int kE4M3Max = 448, kMaxStages = 8;

__device__ int g_stuck;  // set when a wait for a copy ran out

__device__ __forceinline__ float weight_at(const void* w, bool f32, int i, float) {
    return w == nullptr ? 1.0f : static_cast<const float*>(w)[i];
}
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, bool f32, int i, T) {
    if (w == nullptr) return 1.0f;
    return f32 ? static_cast<const float*>(w)[i] : to_f32<T>(static_cast<const T*>(w)[i]);
}

// Waits for the other threads of the row (named barriers where a block holds several rows of several warps).
template <int TPR, int THREADS>
__device__ __forceinline__ void row_sync(int sub) {
    if (TPR == 32) __syncwarp();
    else if (TPR == THREADS) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(sub + 1), "n"(TPR) : "memory");
}

// Two sums over the TPR threads of a row, through one of two buffers in turn, so that a row needs one barrier.
template <int TPR, int THREADS>
__device__ __forceinline__ void row_sums(float& x, float& y, float2* buffer, int sub) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, o));
        y = __fadd_rn(y, __shfl_xor_sync(0xffffffffu, y, o));
    }
    if (TPR == 32) return;
    constexpr int kWarps = TPR / 32;
    if ((threadIdx.x & 31) == 0) buffer[threadIdx.x >> 5] = make_float2(x, y);
    row_sync<TPR, THREADS>(sub);
    const float2 v = buffer[sub * kWarps];
    x = v.x, y = v.y;
#pragma unroll
    for (int i = 1; i < kWarps; ++i) {
        const float2 w = buffer[sub * kWarps + i];
        x = __fadd_rn(x, w.x), y = __fadd_rn(y, w.y);
    }
}
// One sum, or the largest value (a NaN wins).
template <int TPR, int THREADS, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* buffer, int sub) {
    v = MAX ? fg::warp_max(v) : fg::warp_sum(v);
    if (TPR == 32) return v;
    constexpr int kWarps = TPR / 32;
    if ((threadIdx.x & 31) == 0) buffer[threadIdx.x >> 5] = v;
    row_sync<TPR, THREADS>(sub);
    v = buffer[sub * kWarps];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) {
        const float w = buffer[sub * kWarps + i];
        if (MAX) v = (w > v || w != w) ? w : v;
        else v = __fadd_rn(v, w);
    }
    return v;
}

// The scale of an 8-bit row whose largest value is `most`.  The quotient is 0 for a row of zeros, and for one of up to 224 steps
// of 2^-149: 1 then, since a scale of 0 would make NaN of its zeros.  A quotient of few steps is rounded up: to nearest it
// could lose a thirtieth and more, and the largest values would lie beyond 464, the last number that rounds to 448; from 16
// steps on they cannot (448 x 16.5 / 16 = 462).  Infinities and NaN stay what they are.
__device__ __forceinline__ float row_scale(float most) {
    const float s = __fdiv_rn(most, (float)kE4M3Max);
    return s == 0.0f ? 1.0f : s < 0x1p-145f ? __fdiv_ru(most, (float)kE4M3Max) : s;
}

// The ring of a row's TPR threads: `stages` rows of ARRAYS arrays ahead of them in shared memory, filled by bulk copies, so
// that what is in flight takes no registers (the gradient of 32768 x 4096 bf16 took 253 us with the next row in
// registers and 16 warps an SM, 163 us with the ring).  A row that starts off the 16-byte grid is copied from the
// grid point before it on, up to 15 bytes more on either side, in the 16-byte units that hold its first and last values.
// A stage is free again as soon as its values are in registers, which a barrier of the row's threads shows.
template <typename T, int VEC, int ARRAYS>
struct RowRing {
    uint64_t* full;
    const uint8_t* mine;
    int32_t stages, slot, d;
    int* stop;
    int s = 0, parity = 0;
    const T* arrays[ARRAYS];
    int64_t ld[ARRAYS];

    __device__ uint64_t address(int q, int64_t row) const { return reinterpret_cast<uint64_t>(arrays[q] + row * ld[q]); }
    __device__ void request(int stage, int64_t row) const {  // one thread of the row
        const uint32_t bar = fg::smem_address(full + stage), to = fg::smem_address(mine) + stage * ARRAYS * slot;
        uint64_t lo[ARRAYS];
        uint32_t bytes[ARRAYS], all = 0;
#pragma unroll
        for (int q = 0; q < ARRAYS; ++q) {
            const uint64_t from = address(q, row);
            lo[q] = from & ~15ull;
            bytes[q] = (uint32_t)(((from + (uint64_t)d * sizeof(T) + 15) & ~15ull) - lo[q]);
            all += bytes[q];
        }
        fg::barrier_expect(bar, all);
#pragma unroll
        for (int q = 0; q < ARRAYS; ++q) fg::bulk_load(to + q * slot, lo[q], bytes[q], bar);
    }
    // The row's values of array q, in the current stage; rows that are read in vectors start on the grid.
    __device__ const T* values(int q, int64_t row) const {
        return reinterpret_cast<const T*>(mine + (s * ARRAYS + q) * slot + (VEC == 1 ? (uint32_t)address(q, row) & 15 : 0));
    }
    __device__ void wait() { fg::barrier_wait(fg::smem_address(full + s), parity, stop); }  // without the copy: wrong values, and the flag
    __device__ void next() {
        if (++s == stages) s = 0, parity ^= 1;
    }
    __device__ void drain() const {  // a wait ran out: the copies that are left end before the block does
        for (int q = 0; q < stages; ++q) {
            fg::barrier_wait(fg::smem_address(full + q), 0, stop, true);
            fg::barrier_wait(fg::smem_address(full + q), 1, stop, true);
        }
    }
};

struct NormArgs {
    const void *x, *residual, *weight;
    void *h, *y;
    float* scales;
    int64_t ldx, ldr, n;
    int32_t d, stages, slot;  // slot: bytes of one array's row in shared memory
    float eps;
    bool weight_f32, normalize, e4m3;
};

template <typename T, int VEC, int TPR, int E, bool RES>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, TPR <= 256 ? 2 : 1) norm_kernel(const NormArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR, NV = E / VEC, kArrays = RES ? 2 : 1;
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ uint64_t full[kRows][kMaxStages];
    __shared__ float buffer[4][kThreads / 32];  // in turn: a row's barrier shows that the row before it has been read
    __shared__ int stop;
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int64_t first = (int64_t)blockIdx.x * kRows + sub, step = (int64_t)gridDim.x * kRows;
    const float over_d = __fdiv_rn(1.0f, (float)a.d);
    RowRing<T, VEC, kArrays> ring{full[sub], dynamic + sub * a.stages * kArrays * a.slot, a.stages, a.slot, a.d, &stop};
    ring.arrays[0] = static_cast<const T*>(a.x), ring.ld[0] = a.ldx;
    if (RES) ring.arrays[kArrays - 1] = static_cast<const T*>(a.residual), ring.ld[kArrays - 1] = a.ldr;
    if (t == 0)
        for (int s = 0; s < a.stages; ++s) fg::barrier_init(fg::smem_address(&full[sub][s]), 1);
    if (threadIdx.x == 0) stop = 0;
    fg::barrier_init_fence();
    __syncthreads();
    if (t == 0)
        for (int s = 0; s < a.stages; ++s)
            if (first + s * step < a.n) ring.request(s, first + s * step);
    float weight[E];  // the thread's columns: the same for all rows
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int i = (c * TPR + t) * VEC + j;
            weight[c * VEC + j] = i < a.d ? weight_at(a.weight, a.weight_f32, i, T()) : 0.0f;
        }
    int turn = 0;
    for (int64_t row = first; row < a.n; row += step, turn ^= 1) {
        ring.wait();
        Pack<T, VEC> p[NV];
        const T* xs = ring.values(0, row);
        const T* rs = ring.values(kArrays - 1, row);
        T* h = static_cast<T*>(a.h) + row * a.d;
        float v[E], ss = 0.0f;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (i < a.d) {
                p[c] = load_pack<T, VEC>(xs + i);
                if (RES) {
                    const Pack<T, VEC> q = load_pack<T, VEC>(rs + i);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) p[c].v[j] = from_f32<T>(__fadd_rn(to_f32<T>(p[c].v[j]), to_f32<T>(q.v[j])));
                    store_pack<T, VEC>(h + i, p[c]);
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float u = i < a.d ? to_f32<T>(p[c].v[j]) : 0.0f;
                v[c * VEC + j] = u;
                ss = __fmaf_rn(u, u, ss);
            }
        }
        ss = row_reduce<TPR, kThreads, false>(ss, buffer[turn], sub);
        if (TPR == 32) __syncwarp();
        if (t == 0 && row + a.stages * step < a.n) ring.request(ring.s, row + a.stages * step);
        ring.next();
        if (a.normalize) {
            const float r = __frsqrt_rn(__fmaf_rn(ss, over_d, a.eps));
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = __fmul_rn(__fmul_rn(v[e], r), weight[e]);
        }
        if (!a.e4m3) {
            T* y = static_cast<T*>(a.y) + row * a.d;
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const int i = (c * TPR + t) * VEC;
                if (i < a.d) {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o.v[j] = from_f32<T>(v[c * VEC + j]);
                    store_pack<T, VEC>(y + i, o);
                }
            }
            continue;
        }
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float u = fabsf(v[e]);
            most = (u > most || u != u) ? u : most;
        }
        most = row_reduce<TPR, kThreads, true>(most, buffer[2 + turn], sub);
        const float scale = row_scale(most);
        uint8_t* q = static_cast<uint8_t*>(a.y) + row * a.d;
        if (t == 0) a.scales[row] = scale;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (i < a.d) {
                Pack<uint8_t, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    o.v[j] = __nv_cvt_float_to_fp8(__fdiv_rn(v[c * VEC + j], scale), __NV_SATFINITE, __NV_E4M3);
                store_pack<uint8_t, VEC>(q + i, o);
            }
        }
    }
    if (stop) {
        if (t == 0) ring.drain();
        if (threadIdx.x == 0) atomicExch(&g_stuck, 1);
    }
}

struct NormGradArgs {
    const void *h, *weight, *dy, *dh;
    void* dx;
    float* partial;  // [gridDim.x, d], or NULL where the weight's gradient is not wanted
    int64_t ldh, lddy, lddh, n;
    int32_t d, stages, slot;  // slot: bytes of one array's row in shared memory
    float eps;
    bool weight_f32;
};

template <typename T, int VEC, int TPR, int E, bool DH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, TPR <= 256 ? 2 : 1) norm_grad_kernel(const NormGradArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR, NV = E / VEC;
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ uint64_t full[kRows][kMaxStages];
    __shared__ float2 buffer[2][kThreads / 32];
    __shared__ float across[kRows > 1 ? kRows * TPR * E : 1];
    __shared__ int stop;
    constexpr int kArrays = DH ? 3 : 2;
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float over_d = __fdiv_rn(1.0f, (float)a.d);
    const int64_t first = (int64_t)blockIdx.x * kRows + sub, step = (int64_t)gridDim.x * kRows;
    RowRing<T, VEC, kArrays> ring{full[sub], dynamic + sub * a.stages * kArrays * a.slot, a.stages, a.slot, a.d, &stop};
    ring.arrays[0] = static_cast<const T*>(a.h), ring.ld[0] = a.ldh;
    ring.arrays[1] = static_cast<const T*>(a.dy), ring.ld[1] = a.lddy;
    if (DH) ring.arrays[kArrays - 1] = static_cast<const T*>(a.dh), ring.ld[kArrays - 1] = a.lddh;
    if (t == 0)
        for (int s = 0; s < a.stages; ++s) fg::barrier_init(fg::smem_address(&full[sub][s]), 1);
    if (threadIdx.x == 0) stop = 0;
    fg::barrier_init_fence();
    __syncthreads();
    if (t == 0)
        for (int s = 0; s < a.stages; ++s)
            if (first + s * step < a.n) ring.request(s, first + s * step);
    float acc[E], weight[E];  // the thread's columns: the same for all rows
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int i = (c * TPR + t) * VEC + j;
            acc[c * VEC + j] = 0.0f;
            weight[c * VEC + j] = i < a.d ? weight_at(a.weight, a.weight_f32, i, T()) : 0.0f;
        }
    int turn = 0;
    for (int64_t row = first; row < a.n; row += step, turn ^= 1) {
        ring.wait();
        Pack<T, VEC> h[NV], g[NV], d[NV];
        const T* hs = ring.values(0, row);
        const T* gs = ring.values(1, row);
        const T* ds = ring.values(kArrays - 1, row);
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (i < a.d) {
                h[c] = load_pack<T, VEC>(hs + i);
                g[c] = load_pack<T, VEC>(gs + i);
                if (DH) d[c] = load_pack<T, VEC>(ds + i);
            }
        }
        float ss = 0.0f, sg = 0.0f;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (i < a.d) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float u = to_f32<T>(h[c].v[j]);
                    const float v = __fmul_rn(to_f32<T>(g[c].v[j]), weight[c * VEC + j]);
                    ss = __fmaf_rn(u, u, ss);
                    sg = __fmaf_rn(u, v, sg);
                }
            }
        }
        row_sums<TPR, kThreads>(ss, sg, buffer[turn], sub);
        if (TPR == 32) __syncwarp();
        if (t == 0 && row + a.stages * step < a.n) ring.request(ring.s, row + a.stages * step);
        ring.next();
        const float r = __frsqrt_rn(__fmaf_rn(ss, over_d, a.eps));
        const float along = __fmul_rn(r, __fmul_rn(sg, over_d));
        T* dx = static_cast<T*>(a.dx) + row * a.d;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (i < a.d) {
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float u = to_f32<T>(h[c].v[j]), dyj = to_f32<T>(g[c].v[j]);
                    const float v = __fmul_rn(dyj, weight[c * VEC + j]), unit = __fmul_rn(u, r);
                    float w = __fmul_rn(r, __fmaf_rn(-unit, along, v));
                    if (DH) w = __fadd_rn(w, to_f32<T>(d[c].v[j]));
                    o.v[j] = from_f32<T>(w);
                    acc[c * VEC + j] = __fmaf_rn(dyj, unit, acc[c * VEC + j]);
                }
                store_pack<T, VEC>(dx + i, o);
            }
        }
    }
    if (stop) {
        if (t == 0) ring.drain();
        if (threadIdx.x == 0) atomicExch(&g_stuck, 1);
    }
    if (a.partial == nullptr) return;
    float* out = a.partial + (int64_t)blockIdx.x * a.d;
    if (kRows > 1) {  // the block's row groups hold the same columns: add them in order
#pragma unroll
        for (int e = 0; e < E; ++e) across[(sub * E + e) * TPR + t] = acc[e];
        __syncthreads();
        if (sub != 0) return;
        for (int q = 1; q < kRows; ++q)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = __fadd_rn(acc[e], across[(q * E + e) * TPR + t]);
    }
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int i = (c * TPR + t) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (i + j < a.d) out[i + j] = acc[c * VEC + j];
    }
}

// ---- narrow rows ----

// Rows of at most 128 values: LANES lanes of a warp own a row, 8 values each, so that a warp works on 32 / LANES rows at a
// time, straight from memory with the next rows requested ahead.  A warp and a bulk copy a row, as above, spend their time
// on what does not depend on the width: 435845 x 32 bf16 to e4m3 took 200 us.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <typename T, int VEC>
struct Narrow {
    Pack<T, VEC> v[8 / VEC];
    __device__ void load(const T* row, int first, int d, int lanes, bool live) {
#pragma unroll
        for (int c = 0; c < 8 / VEC; ++c) {
            const int i = (c * lanes + first) * VEC;
            if (live && i < d) v[c] = load_pack<T, VEC>(row + i);
        }
    }
};

template <typename T, int VEC, int LANES, bool RES>
__global__ void __launch_bounds__(256) norm_narrow_kernel(const NormArgs a) {
    constexpr int NV = 8 / VEC;
    const int t = threadIdx.x % LANES, sub = (threadIdx.x & 31) / LANES;
    const float over_d = __fdiv_rn(1.0f, (float)a.d);
    const int64_t step = (int64_t)gridDim.x * (256 / LANES);
    int64_t base = (int64_t)blockIdx.x * (256 / LANES) + (threadIdx.x >> 5) * (32 / LANES);  // the warp's first row
    auto row_of = [&](const void* p, int64_t row, int64_t ld) { return static_cast<const T*>(p) + row * ld; };
    float weight[8];
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int i = (c * LANES + t) * VEC + j;
            weight[c * VEC + j] = i < a.d ? weight_at(a.weight, a.weight_f32, i, T()) : 0.0f;
        }
    Narrow<T, VEC> x, res;
    if (base + sub < a.n) {
        x.load(row_of(a.x, base + sub, a.ldx), t, a.d, LANES, true);
        if (RES) res.load(row_of(a.residual, base + sub, a.ldr), t, a.d, LANES, true);
    }
    for (; base < a.n; base += step) {
        const int64_t row = base + sub, next = row + step;
        const bool live = row < a.n;
        Narrow<T, VEC> p = x, q = res;
        if (next < a.n) {
            x.load(row_of(a.x, next, a.ldx), t, a.d, LANES, true);
            if (RES) res.load(row_of(a.residual, next, a.ldr), t, a.d, LANES, true);
        }
        float v[8], ss = 0.0f;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * LANES + t) * VEC;
            const bool in = live && i < a.d;
            if (RES && in) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) p.v[c].v[j] = from_f32<T>(__fadd_rn(to_f32<T>(p.v[c].v[j]), to_f32<T>(q.v[c].v[j])));
                store_pack<T, VEC>(static_cast<T*>(a.h) + row * a.d + i, p.v[c]);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float u = in ? to_f32<T>(p.v[c].v[j]) : 0.0f;
                v[c * VEC + j] = u;
                ss = __fmaf_rn(u, u, ss);
            }
        }
        if (a.normalize) {
            const float r = __frsqrt_rn(__fmaf_rn(lanes_sum<LANES>(ss), over_d, a.eps));
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __fmul_rn(__fmul_rn(v[e], r), weight[e]);
        }
        float scale = 1.0f;
        if (a.e4m3) {
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float u = fabsf(v[e]);
                most = (u > most || u != u) ? u : most;
            }
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) {
                const float u = __shfl_xor_sync(0xffffffffu, most, o);
                most = (u > most || u != u) ? u : most;
            }
            scale = row_scale(most);
            if (live && t == 0) a.scales[row] = scale;
        }
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * LANES + t) * VEC;
            if (live && i < a.d) {
                if (a.e4m3) {
                    Pack<uint8_t, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        o.v[j] = __nv_cvt_float_to_fp8(__fdiv_rn(v[c * VEC + j], scale), __NV_SATFINITE, __NV_E4M3);
                    store_pack<uint8_t, VEC>(static_cast<uint8_t*>(a.y) + row * a.d + i, o);
                } else {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o.v[j] = from_f32<T>(v[c * VEC + j]);
                    store_pack<T, VEC>(static_cast<T*>(a.y) + row * a.d + i, o);
                }
            }
        }
    }
}

template <typename T, int VEC, int LANES, bool DH>
__global__ void __launch_bounds__(256) norm_narrow_grad_kernel(const NormGradArgs a) {
    constexpr int NV = 8 / VEC;
    __shared__ float across[256 * 8];
    const int t = threadIdx.x % LANES, sub = (threadIdx.x & 31) / LANES;
    const float over_d = __fdiv_rn(1.0f, (float)a.d);
    const int64_t step = (int64_t)gridDim.x * (256 / LANES);
    int64_t base = (int64_t)blockIdx.x * (256 / LANES) + (threadIdx.x >> 5) * (32 / LANES);
    auto row_of = [&](const void* p, int64_t row, int64_t ld) { return static_cast<const T*>(p) + row * ld; };
    float weight[8], acc[8];
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int i = (c * LANES + t) * VEC + j;
            weight[c * VEC + j] = i < a.d ? weight_at(a.weight, a.weight_f32, i, T()) : 0.0f;
            acc[c * VEC + j] = 0.0f;
        }
    Narrow<T, VEC> nh, ng, nd;
    auto request = [&](int64_t row) {
        if (row >= a.n) return;
        nh.load(row_of(a.h, row, a.ldh), t, a.d, LANES, true);
        ng.load(row_of(a.dy, row, a.lddy), t, a.d, LANES, true);
        if (DH) nd.load(row_of(a.dh, row, a.lddh), t, a.d, LANES, true);
    };
    request(base + sub);
    for (; base < a.n; base += step) {
        const int64_t row = base + sub;
        const bool live = row < a.n;
        const Narrow<T, VEC> h = nh, g = ng, d = nd;
        request(row + step);
        float ss = 0.0f, sg = 0.0f;
#pragma unroll
        for (int c = 0; c < NV; ++c)
            if (live && (c * LANES + t) * VEC < a.d)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float u = to_f32<T>(h.v[c].v[j]);
                    ss = __fmaf_rn(u, u, ss);
                    sg = __fmaf_rn(u, __fmul_rn(to_f32<T>(g.v[c].v[j]), weight[c * VEC + j]), sg);
                }
        const float r = __frsqrt_rn(__fmaf_rn(lanes_sum<LANES>(ss), over_d, a.eps));
        const float along = __fmul_rn(r, __fmul_rn(lanes_sum<LANES>(sg), over_d));
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * LANES + t) * VEC;
            if (live && i < a.d) {
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float u = to_f32<T>(h.v[c].v[j]), dyj = to_f32<T>(g.v[c].v[j]);
                    const float unit = __fmul_rn(u, r);
                    float w = __fmul_rn(r, __fmaf_rn(-unit, along, __fmul_rn(dyj, weight[c * VEC + j])));
                    if (DH) w = __fadd_rn(w, to_f32<T>(d.v[c].v[j]));
                    o.v[j] = from_f32<T>(w);
                    acc[c * VEC + j] = __fmaf_rn(dyj, unit, acc[c * VEC + j]);
                }
                store_pack<T, VEC>(static_cast<T*>(a.dx) + row * a.d + i, o);
            }
        }
    }
    if (a.partial == nullptr) return;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) across[(threadIdx.x / LANES) * (LANES * 8) + (c * LANES + t) * VEC + j] = acc[c * VEC + j];
    __syncthreads();
    for (int i = threadIdx.x; i < a.d; i += 256) {  // the block's row groups in order
        float sum = across[i];
        for (int q = 1; q < 256 / LANES; ++q) sum = __fadd_rn(sum, across[q * (LANES * 8) + i]);
        a.partial[(int64_t)blockIdx.x * a.d + i] = sum;
    }
}

// dw[c] = sum of partial[0 .. rows)[c]: 32 columns a block, 32 row sequences each, joined in order.
template <typename W>
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* __restrict__ partial, int rows, int d, W* __restrict__ dw) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, seq = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < d)
#pragma unroll 8
        for (int r = seq; r < rows; r += 32) s = __fadd_rn(s, partial[(int64_t)r * d + c]);
    part[seq][lane] = s;
    __syncthreads();
    if (seq == 0 && c < d) {
#pragma unroll
        for (int q = 1; q < 32; ++q) s = __fadd_rn(s, part[q][lane]);
        dw[c] = from_f32<W>(s);
    }
}

constexpr int kMaxWidth = 16384;

// Calls f.template operator()<T, VEC, TPR, E>() with the smallest TPR * E that covers d.  16 values a thread: with 8, the
// work of a row that does not depend on its width (waits, reductions, addresses) made the kernels issue-bound.
template <typename T, int VEC, typename F>
void by_width(int d, F&& f) {
    if (d <= 256) f.template operator()<T, VEC, 32, 8>();
    else if (d <= 512) f.template operator()<T, VEC, 32, 16>();
    else if (d <= 1024) f.template operator()<T, VEC, 64, 16>();
    else if (d <= 2048) f.template operator()<T, VEC, 128, 16>();
    else if (d <= 4096) f.template operator()<T, VEC, 256, 16>();
    else if (d <= 8192) f.template operator()<T, VEC, 512, 16>();
    else f.template operator()<T, VEC, 1024, 16>();
}
template <typename F>
void by_type(int32_t type, bool vec, int d, F&& f) {
    if (type == FG_F32) vec ? by_width<float, 4>(d, f) : by_width<float, 1>(d, f);
    else if (type == FG_F16) vec ? by_width<__half, 8>(d, f) : by_width<__half, 1>(d, f);
    else vec ? by_width<__nv_bfloat16, 8>(d, f) : by_width<__nv_bfloat16, 1>(d, f);
}

// Rows that a block walks at a time, and blocks an SM.
constexpr int kNarrow = 128;
int rows_per_block(int d) { return d <= 32 ? 64 : d <= 64 ? 32 : d <= kNarrow ? 16 : d <= 512 ? 8 : d <= 1024 ? 4 : d <= 2048 ? 2 : 1; }
int blocks_per_sm(int d) { return d <= kNarrow ? 6 : d <= 4096 ? 2 : 1; }

// 128-bit accesses need every row to start on a 16-byte boundary.
bool vector_rows(const void* p, int64_t ld, int32_t type) {
    return p == nullptr || (fg::aligned16(p) && (ld * fg::type_size(type)) % 16 == 0);
}

int64_t grid_blocks(int64_t n, int32_t d) {
    const int rows = rows_per_block(d);
    const int64_t want = (n + rows - 1) / rows, most = (int64_t)fg::device_props().sm_count * blocks_per_sm(d);
    return want < most ? want : most;
}

// Three arrays of the widest fp32 rows, the most that a launch asks for.
constexpr int kWidestRows = 3 * (kMaxWidth * 4 + 16);

// Sets the ring: some 180 KB of rows ahead an SM, no more than a block has rows; a very wide row takes what it takes.
template <typename Args, typename K>
void launch_rows(Args& a, int arrays, int size, int threads, int64_t blocks, K kernel, cudaStream_t s) {
    a.slot = (a.d * size + 15) / 16 * 16 + 16;
    const int rows = rows_per_block(a.d), row = rows * arrays * a.slot, room = 180 * 1024 / blocks_per_sm(a.d), most = room / row;
    const int64_t walks = (a.n + blocks * rows - 1) / (blocks * rows);
    a.stages = most < 1 ? 1 : most < kMaxStages ? most : kMaxStages;
    if (a.stages > walks) a.stages = (int32_t)walks;
    const int smem = a.stages * row;
    // one limit for all widths of a kernel: a smaller one, set by another thread before this launch, would have it refused
    static_assert(kWidestRows + 17 * 1024 <= 227 * 1024, "the widest rows and a kernel's own shared memory fit a block");
    if (smem > 30 * 1024) (void)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kWidestRows);
    kernel<<<(unsigned)blocks, threads, smem, s>>>(a);
}
template <typename T, int VEC, int LANES>
void launch_narrow(const NormArgs& a, int64_t blocks, cudaStream_t s) {
    if (a.residual) norm_narrow_kernel<T, VEC, LANES, true><<<(unsigned)blocks, 256, 0, s>>>(a);
    else norm_narrow_kernel<T, VEC, LANES, false><<<(unsigned)blocks, 256, 0, s>>>(a);
}
template <typename T, int VEC, int LANES>
void launch_narrow(const NormGradArgs& a, int64_t blocks, cudaStream_t s) {
    if (a.dh) norm_narrow_grad_kernel<T, VEC, LANES, true><<<(unsigned)blocks, 256, 0, s>>>(a);
    else norm_narrow_grad_kernel<T, VEC, LANES, false><<<(unsigned)blocks, 256, 0, s>>>(a);
}
template <typename T, int VEC, typename Args>
void narrow(const Args& a, int64_t blocks, cudaStream_t s) {
    if (a.d <= 32) launch_narrow<T, VEC, 4>(a, blocks, s);
    else if (a.d <= 64) launch_narrow<T, VEC, 8>(a, blocks, s);
    else launch_narrow<T, VEC, 16>(a, blocks, s);
}
template <typename Args>
void narrow(int32_t type, bool vec, const Args& a, int64_t blocks, cudaStream_t s) {
    if (type == FG_F32) vec ? narrow<float, 4>(a, blocks, s) : narrow<float, 1>(a, blocks, s);
    else if (type == FG_F16) vec ? narrow<__half, 8>(a, blocks, s) : narrow<__half, 1>(a, blocks, s);
    else vec ? narrow<__nv_bfloat16, 8>(a, blocks, s) : narrow<__nv_bfloat16, 1>(a, blocks, s);
}

struct LaunchNorm {
    NormArgs& a;
    cudaStream_t s;
    template <typename T, int VEC, int TPR, int E>
    void operator()() const {
        launch_rows(a, a.residual ? 2 : 1, sizeof(T), TPR < 256 ? 256 : TPR, grid_blocks(a.n, a.d),
                    a.residual ? norm_kernel<T, VEC, TPR, E, true> : norm_kernel<T, VEC, TPR, E, false>, s);
    }
};
struct LaunchNormGrad {
    NormGradArgs& a;
    int64_t blocks;
    cudaStream_t s;
    template <typename T, int VEC, int TPR, int E>
    void operator()() const {
        launch_rows(a, a.dh ? 3 : 2, sizeof(T), TPR < 256 ? 256 : TPR, blocks,
                    a.dh ? norm_grad_kernel<T, VEC, TPR, E, true> : norm_grad_kernel<T, VEC, TPR, E, false>, s);
    }
};

int launch_norm(NormArgs& a, int32_t type, void* stream) {
    const bool vec = a.d % (16 / fg::type_size(type)) == 0 && vector_rows(a.x, a.ldx, type) &&
                     vector_rows(a.residual, a.ldr, type) && vector_rows(a.h, a.d, type) && fg::aligned16(a.y);
    if (a.d <= kNarrow) narrow(type, vec, a, grid_blocks(a.n, a.d), static_cast<cudaStream_t>(stream));
    else by_type(type, vec, a.d, LaunchNorm{a, static_cast<cudaStream_t>(stream)});
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return FG_OK;
}

int check_rows(int64_t n, int32_t d, int32_t type) {
    if (n < 0 || n > INT_MAX || d < 1 || d > kMaxWidth)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "bad sizes n=%lld d=%d (1 <= d <= %d)", (long long)n, d, kMaxWidth);
    if (!fg::float_type(type)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "unknown value type %d", type);
    return FG_OK;
}

}  // namespace

namespace fg {
int norm_stuck(cudaStream_t s, int* out) {
    FG_CUDA_TRY(cudaMemcpyFromSymbolAsync(out, g_stuck, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
    return FG_OK;
}
}  // namespace fg

extern "C" {

int fg_rms_norm(const void* d_x, int64_t ldx, const void* d_residual, int64_t ldr, const void* d_weight, void* d_h, void* d_y,
                float* d_scales, int64_t n, int32_t d, float eps, int32_t type, int32_t weight_type, int32_t out_type,
                void* stream) {
    if (int rc = check_rows(n, d, type)) return rc;
    if (d_weight && weight_type != type && weight_type != FG_F32)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "the weight is of the rows' type or fp32");
    if (out_type != type && out_type != FG_E4M3) return fg::fail(FG_ERR_INVALID_ARGUMENT, "the output is of the rows' type or e4m3");
    if (!(eps >= 0.0f)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "eps must be >= 0");
    if (ldx == 0) ldx = d;
    if (ldr == 0) ldr = d;
    if (ldx < d || ldr < d) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= d=%d", d);
    if (n == 0) return FG_OK;
    if (!d_x || !d_y || (d_residual && !d_h) || (out_type == FG_E4M3 && !d_scales))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    NormArgs a{d_x, d_residual, d_weight, d_h, d_y, d_scales, ldx, ldr, n, d, 0, 0, eps, weight_type == FG_F32, true, out_type == FG_E4M3};
    return launch_norm(a, type, stream);
}

int fg_quantize_rows(const void* d_x, int64_t ldx, void* d_y, float* d_scales, int64_t n, int32_t d, int32_t type, void* stream) {
    if (int rc = check_rows(n, d, type)) return rc;
    if (ldx == 0) ldx = d;
    if (ldx < d) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= d=%d", d);
    if (n == 0) return FG_OK;
    if (!d_x || !d_y || !d_scales) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    NormArgs a{d_x, nullptr, nullptr, nullptr, d_y, d_scales, ldx, 0, n, d, 0, 0, 0.0f, true, false, true};
    return launch_norm(a, type, stream);
}

int64_t fg_rms_norm_backward_blocks(int64_t n, int32_t d) {
    return n < 1 || d < 1 ? 0 : grid_blocks(n, d);
}

int fg_rms_norm_backward(const void* d_h, int64_t ldh, const void* d_weight, const void* d_dy, int64_t lddy, const void* d_dh,
                         int64_t lddh, void* d_dx, void* d_dweight, float* d_partial, int64_t blocks, int64_t n, int32_t d,
                         float eps, int32_t type, int32_t weight_type, void* stream) {
    if (int rc = check_rows(n, d, type)) return rc;
    if (d_weight && weight_type != type && weight_type != FG_F32)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "the weight is of the rows' type or fp32");
    if (ldh == 0) ldh = d;
    if (lddy == 0) lddy = d;
    if (lddh == 0) lddh = d;
    if (ldh < d || lddy < d || lddh < d) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= d=%d", d);
    if (n == 0) {
        if (d_dweight)
            FG_CUDA_TRY(cudaMemsetAsync(d_dweight, 0, (size_t)d * fg::type_size(weight_type), static_cast<cudaStream_t>(stream)));
        return FG_OK;
    }
    if (!d_h || !d_dy || !d_dx || (d_dweight && !d_partial)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    if (blocks < 1 || blocks > INT_MAX) return fg::fail(FG_ERR_INVALID_ARGUMENT, "blocks must come from fg_rms_norm_backward_blocks");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    NormGradArgs a{d_h, d_weight, d_dy, d_dh, d_dx, d_dweight ? d_partial : nullptr, ldh, lddy, lddh, n, d, 0, 0, eps, weight_type == FG_F32};
    const bool vec = d % (16 / fg::type_size(type)) == 0 && vector_rows(d_h, ldh, type) && vector_rows(d_dy, lddy, type) &&
                     vector_rows(d_dh, lddh, type) && fg::aligned16(d_dx);
    if (d <= kNarrow) narrow(type, vec, a, blocks, s);
    else by_type(type, vec, d, LaunchNormGrad{a, blocks, s});
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    if (d_dweight) {
        const unsigned grid = (unsigned)((d + 31) / 32);
        if (weight_type == FG_F32) weight_grad_kernel<float><<<grid, 1024, 0, s>>>(d_partial, (int)blocks, d, static_cast<float*>(d_dweight));
        else if (weight_type == FG_F16) weight_grad_kernel<__half><<<grid, 1024, 0, s>>>(d_partial, (int)blocks, d, static_cast<__half*>(d_dweight));
        else weight_grad_kernel<__nv_bfloat16><<<grid, 1024, 0, s>>>(d_partial, (int)blocks, d, static_cast<__nv_bfloat16*>(d_dweight));
        FG_CUDA_TRY(cudaGetLastError());
        fg::count_launches(1);
    }
    return FG_OK;
}

}  // extern "C"
