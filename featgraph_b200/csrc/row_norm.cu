// Root-mean-square norm of rows with the residual's addition, its 8-bit form, and its gradient.
//
//   h = round(x + residual)      y = h * r * w,   r = 1 / sqrt(mean(h^2) + eps)
//   8 bits: s = max|h r w| / 448 (1 for a row of zeros),  q = e4m3(h r w / s)
//   dx = dresidual = dh + r g - h r^3 / d * sum(g h),  g = dy w;      dw = sum over rows of dy h r
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

// Sum / maximum over the TPR threads of a row; `slot` picks a buffer so that two reductions in a row need no
// barrier between them.
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* buffer) {
    v = MAX ? fg::warp_max(v) : fg::warp_sum(v);
    if (TPR == 32) return v;
    constexpr int kWarps = TPR / 32;
    const int warp = threadIdx.x >> 5, first = (threadIdx.x / TPR) * kWarps;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buffer[warp] = v;
    __syncthreads();
    v = buffer[first];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) {
        const float w = buffer[first + i];
        if (MAX) v = (w > v || w != w) ? w : v;
        else v = __fadd_rn(v, w);
    }
    return v;
}

__device__ __forceinline__ float weight_at(const void* w, bool f32, int i, float) {
    return w == nullptr ? 1.0f : static_cast<const float*>(w)[i];
}
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, bool f32, int i, T) {
    if (w == nullptr) return 1.0f;
    return f32 ? static_cast<const float*>(w)[i] : to_f32<T>(static_cast<const T*>(w)[i]);
}

struct NormArgs {
    const void *x, *residual, *weight;
    void *h, *y;
    float* scales;
    int64_t ldx, ldr, n;
    int32_t d;
    float eps;
    bool weight_f32, normalize, e4m3;
};

template <typename T, int VEC, int TPR, int E>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) norm_kernel(const NormArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR, NV = E / VEC;
    __shared__ float buffer[kThreads / 32];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
    const bool live = row < a.n;  // a dead row still takes part in the barriers
    const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.ldx;
    float v[E];
    Pack<T, VEC> px[NV];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int i = (c * TPR + t) * VEC;
        if (live && i < a.d) px[c] = load_pack<T, VEC>(x + i);
    }
    if (a.residual != nullptr) {
        const T* res = static_cast<const T*>(a.residual) + (live ? row : 0) * a.ldr;
        T* h = static_cast<T*>(a.h) + row * a.d;
        Pack<T, VEC> pr[NV];
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (live && i < a.d) pr[c] = load_pack<T, VEC>(res + i);
        }
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (live && i < a.d) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    px[c].v[j] = from_f32<T>(__fadd_rn(to_f32<T>(px[c].v[j]), to_f32<T>(pr[c].v[j])));
                store_pack<T, VEC>(h + i, px[c]);
            }
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int i = (c * TPR + t) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float u = (live && i < a.d) ? to_f32<T>(px[c].v[j]) : 0.0f;
            v[c * VEC + j] = u;
            ss = __fmaf_rn(u, u, ss);
        }
    }
    if (a.normalize) {
        ss = row_reduce<TPR, false>(ss, buffer);
        const float r = __frsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)a.d), a.eps));
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (i < a.d) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    v[c * VEC + j] = __fmul_rn(__fmul_rn(v[c * VEC + j], r), weight_at(a.weight, a.weight_f32, i + j, T()));
            }
        }
    }
    if (!a.e4m3) {
        T* y = static_cast<T*>(a.y) + row * a.d;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (live && i < a.d) {
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) o.v[j] = from_f32<T>(v[c * VEC + j]);
                store_pack<T, VEC>(y + i, o);
            }
        }
        return;
    }
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float u = fabsf(v[e]);
        most = (u > most || u != u) ? u : most;
    }
    most = row_reduce<TPR, true>(most, buffer);
    const float scale = most == 0.0f ? 1.0f : __fdiv_rn(most, (float)kE4M3Max);
    uint8_t* q = static_cast<uint8_t*>(a.y) + row * a.d;
    if (live && t == 0) a.scales[row] = scale;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int i = (c * TPR + t) * VEC;
        if (live && i < a.d) {
            Pack<uint8_t, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                o.v[j] = __nv_cvt_float_to_fp8(__fdiv_rn(v[c * VEC + j], scale), __NV_SATFINITE, __NV_E4M3);
            store_pack<uint8_t, VEC>(q + i, o);
        }
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

// The TPR threads of a row walk the rows with a ring of `stages` rows in shared memory ahead of them, filled by bulk copies:
// what is in flight does not take registers (with the next row in registers 16 warps an SM were left, and 32768 x
// 4096 bf16 with dh took 253 us), and a row that starts off the 16-byte grid is copied from the grid point before it
// on, up to 15 bytes more on either side in the 16-byte units that hold the row's first and last values.
// A stage is free again as soon as its values are in registers, which the barrier of the sums shows.
template <typename T, int VEC, int TPR, int E, bool DH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, TPR <= 256 ? 2 : 1) norm_grad_kernel(const NormGradArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR, NV = E / VEC;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ uint64_t full[kRows][kMaxStages];
    __shared__ float2 buffer[2][kThreads / 32];
    __shared__ float across[kRows > 1 ? kRows * TPR * E : 1];
    __shared__ int stop;
    constexpr int arrays = DH ? 3 : 2;
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float over_d = __fdiv_rn(1.0f, (float)a.d);
    const int64_t first = (int64_t)blockIdx.x * kRows + sub, step = (int64_t)gridDim.x * kRows;
    const uint8_t* mine = ring + sub * a.stages * arrays * a.slot;
    const uint32_t base = fg::smem_address(mine);
    if (t == 0)
        for (int s = 0; s < a.stages; ++s) fg::barrier_init(fg::smem_address(&full[sub][s]), 1);
    if (threadIdx.x == 0) stop = 0;
    fg::barrier_init_fence();
    __syncthreads();
    auto address = [&](int array, int64_t row) {
        return array == 0   ? reinterpret_cast<uint64_t>(static_cast<const T*>(a.h) + row * a.ldh)
               : array == 1 ? reinterpret_cast<uint64_t>(static_cast<const T*>(a.dy) + row * a.lddy)
                            : reinterpret_cast<uint64_t>(static_cast<const T*>(a.dh) + row * a.lddh);
    };
    auto request = [&](int s, int64_t row) {  // one thread of the row
        const uint32_t bar = fg::smem_address(&full[sub][s]);
        uint32_t bytes = 0;
        for (int q = 0; q < arrays; ++q) {
            const uint64_t from = address(q, row), lo = from & ~15ull;
            bytes += (uint32_t)(((from + (uint64_t)a.d * sizeof(T) + 15) & ~15ull) - lo);
        }
        fg::barrier_expect(bar, bytes);
        for (int q = 0; q < arrays; ++q) {
            const uint64_t from = address(q, row), lo = from & ~15ull;
            fg::bulk_load(base + (s * arrays + q) * a.slot, lo, (uint32_t)(((from + (uint64_t)a.d * sizeof(T) + 15) & ~15ull) - lo), bar);
        }
    };
    if (t == 0)
        for (int s = 0; s < a.stages; ++s)
            if (first + s * step < a.n) request(s, first + s * step);
    float acc[E], weight[E];  // the thread's columns: the same for all rows
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int i = (c * TPR + t) * VEC + j;
            acc[c * VEC + j] = 0.0f;
            weight[c * VEC + j] = i < a.d ? weight_at(a.weight, a.weight_f32, i, T()) : 0.0f;
        }
    int s = 0, parity = 0, turn = 0;
    for (int64_t row = first; row < a.n; row += step, turn ^= 1) {
        fg::barrier_wait(fg::smem_address(&full[sub][s]), parity, &stop);  // without the copy: wrong values, and the flag
        Pack<T, VEC> h[NV], g[NV], d[NV];
        // where a row starts in its 16-byte unit; rows that are read in vectors start on the grid
        const uint8_t* stage = mine + s * arrays * a.slot;
        const T* hs = reinterpret_cast<const T*>(stage + (VEC == 1 ? (uint32_t)address(0, row) & 15 : 0));
        const T* gs = reinterpret_cast<const T*>(stage + a.slot + (VEC == 1 ? (uint32_t)address(1, row) & 15 : 0));
        const T* ds = reinterpret_cast<const T*>(stage + 2 * a.slot + (VEC == 1 && DH ? (uint32_t)address(2, row) & 15 : 0));
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
        if (t == 0 && row + a.stages * step < a.n) request(s, row + a.stages * step);
        if (++s == a.stages) s = 0, parity ^= 1;
        const float r = __frsqrt_rn(__fmaf_rn(ss, over_d, a.eps));
        const float along = __fmul_rn(__fmul_rn(r, r), __fmul_rn(r, __fmul_rn(sg, over_d)));
        T* dx = static_cast<T*>(a.dx) + row * a.d;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = (c * TPR + t) * VEC;
            if (i < a.d) {
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float u = to_f32<T>(h[c].v[j]), dyj = to_f32<T>(g[c].v[j]);
                    const float v = __fmul_rn(dyj, weight[c * VEC + j]);
                    float w = __fmaf_rn(-u, along, __fmul_rn(r, v));
                    if (DH) w = __fadd_rn(w, to_f32<T>(d[c].v[j]));
                    o.v[j] = from_f32<T>(w);
                    acc[c * VEC + j] = __fmaf_rn(dyj, __fmul_rn(u, r), acc[c * VEC + j]);
                }
                store_pack<T, VEC>(dx + i, o);
            }
        }
    }
    if (stop) {  // a wait ran out: the copies that are left end before the block does
        if (t == 0)
            for (int q = 0; q < a.stages; ++q) {
                fg::barrier_wait(fg::smem_address(&full[sub][q]), 0, &stop, true);
                fg::barrier_wait(fg::smem_address(&full[sub][q]), 1, &stop, true);
            }
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

// Calls f.template operator()<T, VEC, TPR, E>() with the smallest TPR * E that covers d.  Single values straight from memory
// cost an address and a register each, so there (SLIM) a thread holds 8 values rather than 16.
template <typename T, int VEC, bool SLIM, typename F>
void by_width(int d, F&& f) {
    if constexpr (SLIM) {
        if (d <= 256) f.template operator()<T, VEC, 32, 8>();
        else if (d <= 512) f.template operator()<T, VEC, 64, 8>();
        else if (d <= 1024) f.template operator()<T, VEC, 128, 8>();
        else if (d <= 2048) f.template operator()<T, VEC, 256, 8>();
        else if (d <= 4096) f.template operator()<T, VEC, 512, 8>();
        else if (d <= 8192) f.template operator()<T, VEC, 1024, 8>();
        else f.template operator()<T, VEC, 1024, 16>();
    } else {
        if (d <= 256) f.template operator()<T, VEC, 32, 8>();
        else if (d <= 512) f.template operator()<T, VEC, 32, 16>();
        else if (d <= 1024) f.template operator()<T, VEC, 64, 16>();
        else if (d <= 2048) f.template operator()<T, VEC, 128, 16>();
        else if (d <= 4096) f.template operator()<T, VEC, 256, 16>();
        else if (d <= 8192) f.template operator()<T, VEC, 512, 16>();
        else f.template operator()<T, VEC, 1024, 16>();
    }
}
template <bool SLIM, typename F>
void by_type(int32_t type, bool vec, int d, F&& f) {
    if (type == FG_F32) vec ? by_width<float, 4, false>(d, f) : by_width<float, 1, SLIM>(d, f);
    else if (type == FG_F16) vec ? by_width<__half, 8, false>(d, f) : by_width<__half, 1, SLIM>(d, f);
    else vec ? by_width<__nv_bfloat16, 8, false>(d, f) : by_width<__nv_bfloat16, 1, SLIM>(d, f);
}

// Rows that a block of the backward pass walks at a time, and blocks an SM.
int rows_per_block(int d) { return d <= 512 ? 8 : d <= 1024 ? 4 : d <= 2048 ? 2 : 1; }
int blocks_per_sm(int d) { return d <= 4096 ? 2 : 1; }

// 128-bit accesses need every row to start on a 16-byte boundary.
bool vector_rows(const void* p, int64_t ld, int32_t type) {
    return p == nullptr || (fg::aligned16(p) && (ld * fg::type_size(type)) % 16 == 0);
}

struct LaunchNorm {
    const NormArgs& a;
    cudaStream_t s;
    template <typename T, int VEC, int TPR, int E>
    void operator()() const {
        constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR;
        norm_kernel<T, VEC, TPR, E><<<(unsigned)((a.n + kRows - 1) / kRows), kThreads, 0, s>>>(a);
    }
};
struct LaunchNormGrad {
    NormGradArgs& a;
    unsigned blocks;
    cudaStream_t s;
    template <typename T, int VEC, int TPR, int E>
    void operator()() const {
        constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR;
        // rows ahead: some 180 KB of them an SM; a very wide row takes what it takes
        a.slot = (a.d * (int)sizeof(T) + 15) / 16 * 16 + 16;
        const int row = kRows * (a.dh != nullptr ? 3 : 2) * a.slot, room = 180 * 1024 / blocks_per_sm(a.d), most = room / row;
        a.stages = most < 1 ? 1 : most < kMaxStages ? most : kMaxStages;
        const int smem = a.stages * row;
        const auto kernel = a.dh ? norm_grad_kernel<T, VEC, TPR, E, true> : norm_grad_kernel<T, VEC, TPR, E, false>;
        if (smem > 30 * 1024) (void)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem < room ? room : smem);
        kernel<<<blocks, kThreads, smem, s>>>(a);
    }
};

int launch_norm(NormArgs& a, int32_t type, void* stream) {
    const bool vec = a.d % (16 / fg::type_size(type)) == 0 && vector_rows(a.x, a.ldx, type) &&
                     vector_rows(a.residual, a.ldr, type) && vector_rows(a.h, a.d, type) && fg::aligned16(a.y);
    by_type<true>(type, vec, a.d, LaunchNorm{a, static_cast<cudaStream_t>(stream)});
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
    NormArgs a{d_x, d_residual, d_weight, d_h, d_y, d_scales, ldx, ldr, n, d, eps, weight_type == FG_F32, true, out_type == FG_E4M3};
    return launch_norm(a, type, stream);
}

int fg_quantize_rows(const void* d_x, int64_t ldx, void* d_y, float* d_scales, int64_t n, int32_t d, int32_t type, void* stream) {
    if (int rc = check_rows(n, d, type)) return rc;
    if (ldx == 0) ldx = d;
    if (ldx < d) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= d=%d", d);
    if (n == 0) return FG_OK;
    if (!d_x || !d_y || !d_scales) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    NormArgs a{d_x, nullptr, nullptr, nullptr, d_y, d_scales, ldx, 0, n, d, 0.0f, true, false, true};
    return launch_norm(a, type, stream);
}

int64_t fg_rms_norm_backward_blocks(int64_t n, int32_t d) {
    if (n < 1 || d < 1) return 0;
    const int rows = rows_per_block(d);
    const int64_t want = (n + rows - 1) / rows, most = (int64_t)fg::device_props().sm_count * blocks_per_sm(d);
    return want < most ? want : most;
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
    by_type<false>(type, vec, d, LaunchNormGrad{a, (unsigned)blocks, s});
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
