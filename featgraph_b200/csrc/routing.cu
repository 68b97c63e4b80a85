// Routing: the choice of k experts for each row, the lists by expert, and the weighted sum back.
//
// A choice of k of G groups for each of n rows is a bipartite graph with n * k edges ("entries", entry = row * k + j).
// fg_group_rows turns it from row order into CSR by group: a stable counting sort, so the slots of a group hold its
// entries in ascending order and the lists are the same on every run.
//
//   offsets[g] .. offsets[g + 1]  the slots of group g;     order[slot] = entry;     position[entry] = slot
//   an entry whose key is outside [0, G) is in no group: position -1, and the slots from offsets[G] on hold -1
#include <climits>

#include "rows.cuh"

namespace {

using fg::from_f32;
using fg::load_pack;
using fg::Pack;
using fg::store_pack;
using fg::to_f32;

constexpr int kMaxExperts = 1024, kMaxChoices = 32, kMaxGroups = 1024;

// ---- choice ----

// Unsigned keys in the order of the floats, 0 for what can never be chosen (-inf, NaN); +0 and -0 are equal.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (!(v > -INFINITY)) return 0u;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ float sigmoid(float v) {
    const float e = expf(-fabsf(v)), s = __fdiv_rn(1.0f, __fadd_rn(1.0f, e));
    return v >= 0.0f ? s : __fmul_rn(e, s);
}

struct RouteArgs {
    const void* logits;
    int64_t ld, n;
    int32_t experts, k;
    bool sigmoid, normalize;
    float* weights;
    int32_t* chosen;
};

// A warp owns a row; lane l holds experts l, l + 32, ...  Each of the k rounds is one warp-wide maximum of the lanes'
// largest keys and a vote; where several lanes hold it (equal logits), a warp-wide minimum of the indices breaks
// the tie, so it goes to the lowest.  The winner moves to its next largest: up to 4 keys a lane are sorted at the start
// (adjacent swaps of strictly smaller ones, so equal keys stay in order), more are searched again.  Lane j keeps the
// j-th choice.  Bound: instructions, some 40 a row and round; the n * E logits are read once (65,536 x 128: 33.6 MB, 5 us).
template <typename T, int NE>
__device__ __forceinline__ void route_row(const RouteArgs& a, int64_t row) {
    constexpr bool kSorted = NE <= 4;
    const int lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    uint32_t key[NE], index[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = i * 32 + lane;
        key[i] = e < a.experts ? order_key(to_f32<T>(x[e])) : 0u;
        index[i] = e;
    }
    uint32_t best = key[0], slot = 0;
    auto search = [&]() {  // the lane's largest key, and which of its NE it is (the lowest)
        best = key[0], slot = 0;
#pragma unroll
        for (int i = 1; i < NE; ++i)
            if (key[i] > best) best = key[i], slot = i;
    };
    if (kSorted) {
#pragma unroll
        for (int pass = 0; pass < NE; ++pass)
#pragma unroll
            for (int i = pass & 1; i + 1 < NE; i += 2)
                if (key[i + 1] > key[i]) {
                    const uint32_t k0 = key[i], i0 = index[i];
                    key[i] = key[i + 1], index[i] = index[i + 1];
                    key[i + 1] = k0, index[i + 1] = i0;
                }
        best = key[0];
    } else {
        search();
    }
    float all = 0.0f, top = 0.0f;
    if (!a.sigmoid && !a.normalize) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, best);
        top = m ? key_value(m) : 0.0f;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (key[i]) all = __fadd_rn(all, expf(__fsub_rn(key_value(key[i]), top)));
        all = fg::warp_sum(all);
    }
    uint32_t mine = 0, at_mine = 0;
    for (int j = 0; j < a.k; ++j) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, best);
        if (m == 0) break;
        const uint32_t holders = __ballot_sync(0xffffffffu, best == m);
        uint32_t at = kSorted ? index[0] : slot * 32 + lane;
        if (holders & (holders - 1)) at = __reduce_min_sync(0xffffffffu, best == m ? at : 0xffffffffu);
        else at = __shfl_sync(0xffffffffu, at, __ffs(holders) - 1);
        if (lane == j) mine = m, at_mine = at;
        if ((at & 31) == lane) {
            if (kSorted) {
#pragma unroll
                for (int i = 0; i + 1 < NE; ++i) key[i] = key[i + 1], index[i] = index[i + 1];
                key[NE - 1] = 0;
                best = key[0];
            } else {
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if (i == (int)(at >> 5)) key[i] = 0;
                search();
            }
        }
    }
    float score = 0.0f;
    if (!a.sigmoid && a.normalize) {
        const uint32_t m = __shfl_sync(0xffffffffu, mine, 0);
        top = m ? key_value(m) : 0.0f;
    }
    if (mine) score = a.sigmoid ? sigmoid(key_value(mine)) : expf(__fsub_rn(key_value(mine), top));
    if (a.normalize) all = fg::warp_sum(score);
    if (a.normalize || !a.sigmoid) score = all > 0.0f || all != all ? __fdiv_rn(score, all) : 0.0f;
    if (lane < a.k) {
        a.weights[row * a.k + lane] = score;
        a.chosen[row * a.k + lane] = mine ? (int)at_mine : -1;
    }
}

template <typename T, int NE>
__global__ void __launch_bounds__(256) route_kernel(const RouteArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row < a.n) route_row<T, NE>(a, row);
}

struct RouteGradArgs {
    const void* logits;
    int64_t ld, n;
    int32_t experts, k;
    bool sigmoid, normalize;
    const float *weights, *dweights;
    const int32_t* chosen;
    void* dlogits;
};

// softmax, normalised:   dx_i = w_i (g_i - sum g w) for the chosen, 0 elsewhere (the other logits cancel out)
// softmax over all:      dx_i = p_i ([i chosen] g_i - sum g w)
// sigmoid, normalised:   dx_i = s_i (1 - s_i) (g_i - sum g w) / sum s;   not normalised: dx_i = s_i (1 - s_i) g_i
// A warp owns a row: it writes what the row gets without the choice (zeros, or -p sum g w), then lane j writes choice j's
// value over it - for a chosen logit of the softmax over all, p is the weight itself.  Bound: the dense rows' bytes.
template <typename T, int NE>
__global__ void __launch_bounds__(256) route_grad_kernel(const RouteGradArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= a.n) return;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    T* dx = static_cast<T*>(a.dlogits) + row * a.experts;
    int mine = -1;
    float w = 0.0f, g = 0.0f;
    if (lane < a.k) {
        mine = a.chosen[row * a.k + lane];
        w = a.weights[row * a.k + lane];
        g = a.dweights[row * a.k + lane];
        if ((unsigned)mine >= (unsigned)a.experts) mine = -1;
        if (mine < 0) g = 0.0f;
    }
    const float dot = fg::warp_sum(__fmul_rn(g, w));
    if (a.sigmoid || a.normalize) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (i * 32 + lane < a.experts) dx[i * 32 + lane] = from_f32<T>(0.0f);
    } else {
        uint32_t key[NE], m = 0;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = i * 32 + lane;
            key[i] = e < a.experts ? order_key(to_f32<T>(x[e])) : 0u;
            m = max(m, key[i]);
        }
        m = __reduce_max_sync(0xffffffffu, m);
        const float top = m ? key_value(m) : 0.0f;
        float all = 0.0f, p[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            p[i] = key[i] ? expf(__fsub_rn(key_value(key[i]), top)) : 0.0f;
            all = __fadd_rn(all, p[i]);
        }
        all = fg::warp_sum(all);
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (i * 32 + lane < a.experts) dx[i * 32 + lane] = from_f32<T>(m ? -__fmul_rn(__fdiv_rn(p[i], all), dot) : 0.0f);
    }
    __syncwarp();  // the stores above come before those below
    float s = 0.0f, slope = 0.0f;
    if (a.sigmoid) {
        if (mine >= 0) {
            const float v = to_f32<T>(x[mine]);
            s = sigmoid(v);
            slope = __fmul_rn(s, sigmoid(-v));
        }
        if (a.normalize) {
            const float total = fg::warp_sum(s);
            slope = total > 0.0f ? __fdiv_rn(__fmul_rn(slope, __fsub_rn(g, dot)), total) : 0.0f;
        } else {
            slope = __fmul_rn(slope, g);
        }
    } else {
        slope = __fmul_rn(w, __fsub_rn(g, dot));
    }
    if (mine >= 0) dx[mine] = from_f32<T>(slope);
}

// ---- lists ----

// Entries are cut into chunks, a block each; in a chunk every warp owns a run of consecutive entries.  Pass 1 counts
// keys per chunk, pass 2 sums a group's counts over the chunks before (a warp a group), pass 3 scans the totals, counts per warp,
// and walks each run 32 entries at a time: an entry's rank among its warp's equal keys is the number of lower lanes
// with the same key (match_any), so the order is stable.  Key `groups` stands for "in no group".  When one chunk
// holds all entries, pass 3 alone does everything.
struct GroupArgs {
    const int32_t* keys;
    int64_t m;
    int32_t groups, chunk, chunks;
    int32_t *counts;  // [groups + 1][chunks]: counts, then the entries of the group in earlier chunks; then a total each
    int32_t *offsets, *order, *position;
};

__device__ __forceinline__ int key_of(const GroupArgs& a, int64_t e) {
    const int v = a.keys[e];
    return (unsigned)v < (unsigned)a.groups ? v : a.groups;
}

__global__ void __launch_bounds__(256) group_count_kernel(const GroupArgs a) {
    extern __shared__ int hist[];
    for (int g = threadIdx.x; g <= a.groups; g += blockDim.x) hist[g] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * a.chunk, last = min(first + a.chunk, a.m);
    for (int64_t e = first + threadIdx.x; e < last; e += blockDim.x) atomicAdd(&hist[key_of(a, e)], 1);  // whole numbers: any order
    __syncthreads();
    for (int g = threadIdx.x; g <= a.groups; g += blockDim.x) a.counts[(int64_t)g * a.chunks + blockIdx.x] = hist[g];
}

// Exclusive scan of v over the block; total by reference.
__device__ int block_scan(int v, int& total) {
    __shared__ int sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += w;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    if (warp == 0) {
        int w = lane < warps ? sums[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        sums[lane] = w;
    }
    __syncthreads();
    total = sums[31];
    return s - v + (warp ? sums[warp - 1] : 0);
}

__global__ void __launch_bounds__(128) group_scan_kernel(const GroupArgs a) {
    const int lane = threadIdx.x & 31, bins = a.groups + 1, each = (a.chunks + 31) / 32, g = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (g >= bins) return;
    int32_t* row = a.counts + (int64_t)g * a.chunks;
    const int from = min(lane * each, a.chunks), to = min(from + each, a.chunks);
    int own = 0;
#pragma unroll 8
    for (int c = from; c < to; ++c) own += row[c];
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31) a.counts[(int64_t)bins * a.chunks + g] = sum;
    int before = sum - own;
#pragma unroll 8
    for (int c = from; c < to; ++c) {
        const int n = row[c];
        row[c] = before;
        before += n;
    }
}

template <bool SINGLE>
__device__ __forceinline__ void place_entries(const GroupArgs& a, int* cell) {  // cell: [warps][groups + 1]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = a.groups + 1, threads = blockDim.x >> 5;
    const int64_t begin = (int64_t)blockIdx.x * a.chunk, end = min(begin + a.chunk, a.m);
    const int run = ((a.chunk + threads - 1) / threads + 31) / 32 * 32;
    const int warps = (a.chunk + run - 1) / run;  // that have entries
    for (int i = threadIdx.x; i < warps * bins; i += blockDim.x) cell[i] = 0;
    __syncthreads();
    const int64_t first = min(begin + (int64_t)warp * run, end), last = min(first + run, end);
    int* mine = cell + warp * bins;
    for (int64_t e = first + lane; e < last; e += 32) atomicAdd(&mine[key_of(a, e)], 1);
    __syncthreads();
    int carry = 0;
    for (int base = 0; base < bins; base += blockDim.x) {
        const int g = base + threadIdx.x;
        int sum = 0, total;  // the group's entries: counted here, or in the passes before
        if (SINGLE && g < bins)
            for (int w = 0; w < warps; ++w) sum += cell[w * bins + g];
        if (!SINGLE && g < bins) sum = a.counts[(int64_t)bins * a.chunks + g];
        int start = carry + block_scan(sum, total);
        carry += total;
        if (g < bins && blockIdx.x == 0) a.offsets[g] = start;  // group `groups` starts where the last group ends
        if (!SINGLE && g < bins) start += a.counts[(int64_t)g * a.chunks + blockIdx.x];
        if (g < bins)
            for (int w = 0; w < warps; ++w) {
                const int c = cell[w * bins + g];
                cell[w * bins + g] = start;
                start += c;
            }
    }
    __syncthreads();
    for (int64_t base = first; base < last; base += 32) {
        const int64_t e = base + lane;
        const bool live = e < last;
        const unsigned active = __ballot_sync(0xffffffffu, live);
        if (live) {
            const int key = key_of(a, e);
            const unsigned same = __match_any_sync(active, key);
            const int slot = mine[key] + __popc(same & ((1u << lane) - 1u));
            __syncwarp(active);
            if ((same >> lane) == 1u) mine[key] = slot + 1;  // the highest lane of a key moves its cell on
            __syncwarp(active);
            a.position[e] = key < a.groups ? slot : -1;
            a.order[slot] = key < a.groups ? (int32_t)e : -1;
        }
    }
}

template <bool SINGLE>
__global__ void __launch_bounds__(1024) group_place_kernel(const GroupArgs a) {
    extern __shared__ int cell[];
    place_entries<SINGLE>(a, cell);
}

// Choice and lists of a few rows in one launch: one block chooses for all rows, a warp a row, and then lists them.
template <typename T, int NE>
__global__ void __launch_bounds__(1024) route_lists_kernel(const RouteArgs a, const GroupArgs g) {
    extern __shared__ int cell[];
    for (int64_t row = threadIdx.x >> 5; row < a.n; row += blockDim.x >> 5) route_row<T, NE>(a, row);
    __syncthreads();  // the choices are in global memory, written by this block
    place_entries<true>(g, cell);
}

// Calls f.template operator()<T, NE>() with the smallest NE that covers the experts.
template <typename T, typename F>
void by_experts(int experts, F&& f) {
    if (experts <= 32) f.template operator()<T, 1>();
    else if (experts <= 64) f.template operator()<T, 2>();
    else if (experts <= 128) f.template operator()<T, 4>();
    else if (experts <= 256) f.template operator()<T, 8>();
    else if (experts <= 512) f.template operator()<T, 16>();
    else f.template operator()<T, 32>();
}
template <typename F>
void by_logit_type(int32_t type, int experts, F&& f) {
    if (type == FG_F32) by_experts<float>(experts, f);
    else if (type == FG_F16) by_experts<__half>(experts, f);
    else by_experts<__nv_bfloat16>(experts, f);
}
struct LaunchRoute {
    const RouteArgs& a;
    cudaStream_t s;
    template <typename T, int NE>
    void operator()() const { route_kernel<T, NE><<<(unsigned)((a.n + 7) / 8), 256, 0, s>>>(a); }
};
struct LaunchRouteLists {
    const RouteArgs& a;
    const GroupArgs& g;
    cudaStream_t s;
    template <typename T, int NE>
    void operator()() const {
        const int warps = a.n <= 4 ? 4 : a.n <= 8 ? 8 : a.n <= 16 ? 16 : 32;
        const size_t smem = (size_t)warps * (g.groups + 1) * 4;
        if (smem > 40 * 1024) (void)cudaFuncSetAttribute(route_lists_kernel<T, NE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 140 * 1024);
        route_lists_kernel<T, NE><<<1, warps * 32, smem, s>>>(a, g);
    }
};
struct LaunchRouteGrad {
    const RouteGradArgs& a;
    cudaStream_t s;
    template <typename T, int NE>
    void operator()() const { route_grad_kernel<T, NE><<<(unsigned)((a.n + 7) / 8), 256, 0, s>>>(a); }
};

// ---- weighted sum back ----

struct CombineArgs {
    const void *y, *dout;
    const float* weights;
    const int32_t *position, *offsets;
    void *out, *dy;
    float* dweights;
    int64_t n, m, ldy, ldd;
    int32_t k, d, groups;
};

// out[t] = sum over j of weights[t, j] y[position[t, j]], in ascending j, in 32 bits.  A thread owns VEC columns of a
// row; the k slices of a row are independent loads.  Bound: device memory (M rows read, n written): 32768 rows of 2048 bf16,
// k = 4, in 119 us (5.6 TB/s).  Four slices held at a time cost a third of the warps and 148 us.  O: the output's type.
template <typename T, int VEC, typename O = T>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a) {
    const int per_row = (a.d + VEC - 1) / VEC;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = i / per_row;
    if (t >= a.n) return;
    const int c = (int)(i - t * per_row) * VEC;
    float acc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
#pragma unroll 4
    for (int j = 0; j < a.k; ++j) {
        const int p = a.position[t * a.k + j];
        if ((unsigned)p >= (unsigned)a.m) continue;
        const float w = a.weights ? a.weights[t * a.k + j] : 1.0f;
        const Pack<T, VEC> r = load_pack<T, VEC>(static_cast<const T*>(a.y) + (int64_t)p * a.ldy + c);
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = __fmaf_rn(w, to_f32<T>(r.v[v]), acc[v]);
    }
    Pack<O, VEC> o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) o.v[v] = from_f32<O>(acc[v]);
    store_pack<O, VEC>(static_cast<O*>(a.out) + t * a.d + c, o);
}

// dy[position[t, j]] = weights[t, j] dout[t];   dweights[t, j] = dot(dout[t], y[position[t, j]]).
// A warp owns a row t, so that dout[t] is read from memory once for all k; slots that belong to no entry are zeroed.
// Bound: device memory, 1.2 GB for 32768 rows of 2048 bf16, k = 4, in 223 us (5.4 TB/s).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) combine_grad_kernel(const CombineArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t < a.n) {
        const T* g = static_cast<const T*>(a.dout) + t * a.ldd;
        for (int j = 0; j < a.k; ++j) {
            const int p = a.position[t * a.k + j];
            const bool in = (unsigned)p < (unsigned)a.m;
            const float w = a.weights ? a.weights[t * a.k + j] : 1.0f;
            float dot = 0.0f;
            if (in)
#pragma unroll 4
                for (int c = lane * VEC; c < a.d; c += 32 * VEC) {
                    const Pack<T, VEC> pg = load_pack<T, VEC>(g + c);
                    if (a.dy) {
                        Pack<T, VEC> o;
#pragma unroll
                        for (int v = 0; v < VEC; ++v) o.v[v] = from_f32<T>(__fmul_rn(w, to_f32<T>(pg.v[v])));
                        store_pack<T, VEC>(static_cast<T*>(a.dy) + (int64_t)p * a.d + c, o);
                    }
                    if (a.dweights) {
                        const Pack<T, VEC> py = load_pack<T, VEC>(static_cast<const T*>(a.y) + (int64_t)p * a.ldy + c);
#pragma unroll
                        for (int v = 0; v < VEC; ++v) dot = __fmaf_rn(to_f32<T>(pg.v[v]), to_f32<T>(py.v[v]), dot);
                    }
                }
            if (a.dweights) {
                dot = fg::warp_sum(dot);
                if (lane == 0) a.dweights[t * a.k + j] = dot;
            }
        }
    }
    if (!a.dy) return;
    const int used = max(0, a.offsets[a.groups]);
    for (int64_t p = used + t; p < a.m; p += (int64_t)gridDim.x * 8) {
        T* row = static_cast<T*>(a.dy) + p * a.d;
        for (int c = lane; c < a.d; c += 32) row[c] = from_f32<T>(0.0f);
    }
}

template <typename T, typename O = T>
int launch_combine(const CombineArgs& a, bool vec, cudaStream_t s) {
    constexpr int kVec = 16 / sizeof(T);
    const int64_t units = a.n * ((a.d + (vec ? kVec : 1) - 1) / (vec ? kVec : 1)), blocks = (units + 255) / 256;
    if (blocks > INT_MAX) return fg::fail(FG_ERR_INVALID_ARGUMENT, "grid too large");
    if (vec) combine_kernel<T, kVec, O><<<(unsigned)blocks, 256, 0, s>>>(a);
    else combine_kernel<T, 1, O><<<(unsigned)blocks, 256, 0, s>>>(a);
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return FG_OK;
}
template <typename T>
int launch_combine_grad(const CombineArgs& a, bool vec, cudaStream_t s) {
    const unsigned blocks = (unsigned)((a.n + 7) / 8);
    if (vec) combine_grad_kernel<T, 16 / sizeof(T)><<<blocks, 256, 0, s>>>(a);
    else combine_grad_kernel<T, 1><<<blocks, 256, 0, s>>>(a);
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return FG_OK;
}

int check_combine(int64_t n, int32_t k, int32_t d, int32_t type) {
    if (n < 0 || k < 1 || k > kMaxChoices || d < 1 || d > INT_MAX - 1024 || n > INT_MAX / k)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "bad sizes n=%lld k=%d d=%d (1 <= k <= %d, n k < 2^31)", (long long)n, k, d, kMaxChoices);
    if (!fg::float_type(type)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "unknown value type %d", type);
    return FG_OK;
}

int check_route(int64_t n, int32_t experts, int32_t k, int32_t type, int32_t scoring) {
    if (n < 0 || experts < 1 || experts > kMaxExperts || k < 1 || k > kMaxChoices || k > experts || n > INT_MAX / k)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "bad sizes n=%lld experts=%d k=%d (experts <= %d, k <= experts, k <= %d, n k < 2^31)",
                        (long long)n, experts, k, kMaxExperts, kMaxChoices);
    if (!fg::float_type(type)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "unknown value type %d", type);
    if (scoring != FG_SCORE_SOFTMAX && scoring != FG_SCORE_SIGMOID) return fg::fail(FG_ERR_INVALID_ARGUMENT, "unknown scoring %d", scoring);
    return FG_OK;
}

// Rows that one block chooses and lists by itself, a warp each: one launch instead of two.
constexpr int64_t kOneBlockRows = 32;

// 8192 entries or fewer are one chunk; above that chunks of at least 2048, at most 1024 of them.  One launch or three, 128
// groups, called / in a graph: 8192 entries 16 / 14 us in one; 16384 22 / 21 in one and 21 / 10 in three.
int64_t chunk_size(int64_t m) {
    if (m <= 8192) return 8192;
    int64_t c = (m + 1023) / 1024;
    c = c < 2048 ? 2048 : c;
    return (c + 255) / 256 * 256;
}

}  // namespace

namespace fg {
int sum_slots(const float* parts, const int32_t* position, void* out, int64_t n, int32_t k, int32_t d, int32_t type, cudaStream_t s) {
    if (int rc = check_combine(n, k, d, type)) return rc;
    if (n == 0) return FG_OK;
    CombineArgs a{};
    a.y = parts, a.position = position, a.out = out;
    a.n = n, a.m = n * k, a.ldy = d, a.k = k, a.d = d;
    const bool vec = d % 4 == 0 && aligned16(parts) && aligned16(out);
    return type == FG_F32   ? launch_combine<float, float>(a, vec, s)
           : type == FG_F16 ? launch_combine<float, __half>(a, vec, s)
                            : launch_combine<float, __nv_bfloat16>(a, vec, s);
}
}  // namespace fg

extern "C" {

int fg_route_backward(const void* d_logits, int64_t ld, const float* d_weights, const int32_t* d_experts, const float* d_dweights,
                      void* d_dlogits, int64_t n, int32_t experts, int32_t k, int32_t type, int32_t scoring, int32_t normalize,
                      void* stream) {
    if (int rc = check_route(n, experts, k, type, scoring)) return rc;
    if (ld == 0) ld = experts;
    if (ld < experts) return fg::fail(FG_ERR_INVALID_ARGUMENT, "the row stride must be 0 or >= experts=%d", experts);
    if (n == 0) return FG_OK;
    if (!d_logits || !d_weights || !d_experts || !d_dweights || !d_dlogits) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    const RouteGradArgs a{d_logits, ld, n, experts, k, scoring == FG_SCORE_SIGMOID, normalize != 0, d_weights, d_dweights, d_experts, d_dlogits};
    by_logit_type(type, experts, LaunchRouteGrad{a, static_cast<cudaStream_t>(stream)});
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return FG_OK;
}

int64_t fg_group_rows_workspace(int64_t num_entries, int32_t num_groups) {
    if (num_entries <= 0 || num_groups < 1) return 0;
    const int64_t chunk = chunk_size(num_entries), chunks = (num_entries + chunk - 1) / chunk;
    return chunks <= 1 ? 0 : (chunks + 1) * ((int64_t)num_groups + 1) * 4;
}

int fg_group_rows(const int32_t* d_keys, int64_t num_entries, int32_t num_groups, int32_t* d_offsets, int32_t* d_order,
                  int32_t* d_position, void* d_workspace, int64_t workspace_bytes, void* stream) {
    if (num_entries < 0 || num_entries > INT_MAX || num_groups < 1 || num_groups > kMaxGroups)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "bad sizes entries=%lld groups=%d (1 <= groups <= %d)", (long long)num_entries, num_groups, kMaxGroups);
    if (!d_offsets || (num_entries && (!d_keys || !d_order || !d_position))) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    if (workspace_bytes < fg_group_rows_workspace(num_entries, num_groups) || (fg_group_rows_workspace(num_entries, num_groups) && !d_workspace))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "workspace smaller than fg_group_rows_workspace()");
    if (fg_group_rows_workspace(num_entries, num_groups) && !fg::aligned16(d_workspace))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "the workspace must start on a 16-byte boundary");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (num_entries == 0) {
        FG_CUDA_TRY(cudaMemsetAsync(d_offsets, 0, ((size_t)num_groups + 1) * 4, s));
        return FG_OK;
    }
    const int64_t chunk = chunk_size(num_entries), chunks = (num_entries + chunk - 1) / chunk;
    const GroupArgs a{d_keys, num_entries, num_groups, (int32_t)chunk, (int32_t)chunks, static_cast<int32_t*>(d_workspace), d_offsets, d_order, d_position};
    const int bins = num_groups + 1;
    if (chunks == 1) {
        const int warps = num_entries <= 256 ? 4 : num_entries <= 2048 ? 16 : 32;
        GroupArgs one = a;
        one.chunk = (int32_t)num_entries;
        const size_t smem = (size_t)warps * bins * 4;
        if (smem > 40 * 1024) FG_CUDA_TRY(cudaFuncSetAttribute(group_place_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
        group_place_kernel<true><<<1, warps * 32, smem, s>>>(one);
        FG_CUDA_TRY(cudaGetLastError());
        fg::count_launches(1);
        return FG_OK;
    }
    group_count_kernel<<<(unsigned)chunks, 256, (size_t)bins * 4, s>>>(a);
    FG_CUDA_TRY(cudaGetLastError());
    group_scan_kernel<<<(unsigned)((bins + 3) / 4), 128, 0, s>>>(a);
    FG_CUDA_TRY(cudaGetLastError());
    group_place_kernel<false><<<(unsigned)chunks, 256, (size_t)8 * bins * 4, s>>>(a);
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(3);
    return FG_OK;
}

int fg_route(const void* d_logits, int64_t ld, float* d_weights, int32_t* d_experts, int32_t* d_offsets, int32_t* d_order,
             int32_t* d_position, int64_t n, int32_t experts, int32_t k, int32_t type, int32_t scoring, int32_t normalize,
             void* d_workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_route(n, experts, k, type, scoring)) return rc;
    if (ld == 0) ld = experts;
    if (ld < experts) return fg::fail(FG_ERR_INVALID_ARGUMENT, "the row stride must be 0 or >= experts=%d", experts);
    if (n == 0) return d_offsets ? fg_group_rows(d_experts, 0, experts, d_offsets, d_order, d_position, d_workspace, workspace_bytes, stream) : FG_OK;
    if (!d_logits || !d_weights || !d_experts || (d_offsets && (!d_order || !d_position))) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    if (d_offsets && workspace_bytes < fg_group_rows_workspace(n * k, experts))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "workspace smaller than fg_group_rows_workspace()");
    if (d_offsets && fg_group_rows_workspace(n * k, experts) && !fg::aligned16(d_workspace))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "the workspace must start on a 16-byte boundary");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const RouteArgs a{d_logits, ld, n, experts, k, scoring == FG_SCORE_SIGMOID, normalize != 0, d_weights, d_experts};
    if (d_offsets && n <= kOneBlockRows) {
        const GroupArgs g{d_experts, n * k, experts, (int32_t)(n * k), 1, nullptr, d_offsets, d_order, d_position};
        by_logit_type(type, experts, LaunchRouteLists{a, g, s});
        FG_CUDA_TRY(cudaGetLastError());
        fg::count_launches(1);
        return FG_OK;
    }
    by_logit_type(type, experts, LaunchRoute{a, s});
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return d_offsets ? fg_group_rows(d_experts, n * k, experts, d_offsets, d_order, d_position, d_workspace, workspace_bytes, stream) : FG_OK;
}

int fg_combine_rows(const void* d_y, int64_t ldy, const float* d_weights, const int32_t* d_position, void* d_out, int64_t n,
                    int32_t k, int32_t d, int32_t type, void* stream) {
    if (int rc = check_combine(n, k, d, type)) return rc;
    if (ldy == 0) ldy = d;
    if (ldy < d) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= d=%d", d);
    if (n == 0) return FG_OK;
    if (!d_y || !d_position || !d_out) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    CombineArgs a{};
    a.y = d_y, a.weights = d_weights, a.position = d_position, a.out = d_out;
    a.n = n, a.m = n * k, a.ldy = ldy, a.k = k, a.d = d;
    const int per = 16 / fg::type_size(type);
    const bool vec = d % per == 0 && ldy % per == 0 && fg::aligned16(d_y) && fg::aligned16(d_out);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return type == FG_F32 ? launch_combine<float>(a, vec, s) : type == FG_F16 ? launch_combine<__half>(a, vec, s) : launch_combine<__nv_bfloat16>(a, vec, s);
}

int fg_combine_rows_backward(const void* d_y, int64_t ldy, const float* d_weights, const int32_t* d_position, const int32_t* d_offsets,
                             int32_t num_groups, const void* d_dout, int64_t ldd, void* d_dy, float* d_dweights, int64_t n, int32_t k,
                             int32_t d, int32_t type, void* stream) {
    if (int rc = check_combine(n, k, d, type)) return rc;
    if (ldy == 0) ldy = d;
    if (ldd == 0) ldd = d;
    if (ldy < d || ldd < d) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= d=%d", d);
    if (num_groups < 1) return fg::fail(FG_ERR_INVALID_ARGUMENT, "bad sizes groups=%d", num_groups);
    if (n == 0 || (!d_dy && !d_dweights)) return FG_OK;
    if (!d_position || !d_offsets || !d_dout || (d_dweights && !d_y)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    CombineArgs a{};
    a.y = d_y, a.dout = d_dout, a.weights = d_weights, a.position = d_position, a.offsets = d_offsets, a.dy = d_dy, a.dweights = d_dweights;
    a.n = n, a.m = n * k, a.ldy = ldy, a.ldd = ldd, a.k = k, a.d = d, a.groups = num_groups;
    const int per = 16 / fg::type_size(type);
    const bool vec = d % per == 0 && ldy % per == 0 && ldd % per == 0 && fg::aligned16(d_y) && fg::aligned16(d_dout) && fg::aligned16(d_dy);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return type == FG_F32 ? launch_combine_grad<float>(a, vec, s) : type == FG_F16 ? launch_combine_grad<__half>(a, vec, s) : launch_combine_grad<__nv_bfloat16>(a, vec, s);
}

}  // extern "C"
