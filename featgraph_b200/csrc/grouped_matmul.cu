// Products grouped by expert (node type, relation): y[p] = W[g(p)] x[row(p)] for the rows p of each group.
//
// Simple form: 64 x 64 output tiles, 256 threads with 4 x 4 outputs each, 16 values of the inner axis at a time
// through shared memory, 32-bit sums of fused multiply-adds.  Any strides.
#include <climits>

#include "rows.cuh"

namespace {

using fg::from_f32;
using fg::to_f32;

struct ProductArgs {
    const void *x, *w;
    const float *x_scales, *w_scales;
    const int32_t *offsets, *order;
    void* y;
    int64_t ldx, w_group, w_out, w_in, x_rows, m;
    int32_t choices, groups, inner, outer;
};

// First row and end of row tile `tile` (tiles of `size` rows never span two groups; group `groups` stands for the rows
// in no group).  False past the last tile.
__device__ bool locate_tile(const int32_t* offsets, int groups, int64_t m, int size, int64_t tile, int& group, int64_t& first, int64_t& end) {
    int64_t begin = 0;
    for (int g = 0; g <= groups; ++g) {
        const int64_t stop = g < groups ? min((int64_t)max(offsets[g + 1], 0), m) : m;
        const int64_t tiles = stop > begin ? (stop - begin + size - 1) / size : 0;
        if (tile < tiles) {
            group = g, first = begin + tile * size, end = min(first + size, stop);
            return true;
        }
        tile -= tiles;
        begin = max(begin, stop);
    }
    return false;
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) product_kernel(const ProductArgs a) {
    __shared__ float sx[16][65], sw[16][65];
    __shared__ int64_t source[64];
    int g;
    int64_t first, end;
    if (!locate_tile(a.offsets, a.groups, a.m, 64, blockIdx.y, g, first, end)) return;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, col0 = blockIdx.x * 64;
    if (threadIdx.x < 64) {
        const int64_t p = first + threadIdx.x;
        int64_t r = -1;
        if (p < end && g < a.groups) {
            r = p;
            if (a.order) {
                const int e = a.order[p];
                r = e < 0 ? -1 : e / a.choices;
            }
            if (r >= a.x_rows) r = -1;
        }
        source[threadIdx.x] = r;
    }
    __syncthreads();
    float acc[4][4] = {};
    const T* w = static_cast<const T*>(a.w) + (int64_t)(g < a.groups ? g : 0) * a.w_group;
    for (int k0 = 0; k0 < (g < a.groups ? a.inner : 0); k0 += 16) {
        for (int i = threadIdx.x; i < 1024; i += 256) {
            const int kk = i % 16, r = i / 16;
            const bool in = k0 + kk < a.inner;
            sx[kk][r] = in && source[r] >= 0 ? to_f32<T>(static_cast<const T*>(a.x)[source[r] * a.ldx + k0 + kk]) : 0.0f;
            sw[kk][r] = in && col0 + r < a.outer ? to_f32<T>(w[(int64_t)(col0 + r) * a.w_out + (int64_t)(k0 + kk) * a.w_in]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 16; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(sx[kk][ty * 4 + i], sw[kk][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
        const int64_t p = first + ty * 4 + i;
        if (p >= end) continue;
        for (int j = 0; j < 4; ++j) {
            const int c = col0 + tx + 16 * j;
            if (c >= a.outer) continue;
            float v = acc[i][j];
            if (a.x_scales && source[ty * 4 + i] >= 0 && g < a.groups)
                v = __fmul_rn(__fmul_rn(v, a.x_scales[source[ty * 4 + i]]), a.w_scales[(int64_t)g * a.outer + c]);
            static_cast<O*>(a.y)[p * a.outer + c] = from_f32<O>(v);
        }
    }
}

struct WeightGradArgs {
    const void *x, *dy;
    const int32_t *offsets, *order;
    void* dw;
    int64_t ldx, lddy, x_rows, m;
    int32_t choices, groups, inner, outer;
};

template <typename T>
__global__ void __launch_bounds__(256) weight_grad_kernel(const WeightGradArgs a) {
    __shared__ float sx[16][65], sy[16][65];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, in0 = blockIdx.x * 64, out0 = blockIdx.y * 64, g = blockIdx.z;
    const int64_t begin = min((int64_t)max(a.offsets[g], 0), a.m), end = min((int64_t)max(a.offsets[g + 1], 0), a.m);
    float acc[4][4] = {};
    for (int64_t p0 = begin; p0 < end; p0 += 16) {
        for (int i = threadIdx.x; i < 1024; i += 256) {
            const int c = i % 64, r = i / 64;
            const int64_t p = p0 + r;
            int64_t row = p < end ? p : -1;
            if (row >= 0 && a.order) {
                const int e = a.order[p];
                row = e < 0 ? -1 : e / a.choices;
            }
            if (row >= a.x_rows) row = -1;
            sx[r][c] = row >= 0 && in0 + c < a.inner ? to_f32<T>(static_cast<const T*>(a.x)[row * a.ldx + in0 + c]) : 0.0f;
            sy[r][c] = row >= 0 && out0 + c < a.outer ? to_f32<T>(static_cast<const T*>(a.dy)[p * a.lddy + out0 + c]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(sy[r][ty * 4 + i], sx[r][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int o = out0 + ty * 4 + i, c = in0 + tx + 16 * j;
            if (o < a.outer && c < a.inner) static_cast<T*>(a.dw)[((int64_t)g * a.outer + o) * a.inner + c] = from_f32<T>(acc[i][j]);
        }
}

int check_product(int64_t m, int64_t x_rows, int32_t choices, int32_t groups, int32_t inner, int32_t outer) {
    if (m < 0 || m > INT_MAX || x_rows < 0 || x_rows > INT_MAX || choices < 1 || groups < 1 || groups > 1024 || inner < 1 || outer < 1)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "bad sizes rows=%lld of %lld choices=%d groups=%d inner=%d outer=%d (groups <= 1024)",
                        (long long)m, (long long)x_rows, choices, groups, inner, outer);
    return FG_OK;
}

}  // namespace

extern "C" {

int64_t fg_grouped_matmul_workspace(int64_t num_rows, int64_t x_rows, int32_t groups, int32_t inner, int32_t outer, int32_t type) {
    return 0;
}

int fg_grouped_matmul(const void* d_x, int64_t ldx, const float* d_x_scales, const void* d_w, int64_t w_group, int64_t w_out,
                      int64_t w_in, const float* d_w_scales, const int32_t* d_offsets, const int32_t* d_order, int32_t choices,
                      int64_t x_rows, void* d_y, int64_t num_rows, int32_t groups, int32_t inner, int32_t outer, int32_t type,
                      int32_t out_type, void* d_workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_product(num_rows, x_rows, choices, groups, inner, outer)) return rc;
    if (!fg::float_type(type) && type != FG_E4M3) return fg::fail(FG_ERR_INVALID_ARGUMENT, "unknown value type %d", type);
    if (type == FG_E4M3 ? !fg::float_type(out_type) : out_type != type)
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "the output is of the inputs' type, or of a wider one for e4m3");
    if (ldx == 0) ldx = inner;
    if (ldx < inner) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= inner=%d", inner);
    if (num_rows == 0) return FG_OK;
    if (!d_x || !d_w || !d_offsets || !d_y || (type == FG_E4M3 && (!d_x_scales || !d_w_scales)))
        return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    const ProductArgs a{d_x, d_w, d_x_scales, d_w_scales, d_offsets, d_order, d_y, ldx, w_group, w_out, w_in, x_rows, num_rows, choices, groups, inner, outer};
    const int64_t tiles = num_rows / 64 + groups + 1;
    if (tiles > 65535) return fg::fail(FG_ERR_INVALID_ARGUMENT, "grid too large");
    const dim3 grid((outer + 63) / 64, (unsigned)tiles);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == FG_F32) product_kernel<float, float><<<grid, 256, 0, s>>>(a);
    else if (type == FG_F16) product_kernel<__half, __half><<<grid, 256, 0, s>>>(a);
    else if (type == FG_BF16) product_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, s>>>(a);
    else if (out_type == FG_F32) product_kernel<__nv_fp8_e4m3, float><<<grid, 256, 0, s>>>(a);
    else if (out_type == FG_F16) product_kernel<__nv_fp8_e4m3, __half><<<grid, 256, 0, s>>>(a);
    else product_kernel<__nv_fp8_e4m3, __nv_bfloat16><<<grid, 256, 0, s>>>(a);
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return FG_OK;
}

int64_t fg_grouped_matmul_wgrad_workspace(int64_t num_rows, int64_t x_rows, int32_t groups, int32_t inner, int32_t outer, int32_t type) {
    return 0;
}

int fg_grouped_matmul_wgrad(const void* d_x, int64_t ldx, const void* d_dy, int64_t lddy, const int32_t* d_offsets,
                            const int32_t* d_order, int32_t choices, int64_t x_rows, void* d_dw, int64_t num_rows, int32_t groups,
                            int32_t inner, int32_t outer, int32_t type, void* d_workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_product(num_rows, x_rows, choices, groups, inner, outer)) return rc;
    if (!fg::float_type(type)) return fg::fail(FG_ERR_INVALID_ARGUMENT, "unknown value type %d", type);
    if (ldx == 0) ldx = inner;
    if (lddy == 0) lddy = outer;
    if (ldx < inner || lddy < outer) return fg::fail(FG_ERR_INVALID_ARGUMENT, "row strides must be 0 or >= the width");
    if (!d_dw || !d_offsets || (num_rows && (!d_x || !d_dy))) return fg::fail(FG_ERR_INVALID_ARGUMENT, "NULL array argument");
    const WeightGradArgs a{d_x, d_dy, d_offsets, d_order, d_dw, ldx, lddy, x_rows, num_rows, choices, groups, inner, outer};
    const dim3 grid((inner + 63) / 64, (outer + 63) / 64, groups);
    if (grid.y > 65535) return fg::fail(FG_ERR_INVALID_ARGUMENT, "grid too large");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == FG_F32) weight_grad_kernel<float><<<grid, 256, 0, s>>>(a);
    else if (type == FG_F16) weight_grad_kernel<__half><<<grid, 256, 0, s>>>(a);
    else weight_grad_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
    FG_CUDA_TRY(cudaGetLastError());
    fg::count_launches(1);
    return FG_OK;
}

}  // extern "C"
