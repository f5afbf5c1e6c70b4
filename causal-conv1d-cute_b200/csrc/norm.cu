// Gated RMS norm: out = x rsqrt(mean(x^2) + eps) weight silu(z), row by row.
//
// Bound: HBM (x and z read, out written once; about 10 flops and two special-function results per
// element). A group of LANES lanes owns a row: VPL 16-byte vectors of x and of z per lane, all
// loaded before the row's sum of squares is reduced by shuffles, so the row is read once. R rows
// per group keep enough bytes in flight.
#include "common.cuh"
#include "kernels.h"

namespace cc1d {
namespace {

// z sigmoid(z) in fp32. The fast exponential and division err by a few ulp of fp32, far below the
// rounding of a 16-bit output; fp32 outputs take the library's expf and a true division.
template <typename T>
__device__ __forceinline__ float gate(float z) {
    if constexpr (sizeof(T) == 4) {
        return z / (1.f + expf(-z));
    } else {
        return __fdividef(z, 1.f + __expf(-z));
    }
}

// n / d for n below 2^31 by one multiplication (d >= 1), d fixed for a launch.
struct Divider {
    uint32_t d, mul, shift;
    explicit Divider(uint32_t divisor) : d(divisor), mul(0), shift(0) {
        while (shift < 31 && (1u << shift) < d) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        return (__umulhi(n, mul) + n) >> shift;
    }
};

template <typename T, int LANES, int VPL, int R>
__global__ void __launch_bounds__(256)
norm_kernel(const __grid_constant__ cc1d_norm_args a, int rows, Divider by_n1) {
    constexpr int V = Vec<T>::V;
    constexpr int GROUPS = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int first = blockIdx.x * (GROUPS * R) + threadIdx.x / LANES;
    const T* xp = static_cast<const T*>(a.x);
    const T* zp = static_cast<const T*>(a.z);
    T* op = static_cast<T*>(a.out);

    uint4 x[R][VPL], z[R][VPL];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = first + r * GROUPS;
        const int64_t i0 = by_n1(row), i1 = row - i0 * a.n1;
#pragma unroll
        for (int m = 0; m < VPL; ++m) {
            const int e = (m * LANES + lane) * V;
            x[r][m] = z[r][m] = make_uint4(0, 0, 0, 0);
            if (row < rows && e < a.dim) {
                x[r][m] = ldg16_stream(xp + i0 * a.x_s0 + i1 * a.x_s1 + e);
                if (zp != nullptr) z[r][m] = ldg16_stream(zp + i0 * a.z_s0 + i1 * a.z_s1 + e);
            }
        }
    }
    float w[VPL][V];
#pragma unroll
    for (int m = 0; m < VPL; ++m)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = (m * LANES + lane) * V + i;
            w[m][i] = 0.f;
            if (e < a.dim)
                w[m][i] = a.wdtype == CC1D_F32 ? static_cast<const float*>(a.weight)[e]
                                               : to_f32(static_cast<const T*>(a.weight)[e]);
        }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = first + r * GROUPS;
        float f[VPL][V], sum = 0.f;
#pragma unroll
        for (int m = 0; m < VPL; ++m) {
            unpack16<T>(x[r][m], f[m]);
#pragma unroll
            for (int i = 0; i < V; ++i) sum = fmaf(f[m][i], f[m][i], sum);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
        const float inv = rsqrtf(sum / (float)a.dim + a.eps);
        if (row >= rows) continue;
        const int64_t i0 = by_n1(row), i1 = row - i0 * a.n1;
#pragma unroll
        for (int m = 0; m < VPL; ++m) {
            const int e = (m * LANES + lane) * V;
            if (e >= a.dim) continue;
            float g[V];
            unpack16<T>(z[r][m], g);
#pragma unroll
            for (int i = 0; i < V; ++i)
                f[m][i] = f[m][i] * inv * w[m][i] * (zp != nullptr ? gate<T>(g[i]) : 1.f);
            st16_stream(op + i0 * a.o_s0 + i1 * a.o_s1 + e, pack16<T>(f[m]));
        }
    }
}

// Any row length, stride and alignment: one warp per row, element by element, x read twice.
template <typename T>
__global__ void __launch_bounds__(256)
norm_generic_kernel(const __grid_constant__ cc1d_norm_args a, int64_t rows) {
    const int lane = threadIdx.x % 32;
    const int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
    if (row >= rows) return;
    const int64_t i0 = row / a.n1, i1 = row % a.n1;
    const T* xp = static_cast<const T*>(a.x) + i0 * a.x_s0 + i1 * a.x_s1;
    const T* zp = a.z == nullptr ? nullptr : static_cast<const T*>(a.z) + i0 * a.z_s0 + i1 * a.z_s1;
    T* op = static_cast<T*>(a.out) + i0 * a.o_s0 + i1 * a.o_s1;
    float sum = 0.f;
    for (int64_t e = lane; e < a.dim; e += 32) {
        const float f = to_f32(xp[e]);
        sum = fmaf(f, f, sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
    const float inv = rsqrtf(sum / (float)a.dim + a.eps);
    for (int64_t e = lane; e < a.dim; e += 32) {
        const float w = a.wdtype == CC1D_F32 ? static_cast<const float*>(a.weight)[e]
                                             : to_f32(static_cast<const T*>(a.weight)[e]);
        const float g = zp != nullptr ? gate<T>(to_f32(zp[e])) : 1.f;
        op[e] = from_f32<T>(to_f32(xp[e]) * inv * w * g);
    }
}

template <typename T, int LANES, int VPL, int R>
void go(const cc1d_norm_args& a, int64_t rows, cudaStream_t stream) {
    const int64_t grid = ceil_div(rows, (256 / LANES) * R);
    norm_kernel<T, LANES, VPL, R><<<(unsigned)grid, 256, 0, stream>>>(a, (int)rows, Divider((uint32_t)a.n1));
}

template <typename T>
cudaError_t launch(const cc1d_norm_args& a, cudaStream_t stream) {
    constexpr int V = Vec<T>::V;
    const int64_t rows = a.n0 * a.n1;
    if (ceil_div(rows, 8) > INT32_MAX) return cudaErrorInvalidConfiguration;
    const bool vec = a.dim % V == 0 && host_aligned16(a.x) && host_aligned16(a.out) &&
                     (a.z == nullptr || (host_aligned16(a.z) && a.z_s0 % V == 0 && a.z_s1 % V == 0)) &&
                     a.x_s0 % V == 0 && a.x_s1 % V == 0 && a.o_s0 % V == 0 && a.o_s1 % V == 0;
    // 2^30 rows and more (their 32-bit indices and the divider's) take the generic kernel.
    if (!vec || a.dim > 128 * V || rows >= (1 << 30)) {
        norm_generic_kernel<T><<<(unsigned)ceil_div(rows, 8), 256, 0, stream>>>(a, rows);
    } else if (a.dim <= 8 * V) {
        go<T, 8, 1, 4>(a, rows, stream);
    } else if (a.dim <= 16 * V) {
        go<T, 16, 1, 4>(a, rows, stream);
    } else if (a.dim <= 32 * V) {
        go<T, 32, 1, 4>(a, rows, stream);
    } else if (a.dim <= 64 * V) {
        go<T, 32, 2, 2>(a, rows, stream);
    } else {
        go<T, 32, 4, 1>(a, rows, stream);
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_norm(const cc1d_norm_args& a, cudaStream_t stream) {
    CC1D_DISPATCH_DTYPE(a.dtype, return launch<T>(a, stream));
    return cudaErrorInvalidValue;
}

}  // namespace cc1d
