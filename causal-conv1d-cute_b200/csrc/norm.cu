// Gated RMS norm: out = x rsqrt(mean(x^2) + eps) weight silu(z), row by row.
//
// Bound: HBM (x and z read, out written once; about 10 flops and two special-function results per
// element). A group of LANES lanes owns a row: VPL 16-byte vectors of x and of z per lane, all
// loaded before the row's sum of squares is reduced by shuffles, so the row is read once. Two rows
// per group and six CTAs per SM keep enough bytes in flight: 40807 x 48 rows of 128 in bf16 227 us, 6.6
// TB/s, which is the copy rate (four rows and two CTAs 255 us, one row and eight 245 us).
#include "common.cuh"
#include "kernels.h"

namespace cc1d {
namespace {

// Two lanes of x inv w z sigmoid(z), the factors that do not depend on the row in w. For 16-bit types
// the exponential, the reciprocal (a few ulp of fp32 each) and packed arithmetic: with scalar
// arithmetic and a division the kernel was bound by issue (0.84 a cycle). fp32 takes the library's
// expf and a true division.
template <typename T>
__device__ __forceinline__ float2 gated(float2 x, float2 z, float2 w, float inv, bool gate) {
    const float2 y = __fmul2_rn(__fmul2_rn(x, make_float2(inv, inv)), w);
    if (!gate) return y;
    float2 s;
    if constexpr (sizeof(T) == 4) {
        s = make_float2(z.x / (1.f + expf(-z.x)), z.y / (1.f + expf(-z.y)));
    } else {
        constexpr float kNegLog2e = -1.4426950408889634f;
        const float2 e = __fmul2_rn(z, make_float2(kNegLog2e, kNegLog2e));
        float2 t;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(e.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(e.y));
        t = __fadd2_rn(t, make_float2(1.f, 1.f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(t.x));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(t.y));
        s = __fmul2_rn(s, z);
    }
    return __fmul2_rn(y, s);
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
__global__ void __launch_bounds__(256, VPL == 1 ? 6 : 1)
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
    float2 w[VPL][V / 2];
#pragma unroll
    for (int m = 0; m < VPL; ++m)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = (m * LANES + lane) * V + i;
            float& to = i % 2 ? w[m][i / 2].y : w[m][i / 2].x;
            to = 0.f;
            if (e < a.dim)
                to = a.wdtype == CC1D_F32 ? static_cast<const float*>(a.weight)[e]
                                               : to_f32(static_cast<const T*>(a.weight)[e]);
        }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = first + r * GROUPS;
        float2 f[VPL][V / 2], sums = make_float2(0.f, 0.f);
#pragma unroll
        for (int m = 0; m < VPL; ++m) {
            unpack16<T>(x[r][m], &f[m][0].x);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) sums = __ffma2_rn(f[m][i], f[m][i], sums);
        }
        float sum = sums.x + sums.y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
        const float inv = rsqrtf(sum / (float)a.dim + a.eps);
        if (row >= rows) continue;
        const int64_t i0 = by_n1(row), i1 = row - i0 * a.n1;
#pragma unroll
        for (int m = 0; m < VPL; ++m) {
            const int e = (m * LANES + lane) * V;
            if (e >= a.dim) continue;
            float2 g[V / 2];
            unpack16<T>(z[r][m], &g[0].x);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) f[m][i] = gated<T>(f[m][i], g[i], w[m][i], inv, zp != nullptr);
            st16_stream(op + i0 * a.o_s0 + i1 * a.o_s1 + e, pack16<T>(&f[m][0].x));
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
        const float2 x = make_float2(to_f32(xp[e]), 0.f), z = make_float2(zp != nullptr ? to_f32(zp[e]) : 0.f, 0.f);
        op[e] = from_f32<T>(gated<T>(x, z, make_float2(w, 0.f), inv, zp != nullptr).x);
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
        go<T, 8, 1, 2>(a, rows, stream);
    } else if (a.dim <= 16 * V) {
        go<T, 16, 1, 2>(a, rows, stream);
    } else if (a.dim <= 32 * V) {
        go<T, 32, 1, 2>(a, rows, stream);
    } else if (a.dim <= 64 * V) {
        go<T, 32, 2, 1>(a, rows, stream);
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
