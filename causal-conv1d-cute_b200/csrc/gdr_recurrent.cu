// Gated delta rule, token by token: decode of one or a few tokens per batch row, and packed
// prefill of rows too short, or of shapes or types outside, the chunked kernel (gdr_chunk.cu).
//
// Mathematics. With S the (dk, dv) state of a value head, a token does
//     S' = alpha S,  u = beta (v - S'^T k),  S <- S' + k u^T,  o = scale S^T q.
// S^T k and S^T q are taken in ONE pass over the old state: o = scale (alpha S_old^T q + (q.k) u),
// so a token costs one reduction over dk and one rank-1 update.
//
// Bound. A decode step reads and writes the whole state (64 KB per head at dk = dv = 128 in fp32)
// for 6 dk dv flops: HBM bandwidth. Few rows are bound by latency (launch, slot -> state load).
//
// Layout. The columns of S are independent, so they are the parallel axis: a warp owns 16 columns
// and all dk rows. Four lanes hold 4 columns each (one 16-byte vector of fp32 state), eight lane
// groups hold the rows; the reduction over dk is RPT FMAs per lane and three shuffles, with no
// exchange between warps. All state loads of a thread are issued before the token's q and k are
// staged, so they overlap with the gate and norm arithmetic.
#include "gdr.cuh"
#include "kernels.h"

namespace cc1d {
namespace {

constexpr int kTokTile = 4;   // tokens staged in shared memory at a time
constexpr int kWarpCols = 16;

template <typename ST>
__device__ __forceinline__ void load4(const ST* p, bool vec, int valid, float* f) {
    if (vec) {
        unpack_raw<ST, 4 * (int)sizeof(ST)>(ld_raw<4 * (int)sizeof(ST)>(p), f);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = i < valid ? to_f32(p[i]) : 0.f;
    }
}

template <typename ST>
__device__ __forceinline__ void store4(ST* p, bool vec, int valid, const float* f) {
    if (vec) {
        st_raw<4 * (int)sizeof(ST)>(p, pack_raw<ST, 4 * (int)sizeof(ST)>(f));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = from_f32<ST>(f[i]);
    }
}

// RPT: rows of the state per thread (dk <= 8 RPT). WARPS: warps per CTA, 16 columns each.
template <typename T, typename ST, int RPT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
gdr_recurrent_kernel(const __grid_constant__ cc1d_gdr_args a, bool varlen, bool vec, int tiles) {
    constexpr int KP = 8 * RPT;
    __shared__ __align__(16) float sq[kTokTile][KP], sk[kTokTile][KP];
    __shared__ float s_alpha[kTokTile], s_beta[kTokTile];

    const int tile = blockIdx.x % tiles;
    const int64_t rh = blockIdx.x / tiles;
    const int h = (int)(rh % a.heads_v);
    const int64_t row = rh / a.heads_v;
    const int hk = h / (a.heads_v / a.heads_k);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rg = lane / 4;
    const int col = (tile * WARPS + warp) * kWarpCols + (lane % 4) * 4;
    const int valid = min(4, max(0, a.dv - col));

    int64_t tok0, slot;
    int ntok;
    if (!gdr_row(a, varlen, row, tok0, ntok, slot, h == 0 && tile == 0 && threadIdx.x == 0)) return;
    int64_t islot = -1;
    if (a.inter != nullptr) {
        islot = a.inter_indices != nullptr ? a.inter_indices[row] : slot;
        if (islot < 0 || islot >= a.inter_nslots) {
            if (h == 0 && tile == 0 && threadIdx.x == 0)
                flag_status(a.dev_status, CC1D_DEV_BAD_INTER_SLOT);
            islot = -1;
        }
    }

    // Row r of a thread: (r / 4) * 32 + rg * 4 + r % 4, so that q and k come as 16-byte vectors.
    float S[RPT][4];
    const bool initial = !varlen || (a.has_initial_state != nullptr && a.has_initial_state[row]);
    ST* st = nullptr;
    if (slot >= 0) st = static_cast<ST*>(a.states) + slot * a.s_slot + h * a.s_sh + col;
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
        const int k = (r / 4) * 32 + rg * 4 + r % 4;
        if (st != nullptr && initial && valid > 0 && k < a.dk) {
            load4(st + k * a.s_sk, vec, valid, S[r]);
        } else {
            S[r][0] = S[r][1] = S[r][2] = S[r][3] = 0.f;
        }
    }

    const T* qp = static_cast<const T*>(a.q) + (varlen ? 0 : row * a.q_sb) + hk * a.q_sh;
    const T* kp = static_cast<const T*>(a.k) + (varlen ? 0 : row * a.k_sb) + hk * a.k_sh;
    const T* vp = static_cast<const T*>(a.v) + (varlen ? 0 : row * a.v_sb) + h * a.v_sh;
    T* op = static_cast<T*>(a.out) + (varlen ? 0 : row * a.o_sb) + h * a.o_sh;
    const int64_t g0 = (varlen ? 0 : row * a.g_sb) + h * a.g_sh;
    const int64_t b0 = (varlen ? 0 : row * a.b_sb) + h * a.b_sh;

    for (int base = 0; base < ntok; base += kTokTile) {
        const int n = min(kTokTile, ntok - base);
        if (base > 0) __syncthreads();
        for (int i = warp; i < 2 * n; i += WARPS) {
            const int64_t t = tok0 + base + i / 2;
            const T* src = i % 2 ? kp + t * a.k_st : qp + t * a.q_st;
            const int64_t sd = i % 2 ? a.k_sd : a.q_sd;
            float* dst = i % 2 ? sk[i / 2] : sq[i / 2];
            float x[KP / 32], sum = 0.f;
#pragma unroll
            for (int m = 0; m < KP / 32; ++m) {
                const int e = lane + 32 * m;
                x[m] = e < a.dk ? to_f32(src[e * sd]) : 0.f;
                sum += x[m] * x[m];
            }
            float scale = 1.f;
            if (a.l2norm) {
#pragma unroll
                for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
                scale = rsqrtf(sum + kL2Eps);
            }
#pragma unroll
            for (int m = 0; m < KP / 32; ++m) dst[lane + 32 * m] = x[m] * scale;
        }
        if ((int)threadIdx.x < n) {
            const int64_t t = tok0 + base + threadIdx.x;
            float g, beta;
            load_gates(a, g0 + t * a.g_st, b0 + t * a.b_st, h, g, beta);
            s_alpha[threadIdx.x] = expf(g);
            s_beta[threadIdx.x] = beta;
        }
        __syncthreads();
        for (int j = 0; j < n; ++j) {
            const int64_t t = tok0 + base + j;
            float kS[4] = {0.f, 0.f, 0.f, 0.f}, qS[4] = {0.f, 0.f, 0.f, 0.f}, qk = 0.f;
            float vv[4];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                vv[c] = c < valid ? to_f32(vp[t * a.v_st + (int64_t)(col + c) * a.v_sd]) : 0.f;
#pragma unroll
            for (int r = 0; r < RPT; r += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(&sk[j][r * 8 + rg * 4]);
                const float4 q4 = *reinterpret_cast<const float4*>(&sq[j][r * 8 + rg * 4]);
                const float kk[4] = {k4.x, k4.y, k4.z, k4.w}, qq[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    qk = fmaf(kk[e], qq[e], qk);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        kS[c] = fmaf(kk[e], S[r + e][c], kS[c]);
                        qS[c] = fmaf(qq[e], S[r + e][c], qS[c]);
                    }
                }
            }
#pragma unroll
            for (int o = 4; o < 32; o *= 2) {
                qk += __shfl_xor_sync(~0u, qk, o);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    kS[c] += __shfl_xor_sync(~0u, kS[c], o);
                    qS[c] += __shfl_xor_sync(~0u, qS[c], o);
                }
            }
            const float alpha = s_alpha[j], beta = s_beta[j];
            float u[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                u[c] = beta * (vv[c] - alpha * kS[c]);
                // Lane group c writes column c: four groups share the stores.
                if (rg == c && c < valid)
                    op[t * a.o_st + (int64_t)(col + c) * a.o_sd] =
                        from_f32<T>(a.scale * (alpha * qS[c] + qk * u[c]));
            }
#pragma unroll
            for (int r = 0; r < RPT; r += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(&sk[j][r * 8 + rg * 4]);
                const float kk[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        S[r + e][c] = fmaf(kk[e], u[c], alpha * S[r + e][c]);
            }
            if (islot >= 0 && valid > 0) {
                ST* ip = static_cast<ST*>(a.inter) + islot * a.i_slot + (base + j) * a.i_st +
                         h * a.i_sh + col;
#pragma unroll
                for (int r = 0; r < RPT; ++r) {
                    const int k = (r / 4) * 32 + rg * 4 + r % 4;
                    if (k < a.dk) store4(ip + k * a.i_sk, vec, valid, S[r]);
                }
            }
        }
    }

    if (st != nullptr && valid > 0 && (varlen || a.update_states)) {
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            const int k = (r / 4) * 32 + rg * 4 + r % 4;
            if (k < a.dk) store4(st + k * a.s_sk, vec, valid, S[r]);
        }
    }
}

// Whether every 4-column vector of the states is aligned and whole.
bool state_vec(const cc1d_gdr_args& a) {
    const int64_t e = a.sdtype == CC1D_F32 ? 4 : 2;
    auto ok = [&](const void* p, int64_t s0, int64_t s1, int64_t s2, int64_t s3) {
        return (uintptr_t)p % (4 * e) == 0 && s0 % 4 == 0 && s1 % 4 == 0 && s2 % 4 == 0 && s3 % 4 == 0;
    };
    return a.dv % 4 == 0 && ok(a.states, a.s_slot, a.s_sh, a.s_sk, 0) &&
           (a.inter == nullptr || ok(a.inter, a.i_slot, a.i_st, a.i_sh, a.i_sk));
}

template <typename T, typename ST>
cudaError_t launch(const cc1d_gdr_args& a, bool varlen, cudaStream_t stream) {
    constexpr int WARPS = 4;
    const int tiles = (int)ceil_div(a.dv, kWarpCols * WARPS);
    const int64_t grid = a.rows * a.heads_v * tiles;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    const bool vec = state_vec(a);
    if (a.dk <= 64)
        gdr_recurrent_kernel<T, ST, 8, WARPS><<<(unsigned)grid, 32 * WARPS, 0, stream>>>(a, varlen, vec, tiles);
    else if (a.dk <= 128)
        gdr_recurrent_kernel<T, ST, 16, WARPS><<<(unsigned)grid, 32 * WARPS, 0, stream>>>(a, varlen, vec, tiles);
    else
        gdr_recurrent_kernel<T, ST, 32, WARPS><<<(unsigned)grid, 32 * WARPS, 0, stream>>>(a, varlen, vec, tiles);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gdr_recurrent(const cc1d_gdr_args& a, bool varlen, cudaStream_t stream) {
    if (a.sdtype == CC1D_F32) {
        CC1D_DISPATCH_DTYPE(a.dtype, return launch<T, float>(a, varlen, stream));
    } else {
        CC1D_DISPATCH_DTYPE(a.dtype, return launch<T, T>(a, varlen, stream));
    }
    return cudaErrorInvalidValue;
}

}  // namespace cc1d
