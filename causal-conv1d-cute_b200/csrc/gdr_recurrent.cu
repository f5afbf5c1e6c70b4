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
// Layout. The columns of S are independent: a CTA owns 8 CPL columns (a 128-byte line of an fp32 or
// 16-bit state row) and all dk rows, one warp for every 32 rows. Eight lanes cover a row of the tile,
// four lane groups and 8 rows per lane the warp's rows; the reduction over dk is 8 FMAs per lane, two
// shuffles and one exchange through shared memory. Few registers per lane (32 or 64 of state) keep
// many CTAs resident, and all state loads of a thread are issued before the token's q and k are
// staged, so they overlap with the gate and norm arithmetic.
#include <algorithm>
#include <initializer_list>

#include "gdr.cuh"
#include "kernels.h"

namespace cc1d {
namespace {

constexpr int kMaxSteps = 16;
constexpr int kTokTile = 4;  // tokens staged in shared memory at a time
constexpr int kRows = 8;     // rows of the state per lane

// N adjacent values, as one vector where `vec` allows it; only the first `valid` of them exist.
template <int N, typename E>
__device__ __forceinline__ void load_n(const E* p, bool vec, int valid, float* f) {
    if (vec) {
        constexpr int NB = N * (int)sizeof(E) >= 16 ? 16 : 8;
#pragma unroll
        for (int i = 0; i < N; i += NB / (int)sizeof(E)) unpack_raw<E, NB>(ld_raw<NB>(p + i), f + i);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = i < valid ? to_f32(p[i]) : 0.f;
    }
}
template <int N, typename E>
__device__ __forceinline__ void store_n(E* p, bool vec, int valid, const float* f) {
    if (vec) {
        constexpr int NB = N * (int)sizeof(E) >= 16 ? 16 : 8;
#pragma unroll
        for (int i = 0; i < N; i += NB / (int)sizeof(E)) st_raw<NB>(p + i, pack_raw<E, NB>(f + i));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < valid) p[i] = from_f32<E>(f[i]);
    }
}

// NW: warps, 32 rows of the state each (dk <= 32 NW). CPL: columns per lane.
template <typename T, typename ST, int NW, int CPL>
__global__ void __launch_bounds__(32 * NW, NW == 4 ? 6 : 1)
gdr_recurrent_kernel(const __grid_constant__ cc1d_gdr_args a, bool varlen, bool svec, bool iovec,
                     int tiles, const int32_t* list) {
    constexpr int KP = 32 * NW, COLS = 8 * CPL;
    __shared__ __align__(16) float sq[kTokTile][KP], sk[kTokTile][KP];
    __shared__ __align__(16) float part[2][NW][2 * COLS];
    __shared__ float part_qk[2][NW], s_alpha[kTokTile], s_beta[kTokTile];

    const int tile = blockIdx.x % tiles;
    const int64_t rh = blockIdx.x / tiles;
    const int h = (int)(rh % a.heads_v);
    const int64_t row = rh / a.heads_v;
    const int hk = h / (a.heads_v / a.heads_k);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rg = lane / 8, cl = lane % 8 * CPL;
    const int col = tile * COLS + cl, first = warp * 32 + rg * kRows;
    const int valid = min(CPL, max(0, a.dv - col));
    svec = svec && valid == CPL;
    iovec = iovec && valid == CPL;

    int64_t tok0, slot;
    int ntok;
    if (!gdr_row(a, varlen, row, tok0, ntok, slot, h == 0 && tile == 0 && threadIdx.x == 0)) return;
    if (list != nullptr && ntok > list[1]) return;
    int64_t islot = -1;
    if (a.inter != nullptr) {
        islot = a.inter_indices != nullptr ? a.inter_indices[row] : slot;
        if (islot < 0 || islot >= a.inter_nslots) {
            if (h == 0 && tile == 0 && threadIdx.x == 0)
                flag_status(a.dev_status, CC1D_DEV_BAD_INTER_SLOT);
            islot = -1;
        }
    }

    float S[kRows][CPL];
    const bool initial = !varlen || (a.has_initial_state != nullptr && a.has_initial_state[row]);
    ST* st = nullptr;
    if (slot >= 0) st = static_cast<ST*>(a.states) + slot * a.s_slot + h * a.s_sh + first * a.s_sk + col;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (st != nullptr && initial && valid > 0 && first + r < a.dk) {
            load_n<CPL>(st + r * a.s_sk, svec, valid, S[r]);
        } else {
#pragma unroll
            for (int c = 0; c < CPL; ++c) S[r][c] = 0.f;
        }
    }

    const T* qp = static_cast<const T*>(a.q) + (varlen ? 0 : row * a.q_sb) + hk * a.q_sh;
    const T* kp = static_cast<const T*>(a.k) + (varlen ? 0 : row * a.k_sb) + hk * a.k_sh;
    const T* vp = static_cast<const T*>(a.v) + (varlen ? 0 : row * a.v_sb) + h * a.v_sh + col * a.v_sd;
    T* op = static_cast<T*>(a.out) + (varlen ? 0 : row * a.o_sb) + h * a.o_sh + col * a.o_sd;
    const int64_t g0 = (varlen ? 0 : row * a.g_sb) + h * a.g_sh;
    const int64_t b0 = (varlen ? 0 : row * a.b_sb) + h * a.b_sh;

    for (int base = 0; base < ntok; base += kTokTile) {
        const int n = min(kTokTile, ntok - base);
        if (base > 0) __syncthreads();
        for (int i = warp; i < 2 * n; i += NW) {
            const int64_t t = tok0 + base + i / 2;
            const T* src = i % 2 ? kp + t * a.k_st : qp + t * a.q_st;
            const int64_t sd = i % 2 ? a.k_sd : a.q_sd;
            float* dst = i % 2 ? sk[i / 2] : sq[i / 2];
            float x[NW], sum = 0.f;
#pragma unroll
            for (int m = 0; m < NW; ++m) {
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
            for (int m = 0; m < NW; ++m) dst[lane + 32 * m] = x[m] * scale;
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
            float v[CPL];
            if (iovec) {
                load_n<CPL>(vp + t * a.v_st, true, CPL, v);
            } else {
#pragma unroll
                for (int c = 0; c < CPL; ++c) v[c] = c < valid ? to_f32(vp[t * a.v_st + c * a.v_sd]) : 0.f;
            }
            float kk[kRows], kS[CPL], qS[CPL], qk = 0.f;
#pragma unroll
            for (int c = 0; c < CPL; ++c) kS[c] = qS[c] = 0.f;
#pragma unroll
            for (int r = 0; r < kRows; r += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(&sk[j][first + r]);
                const float4 q4 = *reinterpret_cast<const float4*>(&sq[j][first + r]);
                const float qq[4] = {q4.x, q4.y, q4.z, q4.w};
                kk[r] = k4.x;
                kk[r + 1] = k4.y;
                kk[r + 2] = k4.z;
                kk[r + 3] = k4.w;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    qk = fmaf(kk[r + e], qq[e], qk);
#pragma unroll
                    for (int c = 0; c < CPL; ++c) {
                        kS[c] = fmaf(kk[r + e], S[r + e][c], kS[c]);
                        qS[c] = fmaf(qq[e], S[r + e][c], qS[c]);
                    }
                }
            }
#pragma unroll
            for (int o = 8; o < 32; o *= 2) {
                qk += __shfl_xor_sync(~0u, qk, o);
#pragma unroll
                for (int c = 0; c < CPL; ++c) {
                    kS[c] += __shfl_xor_sync(~0u, kS[c], o);
                    qS[c] += __shfl_xor_sync(~0u, qS[c], o);
                }
            }
            if constexpr (NW > 1) {
                // Sums over the warps, always in the same order; two buffers, one barrier a token.
                float (*pp)[2 * COLS] = part[j % 2];
                if (rg == 0) {
#pragma unroll
                    for (int c = 0; c < CPL; c += 4) {
                        *reinterpret_cast<float4*>(&pp[warp][cl + c]) = make_float4(kS[c], kS[c + 1], kS[c + 2], kS[c + 3]);
                        *reinterpret_cast<float4*>(&pp[warp][COLS + cl + c]) = make_float4(qS[c], qS[c + 1], qS[c + 2], qS[c + 3]);
                    }
                    if (lane == 0) part_qk[j % 2][warp] = qk;
                }
                __syncthreads();
                qk = 0.f;
#pragma unroll
                for (int c = 0; c < CPL; ++c) kS[c] = qS[c] = 0.f;
#pragma unroll
                for (int m = 0; m < NW; ++m) {
                    qk += part_qk[j % 2][m];
#pragma unroll
                    for (int c = 0; c < CPL; c += 4) {
                        const float4 k4 = *reinterpret_cast<const float4*>(&pp[m][cl + c]);
                        const float4 q4 = *reinterpret_cast<const float4*>(&pp[m][COLS + cl + c]);
                        kS[c] += k4.x, kS[c + 1] += k4.y, kS[c + 2] += k4.z, kS[c + 3] += k4.w;
                        qS[c] += q4.x, qS[c + 1] += q4.y, qS[c + 2] += q4.z, qS[c + 3] += q4.w;
                    }
                }
            }
            const float alpha = s_alpha[j], beta = s_beta[j];
            float u[CPL];
#pragma unroll
            for (int c = 0; c < CPL; ++c) u[c] = beta * (v[c] - alpha * kS[c]);
            if (warp == j % NW && rg == 0) {
                float o[CPL];
#pragma unroll
                for (int c = 0; c < CPL; ++c) o[c] = a.scale * (alpha * qS[c] + qk * u[c]);
                if (iovec) {
                    store_n<CPL>(op + t * a.o_st, true, CPL, o);
                } else {
#pragma unroll
                    for (int c = 0; c < CPL; ++c)
                        if (c < valid) op[t * a.o_st + c * a.o_sd] = from_f32<T>(o[c]);
                }
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
                for (int c = 0; c < CPL; ++c) S[r][c] = fmaf(kk[r], u[c], alpha * S[r][c]);
            if (islot >= 0 && valid > 0) {
                ST* ip = static_cast<ST*>(a.inter) + islot * a.i_slot + (base + j) * a.i_st +
                         h * a.i_sh + first * a.i_sk + col;
#pragma unroll
                for (int r = 0; r < kRows; ++r)
                    if (first + r < a.dk) store_n<CPL>(ip + r * a.i_sk, svec, valid, S[r]);
            }
        }
    }

    if (st != nullptr && valid > 0 && (varlen || a.update_states)) {
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            if (first + r < a.dk) store_n<CPL>(st + r * a.s_sk, svec, valid, S[r]);
    }
}

// Decode of whole heads, dk = 128 and tiles of 128 columns: a CTA of 8 warps has a (128, 128) state
// tile in registers, 16 rows and 4 columns per lane, so that a warp's access is one whole row and
// the norms, gates and the reduction are done once for the tile. Two CTAs of 64 KB per SM are in
// flight, and the stores are evict-first: a step's states are next read a whole model later.
// Measured at 256 rows x 48 heads, fp32: 274 us, 5.9 TB/s of 6.4 (plain stores 293 us; 16 warps of 8
// rows 300 us, the same with three CTAs an SM, which spills, 538 us).
template <typename T, typename ST>
__global__ void __launch_bounds__(256, 2)
gdr_decode_kernel(const __grid_constant__ cc1d_gdr_args a, int tiles) {
    constexpr int NB = 4 * (int)sizeof(ST), ROWS = 16, WARPS = 128 / ROWS, THREADS = 32 * WARPS;
    __shared__ __align__(16) float sq[kMaxSteps][128], sk[kMaxSteps][128];
    __shared__ __align__(16) float part[2][WARPS][128], total[2][128];
    __shared__ float s_qk[kMaxSteps], s_alpha[kMaxSteps], s_beta[kMaxSteps];

    const int tile = blockIdx.x % tiles;
    const int64_t rh = blockIdx.x / tiles;
    const int h = (int)(rh % a.heads_v);
    const int64_t row = rh / a.heads_v;
    const int hk = h / (a.heads_v / a.heads_k);
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int col = tile * 128 + lane * 4, first = warp * ROWS;

    int64_t tok0, slot;
    int steps;
    if (!gdr_row(a, false, row, tok0, steps, slot, h == 0 && tile == 0 && tid == 0)) return;
    int64_t islot = -1;
    if (a.inter != nullptr) {
        islot = a.inter_indices != nullptr ? a.inter_indices[row] : slot;
        if (islot < 0 || islot >= a.inter_nslots) {
            if (h == 0 && tile == 0 && tid == 0) flag_status(a.dev_status, CC1D_DEV_BAD_INTER_SLOT);
            islot = -1;
        }
    }
    ST* st = static_cast<ST*>(a.states) + slot * a.s_slot + h * a.s_sh + first * a.s_sk + col;
    typename RawVec<NB>::type raw[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) raw[r] = ld_raw<NB>(st + r * a.s_sk);

    // Queries and keys of all steps, one vector per warp in turn; gates by the warps behind.
    for (int i = warp; i < 2 * steps; i += WARPS) {
        const int t = i / 2;
        const T* src = i % 2 ? static_cast<const T*>(a.k) + row * a.k_sb + hk * a.k_sh + t * a.k_st
                             : static_cast<const T*>(a.q) + row * a.q_sb + hk * a.q_sh + t * a.q_st;
        const int64_t sd = i % 2 ? a.k_sd : a.q_sd;
        float x[4], sum = 0.f;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            x[m] = to_f32(src[(lane + 32 * m) * sd]);
            sum += x[m] * x[m];
        }
        float scale = 1.f;
        if (a.l2norm) {
#pragma unroll
            for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
            scale = rsqrtf(sum + kL2Eps);
        }
        float* dst = i % 2 ? sk[t] : sq[t];
#pragma unroll
        for (int m = 0; m < 4; ++m) dst[lane + 32 * m] = x[m] * scale;
    }
    if (tid >= THREADS - steps) {
        const int t = tid - (THREADS - steps);
        float g, beta;
        load_gates(a, row * a.g_sb + t * a.g_st + h * a.g_sh, row * a.b_sb + t * a.b_st + h * a.b_sh, h, g, beta);
        s_alpha[t] = expf(g);
        s_beta[t] = beta;
    }
    const T* vp = static_cast<const T*>(a.v) + row * a.v_sb + h * a.v_sh + col * a.v_sd;
    T* op = static_cast<T*>(a.out) + row * a.o_sb + h * a.o_sh + col * a.o_sd;
    float2 S[ROWS][2];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) unpack_raw<ST, NB>(raw[r], &S[r][0].x);
    __syncthreads();
    for (int t = warp; t < steps; t += WARPS) {
        float qk = 0.f;
#pragma unroll
        for (int m = 0; m < 4; ++m) qk = fmaf(sq[t][lane + 32 * m], sk[t][lane + 32 * m], qk);
#pragma unroll
        for (int o = 16; o > 0; o /= 2) qk += __shfl_xor_sync(~0u, qk, o);
        if (lane == 0) s_qk[t] = qk;
    }

    for (int t = 0; t < steps; ++t) {
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = to_f32(vp[t * a.v_st + c * a.v_sd]);
        float2 kS[2] = {}, qS[2] = {};
#pragma unroll
        for (int r = 0; r < ROWS; r += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(&sk[t][first + r]);
            const float4 q4 = *reinterpret_cast<const float4*>(&sq[t][first + r]);
            const float kk[4] = {k4.x, k4.y, k4.z, k4.w}, qq[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    kS[c] = __ffma2_rn(make_float2(kk[e], kk[e]), S[r + e][c], kS[c]);
                    qS[c] = __ffma2_rn(make_float2(qq[e], qq[e]), S[r + e][c], qS[c]);
                }
        }
        *reinterpret_cast<float4*>(&part[0][warp][lane * 4]) = make_float4(kS[0].x, kS[0].y, kS[1].x, kS[1].y);
        *reinterpret_cast<float4*>(&part[1][warp][lane * 4]) = make_float4(qS[0].x, qS[0].y, qS[1].x, qS[1].y);
        __syncthreads();
        {
            // One column of S^T k or S^T q per thread, summed over the warps in order.
            const float (*p)[128] = part[tid / 128];
            float sum = 0.f;
#pragma unroll
            for (int m = 0; m < WARPS; ++m) sum += p[m][tid % 128];
            total[tid / 128][tid % 128] = sum;
        }
        __syncthreads();
        const float4 k4 = *reinterpret_cast<const float4*>(&total[0][lane * 4]);
        const float alpha = s_alpha[t], beta = s_beta[t];
        const float u[4] = {beta * (v[0] - alpha * k4.x), beta * (v[1] - alpha * k4.y),
                            beta * (v[2] - alpha * k4.z), beta * (v[3] - alpha * k4.w)};
        if (warp == t % WARPS) {
            const float4 q4 = *reinterpret_cast<const float4*>(&total[1][lane * 4]);
            const float q[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                op[t * a.o_st + c * a.o_sd] = from_f32<T>(a.scale * (alpha * q[c] + s_qk[t] * u[c]));
        }
        const float2 u2[2] = {make_float2(u[0], u[1]), make_float2(u[2], u[3])};
#pragma unroll
        for (int r = 0; r < ROWS; r += 4) {
            const float4 kk4 = *reinterpret_cast<const float4*>(&sk[t][first + r]);
            const float kk[4] = {kk4.x, kk4.y, kk4.z, kk4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    S[r + e][c] = __ffma2_rn(make_float2(kk[e], kk[e]), u2[c],
                                             __fmul2_rn(make_float2(alpha, alpha), S[r + e][c]));
        }
        if (islot >= 0) {
            ST* ip = static_cast<ST*>(a.inter) + islot * a.i_slot + t * a.i_st + h * a.i_sh + first * a.i_sk + col;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) st_stream_raw<NB>(ip + r * a.i_sk, pack_raw<ST, NB>(&S[r][0].x));
        }
    }
    if (a.update_states) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) st_stream_raw<NB>(st + r * a.s_sk, pack_raw<ST, NB>(&S[r][0].x));
    }
}

// Whether every N-element vector of a tensor with these strides is aligned and whole.
bool vec_ok(const void* p, int64_t bytes, int64_t n, std::initializer_list<int64_t> strides) {
    bool ok = (uintptr_t)p % std::min<int64_t>(16, bytes * n) == 0;
    for (int64_t s : strides) ok = ok && s % n == 0;
    return ok;
}

template <typename T, typename ST>
cudaError_t launch(const cc1d_gdr_args& a, bool varlen, cudaStream_t stream, const int32_t* list) {
    constexpr int CPL = 4;
    const int tiles = (int)ceil_div(a.dv, 8 * CPL);
    const int64_t grid = a.rows * a.heads_v * tiles;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    const int64_t eb = sizeof(ST), ib = sizeof(T);
    const bool svec = vec_ok(a.states, eb, CPL, {a.s_slot, a.s_sh, a.s_sk}) &&
                      (a.inter == nullptr || vec_ok(a.inter, eb, CPL, {a.i_slot, a.i_st, a.i_sh, a.i_sk}));
    const bool iovec = a.v_sd == 1 && a.o_sd == 1 &&
                       vec_ok(a.v, ib, CPL, {varlen ? 0 : a.v_sb, a.v_st, a.v_sh}) &&
                       vec_ok(a.out, ib, CPL, {varlen ? 0 : a.o_sb, a.o_st, a.o_sh});
    // Whole heads where the shape allows it (one step, fp32: 12288 heads 274 us against 371 us in
    // tiles of 32 columns, 6 heads 5.3 against 5.0). Recorded fp32 states are the exception with few
    // heads: their stores are bound by the SM, and four CTAs a head spread them over more SMs (4
    // steps, 6 heads 8.7 against 11.8 us, 384 heads 36 against 41 us, 768 heads 67 against 66 us).
    const int64_t heads = a.rows * a.heads_v * (a.dv / 128);
    const bool spread = a.inter != nullptr && sizeof(ST) == 4 && heads < 5 * 148;
    if (!varlen && !spread && a.dk == 128 && a.dv % 128 == 0 && a.steps <= kMaxSteps &&
        heads <= INT32_MAX && vec_ok(a.states, eb, 4, {a.s_slot, a.s_sh, a.s_sk}) &&
        (a.inter == nullptr || vec_ok(a.inter, eb, 4, {a.i_slot, a.i_st, a.i_sh, a.i_sk}))) {
        gdr_decode_kernel<T, ST><<<(unsigned)heads, 256, 0, stream>>>(a, a.dv / 128);
        return cudaGetLastError();
    }
    auto go = [&](auto nw) {
        constexpr int NW = decltype(nw)::value;
        gdr_recurrent_kernel<T, ST, NW, CPL>
            <<<(unsigned)grid, 32 * NW, 0, stream>>>(a, varlen, svec, iovec, tiles, list);
    };
    if (a.dk <= 32)
        go(std::integral_constant<int, 1>());
    else if (a.dk <= 64)
        go(std::integral_constant<int, 2>());
    else if (a.dk <= 128)
        go(std::integral_constant<int, 4>());
    else
        go(std::integral_constant<int, 8>());
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gdr_recurrent(const cc1d_gdr_args& a, bool varlen, cudaStream_t stream,
                                 const int32_t* list) {
    if (a.sdtype == CC1D_F32) {
        CC1D_DISPATCH_DTYPE(a.dtype, return launch<T, float>(a, varlen, stream, list));
    } else {
        CC1D_DISPATCH_DTYPE(a.dtype, return launch<T, T>(a, varlen, stream, list));
    }
    return cudaErrorInvalidValue;
}

}  // namespace cc1d
