// Gated delta rule over packed sequences, chunk by chunk on the tensor cores (bf16, dk = 128).
//
// Mathematics. In a chunk of C = 64 tokens that starts from state S0, with b the cumulative log
// decay inside the chunk, r the inverse norms of the keys (1 without l2norm) and s those of the
// queries times the output scale:
//     L_ij = beta_i r_i r_j e^(b_i - b_j) k_i.k_j   (j < i),   T = (I + L)^-1 diag(beta)
//     P_ij = s_i r_j e^(b_i - b_j) q_i.k_j          (j <= i),  G = P T
//     R_i  = v_i - r_i e^(b_i) S0^T k_i
//     u    = T R,      o_i = s_i e^(b_i) S0^T q_i + (G R)_i
//     S    = e^(b_C) S0 + sum_j k_j (r_j e^(b_C - b_j) u_j)^T.
// k and q enter every product as the caller's bf16 values, which are exact; norms, gates and
// decays scale rows in fp32 outside the products. All exponents are differences b_i - b_j <= 0.
//
// Precision. S, R, T, G and u are fp32 quantities. As operands they are split into two bf16 parts
// (2^-17), and the products keep hi*hi + hi*lo + lo*hi, so that fp32 final states are good to about
// 1e-5 where a single bf16 rounding would leave 2e-3. The state itself stays in fp32 registers.
//
// Split of the work. Chunks of one sequence form a chain; heads, sequences and tiles of VS state
// columns are independent and are the grid. A CTA has two warpgroups:
//   - prep: loads K, Q and V of the next chunk (cp.async, zeros behind the sequence's end), forms
//     [K;Q] K^T on the tensor core, L, its inverse by forward substitution, T and G = P T. Nothing
//     of it depends on the state, so it runs a chunk ahead of the chain.
//   - scan: the chain. [K;Q] S0 (one M = 128 product), R, [T;G] R (another), u, K^T u, S.
// Stacking K over Q and T over G makes every product M = 128, the full tensor core rate.
#include <algorithm>

#include "gdr.cuh"
#include "kernels.h"
#include "tc05.cuh"

namespace cc1d {
namespace {

constexpr int C = 64;        // tokens per chunk
constexpr int DK = 128;      // key head dim
constexpr int LPAD = 68;     // fp32 row of L in shared memory: 16-byte stores of 8 rows hit 8 bank groups
constexpr int kOrderMax = 256;  // batches up to this many sequences start with the longest

template <int VS>
struct Layout {
    static constexpr int kRow = VS >= 64 ? 128 : 2 * VS;          // bytes of an operand row of V columns
    static constexpr int kS = 128 * VS * 2;                       // one part (hi or lo) of S
    static constexpr int kR = C * VS * 2;                         // one part of R or u
    static constexpr int KQ = 0;                                  // 2 stages x [2 halves][128 rows][128 B]
    static constexpr int V = KQ + 2 * 32768;                      // 2 stages x [64 rows][VS]
    static constexpr int TG = V + 2 * kR;                         // [hi, lo][128 rows][128 B]
    static constexpr int SB = TG + 32768;                         // S hi, S lo; R in S hi, u in S lo
    static constexpr int L = SB + 2 * kS;                         // fp32 [64][LPAD]
    static constexpr int VEC = L + C * LPAD * 4;                  // 2 stages x Vectors
    static constexpr int END = VEC + 2 * 1040;
};

struct Vectors {     // per chunk: what the scan multiplies rows by
    float in[2 * C];  // r_i e^(b_i) (rows of K), s_i e^(b_i) (rows of Q)
    float out[C];     // r_j e^(b_C - b_j)
    float decay;      // e^(b_C)
};
static_assert(sizeof(Vectors) <= 1040, "");

struct Shared {
    uint64_t kq_full[2], kq_free[2], vec_full[2], tg_full, tg_free, prep_mma, m1, m2, m3;
    uint32_t tmem;
    int abort;
    int row;  // sequence of this CTA
    int len[kOrderMax];
    float bh[C], bl[C], rk[C], beta[C];
    double half;
};

// Row r, 16-byte unit u of an operand image of `row`-byte rows.
template <int ROW>
__device__ __forceinline__ uint32_t swz(int r, int u) {
    if constexpr (ROW == 128) {
        return r * 128 + ((u ^ (r & 7)) << 4);
    } else {
        return r * 64 + ((u ^ ((r >> 1) & 3)) << 4);
    }
}
// The same for a row of VS columns: 128-byte atoms of 64 columns lie `rows` rows apart.
template <int VS>
__device__ __forceinline__ uint32_t swz_cols(int rows, int r, int u) {
    if constexpr (VS >= 64) {
        return (u >> 3) * rows * 128 + swz<128>(r, u & 7);
    } else {
        return swz<64>(r, u);
    }
}

// 32 values of row r, columns 32 g.., as two bf16 parts into an MN-major operand image.
template <int VS>
__device__ __forceinline__ void store_split(uint32_t hi_base, uint32_t lo_base, int rows, int r,
                                            int g, const float* f) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split2(f[u * 8 + 2 * i], f[u * 8 + 2 * i + 1], h[i], l[i]);
        const uint32_t at = swz_cols<VS>(rows, r, g * 4 + u);
        sts16(hi_base + at, h[0], h[1], h[2], h[3]);
        sts16(lo_base + at, l[0], l[1], l[2], l[3]);
    }
}

template <typename ST, int VS>
__global__ void __launch_bounds__(256, 1)
gdr_chunk_kernel(const __grid_constant__ cc1d_gdr_args a, int tiles, bool out32) {
    using Lay = Layout<VS>;
    constexpr int kTmemCols = VS == 32 ? 256 : 512;
    constexpr uint64_t kSwz = VS >= 64 ? kSwizzle128 : kSwizzle64;
    constexpr uint32_t kGroup = 8 * Lay::kRow;  // bytes of eight rows of V columns
    extern __shared__ __align__(1024) unsigned char raw[];
    __shared__ Shared sh;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    Vectors* vec = reinterpret_cast<Vectors*>(raw + (base - smem_addr(raw)) + Lay::VEC);
    float* Lsm = reinterpret_cast<float*>(raw + (base - smem_addr(raw)) + Lay::L);

    const int tid = threadIdx.x, warp = tid / 32, p = tid % 128;
    const int vt = blockIdx.x % tiles;
    const int h = (int)((blockIdx.x / tiles) % a.heads_v);
    int64_t row = blockIdx.x / tiles / a.heads_v;
    const int hk = h / (a.heads_v / a.heads_k);

    // Longest sequences first, so that the last CTAs to start are short. Ties go by index.
    if (a.rows > 1 && a.rows <= kOrderMax) {
        const int n = (int)a.rows;
        if (tid < n) sh.len[tid] = a.query_start_loc[tid + 1] - a.query_start_loc[tid];
        __syncthreads();
        if (tid < n) {
            int rank = 0;
            for (int i = 0; i < n; ++i)
                rank += sh.len[i] > sh.len[tid] || (sh.len[i] == sh.len[tid] && i < tid);
            if (rank == row) sh.row = tid;
        }
        __syncthreads();
        row = sh.row;
    }
    int64_t tok0, slot;
    int ntok;
    if (!gdr_row(a, true, row, tok0, ntok, slot, h == 0 && vt == 0 && tid == 0)) return;
    const int chunks = (ntok + C - 1) / C;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&sh.kq_full[i]), 1);
            mbar_init(smem_addr(&sh.kq_free[i]), 3);  // the last product, and two warps of the scan
            mbar_init(smem_addr(&sh.vec_full[i]), 1);
        }
        for (uint64_t* b : {&sh.tg_full, &sh.tg_free, &sh.prep_mma, &sh.m1, &sh.m2, &sh.m3})
            mbar_init(smem_addr(b), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.abort = 0;
    }
    if (warp == 0) {
        tmem_alloc(smem_addr(&sh.tmem), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t D0 = tmem, DG = tmem + 64, D1 = tmem + 128, D2 = D1 + VS, D3 = D2 + VS;
    const uint32_t lanes = (uint32_t)(warp % 4) << 21;  // the warp's first TMEM lane, in bits 16..

    if (warp >= 4) {
        // -------------------------------------------------------------------------------- prep
        const bf16* qp = static_cast<const bf16*>(a.q) + tok0 * a.q_st + hk * a.q_sh;
        const bf16* kp = static_cast<const bf16*>(a.k) + tok0 * a.k_st + hk * a.k_sh;
        const bf16* vp = static_cast<const bf16*>(a.v) + tok0 * a.v_st + h * a.v_sh + vt * VS;
        const int64_t g0 = tok0 * a.g_st + h * a.g_sh, b0 = tok0 * a.b_st + h * a.b_sh;

        auto load = [&](int c) {
            const uint32_t kq = base + Lay::KQ + (c & 1) * 32768;
            const int left = ntok - c * C;
#pragma unroll 4
            for (int i = p; i < 2 * C * 16; i += 128) {
                const int r = i / 16, u = i % 16, t = r % C;
                const bool in = t < left;
                const int64_t at = c * C + (in ? t : 0);
                const bf16* src = (r < C ? kp + at * a.k_st : qp + at * a.q_st) + u * 8;
                const uint32_t dst = kq + (u >> 3) * 16384 + swz<128>(r, u & 7);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                             "r"(in ? 16 : 0)
                             : "memory");
            }
            const uint32_t vb = base + Lay::V + (c & 1) * Lay::kR;
#pragma unroll 4
            for (int i = p; i < C * (VS / 8); i += 128) {
                const int r = i / (VS / 8), u = i % (VS / 8);
                const bool in = r < left;
                const bf16* src = vp + (c * C + (in ? r : 0)) * a.v_st + u * 8;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                 vb + swz_cols<VS>(C, r, u)),
                             "l"(src), "r"(in ? 16 : 0)
                             : "memory");
            }
            cp_async_commit();
        };

        load(0);
        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1;
            const uint32_t kq = base + Lay::KQ + st * 32768;
            cp_async_wait<0>();
            fence_async_smem();
            named_sync(1, 128);
            if (p == 0) {
                mbar_arrive(smem_addr(&sh.kq_full[st]));
                tc_fence_after();
                // D0 = [K;Q] K^T
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint32_t at = kq + (ks >> 2) * 16384 + (ks & 3) * 32;
                    mma_bf16(D0, operand(at, 16, 1024, kSwizzle128), operand(at, 16, 1024, kSwizzle128),
                             mma_desc(64, false, false), ks > 0);
                }
                mma_commit(smem_addr(&sh.prep_mma));
            }
            // While it runs: gates and cumulative decays (threads of K rows), query norms (Q rows).
            float sq = a.scale;
            double total = 0;
            if (p < C) {
                float g = 0.f, beta = 0.f;
                if (c * C + p < ntok)
                    load_gates(a, g0 + (int64_t)(c * C + p) * a.g_st, b0 + (int64_t)(c * C + p) * a.b_st,
                               h, g, beta);
                // -1e5 decays anything to zero, and its sums stay finite where -inf would give
                // inf - inf below.
                g = g < -1e5f ? -1e5f : g;
                // The sums are carried in 64 bits and kept as two fp32 parts: their differences
                // are exponents, where fp32 sums of strong decays would lose the weak ones.
                total = (double)g * 1.4426950408889634;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const double below = __shfl_up_sync(~0u, total, o);
                    if (p % 32 >= o) total += below;
                }
                if (p == 31) sh.half = total;
                sh.beta[p] = beta;
            } else if (a.l2norm) {
                float sum = 0.f;
#pragma unroll 4
                for (int u = 0; u < 16; ++u) {
                    float f[8];
                    unpack16<bf16>(lds16(kq + (u >> 3) * 16384 + swz<128>(p, u & 7)), f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum = fmaf(f[i], f[i], sum);
                }
                sq *= rsqrtf(sum + kL2Eps);
            }
            named_sync(1, 128);
            if (p < C) {
                if (p >= 32) total += sh.half;
                const float hi = (float)total;
                sh.bh[p] = hi;
                sh.bl[p] = (float)(total - (double)hi);
            }
            mbar_wait(smem_addr(&sh.prep_mma), 0, &sh.abort);
            tc_fence_after();
            float x[C];
            tmem_ld32(D0 + lanes, x);
            tmem_ld32(D0 + lanes + 32, x + 32);
            const int i = p % C;
            if (p < C) {
                float d = 0.f;
#pragma unroll
                for (int j = 0; j < C; ++j) d = j == p ? x[j] : d;
                sh.rk[p] = a.l2norm ? rsqrtf(d + kL2Eps) : 1.f;
            }
            named_sync(1, 128);
            {
                const float bh = sh.bh[i], bl = sh.bl[i];
                const float mul = p < C ? sh.beta[i] * sh.rk[i] : sq;
                const int last = p < C ? i - 1 : i;
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    const float e = exp2_approx((bh - sh.bh[j]) + (bl - sh.bl[j]));
                    x[j] = j <= last ? x[j] * (mul * sh.rk[j] * e) : 0.f;
                }
                const float grow = exp2_approx(bh + bl);
                vec[st].in[p] = grow * (p < C ? sh.rk[i] : sq);
                if (p < C) {
                    vec[st].out[i] = sh.rk[i] * exp2_approx((sh.bh[C - 1] - bh) + (sh.bl[C - 1] - bl));
                    if (i == C - 1) vec[st].decay = grow;
                    // L row by row, for the substitution.
#pragma unroll
                    for (int j = 0; j < C; j += 4)
                        *reinterpret_cast<float4*>(&Lsm[i * LPAD + j]) =
                            make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                }
            }
            named_sync(1, 128);
            if (p == 0) mbar_arrive(smem_addr(&sh.vec_full[st]));
            if (p < C) {
                // Column p of (I + L)^-1 by forward substitution: x_i = [i = p] - sum_m L_im x_m.
#pragma unroll
                for (int r = 0; r < C; ++r) {
                    float s0 = r == p ? 1.f : 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
                    for (int m = 0; m < r; m += 4) {
                        const float4 l = *reinterpret_cast<const float4*>(&Lsm[r * LPAD + m]);
                        s0 = fmaf(-l.x, x[m], s0);
                        if (m + 1 < r) s1 = fmaf(-l.y, x[m + 1], s1);
                        if (m + 2 < r) s2 = fmaf(-l.z, x[m + 2], s2);
                        if (m + 3 < r) s3 = fmaf(-l.w, x[m + 3], s3);
                    }
                    x[r] = (s0 + s1) + (s2 + s3);
                }
            }
            // The chain's product with the previous chunk's T and G must be done with their memory.
            if (c > 0) mbar_wait(smem_addr(&sh.tg_free), (c - 1) & 1, &sh.abort);
            const uint32_t tg = base + Lay::TG;
            if (p < C) {
                const float beta = sh.beta[p];
#pragma unroll
                for (int r = 0; r < C; r += 2) {
                    uint32_t hi, lo;
                    split2(x[r] * beta, x[r + 1] * beta, hi, lo);
                    const uint32_t at0 = tg + swz<128>(r, p >> 3) + (p & 7) * 2;
                    const uint32_t at1 = tg + swz<128>(r + 1, p >> 3) + (p & 7) * 2;
                    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at0), "h"((uint16_t)hi) : "memory");
                    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at1), "h"((uint16_t)(hi >> 16)) : "memory");
                    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at0 + 16384), "h"((uint16_t)lo) : "memory");
                    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at1 + 16384), "h"((uint16_t)(lo >> 16)) : "memory");
                }
            } else {
                store_split<64>(tg, tg + 16384, 128, p, 0, x);
                store_split<64>(tg, tg + 16384, 128, p, 1, x + 32);
            }
            fence_async_smem();
            tc_fence_before();
            named_sync(1, 128);
            if (p == 0) {
                tc_fence_after();
                // DG = [T;P] T, of which the lower half is G.
#pragma unroll
                for (int part = 0; part < 3; ++part) {
                    const uint32_t A = tg + (part == 2 ? 16384 : 0), B = tg + (part == 1 ? 16384 : 0);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        mma_bf16(DG, operand(A + ks * 32, 16, 1024, kSwizzle128),
                                 operand(B + ks * 2048, 16, 1024, kSwizzle128),
                                 mma_desc(64, false, true), part + ks > 0);
                }
                mma_commit(smem_addr(&sh.prep_mma));
            }
            if (c + 1 < chunks) {
                if (c > 0) mbar_wait(smem_addr(&sh.kq_free[(c + 1) & 1]), ((c - 1) >> 1) & 1, &sh.abort);
                load(c + 1);
            }
            mbar_wait(smem_addr(&sh.prep_mma), 1, &sh.abort);
            tc_fence_after();
            if (p >= C) {
                tmem_ld32(DG + lanes, x);
                store_split<64>(tg, tg + 16384, 128, p, 0, x);
                tmem_ld32(DG + lanes + 32, x);
                store_split<64>(tg, tg + 16384, 128, p, 1, x);
            }
            fence_async_smem();
            tc_fence_before();
            named_sync(1, 128);
            if (p == 0) mbar_arrive(smem_addr(&sh.tg_full));
        }
    } else {
        // -------------------------------------------------------------------------------- scan
        const uint32_t s_hi = base + Lay::SB, s_lo = s_hi + Lay::kS;
        const uint32_t r_hi = s_hi, r_lo = s_hi + Lay::kR, u_hi = s_lo, u_lo = s_lo + Lay::kR;
        const uint32_t tg = base + Lay::TG;
        const bool initial = a.states != nullptr && a.has_initial_state != nullptr && a.has_initial_state[row];
        ST* sp = nullptr;
        if (a.states != nullptr)
            sp = static_cast<ST*>(a.states) + slot * a.s_slot + h * a.s_sh + p * a.s_sk + vt * VS;
        float S[VS];  // row p of the state
        constexpr int SV = Vec<ST>::V;
#pragma unroll
        for (int j = 0; j < VS; j += SV) {
            if (initial) {
                unpack16<ST>(ld16(sp + j), S + j);
            } else {
#pragma unroll
                for (int e = 0; e < SV; ++e) S[j + e] = 0.f;
            }
        }
        bf16* op = static_cast<bf16*>(a.out) + tok0 * a.o_st + h * a.o_sh + vt * VS;

        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1;
            const uint32_t kq = base + Lay::KQ + st * 32768;
#pragma unroll
            for (int g = 0; g < VS / 32; ++g) store_split<VS>(s_hi, s_lo, 128, p, g, S + 32 * g);
            fence_async_smem();
            tc_fence_before();
            named_sync(2, 128);
            if (tid == 0) {
                mbar_wait(smem_addr(&sh.kq_full[st]), (c >> 1) & 1, &sh.abort);
                tc_fence_after();
                // D1 = [K;Q] S
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        mma_bf16(D1,
                                 operand(kq + (ks >> 2) * 16384 + (ks & 3) * 32, 16, 1024, kSwizzle128),
                                 operand((part ? s_lo : s_hi) + ks * 2 * kGroup, 128 * 128, kGroup, kSwz),
                                 mma_desc(VS, false, true), part + ks > 0);
                mma_commit(smem_addr(&sh.m1));
            }
            mbar_wait(smem_addr(&sh.vec_full[st]), (c >> 1) & 1, &sh.abort);
            const float in = vec[st].in[p], decay = vec[st].decay;
            const float grow = vec[st].out[p % C];
            if (p >= C) {
                __syncwarp();
                if (p % 32 == 0) mbar_arrive(smem_addr(&sh.kq_free[st]));
            }
            if (p < C) {
                // R = V - r e^b (K S)
                mbar_wait(smem_addr(&sh.m1), c & 1, &sh.abort);
                tc_fence_after();
                const uint32_t vb = base + Lay::V + st * Lay::kR;
#pragma unroll
                for (int g = 0; g < VS / 32; ++g) {
                    float d[32];
                    tmem_ld32(D1 + lanes + 32 * g, d);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        float f[8];
                        unpack16<bf16>(lds16(vb + swz_cols<VS>(C, p, g * 4 + u)), f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) d[u * 8 + e] = fmaf(-in, d[u * 8 + e], f[e]);
                    }
                    store_split<VS>(r_hi, r_lo, C, p, g, d);
                }
                fence_async_smem();
                tc_fence_before();
                named_sync(3, 64);
                if (tid == 0) {
                    mbar_wait(smem_addr(&sh.tg_full), c & 1, &sh.abort);
                    tc_fence_after();
                    // D2 = [T;G] R
#pragma unroll
                    for (int part = 0; part < 3; ++part)
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            mma_bf16(D2, operand(tg + (part == 2 ? 16384 : 0) + ks * 32, 16, 1024, kSwizzle128),
                                     operand((part == 1 ? r_lo : r_hi) + ks * 2 * kGroup, C * 128, kGroup, kSwz),
                                     mma_desc(VS, false, true), part + ks > 0);
                    mma_commit(smem_addr(&sh.m2));
                    mma_commit(smem_addr(&sh.tg_free));
                }
                mbar_wait(smem_addr(&sh.m2), c & 1, &sh.abort);
                tc_fence_after();
#pragma unroll
                for (int g = 0; g < VS / 32; ++g) {
                    float d[32];
                    tmem_ld32(D2 + lanes + 32 * g, d);
#pragma unroll
                    for (int e = 0; e < 32; ++e) d[e] *= grow;
                    store_split<VS>(u_hi, u_lo, C, p, g, d);
                }
                fence_async_smem();
                tc_fence_before();
                named_sync(3, 64);
                if (tid == 0) {
                    tc_fence_after();
                    // D3 = K^T u
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            mma_bf16(D3, operand(kq + ks * 2048, 16384, 1024, kSwizzle128),
                                     operand((part ? u_lo : u_hi) + ks * 2 * kGroup, C * 128, kGroup, kSwz),
                                     mma_desc(VS, true, true), part + ks > 0);
                    mma_commit(smem_addr(&sh.m3));
                    mma_commit(smem_addr(&sh.kq_free[st]));
                }
            } else {
                // o = s e^b (Q S) + G R
                mbar_wait(smem_addr(&sh.m2), c & 1, &sh.abort);
                tc_fence_after();
                const int t = c * C + p - C;
#pragma unroll
                for (int g = 0; g < VS / 32; ++g) {
                    float d[32], e[32];
                    tmem_ld32(D1 + lanes + 32 * g, d);
                    tmem_ld32(D2 + lanes + 32 * g, e);
#pragma unroll
                    for (int i = 0; i < 32; ++i) d[i] = fmaf(in, d[i], e[i]);
                    if (t < ntok) {
                        bf16* o = op + (int64_t)t * a.o_st + 32 * g;
#pragma unroll
                        for (int i = 0; i < 32; i += 16) {
                            const uint4 lo = pack16<bf16>(d + i), hi = pack16<bf16>(d + i + 8);
                            if (out32) {
                                st32_stream(o + i, lo, hi);
                            } else {
                                st16(o + i, lo);
                                st16(o + i + 8, hi);
                            }
                        }
                    }
                }
            }
            mbar_wait(smem_addr(&sh.m3), c & 1, &sh.abort);
            tc_fence_after();
#pragma unroll
            for (int g = 0; g < VS / 32; ++g) {
                float d[32];
                tmem_ld32(D3 + lanes + 32 * g, d);
#pragma unroll
                for (int e = 0; e < 32; ++e) S[32 * g + e] = fmaf(decay, S[32 * g + e], d[e]);
            }
        }
        if (sp != nullptr) {
#pragma unroll
            for (int j = 0; j < VS; j += SV) st16(sp + j, pack16<ST>(S + j));
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, kTmemCols);
    if (tid == 0 && sh.abort) flag_status(a.dev_status, CC1D_DEV_TIMEOUT);
}

template <typename ST, int VS>
cudaError_t go(const cc1d_gdr_args& a, bool out32, cudaStream_t stream) {
    constexpr int smem = Layout<VS>::END + 1024;
    const cudaError_t err =
        cudaFuncSetAttribute(gdr_chunk_kernel<ST, VS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return err;
    const int tiles = a.dv / VS;
    const int64_t grid = a.rows * a.heads_v * tiles;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    gdr_chunk_kernel<ST, VS><<<(unsigned)grid, 256, smem, stream>>>(a, tiles, out32);
    return cudaGetLastError();
}

template <typename ST>
cudaError_t pick(const cc1d_gdr_args& a, bool out32, cudaStream_t stream) {
    const int64_t heads = a.rows * a.heads_v;
    if (a.dv % 128 == 0 && heads * (a.dv / 128) >= 148) return go<ST, 128>(a, out32, stream);
    if (a.dv % 64 == 0 && heads * (a.dv / 64) >= 148) return go<ST, 64>(a, out32, stream);
    return go<ST, 32>(a, out32, stream);
}

}  // namespace

bool gdr_chunk_serves(const cc1d_gdr_args& a) {
    auto rows_ok = [](const void* p, int64_t s0, int64_t s1, int64_t s2, int64_t per) {
        return host_aligned16(p) && s0 % per == 0 && s1 % per == 0 && s2 % per == 0;
    };
    const int64_t sv = a.sdtype == CC1D_F32 ? 4 : 8;
    return a.dtype == CC1D_BF16 && a.dk == DK && a.dv % 32 == 0 && a.q_sd == 1 && a.k_sd == 1 &&
           a.v_sd == 1 && a.o_sd == 1 && rows_ok(a.q, a.q_st, a.q_sh, 0, 8) &&
           rows_ok(a.k, a.k_st, a.k_sh, 0, 8) && rows_ok(a.v, a.v_st, a.v_sh, 0, 8) &&
           rows_ok(a.out, a.o_st, a.o_sh, 0, 8) && rows_ok(a.states, a.s_slot, a.s_sh, a.s_sk, sv) &&
           a.tokens >= 16 * a.rows;
}

cudaError_t launch_gdr_chunk(const cc1d_gdr_args& a, cudaStream_t stream) {
    const bool out32 = host_aligned32(a.out) && a.o_st % 16 == 0 && a.o_sh % 16 == 0;
    return a.sdtype == CC1D_F32 ? pick<float>(a, out32, stream) : pick<bf16>(a, out32, stream);
}

}  // namespace cc1d
