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
// Split of the work. Chunks of one sequence form a chain; heads, sequences and the columns of the
// state are independent. A CTA takes one head of one sequence, NG tiles of VS state columns, and has
//   - prep warps: [K;Q] K^T on the tensor core, L, its inverse, T and G = P T. Nothing of it
//     depends on the state, so it runs ahead of the chain;
//   - NG scan groups of 256 threads (two per row), each with the chain of its own columns: [K;Q] S0,
//     R, [T;G] R, u, K^T u, S. Two chains in a CTA fill each other's waits and share K, Q, T and G.
// K, Q and V come by TMA, K and Q up to three chunks ahead. The state lies in TMEM.
// Stacking K over Q and T over G makes every product M = 128, the full tensor core rate; the two
// parts of an operand lie side by side as one operand of 2 VS columns (measured: a K step of 16
// costs 46 cycles up to 64 columns and 66 with 128, so one wide step beats two narrow ones).
// Loops over columns stay rolled where registers allow it: with all of them unrolled the warps
// spent a quarter of their time waiting for instructions.
#include "gdr.cuh"
#include "kernels.h"
#include "tc05.cuh"

namespace cc1d {
namespace {

constexpr int C = 64;        // tokens per chunk
constexpr int DK = 128;      // key head dim
constexpr int LPAD = 36;     // fp32 row of a 32 x 32 block: 16-byte accesses of 8 rows hit 8 bank groups
constexpr int kOrderMax = 256;  // batches up to this many sequences start with the longest

struct Vectors {     // per chunk: what the scan multiplies rows by
    float in[2 * C];  // r_i e^(b_i) (rows of K), s_i e^(b_i) (rows of Q)
    float out[C];     // r_j e^(b_C - b_j)
    float decay;      // e^(b_C)
    float pad[3];
};

// I + L in 32 x 32 blocks, fp32: the diagonal blocks (L, then their inverses in place) and the
// block below them.
struct Blocks {
    float diag[2][32][LPAD], low[32][LPAD];
};

template <int VS, int NG>
struct Layout {
    static constexpr int kRow = VS >= 64 ? 128 : 2 * VS;  // bytes of an operand row of VS columns
    static constexpr int kS = 128 * kRow;                 // one part (hi or lo) of S
    static constexpr int kR = C * kRow;                   // one part of R or u, or one tile of V
    static constexpr int kStages = NG == 1 ? 3 : 2;       // of K and Q
    static constexpr int KQ = 0;                          // stages x [2 halves][128 rows][128 B]
    static constexpr int V = KQ + kStages * 32768;        // NG x [64 rows]
    static constexpr int TG = V + NG * kR;                // [hi, lo][128 rows][128 B]
    static constexpr int SB = TG + 32768;                 // NG x (S hi, S lo); R in S hi, u in S lo
    static constexpr int P = SB + NG * 2 * kS;            // [hi, lo][64 rows][128 B]
    static constexpr int B = P + 16384;                   // Blocks
    static constexpr int VEC = B + (int)sizeof(Blocks);   // 2 stages x Vectors
    static constexpr int END = VEC + 2 * (int)sizeof(Vectors);
    static constexpr int kTmem = 128 + NG * 3 * VS <= 256 ? 256 : 512;
    static constexpr int kPrepWarps = NG == 1 ? 8 : 4;
    static constexpr int kThreads = 256 * NG + 32 * kPrepWarps;
};
// P as a 128-row operand reads 8 KB behind its last row.
static_assert(sizeof(Blocks) >= 8192, "");

// What a chunk's gates give: cumulative log2 decays b, negated, in two parts each; rates; decays
// e^(b_i), e^(b_C - b_j) and, below 32, e^(b_31 - b_j).
struct Gates {
    alignas(16) float nbh[C], nbl[C], beta[C], grow[C], out[C], far[32];
};

struct Shared {
    uint64_t kq_tma[3], kq_full[3], vec_full[2], v_full[2], tg_full, tg_free, prep_mma, scan_mma[2];
    uint32_t tmem;
    int abort;
    int row;  // sequence of this CTA
    int done[3];  // per stage: scan groups that are through with its K and Q, over all chunks
    int len[kOrderMax];
    alignas(16) float rk[C], ru[32], qq[2][2 * C];
    Gates gates[2];
};

// Row r, 16-byte unit u of an operand image of ROW-byte rows.
template <int ROW>
__device__ __forceinline__ uint32_t swz(int r, int u) {
    if constexpr (ROW == 128) {
        return r * 128 + ((u ^ (r & 7)) << 4);
    } else {
        return r * 64 + ((u ^ ((r >> 1) & 3)) << 4);
    }
}

// 8 values as two bf16 parts, one 16-byte unit each.
__device__ __forceinline__ void store_split8(uint32_t hi, uint32_t lo, const float2* f) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split2(f[i], h[i], l[i]);
    sts16(hi, h[0], h[1], h[2], h[3]);
    sts16(lo, l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ float2 mul2(float2 a, float b) {
    return __fmul2_rn(a, make_float2(b, b));
}
__device__ __forceinline__ float2 bf16_pair(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Row i of the inverse of I + l (l strictly lower triangular, 16 x 16, zeros above) by backward
// substitution: y_m is final once every later y has been taken out of it, and is then taken out of
// the earlier ones along row m of l. A lane owns a row; the rows of l come as broadcasts.
__device__ __forceinline__ void solve_row16(const float (*l)[LPAD], int i, float2* y) {
#pragma unroll
    for (int q = 0; q < 8; ++q) y[q] = make_float2(i == 2 * q ? 1.f : 0.f, i == 2 * q + 1 ? 1.f : 0.f);
#pragma unroll
    for (int m = 15; m > 0; --m) {
        const float v = -(m % 2 ? y[m / 2].y : y[m / 2].x);
        const float2 vv = make_float2(v, v);
#pragma unroll
        for (int r = 0; r < m; r += 4) {
            const float4 f = *reinterpret_cast<const float4*>(&l[m][r]);
            y[r / 2] = __ffma2_rn(make_float2(f.x, f.y), vv, y[r / 2]);
            if (r + 2 < m) y[r / 2 + 1] = __ffma2_rn(make_float2(f.z, f.w), vv, y[r / 2 + 1]);
        }
    }
}

// d (16 x 8) += a (16 x 16) b (16 x 8), bf16 operands, fp32 sums, within a warp.
__device__ __forceinline__ void mma_warp(float* d, const uint32_t* a, const uint32_t* b) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_warp3(float* d, const uint32_t (*a)[4], const uint32_t (*b)[2]) {
    mma_warp(d, a[0], b[0]);
    mma_warp(d, a[0], b[1]);
    mma_warp(d, a[1], b[0]);
}

// The 16 x 16 tile inv1[r0.., :] (low inv0)[:, c0..] of a product of K x K matrices, K = 16 or 32,
// by one warp in two-part bf16. The inner product is formed transposed, (inv0^T low^T): its
// accumulator fragments are then the B fragments of the outer one. d: accumulators of columns c0..
// and c0 + 8...
template <int K>
__device__ __forceinline__ void merge_tile(const float (*inv1)[LPAD], const float (*low)[LPAD],
                                           const float (*inv0)[LPAD], int r0, int c0, int lane,
                                           float (*d)[4]) {
    const int g = lane / 4, t2 = lane % 4 * 2;
    // The two halves of a sum over 32 go to accumulators of their own: shorter chains of products.
    float m[K / 16][K / 8][4];  // (low inv0)^T: rows c0.., 8 columns (rows of low) each
#pragma unroll
    for (int k = 0; k < K / 16; ++k) {
        uint32_t av[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = c0 + g + e % 2 * 8, r = 16 * k + t2 + e / 2 * 8;
            split2(make_float2(inv0[r][col], inv0[r + 1][col]), av[0][e], av[1][e]);
        }
#pragma unroll
        for (int n = 0; n < K / 8; ++n) {
            uint32_t bv[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                split2(*reinterpret_cast<const float2*>(&low[8 * n + g][16 * k + t2 + 8 * e]), bv[0][e], bv[1][e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) m[k][n][e] = 0.f;
            mma_warp3(m[k][n], av, bv);
        }
    }
    float s[K / 16][2][4];
#pragma unroll
    for (int k = 0; k < K / 16; ++k) {
        uint32_t av[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            split2(*reinterpret_cast<const float2*>(&inv1[r0 + g + e % 2 * 8][16 * k + t2 + e / 2 * 8]), av[0][e], av[1][e]);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            uint32_t bv[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float2 f = make_float2(m[0][2 * k + e][2 * n], m[0][2 * k + e][2 * n + 1]);
                if (K > 16)
                    f = __fadd2_rn(f, make_float2(m[K / 16 - 1][2 * k + e][2 * n], m[K / 16 - 1][2 * k + e][2 * n + 1]));
                split2(f, bv[0][e], bv[1][e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[k][n][e] = 0.f;
            mma_warp3(s[k][n], av, bv);
        }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[n][e] = K > 16 ? s[0][n][e] + s[K / 16 - 1][n][e] : s[0][n][e];
}

// Bits of element i of a gate tensor, and its value: the load and its use can lie far apart.
__device__ __forceinline__ uint32_t load_bits(const void* p, int64_t i, int dtype) {
    return dtype == CC1D_F32 ? static_cast<const uint32_t*>(p)[i] : static_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float bits_value(uint32_t b, int dtype) {
    if (dtype == CC1D_BF16) return __uint_as_float(b << 16);
    if (dtype == CC1D_F16) return __half2float(__ushort_as_half((unsigned short)b));
    return __uint_as_float(b);
}

template <typename ST, int VS, int NG>
__global__ void __launch_bounds__(Layout<VS, NG>::kThreads, 1)
gdr_chunk_kernel(const __grid_constant__ cc1d_gdr_args a, const __grid_constant__ CUtensorMap mapq,
                 const __grid_constant__ CUtensorMap mapk, const __grid_constant__ CUtensorMap mapv,
                 int tiles, bool out32) {
    using Lay = Layout<VS, NG>;
    constexpr uint64_t kSwz = VS >= 64 ? kSwizzle128 : kSwizzle64;
    constexpr uint32_t kGroup = 8 * Lay::kRow;  // bytes of eight rows of V columns
    constexpr int kStages = Lay::kStages;
    extern __shared__ __align__(1024) unsigned char raw[];
    __shared__ Shared sh;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    unsigned char* gen = raw + (base - smem_addr(raw));
    Vectors* vec = reinterpret_cast<Vectors*>(gen + Lay::VEC);
    Blocks& blk = *reinterpret_cast<Blocks*>(gen + Lay::B);

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, p = tid % 128, w = warp % 4;
    const int vt = blockIdx.x % tiles;  // columns vt * NG * VS ..
    const int h = (int)((blockIdx.x / tiles) % a.heads_v);
    int64_t row = blockIdx.x / tiles / a.heads_v;
    const int hk = h / (a.heads_v / a.heads_k);

    // Longest sequences first, so that the last CTAs to start are short. Ties go by index.
    if (a.rows > 1 && a.rows <= kOrderMax) {
        const int n = (int)a.rows;
        for (int j = tid; j < n; j += Lay::kThreads)
            sh.len[j] = a.query_start_loc[j + 1] - a.query_start_loc[j];
        __syncthreads();
        for (int j = tid; j < n; j += Lay::kThreads) {
            int rank = 0;
            for (int i = 0; i < n; ++i)
                rank += sh.len[i] > sh.len[j] || (sh.len[i] == sh.len[j] && i < j);
            if (rank == row) sh.row = j;
        }
        __syncthreads();
        row = sh.row;
    }
    int64_t tok0, slot;
    int ntok;
    if (!gdr_row(a, true, row, tok0, ntok, slot, h == 0 && vt == 0 && tid == 0)) return;
    const int chunks = (ntok + C - 1) / C;

    if (tid == 0) {
        for (int i = 0; i < 3; ++i) {
            mbar_init(smem_addr(&sh.kq_tma[i]), 1);
            mbar_init(smem_addr(&sh.kq_full[i]), 1);
            sh.done[i] = 0;
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&sh.vec_full[i]), 1);
            mbar_init(smem_addr(&sh.v_full[i]), 1);
            mbar_init(smem_addr(&sh.scan_mma[i]), 1);
        }
        mbar_init(smem_addr(&sh.tg_full), 1);
        mbar_init(smem_addr(&sh.tg_free), NG);
        mbar_init(smem_addr(&sh.prep_mma), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.abort = 0;
    }
    if (warp == 0) {
        tmem_alloc(smem_addr(&sh.tmem), Lay::kTmem);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t lanes = (uint32_t)w << 21;  // the warp's first TMEM lane, in bits 16..
    const uint32_t tg = base + Lay::TG;

    // K and Q of chunk c into stage st, which must be free; one thread.
    auto load_kq = [&](int c, int st) {
        const uint32_t full = smem_addr(&sh.kq_tma[st]), kq = base + Lay::KQ + st * 32768;
        const int t = (int)tok0 + c * C;
        mbar_expect(full, 32768);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            tma_load(kq + half * 16384, &mapk, half * 64, hk, t, full);
            tma_load(kq + half * 16384 + 8192, &mapq, half * 64, hk, t, full);
        }
    };
    // V of chunk c for scan group g.
    auto load_v = [&](int c, int g) {
        const uint32_t full = smem_addr(&sh.v_full[g]);
        mbar_expect(full, C * VS * 2);
        tma_load(base + Lay::V + g * Lay::kR, &mapv, (vt * NG + g) * VS, h, (int)tok0 + c * C, full);
    };
    if (tid == 0) {
        for (int c = 0; c < kStages && c < chunks; ++c) load_kq(c, c);
        for (int g = 0; g < NG; ++g) load_v(0, g);
    }

    if (warp >= 8 * NG) {
        // --------------------------------------------------------------------------------- prep
        // A thread has row p of [K;Q] K^T: columns 32 half .., both halves in turn with four warps.
        constexpr int kPrep = 32 * Lay::kPrepWarps, kHalves = kPrep / 128;
        const int half0 = (warp - 8 * NG) / 4;
        const int i = p % C;
        const int pt = tid - 256 * NG;
        const bool lead = pt == kPrep - 32;          // issues the products
        const bool gate_warp = pt / 32 == kPrep / 32 - 4 + (kHalves == 1 ? 2 : 0);  // idle while others solve
        const uint32_t D0 = tmem;  // 64 columns of [K;Q] K^T; later 128 of P [T hi | T lo]
        const uint32_t pb = base + Lay::P;
        // T and P are zero above their diagonal blocks; nothing writes there again.
        if (p < 32 && half0 == 0) {
#pragma unroll
            for (int u = 4; u < 8; ++u) {
                sts16(tg + swz<128>(p, u), 0, 0, 0, 0);
                sts16(tg + 16384 + swz<128>(p, u), 0, 0, 0, 0);
                sts16(pb + swz<128>(p, u), 0, 0, 0, 0);
                sts16(pb + 8192 + swz<128>(p, u), 0, 0, 0, 0);
            }
        }
        // Gates of a chunk, by one warp, two tokens a lane. The raw values of the next chunk are
        // loaded here a chunk before they are used.
        float rate = 0.f, dt = 0.f;
        uint32_t g_bits[2] = {0, 0}, b_bits[2] = {0, 0};
        const int64_t g0 = tok0 * a.g_st + h * a.g_sh, b0 = tok0 * a.b_st + h * a.b_sh;
        auto load_gate_bits = [&](int c) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int64_t t = (int64_t)c * C + 2 * lane + e;
                if (t < ntok) {
                    g_bits[e] = load_bits(a.g, g0 + t * a.g_st, a.gdtype);
                    b_bits[e] = load_bits(a.beta, b0 + t * a.b_st, a.bdtype);
                }
            }
        };
        auto make_gates = [&](int c) {
            Gates& to = sh.gates[c & 1];
            double sum[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float g = 0.f, beta = 0.f;
                if (c * C + 2 * lane + e < ntok) {
                    g = bits_value(g_bits[e], a.gdtype);
                    beta = bits_value(b_bits[e], a.bdtype);
                    if (a.a_log != nullptr) {
                        const float z = g + dt;
                        g = rate * (z > 20.f ? z : log1pf(expf(z)));
                        beta = 1.f / (1.f + expf(-beta));
                    }
                    // -1e5 decays anything to zero, and its sums stay finite where -inf would give
                    // inf - inf below.
                    g = g < -1e5f ? -1e5f : g;
                }
                to.beta[2 * lane + e] = beta;
                // The sums are carried in 64 bits and kept as two fp32 parts: their differences
                // are exponents, where fp32 sums of strong decays would lose the weak ones.
                sum[e] = (double)g * 1.4426950408889634;
            }
            load_gate_bits(c + 1);
            sum[1] += sum[0];
            double total = sum[1];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double below = __shfl_up_sync(~0u, total, o);
                if (lane >= o) total += below;
            }
            const double mid = __shfl_sync(~0u, total, 15), end = __shfl_sync(~0u, total, 31);
            const double b[2] = {total - sum[1] + sum[0], total};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = 2 * lane + e;
                const float hi = (float)b[e];
                to.nbh[t] = -hi;
                to.nbl[t] = (float)((double)hi - b[e]);
                to.grow[t] = exp2_approx(hi);
                to.out[t] = exp2_approx((float)(end - b[e]));
                if (t < 32) to.far[t] = exp2_approx((float)(mid - b[e]));
            }
        };
        if (gate_warp) {
            if (a.a_log != nullptr) {
                rate = -expf(load_any(a.a_log, h, a.pdtype));
                dt = load_any(a.dt_bias, h, a.pdtype);
            }
            load_gate_bits(0);
            make_gates(0);
        }

        int st = 0;
        uint32_t st_phase = 0;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
            Vectors& ve = vec[c & 1];
            const Gates& ga = sh.gates[c & 1];
            const uint32_t kq = base + Lay::KQ + st * 32768;
            const int left = ntok - c * C;
            mbar_wait(smem_addr(&sh.kq_tma[st]), st_phase, &sh.abort);
            if (left < C) {
                // The copies went on into the next sequence: zeros there, whatever it holds.
                for (int e = pt; e < (C - left) * 32; e += kPrep) {
                    const int r = left + e / 32, u = e % 16;
                    sts16(kq + (u >> 3) * 16384 + swz<128>(r + (e & 16) * 4, u & 7), 0, 0, 0, 0);
                }
                fence_async_smem();
            }
            tc_fence_before();
            named_sync(8, kPrep);
            if (lead) {
                mbar_arrive(smem_addr(&sh.kq_full[st]));
                tc_fence_after();
                const uint64_t d = operand(kq, 16, 1024, kSwizzle128);
                mma_steps<4, 2, 2>(D0, d, d, mma_desc(64, false, false), false);
                mma_steps<4, 2, 2>(D0, d + 1024, d + 1024, mma_desc(64, false, false), true);
                mma_commit(smem_addr(&sh.prep_mma));
            }
            // While it runs: the norms of its rows.
            for (int hf = half0; hf < 2; hf += kHalves) {
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 4
                for (int u = 0; u < 8; ++u) {
                    const uint4 v = lds16(kq + hf * 16384 + swz<128>(p, u));
                    const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = bf16_pair(vv[e]);
                        sum[e % 2] = __ffma2_rn(f, f, sum[e % 2]);
                    }
                }
                sh.qq[hf][p] = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            named_sync(8, kPrep);
            const float norm = a.l2norm ? rsqrtf(sh.qq[0][p] + sh.qq[1][p] + kL2Eps) : 1.f;
            const float mul = norm * (p < C ? ga.beta[i] : a.scale);  // of row i of L or P
            if (half0 == 0) {
                ve.in[p] = ga.grow[i] * (p < C ? norm : mul);
                if (p < C) {
                    sh.rk[p] = norm;
                    ve.out[i] = norm * ga.out[i];
                    if (p < 32) sh.ru[p] = norm * ga.far[p];
                    if (i == C - 1) ve.decay = ga.grow[i];
                }
            }
            named_sync(8, kPrep);
            if (pt == 0) mbar_arrive(smem_addr(&sh.vec_full[c & 1]));
            mbar_wait(smem_addr(&sh.prep_mma), 0, &sh.abort);
            tc_fence_after();
            // Warps 0 and 1 make L (columns j < i) of rows of K K^T, warps 2 and 3 make P (columns
            // j <= i) of rows of Q K^T. In the columns of a row's own half the decay e^(b_i - b_j)
            // is taken element by element; for the lower left block it splits at the middle of the
            // chunk into two factors of at most 1.
#pragma unroll 1
            for (int hf = half0; hf < 2; hf += kHalves) {
                if (hf > w % 2) continue;  // above the diagonal block
                const bool own = hf == w % 2;
                const float2 bh = make_float2(-ga.nbh[i], -ga.nbh[i]), bl = make_float2(-ga.nbl[i], -ga.nbl[i]);
                const float low_mul = mul * exp2_approx((bh.x + ga.nbh[31]) + (bl.x + ga.nbl[31]));
                const int last = (p < C ? i - 1 : i) - 32 * hf;  // last column of this half that counts
                float (*to)[LPAD] = own ? blk.diag[w % 2] : blk.low;
#pragma unroll 1
                for (int o = 0; o < 32; o += 16) {
                    float2 x[8];
                    tmem_ld16(D0 + lanes + 32 * hf + o, x);
                    if (own) {
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const int jj = o + 2 * e, j = 32 * hf + jj;
                            const float4 h4 = *reinterpret_cast<const float4*>(&ga.nbh[j]);
                            const float4 l4 = *reinterpret_cast<const float4*>(&ga.nbl[j]);
                            const float4 r4 = *reinterpret_cast<const float4*>(&sh.rk[j]);
                            const float2 e0 = __fadd2_rn(__fadd2_rn(bh, make_float2(h4.x, h4.y)),
                                                         __fadd2_rn(bl, make_float2(l4.x, l4.y)));
                            const float2 e1 = __fadd2_rn(__fadd2_rn(bh, make_float2(h4.z, h4.w)),
                                                         __fadd2_rn(bl, make_float2(l4.z, l4.w)));
                            x[e] = __fmul2_rn(__fmul2_rn(x[e], mul2(make_float2(r4.x, r4.y), mul)),
                                              make_float2(exp2_approx(e0.x), exp2_approx(e0.y)));
                            x[e + 1] = __fmul2_rn(__fmul2_rn(x[e + 1], mul2(make_float2(r4.z, r4.w), mul)),
                                                  make_float2(exp2_approx(e1.x), exp2_approx(e1.y)));
                            // Columns behind the last one: their decay may be inf, their value is 0.
                            x[e].x = jj <= last ? x[e].x : 0.f;
                            x[e].y = jj + 1 <= last ? x[e].y : 0.f;
                            x[e + 1].x = jj + 2 <= last ? x[e + 1].x : 0.f;
                            x[e + 1].y = jj + 3 <= last ? x[e + 1].y : 0.f;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const float4 r4 = *reinterpret_cast<const float4*>(&sh.ru[o + 2 * e]);
                            x[e] = __fmul2_rn(x[e], mul2(make_float2(r4.x, r4.y), low_mul));
                            x[e + 1] = __fmul2_rn(x[e + 1], mul2(make_float2(r4.z, r4.w), low_mul));
                        }
                    }
                    if (p < C) {
#pragma unroll
                        for (int e = 0; e < 8; e += 2)
                            *reinterpret_cast<float4*>(&to[lane][o + 2 * e]) =
                                make_float4(x[e].x, x[e].y, x[e + 1].x, x[e + 1].y);
                    } else {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint32_t at = pb + swz<128>(i, 4 * hf + o / 8 + u);
                            store_split8(at, at + 8192, x + 4 * u);
                        }
                    }
                }
            }
            if (gate_warp && c + 1 < chunks) make_gates(c + 1);
            if (p < C && (w % 2 == half0 || kHalves == 1)) {
                // Inverse of this warp's diagonal block: its two 16 x 16 blocks by substitution, a
                // half warp each, then the block below them, -inv_1 (L_21 inv_0).
                float (*dg)[LPAD] = blk.diag[w];
                const int b = lane & 16;
                float2 y[8];
                __syncwarp();
                solve_row16(reinterpret_cast<const float (*)[LPAD]>(&dg[b][b]), lane & 15, y);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    *reinterpret_cast<float4*>(&dg[lane][b + 2 * e]) =
                        make_float4(y[e].x, y[e].y, y[e + 1].x, y[e + 1].y);
                __syncwarp();
                float d[2][4];
                merge_tile<16>(reinterpret_cast<const float (*)[LPAD]>(&dg[16][16]),
                               reinterpret_cast<const float (*)[LPAD]>(&dg[16][0]), dg, 0, 0, lane, d);
                __syncwarp();
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float2*>(&dg[16 + lane / 4 + 8 * e][8 * n + lane % 4 * 2]) =
                            make_float2(-d[n][2 * e], -d[n][2 * e + 1]);
            }
            named_sync(8, kPrep);
            // The chain's products with the previous T and G must be done with their memory.
            if (c > 0) mbar_wait(smem_addr(&sh.tg_free), (c - 1) & 1, &sh.abort);
            if (half0 == 0) {
                // The 32 x 32 block below the diagonal ones, a 16 x 16 tile per warp.
                const int r0 = w / 2 * 16, c0 = w % 2 * 16, fr = r0 + lane / 4, fc = c0 + lane % 4 * 2;
                float d[2][4];
                merge_tile<32>(blk.diag[1], blk.low, blk.diag[0], r0, c0, lane, d);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int col = fc + 8 * n;
                    const float2 bt = make_float2(-ga.beta[col], -ga.beta[col + 1]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t hi, lo;
                        split2(__fmul2_rn(make_float2(d[n][2 * e], d[n][2 * e + 1]), bt), hi, lo);
                        const uint32_t at = tg + swz<128>(32 + fr + 8 * e, col / 8) + col % 8 * 2;
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(hi) : "memory");
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 16384), "r"(lo) : "memory");
                    }
                }
            }
            if (half0 == kHalves - 1) {
                // The diagonal blocks: row p / 2, half of its 32 columns.
                const int r = p / 2, o = p % 2 * 16;
#pragma unroll 1
                for (int u = 0; u < 2; ++u) {
                    const float* from = &blk.diag[r / 32][r % 32][o + 8 * u];
                    const float* bt = &ga.beta[r / 32 * 32 + o + 8 * u];
                    float2 f[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        f[e] = __fmul2_rn(*reinterpret_cast<const float2*>(from + 2 * e),
                                          *reinterpret_cast<const float2*>(bt + 2 * e));
                    const uint32_t at = tg + swz<128>(r, r / 32 * 4 + o / 8 + u);
                    store_split8(at, at + 16384, f);
                }
            }
            fence_async_smem();
            tc_fence_before();
            named_sync(8, kPrep);
            if (lead) {
                tc_fence_after();
                // G = P T in rows 0..63: hi [hi | lo], then lo hi. Rows 64.. are of no use.
                const uint64_t t = operand(tg, 16384, 1024, kSwizzle128);
                mma_steps<4, 2, 128>(D0, operand(pb, 16, 1024, kSwizzle128), t, mma_desc(128, false, true), false);
                mma_steps<4, 2, 128>(D0, operand(pb + 8192, 16, 1024, kSwizzle128), t, mma_desc(64, false, true), true);
                mma_commit(smem_addr(&sh.prep_mma));
            }
            mbar_wait(smem_addr(&sh.prep_mma), 1, &sh.abort);
            tc_fence_after();
            if (p < C) {
#pragma unroll 1
                for (int o = 16 * half0; o < C; o += 16 * kHalves) {
                    float2 x[8], y[8];
                    tmem_ld16(D0 + lanes + o, D0 + lanes + 64 + o, x, y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = __fadd2_rn(x[e], y[e]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t at = tg + swz<128>(C + p, o / 8 + u);
                        store_split8(at, at + 16384, x + 4 * u);
                    }
                }
                fence_async_smem();
            }
            tc_fence_before();
            named_sync(8, kPrep);
            if (pt == 0) mbar_arrive(smem_addr(&sh.tg_full));
            if (++st == kStages) {
                st = 0;
                st_phase ^= 1;
            }
        }
    } else {
        // -------------------------------------------------------------------------------- scan
        // A thread has row p and columns first .. first + W of its group's tile.
        constexpr int W = VS / 2;
        const int grp = warp / 8, first = warp / 4 % 2 * W;
        const int bar = 1 + grp;
        const bool lead = tid % 256 == 0;
        const uint32_t D = tmem + 128 + grp * 3 * VS;  // [product with hi parts | with lo parts]
        const uint32_t Dh = D + lanes + first, Dl = Dh + VS, TS = Dl + VS;  // TS: the state
        const uint32_t mma = smem_addr(&sh.scan_mma[grp]);
        const uint32_t s_hi = base + Lay::SB + grp * 2 * Lay::kS, s_lo = s_hi + Lay::kS;
        const uint32_t r_hi = s_hi, r_lo = r_hi + Lay::kR, u_hi = s_lo, u_lo = u_hi + Lay::kR;
        const uint32_t vb = base + Lay::V + grp * Lay::kR;
        const int col = (vt * NG + grp) * VS + first;
        const bool initial = a.states != nullptr && a.has_initial_state != nullptr && a.has_initial_state[row];
        ST* sp = nullptr;
        if (a.states != nullptr)
            sp = static_cast<ST*>(a.states) + slot * a.s_slot + h * a.s_sh + p * a.s_sk + col;
        constexpr int SV = Vec<ST>::V;
        bf16* op = static_cast<bf16*>(a.out) + tok0 * a.o_st + h * a.o_sh + col;

        int st = 0;
        uint32_t phase = 0, st_phase = 0;
        float decay = 0.f;
#pragma unroll 1
        for (int c = 0;; ++c) {
            // The state after the chunk before, into TMEM, and as an operand if there is another.
#pragma unroll 1
            for (int o = 0; o < W; o += 16) {
                float2 s[8];
                if (c == 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[e] = make_float2(0.f, 0.f);
                    if (initial) {
#pragma unroll
                        for (int e = 0; e < 16; e += SV) unpack16<ST>(ld16(sp + o + e), &s[0].x + e);
                    }
                } else {
                    float2 d[8], e[8];
                    tmem_ld16(Dh + o, Dl + o, TS + o, d, e, s);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        s[k] = __ffma2_rn(make_float2(decay, decay), s[k], __fadd2_rn(d[k], e[k]));
                }
                if (c == chunks) {
                    if (sp != nullptr) {
#pragma unroll
                        for (int e = 0; e < 16; e += SV) st16(sp + o + e, pack16<ST>(&s[0].x + e));
                    }
                } else {
                    tmem_st16(TS + o, s);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t at = swz<Lay::kRow>(p, (first + o) / 8 + u);
                        store_split8(s_hi + at, s_lo + at, s + 4 * u);
                    }
                }
            }
            if (c == chunks) break;
            tmem_wait_st();
            const uint32_t kq = base + Lay::KQ + st * 32768;
            fence_async_smem();
            tc_fence_before();
            named_sync(bar, 256);
            if (lead) {
                mbar_wait(smem_addr(&sh.kq_full[st]), st_phase, &sh.abort);
                tc_fence_after();
                // [K;Q] S
                const uint64_t k = operand(kq, 16, 1024, kSwizzle128), s = operand(s_hi, Lay::kS, kGroup, kSwz);
                mma_steps<4, 2, kGroup / 8>(D, k, s, mma_desc(2 * VS, false, true), false);
                mma_steps<4, 2, kGroup / 8>(D, k + 1024, s + kGroup / 2, mma_desc(2 * VS, false, true), true);
                mma_commit(mma);
            }
            mbar_wait(smem_addr(&sh.vec_full[c & 1]), (c >> 1) & 1, &sh.abort);
            const float in = vec[c & 1].in[p], out = vec[c & 1].out[p % C];
            decay = vec[c & 1].decay;
            float2 q[W / 2];  // rows of Q: their outputs
            if (p < C) mbar_wait(smem_addr(&sh.v_full[grp]), c & 1, &sh.abort);
            mbar_wait(mma, phase, &sh.abort);
            phase ^= 1;
            tc_fence_after();
            if (p < C) {
                // R = V - r e^b (K S), zero behind the sequence's end, whatever V holds there
                const bool live = c * C + p < ntok;
#pragma unroll 1
                for (int o = 0; o < W; o += 16) {
                    float2 d[8], e[8];
                    tmem_ld16(Dh + o, Dl + o, d, e);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t at = swz<Lay::kRow>(p, (first + o) / 8 + u);
                        const uint4 v = lds16(vb + at);
                        const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
                        float2 f[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            f[k] = __ffma2_rn(make_float2(-in, -in), __fadd2_rn(d[4 * u + k], e[4 * u + k]),
                                              bf16_pair(live ? vv[k] : 0u));
                        store_split8(r_hi + at, r_lo + at, f);
                    }
                }
                fence_async_smem();
            } else {
#pragma unroll
                for (int o = 0; o < W; o += 16) {
                    float2 d[8], e[8];
                    tmem_ld16(Dh + o, Dl + o, d, e);
#pragma unroll
                    for (int k = 0; k < 8; ++k) q[o / 2 + k] = mul2(__fadd2_rn(d[k], e[k]), in);
                }
            }
            tc_fence_before();
            named_sync(bar, 256);
            if (lead) {
                if (c + 1 < chunks) load_v(c + 1, grp);
                mbar_wait(smem_addr(&sh.tg_full), c & 1, &sh.abort);
                tc_fence_after();
                // [T;G] R: hi [hi | lo], then lo hi
                const uint64_t r = operand(r_hi, Lay::kR, kGroup, kSwz);
                mma_steps<4, 2, kGroup / 8>(D, operand(tg, 16, 1024, kSwizzle128), r, mma_desc(2 * VS, false, true), false);
                mma_steps<4, 2, kGroup / 8>(D, operand(tg + 16384, 16, 1024, kSwizzle128), r, mma_desc(VS, false, true), true);
                mma_commit(mma);
                mma_commit(smem_addr(&sh.tg_free));
            }
            mbar_wait(mma, phase, &sh.abort);
            phase ^= 1;
            tc_fence_after();
            if (p < C) {
#pragma unroll 1
                for (int o = 0; o < W; o += 16) {
                    float2 d[8], e[8];
                    tmem_ld16(Dh + o, Dl + o, d, e);
#pragma unroll
                    for (int k = 0; k < 8; ++k) d[k] = mul2(__fadd2_rn(d[k], e[k]), out);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t at = swz<Lay::kRow>(p, (first + o) / 8 + u);
                        store_split8(u_hi + at, u_lo + at, d + 4 * u);
                    }
                }
                fence_async_smem();
            } else {
#pragma unroll
                for (int o = 0; o < W; o += 16) {
                    float2 d[8], e[8];
                    tmem_ld16(Dh + o, Dl + o, d, e);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        q[o / 2 + k] = __fadd2_rn(q[o / 2 + k], __fadd2_rn(d[k], e[k]));
                }
            }
            tc_fence_before();
            named_sync(bar, 256);
            if (lead) {
                tc_fence_after();
                // K^T u
                mma_steps<4, 128, kGroup / 8>(D, operand(kq, 16384, 1024, kSwizzle128),
                                              operand(u_hi, Lay::kR, kGroup, kSwz),
                                              mma_desc(2 * VS, true, true), false);
                mma_commit(mma);
            }
            const int t = c * C + p - C;
            if (p >= C && t < ntok) {
                bf16* to = op + (int64_t)t * a.o_st;
#pragma unroll
                for (int k = 0; k < W; k += 16) {
                    const uint4 lo = pack16<bf16>(&q[k / 2].x), hi = pack16<bf16>(&q[k / 2 + 4].x);
                    if (out32) {
                        st32_stream(to + k, lo, hi);
                    } else {
                        st16(to + k, lo);
                        st16(to + k + 8, hi);
                    }
                }
            }
            mbar_wait(mma, phase, &sh.abort);
            phase ^= 1;
            tc_fence_after();
            if (lead && c + kStages < chunks) {
                // The last scan group through with the chunk refills its stage.
                __threadfence_block();
                if (atomicAdd(&sh.done[st], 1) % NG == NG - 1) {
                    __threadfence_block();
                    load_kq(c + kStages, st);
                }
            }
            if (++st == kStages) {
                st = 0;
                st_phase ^= 1;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, Lay::kTmem);
    if (tid == 0 && sh.abort) flag_status(a.dev_status, CC1D_DEV_TIMEOUT);
}

// Tensor map of a (tokens, heads, dim) bf16 view, boxes of 64 tokens of one head.
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                            const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                            CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                            CUtensorMapFloatOOBfill);

Encode encoder() {
    static const Encode f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) !=
                cudaSuccess || found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<Encode>(p);
    }();
    return f;
}

bool make_map(CUtensorMap* map, const void* p, int64_t tokens, int heads, int dim, int64_t st,
              int64_t sh, int cols) {
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)sh * 2, (cuuint64_t)st * 2};
    const cuuint32_t box[3] = {(cuuint32_t)cols, 1, C}, step[3] = {1, 1, 1};
    return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides,
                     box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename ST, int VS, int NG>
cudaError_t go(const cc1d_gdr_args& a, bool out32, cudaStream_t stream) {
    using Lay = Layout<VS, NG>;
    constexpr int smem = Lay::END + 1024;
    const int tiles = a.dv / (VS * NG);
    const int64_t grid = a.rows * a.heads_v * tiles;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    CUtensorMap q, k, v;
    if (!make_map(&q, a.q, a.tokens, a.heads_k, a.dk, a.q_st, a.q_sh, 64) ||
        !make_map(&k, a.k, a.tokens, a.heads_k, a.dk, a.k_st, a.k_sh, 64) ||
        !make_map(&v, a.v, a.tokens, a.heads_v, a.dv, a.v_st, a.v_sh, VS))
        return cudaErrorInvalidValue;
    const cudaError_t err =
        cudaFuncSetAttribute(gdr_chunk_kernel<ST, VS, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return err;
    gdr_chunk_kernel<ST, VS, NG><<<(unsigned)grid, Lay::kThreads, smem, stream>>>(a, q, k, v, tiles, out32);
    return cudaGetLastError();
}

template <typename ST>
cudaError_t pick(const cc1d_gdr_args& a, bool out32, cudaStream_t stream) {
    const int64_t heads = a.rows * a.heads_v;
    if (a.dv % 128 == 0 && heads * (a.dv / 128) >= 148) return go<ST, 64, 2>(a, out32, stream);
    if (a.dv % 64 == 0 && heads * (a.dv / 64) >= 148) return go<ST, 64, 1>(a, out32, stream);
    return go<ST, 32, 1>(a, out32, stream);
}

}  // namespace

bool gdr_chunk_serves(const cc1d_gdr_args& a) {
    auto rows_ok = [](const void* p, int64_t s0, int64_t s1, int64_t per) {
        return host_aligned16(p) && s0 % per == 0 && s1 % per == 0;
    };
    // What a tensor map describes: 16-byte rows, positive strides below 2^40 bytes.
    auto map_ok = [&](const void* p, int64_t st, int64_t sh) {
        return rows_ok(p, st, sh, 8) && st > 0 && sh > 0 && st < (1ll << 38) && sh < (1ll << 38);
    };
    const int64_t sv = a.sdtype == CC1D_F32 ? 4 : 8;
    return a.dtype == CC1D_BF16 && a.dk == DK && a.dv % 32 == 0 && a.q_sd == 1 && a.k_sd == 1 &&
           a.v_sd == 1 && a.o_sd == 1 && map_ok(a.q, a.q_st, a.q_sh) && map_ok(a.k, a.k_st, a.k_sh) &&
           map_ok(a.v, a.v_st, a.v_sh) && rows_ok(a.out, a.o_st, a.o_sh, 8) &&
           rows_ok(a.states, a.s_slot, a.s_sh, sv) && a.s_sk % sv == 0 &&
           a.tokens >= 16 * a.rows && encoder() != nullptr;
}

cudaError_t launch_gdr_chunk(const cc1d_gdr_args& a, cudaStream_t stream) {
    const bool out32 = host_aligned32(a.out) && a.o_st % 16 == 0 && a.o_sh % 16 == 0;
    return a.sdtype == CC1D_F32 ? pick<float>(a, out32, stream) : pick<bf16>(a, out32, stream);
}

}  // namespace cc1d
