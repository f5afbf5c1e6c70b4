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
//   - a prep warpgroup: [K;Q] K^T on the tensor core, L, its inverse, T and G = P T. Nothing of it
//     depends on the state, so it runs ahead of the chain;
//   - NG scan warpgroups, each with the chain of its own columns: [K;Q] S0, R, [T;G] R, u, K^T u, S.
//     Two chains in a CTA fill each other's waits and share K, Q, T and G. K, Q and V come by TMA
//     up to three chunks ahead.
// Stacking K over Q and T over G makes every product M = 128, the full tensor core rate; the two
// parts of an operand lie side by side as one operand of 2 VS columns (measured: a K step of 16
// costs 46 cycles up to 64 columns and 66 with 128, so one wide step beats two narrow ones).

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

// I + L in 32 x 32 blocks, fp32: the diagonal blocks (L, then their inverses in place), the block
// below them, and L_21 inv_0 transposed.
struct Blocks {
    float diag[2][32][LPAD], low[32][LPAD], prod[32][LPAD];
};

template <int VS, int NG>
struct Layout {
    static constexpr int kRow = VS >= 64 ? 128 : 2 * VS;  // bytes of an operand row of VS columns
    static constexpr int kS = 128 * kRow;                 // one part (hi or lo) of S
    static constexpr int kR = C * kRow;                   // one part of R or u, or one tile of V
    static constexpr int kStages = NG == 1 ? 3 : 2;       // of K, Q, V
    static constexpr int KQ = 0;                          // stages x [2 halves][128 rows][128 B]
    static constexpr int V = KQ + kStages * 32768;        // stages x NG x [64 rows]
    static constexpr int TG = V + kStages * NG * kR;      // [hi, lo][128 rows][128 B]
    static constexpr int SB = TG + 32768;                 // NG x (S hi, S lo); R in S hi, u in S lo
    static constexpr int B = SB + NG * 2 * kS;            // Blocks
    static constexpr int VEC = B + (int)sizeof(Blocks);   // 2 stages x Vectors
    static constexpr int END = VEC + 2 * (int)sizeof(Vectors);
    static constexpr int kTmem = 128 + NG * 2 * VS <= 256 ? 256 : 512;
    static constexpr int kThreads = 128 * (NG + 1);
};

struct Shared {
    uint64_t tma_full[3], kq_full[3], vec_full[2], tg_full, tg_free, prep_mma, scan_mma[2];
    uint32_t tmem;
    int abort;
    int row;  // sequence of this CTA
    int done[3];  // per stage: scan warpgroups that are through with its K, Q and V, over all chunks
    int len[kOrderMax];
    alignas(16) float bh[C], bl[C], rk[C], ru[32], beta[C];
    double half;
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
__device__ __forceinline__ void store_split8(uint32_t hi, uint32_t lo, const float* f) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split2(f[2 * i], f[2 * i + 1], h[i], l[i]);
    sts16(hi, h[0], h[1], h[2], h[3]);
    sts16(lo, l[0], l[1], l[2], l[3]);
}

// Row i of the inverse of I + l (l strictly lower triangular, 32 x 32, zeros above) by backward
// substitution: y_m is final once every later y has been taken out of it, and is then taken out of
// the earlier ones along row m of l. A lane owns a row; the rows of l come as broadcasts.
__device__ __forceinline__ void solve_row(const float (*l)[LPAD], int i, float* y) {
    float2 acc[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) acc[q] = make_float2(i == 2 * q ? 1.f : 0.f, i == 2 * q + 1 ? 1.f : 0.f);
#pragma unroll
    for (int m = 31; m > 0; --m) {
        const float v = -(m % 2 ? acc[m / 2].y : acc[m / 2].x);
        const float2 vv = make_float2(v, v);
#pragma unroll
        for (int r = 0; r < m; r += 4) {
            const float4 f = *reinterpret_cast<const float4*>(&l[m][r]);
            acc[r / 2] = __ffma2_rn(make_float2(f.x, f.y), vv, acc[r / 2]);
            if (r + 2 < m) acc[r / 2 + 1] = __ffma2_rn(make_float2(f.z, f.w), vv, acc[r / 2 + 1]);
        }
    }
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        y[2 * q] = acc[q].x;
        y[2 * q + 1] = acc[q].y;
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

// The warp's 16 x 16 tile at (r0, c0) of a 32 x 32 product a b, in two-part bf16. a is row-major;
// b is row-major, or transposed (kBt). d: two 16 x 8 accumulator fragments.
template <bool kBt>
__device__ __forceinline__ void block_product(const float (*a)[LPAD], const float (*b)[LPAD], int r0,
                                              int c0, int lane, float (*d)[4]) {
    const int g = lane / 4, t2 = lane % 4 * 2;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[n][e] = 0.f;
#pragma unroll
    for (int k0 = 0; k0 < 32; k0 += 16) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = *reinterpret_cast<const float2*>(&a[r0 + g + e % 2 * 8][k0 + t2 + e / 2 * 8]);
            split2(f.x, f.y, ah[e], al[e]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            uint32_t bh[2], bl[2];
            const int col = c0 + 8 * n + g;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = k0 + t2 + 8 * e;
                const float2 f = kBt ? *reinterpret_cast<const float2*>(&b[col][k])
                                     : make_float2(b[k][col], b[k + 1][col]);
                split2(f.x, f.y, bh[e], bl[e]);
            }
            mma_warp(d[n], ah, bh);
            mma_warp(d[n], ah, bl);
            mma_warp(d[n], al, bh);
        }
    }
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
    extern __shared__ __align__(1024) unsigned char raw[];
    __shared__ Shared sh;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    unsigned char* gen = raw + (base - smem_addr(raw));
    Vectors* vec = reinterpret_cast<Vectors*>(gen + Lay::VEC);
    Blocks& blk = *reinterpret_cast<Blocks*>(gen + Lay::B);

    const int tid = threadIdx.x, warp = tid / 32, p = tid % 128;
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
            mbar_init(smem_addr(&sh.tma_full[i]), 1);
            mbar_init(smem_addr(&sh.kq_full[i]), 1);
            sh.done[i] = 0;
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&sh.vec_full[i]), 1);
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
    const uint32_t lanes = (uint32_t)(warp % 4) << 21;  // the warp's first TMEM lane, in bits 16..
    const uint32_t tg = base + Lay::TG;

    // K, Q and V of chunk c into stage st, which must be free; one thread.
    constexpr int kStages = Lay::kStages;
    auto load = [&](int c, int st) {
        const uint32_t full = smem_addr(&sh.tma_full[st]), kq = base + Lay::KQ + st * 32768;
        const int t = (int)tok0 + c * C;
        mbar_expect(full, 32768 + NG * C * VS * 2);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            tma_load(kq + half * 16384, &mapk, half * 64, hk, t, full);
            tma_load(kq + half * 16384 + 8192, &mapq, half * 64, hk, t, full);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
            tma_load(base + Lay::V + (st * NG + g) * Lay::kR, &mapv, (vt * NG + g) * VS, h, t, full);
    };
    if (tid == 0) {
        for (int c = 0; c < kStages && c < chunks; ++c) load(c, c);
    }

    if (warp >= 4 * NG) {
        // --------------------------------------------------------------------------------- prep
        const int w = warp % 4, lane = tid % 32, i = p % C;
        const uint32_t D0 = tmem;  // 64 columns of [K;Q] K^T; later 128 of P [T hi | T lo]
        const int64_t g0 = tok0 * a.g_st + h * a.g_sh, b0 = tok0 * a.b_st + h * a.b_sh;
        // T is zero above its diagonal blocks; nothing writes there again.
        if (p < 32) {
#pragma unroll
            for (int u = 4; u < 8; ++u) {
                sts16(tg + swz<128>(p, u), 0, 0, 0, 0);
                sts16(tg + 16384 + swz<128>(p, u), 0, 0, 0, 0);
            }
        }
        float rate = 0.f, dt = 0.f;
        if (a.a_log != nullptr) {
            rate = -expf(load_any(a.a_log, h, a.pdtype));
            dt = load_any(a.dt_bias, h, a.pdtype);
        }
        uint32_t g_bits = 0, b_bits = 0;
        auto load_gate_bits = [&](int c) {
            const int64_t t = (int64_t)c * C + p;
            if (p < C && t < ntok) {
                g_bits = load_bits(a.g, g0 + t * a.g_st, a.gdtype);
                b_bits = load_bits(a.beta, b0 + t * a.b_st, a.bdtype);
            }
        };
        load_gate_bits(0);

        int st = 0;
        uint32_t st_phase = 0;
        for (int c = 0; c < chunks; ++c) {
            Vectors& ve = vec[c & 1];
            const uint32_t kq = base + Lay::KQ + st * 32768;
            const int left = ntok - c * C;
            // Gates of this chunk, bits of the next one's.
            float g = 0.f, beta = 0.f;
            if (p < C && p < left) {
                g = bits_value(g_bits, a.gdtype);
                beta = bits_value(b_bits, a.bdtype);
                if (a.a_log != nullptr) {
                    const float z = g + dt;
                    g = rate * (z > 20.f ? z : log1pf(expf(z)));
                    beta = 1.f / (1.f + expf(-beta));
                }
            }
            load_gate_bits(c + 1);
            mbar_wait(smem_addr(&sh.tma_full[st]), st_phase, &sh.abort);
            if (left < C) {
                // The copies went on into the next sequence: zeros there, whatever it holds.
                for (int e = p; e < (C - left) * 32; e += 128) {
                    const int r = left + e / 32, u = e % 16;
                    sts16(kq + (u >> 3) * 16384 + swz<128>(r + (e & 16) * 4, u & 7), 0, 0, 0, 0);
                }
                for (int e = p; e < (C - left) * (NG * VS / 8); e += 128) {
                    const int r = left + e / (NG * VS / 8), u = e % (NG * VS / 8);
                    sts16(base + Lay::V + (st * NG + u / (VS / 8)) * Lay::kR +
                              swz<Lay::kRow>(r, u % (VS / 8)), 0, 0, 0, 0);
                }
                fence_async_smem();
            }
            tc_fence_before();
            named_sync(8, 128);
            if (p == 0) {
                mbar_arrive(smem_addr(&sh.kq_full[st]));
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint32_t at = kq + (ks >> 2) * 16384 + (ks & 3) * 32;
                    mma_bf16(D0, operand(at, 16, 1024, kSwizzle128), operand(at, 16, 1024, kSwizzle128),
                             mma_desc(64, false, false), ks > 0);
                }
                mma_commit(smem_addr(&sh.prep_mma));
            }
            // While it runs: cumulative decays (threads of K rows), query norms (Q rows).
            float row_mul = a.scale;  // of row i of Q K^T; of K K^T below
            double total = 0;
            if (p < C) {
                // -1e5 decays anything to zero, and its sums stay finite where -inf would give
                // inf - inf below.
                g = g < -1e5f ? -1e5f : g;
                // The sums are carried in 64 bits and kept as two fp32 parts: their differences
                // are exponents, where fp32 sums of strong decays would lose the weak ones.
                total = (double)g * 1.4426950408889634;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const double below = __shfl_up_sync(~0u, total, o);
                    if (lane >= o) total += below;
                }
                if (p == 31) sh.half = total;
                sh.beta[p] = beta;
            } else if (a.l2norm) {
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    float f[8];
                    unpack16<bf16>(lds16(kq + (u >> 3) * 16384 + swz<128>(p, u & 7)), f);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 ff = make_float2(f[2 * e], f[2 * e + 1]);
                        sum[e % 2] = __ffma2_rn(ff, ff, sum[e % 2]);
                    }
                }
                row_mul *= rsqrtf((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y) + kL2Eps);
            }
            named_sync(8, 128);
            float far = 0.f;  // decay between token i and the middle of the chunk
            if (p < C) {
                const double mid = sh.half;
                if (p >= 32) total += mid;
                const float hi = (float)total;
                sh.bh[p] = hi;
                sh.bl[p] = (float)(total - (double)hi);
                far = exp2_approx((float)(mid - total));  // used below 32 only
            }
            mbar_wait(smem_addr(&sh.prep_mma), 0, &sh.abort);
            tc_fence_after();
            float x[C];
            tmem_ld32(D0 + lanes, x);
            tmem_ld32(D0 + lanes + 32, x + 32);
            if (p < C) {
                float d = 0.f;
#pragma unroll
                for (int j = 0; j < C; ++j) d = j == p ? x[j] : d;
                const float rk = a.l2norm ? rsqrtf(d + kL2Eps) : 1.f;
                sh.rk[p] = rk;
                if (p < 32) sh.ru[p] = rk * far;
                row_mul = beta * rk;
            }
            named_sync(8, 128);
            // Warps 0 and 1 hold rows of K K^T and make L (columns j < i), warps 2 and 3 rows of
            // Q K^T and make P (columns j <= i). In the columns of a row's own half the decay
            // e^(b_i - b_j) is taken element by element; for the lower left block it splits at the
            // middle of the chunk into two factors of at most 1.
            {
                const float bh = sh.bh[i], bl = sh.bl[i], rk = sh.rk[i];
                const float grow = exp2_approx(bh + bl);
                ve.in[p] = grow * (p < C ? rk : row_mul);
                if (p < C) {
                    ve.out[i] = rk * exp2_approx((sh.bh[C - 1] - bh) + (sh.bl[C - 1] - bl));
                    if (i == C - 1) ve.decay = grow;
                }
                const int last = p < C ? i - 1 : i;
                const float mid = sh.bh[31], mid_l = sh.bl[31];
                const float low_mul = row_mul * exp2_approx((bh - mid) + (bl - mid_l));
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    float* y = x + 32 * hf;
                    if (w % 2 == hf) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const int j = 32 * hf + e;
                            const float4 h4 = *reinterpret_cast<const float4*>(&sh.bh[j]);
                            const float4 l4 = *reinterpret_cast<const float4*>(&sh.bl[j]);
                            const float4 r4 = *reinterpret_cast<const float4*>(&sh.rk[j]);
                            const float hj[4] = {h4.x, h4.y, h4.z, h4.w}, lj[4] = {l4.x, l4.y, l4.z, l4.w};
                            const float rj[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float ex = exp2_approx((bh - hj[k]) + (bl - lj[k]));
                                y[e + k] = j + k <= last ? y[e + k] * (row_mul * rj[k]) * ex : 0.f;
                            }
                        }
                    } else if (hf == 0) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 r4 = *reinterpret_cast<const float4*>(&sh.ru[e]);
                            y[e] *= low_mul * r4.x;
                            y[e + 1] *= low_mul * r4.y;
                            y[e + 2] *= low_mul * r4.z;
                            y[e + 3] *= low_mul * r4.w;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) y[e] = 0.f;
                    }
                }
            }
            // What this thread writes into T (its row of a diagonal block) or P (its row).
            uint32_t part[2][32];
            if (w < 2) {
                float (*dg)[LPAD] = blk.diag[w];
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    if (w == 0) {
                        *reinterpret_cast<float4*>(&dg[lane][e]) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                    } else {
                        *reinterpret_cast<float4*>(&blk.low[lane][e]) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                        *reinterpret_cast<float4*>(&dg[lane][e]) =
                            make_float4(x[32 + e], x[33 + e], x[34 + e], x[35 + e]);
                    }
                }
                __syncwarp();
                solve_row(dg, lane, x);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<float4*>(&dg[lane][e]) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
#pragma unroll
                for (int e = 0; e < 32; e += 2)
                    split2(x[e] * sh.beta[32 * w + e], x[e + 1] * sh.beta[32 * w + e + 1], part[0][e / 2], part[1][e / 2]);
            } else {
#pragma unroll
                for (int e = 0; e < C; e += 2) split2(x[e], x[e + 1], part[0][e / 2], part[1][e / 2]);
            }
            named_sync(8, 128);
            if (p == 0) mbar_arrive(smem_addr(&sh.vec_full[c & 1]));
            // The block below: -inv_1 (L_21 inv_0), a 16 x 16 tile per warp.
            const int r0 = w / 2 * 16, c0 = w % 2 * 16, fr = r0 + lane / 4, fc = c0 + lane % 4 * 2;
            float d[2][4];
            block_product<false>(blk.low, blk.diag[0], r0, c0, lane, d);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) blk.prod[fc + 8 * n + e % 2][fr + e / 2 * 8] = d[n][e];
            named_sync(8, 128);
            block_product<true>(blk.diag[1], blk.prod, r0, c0, lane, d);
            // The chain's products with the previous T and G must be done with their memory.
            if (c > 0) mbar_wait(smem_addr(&sh.tg_free), (c - 1) & 1, &sh.abort);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int col = fc + 8 * n;
                const float bt0 = -sh.beta[col], bt1 = -sh.beta[col + 1];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t hi, lo;
                    split2(d[n][2 * e] * bt0, d[n][2 * e + 1] * bt1, hi, lo);
                    const uint32_t at = tg + swz<128>(32 + fr + 8 * e, col / 8) + col % 8 * 2;
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(hi) : "memory");
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 16384), "r"(lo) : "memory");
                }
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (w < 2 && u >= 4) continue;
                const uint32_t at = tg + (w < 2 ? swz<128>(i, 4 * w + u) : swz<128>(p, u));
                sts16(at, part[0][4 * u], part[0][4 * u + 1], part[0][4 * u + 2], part[0][4 * u + 3]);
                sts16(at + 16384, part[1][4 * u], part[1][4 * u + 1], part[1][4 * u + 2], part[1][4 * u + 3]);
            }
            fence_async_smem();
            tc_fence_before();
            named_sync(8, 128);
            if (p == 0) {
                tc_fence_after();
                // [T;P] T, of which the lower half is G: hi [hi | lo], then lo hi.
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma_bf16(D0, operand(tg + ks * 32, 16, 1024, kSwizzle128),
                             operand(tg + ks * 2048, 16384, 1024, kSwizzle128),
                             mma_desc(128, false, true), ks > 0);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma_bf16(D0, operand(tg + 16384 + ks * 32, 16, 1024, kSwizzle128),
                             operand(tg + ks * 2048, 16384, 1024, kSwizzle128),
                             mma_desc(64, false, true), true);
                mma_commit(smem_addr(&sh.prep_mma));
            }
            mbar_wait(smem_addr(&sh.prep_mma), 1, &sh.abort);
            tc_fence_after();
            if (w >= 2) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    tmem_ld32(D0 + lanes + 32 * hf, x);
                    tmem_ld32(D0 + lanes + 64 + 32 * hf, x + 32);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[8 * u + e] += x[32 + 8 * u + e];
                        const uint32_t at = tg + swz<128>(p, 4 * hf + u);
                        store_split8(at, at + 16384, x + 8 * u);
                    }
                }
                fence_async_smem();
            }
            tc_fence_before();
            named_sync(8, 128);
            if (p == 0) mbar_arrive(smem_addr(&sh.tg_full));
            if (++st == kStages) {
                st = 0;
                st_phase ^= 1;
            }
        }
    } else {
        // -------------------------------------------------------------------------------- scan
        const int grp = warp / 4;
        const int bar = 1 + grp;
        const uint32_t D = tmem + 128 + grp * 2 * VS;  // [product with hi parts | with lo parts]
        const uint32_t mma = smem_addr(&sh.scan_mma[grp]);
        const uint32_t s_hi = base + Lay::SB + grp * 2 * Lay::kS, s_lo = s_hi + Lay::kS;
        const uint32_t r_hi = s_hi, r_lo = r_hi + Lay::kR, u_hi = s_lo, u_lo = u_hi + Lay::kR;
        const int col = (vt * NG + grp) * VS;
        const bool initial = a.states != nullptr && a.has_initial_state != nullptr && a.has_initial_state[row];
        ST* sp = nullptr;
        if (a.states != nullptr)
            sp = static_cast<ST*>(a.states) + slot * a.s_slot + h * a.s_sh + p * a.s_sk + col;
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
        bf16* op = static_cast<bf16*>(a.out) + tok0 * a.o_st + h * a.o_sh + col;

        int st = 0;
        uint32_t phase = 0, st_phase = 0;
        for (int c = 0; c < chunks; ++c) {
            const uint32_t kq = base + Lay::KQ + st * 32768;
#pragma unroll
            for (int u = 0; u < VS / 8; ++u) {
                const uint32_t at = swz<Lay::kRow>(p, u);
                store_split8(s_hi + at, s_lo + at, S + 8 * u);
            }
            fence_async_smem();
            tc_fence_before();
            named_sync(bar, 128);
            if (p == 0) {
                mbar_wait(smem_addr(&sh.kq_full[st]), st_phase, &sh.abort);
                tc_fence_after();
                // [K;Q] S
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    mma_bf16(D, operand(kq + (ks >> 2) * 16384 + (ks & 3) * 32, 16, 1024, kSwizzle128),
                             operand(s_hi + ks * 2 * kGroup, Lay::kS, kGroup, kSwz),
                             mma_desc(2 * VS, false, true), ks > 0);
                mma_commit(mma);
            }
            mbar_wait(smem_addr(&sh.vec_full[c & 1]), (c >> 1) & 1, &sh.abort);
            const float in = vec[c & 1].in[p], decay = vec[c & 1].decay, out = vec[c & 1].out[p % C];
            float o[VS];  // rows of Q: their outputs
            mbar_wait(mma, phase, &sh.abort);
            phase ^= 1;
            tc_fence_after();
            const uint32_t vb = base + Lay::V + (st * NG + grp) * Lay::kR;
#pragma unroll
            for (int g = 0; g < VS / 16; ++g) {
                float d[16], e[16];
                tmem_ld16x2(D + lanes + 16 * g, D + lanes + VS + 16 * g, d, e);
                if (p < C) {
                    // R = V - r e^b (K S)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float f[8];
                        unpack16<bf16>(lds16(vb + swz<Lay::kRow>(p, 2 * g + u)), f);
#pragma unroll
                        for (int k = 0; k < 8; ++k) f[k] = fmaf(-in, d[8 * u + k] + e[8 * u + k], f[k]);
                        const uint32_t at = swz<Lay::kRow>(p, 2 * g + u);
                        store_split8(r_hi + at, r_lo + at, f);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[16 * g + k] = in * (d[k] + e[k]);
                }
            }
            fence_async_smem();
            tc_fence_before();
            named_sync(bar, 128);
            if (p == 0) {
                mbar_wait(smem_addr(&sh.tg_full), c & 1, &sh.abort);
                tc_fence_after();
                // [T;G] R: hi [hi | lo], then lo hi
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma_bf16(D, operand(tg + ks * 32, 16, 1024, kSwizzle128),
                             operand(r_hi + ks * 2 * kGroup, Lay::kR, kGroup, kSwz),
                             mma_desc(2 * VS, false, true), ks > 0);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma_bf16(D, operand(tg + 16384 + ks * 32, 16, 1024, kSwizzle128),
                             operand(r_hi + ks * 2 * kGroup, Lay::kR, kGroup, kSwz),
                             mma_desc(VS, false, true), true);
                mma_commit(mma);
                mma_commit(smem_addr(&sh.tg_free));
            }
            mbar_wait(mma, phase, &sh.abort);
            phase ^= 1;
            tc_fence_after();
#pragma unroll
            for (int g = 0; g < VS / 16; ++g) {
                float d[16], e[16];
                tmem_ld16x2(D + lanes + 16 * g, D + lanes + VS + 16 * g, d, e);
                if (p < C) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float f[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) f[k] = out * (d[8 * u + k] + e[8 * u + k]);
                        const uint32_t at = swz<Lay::kRow>(p, 2 * g + u);
                        store_split8(u_hi + at, u_lo + at, f);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[16 * g + k] += d[k] + e[k];
                }
            }
            fence_async_smem();
            tc_fence_before();
            named_sync(bar, 128);
            if (p == 0) {
                tc_fence_after();
                // K^T u
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma_bf16(D, operand(kq + ks * 2048, 16384, 1024, kSwizzle128),
                             operand(u_hi + ks * 2 * kGroup, Lay::kR, kGroup, kSwz),
                             mma_desc(2 * VS, true, true), ks > 0);
                mma_commit(mma);
            }
            const int t = c * C + p - C;
            if (p >= C && t < ntok) {
                bf16* to = op + (int64_t)t * a.o_st;
#pragma unroll
                for (int k = 0; k < VS; k += 16) {
                    const uint4 lo = pack16<bf16>(o + k), hi = pack16<bf16>(o + k + 8);
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
            if (p == 0 && c + kStages < chunks) {
                // The last scan warpgroup through with the chunk refills its stage.
                __threadfence_block();
                if (atomicAdd(&sh.done[st], 1) % NG == NG - 1) {
                    __threadfence_block();
                    load(c + kStages, st);
                }
            }
#pragma unroll
            for (int g = 0; g < VS / 16; ++g) {
                float d[16], e[16];
                tmem_ld16x2(D + lanes + 16 * g, D + lanes + VS + 16 * g, d, e);
#pragma unroll
                for (int k = 0; k < 16; ++k) S[16 * g + k] = fmaf(decay, S[16 * g + k], d[k] + e[k]);
            }
            if (++st == kStages) {
                st = 0;
                st_phase ^= 1;
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
