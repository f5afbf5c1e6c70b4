// Gated delta rule in chunks, first kernel: everything of a chunk that does not depend on the state.
// gdr_chunk.cu has the mathematics; here, per chunk of 64 tokens and value head,
//     L_ij = beta_i r_i r_j e^(b_i - b_j) k_i.k_j  (j < i),   T = (I + L)^-1 diag(beta),
//     P_ij = s_i r_j e^(b_i - b_j) q_i.k_j         (j <= i),  G = P T,
// and the row factors of the scan. The chunks are independent, so latency is hidden by three
// CTAs per SM (fp16: two) rather than inside one.
//
// A CTA of four warps takes one chunk of one query/key head: K and Q by TMA, [K;Q] K^T on the tensor
// core and the norms once, then the value heads of the group one after another. The inverse goes in
// blocks: 16 x 16 by substitution in registers (a lane owns a row, rows of L come as broadcasts),
// the blocks below the diagonal by -inv_1 (L_21 inv_0) in three-part bf16 on the warp-level tensor
// core (120 dependent fp32 steps a row instead of the 2016 of plain substitution). G is a product on
// the tensor core again. T leaves by a bulk copy, G from registers.
//
// Bound: instruction latency and issue, with 12 warps an SM (the parts of T and P leave shared memory
// for three CTAs). 30600 chunks and heads take 632 us, 1.5 GB written. With T, P and G in two parts and
// four CTAs it was 424 us (6200 warp instructions per chunk and value head at 0.4 a cycle and
// scheduler). Plain substitution over the whole chunk took 5000 to 15000 cycles for the inverse alone.
#include "gdr_chunk.cuh"

namespace cc1d {
namespace {

constexpr int LPAD = 36;  // fp32 row of a 32 x 32 block: 16-byte accesses of 8 rows hit 8 bank groups
constexpr int kHeads = 4;  // value heads whose gates are made at a time, one warp each

// I + L in 32 x 32 blocks, fp32: the diagonal blocks (L, then their inverses in place) and the
// block below them.
struct Blocks {
    float diag[2][32][LPAD], low[32][LPAD];
};
// What a chunk's gates give: cumulative log2 decays b, negated, in two parts each; rates; decays
// e^(b_i), e^(b_C - b_j) and, below 32, e^(b_31 - b_j).
struct Gates {
    alignas(16) float nbh[C], nbl[C], beta[C], grow[C], out[C], far[32];
};

template <bool kLo>
struct Smem {
    // K and Q; later the parts of T, then those of P
    unsigned char kq[Parts<kLo>::kBytes > 6 * 8192 ? Parts<kLo>::kBytes : 6 * 8192];
    Blocks blk;
    Gates gates[kHeads];
    alignas(16) float rk[C], ru[kHeads][32];  // inverse norms of the keys; with e^(b_31 - b_j)
    uint64_t full, mma, last;
    uint32_t tmem;
    int abort, late, seq;
};

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
// The same of operands in three parts, the smallest products first: a sum is cut to fp32 after every
// step. The products left out are 2^-27 of the whole.
__device__ __forceinline__ void mma_warp_parts(float* d, const uint32_t (*a)[4], const uint32_t (*b)[2]) {
    mma_warp(d, a[0], b[2]);
    mma_warp(d, a[2], b[0]);
    mma_warp(d, a[1], b[1]);
    mma_warp(d, a[0], b[1]);
    mma_warp(d, a[1], b[0]);
    mma_warp(d, a[0], b[0]);
}

// The 16 x 16 tile inv1[r0.., :] (low inv0)[:, c0..] of a product of K x K matrices, K = 16 or 32,
// by one warp in three-part bf16. The inner product is formed transposed, (inv0^T low^T): its
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
        uint32_t av[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = c0 + g + e % 2 * 8, r = 16 * k + t2 + e / 2 * 8;
            split3(make_float2(inv0[r][col], inv0[r + 1][col]), av[0][e], av[1][e], av[2][e]);
        }
#pragma unroll
        for (int n = 0; n < K / 8; ++n) {
            uint32_t bv[3][2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                split3(*reinterpret_cast<const float2*>(&low[8 * n + g][16 * k + t2 + 8 * e]), bv[0][e], bv[1][e], bv[2][e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) m[k][n][e] = 0.f;
            mma_warp_parts(m[k][n], av, bv);
        }
    }
    float s[K / 16][2][4];
#pragma unroll
    for (int k = 0; k < K / 16; ++k) {
        uint32_t av[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            split3(*reinterpret_cast<const float2*>(&inv1[r0 + g + e % 2 * 8][16 * k + t2 + e / 2 * 8]), av[0][e], av[1][e], av[2][e]);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            uint32_t bv[3][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float2 f = make_float2(m[0][2 * k + e][2 * n], m[0][2 * k + e][2 * n + 1]);
                if (K > 16)
                    f = __fadd2_rn(f, make_float2(m[K / 16 - 1][2 * k + e][2 * n], m[K / 16 - 1][2 * k + e][2 * n + 1]));
                split3(f, bv[0][e], bv[1][e], bv[2][e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[k][n][e] = 0.f;
            mma_warp_parts(s[k][n], av, bv);
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

template <bool kLo>
__global__ void __launch_bounds__(128, kLo ? 2 : 3)
gdr_prep_kernel(const __grid_constant__ cc1d_gdr_args a, const __grid_constant__ CUtensorMap mapq,
                const __grid_constant__ CUtensorMap mapk, Sequences seqs, int64_t wait_ns) {
    extern __shared__ __align__(1024) unsigned char raw[];
    Smem<kLo>& sh = *reinterpret_cast<Smem<kLo>*>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
    const uint32_t kq = smem_addr(sh.kq), tb = kq, pb = kq + 24576;
    const int p = threadIdx.x, w = p / 32, lane = p % 32, i = p % C;
    const int hk = blockIdx.x % a.heads_k;
    const int64_t image = blockIdx.x / a.heads_k;

    // The scan kernel may come up (its CTAs wait there for this kernel's end).
    allow_dependent_launch();
    // The sequence whose chunk this is.
    if (p == 0) sh.seq = -1;
    __syncthreads();
    const int64_t n_seqs = seqs.list != nullptr ? seqs.list[0] : seqs.n;
    for (int64_t n = p; n < n_seqs; n += 128) {
        const int64_t at = seqs.list != nullptr ? seqs.list[2 + n] : n;
        const int64_t t0 = a.query_start_loc[at], t1 = a.query_start_loc[at + 1];
        if (t0 < 0 || t1 <= t0 || t1 > a.tokens) continue;
        const int64_t first = chunk_base(t0, n);
        if (image >= first && image < first + (t1 - t0 + C - 1) / C) sh.seq = (int)n;
    }
    __syncthreads();
    const int seq = sh.seq;
    int64_t tok0, slot;
    int ntok;
    if (seq < 0 || !gdr_row(a, true, seqs.list != nullptr ? seqs.list[2 + seq] : seq, tok0, ntok, slot, false)) return;
    const int c = (int)(image - chunk_base(tok0, seq));
    tok0 += c * C;
    const int left = ntok - c * C;

    if (p == 0) {
        mbar_init(smem_addr(&sh.full), 1);
        mbar_init(smem_addr(&sh.mma), 1);
        mbar_init(smem_addr(&sh.last), 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.abort = sh.late = 0;
    }
    if (w == 0) {
        tmem_alloc(smem_addr(&sh.tmem), 128);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t D0 = sh.tmem, DG = D0 + 64;  // [K;Q] K^T; G
    const uint32_t lanes = (uint32_t)w << 21;   // the warp's first TMEM lane, in bits 16..
    if (p == 0 && wait_ns > 0) {
        const uint32_t full = smem_addr(&sh.full);
        mbar_expect(full, Parts<kLo>::kBytes);
        load_kq<kLo>(kq, &mapk, &mapq, hk, (int)tok0, full);
    }

    // Gates of one value head by one warp, two tokens a lane: the loads, all at once, and the rest.
    const int group = a.heads_v / a.heads_k;
    uint32_t g_bits[2] = {0, 0}, b_bits[2] = {0, 0}, rate_bits = 0, dt_bits = 0;
    auto load_gates = [&](int h) {
        if (a.a_log != nullptr) {
            rate_bits = load_bits(a.a_log, h, a.pdtype);
            dt_bits = load_bits(a.dt_bias, h, a.pdtype);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int64_t t = tok0 + 2 * lane + e;
            if (2 * lane + e < left) {
                g_bits[e] = load_bits(a.g, t * a.g_st + h * a.g_sh, a.gdtype);
                b_bits[e] = load_bits(a.beta, t * a.b_st + h * a.b_sh, a.bdtype);
            }
        }
    };
    auto make_gates = [&](Gates& to) {
        const float rate = -expf(bits_value(rate_bits, a.pdtype)), dt = bits_value(dt_bits, a.pdtype);
        double sum[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float g = 0.f, beta = 0.f;
            if (2 * lane + e < left) {
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
            // The sums are carried in 64 bits and kept as two fp32 parts: their differences are
            // exponents, where fp32 sums of strong decays would lose the weak ones.
            sum[e] = (double)g * 1.4426950408889634;
        }
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
    if (w < group) load_gates(hk * group + w);
    if (w < group) make_gates(sh.gates[w]);

    mbar_wait(smem_addr(&sh.full), 0, &sh.abort, wait_ns);
    if (left < C) {
        // The copies went on into the next sequence: zeros there, whatever it holds.
        for (int e = p; e < (C - left) * 32; e += 128) {
            const int r = left + e / 32, u = e % 16;
#pragma unroll
            for (int part = 0; part <= (kLo ? 1 : 0); ++part)
                sts16(kq + part * 32768 + (u >> 3) * 16384 + swz<128>(r + (e & 16) * 4, u & 7), 0, 0, 0, 0);
        }
        fence_async_smem();
    }
    __syncthreads();
    uint32_t phase = 0;
    if (p == 0) {
        tc_fence_after();
        const uint64_t d = operand(kq, 16, 1024, kSwizzle128);
        if constexpr (kLo) {
            // lo lo, then hi lo and lo hi, over the halves of dk
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint64_t lo = d + half * 1024 + 2048;
                mma_steps<4, 2, 2>(D0, lo, lo, mma_desc(64, false, false), half > 0);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint64_t hi = d + half * 1024, lo = hi + 2048;
                mma_steps<4, 2, 2>(D0, hi, lo, mma_desc(64, false, false), true);
                mma_steps<4, 2, 2>(D0, lo, hi, mma_desc(64, false, false), true);
            }
        }
        mma_steps<4, 2, 2>(D0, d, d, mma_desc(64, false, false), kLo);
        mma_steps<4, 2, 2>(D0, d + 1024, d + 1024, mma_desc(64, false, false), true);
        mma_commit(smem_addr(&sh.mma));
    }
    // Norm of row p of [K;Q].
    float norm = 1.f;
    if (a.l2norm) {
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 4
        for (int u = 0; u < 16; ++u) {
            const uint32_t at = kq + (u >> 3) * 16384 + swz<128>(p, u & 7);
            const uint4 v = lds16(at), l = kLo ? lds16(at + 32768) : make_uint4(0, 0, 0, 0);
            const uint32_t vv[4] = {v.x, v.y, v.z, v.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float2 f = bf16_pair(vv[e]);
                if (kLo) f = add_pair<bf16>(ll[e], f);
                sum[e % 2] = __ffma2_rn(f, f, sum[e % 2]);
            }
        }
        norm = rsqrtf((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y) + kL2Eps);
    }
    if (p < C) sh.rk[p] = norm;
    __syncthreads();
    sh.ru[w][lane] = sh.rk[lane] * sh.gates[w].far[lane];
    mbar_wait(smem_addr(&sh.mma), phase, &sh.abort, wait_ns);
    phase ^= 1;
    // K and Q are through; T and P are zero above their diagonal blocks from here on.
    if (p < 32) {
#pragma unroll
        for (int u = 4; u < 8; ++u) {
#pragma unroll
            for (int m = 0; m < 6; ++m) sts16(kq + m * 8192 + swz<128>(p, u), 0, 0, 0, 0);
        }
    }
    __syncthreads();
    tc_fence_after();

    Blocks& blk = sh.blk;
    // G of value head h, once its product is there: rows 64.. of the product, by warps 2 and 3.
    auto store_g = [&](int h) {
        ChunkImage* out = static_cast<ChunkImage*>(a.workspace) + image * a.heads_v + h;
        mbar_wait(smem_addr(&sh.mma), phase, &sh.abort, wait_ns);
        phase ^= 1;
        tc_fence_after();
#pragma unroll 1
        for (int o = 0; o < C; o += 16) {
            float2 x[8];
            tmem_ld16(DG + lanes + o, x);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t g[3][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) split3(x[4 * u + e], g[0][e], g[1][e], g[2][e]);
                const uint32_t at = swz<128>(p, o / 8 + u);
#pragma unroll
                for (int m = 0; m < 3; ++m) st16(out->tg[m] + at, make_uint4(g[m][0], g[m][1], g[m][2], g[m][3]));
            }
        }
        tc_fence_before();
    };
#pragma unroll 1
    for (int v = 0; v < group; ++v) {
        const int h = hk * group + v;
        if (v > 0 && v % kHeads == 0) {
            if (v + w < group) {
                load_gates(h + w);
                make_gates(sh.gates[w]);
            }
            __syncwarp();
            sh.ru[w][lane] = sh.rk[lane] * sh.gates[w].far[lane];
            __syncthreads();
        }
        const Gates& ga = sh.gates[v % kHeads];
        ChunkImage* out = static_cast<ChunkImage*>(a.workspace) + image * a.heads_v + h;
        const float mul = norm * (p < C ? ga.beta[i] : a.scale);  // of row i of L or P
        out->in[p] = ga.grow[i] * (p < C ? norm : mul);
        if (p < C) out->out[i] = norm * ga.out[i];
        if (p == C - 1) {
            out->decay = ga.grow[i];
            out->failed = 0;
        }
        // The head before: its G, while warps 0 and 1 are at L and its inverse.
        if (p >= C && v > 0) store_g(h - 1);
        // Warps 0 and 1 make L (columns j < i) of rows of K K^T, warps 2 and 3 make P (columns
        // j <= i) of rows of Q K^T. In the columns of a row's own half the decay e^(b_i - b_j) is
        // taken element by element; for the lower left block it splits at the middle of the chunk
        // into two factors of at most 1.
        const float2 bh = make_float2(-ga.nbh[i], -ga.nbh[i]), bl = make_float2(-ga.nbl[i], -ga.nbl[i]);
        const float low_mul = mul * exp2_approx((bh.x + ga.nbh[31]) + (bl.x + ga.nbl[31]));
#pragma unroll 1
        for (int hf = 0; hf <= w % 2; ++hf) {
            const bool own = hf == w % 2;
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
                        const float4 r4 = *reinterpret_cast<const float4*>(&sh.ru[v % kHeads][o + 2 * e]);
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
                        store_split8(at, 8192, x + 4 * u);
                    }
                }
            }
        }
        if (p < C) {
            // Inverse of this warp's diagonal block: its two 16 x 16 blocks by substitution, a half
            // warp each, then the block below them, -inv_1 (L_21 inv_0).
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
        // The bulk copies of the T before have read it.
        if (p == 96) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncthreads();
        {
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
                    uint32_t x[3];
                    split3(__fmul2_rn(make_float2(d[n][2 * e], d[n][2 * e + 1]), bt), x[0], x[1], x[2]);
                    const uint32_t at = tb + swz<128>(32 + fr + 8 * e, col / 8) + col % 8 * 2;
#pragma unroll
                    for (int m = 0; m < 3; ++m)
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + m * 8192), "r"(x[m]) : "memory");
                }
            }
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
                const uint32_t at = tb + swz<128>(r, r / 32 * 4 + o / 8 + u);
                store_split8(at, 8192, f);
            }
        }
        fence_async_smem();
        tc_fence_before();
        __syncthreads();
        if (p == 96) {
            // A thread of the warps that wait for this product next.
            tc_fence_after();
            // G = P T in rows 64.., by parts. The 8 KB before a part of P are other parts of T or P;
            // the rows 0..63 they make are of no use.
            const uint64_t P = operand(pb - 8192, 16, 1024, kSwizzle128);
            const uint64_t T = operand(tb, 16384, 1024, kSwizzle128);
#pragma unroll
            for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                for (int m = 0; m <= sum; ++m)
                    mma_steps<4, 2, 128>(DG, P + m * 512, T + (sum - m) * 512, mma_desc(64, false, true),
                                         sum < 2 || m > 0);
            mma_commit(smem_addr(&sh.mma));
#pragma unroll
            for (int part = 0; part < 3; ++part)
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], 8192;" ::"l"(
                                 out->tg[part]), "r"(tb + part * 8192)
                             : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        __syncwarp();
    }
    if (p >= C) store_g(hk * group + group - 1);
    if (p == 96) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncthreads();
    tc_fence_after();
    if (sh.abort) {
        // What the two threads that issue products have issued.
        if (p == 0 || p == 96) mma_commit(smem_addr(&sh.last));
        if (p == 0) {
            mbar_wait(smem_addr(&sh.last), 0, &sh.late, kDrainNs);
            if (wait_ns > 0) mbar_wait(smem_addr(&sh.full), 0, &sh.late, kDrainNs);
        }
        for (int v = p; v < group; v += 128)
            (static_cast<ChunkImage*>(a.workspace) + image * a.heads_v + hk * group + v)->failed = 1;
        if (p == 0) flag_status(a.dev_status, CC1D_DEV_TIMEOUT);
        __syncthreads();
    }
    if (w == 0) tmem_dealloc(sh.tmem, 128);
}

// fp16 keys and queries to bf16 parts, four values a lane; bound by HBM. One warp per token and head.
__global__ void __launch_bounds__(256)
gdr_split_kernel(const __grid_constant__ cc1d_gdr_args a, uint2* to) {
    const int64_t item = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
    if (item >= a.tokens * a.heads_k) return;
    const int64_t t = item / a.heads_k;
    const int h = (int)(item - t * a.heads_k), lane = threadIdx.x % 32;
    const f16* src[2] = {static_cast<const f16*>(a.k) + t * a.k_st + h * a.k_sh,
                         static_cast<const f16*>(a.q) + t * a.q_st + h * a.q_sh};
    uint2* dst = to + item * (4 * DK / 4) + lane;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const uint2 v = ldg_raw<8>(src[m] + 4 * lane);
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
        uint2 hi, lo;
        split2(x, hi.x, lo.x);
        split2(y, hi.y, lo.y);
        dst[m * (DK / 4)] = hi;
        dst[(2 + m) * (DK / 4)] = lo;
    }
}

// Lists at most `most_listed` sequences of more than kLong tokens, in order: those above the smallest of
// kLong, 2 kLong, 4 kLong, .. tokens that leaves so few. One CTA.
__global__ void __launch_bounds__(1024)
gdr_list_kernel(const __grid_constant__ cc1d_gdr_args a, int most_listed, int32_t* list) {
    __shared__ int above[27], warp_sum[32], most;  // above[k]: sequences of more than kLong 2^k tokens
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    auto length = [&](int64_t n) {
        int64_t tok0, slot;
        int ntok;
        return n < a.rows && gdr_row(a, true, n, tok0, ntok, slot, false) ? ntok : 0;
    };
    if (tid < 27) above[tid] = 0;
    __syncthreads();
    for (int64_t n = tid; n < a.rows; n += 1024) {
        const int ntok = length(n);
        for (int k = 0; k < 26 && ntok > ((int64_t)kLong << k); ++k) atomicAdd(&above[k], 1);
    }
    __syncthreads();
    if (tid == 0) {
        int k = 0;
        while (above[k] > most_listed) ++k;  // above[26] is 0
        list[0] = above[k];
        list[1] = most = k < 26 ? kLong << k : INT32_MAX;
    }
    __syncthreads();
    int base = 0;
    for (int64_t at = 0; at < a.rows; at += 1024) {
        const bool on = length(at + tid) > most;
        const unsigned mask = __ballot_sync(~0u, on);
        __syncthreads();
        if (lane == 0) warp_sum[warp] = __popc(mask);
        __syncthreads();
        int before = 0, all = 0;
        for (int m = 0; m < 32; ++m) {
            before += m < warp ? warp_sum[m] : 0;
            all += warp_sum[m];
        }
        if (on) list[2 + base + before + __popc(mask & ((1u << lane) - 1u))] = (int32_t)(at + tid);
        base += all;
    }
}

}  // namespace

cudaError_t launch_gdr_list(const cc1d_gdr_args& a, const Sequences& seqs, int32_t* list,
                            cudaStream_t stream) {
    gdr_list_kernel<<<1, 1024, 0, stream>>>(a, (int)seqs.n, list);
    return cudaGetLastError();
}

cudaError_t launch_gdr_prep(const cc1d_gdr_args& a, const Sequences& seqs, const CUtensorMap& q,
                            const CUtensorMap& k, cudaStream_t stream) {
    const int64_t grid = chunk_slots(a.tokens, seqs.n) * a.heads_k;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    auto go = [&](auto lo) {
        constexpr bool kLo = decltype(lo)::value;
        constexpr int smem = (int)sizeof(Smem<kLo>) + 1024;
        static SmemLimit limit;
        const cudaError_t err = limit.raise(gdr_prep_kernel<kLo>, smem);
        if (err != cudaSuccess) return err;
        gdr_prep_kernel<kLo><<<(unsigned)grid, 128, smem, stream>>>(a, q, k, seqs, wait_limit_ns());
        return cudaGetLastError();
    };
    return a.dtype == CC1D_F16 ? go(std::true_type()) : go(std::false_type());
}

cudaError_t launch_gdr_split(const cc1d_gdr_args& a, void* to, cudaStream_t stream) {
    const int64_t grid = ceil_div(a.tokens * a.heads_k, 8);
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    gdr_split_kernel<<<(unsigned)grid, 256, 0, stream>>>(a, static_cast<uint2*>(to));
    return cudaGetLastError();
}

}  // namespace cc1d
