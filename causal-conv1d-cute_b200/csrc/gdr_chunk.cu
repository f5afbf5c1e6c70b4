// Gated delta rule over packed sequences, chunk by chunk on the tensor cores (bf16 and fp16, dk = 128).
//
// Mathematics. In a chunk of C = 64 tokens that starts from state S0, with b the cumulative log
// decay inside the chunk, r the inverse norms of the keys (1 without l2norm) and s those of the
// queries times the output scale:
//     L_ij = beta_i r_i r_j e^(b_i - b_j) k_i.k_j   (j < i),   T = (I + L)^-1 diag(beta)
//     P_ij = s_i r_j e^(b_i - b_j) q_i.k_j          (j <= i),  G = P T
//     R_i  = v_i - r_i e^(b_i) S0^T k_i
//     u    = T R,      o_i = s_i e^(b_i) S0^T q_i + (G R)_i
//     S    = e^(b_C) S0 + sum_j k_j (r_j e^(b_C - b_j) u_j)^T.
// k and q enter every product as the caller's bf16 values (fp16 ones as two bf16 parts), which are
// exact; norms, gates and decays scale rows in fp32 outside the products. All exponents are
// differences b_i - b_j <= 0. Within a chunk, as in any chunked form, a value that is not finite
// spoils the rows of its chunk, earlier ones included; it reaches no earlier chunk, and no other
// sequence (rows behind a sequence's end are zeroed).
//
// Precision. S, R, T, G and u are fp32 quantities. As operands they are split into three bf16 parts,
// which hold all 24 bits; of the products of two split operands those of 2^-27 are left out, and
// small products are added among themselves before they meet the large ones, because the tensor core
// cuts its sums to fp32 after every step (summed the other way the errors are two to five times as
// large). fp32 final states come out within 2.5e-7 of the definition (2-norm) where keys are random, and
// within 7e-7 where the keys of a sequence repeat and u cancels over its tokens; fp32 arithmetic token by
// token leaves up to 4e-7 and 9e-7. Two parts, which need 0.6 of the products, left 2e-6 to 9e-6, and 7e-5.
// The state itself is carried in fp32 from chunk to chunk.
//
// Split of the work. Chunks of one sequence form a chain; heads, sequences and the columns of the
// state are independent. T, G and the row factors do not depend on the state: a first kernel
// (gdr_prep.cu) makes them for all chunks in parallel and leaves them in a workspace, 50 KB per
// chunk and head. (One kernel with warps for either part was tried first: a chunk's T and G take
// longer than its step of the chain, and shared memory has no room for more of them in flight.)
// The kernel here walks the chain: [K;Q] S0, R, [T;G] R, u, K^T u, S. A CTA takes one head of one
// sequence and VS state columns; all its warps turn a product into the operand of the next together.
// K, Q, T and G come by TMA and bulk copies a chunk or two ahead.
//
// Bound. The latency of the chain: 2.2 us a chunk at VS = 32 (8192 tokens x 12 heads 285 us), of which
// the products take half and the rest is TMEM loads, splitting, barriers. Tiles of 128 columns, for
// many heads, have a kernel of their own (gdr_wide.cu). Measured with operands in two parts: 2950
// cycles a chunk at VS = 32; in this form 6800 with 128 columns, two independent chains of 64 in one CTA
// 7700, and two tiles in turn, with warps of their own for products and loads, 7400 (3500 at 32
// columns); twice the threads at 32 columns 3050.
//
// Stacking K over Q and T over G makes every product M = 128, the full tensor core rate; the parts of
// an operand lie side by side as one operand of 3 VS columns (measured: a K step of 16 costs 46 cycles
// up to 64 columns, 66 with 128 and 137 with 256, so one wide step beats two narrow ones).
#include <algorithm>

#include "gdr_chunk.cuh"

namespace cc1d {
namespace {

template <int VS, bool kLo>
struct Layout {
    static constexpr int kRow = 2 * VS;        // bytes of a row of columns
    static constexpr int kS = 128 * kRow;      // one part of S
    static constexpr int kR = C * kRow;        // one part of R or u, or V
    static constexpr int kKQ = Parts<kLo>::kBytes;
    static constexpr int kStages = 2;                  // of K, Q and the row factors
    static constexpr int kTgStages = kLo ? 1 : 2;      // of T and G
    static constexpr int KQ = 0;                       // stages x K and Q
    static constexpr int TG = KQ + kStages * kKQ;      // stages x [3 parts][128 rows][128 B]
    static constexpr int SB = TG + kTgStages * kTgBytes;  // the parts of S; in their place those of R and u
    static constexpr int V = SB + 3 * kS;              // [64 rows]
    static constexpr int VEC = V + kR;                 // stages x row factors
    static constexpr int END = VEC + kStages * kVectorBytes;
    static constexpr int kTmem = VS == 32 ? 128 : 256;  // a power of two from 3 VS on
};
constexpr int kThreads = 256;

struct Shared {
    uint64_t full[2], tg_full[2], v_full, mma, last;
    int begun[5];  // copies begun on the first five of these
    uint32_t tmem;
    int abort, late;
    int row;  // sequence of this CTA
};

// One thread: D (+)= A B over kSteps K steps, the first kParts parts of B side by side as one operand
// of kParts VS columns, whose products are added on the way out of TMEM.
template <int VS, int kParts, int kSteps, int kA, bool kTransposedA>
__device__ __forceinline__ void parts_product(uint32_t d, uint64_t a, uint64_t b, bool accumulate) {
    mma_steps<kSteps, kA, 2 * VS>(d, a, b, mma_desc(kParts * VS, kTransposedA, true), accumulate);
}

// 16 columns of a product, its parts added.
template <int VS>
__device__ __forceinline__ void load_sum(uint32_t d, float2* f) {
    float2 e[8], g[8];
    tmem_ld16_async(d, f);
    tmem_ld16_async(d + VS, e);
    tmem_ld16_async(d + 2 * VS, g);
    tmem_wait_ld();
    tmem_ready(f);
    tmem_ready(e);
    tmem_ready(g);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = __fadd2_rn(f[k], __fadd2_rn(e[k], g[k]));
}

template <typename T, typename ST, int VS>
__global__ void __launch_bounds__(kThreads, 1)
gdr_chunk_kernel(const __grid_constant__ cc1d_gdr_args a, const __grid_constant__ CUtensorMap mapq,
                 const __grid_constant__ CUtensorMap mapk, const __grid_constant__ CUtensorMap mapv,
                 int tiles, bool out32, Sequences seqs, int64_t wait_ns) {
    constexpr bool kLo = std::is_same<T, f16>::value;  // fp16 keys and queries come in two bf16 parts
    using Lay = Layout<VS, kLo>;
    constexpr uint64_t kSwz = VS == 64 ? kSwizzle128 : kSwizzle64;
    constexpr uint32_t kGroup = 8 * Lay::kRow;  // bytes of eight rows of V columns
    constexpr int kStages = Lay::kStages, kTgStages = Lay::kTgStages;
    extern __shared__ __align__(1024) unsigned char raw[];
    __shared__ Shared sh;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    unsigned char* gen = raw + (base - smem_addr(raw));
    const Vectors* vec = reinterpret_cast<const Vectors*>(gen + Lay::VEC);

    const int tid = threadIdx.x, warp = tid / 32, p = tid % 128, w = warp % 4;
    const int vt = blockIdx.x % tiles;  // columns vt * VS ..
    const int h = (int)((blockIdx.x / tiles) % a.heads_v);
    int64_t row = blockIdx.x / tiles / a.heads_v;
    const int hk = h / (a.heads_v / a.heads_k);

    int64_t seq = row;
    if (seqs.list != nullptr) {
        if (seq >= seqs.list[0]) return;
        row = seqs.list[2 + seq];
    } else {
        seq = row = longest_first(a, row, reinterpret_cast<int*>(gen), &sh.row);
    }
    int64_t tok0, slot;
    int ntok;
    if (!gdr_row(a, true, row, tok0, ntok, slot, h == 0 && vt == 0 && tid == 0)) return;
    const int chunks = (ntok + C - 1) / C;
    const ChunkImage* image =
        static_cast<const ChunkImage*>(a.workspace) + chunk_base(tok0, seq) * a.heads_v + h;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&sh.full[i]), 1);
            mbar_init(smem_addr(&sh.tg_full[i]), 1);
        }
        mbar_init(smem_addr(&sh.v_full), 1);
        mbar_init(smem_addr(&sh.mma), 1);
        mbar_init(smem_addr(&sh.last), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < 5; ++i) sh.begun[i] = 0;
        sh.abort = sh.late = 0;
    }
    if (warp == 0) {
        tmem_alloc(smem_addr(&sh.tmem), Lay::kTmem);
        tmem_relinquish();
    }
    // The bulk copies below overwrite what the ordering above kept in shared memory.
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t lanes = (uint32_t)w << 21;  // the warp's first TMEM lane, in bits 16..

    // Copies may be started: those of earlier chunks have been waited for.
    auto live = [&] { return *(volatile int*)&sh.abort == 0 && wait_ns > 0; };
    // K, Q and the row factors of chunk c into stage st, which must be free; one thread.
    auto load = [&](int c, int st) {
        if (!live()) return;
        sh.begun[st] = c / kStages + 1;
        const uint32_t full = smem_addr(&sh.full[st]);
        const ChunkImage* from = image + (int64_t)c * a.heads_v;
        mbar_expect(full, Lay::kKQ + kVectorBytes);
        load_kq<kLo>(base + Lay::KQ + st * Lay::kKQ, &mapk, &mapq, hk, (int)tok0 + c * C, full);
        bulk_load(base + Lay::VEC + st * kVectorBytes, from->in, kVectorBytes, full);
    };
    // T and G of chunk c, into the stage of their own.
    auto load_tg = [&](int c) {
        if (!live()) return;
        const int st = c % kTgStages;
        sh.begun[2 + st] = c / kTgStages + 1;
        const uint32_t full = smem_addr(&sh.tg_full[st]);
        mbar_expect(full, kTgBytes);
        bulk_load(base + Lay::TG + st * kTgBytes, image[(int64_t)c * a.heads_v].tg, kTgBytes, full);
    };
    // V of chunk c.
    auto load_v = [&](int c) {
        if (!live()) return;
        sh.begun[4] = c + 1;
        const uint32_t full = smem_addr(&sh.v_full);
        mbar_expect(full, C * VS * 2);
        tma_load(base + Lay::V, &mapv, vt * VS, h, (int)tok0 + c * C, full);
    };
    grid_dependency_wait();  // for the prep kernel's images
    if (tid == 0) {
        for (int c = 0; c < kStages && c < chunks; ++c) load(c, c);
        for (int c = 0; c < kTgStages && c < chunks; ++c) load_tg(c);
        load_v(0);
    }

    // A thread has row p and columns first .. first + W of the tile.
    constexpr int W = VS * 128 / kThreads;
    const int first = warp / 4 * W;
    const bool lead = tid == 0;
    const uint32_t D = tmem;  // products with the parts of B, side by side
    const uint32_t Dp = D + lanes + first;
    const uint32_t mma = smem_addr(&sh.mma);
    const uint32_t sb = base + Lay::SB, rb = sb, ub = rb + 3 * Lay::kR;
    const uint32_t vb = base + Lay::V;
    const int col = vt * VS + first;
    const bool initial = a.states != nullptr && a.has_initial_state != nullptr && a.has_initial_state[row];
    ST* sp = nullptr;
    if (a.states != nullptr)
        sp = static_cast<ST*>(a.states) + slot * a.s_slot + h * a.s_sh + p * a.s_sk + col;
    constexpr int SV = Vec<ST>::V;
    T* op = static_cast<T*>(a.out) + tok0 * a.o_st + h * a.o_sh + col;

    float2 s[W / 16][8];  // the state
#pragma unroll
    for (int g = 0; g < W / 16; ++g) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s[g][k] = make_float2(0.f, 0.f);
        if (initial) {
#pragma unroll
            for (int k = 0; k < 16; k += SV) unpack16<ST>(ld16(sp + 16 * g + k), &s[g][0].x + k);
        }
    }
    int st = 0;
    uint32_t phase = 0, st_phase = 0;
    float decay = 1.f;
    mbar_wait(smem_addr(&sh.full[0]), 0, &sh.abort, wait_ns);
#pragma unroll 1
    for (int c = 0;; ++c) {
        // The state after the chunk before, and as an operand if there is another.
        if (c > 0) {
#pragma unroll
            for (int g = 0; g < W / 16; ++g) {
                float2 d[8];
                load_sum<VS>(Dp + 16 * g, d);
#pragma unroll
                for (int k = 0; k < 8; ++k) s[g][k] = __ffma2_rn(make_float2(decay, decay), s[g][k], d[k]);
            }
        }
        if (c == chunks) break;
#pragma unroll
        for (int g = 0; g < W / 16; ++g)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t at = swz<Lay::kRow>(p, first / 8 + 2 * g + u);
                store_split8(sb + at, Lay::kS, s[g] + 4 * u);
            }
        const uint32_t kq = base + Lay::KQ + st * Lay::kKQ, tg = base + Lay::TG + c % kTgStages * kTgBytes;
        const int left = ntok - c * C;
        if (left < C) {
            // The copies of K went on into the next sequence: zeros there, whatever it holds
            // (rows of Q there make outputs that are not stored).
            for (int e = tid; e < (C - left) * 16; e += kThreads)
#pragma unroll
                for (int part = 0; part <= (kLo ? 1 : 0); ++part)
                    sts16(kq + part * 32768 + (e % 16 >> 3) * 16384 + swz<128>(left + e / 16, e % 8), 0, 0, 0, 0);
        }
        fence_async_smem();
        tc_fence_before();
        __syncthreads();
        if (lead) {
            tc_fence_after();
            // [K;Q] S
            const uint64_t k = operand(kq, 16, 1024, kSwizzle128), s = operand(sb, Lay::kS, kGroup, kSwz);
            parts_product<VS, 3, 4, 2, false>(D, k, s, false);
            parts_product<VS, 3, 4, 2, false>(D, k + 1024, s + kGroup / 2, true);
            if constexpr (kLo) {
                // Their sums belong to the second and third parts'.
                parts_product<VS, 2, 4, 2, false>(D + VS, k + 2048, s, true);
                parts_product<VS, 2, 4, 2, false>(D + VS, k + 3072, s + kGroup / 2, true);
            }
            mma_commit(mma);
        }
        // While it runs, a thread with little else to do (six copies take 560 cycles to issue) refills
        // the stage of the chunk before.
        if (tid == 64 && c > 0 && c - 1 + kStages < chunks) load(c - 1 + kStages, st > 0 ? st - 1 : kStages - 1);
        const float in = vec[st].in[p], out = vec[st].out[p % C];
        decay = vec[st].decay;
        if (tid == 96 && vec[st].failed) *(volatile int*)&sh.abort = 1;
        float2 q[W / 2];  // rows of Q: their outputs
        if (p < C) mbar_wait(smem_addr(&sh.v_full), c & 1, &sh.abort, wait_ns);
        mbar_wait(mma, phase, &sh.abort, wait_ns);
        phase ^= 1;
        tc_fence_after();
        if (p < C) {
            // R = V - r e^b (K S), zero behind the sequence's end, whatever V holds there
            const bool live = p < left;
#pragma unroll
            for (int g = 0; g < W / 16; ++g) {
                uint4 v[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) v[u] = lds16(vb + swz<Lay::kRow>(p, first / 8 + 2 * g + u));
                float2 d[8];
                load_sum<VS>(Dp + 16 * g, d);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t vv[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
                    float2 f[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) f[k] = add_pair<T>(live ? vv[k] : 0u, mul2(d[4 * u + k], -in));
                    store_split8(rb + swz<Lay::kRow>(p, first / 8 + 2 * g + u), Lay::kR, f);
                }
            }
            fence_async_smem();
        } else {
#pragma unroll
            for (int g = 0; g < W / 16; ++g) {
                float2 d[8];
                load_sum<VS>(Dp + 16 * g, d);
#pragma unroll
                for (int k = 0; k < 8; ++k) q[8 * g + k] = mul2(d[k], in);
            }
        }
        tc_fence_before();
        __syncthreads();
        if (lead) mbar_wait(smem_addr(&sh.tg_full[c % kTgStages]), c / kTgStages & 1, &sh.abort, wait_ns);
        if (lead) {
            tc_fence_after();
            // [T;G] R, part by part of [T;G]
            const uint64_t r = operand(rb, Lay::kR, kGroup, kSwz), g = operand(tg, 16, 1024, kSwizzle128);
            parts_product<VS, 3, 4, 2, false>(D, g, r, false);
            parts_product<VS, 2, 4, 2, false>(D + VS, g + 1024, r, true);
            parts_product<VS, 1, 4, 2, false>(D + 2 * VS, g + 2048, r, true);
            mma_commit(mma);
            if (c + 1 < chunks) load_v(c + 1);
        }
        mbar_wait(mma, phase, &sh.abort, wait_ns);
        phase ^= 1;
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < W / 16; ++g) {
            float2 d[8];
            load_sum<VS>(Dp + 16 * g, d);
            if (p < C) {
#pragma unroll
                for (int k = 0; k < 8; ++k) d[k] = mul2(d[k], out);
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    store_split8(ub + swz<Lay::kRow>(p, first / 8 + 2 * g + u), Lay::kR, d + 4 * u);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) q[8 * g + k] = __fadd2_rn(q[8 * g + k], d[k]);
            }
        }
        if (p < C) fence_async_smem();
        tc_fence_before();
        __syncthreads();
        if (lead) {
            tc_fence_after();
            // K^T u
            const uint64_t k = operand(kq, 16384, 1024, kSwizzle128), u = operand(ub, Lay::kR, kGroup, kSwz);
            parts_product<VS, 3, 4, 128, true>(D, k, u, false);
            if constexpr (kLo) parts_product<VS, 2, 4, 128, true>(D + VS, k + 2048, u, true);
            mma_commit(mma);
        }
        // [T;G] R is through: the next T and G into its place.
        if (tid == 64 && c + kTgStages < chunks) load_tg(c + kTgStages);
        const int t = c * C + p - C;
        if (p >= C && t < ntok) {
            T* to = op + (int64_t)t * a.o_st;
#pragma unroll
            for (int k = 0; k < W; k += 16) {
                const uint4 lo = pack16<T>(&q[k / 2].x), hi = pack16<T>(&q[k / 2 + 4].x);
                if (out32) {
                    st32_stream(to + k, lo, hi);
                } else {
                    st16(to + k, lo);
                    st16(to + k + 8, hi);
                }
            }
        }
        if (++st == kStages) {
            st = 0;
            st_phase ^= 1;
        }
        // The next chunk's K, Q, T, G: there by now, and the look costs less here.
        if (c + 1 < chunks) mbar_wait(smem_addr(&sh.full[st]), st_phase, &sh.abort, wait_ns);
        mbar_wait(mma, phase, &sh.abort, wait_ns);
        phase ^= 1;
        tc_fence_after();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (sh.abort) {
        // The cache keeps its state, and the outputs say that they are none.
        if (tid == 0) {
            mma_commit(smem_addr(&sh.last));
            mbar_wait(smem_addr(&sh.last), 0, &sh.late, kDrainNs);
            for (int i = 0; i < 5; ++i)
                if (sh.begun[i] > 0)
                    mbar_wait(smem_addr(sh.full) + 8 * i, (sh.begun[i] - 1) & 1, &sh.late, kDrainNs);
            flag_status(a.dev_status, CC1D_DEV_TIMEOUT);
        }
        __syncthreads();
        for (int64_t t = p - C; p >= C && t < ntok; t += C)
#pragma unroll
            for (int k = 0; k < W; k += 8) st16(op + t * a.o_st + k, nan16());
    } else if (sp != nullptr) {
#pragma unroll
        for (int g = 0; g < W / 16; ++g)
#pragma unroll
            for (int k = 0; k < 16; k += SV) st16(sp + 16 * g + k, pack16<ST>(&s[g][0].x + k));
    }
    if (warp == 0) tmem_dealloc(tmem, Lay::kTmem);
}

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

// The chunk images, in whole 128-byte lines.
int64_t images_bytes(const cc1d_gdr_args& a, const Sequences& seqs) {
    return ceil_div(chunk_slots(a.tokens, seqs.n) * a.heads_v * (int64_t)sizeof(ChunkImage), 128) * 128;
}

// Whether a batch is of mostly short sequences, and may hold long ones all the same.
bool mostly_short(const cc1d_gdr_args& a) { return a.tokens < 12 * a.rows; }

// Those that run in chunks, with their list (in the workspace, behind the rest) still to come.
Sequences sequences(const cc1d_gdr_args& a) {
    return {nullptr, mostly_short(a) ? std::min<int64_t>(kListMax, a.tokens / (kLong + 1)) : a.rows};
}
constexpr int64_t kListBytes = 256;  // of a list

template <typename T, typename ST, int VS>
cudaError_t go(const cc1d_gdr_args& a, const Sequences& seqs, const CUtensorMap& q, const CUtensorMap& k,
               bool out32, cudaStream_t stream) {
    constexpr int smem = Layout<VS, std::is_same<T, f16>::value>::END + 1024;
    const int tiles = a.dv / VS;
    const int64_t grid = seqs.n * a.heads_v * tiles;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    CUtensorMap v;
    if (!make_map(&v, a.v, a.tokens, a.heads_v, a.dv, a.v_st, a.v_sh, VS)) return cudaErrorInvalidValue;
    static SmemLimit limit;
    const cudaError_t err = limit.raise(gdr_chunk_kernel<T, ST, VS>, smem);
    if (err != cudaSuccess) return err;
    return launch_dependent(gdr_chunk_kernel<T, ST, VS>, (unsigned)grid, kThreads, smem, stream, a, q, k, v,
                            tiles, out32, seqs, wait_limit_ns());
}

template <typename T, typename ST>
cudaError_t pick(const cc1d_gdr_args& a, const Sequences& seqs, const CUtensorMap& q, const CUtensorMap& k,
                 cudaStream_t stream) {
    const bool out32 = host_aligned32(a.out) && a.o_st % 16 == 0 && a.o_sh % 16 == 0;
    // Columns per CTA. A chunk's step takes 2.2, 3.0 and 4.0 us with 32, 64 and 128 columns: wide
    // tiles do more per SM, narrow ones finish a chain sooner. Many heads (sequences x heads) take the
    // widest (bf16, uneven lengths, us with 32, 64, 128 columns: 768 heads, 16384 tokens 1006, 826, 641;
    // 336 heads 290, 236, 224; 288 heads 281, 232, 240; 240 heads 274, 226, 274), few the narrowest
    // (144 heads 262, 286, 352 in 12 sequences, 260, 298, 367 in six of 8192 tokens; 96 heads 272, 372,
    // 465; 48 heads, 4096 tokens 131, 179, 227), the more so as long as the CTAs of the longest sequences
    // find an SM of their own. With fewer than four sequences all CTAs are long ones, and a second wave
    // costs a whole chain (48 heads in one sequence 332, 273, 333; 12 heads 160, 220, 281). fp16 has no
    // tile of 64, which would load twice the keys for no more than the narrow one's speed (us with 32,
    // 128: 768 heads 1273, 853; 240 heads 340, 347 and in five sequences 1194, 1099; 192 heads 330, 380;
    // 144 heads 328, 442). Listed sequences, few as a rule, take the narrowest.
    constexpr bool kF16 = std::is_same<T, f16>::value;
    const int64_t heads = seqs.list != nullptr ? 0 : a.rows * a.heads_v;
    if (a.dv % 128 == 0 && heads * (a.dv / 128) >= (kF16 ? 222 : 296)) return launch_gdr_wide(a, q, k, stream);
    if constexpr (!kF16) {
        if (a.dv % 64 == 0 && heads * (a.dv / 32) > (a.rows >= 4 ? 592 : 148))
            return go<T, ST, 64>(a, seqs, q, k, out32, stream);
    }
    return go<T, ST, 32>(a, seqs, q, k, out32, stream);
}

}  // namespace

bool have_maps() { return encoder() != nullptr; }

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

int64_t gdr_chunk_workspace(const cc1d_gdr_args& a) {
    return images_bytes(a, sequences(a)) + (a.dtype == CC1D_F16 ? a.tokens * a.heads_k * 4 * DK * 2 : 0) +
           (mostly_short(a) ? kListBytes : 0);
}

bool gdr_chunk_serves(const cc1d_gdr_args& a) {
    constexpr int64_t kMixed = 128;
    auto rows_ok = [](const void* p, int64_t s0, int64_t s1, int64_t per) {
        return host_aligned16(p) && s0 % per == 0 && s1 % per == 0;
    };
    // What a tensor map describes: 16-byte rows, positive strides below 2^40 bytes.
    auto map_ok = [&](const void* p, int64_t st, int64_t sh) {
        return rows_ok(p, st, sh, 8) && st > 0 && sh > 0 && st < (1ll << 38) && sh < (1ll << 38);
    };
    const int64_t sv = a.sdtype == CC1D_F32 ? 4 : 8;
    // Token by token is faster up to some 12 tokens a sequence where the GPU is full, and up to 16 or 20
    // with few heads (measured: 48 heads, 128 sequences of 8, 12, 16 tokens 480, 677, 876 us, in chunks 682;
    // 12 heads, 32 sequences 35, 48, 61, chunks 51; 6 heads, 4 sequences 13, 18, 22, chunks 24). Whether a batch with fewer
    // on average holds a long sequence all the same is known on the device only: from kMixed tokens on,
    // which would take 1.2 us each in a row, the device lists those for the chunks, and the rest goes token
    // by token. 512 sequences of one token and one of 4096, 48 heads: 7243 us token by token, 2749 all in
    // chunks, 1090 like this; 64 of one and one of 100, 6 heads: 122, 52, 43. Batches without a long
    // sequence pay for launches that find nothing to do (512 of 8, 48 heads 1872 -> 1930 us; 16 of 9, 6
    // heads 18 -> 25).
    return (a.dtype == CC1D_BF16 || a.dtype == CC1D_F16) && a.dk == DK && a.dv % 32 == 0 && a.q_sd == 1 && a.k_sd == 1 &&
           a.v_sd == 1 && a.o_sd == 1 && map_ok(a.q, a.q_st, a.q_sh) && map_ok(a.k, a.k_st, a.k_sh) &&
           map_ok(a.v, a.v_st, a.v_sh) && rows_ok(a.out, a.o_st, a.o_sh, 8) &&
           rows_ok(a.states, a.s_slot, a.s_sh, sv) && a.s_sk % sv == 0 &&
           (!mostly_short(a) || (a.tokens >= kMixed && (a.steps < 1 || a.steps > kLong))) && have_maps();
}

cudaError_t launch_gdr_chunk(const cc1d_gdr_args& a, cudaStream_t stream) {
    CUtensorMap q, k;
    Sequences seqs = sequences(a);
    if (mostly_short(a)) {
        int32_t* list = reinterpret_cast<int32_t*>(static_cast<char*>(a.workspace) + gdr_chunk_workspace(a) - kListBytes);
        cudaError_t err = launch_gdr_list(a, seqs, list, stream);
        if (err == cudaSuccess) err = launch_gdr_recurrent(a, true, stream, list);
        if (err != cudaSuccess) return err;
        seqs.list = list;
    }
    if (a.dtype == CC1D_F16) {
        void* parts = static_cast<char*>(a.workspace) + images_bytes(a, seqs);
        const cudaError_t err = launch_gdr_split(a, parts, stream);
        if (err != cudaSuccess) return err;
        if (!make_map(&k, parts, a.tokens, 4 * a.heads_k, a.dk, 4 * a.heads_k * a.dk, a.dk, 64))
            return cudaErrorInvalidValue;
        q = k;
    } else if (!make_map(&q, a.q, a.tokens, a.heads_k, a.dk, a.q_st, a.q_sh, 64) ||
               !make_map(&k, a.k, a.tokens, a.heads_k, a.dk, a.k_st, a.k_sh, 64)) {
        return cudaErrorInvalidValue;
    }
    const cudaError_t err = launch_gdr_prep(a, seqs, q, k, stream);
    if (err != cudaSuccess) return err;
    if (a.dtype == CC1D_F16)
        return a.sdtype == CC1D_F32 ? pick<f16, float>(a, seqs, q, k, stream) : pick<f16, f16>(a, seqs, q, k, stream);
    return a.sdtype == CC1D_F32 ? pick<bf16, float>(a, seqs, q, k, stream) : pick<bf16, bf16>(a, seqs, q, k, stream);
}

}  // namespace cc1d
