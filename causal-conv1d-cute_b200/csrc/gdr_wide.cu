// Gated delta rule over packed sequences, the scan of gdr_chunk.cu with 128 state columns to a CTA.
//
// The mathematics, the images of the prep kernel, the precision and the loop are those of
// gdr_chunk.cu, transposed: state columns lie along M, so
//     [K;Q] S  is  S^T [K;Q]^T,    [T;G] R  is  R^T [T;G]^T,    K^T u  is  u^T K.
// The operands that the CTA makes (S, R, u, in three bf16 parts) are then the A of their products,
// which the tensor core reads from tensor memory: shared memory holds copies only, and every warp
// has a share of every row (with the rows of K and Q along M, the warps of two of the SM's four
// partitions made all of R and u). The state stays in registers, fp32. R, u and the outputs use
// the matrix fragment shapes of tensor memory, so that V comes in and outputs go out by transposes of
// 8 x 8 matrices instead of 2-byte accesses.
//
// Bound. The products, 60 steps of some 76 cycles and their latency, take two thirds of a chunk; the
// rest is splitting S, R and u, outputs and waits. 40807 tokens x 48 heads: 937 us. Measured on the way
// with operands in two parts (36 steps): the form of gdr_chunk.cu 845 us; products issued by a worker
// (58 cycles a step, which it waits for) 812; by a warp of their own, 739; outputs read before the last
// product is issued, since a TMEM load that starts beside a product waits for its end, 708; fragments
// instead of a row to a thread for V and the outputs, 691; rows of the state by thread, 687. Slower:
// those reads in flight across the arrival (772), the state's update and split interleaved in two
// halves (726).
#include "gdr_chunk.cuh"

namespace cc1d {
namespace {

constexpr int VS = 128;
constexpr int kWorkers = 512, kThreads = kWorkers + 64;  // a warp each issues products and copies

template <bool kLo>
struct Layout {
    static constexpr int kKQ = Parts<kLo>::kBytes;
    static constexpr int kStages = 2;                      // of K, Q and the row factors
    static constexpr int kTgStages = kLo ? 1 : 2;          // of T and G
    static constexpr int KQ = 0;                           // stages x K and Q
    static constexpr int TG = KQ + kStages * kKQ;          // stages x [3 parts][T, G rows][128 B]
    static constexpr int V = TG + kTgStages * kTgBytes;    // [2 halves of 64 columns][64 rows][128 B]
    static constexpr int O = V + C * VS * 2;               // 512 bytes a warp: outputs on their way out
    static constexpr int VEC = O + kWorkers / 32 * 512;    // stages x row factors
    static constexpr int END = VEC + kStages * kVectorBytes;
};

// Tensor memory columns. An operand's three parts lie one behind the other, two values to a column.
enum : uint32_t {
    kSP = 0,           // S (64 columns each part)
    kRP = 0, kUP = 96, // R and u in its place (32 each part)
    kDK = 192,         // S^T [K;Q]^T
    kDT = 320,         // R^T [T;G]^T
    kDS = kDT,         // u^T K: all of kDT has been read by then
    // All of it: a prep CTA could not start beside this one, and this one waits for the prep kernel. Their
    // shared memory (above 180 KB and above 70 KB) keeps them from meeting on an SM.
    kColumns = 512
};

// Named barriers: the operand of a product is written; nobody starts anything any more.
enum { kHaveS = 1, kHaveR, kHaveU, kDone };

struct Shared {
    uint64_t full[2], tg_full[2], v_full, mma, last;
    int begun[5];  // copies begun on the first five of these
    uint32_t tmem;
    int abort, late;
    int row;  // sequence of this CTA
};

// Workers arrive, the issuing warps wait for them.
__device__ __forceinline__ void arrive(int id) {
    tmem_wait_st();
    tc_fence_before();
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kThreads) : "memory");
}

// Fragments: a warp's 32 rows (of M) by 16 columns, eight pairs of neighbouring columns to a lane.
// Pair 4 half + 2 block + below is row 16 half + 8 below + lane / 4, columns 8 block + lane % 4 * 2.
constexpr uint32_t kHalf = 16u << 16;  // 16 TMEM lanes
__device__ __forceinline__ void tmem_ld_frag(uint32_t t0, float2* f) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
            : "=f"(f[4 * h].x), "=f"(f[4 * h].y), "=f"(f[4 * h + 1].x), "=f"(f[4 * h + 1].y),
              "=f"(f[4 * h + 2].x), "=f"(f[4 * h + 2].y), "=f"(f[4 * h + 3].x), "=f"(f[4 * h + 3].y)
            : "r"(t0 + h * kHalf)
            : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t t0, const uint32_t* x) {
    __syncwarp();
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(x[0]), "r"(x[1]),
        "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(t0)
        : "memory");
}
// Pairs as words: 8 columns.
__device__ __forceinline__ void tmem_st_frag(uint32_t t0, const uint32_t* x) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%4], {%0,%1,%2,%3};" ::"r"(x[4 * h]),
                     "r"(x[4 * h + 1]), "r"(x[4 * h + 2]), "r"(x[4 * h + 3]), "r"(t0 + h * kHalf)
                     : "memory");
}

// Four 8 x 8 matrices of 16-bit values, transposed between shared memory and registers. A lane gives
// the address of row lane % 8 of matrix lane / 8 and has pair lane % 4 of column lane / 4 of each.
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t* x) {
    __syncwarp();
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void stsm_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    __syncwarp();
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a),
                 "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ float2 lds_pair(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// Two values as T, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float2 f) {
    uint32_t v;
    if constexpr (std::is_same<T, f16>::value) {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(f.y), "f"(f.x));
    } else {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(f.y), "f"(f.x));
    }
    return v;
}

template <typename T, typename ST>
__global__ void __launch_bounds__(kThreads, 1)
gdr_wide_kernel(const __grid_constant__ cc1d_gdr_args a, const __grid_constant__ CUtensorMap mapq,
                const __grid_constant__ CUtensorMap mapk, const __grid_constant__ CUtensorMap mapv, int tiles,
                int64_t wait_ns) {
    constexpr bool kLo = std::is_same<T, f16>::value;  // fp16 keys and queries come in two bf16 parts
    using Lay = Layout<kLo>;
    constexpr int kStages = Lay::kStages, kTgStages = Lay::kTgStages;
    extern __shared__ __align__(1024) unsigned char raw[];
    __shared__ Shared sh;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    unsigned char* gen = raw + (base - smem_addr(raw));
    const uint32_t vec_at = base + Lay::VEC;

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, w = warp % 4;
    const int part = warp / 4;  // 32 rows of the state, 16 tokens
    const int vt = blockIdx.x % tiles;
    const int h = (int)((blockIdx.x / tiles) % a.heads_v);
    const int hk = h / (a.heads_v / a.heads_k);
    const int64_t row =
        longest_first(a, blockIdx.x / tiles / a.heads_v, reinterpret_cast<int*>(gen), &sh.row);
    int64_t tok0, slot;
    int ntok;
    if (!gdr_row(a, true, row, tok0, ntok, slot, h == 0 && vt == 0 && tid == 0)) return;
    const int chunks = (ntok + C - 1) / C;
    const ChunkImage* image =
        static_cast<const ChunkImage*>(a.workspace) + chunk_base(tok0, row) * a.heads_v + h;

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
        tmem_alloc(smem_addr(&sh.tmem), kColumns);
        tmem_relinquish();
    }
    // The bulk copies below overwrite what the ordering above kept in shared memory.
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t mine = tmem + ((uint32_t)w << 21);  // with the warp's first lane

    if (warp == kWorkers / 32) {
        // Products, one thread.
        uint32_t st_phase = 0;
        for (int c = 0, st = 0; c < chunks; ++c) {
            const uint32_t kq = base + Lay::KQ + st * Lay::kKQ, tg = base + Lay::TG + c % kTgStages * kTgBytes;
            const uint32_t mma = smem_addr(&sh.mma);
            mbar_wait(smem_addr(&sh.full[st]), st_phase, &sh.abort, wait_ns);
            named_sync(kHaveS, kThreads);
            if (lane == 0) {
                tc_fence_after();
                // S^T [K;Q]^T, over the halves of dk. Here as below the smallest products come first: a
                // sum is cut to fp32 after every step.
                if constexpr (kLo)
#pragma unroll
                    for (int m = 1; m >= 0; --m)
#pragma unroll
                        for (int half = 0; half < 2; ++half)
                            mma_steps_ts<4, 2>(tmem + kDK, tmem + kSP + 64 * m + 32 * half,
                                               operand(kq + 32768 + half * 16384, 16, 1024, kSwizzle128),
                                               mma_desc(128, false, false), m == 0 || half > 0);
#pragma unroll
                for (int m = 2; m >= 0; --m)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        mma_steps_ts<4, 2>(tmem + kDK, tmem + kSP + 64 * m + 32 * half,
                                           operand(kq + half * 16384, 16, 1024, kSwizzle128),
                                           mma_desc(128, false, false), kLo || m < 2 || half > 0);
                mma_commit(mma);
            }
            mbar_wait(smem_addr(&sh.tg_full[c % kTgStages]), c / kTgStages & 1, &sh.abort, wait_ns);
            named_sync(kHaveR, kThreads);
            if (lane == 0) {
                tc_fence_after();
                // R^T [T;G]^T, by parts of both
                const uint64_t g = operand(tg, 16, 1024, kSwizzle128);
#pragma unroll
                for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                    for (int m = 0; m <= sum; ++m)
                        mma_steps_ts<4, 2>(tmem + kDT, tmem + kRP + 32 * m, g + 1024 * (sum - m),
                                           mma_desc(128, false, false), sum < 2 || m > 0);
                mma_commit(mma);
            }
            named_sync(kHaveU, kThreads);
            if (lane == 0) {
                tc_fence_after();
                // u^T K
                const uint64_t k = operand(kq, 16384, 1024, kSwizzle128);
                if constexpr (kLo)
#pragma unroll
                    for (int m = 1; m >= 0; --m)
                        mma_steps_ts<4, 128>(tmem + kDS, tmem + kUP + 32 * m, k + 2048, mma_desc(128, false, true),
                                             m == 0);
#pragma unroll
                for (int m = 2; m >= 0; --m)
                    mma_steps_ts<4, 128>(tmem + kDS, tmem + kUP + 32 * m, k, mma_desc(128, false, true), kLo || m < 2);
                mma_commit(mma);
            }
            if (++st == kStages) {
                st = 0;
                st_phase ^= 1;
            }
        }
        named_sync(kDone, kThreads);
        if (sh.abort && lane == 0) {
            mma_commit(smem_addr(&sh.last));
            mbar_wait(smem_addr(&sh.last), 0, &sh.late, kDrainNs);
        }
    } else if (warp > kWorkers / 32) {
        // Copies, one thread: K, Q and the row factors of chunk c into stage st, which must be free;
        // T and G, into the stage of their own; V.
        // Copies may be started: those of earlier chunks have been waited for.
        auto live = [&] { return *(volatile int*)&sh.abort == 0 && wait_ns > 0; };
        auto load = [&](int c, int st) {
            if (!live()) return;
            sh.begun[st] = c / kStages + 1;
            const uint32_t full = smem_addr(&sh.full[st]);
            const ChunkImage* from = image + (int64_t)c * a.heads_v;
            mbar_expect(full, Lay::kKQ + kVectorBytes);
            load_kq<kLo>(base + Lay::KQ + st * Lay::kKQ, &mapk, &mapq, hk, (int)tok0 + c * C, full);
            bulk_load(base + Lay::VEC + st * kVectorBytes, from->in, kVectorBytes, full);
        };
        auto load_tg = [&](int c) {
            if (!live()) return;
            const int st = c % kTgStages;
            sh.begun[2 + st] = c / kTgStages + 1;
            const uint32_t full = smem_addr(&sh.tg_full[st]);
            mbar_expect(full, kTgBytes);
            bulk_load(base + Lay::TG + st * kTgBytes, image[(int64_t)c * a.heads_v].tg, kTgBytes, full);
        };
        auto load_v = [&](int c) {
            if (!live()) return;
            sh.begun[4] = c + 1;
            const uint32_t full = smem_addr(&sh.v_full);
            mbar_expect(full, C * VS * 2);
            for (int half = 0; half < 2; ++half)
                tma_load(base + Lay::V + half * 8192, &mapv, vt * VS + half * 64, h, (int)tok0 + c * C, full);
        };
        grid_dependency_wait();  // for the prep kernel's images
        if (lane == 0) {
            for (int c = 0; c < kStages && c < chunks; ++c) load(c, c);
            for (int c = 0; c < kTgStages && c < chunks; ++c) load_tg(c);
            load_v(0);
        }
        for (int c = 0, st = 0; c < chunks; ++c) {
            // The workers are through with the chunk before, and its products are.
            named_sync(kHaveS, kThreads);
            if (lane == 0 && c > 0 && c - 1 + kStages < chunks)
                load(c - 1 + kStages, st > 0 ? st - 1 : kStages - 1);
            // They have read V.
            named_sync(kHaveR, kThreads);
            if (lane == 0 && c + 1 < chunks) load_v(c + 1);
            // They have the product of T and G.
            named_sync(kHaveU, kThreads);
            if (lane == 0 && c + kTgStages < chunks) load_tg(c + kTgStages);
            if (++st == kStages) st = 0;
        }
        named_sync(kDone, kThreads);
        if (sh.abort && lane == 0) {
            for (int i = 0; i < 5; ++i)
                if (sh.begun[i] > 0)
                    mbar_wait(smem_addr(sh.full) + 8 * i, (sh.begun[i] - 1) & 1, &sh.late, kDrainNs);
            flag_status(a.dev_status, CC1D_DEV_TIMEOUT);
        }
    } else {
        // This thread's state: column 32 w + lane of the tile, rows 32 part ..
        const int pair = lane % 4 * 2;
        const bool initial = a.states != nullptr && a.has_initial_state != nullptr && a.has_initial_state[row];
        ST* sp = nullptr;
        if (a.states != nullptr)
            sp = static_cast<ST*>(a.states) + slot * a.s_slot + h * a.s_sh + 32 * part * a.s_sk + vt * VS +
                 32 * w + lane;
        float2 s[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            s[k] = make_float2(0.f, 0.f);
            const ST* at = sp + 2 * k * a.s_sk;
            if (initial) s[k] = make_float2(to_f32(at[0]), to_f32(at[a.s_sk]));
        }
        // Outputs leave in rows of 32 columns, 16 bytes a lane.
        T* op = static_cast<T*>(a.out) + (tok0 + 16 * part + lane / 4) * a.o_st + h * a.o_sh + vt * VS + 32 * w +
                lane % 4 * 8;
        // Matrices of V: [block of tokens][below] of a half.
        const uint32_t vb = base + Lay::V + (w >> 1) * 8192;
        const int v_row = 16 * part + (lane >> 4) * 8 + lane % 8, v_unit = (w & 1) * 4 + (lane >> 3 & 1);
        const uint32_t mma = smem_addr(&sh.mma);
        const uint32_t patch = base + Lay::O + warp * 512;
        const uint32_t patch_st = patch + swz<64>(lane % 8, lane / 8);
        const uint32_t patch_ld = patch + swz<64>(lane / 4, lane % 4);

        int st = 0;
        uint32_t phase = 0, st_phase = 0;
        mbar_wait(smem_addr(&sh.full[0]), 0, &sh.abort, wait_ns);
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
            const uint32_t kq = base + Lay::KQ + st * Lay::kKQ;
            const int left = ntok - c * C;
            // The state as an operand.
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint32_t x[3][8];
#pragma unroll
                for (int k = 0; k < 8; ++k) split3(s[8 * g + k], x[0][k], x[1][k], x[2][k]);
#pragma unroll
                for (int m = 0; m < 3; ++m) tmem_st8(mine + kSP + 64 * m + 16 * part + 8 * g, x[m]);
            }
            if (left < C) {
                // The copies of K went on into the next sequence: zeros there, whatever it holds
                // (rows of Q there make outputs that are not stored).
                for (int e = tid; e < (C - left) * 16; e += kWorkers)
#pragma unroll
                    for (int p = 0; p <= (kLo ? 1 : 0); ++p)
                        sts16(kq + p * 32768 + (e % 16 >> 3) * 16384 + swz<128>(left + e / 16, e % 8), 0, 0, 0, 0);
                fence_async_smem();
            }
            arrive(kHaveS);
            {
                // R = V - r e^b (K S)
                mbar_wait(smem_addr(&sh.v_full), c & 1, &sh.abort, wait_ns);
                uint32_t vv[8];
                ldsm_t(vb + swz<128>(v_row, v_unit), vv);
                ldsm_t(vb + swz<128>(v_row, v_unit + 2), vv + 4);
                const uint32_t at = vec_at + st * kVectorBytes + 4 * (16 * part + pair);
                const float2 f[2] = {lds_pair(at), lds_pair(at + 32)};
                mbar_wait(mma, phase, &sh.abort, wait_ns);
                phase ^= 1;
                tc_fence_after();
                float2 d[8];
                tmem_ld_frag(mine + kDK + 16 * part, d);
                tmem_wait_ld();
                tmem_ready(d);
                uint32_t x[3][8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    d[k] = add_pair<T>(vv[k], __fmul2_rn(d[k], make_float2(-f[k >> 1 & 1].x, -f[k >> 1 & 1].y)));
                if (left < C) {
                    // zero behind the sequence's end, whatever V holds there
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int t = 16 * part + 8 * (k >> 1 & 1) + pair;
                        d[k].x = t < left ? d[k].x : 0.f;
                        d[k].y = t + 1 < left ? d[k].y : 0.f;
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) split3(d[k], x[0][k], x[1][k], x[2][k]);
#pragma unroll
                for (int m = 0; m < 3; ++m) tmem_st_frag(mine + kRP + 32 * m + 8 * part, x[m]);
            }
            arrive(kHaveR);
            uint32_t o[8];
            {
                // u, scaled for the end of the chunk
                const uint32_t at = vec_at + st * kVectorBytes + 4 * (16 * part + pair);
                const float2 f[2] = {lds_pair(at + 8 * C), lds_pair(at + 8 * C + 32)};
                const float2 fq[2] = {lds_pair(at + 4 * C), lds_pair(at + 4 * C + 32)};
                mbar_wait(mma, phase, &sh.abort, wait_ns);
                phase ^= 1;
                tc_fence_after();
                float2 d[8];
                tmem_ld_frag(mine + kDT + 16 * part, d);
                tmem_wait_ld();
                tmem_ready(d);
                uint32_t x[3][8];
#pragma unroll
                for (int k = 0; k < 8; ++k) split3(__fmul2_rn(d[k], f[k >> 1 & 1]), x[0][k], x[1][k], x[2][k]);
#pragma unroll
                for (int m = 0; m < 3; ++m) tmem_st_frag(mine + kUP + 32 * m + 8 * part, x[m]);
                // Outputs: read here, because a load that runs beside a product waits for its end.
                float2 q[8];
                tmem_ld_frag(mine + kDK + C + 16 * part, q);
                tmem_ld_frag(mine + kDT + C + 16 * part, d);
                tmem_wait_ld();
                tmem_ready(q);
                tmem_ready(d);
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] = pack2<T>(__ffma2_rn(q[k], fq[k >> 1 & 1], d[k]));
            }
            arrive(kHaveU);
            {
                // Outputs leave while it runs.
                T* to = op + (int64_t)c * C * a.o_st;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    stsm_t(patch_st, o[2 * b], o[2 * b + 1], o[4 + 2 * b], o[5 + 2 * b]);
                    __syncwarp();
                    const uint4 x = lds16(patch_ld);
                    if (16 * part + 8 * b + lane / 4 < left) st16_stream(to + 8 * b * a.o_st, x);
                }
            }
            const Vectors& vec = reinterpret_cast<const Vectors*>(gen + Lay::VEC)[st];
            const float decay = vec.decay;
            if (tid == 0 && vec.failed) *(volatile int*)&sh.abort = 1;
            if (++st == kStages) {
                st = 0;
                st_phase ^= 1;
            }
            if (c + 1 < chunks) mbar_wait(smem_addr(&sh.full[st]), st_phase, &sh.abort, wait_ns);
            mbar_wait(mma, phase, &sh.abort, wait_ns);
            phase ^= 1;
            tc_fence_after();
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float2 d[8];
                tmem_ld16(mine + kDS + 32 * part + 16 * g, d);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    s[8 * g + k] = __ffma2_rn(make_float2(decay, decay), s[8 * g + k], d[k]);
            }
        }
        named_sync(kDone, kThreads);
        if (sh.abort) {
            // The cache keeps its state, and the outputs say that they are none.
            for (int64_t t = 16 * part + lane / 4; t < ntok; t += t % 16 < 8 ? 8 : C - 8)
                st16(op + (t - 16 * part - lane / 4) * a.o_st, nan16());
        } else if (sp != nullptr) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                ST* at = sp + 2 * k * a.s_sk;
                at[0] = from_f32<ST>(s[k].x);
                at[a.s_sk] = from_f32<ST>(s[k].y);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, kColumns);
}

template <typename T, typename ST>
cudaError_t go(const cc1d_gdr_args& a, const CUtensorMap& q, const CUtensorMap& k, cudaStream_t stream) {
    constexpr int smem = Layout<std::is_same<T, f16>::value>::END + 1024;
    const int tiles = a.dv / VS;
    const int64_t grid = a.rows * a.heads_v * tiles;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    CUtensorMap v;
    if (!make_map(&v, a.v, a.tokens, a.heads_v, a.dv, a.v_st, a.v_sh, 64)) return cudaErrorInvalidValue;
    static SmemLimit limit;
    const cudaError_t err = limit.raise(gdr_wide_kernel<T, ST>, smem);
    if (err != cudaSuccess) return err;
    return launch_dependent(gdr_wide_kernel<T, ST>, (unsigned)grid, kThreads, smem, stream, a, q, k, v, tiles,
                            wait_limit_ns());
}

}  // namespace

cudaError_t launch_gdr_wide(const cc1d_gdr_args& a, const CUtensorMap& q, const CUtensorMap& k,
                            cudaStream_t stream) {
    if (a.dtype == CC1D_F16)
        return a.sdtype == CC1D_F32 ? go<f16, float>(a, q, k, stream) : go<f16, f16>(a, q, k, stream);
    return a.sdtype == CC1D_F32 ? go<bf16, float>(a, q, k, stream) : go<bf16, bf16>(a, q, k, stream);
}

}  // namespace cc1d
