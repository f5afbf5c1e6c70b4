// What the two kernels of the chunked gated delta rule share: the image of a chunk in the workspace,
// operand images in shared memory, tensor maps.
#pragma once

#include <atomic>

#include "gdr.cuh"
#include "kernels.h"
#include "tc05.cuh"

namespace cc1d {

constexpr int C = 64;    // tokens per chunk
constexpr int DK = 128;  // key head dim

// What the prep kernel leaves of a chunk and value head for the scan kernel.
struct ChunkImage {
    unsigned char tg[3][128 * 128];  // [T;G] in three bf16 parts, 128-byte rows, swizzled
    float in[2 * C];                 // r_i e^(b_i) (rows of K), s_i e^(b_i) (rows of Q)
    float out[C];                    // r_j e^(b_C - b_j)
    float decay;                     // e^(b_C)
    int32_t failed;                  // the prep kernel gave up a wait: nothing here is valid
    int32_t pad[2];
};
constexpr int kTgBytes = 3 * 128 * 128;
constexpr int kVectorBytes = (int)sizeof(ChunkImage) - kTgBytes;  // what follows tg

// The row factors of a ChunkImage, as they follow its T and G.
struct Vectors {
    float in[2 * C], out[C], decay;
    int32_t failed, pad[2];
};
static_assert(sizeof(Vectors) == kVectorBytes, "");

// The sequences that run in chunks: all of them, or in a batch of mostly short ones those that the
// device has listed, list = {count, tokens of the longest sequence left out, indices in order}.
struct Sequences {
    const int32_t* list;  // NULL: all
    int64_t n;            // how many there are at most
};
constexpr int kListMax = 32;  // sequences a list holds
constexpr int kLong = 32;     // they have more tokens than this

// Image slots: the chunks of the n-th of them start at slot floor(first token / 64) + n, which leaves
// every sequence room for its chunks without a prefix sum over the lengths.
__device__ __forceinline__ int64_t chunk_base(int64_t first_token, int64_t n) {
    return first_token / C + n;
}
__host__ __device__ inline int64_t chunk_slots(int64_t tokens, int64_t rows) {
    return tokens / C + rows;
}

// Row r, 16-byte unit u of an operand image of ROW-byte rows.
template <int ROW>
__device__ __forceinline__ uint32_t swz(int r, int u) {
    if constexpr (ROW == 128) {
        return r * 128 + ((u ^ (r & 7)) << 4);
    } else {
        return r * 64 + ((u ^ ((r >> 1) & 3)) << 4);
    }
}

// 8 values as three bf16 parts, one 16-byte unit each, `part` bytes apart.
__device__ __forceinline__ void store_split8(uint32_t at, uint32_t part, const float2* f) {
    uint32_t x[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split3(f[i], x[0][i], x[1][i], x[2][i]);
#pragma unroll
    for (int m = 0; m < 3; ++m) sts16(at + m * part, x[m][0], x[m][1], x[m][2], x[m][3]);
}
__device__ __forceinline__ float2 mul2(float2 a, float b) {
    return __fmul2_rn(a, make_float2(b, b));
}
__device__ __forceinline__ float2 bf16_pair(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// fp16 keys and queries as two bf16 parts, which hold their 11 bits: the first kernel of the fp16
// path writes (tokens, heads_k, 4, 128) bf16, parts k hi, q hi, k lo, q lo, behind the chunk images,
// and the kernels after it add the products with the low parts.
template <bool kLo>
struct Parts {
    static constexpr int kBytes = kLo ? 65536 : 32768;  // K and Q of a chunk in shared memory
    static __device__ __forceinline__ int k(int hk) { return kLo ? 4 * hk : hk; }
    static __device__ __forceinline__ int q(int hk) { return kLo ? 4 * hk + 1 : hk; }
};
// K and Q of 64 tokens: [hi, lo][2 halves of 64 columns][K 64 rows, Q 64 rows][128 B].
template <bool kLo>
__device__ __forceinline__ void load_kq(uint32_t dst, const CUtensorMap* mapk, const CUtensorMap* mapq,
                                        int hk, int t, uint32_t bar) {
#pragma unroll
    for (int part = 0; part <= (kLo ? 1 : 0); ++part)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t at = dst + part * 32768 + half * 16384;
            tma_load(at, mapk, half * 64, Parts<kLo>::k(hk) + 2 * part, t, bar);
            tma_load(at + 8192, mapq, half * 64, Parts<kLo>::q(hk) + 2 * part, t, bar);
        }
}

// The sequence of a CTA that was given index `row`: the row-th longest, so that the last CTAs to
// start are short. Ties go by index. All threads of the CTA call it; len and *mine are shared.
constexpr int kOrderMax = 256;  // batches up to this many sequences are ordered
__device__ __forceinline__ int64_t longest_first(const cc1d_gdr_args& a, int64_t row, int* len, int* mine) {
    if (a.rows < 2 || a.rows > kOrderMax) return row;
    const int n = (int)a.rows;
    for (int j = threadIdx.x; j < n; j += blockDim.x)
        len[j] = a.query_start_loc[j + 1] - a.query_start_loc[j];
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += len[i] > len[j] || (len[i] == len[j] && i < j);
        if (rank == row) *mine = j;
    }
    __syncthreads();
    return *mine;
}

// Dynamic shared memory above 48 KB, asked for once per kernel and device.
struct SmemLimit {
    std::atomic<uint64_t> done{0};  // a bit per device
    template <typename K>
    cudaError_t raise(K kernel, int bytes) {
        int dev = 0;
        cudaError_t err = cudaGetDevice(&dev);
        if (err != cudaSuccess) return err;
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (err == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
        return err;
    }
};

// A launch whose CTAs may come up while the kernel before drains; they wait for its end themselves.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), unsigned grid, int threads, int smem,
                             cudaStream_t stream, const Args&... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// One box (cols x 64 tokens of a head) of the tensor map of a (tokens, heads, dim) view of 16-bit values.
bool make_map(CUtensorMap* map, const void* p, int64_t tokens, int heads, int dim, int64_t st,
              int64_t sh, int cols);
// gdr_wide.cu: the scan with 128 state columns to a CTA.
cudaError_t launch_gdr_wide(const cc1d_gdr_args& a, const CUtensorMap& q, const CUtensorMap& k,
                            cudaStream_t stream);
// Whether the driver offers tensor maps.
bool have_maps();

cudaError_t launch_gdr_prep(const cc1d_gdr_args& a, const Sequences& seqs, const CUtensorMap& q,
                            const CUtensorMap& k, cudaStream_t stream);
// Lists the sequences that are long enough for chunks, seqs.n at most.
cudaError_t launch_gdr_list(const cc1d_gdr_args& a, const Sequences& seqs, int32_t* list,
                            cudaStream_t stream);
// What a CTA that has given up waits for its own copies and products at most, one by one.
constexpr int64_t kDrainNs = 2000000000;

// 16 bytes of NaN of either 16-bit type: the outputs of a CTA that gave up.
__device__ __forceinline__ uint4 nan16() { return make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu); }

// The split of fp16 keys and queries, into the workspace at `to`.
cudaError_t launch_gdr_split(const cc1d_gdr_args& a, void* to, cudaStream_t stream);

}  // namespace cc1d
