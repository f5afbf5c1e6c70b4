// Slot moves between state caches: copy, fork, clear and compaction of whole slots, for every
// cache of a group (conv states and delta-rule states of all layers) in one launch.
//
// Bound: HBM (each moved slot read and written once). The bytes of a slot are cut into tiles of
// one 16-byte unit per thread (smaller units where pointers, strides or row sizes ask for it); a
// CTA owns one tile of one cache for its share of the pairs. With that ownership the pairs of one
// CTA can run in list order with no exchange between CTAs, which gives the sequential meaning
// (later pairs see earlier ones) for any list; whether a list has such dependences is found by
// each CTA in a bitmap of destinations, and only a list that has none is also split over the grid
// and loaded kUnroll pairs at a time. Results do not depend on timing.
#include "common.cuh"
#include "kernels.h"

namespace cc1d {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 8;
constexpr int kMaxBits = 1 << 18;  // destinations the bitmap holds (32 KB of shared memory)

struct SlotTable {
    cc1d_slot_cache c[CC1D_MAX_CACHES];
    int64_t end[CC1D_MAX_CACHES];  // tiles of caches 0..i
    uint8_t unit[CC1D_MAX_CACHES];  // log2 bytes per thread and pair
    int32_t n;
};

template <typename U>
__device__ __forceinline__ void move_pairs(const cc1d_slot_cache& c, int64_t unit,
                                           const int32_t* __restrict__ src,
                                           const int32_t* __restrict__ dst, int n, int first,
                                           int step, bool ordered, int64_t src_slots,
                                           int64_t dst_slots, int pad) {
    const char* from = static_cast<const char*>(c.src) + unit * (int64_t)sizeof(U);
    char* to = static_cast<char*>(c.dst) + unit * (int64_t)sizeof(U);
    if (ordered) {
        for (int i = 0; i < n; ++i) {
            const int s = src[i], d = dst[i];
            if (d == pad || d < 0 || d >= dst_slots || (s != pad && (s < 0 || s >= src_slots))) continue;
            U v{};
            if (s != pad) v = *reinterpret_cast<const U*>(from + s * c.src_stride);
            *reinterpret_cast<U*>(to + d * c.dst_stride) = v;
        }
        return;
    }
    for (int base = first; base < n; base += step * kUnroll) {
        U v[kUnroll];
        int d[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int i = base + j * step;
            v[j] = U{};
            d[j] = -1;
            if (i < n) {
                const int s = src[i];
                d[j] = dst[i];
                if (d[j] == pad || d[j] >= dst_slots || (s != pad && (s < 0 || s >= src_slots))) d[j] = -1;
                if (d[j] >= 0 && s != pad) v[j] = *reinterpret_cast<const U*>(from + s * c.src_stride);
            }
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j)
            if (d[j] >= 0) *reinterpret_cast<U*>(to + d[j] * c.dst_stride) = v[j];
    }
}

// With a plan, the pairs come from it, {count, sources[nslots], destinations[nslots]}
// and have no dependences. bits: destinations the bitmap of dynamic shared memory holds, 0 when a
// list is to run in order without a check.
__global__ void __launch_bounds__(kThreads)
slots_move_kernel(const __grid_constant__ SlotTable t, const int32_t* src, const int32_t* dst,
                  int npairs, const int32_t* plan, int64_t src_slots, int64_t dst_slots, int pad,
                  int bits, bool same, int32_t* status) {
    extern __shared__ uint32_t map[];
    const int64_t tile = blockIdx.x;
    int c = 0;
    while (c + 1 < t.n && tile >= t.end[c]) ++c;

    bool ordered = false;
    if (plan != nullptr) {
        npairs = plan[0];
        src = plan + 1;
        dst = plan + 1 + dst_slots;
    } else if (npairs > 1) {
        ordered = bits == 0;
        if (bits > 0) {
            for (int i = threadIdx.x; i < (bits + 31) / 32; i += kThreads) map[i] = 0;
            __syncthreads();
            int clash = 0;
            for (int i = threadIdx.x; i < npairs; i += kThreads) {
                const int d = dst[i];
                if (d == pad || d < 0 || d >= dst_slots) continue;
                clash |= (atomicOr(&map[d / 32], 1u << (d % 32)) >> (d % 32)) & 1;
            }
            clash = __syncthreads_or(clash);
            if (same && !clash) {
                for (int i = threadIdx.x; i < npairs; i += kThreads) {
                    const int s = src[i];
                    if (s == pad || s < 0 || s >= src_slots || s == dst[i]) continue;
                    clash |= (map[s / 32] >> (s % 32)) & 1;
                }
                clash = __syncthreads_or(clash);
            }
            ordered = clash != 0;
        }
    }
    if (plan == nullptr && tile == 0 && blockIdx.y == 0 && status != nullptr) {
        for (int i = threadIdx.x; i < npairs; i += kThreads) {
            const int s = src[i], d = dst[i];
            if (d != pad && (d < 0 || d >= dst_slots || (s != pad && (s < 0 || s >= src_slots))))
                flag_status(status, CC1D_DEV_BAD_SLOT);
        }
    }
    if (ordered && blockIdx.y > 0) return;

    const int64_t unit = (tile - (c > 0 ? t.end[c - 1] : 0)) * kThreads + threadIdx.x;
    if ((unit << t.unit[c]) >= t.c[c].row_bytes) return;
    const int first = blockIdx.y, step = gridDim.y;
    switch (t.unit[c]) {
        case 4: move_pairs<uint4>(t.c[c], unit, src, dst, npairs, first, step, ordered, src_slots, dst_slots, pad); break;
        case 3: move_pairs<uint2>(t.c[c], unit, src, dst, npairs, first, step, ordered, src_slots, dst_slots, pad); break;
        case 2: move_pairs<uint32_t>(t.c[c], unit, src, dst, npairs, first, step, ordered, src_slots, dst_slots, pad); break;
        case 1: move_pairs<uint16_t>(t.c[c], unit, src, dst, npairs, first, step, ordered, src_slots, dst_slots, pad); break;
        default: move_pairs<uint8_t>(t.c[c], unit, src, dst, npairs, first, step, ordered, src_slots, dst_slots, pad); break;
    }
}

// One CTA: m = number of live slots; the i-th free slot below m and the i-th live slot from m on
// (equally many) become pair i of the plan.
__global__ void __launch_bounds__(1024)
slots_plan_kernel(const uint8_t* __restrict__ live, int nslots, int32_t* __restrict__ remap,
                  int32_t* __restrict__ count, int32_t* __restrict__ plan) {
    __shared__ int warp_sum[32];
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    int m = 0;
    for (int i = tid; i < nslots; i += 1024) m += live[i] != 0;
#pragma unroll
    for (int o = 16; o > 0; o /= 2) m += __shfl_xor_sync(~0u, m, o);
    if (lane == 0) warp_sum[warp] = m;
    __syncthreads();
    m = warp_sum[lane];
#pragma unroll
    for (int o = 16; o > 0; o /= 2) m += __shfl_xor_sync(~0u, m, o);
    if (tid == 0) *count = m;
    int32_t* src = plan + 1;
    int32_t* dst = plan + 1 + nslots;
    // Pairs are numbered by rank: holes below m and movers from m on, each in ascending order. Both
    // counts travel in one word (at most 1024 of either in a step of 1024 slots).
    int base[2] = {0, 0};
    for (int at = 0; at < nslots; at += 1024) {
        const int i = at + tid;
        const bool on = i < nslots && live[i] != 0;
        const bool hole = i < nslots && !on && i < m, mover = on && i >= m;
        const unsigned holes = __ballot_sync(~0u, hole), movers = __ballot_sync(~0u, mover);
        __syncthreads();
        if (lane == 0) warp_sum[warp] = __popc(holes) | __popc(movers) << 16;
        __syncthreads();
        int sum = warp_sum[lane];  // to the running sum over the warps
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int below = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += below;
        }
        const int all = __shfl_sync(~0u, sum, 31);
        const int before = __shfl_sync(~0u, sum, warp > 0 ? warp - 1 : 0) & (warp > 0 ? ~0 : 0);
        const unsigned under = (1u << lane) - 1u;
        if (hole) dst[base[0] + (before & 0xffff) + __popc(holes & under)] = i;
        if (mover) src[base[1] + (before >> 16) + __popc(movers & under)] = i;
        if (i < nslots && !mover) remap[i] = on ? i : -1;
        base[0] += all & 0xffff;
        base[1] += all >> 16;
    }
    if (tid == 0) plan[0] = base[1];
    __syncthreads();
    for (int i = tid; i < base[1]; i += 1024) remap[src[i]] = dst[i];
}

int64_t build_table(const cc1d_slot_cache* table, int ncaches, SlotTable& t) {
    int64_t tiles = 0;
    t.n = ncaches;
    for (int i = 0; i < ncaches; ++i) {
        t.c[i] = table[i];
        const uint64_t all = (uint64_t)(uintptr_t)table[i].dst | (uint64_t)(uintptr_t)table[i].src |
                             (uint64_t)table[i].dst_stride | (uint64_t)table[i].src_stride |
                             (uint64_t)table[i].row_bytes;
        int unit = 4;
        while (unit > 0 && (all & ((1u << unit) - 1))) --unit;
        t.unit[i] = (uint8_t)unit;
        tiles += ceil_div(table[i].row_bytes, (int64_t)kThreads << unit);
        t.end[i] = tiles;
    }
    return tiles;
}

// CTAs that one tile's pairs are split over: enough for a few waves when the slots are small.
int pair_split(int64_t tiles, int64_t npairs) {
    const int64_t want = ceil_div(148 * 8 * 4, tiles);
    const int64_t most = ceil_div(npairs, kUnroll);
    return (int)(want < 1 ? 1 : want > most ? most : want);
}

}  // namespace

cudaError_t launch_slots_copy(const cc1d_slot_cache* table, int ncaches, const int32_t* src,
                              const int32_t* dst, int64_t npairs, int64_t src_nslots,
                              int64_t dst_nslots, bool same, int pad, int32_t* status,
                              cudaStream_t stream) {
    SlotTable t;
    const int64_t tiles = build_table(table, ncaches, t);
    if (tiles == 0) return cudaSuccess;
    if (tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
    const int bits = dst_nslots <= kMaxBits ? (int)dst_nslots : 0;
    const dim3 grid((unsigned)tiles, bits > 0 ? pair_split(tiles, npairs) : 1);
    slots_move_kernel<<<grid, kThreads, npairs > 1 ? (bits + 31) / 32 * 4 : 0, stream>>>(
        t, src, dst, (int)npairs, nullptr, src_nslots, dst_nslots, pad, bits, same, status);
    return cudaGetLastError();
}

cudaError_t launch_slots_compact(const cc1d_slot_cache* table, int ncaches, const uint8_t* live,
                                 int64_t nslots, int32_t* remap, int32_t* count, int32_t* moves,
                                 cudaStream_t stream) {
    slots_plan_kernel<<<1, 1024, 0, stream>>>(live, (int)nslots, remap, count, moves);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess || ncaches == 0 || nslots == 0) return err;
    SlotTable t;
    const int64_t tiles = build_table(table, ncaches, t);
    if (tiles == 0) return cudaSuccess;
    if (tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)tiles, pair_split(tiles, ceil_div(nslots, 2)));
    slots_move_kernel<<<grid, kThreads, 0, stream>>>(t, nullptr, nullptr, 0, moves, nslots, nslots,
                                                     -1, 0, true, nullptr);
    return cudaGetLastError();
}

}  // namespace cc1d
