// Shared pieces of the gated delta rule kernels: token ranges, slots and gates.
#pragma once

#include "common.cuh"

namespace cc1d {

constexpr float kL2Eps = 1e-6f;

// Element i of a tensor of run-time dtype (gates and their parameters: a few values per token).
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
    if (dtype == CC1D_BF16) return __bfloat162float(static_cast<const bf16*>(p)[i]);
    if (dtype == CC1D_F16) return __half2float(static_cast<const f16*>(p)[i]);
    return static_cast<const float*>(p)[i];
}

// Log decay and update rate of one (token, head): given, or made of the raw projections.
// softplus(x) = log(1 + e^x) is x itself in fp32 from x = 20 on (e^-20 is below half an ulp).
__device__ __forceinline__ void load_gates(const cc1d_gdr_args& a, int64_t g_at, int64_t b_at,
                                           int h, float& g, float& beta) {
    g = load_any(a.g, g_at, a.gdtype);
    beta = load_any(a.beta, b_at, a.bdtype);
    if (a.a_log != nullptr) {
        const float x = g + load_any(a.dt_bias, h, a.pdtype);
        const float sp = x > 20.f ? x : log1pf(expf(x));
        g = -expf(load_any(a.a_log, h, a.pdtype)) * sp;
        beta = 1.f / (1.f + expf(-beta));
    }
}

// The tokens and the cache slot of work row `row`. False: nothing to do (a skipped or empty row,
// or an index outside its tensor, which is reported). slot is -1 without a cache.
__device__ __forceinline__ bool gdr_row(const cc1d_gdr_args& a, bool varlen, int64_t row,
                                        int64_t& tok0, int& ntok, int64_t& slot, bool report) {
    slot = -1;
    if (a.states != nullptr) {
        slot = a.indices != nullptr ? a.indices[row] : row;
        if (a.indices != nullptr && slot == a.pad) return false;
        if (slot < 0 || slot >= a.nslots) {
            if (report) flag_status(a.dev_status, CC1D_DEV_BAD_SLOT);
            return false;
        }
    }
    if (!varlen) {
        tok0 = 0;
        ntok = a.steps;
        return true;
    }
    const int64_t t0 = a.query_start_loc[row], t1 = a.query_start_loc[row + 1];
    if (t0 < 0 || t1 < t0 || t1 > a.tokens) {
        if (report) flag_status(a.dev_status, CC1D_DEV_BAD_QSL);
        return false;
    }
    tok0 = t0;
    ntok = (int)(t1 - t0);
    return ntok > 0;
}

}  // namespace cc1d
