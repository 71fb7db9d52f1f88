// The forward of range attention (range_dense.cu) for its callers: one problem or several, plain scores or changed ones (score.cuh).
#pragma once
#include "score.cuh"
#include "sel_launch.cuh"

namespace fsa {

struct RangeDenseParams {
    const int32_t* cu_q;    // [B + 1]
    const int32_t* cu_k;    // [B + 1] first K/V row of every sequence
    const int32_t* kv_lo;   // [N] lowest visible K/V row of every token, or null (the sequence's first row)
    const int32_t* kv_hi;   // [N] highest visible K/V row, lower than kv_lo when the token sees nothing
    int64_t N, Nk;
    int B, Hq, Hk, G, TPT;
    float scale_log2;
    void* o;  int64_t o_sn, o_sh;     // [N, Hq, D]
    float* lse;                       // [Hq, N] log2 units
    int* status;
};

// Up to three problems in one launch (blockIdx.z): branches of a layer that do not wait for one another.  A short prompt has fewer tiles
// than the SMs hold CTAs, and each launch of its own left most of them empty (517 tokens, 32 / 8 heads: 3 x 11 us, together 19: prefill 158 -> 138 us).
constexpr int kRdProblems = 3;
struct RangeDenseLaunch {
    CUtensorMap q[kRdProblems], k[kRdProblems], v[kRdProblems], o[kRdProblems];
    RangeDenseParams p[kRdProblems];
    // kernels with a MOD: one problem
    ScoreMod mod;
    // kModSplit: the K/V rows of every tile are cut into nchunk chunks (blockIdx.z); chunk c of a row writes partial c of P
    float* o_part;          // [N, Hq, P, D] unnormalised
    float2* ml;             // [N, Hq, P] reference maximum (log2 units) and sum
    int P, nchunk;
};

// The forward with changed scores (range_dense.cu): l.p[0] and l.mod, tiles of l.p[0].TPT tokens; nchunk > 0: kModSplit.
cudaError_t launch_range_fwd_mod(int D, int dtype, int mod, const RangeDenseLaunch& l, int max_tiles, cudaStream_t stream);

}  // namespace fsa
