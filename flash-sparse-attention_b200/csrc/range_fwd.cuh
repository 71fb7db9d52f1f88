// The forwards of range attention (range_dense.cu) and of attention with changed scores (biased_fwd.cu) for their callers.
#pragma once
#include "score.cuh"
#include "sel_launch.cuh"

namespace fsa {

constexpr int kRdBK = 64;

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
};

// First and last K/V row that token `tok` of a sequence sees, and its place, without documents.  The sequence has the rows [k0, k1); its last token is
// the one before q1 and stands at row k1 - 1.  window: -1 for none; prefix: rows at its beginning that all tokens see.
struct Sees { int lo, hi, pos; };
__device__ __forceinline__ Sees place_limits(int tok, int k0, int k1, int q1, int window, int prefix) {
    Sees x;
    x.pos = tok + k1 - q1;
    const bool in = x.pos >= k0;            // (else the sequence has fewer keys than queries, and this one precedes them)
    x.lo = in && window >= 0 ? max(k0, x.pos - window) : k0;
    x.hi = in ? max(x.pos, min(k0 + prefix, k1) - 1) : -1;
    return x;
}

// Attention with changed scores: the same problem, one a launch.
struct BiasedFwdLaunch {
    CUtensorMap q, k, v;
    RangeDenseParams p;     // (o_sn and o_sh are not used: o is contiguous; kv_lo null: place_limits)
    ScoreMod mod;
    int window;                     // -1: none
    const int32_t* prefix_lens;     // [B] or null
    // kModSplit: rows that several sequences share, a "token" is a sequence of the batch (kv_lo and kv_hi are not used).  The K/V rows of every
    // tile are cut into nchunk chunks (blockIdx.y) of `chunk` tiles; chunk c of a row writes partial c of P
    const int32_t* seq_len; // [N] own tokens of every sequence, the new one among them
    float* o_part;          // [N, Hq, P, D] unnormalised
    float2* ml;             // [N, Hq, P] reference maximum (log2 units) and sum
    int P, nchunk, chunk;
};
// which: kModCap, kModBias; split: with kModSplit.  l.p.TPT tokens a tile, max_tiles tiles at most.
cudaError_t launch_biased_fwd(int D, int dtype, int which, bool split, const BiasedFwdLaunch& l, int max_tiles, cudaStream_t stream);

}  // namespace fsa
