// Attention with changed scores: its kernels (biased_fwd.cu, biased_bwd_dq.cu, biased_bwd_dkdv.cu) for their callers (biased_attn.cu, biased_decode.cu).
#pragma once
#include "score.cuh"
#include "sel_launch.cuh"

namespace fsa {

constexpr int kBiasedBK = 64;       // K/V rows of a tile
constexpr int kBiasedLeast = 4;     // K/V tiles of a chunk (an item's beginning and end are as long as 4 to 5 of them)
// Tiles of `tokens` tokens in B sequences, at most; of all kv heads there are fewer than kBiasedMaxPlaces (32-bit numbers of items and CTAs, some to spare).
inline int64_t biased_places(int64_t tokens, int TPT, int64_t B) { return (tokens + TPT - 1) / TPT + B; }
constexpr int64_t kBiasedMaxPlaces = (int64_t)1 << 30;

// The operators' status word (one a device): what a wait that ran out left, and above it when that was, in units of 2^30 ns of the device's timer.
// The later CTAs of a launch that has failed are not to take 0.2 s each for their waits: up to two units after a failure waits are short.  What
// failed before that is over, whoever has read it or not.  (biased_bwd_dq and _dkdv, whose CTAs all run at once, leave the time out.)
constexpr int kStampBits = 22;
__device__ __forceinline__ int now_stamp() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return (int)(t >> 30) & ((1 << kStampBits) - 1);
}
__device__ __forceinline__ void stamp_status(int* word, int status) { atomicMax(word, now_stamp() << 8 | status); }
__device__ __forceinline__ uint32_t stamped_wait_limit(const int* word) {
    const int failed = *reinterpret_cast<const volatile int*>(word);
    return failed && ((now_stamp() - (failed >> 8)) & ((1 << kStampBits) - 1)) < 2 ? FSA_WAIT_CLOCKS / 64 : FSA_WAIT_CLOCKS;
}
__device__ __forceinline__ bool mbar_wait_stamped(uint64_t* bar, uint32_t parity, int* word, uint32_t limit) {
    if (mbar_poll(bar, parity, limit)) return true;
    stamp_status(word, kStatusWaitTimeout);
    return false;
}

struct BiasedFwdParams {
    const int32_t* cu_q;    // [B + 1]
    const int32_t* cu_k;    // [B + 1] first K/V row of every sequence
    const int32_t* kv_lo;   // [N] first K/V row that every token sees, or null: place_limits
    const int32_t* kv_hi;   // [N] last one, lower than kv_lo where a token sees nothing
    int64_t N, Nk;
    int B, Hq, Hk, G, TPT;
    float scale_log2;
    void* o;                // [N, Hq, D] contiguous
    float* lse;             // [Hq, N] log2 units
    int* status;
};

// First and last K/V row that token `tok` of a sequence sees, and its place, without documents.  The sequence has the rows [k0, k1); its last token is
// the one before q1 and stands at row k1 - 1.  window: -1 for none; prefix: rows at its beginning that all tokens see (below 0: none).
struct Sees { int lo, hi, pos; };
__device__ __forceinline__ Sees place_limits(int tok, int k0, int k1, int q1, int window, int prefix) {
    Sees x;
    x.pos = tok + k1 - q1;
    const bool in = x.pos >= k0;            // (else the sequence has fewer keys than queries, and this one precedes them)
    x.lo = in && window >= 0 ? max(k0, x.pos - window) : k0;
    x.hi = in ? max(x.pos, k0 + min(max(prefix, 0), k1 - k0) - 1) : -1;
    return x;
}

struct BiasedFwdLaunch {
    CUtensorMap q, k, v;
    BiasedFwdParams p;
    ScoreMod mod;
    int window;                     // -1: none
    const int32_t* prefix_lens;     // [B] or null
    // kModSplit: the K/V rows of every tile are cut into nchunk chunks (blockIdx.y) of `chunk` tiles (0: an equal share, at least kBiasedLeast);
    // chunk c of a row writes partial c of P.
    // seq_len: rows that several sequences share, a "token" is a sequence of the batch (kv_lo and kv_hi are not used), and the kernel runs beside the
    // one before it
    const int32_t* seq_len; // [N] own tokens of every sequence, the new one among them; or null
    float* o_part;          // [N, Hq, P, D] unnormalised
    float2* ml;             // [N, Hq, P] reference maximum (log2 units) and sum
    int P, nchunk, chunk;
};
// which: kModCap, kModBias; split: with kModSplit.  l.p.TPT tokens a tile, max_tiles tiles at most.
cudaError_t launch_biased_fwd(int D, int dtype, int which, bool split, const BiasedFwdLaunch& l, int max_tiles, cudaStream_t stream);

// o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, lse = M + log2 of the latter, of rows = tokens x Hq over their P partials.  The first nshared
// partials of tokens outside [cu[0], cu[groups]) are left out.  lse[token * lse_sn + head * lse_sh].  (biased_decode.cu)
struct BiasedMerge {
    const float* o_part;
    const float2* ml;
    int64_t rows;
    int Hq, P, nshared;
    const int32_t* cu;
    int groups;
    void* o;
    float* lse;
    int64_t lse_sn, lse_sh;
};
cudaError_t launch_biased_merge(int D, int dtype, const BiasedMerge& m, cudaStream_t stream);

// Which of the items, longest first, is this CTA's n-th: forth and back, so that who has the longer item of one round has the shorter one of the next (always
// forth, the first CTA has the longest of every round: dQ of 2 x 8192 tokens, 8 / 4 heads, takes 445 us instead of 401).
__device__ __forceinline__ int forth_and_back(int n) { return n * (int)gridDim.x + (int)(n & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x); }

struct RangeKvPlan;      // range_bwd.cuh
// The backward, a.bd's limits given; as parts of a chain of dependent launches, dK / dV beside dQ.  nchunk > 1: dQ cut into chunks along the keys, part
// [N, Hq, nchunk, D], which launch_biased_dq_sum joins after both.
cudaError_t launch_biased_bwd_dq(int dtype, const SelBwdArgs& a, const SelShape& s, const CUtensorMap& kmap, const CUtensorMap& vmap, int* status,
                                 const ScoreMod& mod, int which, int nchunk, float* part, cudaStream_t stream);
cudaError_t launch_biased_dq_sum(int dtype, const float* part, const SelBwdArgs& a, const SelShape& s, int nchunk, cudaStream_t stream);
cudaError_t launch_biased_bwd_dkdv(int dtype, const RangeKvPlan& plan, const SelBwdArgs& a, const SelShape& s, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                   int* status, const ScoreMod& mod, int which, cudaStream_t stream);

}  // namespace fsa
