// Attention with changed scores (capped by a tanh, biased by distance) under causal, window, document and prefix masks, packed
// sequences: the limits of every token and the entry points.  Under each of these masks a token sees one stretch of
// K/V rows.  Forward: biased_fwd.cu; backward: biased_bwd_dq.cu and biased_bwd_dkdv.cu, on the plan of range_bwd_dkdv.cu.
#include "../../include/fsa_sm100.h"

#include "range_bwd.cuh"
#include "biased.cuh"

namespace fsa {

int make_tile_map(CUtensorMap* map, const void* base, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int box_rows);
int make_tile_map_3d_box(CUtensorMap* map, const void* base, int dtype, int64_t d0, int64_t d1, int64_t d2, int64_t stride1,
                         int64_t stride2, int box1, int box2);
int cuda_failed(cudaError_t e);

// Set (biased.cuh) by a kernel of these operators whose bounded wait ran out; read, and cleared, with fsa_biased_read_status.
static __device__ int g_biased_status;

// Its address on the current device (once per thread and device: a driver call).
cudaError_t biased_status_word(int** out) {
    static thread_local struct { int dev = -1; int* word = nullptr; } seen;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && seen.dev != dev) {
        void* p = nullptr;
        if ((e = cudaGetSymbolAddress(&p, g_biased_status)) == cudaSuccess) { seen.dev = dev; seen.word = (int*)p; }
    }
    *out = seen.word;
    return e;
}

// For every token the first and last K/V row that it sees and its own place.
struct BiasedLimits {
    int *lo, *hi, *pos;
    BiasedLimits(void* ws, int64_t N) : lo((int*)ws), hi(lo + N), pos(hi + N) {}
    static int64_t bytes(int64_t N) { return 3 * N * 4; }
};

constexpr int kLimThreads = 256;

// Last row j <= row of [first, row] that begins a document: whose id differs from that of the row before, or `first` itself.  All lanes of a
// warp call it; 512 ids a step (one load is as long on its way as sixteen).
__device__ __forceinline__ int document_start(const int32_t* __restrict__ ids, int first, int row, int lane) {
    const int id = __ldcg(ids + row);
    for (int end = row; end > first; end -= 512) {      // rows [end - 512, end) are looked at
        int found = -1;                                 // last row of another document among them
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int j = end - 1 - (i * 32 + lane);
            if (j >= first && __ldcg(ids + j) != id) found = max(found, j);
        }
        found = __reduce_max_sync(0xffffffffu, found);
        if (found >= 0) return found + 1;
    }
    return first;
}

// One thread per token.  Tokens of one sequence stand at consecutive K/V rows.  Documents: a token whose row does not begin one sees from where the
// token before it does, so a CTA scans its tokens.  What is searched for backwards is the beginning for a sequence's first token (with rows in
// front of it), by its warp, and for the CTA's first token, by the whole CTA, 4096 ids a step.
__global__ void __launch_bounds__(kLimThreads) biased_limits(const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k,
                                                             const int32_t* __restrict__ doc_ids, int B, int64_t N, int window, BiasedLimits out) {
    __shared__ int s_start[kLimThreads / 32], s_seq[kLimThreads / 32], s_found[kLimThreads / 32], s_first[4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t n = (int64_t)blockIdx.x * kLimThreads + tid;
    follow();
    const int used = __ldcg(cu_q + B);
    int seq = -1, k0 = 0;
    Sees x = {0, -1, 0};
    if (n < used && n < N) {
        seq = find_seq<true>(cu_q, B, (int)n);
        k0 = __ldcg(cu_k + seq);
        x = place_limits((int)n, k0, __ldcg(cu_k + seq + 1), __ldcg(cu_q + seq + 1), window, 0);
    }
    const bool in = x.hi >= 0;
    const int id = in ? __ldcg(doc_ids + x.pos) : -1;
    const bool begins = !in || x.pos == k0 || __ldcg(doc_ids + x.pos - 1) != id;
    if (lane == 31) s_seq[warp] = seq;
    // the CTA's first token
    if (tid == 0) { s_first[0] = begins; s_first[1] = k0; s_first[2] = x.pos; s_first[3] = id; }
    __syncthreads();
    int first = s_first[2];
    if (!s_first[0]) {
        const int from = s_first[1], want = s_first[3];
        first = from;
        for (int end = s_first[2]; end > from; end -= 16 * kLimThreads) {      // rows [end - 4096, end) are looked at
            int found = -1;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = end - 1 - (i * kLimThreads + tid);
                if (j >= from && __ldcg(doc_ids + j) != want) found = max(found, j);
            }
            found = __reduce_max_sync(0xffffffffu, found);
            if (lane == 0) s_found[warp] = found;
            __syncthreads();
            found = __reduce_max_sync(0xffffffffu, lane < kLimThreads / 32 ? s_found[lane] : -1);
            __syncthreads();
            if (found >= 0) { first = found + 1; break; }
        }
    }
    int seq_before = __shfl_up_sync(0xffffffffu, seq, 1);
    if (lane == 0) seq_before = warp ? s_seq[warp - 1] : seq;
    // of the document, where it is known (a token before the first row stands at a negative place and sees nothing)
    int start = begins ? max(x.pos, 0) : tid == 0 ? first : -1;
    for (unsigned todo = __ballot_sync(0xffffffffu, start < 0 && seq_before != seq); todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        const int found = document_start(doc_ids, __shfl_sync(0xffffffffu, k0, src), __shfl_sync(0xffffffffu, x.pos, src), lane);
        if (lane == src) start = found;
    }
    // the nearest lane at or below this one that knows, or the end of a warp before
    const unsigned known = __ballot_sync(0xffffffffu, start >= 0) & (0xffffffffu >> (31 - lane));
    start = __shfl_sync(0xffffffffu, start, known ? 31 - __clz(known) : lane);
    if (lane == 31) s_start[warp] = start;
    __syncthreads();
    for (int w = warp - 1; start < 0; --w) start = s_start[w];              // (warp 0 knows all of its)
    if (n < N) {
        const bool sees = in && id >= 0;
        out.lo[n] = sees ? max(x.lo, start) : 0;
        out.hi[n] = sees ? x.hi : -1;
        out.pos[n] = x.pos;
    }
}

static cudaError_t launch_limits(const int32_t* cu_q, const int32_t* cu_k, const int32_t* doc_ids, int B, int64_t N, int window, const BiasedLimits& out,
                                 cudaStream_t stream) {
    return launch_dependent(biased_limits, dim3((unsigned)((N + kLimThreads - 1) / kLimThreads)), kLimThreads, 0, stream, 1, cu_q, cu_k, doc_ids, B, N, window, out);
}

// ------------------------------------------------------------------------------------------------ what the backward's kernels need
// One launch: CTA 0 plans the items of dK / dV, the others work out delta = sum_d o dO, without documents the limits, and clear what lies outside of the
// sequences.  Without documents the stretch of tokens that sees a tile of K/V rows follows from the rule: from the token at the tile's first row
// (with a prefix that the tile is part of: the sequence's first) to the one at its last row (with a window: that far behind).  2 x 8192 tokens, 8 heads
// of 128: 15 us, bound by memory (67 MB of o and dO); delta alone took 20, limits, stretches and plan a launch each besides.
struct BiasedPrep {
    RangeKvPlan plan;
    BiasedLimits lim;
    const int32_t* prefix_lens;
    int window, docs;               // docs: plan.tiles and the limits are there, dk's and dv's last rows cleared
    const void *o, *d_o;            // [N, Hq, D], o contiguous
    int64_t do_sn, do_sh;
    int Hq;
    float* delta;                   // [Hq, N]
    uint4 *dq, *dk, *dv;
};
constexpr int kPrThreads = 512;

template <int D, typename ET>
__global__ void __launch_bounds__(kPrThreads) biased_prep(const BiasedPrep p) {
    constexpr int L = D / 8, R = kPrThreads / L, U = 4;         // lanes a row, rows of a turn, turns in flight
    const int tid = threadIdx.x, lane = tid & 31;
    const int64_t N = p.plan.N;
    const int B = p.plan.B;
    follow();
    if (blockIdx.x == 0) {
        if (!p.docs) {
            // as many sequences as threads at a time: their tiles are counted, and a tile finds its sequence among the counts
            __shared__ int s_first[kPrThreads + 1], s_sum[kPrThreads / 32];
            int done = 0;
            for (int b0 = 0; b0 < B; b0 += kPrThreads) {
                const int rows = b0 + tid < B ? __ldcg(p.plan.cu_k + b0 + tid + 1) - __ldcg(p.plan.cu_k + b0 + tid) : 0;
                int incl = (rows + kTileRows - 1) / kTileRows;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, incl, d);
                    if (lane >= d) incl += up;
                }
                if (lane == 31) s_sum[tid >> 5] = incl;
                __syncthreads();
                s_first[tid + 1] = incl + __reduce_add_sync(0xffffffffu, lane < tid >> 5 ? s_sum[lane] : 0);
                if (tid == 0) s_first[0] = 0;
                __syncthreads();
                const int total = min(s_first[kPrThreads], p.plan.max_tiles - done);
                for (int i = tid; i < total; i += kPrThreads) {
                    int s = 0;                              // the last one that begins at or before tile i
#pragma unroll
                    for (int step = kPrThreads / 2; step; step >>= 1) s += s_first[s + step] <= i ? step : 0;
                    const int seq = b0 + s, t0 = __ldcg(p.plan.cu_q + seq), t1 = __ldcg(p.plan.cu_q + seq + 1), k0 = __ldcg(p.plan.cu_k + seq), k1 = __ldcg(p.plan.cu_k + seq + 1);
                    const int key0 = k0 + (i - s_first[s]) * kTileRows, nkeys = min(kTileRows, k1 - key0);
                    const int to_tok = t1 - k1;             // from a row to the token that stands there
                    const bool shared = p.prefix_lens && key0 - k0 < __ldcg(p.prefix_lens + seq);
                    // (with fewer rows than tokens the first tokens stand before row k0 and see nothing)
                    const int first = max(max(t0, k0 + to_tok), shared ? t0 : key0 + to_tok);
                    const int last = p.window >= 0 ? (int)min((int64_t)t1 - 1, (int64_t)key0 + nkeys - 1 + to_tok + p.window) : t1 - 1;
                    p.plan.tiles[done + i] = make_int4(key0, nkeys, last >= first ? first : 0, last >= first ? last : -1);
                }
                done += total;
                __syncthreads();
            }
            for (int i = done + tid; i < p.plan.max_tiles; i += kPrThreads) p.plan.tiles[i] = make_int4(0, 0, 0, -1);
            __syncthreads();
        }
        plan_items<kPrThreads>(p.plan);
        return;
    }
    const int64_t ctas = gridDim.x - 1, me = (int64_t)(blockIdx.x - 1) * kPrThreads + tid, all = ctas * kPrThreads;
    const int64_t row16 = (int64_t)p.plan.Hk * L, qrow16 = (int64_t)p.Hq * L;
    const int k_first = __ldcg(p.plan.cu_k), k_end = __ldcg(p.plan.cu_k + B), q_end = __ldcg(p.plan.cu_q + B);
    if (!p.docs) {
        for (int64_t n = me; n < N; n += all) {
            Sees x = {0, -1, 0};
            if (n < q_end) {
                const int seq = find_seq<true>(p.plan.cu_q, B, (int)n);
                x = place_limits((int)n, __ldcg(p.plan.cu_k + seq), __ldcg(p.plan.cu_k + seq + 1), __ldcg(p.plan.cu_q + seq + 1), p.window,
                                 p.prefix_lens ? __ldcg(p.prefix_lens + seq) : 0);
            }
            p.lim.lo[n] = x.hi >= 0 ? x.lo : 0;
            p.lim.hi[n] = x.hi;
            p.lim.pos[n] = x.pos;
        }
        for (int64_t i = k_end * row16 + me; i < p.plan.Nk * row16; i += all) p.dk[i] = p.dv[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    // (K/V rows in front of the first sequence: where cu_seqlens_k is a part of a longer one)
    for (int64_t i = me; i < k_first * row16; i += all) p.dk[i] = p.dv[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int64_t i = q_end * qrow16 + me; i < N * qrow16; i += all) p.dq[i] = make_uint4(0u, 0u, 0u, 0u);
    // delta: L lanes a row of one head, U rows of a thread in flight
    const int part = tid % L;
    const uint32_t rows = (uint32_t)(N * p.Hq);
    for (int64_t r0 = (int64_t)(blockIdx.x - 1) * (R * U) + tid / L; r0 - tid / L < rows; r0 += ctas * (R * U)) {
        uint4 a[U], b[U];
        uint32_t n[U], h[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t r = min((uint32_t)r0 + u * R, rows - 1);
            n[u] = r / (uint32_t)p.Hq;
            h[u] = r - n[u] * (uint32_t)p.Hq;
            a[u] = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const ET*>(p.o) + ((int64_t)n[u] * p.Hq + h[u]) * D) + part);
            b[u] = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const ET*>(p.d_o) + (int64_t)n[u] * p.do_sn + (int64_t)h[u] * p.do_sh) + part);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t *x = &a[u].x, *y = &b[u].x;
            float acc = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = ElemTraits<ET>::unpack2(x[i]), w = ElemTraits<ET>::unpack2(y[i]);
                acc = fmaf(v.x, w.x, acc);
                acc = fmaf(v.y, w.y, acc);
            }
#pragma unroll
            for (int d = L / 2; d; d >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, d);
            if (part == 0 && r0 + u * R < rows) p.delta[(int64_t)h[u] * N + n[u]] = acc;
        }
    }
}

template <int D, typename ET>
static cudaError_t launch_prep(const BiasedPrep& p, cudaStream_t stream) {
    constexpr int per = kPrThreads / (D / 8) * 4;
    const int64_t want = (p.plan.N * p.Hq + per - 1) / per, most = 4 * (int64_t)sm_count();
    return launch_dependent(biased_prep<D, ET>, dim3((unsigned)(1 + (want < most ? want : most))), kPrThreads, 0, stream, 1, p);
}

static int biased_shape(int64_t N, int64_t Nk, int B, int Hq, int Hk, int D, SelShape* s) {
    if (N < 0 || Nk < 0 || B < 1 || Hq <= 0 || Hk <= 0 || Hq % Hk) return FSA_ERR_BAD_ARG;
    if ((D != 64 && D != 128) || Hq / Hk > 32 || Hk > 65535 || N >= kMaxTokens || Nk >= kMaxTokens || B >= kMaxTokens ||
        N * Hq >= ((int64_t)1 << 31)) return FSA_ERR_UNSUPPORTED;
    *s = SelShape{};
    s->N = N; s->Nk = Nk; s->B = B; s->Hq = Hq; s->Hk = Hk; s->G = Hq / Hk; s->D = D;
    s->TPT = (kTileRows / s->G) & ~3;
    // (places in the kernels' lists of tiles)
    return (biased_places(N, s->TPT, B) * Hk >= kBiasedMaxPlaces) ? FSA_ERR_UNSUPPORTED : FSA_OK;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int biased_mod(float sm_scale, float softcap, const float* slopes, const int32_t* doc_ids, int ahead, ScoreMod* m, int* which) {
    if (!(sm_scale > 0.f) || !(softcap >= 0.f)) return FSA_ERR_BAD_ARG;
    *which = (softcap > 0.f ? kModCap : 0) | (slopes ? kModBias : 0);
    *m = ScoreMod{};
    if (softcap > 0.f && !set_cap(m, sm_scale, softcap)) return FSA_ERR_BAD_ARG;
    m->slopes = slopes; m->key_ids = doc_ids; m->ahead = ahead;
    return FSA_OK;
}

}  // namespace fsa

using namespace fsa;

extern "C" int fsa_biased_attn_limits_bytes(int64_t N, int64_t* bytes_out) {
    if (!bytes_out || N < 0) return FSA_ERR_BAD_ARG;
    *bytes_out = BiasedLimits::bytes(N);
    return FSA_OK;
}

// How the forward is cut.  While its items leave SMs idle (two run on one), a tile's K/V rows are cut into chunks, no more than run at once, whose
// partial results are merged, where that is expected to gain: 0.75 us for every K/V tile that the longest item has fewer, against 4 us of the second
// launch and the partials' way to memory and back.  How long the longest is the host does not know: of several sequences, twice the mean.
// 16 tokens, 32 / 8 heads of 128, after 65536 in the cache: 80 us with 36 chunks, 799 uncut; 2000 tokens of 8 / 2 heads: 36 us with 2 chunks, 32 uncut.
struct ForwardCut {
    int nchunk = 1;
    ForwardCut(const SelShape& s, int window) {
        if (s.N == 0) return;
        const int64_t row_tiles = (s.N + s.TPT - 1) / s.TPT, items = (row_tiles > s.B ? row_tiles : s.B) * s.Hk;
        int64_t most = s.Nk, keys = s.Nk / s.B - s.N / s.B / 2;         // that a token sees, at most and about
        if (s.B > 1) keys *= 2;
        if (window >= 0 && most > (int64_t)window + s.TPT) most = (int64_t)window + s.TPT;
        if (keys > most) keys = most;
        int64_t n = 2 * sm_count() / items;
        if (n > most / (kBiasedBK * kBiasedLeast)) n = most / (kBiasedBK * kBiasedLeast);
        double best = 0.0;
        for (; n >= 2; n /= 2) {
            const double gain = 0.75 * (double)keys / kBiasedBK * (double)(n - 1) / (double)n - 4.0 - (double)(s.N * s.Hq * n * s.D * 8) / 5e6;
            if (gain > best) { best = gain; nchunk = (int)n; }
        }
    }
    int64_t bytes(const SelShape& s) const { return nchunk > 1 ? align_up(s.N * s.Hq * nchunk * s.D * 4, 256) + s.N * s.Hq * nchunk * 8 : 0; }
};

extern "C" int fsa_biased_attn_fwd_bytes(int64_t N, int64_t Nk, int B, int Hq, int Hk, int D, int window, int64_t* bytes_out) {
    SelShape s;
    const int rc = biased_shape(N, Nk, B, Hq, Hk, D, &s);
    if (rc) return rc;
    if (!bytes_out) return FSA_ERR_BAD_ARG;
    *bytes_out = ForwardCut(s, window).bytes(s);
    return FSA_OK;
}

extern "C" int fsa_biased_attn_fwd(const void* q, const void* k, const void* v, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                   const int32_t* doc_ids, const int32_t* prefix_lens, const float* slopes, int64_t N, int64_t Nk, int B, int Hq, int Hk,
                                   int D, int dtype, int64_t q_sn, int64_t q_sh, int64_t k_sn, int64_t v_sn, float sm_scale, float softcap, int window,
                                   void* o, float* lse, void* limits, int64_t limits_bytes, void* scratch, int64_t scratch_bytes, void* stream_) {
    SelShape s;
    int rc = biased_shape(N, Nk, B, Hq, Hk, D, &s);
    if (rc) return rc;
    if (dtype != FSA_DTYPE_BF16 && dtype != FSA_DTYPE_FP16) return FSA_ERR_BAD_ARG;
    // under these pairs a token would not see one stretch of rows
    if (prefix_lens && (window >= 0 || doc_ids)) return FSA_ERR_UNSUPPORTED;
    BiasedFwdLaunch l = {};
    int which;
    if ((rc = biased_mod(sm_scale, softcap, slopes, doc_ids, prefix_lens != nullptr, &l.mod, &which))) return rc;
    if (N == 0) return FSA_OK;
    if (!q || !k || !v || !cu_seqlens_q || !cu_seqlens_k || !o || !lse || !limits || Nk == 0) return FSA_ERR_BAD_ARG;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || ((uintptr_t)o & 31) || !aligned16(limits)) return FSA_ERR_BAD_ARG;
    if ((q_sn % 8) || (q_sh % 8) || (k_sn % 8) || (v_sn % 8) || k_sn < (int64_t)Hk * D || v_sn < (int64_t)Hk * D) return FSA_ERR_BAD_ARG;
    const ForwardCut cut(s, window);
    if (cut.nchunk > 1 && (!scratch || ((uintptr_t)scratch & 31))) return FSA_ERR_BAD_ARG;
    if (limits_bytes < BiasedLimits::bytes(N) || scratch_bytes < cut.bytes(s)) return FSA_ERR_WORKSPACE;
    (void)cudaGetLastError();
    if ((rc = ensure_context())) return rc;
    if ((rc = make_tile_map_3d_box(&l.q, q, dtype, D, N, Hq, q_sn, q_sh, s.TPT, s.G))) return rc;
    if ((rc = make_tile_map(&l.k, k, dtype, Nk, (int64_t)Hk * D, k_sn, 64))) return rc;
    if ((rc = make_tile_map(&l.v, v, dtype, Nk, (int64_t)Hk * D, v_sn, 64))) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    const BiasedLimits lim(limits, N);
    cudaError_t e;
    BiasedFwdParams& p = l.p;
    if ((e = biased_status_word(&p.status)) != cudaSuccess) return cuda_failed(e);
    p.cu_q = cu_seqlens_q; p.cu_k = cu_seqlens_k;
    l.window = window; l.prefix_lens = prefix_lens;
    if (doc_ids) {          // (else the kernel works them out for itself)
        if ((e = launch_limits(cu_seqlens_q, cu_seqlens_k, doc_ids, B, N, window, lim, stream)) != cudaSuccess) return cuda_failed(e);
        p.kv_lo = lim.lo; p.kv_hi = lim.hi;
        l.mod.pos = lim.pos;
    }
    p.N = N; p.Nk = Nk; p.B = B; p.Hq = Hq; p.Hk = Hk; p.G = s.G; p.TPT = s.TPT;
    p.scale_log2 = sm_scale * kLog2e;
    p.o = o; p.lse = lse;
    if (cut.nchunk > 1) {
        l.o_part = (float*)scratch;
        l.ml = (float2*)((char*)scratch + align_up(N * Hq * cut.nchunk * D * 4, 256));
        l.P = l.nchunk = cut.nchunk;
    }
    e = launch_biased_fwd(D, dtype, which, cut.nchunk > 1, l, (int)biased_places(N, s.TPT, B), stream);
    if (e == cudaSuccess && cut.nchunk > 1)     // (tokens outside the sequences have no partials)
        e = launch_biased_merge(D, dtype, BiasedMerge{l.o_part, l.ml, N * Hq, Hq, cut.nchunk, cut.nchunk, cu_seqlens_q, B, o, lse, 1, N}, stream);
    return e == cudaSuccess ? FSA_OK : cuda_failed(e);
}

// Items of dK / dV that the plan aims at.  (2 x 4096 tokens of documents: 636 us a pass with 5 an SM, 653 with 8, whose slabs take longer to join;
// 2 x 8192 capped: 1339 and 1366)
static int dkdv_items() { return 5 * sm_count(); }

// The same for dQ, one item an SM.  An SM needs about 1 us a K/V tile and 3 an item; uncut, as long as the longest item if that is more than an even share
// of all.  Cut, the parts' way to memory and back and 5 us of the launch that sums them come on top.  8192 tokens of one head: 41 us with four
// chunks, 113 uncut; of four sequences of 1000 and four heads 27 with two chunks, 22 uncut.
struct DqCut {
    int nchunk = 1;
    DqCut(const SelShape& s, int window) {
        if (s.N == 0) return;
        const int64_t row_tiles = (s.N + s.TPT - 1) / s.TPT, items = (row_tiles > s.B ? row_tiles : s.B) * s.Hk;
        double longest = (double)(s.Nk / s.B), mean = (double)(s.Nk / s.B - s.N / s.B / 2);
        if (s.B > 1) longest *= 1.25;           // (the host does not know)
        if (window >= 0 && longest > (double)window + s.TPT) longest = (double)window + s.TPT;
        if (mean > longest) mean = longest;
        longest /= kBiasedBK;
        const double shared = mean / kBiasedBK * (double)items / sm_count(), each = 3.0 * (double)items / sm_count();
        double best = 0.0;
        for (int n = 1; n == 1 || (n <= 64 && (double)n * kBiasedLeast <= longest); n *= 2) {
            const double part = longest / n + 3.0, all = shared + n * each;
            const double t = (part > all ? part : all) + (n > 1 ? 5.0 + (double)(s.N * s.Hq * n * s.D * 8) / 5e6 : 0.0);
            if (n == 1 || t < best) { best = t; nchunk = n; }
        }
    }
    int64_t bytes(const SelShape& s) const { return nchunk > 1 ? s.N * s.Hq * nchunk * s.D * 4 : 0; }
};

extern "C" int fsa_biased_attn_bwd_bytes(int64_t N, int64_t Nk, int B, int Hq, int Hk, int D, int window, int64_t* bytes_out) {
    SelShape s;
    const int rc = biased_shape(N, Nk, B, Hq, Hk, D, &s);
    if (rc) return rc;
    if (!bytes_out) return FSA_ERR_BAD_ARG;
    *bytes_out = align_up(N * Hq * 4, 1024) + align_up(range_kv_plan_bytes(s, dkdv_items()), 1024) + align_up(range_kv_slab_bytes(s, dkdv_items()), 1024) + DqCut(s, window).bytes(s);
    return FSA_OK;
}

extern "C" int fsa_biased_attn_bwd(const void* q, const void* k, const void* v, const void* o, const float* lse, const void* d_o,
                                   const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, const int32_t* doc_ids, const int32_t* prefix_lens, const float* slopes,
                                   int64_t N, int64_t Nk, int B, int Hq, int Hk, int D, int dtype, int64_t q_sn, int64_t q_sh, int64_t k_sn, int64_t v_sn,
                                   int64_t do_sn, int64_t do_sh, float sm_scale, float softcap, int window, void* dq, void* dk, void* dv, void* limits,
                                   int64_t limits_bytes, void* scratch, int64_t scratch_bytes, void* stream_) {
    SelShape s;
    int rc = biased_shape(N, Nk, B, Hq, Hk, D, &s);
    if (rc) return rc;
    if (dtype != FSA_DTYPE_BF16 && dtype != FSA_DTYPE_FP16) return FSA_ERR_BAD_ARG;
    ScoreMod mod;
    int which;
    if ((rc = biased_mod(sm_scale, softcap, slopes, doc_ids, prefix_lens != nullptr, &mod, &which))) return rc;
    if (N == 0) {           // nobody sees the keys
        if (Nk > 0 && (!dk || !dv)) return FSA_ERR_BAD_ARG;
        (void)cudaGetLastError();
        cudaError_t e = cudaSuccess;
        for (void* x : {dk, dv})
            if (e == cudaSuccess && Nk > 0) e = cudaMemsetAsync(x, 0, (size_t)(Nk * Hk * D * 2), (cudaStream_t)stream_);
        return e == cudaSuccess ? FSA_OK : cuda_failed(e);
    }
    if (!q || !k || !v || !o || !lse || !d_o || !cu_seqlens_q || !cu_seqlens_k || !dq || !dk || !dv || !limits || !scratch || Nk == 0) return FSA_ERR_BAD_ARG;
    for (const void* x : {q, k, v, o, d_o, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)limits, (const void*)scratch})
        if (!aligned16(x)) return FSA_ERR_BAD_ARG;
    if (((uintptr_t)dq & 31) || ((uintptr_t)dk & 31) || ((uintptr_t)dv & 31)) return FSA_ERR_BAD_ARG;
    if ((q_sn % 8) || (q_sh % 8) || (k_sn % 8) || (v_sn % 8) || (do_sn % 8) || (do_sh % 8) || k_sn < (int64_t)Hk * D || v_sn < (int64_t)Hk * D) return FSA_ERR_BAD_ARG;
    int64_t need = 0;
    if ((rc = fsa_biased_attn_bwd_bytes(N, Nk, B, Hq, Hk, D, window, &need))) return rc;
    if (limits_bytes < BiasedLimits::bytes(N) || scratch_bytes < need) return FSA_ERR_WORKSPACE;
    (void)cudaGetLastError();
    if ((rc = ensure_context())) return rc;
    CUtensorMap kmap, vmap;
    if ((rc = make_tile_map(&kmap, k, dtype, Nk, (int64_t)Hk * D, k_sn, 64))) return rc;
    if ((rc = make_tile_map(&vmap, v, dtype, Nk, (int64_t)Hk * D, v_sn, 64))) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    const BiasedLimits lim(limits, N);
    mod.pos = lim.pos;
    char* sp = (char*)scratch;
    SelBwdArgs a = {};
    a.q = q; a.d_o = d_o; a.o = o;
    a.q_sn = q_sn; a.q_sh = q_sh; a.do_sn = do_sn; a.do_sh = do_sh; a.o_sn = (int64_t)Hq * D; a.o_sh = D;
    a.lse = lse; a.cu = cu_seqlens_q; a.sm_scale = sm_scale;
    a.delta = (float*)sp;           sp += align_up(N * Hq * 4, 1024);
    a.bd = SelBounds{cu_seqlens_k, lim.lo, lim.hi};
    a.dq = dq; a.dk = dk; a.dv = dv;
    RangeKvPlan plan = {};
    plan.cu_q = cu_seqlens_q; plan.cu_k = cu_seqlens_k; plan.kv_lo = lim.lo; plan.kv_hi = lim.hi;
    plan.N = N; plan.Nk = Nk; plan.B = B; plan.Hk = Hk; plan.TPT = s.TPT;
    plan.aim = dkdv_items();
    plan.max_tiles = (int)range_kv_max_tiles(s);
    plan.D = D;
    plan.counts = (int*)sp;
    plan.tiles = (int4*)(sp + 256);
    plan.multi = plan.tiles + plan.max_tiles;
    plan.items = plan.multi + plan.max_tiles;
    sp += align_up(range_kv_plan_bytes(s, dkdv_items()), 1024);
    a.slabs = (float*)sp;           sp += align_up(range_kv_slab_bytes(s, dkdv_items()), 1024);
    float* part = (float*)sp;
    const DqCut cut(s, window);
    int* status = nullptr;
    cudaError_t e = biased_status_word(&status);
    BiasedPrep prep = {plan, lim, prefix_lens, window, doc_ids != nullptr, o, d_o, do_sn, do_sh, Hq, a.delta, (uint4*)dq, (uint4*)dk, (uint4*)dv};
    // with documents the forward has left the limits, and the stretches are looked for
    if (e == cudaSuccess && doc_ids) e = launch_range_key_tiles(plan, a, stream);
    const bool bf16 = dtype == FSA_DTYPE_BF16;
    if (e == cudaSuccess && D == 128) e = bf16 ? launch_prep<128, __nv_bfloat16>(prep, stream) : launch_prep<128, __half>(prep, stream);
    if (e == cudaSuccess && D == 64) e = bf16 ? launch_prep<64, __nv_bfloat16>(prep, stream) : launch_prep<64, __half>(prep, stream);
    if (e == cudaSuccess) e = launch_biased_bwd_dq(dtype, a, s, kmap, vmap, status, mod, which, cut.nchunk, part, stream);
    if (e == cudaSuccess) e = launch_biased_bwd_dkdv(dtype, plan, a, s, kmap, vmap, status, mod, which, stream);
    // (no stretch of so few row tiles is cut)
    if (e == cudaSuccess && N > (int64_t)kRkMinTiles * s.TPT) e = launch_range_dkdv_reduce(dtype, plan, a.slabs, dk, dv, sm_count(), stream);
    if (e == cudaSuccess && cut.nchunk > 1) e = launch_biased_dq_sum(dtype, part, a, s, cut.nchunk, stream);
    return e == cudaSuccess ? FSA_OK : cuda_failed(e);
}

extern "C" int fsa_biased_read_status(int* status_out) {
    if (!status_out) return FSA_ERR_BAD_ARG;
    // (of all streams: torch's own do not wait for the legacy one, which the copies go through)
    int word = 0;
    const int none = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&word, g_biased_status, sizeof(int));
    if (e == cudaSuccess && word) e = cudaMemcpyToSymbol(g_biased_status, &none, sizeof(int));
    *status_out = word & 255;
    return e == cudaSuccess ? FSA_OK : cuda_failed(e);
}

// A wait of these operators that runs out, harmlessly: nobody arrives at the barrier.
static __global__ void biased_wait_timeout_probe(int* word) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        mbar_init(&bar, 1);
        mbar_init_fence();
        mbar_wait_stamped(&bar, 0, word, stamped_wait_limit(word));
    }
}

extern "C" int fsa_biased_debug_wait_timeout(void* stream_) {
    (void)cudaGetLastError();
    int* word = nullptr;
    cudaError_t e = biased_status_word(&word);
    if (e == cudaSuccess) {
        biased_wait_timeout_probe<<<1, 32, 0, (cudaStream_t)stream_>>>(word);
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? FSA_OK : cuda_failed(e);
}
