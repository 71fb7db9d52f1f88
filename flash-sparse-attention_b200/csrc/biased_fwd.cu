// Forward of attention with changed scores (score.cuh) for sm_100a: every token attends one stretch of K/V rows, its scores capped by a tanh
// and / or biased by distance.  Also its form with the K/V rows cut into chunks (kModSplit), whose partial results are merged afterwards
// (biased_decode.cu): few queries over many rows, and rows that many sequences of a decoded batch share.
//
// An item is a tile of <= 128 rows (query head of a GQA group, TPT consecutive tokens of one sequence) x one KV head, as in range_dense.cu; the
// CTA walks the K/V tiles that the rows see, 64 rows each, from the nearest to the furthest, with the accumulator in TMEM, and writes o and
// lse once.  Two CTAs share an SM (113 KB of shared memory at D = 128, 256 TMEM columns each).
//   warp 0      finds the items (cluster launch control: a running CTA takes over those whose CTA has not started); TMA producer
//   warp 1      one elected thread issues S = Q K^T of the next K/V tile into the other of two TMEM buffers, then O (+)= P V of this one
//   warps 2..5  one row per thread: changed scores, running maximum and sum, P -> TMEM over S; epilogue
// (S of two K/V tiles at a time, N = 128, reads Q from shared memory half as often, but waits for two tiles: 314 us for what takes 282, capped.)
// The row threads do their arithmetic in one pass over a tile: it takes the rows' references for given and the tanh's arguments for near,
// so that the polynomial and the sums run under the exp2 (16 a cycle and SM, 512 cycles a tile, like the products).  What it assumed is looked
// at afterwards; where it does not hold (a row's first tile, a maximum far above the reference, scores near the cap, keys that some row
// does not see) the tile takes three passes: scores, maximum, exp2.  The nearest tile comes first because a distance bias sets the reference
// there (furthest first, every tile raised it: 676 us for what now takes 248).
// 2 x 8192 tokens, 8 / 4 heads of 128: 240 us plain, 282 capped (975 TFLOP/s), 248 with a distance bias, 299 with both.  Capped, the tensor cores' queue
// is 64 % busy, exp2 49 %, issue 49 %: two row warps a scheduler do not hide each other's loads from TMEM and chains of arithmetic altogether.
#include "../../include/fsa_sm100.h"
#include <climits>

#include "biased.cuh"

namespace fsa {

constexpr int kBfThreads = 192;
constexpr int kBfV = 3;             // V tiles in flight

struct BfItem {
    int z, h, seq, tok0, ne, row_lo, nblk, row_hi;     // chunk (-1: no more items); rows [row_lo, row_hi] are those that a row of the item sees
};

// How far (log2 units) a row's maximum may be above its reference before that is raised.  Nothing is lost by a low reference as long as P is in
// range of its type: bf16 reaches as far as the 32-bit sums do; fp16 ends at 2^16, and the lower the reference, the fewer P are below its
// normal numbers.
template <typename ET> constexpr float kBfLazy = ElemTraits<ET>::kIsBF16 ? 64.f : 14.f;

template <int D, int MOD, typename ET>
__global__ void __launch_bounds__(kBfThreads, 2) biased_fwd(const __grid_constant__ BiasedFwdLaunch launch) {
    constexpr int BK = kBiasedBK, KH = D / 64;
    constexpr int kQ = kTileRows * D * 2;
    constexpr int kSlabQ = kTileRows * 128;          // 64 columns of the Q tile
    constexpr int kKt = BK * D * 2;                  // one K (or V) tile
    constexpr uint32_t kCols = 256;
    constexpr int cS = 0, cO = 2 * BK;
    constexpr bool kSplit = (MOD & kModSplit) != 0;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + kQ;                           // [2]
    uint8_t* sV = sK + 2 * kKt;                      // [kBfV]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kBfV * kKt);
    uint64_t* q_full = bars;
    uint64_t* q_empty = bars + 1;       // the item's last S product is done
    uint64_t* k_full = bars + 2;        // [2]
    uint64_t* k_empty = bars + 4;       // [2] S of the tile is done with K
    uint64_t* s_full = bars + 6;        // [2] ... and there to be read
    uint64_t* p_full = bars + 8;        // [2] P is in its place
    uint64_t* pv_done = bars + 10;      // [2] ... and has been multiplied
    uint64_t* v_full = bars + 12;       // [kBfV]
    uint64_t* v_empty = v_full + kBfV;  // [kBfV]
    uint64_t* o_free = v_empty + kBfV;  // the 128 row threads have read an item's accumulator
    uint64_t* it_full = o_free + 1;     // the next item is known
    uint64_t* it_empty = o_free + 2;    // ... has been taken by the five other warps
    uint64_t* claim = o_free + 3;       // the answer to a claim has arrived
    int* s_claim = reinterpret_cast<int*>(bars + 22);    // 16 bytes
    int4* s_item = reinterpret_cast<int4*>(bars + 24);   // [2 items][2]
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 32);
    int* status = reinterpret_cast<int*>(bars + 32) + 1;     // of this CTA

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const BiasedFwdParams& p = launch.p;
    const uint32_t limit = stamped_wait_limit(p.status);
    const int G = p.G, TPT = p.TPT;
    // First and last K/V row that a token sees, and its place.  kModSplit: with shared rows a token is a sequence of the batch, whose own rows
    // follow them.
    auto limits = [&](int seq, int tok) {
        Sees x;
        if (kSplit && launch.seq_len) {
            const int k0 = __ldcg(p.cu_k + seq), k1 = __ldcg(p.cu_k + seq + 1), len = __ldcg(launch.seq_len + tok);
            x.pos = k1 + len - 1;
            x.lo = launch.window >= 0 ? max(k0, x.pos - launch.window) : k0;
            x.hi = len > 0 ? k1 - 1 : -1;
        } else if (p.kv_lo) {
            x.lo = __ldcg(p.kv_lo + tok);
            x.hi = __ldcg(p.kv_hi + tok);
            x.pos = (MOD & kModBias) ? __ldcg(launch.mod.pos + tok) : 0;
        } else {
            const int k0 = __ldcg(p.cu_k + seq), k1 = __ldcg(p.cu_k + seq + 1);
            x = place_limits(tok, k0, k1, __ldcg(p.cu_q + seq + 1), launch.window, launch.prefix_lens ? __ldcg(launch.prefix_lens + seq) : 0);
        }
        return x;
    };
    const bool beside = kSplit && launch.seq_len;        // it needs nothing of the kernel before it
    if (!beside) follow_late();
    if (tid == 0) {
        *status = kStatusOk;
        mbar_init(q_full, 1); mbar_init(q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128); mbar_init(&pv_done[i], 1);
        }
        for (int i = 0; i < kBfV; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
        mbar_init(o_free, 128); mbar_init(it_full, 1); mbar_init(it_empty, 5); mbar_init(claim, 1);
        mbar_init_fence();
    }
    // (warp 0 has set the barriers up itself and needs no TMEM: it goes on to find its item)
    if (warp == 0) {
        __syncwarp();
        asm volatile("bar.arrive 2, 192;" ::: "memory");
    } else {
        // Rows past G * TPT of the Q tile are never loaded, and their scores go nowhere; but they have a part in their warp's choice of the way through a tile, and with
        // what a kernel before left there the other rows' last bits changed from run to run.
        for (int i = G * TPT * 8 + tid - 32; i < kTileRows * 8; i += kBfThreads - 32)
            for (int b = 0; b < KH; ++b) reinterpret_cast<uint4*>(sQ + b * kSlabQ)[i] = make_uint4(0u, 0u, 0u, 0u);
        fence_async_smem();
        if (warp == 1) tmem_alloc(&tmem_slot, kCols);
        tc_fence_before();
        asm volatile("bar.sync 2, 192;" ::: "memory");
        tc_fence_after();
        if (!beside) let_next_start();
    }
    const uint32_t tbase = warp ? tmem_slot : 0u;
    // Item n of this CTA.  Each of the five other warps takes every item once, in order; z < 0 ends the list.
    auto read_item = [&](int n) {
        const int4 x = s_item[(n & 1) * 2], y = s_item[(n & 1) * 2 + 1];
        BfItem m;
        m.z = x.x; m.h = x.y; m.seq = x.z; m.tok0 = x.w;
        m.ne = y.x; m.row_lo = y.y; m.nblk = y.z; m.row_hi = y.w;
        return m;
    };
    auto take_item = [&](int n, bool& ok) {
        ok = ok && mbar_wait(it_full, n & 1, status, limit);
        BfItem m = read_item(n);
        ok = warp_ok(ok);
        if (!ok) m.z = -1;
        if (lane == 0) mbar_arrive(it_empty);
        return m;
    };

    if (warp == 0) {
        // ------------------------------------------------------------------ items and TMA producer
        bool ok = true;
        int n = 0, claims = 0, qi = 0, c = 0;           // items, claims, non-empty items, K/V tiles so far
        int bx = blockIdx.x, z = blockIdx.y;
        while (ok) {
            bool asked = false;
            auto ask = [&]() {
                mbar_expect_tx(claim, 16);
                claim_next_cta(smem_u32(s_claim), claim);
                asked = true;
            };
            int seq, tok0, ne;
            const int h = bx % p.Hk;
            find_ranked_tile(p.cu_q, p.cu_k, p.B, TPT, bx / p.Hk, lane, seq, tok0, ne);
            if (seq >= 0) {
                // lowest and highest K/V row any token of the tile sees
                int lo = INT_MAX, hi = -1;
                for (int e = lane; e < ne; e += 32) {
                    const Sees x = limits(seq, tok0 + e);
                    if (x.hi >= x.lo) { lo = min(lo, x.lo); hi = max(hi, x.hi); }
                }
                lo = max(__reduce_min_sync(0xffffffffu, lo), 0);
                hi = min(__reduce_max_sync(0xffffffffu, hi), (int)p.Nk - 1);
                int nblk = hi >= lo ? (hi - lo) / BK + 1 : 0;
                if constexpr (kSplit) {
                    // chunks of one size (the last one takes what is left), so that long shared rows are cut more often than short ones, or equal ones
                    const int size = launch.chunk ? launch.chunk : max(kBiasedLeast, (nblk + launch.nchunk - 1) / launch.nchunk);
                    const int b0 = min(z * size, nblk);
                    nblk = z + 1 < launch.nchunk ? min(size, nblk - b0) : nblk - b0;
                    lo += b0 * BK;
                    hi = min(hi, lo + nblk * BK - 1);
                }
                if (n > 0) ok = ok && mbar_wait(it_empty, (n - 1) & 1, status, limit);
                ok = warp_ok(ok);
                if (ok && lane == 0) {
                    s_item[(n & 1) * 2] = make_int4(z, h, seq, tok0);
                    s_item[(n & 1) * 2 + 1] = make_int4(ne, lo, nblk, hi);
                    mbar_arrive(it_full);
                }
                ++n;
                if (lane == 0 && nblk > 0) {
                    ok = ok && mbar_wait(q_empty, (qi & 1) ^ 1, status, limit);
                    if constexpr (!kSplit) ask();       // not earlier: a CTA is to be one item ahead, not to take the share of others
                    if (ok) {
                        mbar_expect_tx(q_full, (uint32_t)(KH * 128 * TPT * G));
#pragma unroll
                        for (int b = 0; b < KH; ++b) tma_load_3d(smem_u32(sQ + b * kSlabQ), &launch.q, b * 64, tok0, h * G, q_full);
                    }
                    // K and V tiles in the order that the MMA warp needs them: K(0), K(1), V(0), K(2), V(1), ...
                    for (int step = 0; step < nblk + 1 && ok; ++step) {
                        const int jk = c + step, jv = jk - 1;
                        if (step < nblk) {
                            const int st = jk & 1;
                            ok = ok && mbar_wait(&k_empty[st], ((jk >> 1) & 1) ^ 1, status, limit);
                            if (!ok) break;
                            mbar_expect_tx(&k_full[st], (uint32_t)kKt);
#pragma unroll
                            for (int b = 0; b < KH; ++b)
                                tma_load_2d(smem_u32(sK + st * kKt + b * (BK * 128)), &launch.k, h * D + b * 64, lo + (nblk - 1 - step) * BK, &k_full[st]);
                        }
                        if (step > 0) {
                            const int st = jv % kBfV;
                            ok = ok && mbar_wait(&v_empty[st], ((jv / kBfV) & 1) ^ 1, status, limit);
                            if (!ok) break;
                            mbar_expect_tx(&v_full[st], (uint32_t)kKt);
#pragma unroll
                            for (int b = 0; b < KH; ++b)
                                tma_load_2d(smem_u32(sV + st * kKt + b * (BK * 128)), &launch.v, h * D + b * 64, lo + (nblk - step) * BK, &v_full[st]);
                        }
                    }
                }
                c += nblk;
                qi += nblk > 0;
            } else if (!kSplit && ne == 0) {
                // There are max_tiles >= N / TPT + B places in the list and at most used / TPT + B tiles: those left over clear the rows behind the
                // last sequence, TPT tokens each.
                const int64_t t0 = (int64_t)__ldcg(p.cu_q + p.B) + (int64_t)tok0 * TPT;
                const int nt = (int)min((int64_t)TPT, p.N - t0);
                for (int i = lane; i < nt * G; i += 32) p.lse[(int64_t)(h * G + i % G) * p.N + t0 + i / G] = -INFINITY;
                for (int i = lane; i < nt * (G * D / 8); i += 32)
                    reinterpret_cast<uint4*>(p.o)[((t0 + i / (G * D / 8)) * p.Hq + h * G) * (D / 8) + i % (G * D / 8)] = make_uint4(0u, 0u, 0u, 0u);
            }
            // (chunks: an item a CTA.  Beside another kernel some CTAs start late, and the early ones would have taken their items: twice the time)
            if constexpr (kSplit) break;
            if (lane == 0 && !asked) ask();
            // (the answer is in shared memory before this CTA may end, whatever happened above)
            const bool answered = mbar_wait(claim, claims & 1, status, limit);
            ok = ok && answered;
            ++claims;
            int none;
            const bool more = claimed_cta(smem_u32(s_claim), bx, z, none);
            ok = warp_ok(ok);
            fence_async_smem();
            if (!more) break;
        }
        if (n > 0) ok = ok && mbar_wait(it_empty, (n - 1) & 1, status, limit);
        ok = warp_ok(ok);
        if (ok && lane == 0) {          // (else the other warps give up by themselves: one may still read this place)
            s_item[(n & 1) * 2] = make_int4(-1, 0, -1, 0);
            s_item[(n & 1) * 2 + 1] = make_int4(0, 0, 0, 0);
            mbar_arrive(it_full);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        const bool leader = elect_one();
        constexpr uint32_t idesc_s = umma_idesc(ElemTraits<ET>::kIsBF16, 128, BK, false, false);
        constexpr uint32_t idesc_o = umma_idesc(ElemTraits<ET>::kIsBF16, 128, D, false, true);
        constexpr uint32_t hi_1024 = umma_desc_hi(1024);
        const uint32_t q_lo = umma_desc_lo(smem_u32(sQ), 16);
        const uint32_t k_lo = umma_desc_lo(smem_u32(sK), 16);
        const uint32_t v_lo = umma_desc_lo(smem_u32(sV), BK * 128);     // MN-major: LBO = slab stride
        bool ok = true;
        int n = 0, qi = 0, c = 0;
        // S(t) takes the place of P(t - 2): products of two shapes may run in another order than they were issued, so it waits for the one that
        // reads P(t - 2)
        auto issue_s = [&](int t, bool last) {
            const int st = t & 1;
            ok = ok && mbar_wait(&k_full[st], (t >> 1) & 1, status, limit);
            if (t >= 2) ok = ok && mbar_wait(&pv_done[st], ((t - 2) >> 1) & 1, status, limit);
            ok = warp_ok(ok);
            if (!ok) return;
            tc_fence_after();
            if (leader) {
                constexpr int kSlabB = (BK * 128) >> 4;
                const uint32_t b_lo = k_lo + (uint32_t)(st * (kKt >> 4));
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma_ss(tbase + cS + st * BK, umma_desc_pack(q_lo + (ks >> 2) * (kSlabQ >> 4) + (ks & 3) * 2, hi_1024),
                            umma_desc_pack(b_lo + (ks >> 2) * kSlabB + (ks & 3) * 2, hi_1024), idesc_s, ks > 0);
                umma_commit(&k_empty[st]);
                umma_commit(&s_full[st]);
                if (last) umma_commit(q_empty);
            }
            __syncwarp();
        };
        for (BfItem m = take_item(n, ok); m.z >= 0; m = take_item(++n, ok)) {
            if (m.nblk == 0) continue;
            ok = ok && mbar_wait(q_full, qi & 1, status, limit);
            issue_s(c, m.nblk == 1);
            for (int j = 0; j < m.nblk && ok; ++j, ++c) {
                const int st = c & 1, sv = c % kBfV;
                if (j + 1 < m.nblk) issue_s(c + 1, j + 2 == m.nblk);
                if (j == 0 && qi > 0) ok = ok && mbar_wait(o_free, (qi - 1) & 1, status, limit);
                ok = ok && mbar_wait(&p_full[st], (c >> 1) & 1, status, limit);
                ok = ok && mbar_wait(&v_full[sv], (c / kBfV) & 1, status, limit);
                ok = warp_ok(ok);
                if (!ok) break;
                tc_fence_after();
                if (leader) {
                    const uint32_t b_lo = v_lo + (uint32_t)(sv * (kKt >> 4));
#pragma unroll
                    for (int ks = 0; ks < BK / 16; ++ks)
                        umma_ts(tbase + cO, tbase + cS + st * BK + ks * 8, umma_desc_pack(b_lo + ks * (2048 >> 4), hi_1024), idesc_o,
                                (j > 0 || ks > 0) ? 1u : 0u);
                    umma_commit(&v_empty[sv]);
                    umma_commit(&pv_done[st]);
                }
                __syncwarp();
            }
            ++qi;
        }
    } else {
        // ------------------------------------------------------------------ softmax and epilogue: one row per thread
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
        const int g = r / TPT, e = r - g * TPT;
        const float to_log2 = (MOD & kModCap) ? launch.mod.cap_log2 : p.scale_log2;
        const float scale_log2 = (MOD & kModBias) ? 1.f : to_log2;           // from v to log2 units, once it has been changed
        const NearTanh near(launch.mod, to_log2);
        // What the row of an item needs: the K/V rows that it sees, and with a bias the slope of its head (log2 units) and its token's place.
        // (A place without a row sees everything: it is not what keeps its warp from the short way.)
        struct Row { int lo, hi; float slope; int pos; };
        auto load_row = [&](const BfItem& m) {
            Row x = {0, INT_MAX, 0.f, INT_MAX};
            if (m.z >= 0 && g < G && e < m.ne) {
                const Sees s = limits(m.seq, m.tok0 + e);
                x.lo = s.lo; x.hi = s.hi;
                if constexpr (MOD & kModBias) {
                    x.slope = __ldcg(launch.mod.slopes + m.h * G + g) * kLog2e;
                    x.pos = s.pos;
                }
            }
            return x;
        };
        bool ok = true, far = false;
        int n = 0, c = 0;
        BfItem m = take_item(n, ok);
        Row row = load_row(m);
        // (the four warps leave the loop together: they meet at barriers in it)
        for (ok = bar_all(1, 128, ok); ok && m.z >= 0;) {
            const int lo_r = row.lo - m.row_lo, hi_r = min(row.hi, (int)p.Nk - 1) - m.row_lo;      // rows past the end of K/V do not exist
            const float slope_r = row.slope;
            const int pos_r = row.pos - m.row_lo;
            const int nblk = m.nblk;
            // What decides on a warp's way through a tile, and with it on last bits, are scores of its tokens with keys that they see: not those of places without
            // a token, whose reference is infinite, and none of a tile that is not seen whole (rows of other sequences or of none, which may hold anything).
            float m_ref = g < G && e < m.ne ? -INFINITY : INFINITY, l_run = 0.f;
            // tiles that all rows of the warp see whole (and none of them behind a token's place): [whole_lo, whole_hi]
            const int whole_lo = __reduce_max_sync(0xffffffffu, (max(lo_r, 0) + BK - 1) / BK);
            const int whole_hi = __reduce_min_sync(0xffffffffu, (((MOD & kModBias) && launch.mod.ahead ? min(hi_r, pos_r) : hi_r) + 1 >> 6) - 1);
            bool fresh = true;                             // some row of the warp has no reference yet
            for (int t = nblk - 1; t >= 0; --t, ++c) {     // (left by all lanes at the vote below)
                const int st = c & 1;
                ok = ok && mbar_wait(&s_full[st], (c >> 1) & 1, status, limit);
                tc_fence_after();
                const uint32_t tS = tbase + lane_off + cS + st * BK;
                uint32_t v[BK], pk[BK / 2];
                tmem_ld32(tS, *reinterpret_cast<uint32_t (*)[32]>(&v[0]));
                tmem_ld32(tS + 32, *reinterpret_cast<uint32_t (*)[32]>(&v[32]));
                tmem_ld_wait();
                // p = exp2(score - reference) of two columns
                uint64_t ls[2] = {0, 0};
                auto two = [&](int i, uint64_t s) {
                    const float2 x = f32x2_get(s);
                    const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
                    ls[(i >> 1) & 1] = add_f32x2(ls[(i >> 1) & 1], f32x2(p0, p1));
                    pk[i >> 1] = ElemTraits<ET>::pack2(p0, p1);
                };
                auto pair = [&](int i) { return f32x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])); };
                const float rel = (float)(pos_r - t * BK);
                bool passes = far || fresh || t < whole_lo || t > whole_hi;
                if (!passes) {
                    const uint64_t s2 = f32x2(to_log2, to_log2);
                    const float base = (MOD & kModBias) ? fmaf(-slope_r, rel, -m_ref) : -m_ref;
                    float top[2] = {-INFINITY, -INFINITY}, big[2] = {0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < BK; i += 2) {
                        if constexpr (MOD & kModCap) big[(i >> 1) & 1] = max3_abs(big[(i >> 1) & 1], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                        const uint64_t x = fma_f32x2(pair(i), (MOD & kModCap) ? near.slope(pair(i)) : s2,
                                                     (MOD & kModBias) ? f32x2(fmaf(slope_r, (float)i, base), fmaf(slope_r, (float)(i + 1), base)) : f32x2(base, base));
                        const float2 y = f32x2_get(x);
                        top[(i >> 1) & 1] = max3(top[(i >> 1) & 1], y.x, y.y);
                        two(i, x);
                    }
                    passes = __any_sync(0xffffffffu, !(fmaxf(top[0], top[1]) <= kBfLazy<ET>) || ((MOD & kModCap) && !(fmaxf(big[0], big[1]) <= launch.mod.near_v) && m_ref < INFINITY) || !ok);
                }
                if (passes) {
                    if (!warp_stays(ok)) break;
                    const int c_lo = max(0, lo_r - t * BK), c_hi = min(BK, hi_r - t * BK + 1);      // visible columns [c_lo, c_hi)
                    if constexpr (MOD & kModCap) far = cap_scores(v, launch.mod.x_scale, launch.mod.near_v, m_ref < INFINITY) && t >= whole_lo && t <= whole_hi;
                    if constexpr (MOD & kModBias)
                        bias_scores(v, to_log2, slope_r, rel, launch.mod.ahead && __any_sync(0xffffffffu, t * BK + c_hi - 1 > pos_r));
                    if (c_lo > 0 || c_hi < BK) {
                        // bit i: column i is seen
                        const int v_hi = max(c_hi, 0), v_lo = min(c_lo, BK);
                        const uint64_t vis = v_hi > v_lo ? (~0ull >> (BK - v_hi + v_lo)) << v_lo : 0ull;
                        const uint32_t vis2[2] = {(uint32_t)vis, (uint32_t)(vis >> 32)};
#pragma unroll
                        for (int i = 0; i < BK; ++i)
                            if (!(vis2[i >> 5] >> (i & 31) & 1u)) v[i] = 0xff800000u;      // -inf: exp2 gives exactly 0
                    }
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < BK; i += 4) {
                        mx[0] = max3(mx[0], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                        mx[1] = max3(mx[1], __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
                    }
                    const float m_blk = fmaxf(mx[0], mx[1]) * scale_log2;
                    // raise the reference only when this tile exceeds it by a lot; the first finite maximum sets it
                    float alpha = 1.f;
                    const bool raise = m_blk > m_ref + kBfLazy<ET>;     // false when m_blk is -inf; true when m_ref is -inf and m_blk finite
                    if (raise) {
                        alpha = m_ref == -INFINITY ? 0.f : ex2_approx(m_ref - m_blk);
                        m_ref = m_blk;
                        l_run *= alpha;
                    }
                    // accumulator rows already hold products: rescale them when any row of the warp changes reference
                    const bool scale_acc = __any_sync(0xffffffffu, (raise && t < nblk - 1) || !ok);
                    if (scale_acc) {
                        ok = ok && mbar_wait(&pv_done[(c - 1) & 1], ((c - 1) >> 1) & 1, status, limit);
                        if (!warp_stays(ok)) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c0 = 0; c0 < D; c0 += 32) {
                            uint32_t a[32];
                            tmem_ld32(tbase + lane_off + cO + c0, a);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) a[i] = __float_as_uint(__uint_as_float(a[i]) * alpha);
                            tmem_st32(tbase + lane_off + cO + c0, a);
                        }
                    }
                    fresh = __any_sync(0xffffffffu, m_ref == -INFINITY);
                    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;     // all columns masked so far: every p is exp2(-inf) = 0
                    const uint64_t scale2 = f32x2(scale_log2, scale_log2), m2 = f32x2(-m_use, -m_use);
                    ls[0] = ls[1] = 0;
#pragma unroll
                    for (int i = 0; i < BK; i += 2) two(i, (MOD & kModBias) ? add_f32x2(pair(i), m2) : fma_f32x2(pair(i), scale2, m2));
                }
                const float2 l2 = f32x2_get(add_f32x2(ls[0], ls[1]));
                l_run += l2.x + l2.y;
                tmem_st32(tS, pk);
                tmem_st_wait();
                if (launch.mod.key_ids || t == nblk - 1) {
                    // V rows that no row of the item sees are multiplied by p = 0, but 0 x NaN is NaN: zeros take their place.  Every thread
                    // has half of one of the 64 rows.
                    const int kr = m.row_lo + t * BK + (r & (BK - 1));
                    const bool unseen = kr > m.row_hi || (launch.mod.key_ids && __ldcg(launch.mod.key_ids + kr) < 0);
                    if (__any_sync(0xffffffffu, unseen)) {
                        const int sv = c % kBfV;
                        ok = ok && mbar_wait(&v_full[sv], (c / kBfV) & 1, status, limit);
                        if (unseen && ok)
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                const int chunk = (r >> 6) * (D / 16) + i;
                                *reinterpret_cast<uint4*>(sV + sv * kKt + (chunk >> 3) * (BK * 128) + sw128_chunk_off(r & (BK - 1), chunk & 7)) =
                                    make_uint4(0u, 0u, 0u, 0u);
                            }
                        fence_async_smem();
                    }
                }
                tc_fence_before();
                mbar_arrive(&p_full[st]);
            }
            m = read_item(n);
            const bool row_valid = g < G && e < m.ne;
            const int tok = m.tok0 + e;
            // the next item's numbers arrive under this item's epilogue
            const BfItem next = take_item(++n, ok);
            row = load_row(next);
            // ---- epilogue
            if (m.nblk > 0) {
                ok = ok && mbar_wait(&pv_done[(c - 1) & 1], ((c - 1) >> 1) & 1, status, limit);
                tc_fence_after();
            }
            ok = bar_all(1, 128, ok);
            const bool write = row_valid && ok;
            const int64_t head_row = (int64_t)tok * p.Hq + m.h * G + g;
            // (a sum of 0: nothing was seen.  NaN, from NaN or infinity in what was seen, goes on into o and lse)
            const bool none = l_run == 0.f;
            const float inv_l = none ? 0.f : 1.f / l_run;
            if (write) {
                if constexpr (kSplit) launch.ml[head_row * launch.P + m.z] = none ? make_float2(-INFINITY, 0.f) : make_float2(m_ref, l_run);
                else p.lse[(int64_t)(m.h * G + g) * p.N + tok] = none ? -INFINITY : m_ref + log2f(l_run);
            }
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t a[32];
                if (m.nblk > 0) {
                    tmem_ld32(tbase + lane_off + cO + c0, a);
                    tmem_ld_wait();
                    if (c0 + 32 == D) {
                        tc_fence_before();
                        mbar_arrive(o_free);            // the accumulator may take the next item
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) a[i] = 0u;
                }
                // every thread stores its own row, whole sectors of 32 bytes
                if constexpr (kSplit) {
                    if (write && !none)
#pragma unroll
                        for (int i = 0; i < 32; i += 8) st_global32(launch.o_part + (head_row * launch.P + m.z) * D + c0 + i, &a[i]);
                } else {
                    uint32_t x[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = ElemTraits<ET>::pack2(__uint_as_float(a[2 * i]) * inv_l, __uint_as_float(a[2 * i + 1]) * inv_l);
                    ET* dst = reinterpret_cast<ET*>(p.o) + head_row * D + c0;
                    if (write) {
                        st_global32(dst, &x[0]);
                        st_global32(dst + 16, &x[8]);
                    }
                }
            }
            m = next;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tbase, kCols);
    if (beside) follow_late();
    if (tid == 0 && *status != kStatusOk) stamp_status(p.status, *status);
}

template <int D, int MOD, typename ET>
static cudaError_t launch_bf(const BiasedFwdLaunch& l, int max_tiles, cudaStream_t stream) {
    constexpr int smem = kTileRows * D * 2 + (2 + kBfV) * kBiasedBK * D * 2 + 512;
    auto kern = biased_fwd<D, MOD, ET>;
    const cudaError_t e = allow_smem((const void*)kern, smem);
    if (e != cudaSuccess) return e;
    // (shared rows: beside the kernel before it, which is the one of the own rows, biased_decode.cu)
    return launch_dependent(kern, dim3((unsigned)max_tiles * (unsigned)l.p.Hk, (MOD & kModSplit) ? (unsigned)l.nchunk : 1u), kBfThreads, smem, stream, 1, l);
}

template <int D, typename ET>
static cudaError_t launch_which(int mod, const BiasedFwdLaunch& l, int max_tiles, cudaStream_t stream) {
    switch (mod) {
#define FSA_CASE(M) case M: return launch_bf<D, M, ET>(l, max_tiles, stream);
        FSA_CASE(0) FSA_CASE(kModCap) FSA_CASE(kModBias) FSA_CASE(kModCap | kModBias)
        FSA_CASE(kModSplit) FSA_CASE(kModSplit | kModCap) FSA_CASE(kModSplit | kModBias) FSA_CASE(kModSplit | kModCap | kModBias)
#undef FSA_CASE
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_biased_fwd(int D, int dtype, int which, bool split, const BiasedFwdLaunch& l, int max_tiles, cudaStream_t stream) {
    const int mod = which | (split ? kModSplit : 0);
    if (D == 128) return dtype == kBF16 ? launch_which<128, __nv_bfloat16>(mod, l, max_tiles, stream) : launch_which<128, __half>(mod, l, max_tiles, stream);
    return dtype == kBF16 ? launch_which<64, __nv_bfloat16>(mod, l, max_tiles, stream) : launch_which<64, __half>(mod, l, max_tiles, stream);
}

}  // namespace fsa
