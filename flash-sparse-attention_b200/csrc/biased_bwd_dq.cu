// dQ of attention with changed scores (score.cuh), query-tile-major, for sm_100a: the tiling of the forward (biased_fwd.cu), per K/V tile of 64 rows
//   S = Q K^T, dP = dO V^T, P = exp2(s - lse), dS = P (dP - delta) ds/dx, dQ (+)= dS K
// with ds/dx = 1 - tanh^2 under a cap; dQ accumulated in TMEM over the tiles, multiplied with the scale and written once.  (dS without the scale: 1 / 11 of it
// at head size 128, it would lose three bits more of small gradients to fp16's subnormal numbers: dq over 4096 keys, dO of size 1e-3, was off by 9.1e-7 and is by less than 1.8e-7.
// The other end of fp16: P (dP - delta) up to 65504.)  One CTA per SM, 640 threads:
//   warp 0       TMA producer: Q and dO tiles of every item, (K, V) tiles through a ring of kBqStages
//   warp 1       one elected thread issues S and dP (two TMEM buffers)      warp 2    ... dQ
//   warp 3       finds the items, up to four ahead, longest first
//   warps 4..19  four groups of 128 row threads: two on the tiles of each TMEM buffer, 32 of the 64 key columns each.  dS goes over dP (D = 64: into
//                columns of its own, so that S and dP of the buffer's next tile need not wait for the dQ product); the next item's Q and dO to
//                TMEM; epilogue, a quarter of the dQ columns each.
// The left operand of every product comes from TMEM (in shared memory it would be read at every tile, 48 KB a product of 256 cycles).  The products
// take 768 cycles a tile at D = 128, exp2 512.  What bounds the tile is the row threads' chain of loads, arithmetic and stores: with eight row warps in
// step on one tile (range_dense.cu) it takes 1540 cycles, capped 1990; sixteen on two tiles hide one another's latencies.  2 x 8192 tokens, 8 / 4 heads of
// 128, capped: 392 us (1051 TFLOP/s of the three products); the tensor cores 51 % busy, issue 52 % before the items went forth and back.
#include "../../include/fsa_sm100.h"
#include <climits>

#include "biased.cuh"

namespace fsa {

int make_tile_map_3d_box(CUtensorMap* map, const void* base, int dtype, int64_t d0, int64_t d1, int64_t d2, int64_t stride1,
                         int64_t stride2, int box1, int box2);
int device_sm_count(int* out);

struct BiasedDqParams {
    const int32_t *cu_q, *cu_k, *kv_lo, *kv_hi;
    int64_t N, Nk;
    int B, Hq, Hk, G, TPT;
    float scale, scale_log2;
    const float* lse;       // [Hq, N] log2 units
    const float* delta;     // [Hq, N] sum_d o dO
    void* dq;               // [N, Hq, D] contiguous
    int nchunk;             // the K/V tiles of an item are cut into so many chunks, whose dQ go to part, unless there is only one
    float* part;            // [N, Hq, nchunk, D]
    int* status;
    ScoreMod mod;
};

constexpr int kBqThreads = 640;
constexpr int kBqRows = 512;
constexpr int kBqStages = 5;
constexpr int kBqItems = 4;         // items known ahead
// The item warp is ahead, so that its wait for a free entry lasts as long as an item: this many cycles more for each tile of the longest item so far
// (a tile takes some 1200).
constexpr uint32_t kBqTileClocks = 4096;
static_assert(kMaxTokens / kBiasedBK * kBqTileClocks + FSA_WAIT_CLOCKS < (int64_t)1 << 32, "the counter comes round");

struct BqItem {
    int seq, tok0, ne, row_lo, nblk, h, row_hi, z;     // z: chunk
};

// Work item w of the list.  (Chunks of equal size, kBiasedLeast tiles at least; the last ones may be empty.)  All 32 lanes call it and get the same answer.
__device__ __forceinline__ BqItem bq_item(const BiasedDqParams& p, int w, int lane) {
    BqItem m;
    m.z = w % p.nchunk;
    w /= p.nchunk;
    m.h = w % p.Hk;
    m.row_lo = 0; m.nblk = 0; m.row_hi = -1;
    find_ranked_tile(p.cu_q, p.cu_k, p.B, p.TPT, w / p.Hk, lane, m.seq, m.tok0, m.ne);
    if (m.seq < 0) return m;
    int lo = INT_MAX, hi = -1;
    for (int e = lane; e < m.ne; e += 32) {
        const int l = __ldcg(p.kv_lo + m.tok0 + e), u = __ldcg(p.kv_hi + m.tok0 + e);
        if (u >= l) { lo = min(lo, l); hi = max(hi, u); }
    }
    m.row_lo = max(__reduce_min_sync(0xffffffffu, lo), 0);
    m.row_hi = min(__reduce_max_sync(0xffffffffu, hi), (int)p.Nk - 1);
    m.nblk = m.row_hi >= m.row_lo ? (m.row_hi - m.row_lo) / kBiasedBK + 1 : 0;
    if (p.nchunk > 1) {
        const int size = max(kBiasedLeast, (m.nblk + p.nchunk - 1) / p.nchunk), first = min(m.z * size, m.nblk);
        m.nblk = min(size, m.nblk - first);
        m.row_lo += first * kBiasedBK;
        m.row_hi = min(m.row_hi, m.row_lo + m.nblk * kBiasedBK - 1);
    }
    return m;
}

template <int D, int MOD, typename ET>
__global__ void __launch_bounds__(kBqThreads, 1) biased_bwd_dq(const BiasedDqParams p, const __grid_constant__ CUtensorMap qmap,
                                                              const __grid_constant__ CUtensorMap domap, const __grid_constant__ CUtensorMap kmap,
                                                              const __grid_constant__ CUtensorMap vmap) {
    constexpr int BK = kBiasedBK, KH = D / 64;
    constexpr int kQ = kTileRows * D * 2;            // Q tile, same for dO
    constexpr int kKt = BK * D * 2;
    constexpr bool kOwnDs = D == 64;                 // dS has columns of its own
    // S(b) at 128 b, dP(b) at 128 b + 64; Q, dO and dS two values a column
    constexpr int cDQ = 256, cQ = cDQ + D, cDO = cQ + D / 2, cDS = cDO + D / 2;
    constexpr uint32_t kCols = 512;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;
    uint8_t* sDO = sQ + kQ;
    uint8_t* sKV = sDO + kQ;                         // stage: K then V
    uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + kBqStages * 2 * kKt);
    uint64_t* qd_full = bars;           // Q and dO tiles of an item have landed
    uint64_t* qd_empty = bars + 1;      // ... have been read by the row threads
    uint64_t* kv_full = bars + 2;                        // [stages]
    uint64_t* kv_empty = kv_full + kBqStages;            // [stages] the dQ product of the tile is done
    uint64_t* sdp_full = kv_empty + kBqStages;           // [2]
    uint64_t* sdp_free = sdp_full + 2;                   // [2] the buffer's 256 row threads have read S and dP
    uint64_t* ds_full = sdp_free + 2;                    // [2] ... have written dS
    uint64_t* ds_empty = ds_full + 2;                    // [2] the dQ product has read dS
    uint64_t* dq_free = ds_empty + 2;                    // the row threads have read an item's dQ accumulator
    uint64_t* qt_full = dq_free + 1;                     // ... have written an item's Q and dO to TMEM
    uint64_t* it_full = qt_full + 1;                     // [items]
    uint64_t* it_empty = it_full + kBqItems;             // [items] the other warps have read the entry
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(it_empty + kBqItems);
    int4* s_item = reinterpret_cast<int4*>(bars + 34);   // [items][2]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int* status = p.status;
    follow_late();
    if (tid == 0) {
        mbar_init(qd_full, 1); mbar_init(qd_empty, kBqRows);
        for (int i = 0; i < kBqStages; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sdp_full[i], 1); mbar_init(&sdp_free[i], 256);
            mbar_init(&ds_full[i], 256); mbar_init(&ds_empty[i], 1);
        }
        for (int i = 0; i < kBqItems; ++i) { mbar_init(&it_full[i], 1); mbar_init(&it_empty[i], kBqThreads / 32 - 1); }
        mbar_init(dq_free, kBqRows); mbar_init(qt_full, kBqRows);
        mbar_init_fence();
    }
    // rows past G * TPT of the Q and dO tiles are never loaded, but have a part in their warp's choice of a tanh (biased_fwd.cu)
    for (int i = p.G * p.TPT * 8 + tid; i < kTileRows * 8; i += kBqThreads)
        for (int b = 0; b < KH; ++b) reinterpret_cast<uint4*>(sQ + b * (kTileRows * 128))[i] = reinterpret_cast<uint4*>(sDO + b * (kTileRows * 128))[i] = make_uint4(0u, 0u, 0u, 0u);
    if (warp == 0) tmem_alloc(&tmem_slot, kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tmem_slot;
    let_next_start();
    const int nitems = count_ranked_tiles(p.cu_q, p.B, p.TPT, lane) * p.Hk * p.nchunk;
    // Entry n of this CTA's items: every warp but the one that fills the ring takes each of them once, in order.
    auto take_item = [&](int n, bool& ok) {
        ok = ok && mbar_wait(&it_full[n % kBqItems], (n / kBqItems) & 1, status);
        const int4 x = s_item[(n % kBqItems) * 2], y = s_item[(n % kBqItems) * 2 + 1];
        ok = warp_ok(ok);
        if (lane == 0) mbar_arrive(&it_empty[n % kBqItems]);
        BqItem m;
        m.seq = x.x; m.tok0 = x.y; m.ne = x.z; m.row_lo = x.w; m.nblk = y.x; m.h = y.y; m.row_hi = y.z; m.z = y.w;
        if (!ok) m.ne = m.nblk = 0;
        return m;
    };

    if (warp < 4) {
        reg_dec<64>();
        if (warp == 3) {
            // -------------------------------------------------------------- items
            bool ok = true;
            int n = 0, longest = 0;
            for (int w; (w = forth_and_back(n)) < nitems && ok; ++n) {
                const BqItem m = bq_item(p, w, lane);
                ok = ok && mbar_wait(&it_empty[n % kBqItems], ((n / kBqItems) & 1) ^ 1, status, FSA_WAIT_CLOCKS + longest * kBqTileClocks);
                ok = warp_ok(ok);
                longest = max(longest, m.nblk);
                if (ok && lane == 0) {
                    s_item[(n % kBqItems) * 2] = make_int4(m.seq, m.tok0, m.ne, m.row_lo);
                    s_item[(n % kBqItems) * 2 + 1] = make_int4(m.nblk, m.h, m.row_hi, m.z);
                    mbar_arrive(&it_full[n % kBqItems]);
                }
            }
        } else if (warp == 0) {
            // -------------------------------------------------------------- TMA producer
            bool ok = true;
            int kvc = 0, qi = 0, n = 0;    // K/V tiles and non-empty items so far
            for (; forth_and_back(n) < nitems && ok; ++n) {
                const BqItem m = take_item(n, ok);
                if (m.nblk == 0) continue;
                if (lane == 0) {
                    ok = ok && mbar_wait(qd_empty, (qi & 1) ^ 1, status);
                    if (ok) {
                        mbar_expect_tx(qd_full, (uint32_t)(2 * KH * 128 * p.TPT * p.G));
#pragma unroll
                        for (int b = 0; b < KH; ++b) {
                            tma_load_3d(smem_u32(sQ + b * (kTileRows * 128)), &qmap, b * 64, m.tok0, m.h * p.G, qd_full);
                            tma_load_3d(smem_u32(sDO + b * (kTileRows * 128)), &domap, b * 64, m.tok0, m.h * p.G, qd_full);
                        }
                    }
                }
                ++qi;
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                for (int j = 0; j < m.nblk && ok; ++j, ++kvc) {
                    if (lane == 0) {
                        const int st = kvc % kBqStages;
                        ok = ok && mbar_wait(&kv_empty[st], ((kvc / kBqStages) & 1) ^ 1, status);
                        if (ok) {
                            mbar_expect_tx(&kv_full[st], (uint32_t)(2 * kKt));
                            uint8_t* dK = sKV + st * 2 * kKt;
                            uint8_t* dV = dK + kKt;
#pragma unroll
                            for (int b = 0; b < KH; ++b) {
                                tma_load_2d(smem_u32(dK + b * (BK * 128)), &kmap, m.h * D + b * 64, m.row_lo + j * BK, &kv_full[st]);
                                tma_load_2d(smem_u32(dV + b * (BK * 128)), &vmap, m.h * D + b * 64, m.row_lo + j * BK, &kv_full[st]);
                            }
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                }
            }
        } else {
            // -------------------------------------------------------------- MMA issuers: warp 1 S and dP, warp 2 dQ
            // The K/V tiles of all items form one sequence c = 0, 1, ...; S / dP run ahead of dQ as far as their two TMEM buffers and the K/V ring
            // allow, also across the boundary between two items.
            const bool leader = elect_one();
            constexpr uint32_t idesc_s = umma_idesc(ElemTraits<ET>::kIsBF16, 128, BK, false, false);
            constexpr uint32_t idesc_dq = umma_idesc(ElemTraits<ET>::kIsBF16, 128, D, false, true);     // dS (K-major) x K (MN-major)
            constexpr uint32_t hi_1024 = umma_desc_hi(1024);
            constexpr int kSlabB = (BK * 128) >> 4;
            const uint32_t kv_lo_ = umma_desc_lo(smem_u32(sKV), 16);
            const uint32_t k_mn_lo = umma_desc_lo(smem_u32(sKV), BK * 128);
            bool ok = true;
            int c = 0, qi = 0, n = 0;
            for (; forth_and_back(n) < nitems && ok; ++n) {
                const BqItem m = take_item(n, ok);
                if (m.nblk == 0) continue;
                if (warp == 1) {
                    ok = ok && mbar_wait(qt_full, qi & 1, status);
                    ok = warp_ok(ok);
                    for (int j = 0; j < m.nblk && ok; ++j, ++c) {
                        const int b = c & 1, st = c % kBqStages;
                        const uint32_t k_lo = kv_lo_ + (uint32_t)(st * ((2 * kKt) >> 4));
                        const uint32_t v_lo = k_lo + (uint32_t)(kKt >> 4);
                        ok = ok && mbar_wait(&kv_full[st], (c / kBqStages) & 1, status);
                        ok = ok && mbar_wait(&sdp_free[b], ((c >> 1) & 1) ^ 1, status);     // S / dP of tile c - 2 have been read
                        ok = warp_ok(ok);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
#pragma unroll
                            for (int ks = 0; ks < D / 16; ++ks)
                                umma_ts(tbase + b * 128, tbase + cQ + ks * 8, umma_desc_pack(k_lo + (ks >> 2) * kSlabB + (ks & 3) * 2, hi_1024), idesc_s, ks > 0);
                        }
                        __syncwarp();
                        if constexpr (!kOwnDs) {
                            ok = ok && mbar_wait(&ds_empty[b], ((c >> 1) & 1) ^ 1, status);     // the dQ product of tile c - 2 has read dS
                            ok = warp_ok(ok);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        if (leader) {
#pragma unroll
                            for (int ks = 0; ks < D / 16; ++ks)
                                umma_ts(tbase + b * 128 + BK, tbase + cDO + ks * 8, umma_desc_pack(v_lo + (ks >> 2) * kSlabB + (ks & 3) * 2, hi_1024), idesc_s, ks > 0);
                            umma_commit(&sdp_full[b]);
                        }
                        __syncwarp();
                    }
                } else {
                    for (int j = 0; j < m.nblk && ok; ++j, ++c) {
                        const int b = c & 1, st = c % kBqStages;
                        ok = ok && mbar_wait(&ds_full[b], (c >> 1) & 1, status);      // (implies S / dP of the tile are done with K and V)
                        if (j == 0 && qi > 0) ok = ok && mbar_wait(dq_free, (qi - 1) & 1, status);     // the previous item's dQ has been read
                        ok = warp_ok(ok);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
                            const uint32_t b_lo = k_mn_lo + (uint32_t)(st * ((2 * kKt) >> 4));
#pragma unroll
                            for (int ks = 0; ks < BK / 16; ++ks)      // (over dP, the two column halves are 32 columns apart)
                                umma_ts(tbase + cDQ, kOwnDs ? tbase + cDS + b * 32 + ks * 8 : tbase + b * 128 + BK + (ks >> 1) * 32 + (ks & 1) * 8,
                                        umma_desc_pack(b_lo + ks * (2048 >> 4), hi_1024), idesc_dq, (j > 0 || ks > 0) ? 1u : 0u);
                            umma_commit(&kv_empty[st]);
                            umma_commit(&ds_empty[b]);
                        }
                        __syncwarp();
                    }
                }
                ++qi;
            }
        }
    } else {
        reg_inc<104>();
        // ------------------------------------------------------------------ dS and the epilogue: one row; half the columns of every other tile
        const int grp = (warp - 4) >> 2, tb = grp >> 1, sb = grp & 1;
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
        const int g = r / p.TPT, e = r - g * p.TPT;
        constexpr int HC = BK / 2;
        const int cb = sb * HC;
        const uint32_t tS = tbase + lane_off + tb * 128 + cb, tP = tS + BK, tDS = kOwnDs ? tbase + lane_off + cDS + tb * 32 + sb * 16 : tP;
        const float to_log2 = (MOD & kModCap) ? p.mod.cap_log2 : p.scale_log2;
        bool ok = true;
        int c = 0, qi = 0;
        // A row of an item's Q (groups 0 and 1, half each) or dO (2 and 3) to TMEM.  Not before the last S / dP products of the item before are done.
        auto take_row = [&]() {
            ok = ok && mbar_wait(qd_full, qi & 1, status);
            ++qi;
            const uint8_t* src = tb ? sDO : sQ;
            const uint32_t dst = tbase + lane_off + (tb ? cDO : cQ) + sb * (D / 4);
#pragma unroll
            for (int i0 = 0; i0 < D / 16; i0 += 4) {        // 16-byte chunks of this half row
                uint32_t x[16];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int chunk = sb * (D / 16) + i0 + i;
                    *reinterpret_cast<uint4*>(&x[i * 4]) = *reinterpret_cast<const uint4*>(src + (chunk >> 3) * (kTileRows * 128) + sw128_chunk_off(r, chunk & 7));
                }
                tmem_st16(dst + i0 * 4, x);
            }
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(qd_empty);
            mbar_arrive(qt_full);
        };
        // This row's numbers, loaded an item ahead.
        struct Row { int lo, hi; float lse, delta, slope; int pos; };
        auto load_numbers = [&](const BqItem& m) {
            Row x = {0, INT_MAX, 0.f, 0.f, 0.f, INT_MAX};       // (a place without a token sees everything: its row goes nowhere)
            if (g < p.G && e < m.ne) {
                x.lo = __ldcg(p.kv_lo + m.tok0 + e);
                x.hi = __ldcg(p.kv_hi + m.tok0 + e);
                const int64_t idx = (int64_t)(m.h * p.G + g) * p.N + m.tok0 + e;
                x.lse = __ldcg(p.lse + idx);
                x.delta = __ldcg(p.delta + idx);        // (the kernel before wrote it)
                if constexpr (MOD & kModBias) {
                    x.slope = __ldcg(p.mod.slopes + m.h * p.G + g) * kLog2e;
                    x.pos = __ldcg(p.mod.pos + m.tok0 + e);
                }
            }
            return x;
        };
        const NearTanh near(p.mod, 1.f);
        BqItem m;
        m.nblk = m.ne = 0;
        int n = 0;
        if (forth_and_back(0) < nitems) {
            m = take_item(n, ok);
            if (m.nblk > 0) take_row();
        }
        Row row = load_numbers(m);
        while (forth_and_back(n) < nitems && warp_stays(ok)) {
            const bool row_valid = g < p.G && e < m.ne;
            const int tok = m.tok0 + e;
            const int lo_r = row.lo;
            const float lse_r = row.lse, delta_r = row.delta, slope_r = row.slope;
            const int pos_r = row.pos;
            int hi_r = min(row.hi, (int)p.Nk - 1);              // rows past the end of K/V do not exist
            if (lse_r == -INFINITY) hi_r = lo_r - 1;            // a row that saw nothing in the forward sees nothing here (one that saw NaN gets NaN)
            BqItem next;
            next.nblk = next.ne = 0;
            if (forth_and_back(++n) < nitems) next = take_item(n, ok);
            row = load_numbers(next);
            const int c0 = c;
            c += m.nblk;
            for (int j = (c0 & 1) ^ tb; j < m.nblk; j += 2) {        // (left by all lanes at the vote below)
                const int k = (c0 + j) >> 1;            // tiles of this buffer so far
                const int R0 = m.row_lo + j * BK;
                const int c_lo = max(0, lo_r - R0), c_hi = min(BK, hi_r - R0 + 1);
                ok = ok && mbar_wait(&sdp_full[tb], k & 1, status);
                tc_fence_after();
                uint32_t dd[HC / 2];
                const bool all_visible = __all_sync(0xffffffffu, ok && c_lo <= cb && c_hi >= cb + HC);
                if (!all_visible && !warp_stays(ok)) break;
                {
                    uint32_t sv[32], dv[32];
                    tmem_ld32(tS, sv);
                    tmem_ld32(tP, dv);
                    tmem_ld_wait();
                    tc_fence_before();
                    mbar_arrive(&sdp_free[tb]);       // both are in registers: the buffer may take its next tile
                    // bit i: column cb + i is seen
                    const int v_lo = min(max(c_lo - cb, 0), HC), v_hi = min(max(c_hi - cb, 0), HC);
                    const uint32_t vis = v_hi > v_lo ? (0xffffffffu >> (HC - v_hi + v_lo)) << v_lo : 0u;
                    const uint64_t s2 = f32x2(to_log2, to_log2), d2 = f32x2(-delta_r, -delta_r), one2 = f32x2(1.f, 1.f);
                    const float rel = (float)(pos_r - R0 - cb);
                    const float base = (MOD & kModBias) ? fmaf(-slope_r, rel, -lse_r) : -lse_r;
                    // dS of the columns, two at a time.  NEAR: products whose tanh is near's, else sv has been changed already; BOTH: keys behind the token's
                    // place are seen too; ALL: no mask
                    auto pairs = [&](auto is_near, auto both, auto all) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float b0 = base, b1 = base;
                            if constexpr (MOD & kModBias) {
                                b0 = decltype(both)::on ? fmaf(-slope_r, fabsf(rel - (float)i), -lse_r) : fmaf(slope_r, (float)i, base);
                                b1 = decltype(both)::on ? fmaf(-slope_r, fabsf(rel - (float)(i + 1)), -lse_r) : fmaf(slope_r, (float)(i + 1), base);
                            }
                            uint64_t x = f32x2(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
                            if constexpr (decltype(is_near)::on) x = mul_f32x2(x, near.slope(x));
                            const float2 s = f32x2_get(fma_f32x2(x, s2, f32x2(b0, b1)));
                            uint64_t gr = add_f32x2(f32x2(__uint_as_float(dv[i]), __uint_as_float(dv[i + 1])), d2);
                            // d tanh(x) = 1 - tanh(x)^2
                            if constexpr (MOD & kModCap) {
                                const float2 th = f32x2_get(x);
                                gr = mul_f32x2(gr, fma_f32x2(f32x2(-th.x, -th.y), x, one2));
                            }
                            const float2 ds = f32x2_get(mul_f32x2(f32x2(ex2_approx(s.x), ex2_approx(s.y)), gr));
                            dd[i >> 1] = decltype(all)::on ? ElemTraits<ET>::pack2(ds.x, ds.y)
                                                           : ElemTraits<ET>::pack2(vis >> i & 1u ? ds.x : 0.f, vis >> (i + 1) & 1u ? ds.y : 0.f);
                        }
                    };
                    const bool both = (MOD & kModBias) && p.mod.ahead && __any_sync(0xffffffffu, hi_r > pos_r);
                    constexpr bool kCap = (MOD & kModCap) != 0;
                    // (what decides: scores of tokens with keys that they see, as in the forward)
                    bool is_far = both || (kCap && !all_visible);
                    if constexpr (kCap) {       // (before, not afterwards as in the forward: the products would have to be kept beside the dS)
                        float big[2] = {0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            big[0] = max3_abs(big[0], __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
                            big[1] = max3_abs(big[1], __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
                        }
                        is_far |= __any_sync(0xffffffffu, row_valid && !(fmaxf(big[0], big[1]) <= p.mod.near_v));
                    }
                    if (!is_far) {
                        if (kCap || all_visible) pairs(Flag<kCap>{}, Flag<false>{}, Flag<true>{});
                        else pairs(Flag<false>{}, Flag<false>{}, Flag<false>{});
                    } else {
                        if constexpr (kCap) cap_scores(sv, p.mod.x_scale, p.mod.near_v);
                        if (both) pairs(Flag<false>{}, Flag<true>{}, Flag<false>{});
                        else pairs(Flag<false>{}, Flag<false>{}, Flag<false>{});
                    }
                }
                if (j + 1 == m.nblk && next.nblk > 0) take_row();      // the next item's S / dP run under this item's end
                if constexpr (kOwnDs) {
                    ok = ok && mbar_wait(&ds_empty[tb], (k & 1) ^ 1, status);       // the dQ product of the buffer's tile before has read its dS
                    tc_fence_after();
                }
                tmem_st16(tDS, dd);
                tmem_st_wait();
                if (p.mod.key_ids || j + 1 == m.nblk) {
                    // K rows that no row of the item sees are multiplied by dS = 0: zeros take the place of what may be NaN (the tile's S is
                    // done).  Every thread of the buffer's two groups has a quarter of one of the 64 rows.
                    const int kr = R0 + (r & (BK - 1)), part = sb * 2 + (r >> 6);
                    const bool unseen = kr > m.row_hi || (p.mod.key_ids && __ldcg(p.mod.key_ids + kr) < 0);
                    if (__any_sync(0xffffffffu, unseen)) {
                        if (unseen && ok)
#pragma unroll
                            for (int i = 0; i < D / 32; ++i) {
                                const int chunk = part * (D / 32) + i;
                                *reinterpret_cast<uint4*>(sKV + ((c0 + j) % kBqStages) * 2 * kKt + (chunk >> 3) * (BK * 128) + sw128_chunk_off(r & (BK - 1), chunk & 7)) =
                                    make_uint4(0u, 0u, 0u, 0u);
                            }
                        fence_async_smem();
                    }
                }
                tc_fence_before();
                mbar_arrive(&ds_full[tb]);
            }
            const int last = (c - 1) & 1, klast = (c - 1) >> 1;
            if (next.nblk > 0 && (m.nblk == 0 || last != tb)) {
                // (the item's last tile is the other buffer's)
                if (m.nblk > 0) ok = ok && mbar_wait(&sdp_full[last], klast & 1, status);
                tc_fence_after();
                take_row();
            }
            // ---- epilogue of the item: this group's quarter of the dQ columns
            if (m.nblk > 0) {
                // The item's last dQ product is done.  A group whose buffer it was not in waits for its own last one first: a barrier tells the phase asked
                // for only from those after the one before, which the product before the last comes after.
                if (last != tb && m.nblk > 1) ok = ok && mbar_wait(&ds_empty[tb], ((c - 2) >> 1) & 1, status);
                ok = ok && mbar_wait(&ds_empty[last], klast & 1, status);
                tc_fence_after();
            }
            if (!warp_stays(ok)) break;
            constexpr int kOwn = D / 4;
            const int64_t drow = (int64_t)tok * p.Hq + (m.h * p.G + g);
            uint32_t a[kOwn];
            if (m.nblk > 0) {
                if constexpr (D == 128) tmem_ld32(tbase + lane_off + cDQ + grp * kOwn, a);
                else tmem_ld16(tbase + lane_off + cDQ + grp * kOwn, a);
                tmem_ld_wait();
                tc_fence_before();
                mbar_arrive(dq_free);            // the accumulator may take the next item
#pragma unroll
                for (int i = 0; i < kOwn; ++i) a[i] = __float_as_uint(__uint_as_float(a[i]) * p.scale);
            } else {
#pragma unroll
                for (int i = 0; i < kOwn; ++i) a[i] = 0u;
            }
            if (p.nchunk > 1) {
                float* dst = p.part + (drow * p.nchunk + m.z) * D + grp * kOwn;
                if (row_valid)
#pragma unroll
                    for (int i = 0; i < kOwn; i += 8) st_global32(dst + i, &a[i]);
            } else if (row_valid) {
                ET* dst = reinterpret_cast<ET*>(p.dq) + drow * D + grp * kOwn;
#pragma unroll
                for (int i = 0; i < kOwn; i += 16) {
                    uint32_t x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = ElemTraits<ET>::pack2(__uint_as_float(a[i + 2 * j]), __uint_as_float(a[i + 2 * j + 1]));
                    st_global32(dst + i, x);
                }
            }
            m = next;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tbase, kCols);
}

// dQ of the tokens of the sequences: the sum of the chunks in order, rounded once.  A thread has 8 columns of a row; bound by memory.
constexpr int kDsThreads = 256;
template <int D, typename ET>
__global__ void __launch_bounds__(kDsThreads) biased_dq_sum(const float* part, const int32_t* cu_q, int B, int64_t rows, int Hq, int nchunk, ET* __restrict__ dq) {
    constexpr int L = D / 8;
    const int64_t i = (int64_t)blockIdx.x * kDsThreads + threadIdx.x, row = i / L;
    follow();
    if (row >= rows) return;
    const int tok = (int)((uint32_t)row / (uint32_t)Hq);
    if (tok < __ldcg(cu_q) || tok >= __ldcg(cu_q + B)) return;      // (the row is cleared)
    const float* src = part + row * nchunk * D + i % L * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int z = 0; z < nchunk; ++z) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(src + z * D)), y = __ldcg(reinterpret_cast<const float4*>(src + z * D + 4));
        acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w;
        acc[4] += y.x; acc[5] += y.y; acc[6] += y.z; acc[7] += y.w;
    }
    *reinterpret_cast<uint4*>(dq + i * 8) = make_uint4(ElemTraits<ET>::pack2(acc[0], acc[1]), ElemTraits<ET>::pack2(acc[2], acc[3]),
                                                       ElemTraits<ET>::pack2(acc[4], acc[5]), ElemTraits<ET>::pack2(acc[6], acc[7]));
}

template <int D, typename ET>
static cudaError_t launch_sum(const float* part, const SelBwdArgs& a, const SelShape& s, int nchunk, cudaStream_t stream) {
    const int64_t rows = s.N * s.Hq, blocks = (rows * (D / 8) + kDsThreads - 1) / kDsThreads;
    return launch_dependent(biased_dq_sum<D, ET>, dim3((unsigned)blocks), kDsThreads, 0, stream, 1, part, a.cu, s.B, rows, s.Hq, nchunk, (ET*)a.dq);
}

cudaError_t launch_biased_dq_sum(int dtype, const float* part, const SelBwdArgs& a, const SelShape& s, int nchunk, cudaStream_t stream) {
    const bool bf16 = dtype == kBF16;
    if (s.D == 128) return bf16 ? launch_sum<128, __nv_bfloat16>(part, a, s, nchunk, stream) : launch_sum<128, __half>(part, a, s, nchunk, stream);
    return bf16 ? launch_sum<64, __nv_bfloat16>(part, a, s, nchunk, stream) : launch_sum<64, __half>(part, a, s, nchunk, stream);
}

template <int D, int MOD, typename ET>
static cudaError_t launch_bq(const BiasedDqParams& p, const CUtensorMap* maps, unsigned grid, cudaStream_t stream) {
    constexpr int smem = 2 * kTileRows * D * 2 + kBqStages * 2 * kBiasedBK * D * 2 + 272 + kBqItems * 32;
    auto kern = biased_bwd_dq<D, MOD, ET>;
    const cudaError_t e = allow_smem((const void*)kern, smem);
    if (e != cudaSuccess) return e;
    return launch_dependent(kern, dim3(grid), kBqThreads, smem, stream, 1, p, maps[0], maps[1], maps[2], maps[3]);
}

template <int D, typename ET>
static cudaError_t launch_bq_which(int which, const BiasedDqParams& p, const CUtensorMap* maps, unsigned grid, cudaStream_t stream) {
    switch (which) {
#define FSA_CASE(M) case M: return launch_bq<D, M, ET>(p, maps, grid, stream);
        FSA_CASE(0) FSA_CASE(kModCap) FSA_CASE(kModBias) FSA_CASE(kModCap | kModBias)
#undef FSA_CASE
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_biased_bwd_dq(int dtype, const SelBwdArgs& a, const SelShape& s, const CUtensorMap& kmap, const CUtensorMap& vmap, int* status,
                                 const ScoreMod& mod, int which, int nchunk, float* part, cudaStream_t stream) {
    CUtensorMap maps[4];        // Q, dO, K, V
    if (make_tile_map_3d_box(&maps[0], a.q, dtype, s.D, s.N, s.Hq, a.q_sn, a.q_sh, s.TPT, s.G)) return cudaErrorInvalidValue;
    if (make_tile_map_3d_box(&maps[1], a.d_o, dtype, s.D, s.N, s.Hq, a.do_sn, a.do_sh, s.TPT, s.G)) return cudaErrorInvalidValue;
    maps[2] = kmap; maps[3] = vmap;
    BiasedDqParams p;
    p.cu_q = a.cu; p.cu_k = a.bd.cu_k; p.kv_lo = a.bd.kv_lo; p.kv_hi = a.bd.kv_hi;
    p.N = s.N; p.Nk = s.Nk; p.B = s.B; p.Hq = s.Hq; p.Hk = s.Hk; p.G = s.G; p.TPT = s.TPT;
    p.scale = a.sm_scale; p.scale_log2 = a.sm_scale * kLog2e;
    p.lse = a.lse; p.delta = a.delta; p.dq = a.dq; p.status = status;
    p.mod = mod;
    p.nchunk = nchunk; p.part = part;
    const int64_t max_items = ((s.N + s.TPT - 1) / s.TPT + s.B) * (int64_t)s.Hk * nchunk;
    if (max_items >= (int64_t)1 << 30) return cudaErrorInvalidValue;
    int sms = 0;
    if (device_sm_count(&sms) != 0 || sms <= 0) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)(max_items < sms ? max_items : sms);
    const bool bf16 = dtype == kBF16;
    if (s.D == 128) return bf16 ? launch_bq_which<128, __nv_bfloat16>(which, p, maps, grid, stream) : launch_bq_which<128, __half>(which, p, maps, grid, stream);
    return bf16 ? launch_bq_which<64, __nv_bfloat16>(which, p, maps, grid, stream) : launch_bq_which<64, __half>(which, p, maps, grid, stream);
}

}  // namespace fsa
