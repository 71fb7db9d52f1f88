// dK and dV of attention with changed scores (score.cuh), key-tile-major, for sm_100a: the plan and the products of range_bwd_dkdv.cu (which sums the
// parts of the K/V tiles that were cut, too).  An item is a tile of 128 K/V rows of one sequence x one KV head x a stretch of tokens, walked in
// tiles of <= 128 rows (query head of the GQA group, token); a TMEM lane is a K/V row:
//   S^T = K Q^T, dP^T = V dO^T, P = exp2(s - lse), dS = P (dP - delta) ds/dx, dV += P^T dO, dK += scale dS^T Q
// with the scale in the epilogue, as in biased_bwd_dq.cu.
// One CTA per SM, 640 threads:
//   warp 0       TMA producer: K and V of an item, and Q, dO, Q, dO, ... through a ring of five tiles
//   warp 1       issues S(i) and dV(i)            warp 2    issues dP(i) and dK(i)
//   warp 3       lse, delta and visible rows of every row of a tile, two stages
//   warps 4..19  one K/V row per thread and a quarter of the tile's rows: P and dS; epilogue: dV the first two groups, dK the others, half the
//                columns each.
// A tile's products read 256 KB of shared memory and its loads write 64 KB, 2560 cycles (D = 128); sixteen row warps instead of eight, because with
// eight the capped scores took 4050 cycles and a distance bias 3860.  2 x 8192 tokens, 8 / 4 heads of 128, capped: 529 us (1039 TFLOP/s of the four
// products), the tensor cores' queue 72 % busy, issue 53 %.
#include "../../include/fsa_sm100.h"

#include "biased.cuh"
#include "range_bwd.cuh"

namespace fsa {

int make_tile_map_3d_box(CUtensorMap* map, const void* base, int dtype, int64_t d0, int64_t d1, int64_t d2, int64_t stride1,
                         int64_t stride2, int box1, int box2);
int device_sm_count(int* out);

constexpr int kBkThreads = 640;
constexpr int kBkUnits = 5;             // Q / dO tiles in the ring

struct BiasedKvParams {
    RangeKvPlan plan;
    int Hq, G;
    float scale, scale_log2;
    const float* lse;       // [Hq, N] log2 units
    const float* delta;     // [Hq, N]
    float4* slabs;
    void *dk, *dv;          // [Nk, Hk, D] contiguous
    int* status;
    ScoreMod mod;
};

// (Plan, limits and delta are from the kernel before dQ, which every dQ CTA has waited for before it let this kernel start; this one waits at its end
// only.  They are read through L2: the non-coherent path need not see what was written while a kernel before ran.)
// One work item: K/V rows [key0, key0 + nkeys) of head h, n row tiles of TPT tokens from tok0 on, tokens up to tok_last.
struct BkItem {
    int h, key0, nkeys, tok0, tok_last, n, slab;
};
__device__ __forceinline__ BkItem bk_item(const RangeKvPlan& p, int w) {
    BkItem m;
    const int4 it = __ldcg(p.items + w / p.Hk);
    const int4 t = __ldcg(p.tiles + it.x);
    m.h = w % p.Hk;
    m.key0 = t.x; m.nkeys = t.y;
    m.tok0 = t.z + it.y * p.TPT;
    m.tok_last = min(t.w, m.tok0 + it.z * p.TPT - 1);
    m.n = it.z;
    m.slab = it.w;
    return m;
}

template <int D, int MOD, typename ET>
__global__ void __launch_bounds__(kBkThreads, 1) biased_bwd_dkdv(const BiasedKvParams p, const __grid_constant__ CUtensorMap qmap,
                                                                const __grid_constant__ CUtensorMap domap, const __grid_constant__ CUtensorMap kmap,
                                                                const __grid_constant__ CUtensorMap vmap) {
    constexpr int KH = D / 64, kTile = kTileRows * D * 2;
    constexpr int kSlab = kTileRows * 128;           // 64 columns of a tile
    constexpr int cS = 0, cP = 128, cDV = 256, cDK = 384;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sK = smem;
    uint8_t* sV = sK + kTile;
    uint8_t* sU = sV + kTile;                        // [kBkUnits] Q, dO, Q, dO, ...
    float* sC = reinterpret_cast<float*>(sU + kBkUnits * kTile);          // [2][128] what a score gets besides: -lse and the bias at the item's first key
    float* sDel = sC + 2 * 128;                                           // [2][128] delta
    uint8_t* sVis = reinterpret_cast<uint8_t*>(sDel + 2 * 128);           // [2][2][128] first visible row; last one | 128
    uint64_t* bars = reinterpret_cast<uint64_t*>(sVis + 4 * 128);
    uint64_t* k_full = bars;            // K of an item has landed
    uint64_t* k_empty = bars + 1;       // ... has been read by the item's last S product
    uint64_t* v_full = bars + 2;
    uint64_t* v_empty = bars + 3;
    uint64_t* u_full = bars + 4;                     // [units]
    uint64_t* u_empty = u_full + kBkUnits;           // [units] the two products that read a Q or dO tile are done
    uint64_t* st_full = u_empty + kBkUnits;          // [2]
    uint64_t* st_empty = st_full + 2;                // [2]
    uint64_t* s_full = st_empty + 2;    // [2 halves] S(i) is done
    uint64_t* p_full = s_full + 2;      // [2] P(i) is in its place
    uint64_t* dp_full = s_full + 4;     // [2]
    uint64_t* ds_full = s_full + 6;     // [2]
    uint64_t* dv_done = s_full + 8;     // the item's last dV product is done
    uint64_t* dk_done = s_full + 9;
    uint64_t* dv_free = s_full + 10;    // the accumulator has been read
    uint64_t* dk_free = s_full + 11;
    uint64_t* p_read = s_full + 12;     // [2 halves] dV(i) has read P
    uint64_t* ds_read = s_full + 14;    // [2] dK(i) has read dS
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(s_full + 16);
    uint64_t* it_full = s_full + 18;    // [2] the next item is known
    uint64_t* it_empty = s_full + 20;   // [2] ... has been taken by the 19 other warps
    int* s_it = reinterpret_cast<int*>(s_full + 22);                      // [2] its place in the list, -1: there are no more
    int* s_masked = reinterpret_cast<int*>(s_full + 16) + 2;              // [2] some row of the tile does not see all K/V rows; 2: or sees none

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int* status = p.status;
    if (tid == 0) {
        mbar_init(k_full, 1); mbar_init(k_empty, 1); mbar_init(v_full, 1); mbar_init(v_empty, 1);
        for (int i = 0; i < kBkUnits; ++i) { mbar_init(&u_full[i], 1); mbar_init(&u_empty[i], 2); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&st_full[i], 32); mbar_init(&st_empty[i], 512);
            mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 256); mbar_init(&dp_full[i], 1); mbar_init(&ds_full[i], 256);
            mbar_init(&p_read[i], 1); mbar_init(&ds_read[i], 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(&it_full[i], 1); mbar_init(&it_empty[i], kBkThreads / 32 - 1); }
        mbar_init(dv_done, 1); mbar_init(dk_done, 1); mbar_init(dv_free, 256); mbar_init(dk_free, 256);
        mbar_init_fence();
    }
    // rows past G * TPT of a Q or dO tile are never loaded, but they are multiplied (by P = dS = 0)
    for (int i = p.G * p.plan.TPT * 8 + tid; i < kTileRows * 8; i += kBkThreads)
        for (int u = 0; u < KH * kBkUnits; ++u) reinterpret_cast<uint4*>(sU + u * kSlab)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_async_smem();
    if (warp == 0) tmem_alloc(&tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tmem_slot;
    const int nitems = __ldcg(p.plan.counts) * p.plan.Hk;
    const int TPT = p.plan.TPT;
    // Item n of this CTA: every warp but the producer's takes each of them once, in order; below 0 ends the list.
    auto take_item = [&](int n, bool& ok) {
        ok = ok && mbar_wait(&it_full[n & 1], (n >> 1) & 1, status);
        const int w = s_it[n & 1];
        ok = warp_ok(ok);
        if (lane == 0) mbar_arrive(&it_empty[n & 1]);
        return ok ? w : -1;
    };

    if (warp < 4) {
        reg_dec<64>();
        if (warp == 0) {
            // -------------------------------------------------------------- TMA producer
            if (lane == 0) {
                bool ok = true;
                int u = 0, qi = 0;             // Q / dO tiles and non-empty items so far
                const uint32_t unit_bytes = (uint32_t)(KH * 128 * TPT * p.G);
                for (int n = 0;; ++n) {
                    // the next item that nobody has: CTAs that start late, where a dQ CTA was at work, take fewer (every CTA its share of the list
                    // beforehand: 641 us instead of 628 for a pass over 2 x 4096 tokens of documents; longest first: 655, their Q and dO meet less in L2)
                    const int w = atomicAdd(p.plan.counts + 2, 1);
                    ok = ok && mbar_wait(&it_empty[n & 1], ((n >> 1) & 1) ^ 1, status);
                    if (!ok) break;
                    s_it[n & 1] = w < nitems ? w : -1;
                    mbar_arrive(&it_full[n & 1]);
                    if (w >= nitems) break;
                    const BkItem m = bk_item(p.plan, w);
                    if (m.n == 0) continue;
                    auto load_unit = [&](const CUtensorMap* map, int tok) {
                        const int st = u % kBkUnits;
                        ok = ok && mbar_wait(&u_empty[st], ((u / kBkUnits) & 1) ^ 1, status);
                        if (!ok) return;
                        mbar_expect_tx(&u_full[st], unit_bytes);
#pragma unroll
                        for (int b = 0; b < KH; ++b) tma_load_3d(smem_u32(sU + st * kTile + b * kSlab), map, b * 64, tok, m.h * p.G, &u_full[st]);
                        ++u;
                    };
                    auto load_kv = [&](const CUtensorMap* map, uint8_t* dst, uint64_t* full, uint64_t* empty) {
                        ok = ok && mbar_wait(empty, (qi & 1) ^ 1, status);
                        if (!ok) return;
                        mbar_expect_tx(full, (uint32_t)kTile);
#pragma unroll
                        for (int b = 0; b < KH; ++b)
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                tma_load_2d(smem_u32(dst + b * kSlab + r * (kSlab / 2)), map, m.h * D + b * 64, m.key0 + r * 64, full);
                    };
                    load_kv(&kmap, sK, k_full, k_empty);
                    load_unit(&qmap, m.tok0);
                    load_kv(&vmap, sV, v_full, v_empty);
                    load_unit(&domap, m.tok0);
                    for (int i = 1; i < m.n && ok; ++i) {
                        load_unit(&qmap, m.tok0 + i * TPT);
                        load_unit(&domap, m.tok0 + i * TPT);
                    }
                    ++qi;
                }
            }
        } else if (warp < 3) {
            // -------------------------------------------------------------- MMA issuers: warp 1 S and dV, warp 2 dP and dK
            const bool first = warp == 1;
            const bool leader = elect_one();
            constexpr uint32_t idesc_s = umma_idesc(ElemTraits<ET>::kIsBF16, 128, 64, false, false);
            constexpr uint32_t idesc_acc = umma_idesc(ElemTraits<ET>::kIsBF16, 128, D, false, true);     // P^T / dS^T (TMEM) x dO / Q (MN-major)
            constexpr uint32_t hi_1024 = umma_desc_hi(1024);
            const uint32_t a_lo = umma_desc_lo(smem_u32(first ? sK : sV), 16);
            const uint32_t b_lo = umma_desc_lo(smem_u32(sU), 16);
            const uint32_t b_mn_lo = umma_desc_lo(smem_u32(sU), kSlab);
            const uint32_t c_s = tbase + (first ? cS : cP), c_acc = tbase + (first ? cDV : cDK);
            uint64_t *kv_full = first ? k_full : v_full, *kv_empty = first ? k_empty : v_empty;
            uint64_t *out_full = first ? s_full : dp_full, *in_full = first ? p_full : ds_full, *in_read = first ? p_read : ds_read;
            uint64_t *acc_done = first ? dv_done : dk_done, *acc_free = first ? dv_free : dk_free;
            bool ok = true;
            int c = 0, qi = 0;
            // S^T (dP^T) of half a row tile t into its place, when the product that reads P^T (dS^T) of the tile before from there is done
            // (products of two shapes may run in another order than they were issued)
            auto issue_s = [&](int t, int half, bool last) {
                const int u = 2 * t + (first ? 0 : 1), st = u % kBkUnits;
                if (half == 0) ok = ok && mbar_wait(&u_full[st], (u / kBkUnits) & 1, status);
                if (t > 0) ok = ok && mbar_wait(&in_read[half], (t - 1) & 1, status);
                ok = warp_ok(ok);
                if (!ok) return;
                tc_fence_after();
                if (leader) {
                    const uint32_t bu = b_lo + (uint32_t)(st * (kTile >> 4) + half * (8192 >> 4));
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t off = (ks >> 2) * (kSlab >> 4) + (ks & 3) * 2;
                        umma_ss(c_s + half * 64, umma_desc_pack(a_lo + off, hi_1024), umma_desc_pack(bu + off, hi_1024), idesc_s, ks > 0);
                    }
                    umma_commit(&out_full[half]);
                    if (half) umma_commit(&u_empty[st]);
                    if (half && last) umma_commit(kv_empty);
                }
                __syncwarp();
            };
            for (int n = 0, w; (w = take_item(n, ok)) >= 0; ++n) {
                const BkItem m = bk_item(p.plan, w);
                if (m.n == 0) continue;
                ok = ok && mbar_wait(kv_full, qi & 1, status);
                issue_s(c, 0, m.n == 1);
                issue_s(c, 1, m.n == 1);
                for (int i = 0; i < m.n && ok; ++i, ++c) {
                    const int u = 2 * c + (first ? 1 : 0), st = u % kBkUnits;       // dV takes dO, dK takes Q
                    ok = ok && mbar_wait(&u_full[st], (u / kBkUnits) & 1, status);
                    if (i == 0 && qi > 0) ok = ok && mbar_wait(acc_free, (qi - 1) & 1, status);
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        ok = ok && mbar_wait(&in_full[half], c & 1, status);
                        ok = warp_ok(ok);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
                            const uint32_t bu = b_mn_lo + (uint32_t)(st * (kTile >> 4) + half * (8192 >> 4));
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks)      // (two groups of row threads, 32 columns apart)
                                umma_ts(c_acc, c_s + half * 64 + (ks >> 1) * 32 + (ks & 1) * 8, umma_desc_pack(bu + ks * (2048 >> 4), hi_1024), idesc_acc,
                                        (i > 0 || half > 0 || ks > 0) ? 1u : 0u);
                            umma_commit(&in_read[half]);
                            if (half) umma_commit(&u_empty[st]);
                            if (half && i + 1 == m.n) umma_commit(acc_done);
                        }
                        __syncwarp();
                        if (i + 1 < m.n) issue_s(c + 1, half, i + 2 == m.n);
                    }
                }
                ++qi;
            }
        } else {
            // -------------------------------------------------------------- per-row numbers of the tiles
            bool ok = true;
            int c = 0;
            int g[4], e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { g[j] = (lane + 32 * j) / TPT; e[j] = lane + 32 * j - g[j] * TPT; }
            for (int n = 0, w; (w = take_item(n, ok)) >= 0 && warp_stays(ok); ++n) {
                const BkItem m = bk_item(p.plan, w);
                float slope[4] = {0.f, 0.f, 0.f, 0.f};
                int far = 0;            // from the item's first key to its first token's place
                if ((MOD & kModBias) && m.n > 0 && !p.mod.ahead) {
                    far = __ldcg(p.mod.pos + m.tok0) - m.key0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) slope[j] = g[j] < p.G ? __ldcg(p.mod.slopes + m.h * p.G + g[j]) * kLog2e : 0.f;
                }
                for (int i = 0; i < m.n && warp_stays(ok); ++i, ++c) {
                    float cc[4], del[4];
                    int lo[4], hi[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int tok = m.tok0 + i * TPT + e[j];
                        cc[j] = -INFINITY; del[j] = 0.f; lo[j] = 0; hi[j] = -1;
                        if (g[j] < p.G && tok <= m.tok_last) {
                            const int64_t idx = (int64_t)(m.h * p.G + g[j]) * p.plan.N + tok;
                            cc[j] = -__ldcg(p.lse + idx);
                            del[j] = __ldcg(p.delta + idx);
                            lo[j] = __ldcg(p.plan.kv_lo + tok);
                            hi[j] = __ldcg(p.plan.kv_hi + tok);
                        }
                    }
                    bool masked = false, unseen = false;
                    int vis[4][2];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int l = max(lo[j] - m.key0, 0), u = min(hi[j] - m.key0, kTileRows - 1);
                        const bool sees = u >= l && fabsf(cc[j]) != INFINITY;      // a row that saw nothing in the forward sees nothing here (one that saw NaN has NaN)
                        masked |= sees && (l > 0 || u < m.nkeys - 1);
                        unseen |= !sees && g[j] < p.G;
                        if (!sees) { cc[j] = -INFINITY; del[j] = 0.f; }                        // exp2(s - inf) = 0
                        else if constexpr (MOD & kModBias) cc[j] = fmaf(-slope[j], (float)(far + i * TPT + e[j]), cc[j]);
                        vis[j][0] = sees ? l : kTileRows - 1;
                        vis[j][1] = sees ? u | 128 : 128;
                    }
                    masked = __any_sync(0xffffffffu, masked);
                    unseen = __any_sync(0xffffffffu, unseen);
                    const int b = c & 1;
                    ok = ok && mbar_wait(&st_empty[b], ((c >> 1) & 1) ^ 1, status);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        sC[b * 128 + lane + 32 * j] = cc[j];
                        sDel[b * 128 + lane + 32 * j] = del[j];
                        sVis[b * 256 + lane + 32 * j] = (uint8_t)vis[j][0];
                        sVis[b * 256 + 128 + lane + 32 * j] = (uint8_t)vis[j][1];
                    }
                    if (lane == 0) s_masked[b] = unseen ? 2 : masked;
                    mbar_arrive(&st_full[b]);
                }
            }
        }
    } else {
        reg_inc<104>();
        // ------------------------------------------------------------------ P, dS and the epilogue: one K/V row, a quarter of the tile's rows
        const int grp = (warp - 4) >> 2, half = grp >> 1;
        const int quarter = warp & 3;
        const int key = quarter * 32 + lane;
        const int r0 = grp * 32;            // first row of the tile (column of S^T)
        const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
        const uint32_t tS = tbase + lane_off + cS + r0, tP = tbase + lane_off + cP + r0;
        const NearTanh near(p.mod, 1.f);
        const float to_log2 = (MOD & kModCap) ? p.mod.cap_log2 : p.scale_log2;
        // lane j < 8 knows the head and the first token of the columns 4 j .. 4 j + 3 (tokens of one head follow one another in fours)
        const int q_col = r0 + 4 * (lane & 7), q_g = min(q_col / TPT, p.G - 1), q_e = q_col - q_col / TPT * TPT;
        bool ok = true;
        int c = 0, qi = 0;
        for (int n = 0, w; (w = take_item(n, ok)) >= 0 && warp_stays(ok); ++n) {
            const BkItem m = bk_item(p.plan, w);
            const float q_slope = (MOD & kModBias) ? __ldcg(p.mod.slopes + m.h * p.G + q_g) * kLog2e : 0.f;
            // with keys behind a token's place: place of this K/V row before (negative) or behind the item's first token
            const int key_rel = (MOD & kModBias) && p.mod.ahead && m.n > 0 ? m.key0 + key - __ldcg(p.mod.pos + m.tok0) : 0;
            for (int i = 0; i < m.n && warp_stays(ok); ++i, ++c) {
                const int b = c & 1;
                ok = ok && mbar_wait(&st_full[b], (c >> 1) & 1, status);
                ok = ok && mbar_wait(&s_full[half], c & 1, status);
                tc_fence_after();
                const int masked = s_masked[b];
                const float4* c4 = reinterpret_cast<const float4*>(sC + b * 128 + r0);
                const float4* del4 = reinterpret_cast<const float4*>(sDel + b * 128 + r0);
                uint32_t v[32], pk[16];
                tmem_ld32(tS, v);
                tmem_ld_wait();
                {
                    // v: P ds/dx, what dS takes; pk: P.  NEAR: products whose tanh is near's, else v has been changed already
                    const uint64_t s2 = f32x2(to_log2, to_log2), one2 = f32x2(1.f, 1.f);
                    auto pairs = [&](auto is_near) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float4 l = c4[j];
                            float cc[4] = {l.x, l.y, l.z, l.w};
                            if constexpr (MOD & kModBias) {
                                const float slope = __shfl_sync(0xffffffffu, q_slope, j);
                                if (p.mod.ahead) {
                                    const float d = (float)(key_rel - i * TPT - __shfl_sync(0xffffffffu, q_e, j));
#pragma unroll
                                    for (int q = 0; q < 4; ++q) cc[q] = fmaf(-slope, fabsf(d - (float)q), cc[q]);
                                } else {
                                    const float at = slope * (float)key;
#pragma unroll
                                    for (int q = 0; q < 4; ++q) cc[q] += at;
                                }
                            }
#pragma unroll
                            for (int q = 0; q < 4; q += 2) {
                                const int k = 4 * j + q;
                                uint64_t x = f32x2(__uint_as_float(v[k]), __uint_as_float(v[k + 1]));
                                if constexpr (decltype(is_near)::on) x = mul_f32x2(x, near.slope(x));
                                const float2 s = f32x2_get(fma_f32x2(x, s2, f32x2(cc[q], cc[q + 1])));
                                float2 pr = make_float2(ex2_approx(s.x), ex2_approx(s.y));
                                pk[k >> 1] = ElemTraits<ET>::pack2(pr.x, pr.y);
                                if constexpr (MOD & kModCap) {
                                    const float2 th = f32x2_get(x);
                                    pr = f32x2_get(mul_f32x2(f32x2(pr.x, pr.y), fma_f32x2(f32x2(-th.x, -th.y), x, one2)));
                                }
                                v[k] = __float_as_uint(pr.x);
                                v[k + 1] = __float_as_uint(pr.y);
                            }
                        }
                    };
                    constexpr bool kCap = (MOD & kModCap) != 0;
                    bool is_far = false;
                    if constexpr (kCap) {
                        float big[2] = {0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            big[0] = max3_abs(big[0], __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                            big[1] = max3_abs(big[1], __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
                        }
                        // (what decides: scores of tokens with keys that they see, as in the forward; a K/V row past the item's may be another sequence's or nobody's)
                        is_far = masked || __any_sync(0xffffffffu, key < m.nkeys && !(fmaxf(big[0], big[1]) <= p.mod.near_v));
                    }
                    if (!is_far) {
                        pairs(Flag<kCap>{});
                    } else {
                        if constexpr (kCap) cap_scores(v, p.mod.x_scale, p.mod.near_v);
                        pairs(Flag<false>{});
                    }
                }
                if (masked) {
                    // four rows at a time: bit 7 of a byte of (128 | key) - first says key >= first, of (128 | last) - key that key <= last
                    const uint32_t key4 = (uint32_t)key * 0x01010101u;
                    const uint4* first4 = reinterpret_cast<const uint4*>(sVis + b * 256 + r0);
                    const uint4* last4 = reinterpret_cast<const uint4*>(sVis + b * 256 + 128 + r0);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint4 f = first4[j], l = last4[j];
                        const uint32_t seen[4] = {((key4 | 0x80808080u) - f.x) & (l.x - key4), ((key4 | 0x80808080u) - f.y) & (l.y - key4),
                                                  ((key4 | 0x80808080u) - f.z) & (l.z - key4), ((key4 | 0x80808080u) - f.w) & (l.w - key4)};
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            if (!(seen[q >> 2] & (0x80u << ((q & 3) * 8)))) {
                                v[16 * j + q] = 0u;
                                pk[8 * j + (q >> 1)] &= (q & 1) ? 0x0000ffffu : 0xffff0000u;
                            }
                    }
                }
                if (masked == 2) {
                    // Q and dO rows that see nothing here are multiplied by dS = P = 0: zeros take the place of what may be NaN.  The half's S and dP
                    // are done; every thread of its two groups has a quarter of one of its 64 rows.
                    ok = ok && mbar_wait(&dp_full[half], c & 1, status);
                    tc_fence_after();
                    const int row = half * 64 + (key & 63), part = (grp & 1) * 2 + (key >> 6);
                    if (ok && sC[b * 128 + row] == -INFINITY)
#pragma unroll 1
                        for (int u = 2 * c; u < 2 * c + 2; ++u)
#pragma unroll
                            for (int n = 0; n < D / 32; ++n) {
                                const int chunk = part * (D / 32) + n;
                                *reinterpret_cast<uint4*>(sU + (u % kBkUnits) * kTile + (chunk >> 3) * kSlab + sw128_chunk_off(row, chunk & 7)) = make_uint4(0u, 0u, 0u, 0u);
                            }
                    fence_async_smem();
                }
                tmem_st16(tS, pk);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&p_full[half]);
                ok = ok && mbar_wait(&dp_full[half], c & 1, status);
                tc_fence_after();
                {
                    uint32_t d[32];
                    tmem_ld32(tP, d);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 dl = del4[j];
                        const int k = 4 * j;
                        const float2 x = f32x2_get(mul_f32x2(f32x2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])),
                                                             add_f32x2(f32x2(__uint_as_float(d[k]), __uint_as_float(d[k + 1])), f32x2(-dl.x, -dl.y))));
                        const float2 y = f32x2_get(mul_f32x2(f32x2(__uint_as_float(v[k + 2]), __uint_as_float(v[k + 3])),
                                                             add_f32x2(f32x2(__uint_as_float(d[k + 2]), __uint_as_float(d[k + 3])), f32x2(-dl.z, -dl.w))));
                        pk[2 * j] = ElemTraits<ET>::pack2(x.x, x.y);
                        pk[2 * j + 1] = ElemTraits<ET>::pack2(y.x, y.y);
                    }
                    if (masked) {           // (dP may be NaN where nothing is seen)
#pragma unroll
                        for (int j = 0; j < 16; ++j) pk[j] &= (v[2 * j] ? 0x0000ffffu : 0u) | (v[2 * j + 1] ? 0xffff0000u : 0u);
                    }
                    tmem_st16(tP, pk);
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&ds_full[half]);
                mbar_arrive(&st_empty[b]);
            }
            // ---- epilogue of the item: groups 0 and 1 dV, 2 and 3 dK, half the columns each
            if (m.n > 0) {
                ok = ok && mbar_wait(half ? dk_done : dv_done, qi & 1, status);
                tc_fence_after();
            }
            if (!warp_stays(ok)) break;
            const bool write = key < m.nkeys;
            constexpr int kOwn = D / 2;
            const int col0 = (grp & 1) * kOwn;
            ET* dst = reinterpret_cast<ET*>(half ? p.dk : p.dv) + ((int64_t)(m.key0 + key) * p.plan.Hk + m.h) * D + col0;
            float4* slab = p.slabs + ((int64_t)m.slab * p.plan.Hk + m.h) * (2 * (D / 4) * 128) + half * ((D / 4) * 128) + (col0 / 4) * 128 + key;
#pragma unroll 1
            for (int c0 = 0; c0 < kOwn; c0 += 32) {
                uint32_t a[32];
                if (m.n > 0) {
                    tmem_ld32(tbase + lane_off + (half ? cDK : cDV) + col0 + c0, a);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) a[j] = 0u;
                }
                if (c0 + 32 == kOwn && m.n > 0) {
                    tc_fence_before();
                    mbar_arrive(half ? dk_free : dv_free);            // the accumulator may take the next item
                }
                if (half) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) * p.scale);
                }
                if (write && m.slab >= 0) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        slab[(c0 / 4 + j) * 128] = make_float4(__uint_as_float(a[4 * j]), __uint_as_float(a[4 * j + 1]),
                                                               __uint_as_float(a[4 * j + 2]), __uint_as_float(a[4 * j + 3]));
                } else if (write) {
                    uint32_t x[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = ElemTraits<ET>::pack2(__uint_as_float(a[2 * j]), __uint_as_float(a[2 * j + 1]));
                    st_global32(dst + c0, &x[0]);
                    st_global32(dst + c0 + 16, &x[8]);
                }
            }
            if (m.n > 0) ++qi;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tbase, 512);
    follow_late();      // it runs beside the dQ kernel, of which it needs nothing
}

template <int D, int MOD, typename ET>
static cudaError_t launch_bk(const BiasedKvParams& p, const CUtensorMap* maps, unsigned grid, cudaStream_t stream) {
    constexpr int smem = (2 + kBkUnits) * (kTileRows * D * 2) + 2 * 128 * (4 + 4 + 2) + 512;
    auto kern = biased_bwd_dkdv<D, MOD, ET>;
    const cudaError_t e = allow_smem((const void*)kern, smem);
    if (e != cudaSuccess) return e;
    return launch_dependent(kern, dim3(grid), kBkThreads, smem, stream, 1, p, maps[0], maps[1], maps[2], maps[3]);
}

template <int D, typename ET>
static cudaError_t launch_bk_which(int which, const BiasedKvParams& p, const CUtensorMap* maps, unsigned grid, cudaStream_t stream) {
    switch (which) {
#define FSA_CASE(M) case M: return launch_bk<D, M, ET>(p, maps, grid, stream);
        FSA_CASE(0) FSA_CASE(kModCap) FSA_CASE(kModBias) FSA_CASE(kModCap | kModBias)
#undef FSA_CASE
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_biased_bwd_dkdv(int dtype, const RangeKvPlan& plan, const SelBwdArgs& a, const SelShape& s, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                   int* status, const ScoreMod& mod, int which, cudaStream_t stream) {
    CUtensorMap maps[4];        // Q, dO, K, V
    if (make_tile_map_3d_box(&maps[0], a.q, dtype, s.D, s.N, s.Hq, a.q_sn, a.q_sh, s.TPT, s.G)) return cudaErrorInvalidValue;
    if (make_tile_map_3d_box(&maps[1], a.d_o, dtype, s.D, s.N, s.Hq, a.do_sn, a.do_sh, s.TPT, s.G)) return cudaErrorInvalidValue;
    maps[2] = kmap; maps[3] = vmap;
    BiasedKvParams p;
    p.plan = plan;
    p.Hq = s.Hq; p.G = s.G;
    p.scale = a.sm_scale; p.scale_log2 = a.sm_scale * kLog2e;
    p.lse = a.lse; p.delta = a.delta; p.slabs = (float4*)a.slabs; p.dk = a.dk; p.dv = a.dv; p.status = status;
    p.mod = mod;
    int sms = 0;
    if (device_sm_count(&sms) != 0 || sms <= 0) return cudaErrorInvalidValue;
    const int64_t max_items = (range_kv_max_tiles(s) + range_kv_max_cut(s)) * s.Hk;
    const unsigned grid = (unsigned)(max_items < sms ? max_items : sms);
    const bool bf16 = dtype == kBF16;
    if (s.D == 128) return bf16 ? launch_bk_which<128, __nv_bfloat16>(which, p, maps, grid, stream) : launch_bk_which<128, __half>(which, p, maps, grid, stream);
    return bf16 ? launch_bk_which<64, __nv_bfloat16>(which, p, maps, grid, stream) : launch_bk_which<64, __half>(which, p, maps, grid, stream);
}

}  // namespace fsa
