// One new token per sequence with changed scores (score.cuh) over a K/V cache: split over the rows, merged by log-sum-exp; and the same for
// batches whose sequences continue rows that they share.
//
// A sequence's own rows: every K/V row of a sequence and kv head is read once, by a CTA that takes a chunk of them; 4 d flops a row and query
// head, far below what HBM allows, so the kernel is bound by the bytes in flight: TMA through a ring of 64-row stages, warp-level MMA
// (m16n8k16) whose 16 rows are the query heads of the group.
// Shared rows: the queries of all sequences that share them make MMA tiles of 128 rows (biased_fwd.cu with kModSplit), so the rows are read once for
// 128 queries of a kv head instead of once for every sequence.
// Both write partial results (unnormalised o, maximum, sum) side by side; the last kernel merges them.
#include "../../include/fsa_sm100.h"

#include "biased.cuh"

namespace fsa {

int make_tile_map(CUtensorMap* map, const void* base, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int box_rows);
int make_tile_map_3d_box(CUtensorMap* map, const void* base, int dtype, int64_t d0, int64_t d1, int64_t d2, int64_t stride1,
                         int64_t stride2, int box1, int box2);
int device_sm_count(int* out);
int cuda_failed(cudaError_t e);
cudaError_t biased_status_word(int** out);      // biased_attn.cu

constexpr int kBdKT = 64;           // rows of a stage
constexpr int kBdStages = 3;
constexpr int kBdThreads = 160;     // four consumer warps and the producer

struct BiasedDecodeParams {
    const void* q;              // [B, Hq, D]
    const int32_t* seq_len;     // [B]
    const int32_t* row0;        // [B] first cache row
    int B, Hq, Hk, G, parts;    // parts: CTAs that take up to 16 query heads of a group each
    int window;                 // -1: none
    int chunk, nchunk;          // rows of a chunk; the last one takes what is left
    int P, p0;                  // partials of a row, the first of this kernel's
    float scale_log2;
    ScoreMod mod;
    float* o_part;              // [B, Hq, P, D]
    float2* ml;                 // [B, Hq, P]
    int* status;
};

template <int D, bool HI, int MOD, typename ET>
__global__ void __launch_bounds__(kBdThreads) biased_decode_partial(const BiasedDecodeParams p, const __grid_constant__ CUtensorMap kmap,
                                                                    const __grid_constant__ CUtensorMap vmap) {
    extern __shared__ __align__(1024) unsigned char dsm_raw[];
    constexpr int HALF_BYTES = kBdKT * 128;              // one 64-column half of a stage's rows
    constexpr int KV_BYTES = (D / 64) * HALF_BYTES;
    constexpr int STAGE_BYTES = 2 * KV_BYTES;
    constexpr int NK = D / 16;                           // k-steps of Q K^T
    constexpr int NO = D / 8;                            // 8-column output tiles of P V
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dsm_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t limit = stamped_wait_limit(p.status);
    uint64_t* full = reinterpret_cast<uint64_t*>(base + (size_t)kBdStages * STAGE_BYTES);
    uint64_t* empty = full + kBdStages;
    float* smm = reinterpret_cast<float*>(empty + kBdStages);    // [4][16]
    float* sll = smm + 64;
    float* so = reinterpret_cast<float*>(base);          // [4][heads][D], aliases the stages after the loop

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int gid = lane >> 2, tig = lane & 3;
    const int c = blockIdx.x % p.nchunk;
    const int part = (blockIdx.x / p.nchunk) % p.parts;
    const int h = (blockIdx.x / (p.nchunk * p.parts)) % p.Hk;
    const int b = blockIdx.x / (p.nchunk * p.parts * p.Hk);
    const int per = (p.G + p.parts - 1) / p.parts, g0 = part * per, NG = min(per, p.G - g0);     // query heads of this CTA
    const int64_t pbase = ((int64_t)b * p.Hq + h * p.G + g0) * p.P + p.p0 + c;
    if (tid == 0) {
        for (int s = 0; s < kBdStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 4); }
        mbar_init_fence();
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    follow();
    // rows [lo, lo + n) of the sequence, counted from its first one
    const int len = p.seq_len[b];
    const int from = p.window >= 0 ? max(0, len - 1 - p.window) : 0;
    const int lo = from + min((int64_t)c * p.chunk, (int64_t)max(0, len - from));
    const int n = max(c + 1 < p.nchunk ? min(p.chunk, len - lo) : len - lo, 0);
    if (n == 0) {
        if (tid < NG) p.ml[pbase + (int64_t)tid * p.P] = make_float2(-INFINITY, 0.f);
        return;
    }
    __syncthreads();
    const uint32_t sbase = smem_u32(base);
    float acc[NO][4];
    float m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.f, l1 = 0.f;      // (not -inf: as long as all scores of a row are that, every p is exp2(-inf) = 0)

    if (warp == 4) {
        if (elect_one()) {
            const int row = p.row0[b] + lo;
            for (int it = 0; it * kBdKT < n; ++it) {
                const int s = it % kBdStages;
                if (it >= kBdStages && !mbar_wait_stamped(&empty[s], ((it / kBdStages) - 1) & 1, p.status, limit)) break;
                mbar_expect_tx(&full[s], STAGE_BYTES);
                const uint32_t kb = sbase + s * STAGE_BYTES;
#pragma unroll
                for (int hf = 0; hf < D / 64; ++hf) {
                    tma_load_2d(kb + hf * HALF_BYTES, &kmap, h * D + hf * 64, row + it * kBdKT, &full[s]);
                    tma_load_2d(kb + KV_BYTES + hf * HALF_BYTES, &vmap, h * D + hf * 64, row + it * kBdKT, &full[s]);
                }
            }
        }
        __syncwarp();
    } else {
        uint32_t qf[NK][2], qh[NK][2];
        {
            const ET* q = (const ET*)p.q + ((int64_t)b * p.Hq + h * p.G + g0) * D;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                qf[kk][0] = gid < NG ? *reinterpret_cast<const uint32_t*>(q + gid * D + kk * 16 + tig * 2) : 0u;
                qf[kk][1] = gid < NG ? *reinterpret_cast<const uint32_t*>(q + gid * D + kk * 16 + 8 + tig * 2) : 0u;
                qh[kk][0] = (HI && gid + 8 < NG) ? *reinterpret_cast<const uint32_t*>(q + (gid + 8) * D + kk * 16 + tig * 2) : 0u;
                qh[kk][1] = (HI && gid + 8 < NG) ? *reinterpret_cast<const uint32_t*>(q + (gid + 8) * D + kk * 16 + 8 + tig * 2) : 0u;
            }
        }
        float slope[2] = {0.f, 0.f};
        if constexpr (MOD & kModBias) {
            slope[0] = gid < NG ? p.mod.slopes[h * p.G + g0 + gid] * kLog2e : 0.f;
            slope[1] = HI && gid + 8 < NG ? p.mod.slopes[h * p.G + g0 + gid + 8] * kLog2e : 0.f;
        }
        const float to_log2 = (MOD & kModCap) ? p.mod.cap_log2 : p.scale_log2;
        // score (log2 units) of a product, or of its tanh; dist: tokens between the key and the new token
        auto score = [&](float x, float sl, float dist) { return (MOD & kModBias) ? fmaf(-sl, dist, x * to_log2) : x * to_log2; };
#pragma unroll
        for (int i = 0; i < NO; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        const int lrow = lane & 7, lmat = lane >> 3;
        bool ok = true;
        for (int it = 0; it * kBdKT < n; ++it) {
            const int s = it % kBdStages;
            ok = mbar_wait_stamped(&full[s], (it / kBdStages) & 1, p.status, limit);
            if (!warp_stays(ok)) break;
            const int k0 = it * kBdKT + warp * 16;               // first key of this warp's tile
            if (k0 < n) {
                const uint32_t kb = sbase + s * STAGE_BYTES, vb = kb + KV_BYTES;
                float sc[2][4];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
                    const int row = warp * 16 + nt * 8 + lrow;
#pragma unroll
                    for (int c0 = 0; c0 < D / 8; c0 += 4) {
                        const int cg = c0 + lmat;
                        uint32_t r0, r1, r2, r3;
                        ldsm_x4(kb + (cg >> 3) * HALF_BYTES + row * 128 + (((cg & 7) ^ (row & 7)) << 4), r0, r1, r2, r3);
                        mma16816<ET>(sc[nt], qf[c0 / 2][0], qh[c0 / 2][0], qf[c0 / 2][1], qh[c0 / 2][1], r0, r1);
                        mma16816<ET>(sc[nt], qf[c0 / 2 + 1][0], qh[c0 / 2 + 1][0], qf[c0 / 2 + 1][1], qh[c0 / 2 + 1][1], r2, r3);
                    }
                }
                if constexpr (MOD & kModCap) {
                    uint32_t x[HI ? 8 : 4];
#pragma unroll
                    for (int i = 0; i < (HI ? 8 : 4); ++i) x[i] = __float_as_uint(HI ? sc[i >> 2][i & 3] : sc[i >> 1][i & 1]);
                    cap_scores(x, p.mod.x_scale, p.mod.near_v);
#pragma unroll
                    for (int i = 0; i < (HI ? 8 : 4); ++i) (HI ? sc[i >> 2][i & 3] : sc[i >> 1][i & 1]) = __uint_as_float(x[i]);
                }
                float tmax0 = -INFINITY, tmax1 = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = k0 + nt * 8 + tig * 2 + e;
                        const float dist = (float)(len - 1 - lo - key);
                        sc[nt][e] = key < n ? score(sc[nt][e], slope[0], dist) : -INFINITY;
                        tmax0 = fmaxf(tmax0, sc[nt][e]);
                        if (HI) {
                            sc[nt][2 + e] = key < n ? score(sc[nt][2 + e], slope[1], dist) : -INFINITY;
                            tmax1 = fmaxf(tmax1, sc[nt][2 + e]);
                        }
                    }
                tmax0 = fmaxf(tmax0, __shfl_xor_sync(0xffffffffu, tmax0, 1));
                tmax0 = fmaxf(tmax0, __shfl_xor_sync(0xffffffffu, tmax0, 2));
                if (HI) {
                    tmax1 = fmaxf(tmax1, __shfl_xor_sync(0xffffffffu, tmax1, 1));
                    tmax1 = fmaxf(tmax1, __shfl_xor_sync(0xffffffffu, tmax1, 2));
                }
                const float mn0 = fmaxf(m0, tmax0), mn1 = HI ? fmaxf(m1, tmax1) : m1;
                if (__any_sync(0xffffffffu, mn0 > m0 || (HI && mn1 > m1))) {
                    const float a0 = ex2_approx(m0 - mn0), a1 = HI ? ex2_approx(m1 - mn1) : 1.f;
                    l0 *= a0;
                    l1 *= a1;
#pragma unroll
                    for (int t = 0; t < NO; ++t) {
                        acc[t][0] *= a0; acc[t][1] *= a0;
                        if (HI) { acc[t][2] *= a1; acc[t][3] *= a1; }
                    }
                    m0 = mn0;
                    m1 = mn1;
                }
                uint32_t pa[4];
                {
                    const float e00 = ex2_approx(sc[0][0] - m0), e01 = ex2_approx(sc[0][1] - m0), e10 = ex2_approx(sc[1][0] - m0), e11 = ex2_approx(sc[1][1] - m0);
                    l0 += e00 + e01 + e10 + e11;
                    pa[0] = ElemTraits<ET>::pack2(e00, e01);
                    pa[2] = ElemTraits<ET>::pack2(e10, e11);
                    if (HI) {
                        const float f00 = ex2_approx(sc[0][2] - m1), f01 = ex2_approx(sc[0][3] - m1), f10 = ex2_approx(sc[1][2] - m1), f11 = ex2_approx(sc[1][3] - m1);
                        l1 += f00 + f01 + f10 + f11;
                        pa[1] = ElemTraits<ET>::pack2(f00, f01);
                        pa[3] = ElemTraits<ET>::pack2(f10, f11);
                    } else {
                        pa[1] = pa[3] = 0u;
                    }
                }
                if (k0 + 16 > n) {
                    // V rows behind the sequence are multiplied by p = 0, but may hold NaN: zeros take their place (each warp has its own 16 rows)
                    for (int i = lane; i < 16 * (D / 8); i += 32) {
                        const int row = warp * 16 + i / (D / 8), chunk = i % (D / 8);
                        if (it * kBdKT + row >= n)
                            *reinterpret_cast<uint4*>(base + s * STAGE_BYTES + KV_BYTES + (chunk >> 3) * HALF_BYTES + sw128_chunk_off(row, chunk & 7)) =
                                make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_async_smem();     // (before TMA writes there again)
                    __syncwarp();
                }
                {
                    const int row = warp * 16 + (lmat & 1) * 8 + lrow;
#pragma unroll
                    for (int c0 = 0; c0 < D / 8; c0 += 2) {
                        const int cg = c0 + (lmat >> 1);
                        uint32_t r0, r1, r2, r3;
                        ldsm_x4_trans(vb + (cg >> 3) * HALF_BYTES + row * 128 + (((cg & 7) ^ (row & 7)) << 4), r0, r1, r2, r3);
                        mma16816<ET>(acc[c0], pa[0], pa[1], pa[2], pa[3], r0, r1);
                        mma16816<ET>(acc[c0 + 1], pa[0], pa[1], pa[2], pa[3], r2, r3);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    }
    __syncthreads();                                     // every stage has been consumed: stage memory is free
    if (warp < 4) {
#pragma unroll
        for (int half = 0; half < (HI ? 2 : 1); ++half) {
            const int g = gid + half * 8;
            if (g < NG) {
                float* dst = so + ((size_t)warp * NG + g) * D;
#pragma unroll
                for (int t = 0; t < NO; ++t)
                    *reinterpret_cast<float2*>(dst + t * 8 + tig * 2) = make_float2(acc[t][half * 2], acc[t][half * 2 + 1]);
                if (tig == 0) {
                    smm[warp * 16 + g] = half ? m1 : m0;
                    sll[warp * 16 + g] = half ? l1 : l0;
                }
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < NG * D; i += kBdThreads) {
        const int g = i / D;
        const float M = fmaxf(fmaxf(smm[g], smm[16 + g]), fmaxf(smm[32 + g], smm[48 + g]));
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = smm[w * 16 + g];
            if (sll[w * 16 + g] != 0.f) o += ex2_approx(mw - M) * so[(size_t)w * NG * D + i];        // (0: a warp without keys)
        }
        p.o_part[(pbase + (int64_t)g * p.P) * D + (i - g * D)] = o;
    }
    if (tid < NG) {
        const int g = tid;
        const float M = fmaxf(fmaxf(smm[g], smm[16 + g]), fmaxf(smm[32 + g], smm[48 + g]));
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = smm[w * 16 + g];
            if (sll[w * 16 + g] != 0.f) L += ex2_approx(mw - M) * sll[w * 16 + g];
        }
        p.ml[pbase + (int64_t)g * p.P] = make_float2(M, L);
    }
}

// BiasedMerge; 0 and -inf for a row that saw nothing (partials whose sum is 0), NaN for one that saw NaN.  WARPS warps a row: what it takes is round trips to L2,
// so all maxima and sums, and the first AHEAD partials of every warp, are asked for at once (1 x 8191 tokens, 32 heads, 64 partials a row: 12 us with
// a round trip for every four partials of a warp).  Of few partials many rows: AHEAD 4, whose registers leave room for more warps (16544 rows of 2: 8 us less).
constexpr int kMgThreads = 128;
template <int D, int WARPS, int AHEAD, typename ET>
__global__ void __launch_bounds__(kMgThreads) biased_decode_merge(const BiasedMerge a) {
    constexpr int V = D / 32;           // columns of a lane
    __shared__ float s_m[4], s_l[4];
    __shared__ float4 s_acc[4][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w = warp % WARPS;
    const int64_t row = (int64_t)blockIdx.x * (4 / WARPS) + warp / WARPS;
    follow();
    if (row >= a.rows) return;            // (with WARPS = 4 there is no such CTA)
    const int P = a.P, b = (int)((uint32_t)row / (uint32_t)a.Hq);
    const int first = a.nshared > 0 && (b < __ldcg(a.cu) || b >= __ldcg(a.cu + a.groups)) ? a.nshared : 0;
    const float2* mlr = a.ml + row * P;
    const float* src = a.o_part + row * P * D + lane * V;
    auto load = [&](int i, float (&x)[4]) {
        x[2] = x[3] = 0.f;
        if constexpr (V == 4) *reinterpret_cast<float4*>(x) = __ldcg(reinterpret_cast<const float4*>(src + (int64_t)i * D));
        else *reinterpret_cast<float2*>(x) = __ldcg(reinterpret_cast<const float2*>(src + (int64_t)i * D));
    };
    float x[AHEAD][4];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
        if (first + w + WARPS * j < P) load(first + w + WARPS * j, x[j]);
    float M = -INFINITY, L = 0.f;
    for (int i = first + w * 32 + lane; i < P; i += 32 * WARPS) {
        const float2 v = __ldcg(mlr + i);
        if (v.y != 0.f) {
            const float m = fmaxf(M, v.x);
            L = L * ex2_approx(M - m) + v.y * ex2_approx(v.x - m);
            M = m;
        }
    }
    auto join = [&](float m2, float l2) {
        const float m = fmaxf(M, m2), use = m == -INFINITY ? 0.f : m;
        L = L * ex2_approx(M - use) + l2 * ex2_approx(m2 - use);
        M = m;
    };
#pragma unroll
    for (int d = 16; d; d >>= 1) join(__shfl_xor_sync(0xffffffffu, M, d), __shfl_xor_sync(0xffffffffu, L, d));
    if constexpr (WARPS > 1) {
        if (lane == 0) { s_m[warp] = M; s_l[warp] = L; }
        __syncthreads();
        M = -INFINITY; L = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) join(s_m[i], s_l[i]);
    }
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](int i, const float (&y)[4]) {
        const float2 v = __ldcg(mlr + i);
        if (v.y != 0.f) {               // (a partial without keys has no o)
            const float f = ex2_approx(v.x - M);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = fmaf(f, y[k], acc[k]);
        }
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
        if (first + w + WARPS * j < P) add(first + w + WARPS * j, x[j]);
    for (int i = first + w + WARPS * AHEAD; i < P; i += WARPS) {
        float y[4];
        load(i, y);
        add(i, y);
    }
    if constexpr (WARPS > 1) {
        s_acc[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int j = 1; j < WARPS; ++j) {
            const float4 y = s_acc[j][lane];
            acc[0] += y.x; acc[1] += y.y; acc[2] += y.z; acc[3] += y.w;
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    ET* dst = (ET*)a.o + row * D + lane * V;
    if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(ElemTraits<ET>::pack2(acc[0] * inv, acc[1] * inv), ElemTraits<ET>::pack2(acc[2] * inv, acc[3] * inv));
    else *reinterpret_cast<uint32_t*>(dst) = ElemTraits<ET>::pack2(acc[0] * inv, acc[1] * inv);
    if (lane == 0) a.lse[b * a.lse_sn + (row - (int64_t)b * a.Hq) * a.lse_sh] = L == 0.f ? -INFINITY : M + log2f(L);
}

template <int D, bool HI, int MOD, typename ET>
static cudaError_t launch_bd(const BiasedDecodeParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream) {
    constexpr int smem = kBdStages * 2 * (D / 64) * kBdKT * 128 + 1024 /* alignment */ + 1024 /* barriers, statistics */;
    auto kern = biased_decode_partial<D, HI, MOD, ET>;
    const cudaError_t e = allow_smem((const void*)kern, smem);
    if (e != cudaSuccess) return e;
    return launch_dependent(kern, dim3((unsigned)((int64_t)p.B * p.Hk * p.parts * p.nchunk)), kBdThreads, smem, stream, 1, p, kmap, vmap);
}

template <int D, typename ET>
static cudaError_t launch_bd_which(int which, const BiasedDecodeParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream) {
    const bool hi = (p.G + p.parts - 1) / p.parts > 8;
    switch (which) {
#define FSA_CASE(M) case M: return hi ? launch_bd<D, true, M, ET>(p, kmap, vmap, stream) : launch_bd<D, false, M, ET>(p, kmap, vmap, stream);
        FSA_CASE(0) FSA_CASE(1) FSA_CASE(2) FSA_CASE(3)
#undef FSA_CASE
        default: return cudaErrorInvalidValue;
    }
}

template <int D, typename ET>
static cudaError_t launch_merge(const BiasedMerge& m, cudaStream_t stream) {
    // a CTA per row while all of them still run at once
    if (m.rows <= 4 * sm_count()) return launch_dependent(biased_decode_merge<D, 4, 16, ET>, dim3((unsigned)m.rows), kMgThreads, 0, stream, 1, m);
    const dim3 grid((unsigned)((m.rows + 3) / 4));
    if (m.P <= 4) return launch_dependent(biased_decode_merge<D, 1, 4, ET>, grid, kMgThreads, 0, stream, 1, m);
    return launch_dependent(biased_decode_merge<D, 1, 16, ET>, grid, kMgThreads, 0, stream, 1, m);
}

cudaError_t launch_biased_merge(int D, int dtype, const BiasedMerge& m, cudaStream_t stream) {
    if (D == 128) return dtype == kBF16 ? launch_merge<128, __nv_bfloat16>(m, stream) : launch_merge<128, __half>(m, stream);
    return dtype == kBF16 ? launch_merge<64, __nv_bfloat16>(m, stream) : launch_merge<64, __half>(m, stream);
}

// How a decode call is cut: partials of the shared rows, of the own ones.  Own rows: as many chunks as run at once, two CTAs an SM, and chunks of up to
// 1024 rows where there is more to read than that.  Shared rows: as many items as run at once as well, of at least two tiles.
struct DecodeCut {
    int parts, own, nown, tiles, nshared, mtiles;       // own: rows of a chunk; tiles: 64-row tiles of a shared chunk; mtiles: tiles of 128 queries at most
    DecodeCut(int B, int Hk, int G, int TPT, int groups, int64_t max_len, int64_t max_shared, int window) {
        const int sms = sm_count();
        parts = (G + 15) / 16;
        int64_t rows = max_len < 1 ? 1 : max_len;
        if (window >= 0 && rows > (int64_t)window + 1) rows = (int64_t)window + 1;
        const int64_t heads = (int64_t)B * Hk * parts, each = heads > 0 ? 2 * sms / heads : 1;      // chunks of a sequence and kv head
        int64_t c = each > 0 ? (rows + each - 1) / each : 1024;
        // (more sequences and kv heads than run at once, of unlike lengths: about four turns)
        if (each == 0 && rows * heads < 8 * (int64_t)sms * 1024) c = (rows * heads + 8 * sms - 1) / (8 * sms);
        c = (c + kBdKT - 1) / kBdKT * kBdKT;
        c = c < kBdKT ? kBdKT : c > 1024 ? 1024 : c;
        own = (int)c;
        nown = (int)((rows + c - 1) / c);
        tiles = nshared = mtiles = 0;
        if (groups > 0) {
            // (a group's last tile has one sequence at least; a place in the grid that no tile takes would hold up one that does)
            mtiles = groups > kRankedSeqs ? B / TPT + groups : B > groups ? (B - groups) / TPT + groups : B > 0 ? B : 1;
            const int64_t blocks = max_shared < 1 ? 1 : (max_shared + kBiasedBK - 1) / kBiasedBK;
            int64_t n = 2 * sms / ((int64_t)mtiles * Hk);
            if (n < 1) n = 1;
            if (n > (blocks + 1) / 2) n = (blocks + 1) / 2;
            if (n > 256) n = 256;
            tiles = (int)((blocks + n - 1) / n);
            nshared = (int)((blocks + tiles - 1) / tiles);
        }
    }
    int partials() const { return nshared + nown; }
};

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace fsa

using namespace fsa;

extern "C" int fsa_biased_decode_bytes(int batch, int num_q_heads, int num_kv_heads, int head_dim, int num_groups, int64_t max_len, int64_t max_shared, int window,
                                       int64_t* bytes_out) {
    if (!bytes_out || batch < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || num_groups < 0 || max_len < 0 || max_shared < 0)
        return FSA_ERR_BAD_ARG;
    const int G = num_q_heads / num_kv_heads;
    if ((head_dim != 64 && head_dim != 128) || G > 32 || max_len >= ((int64_t)1 << 30) || max_shared >= kMaxTokens) return FSA_ERR_UNSUPPORTED;
    if (biased_places(batch, (kTileRows / G) & ~3, num_groups) * num_kv_heads >= kBiasedMaxPlaces) return FSA_ERR_UNSUPPORTED;
    const DecodeCut cut(batch, num_kv_heads, G, (kTileRows / G) & ~3, num_groups, max_len, max_shared, window);
    const int64_t rows = (int64_t)batch * num_q_heads * cut.partials();
    *bytes_out = align_up(rows * head_dim * 4, 256) + align_up(rows * 8, 256);
    return FSA_OK;
}

extern "C" int fsa_biased_decode(const void* q, const void* k, const void* v, int64_t kv_rows, int64_t k_stride_n, int64_t v_stride_n, const int32_t* seq_len,
                                 const int32_t* seq_row0, const void* shared_k, const void* shared_v, int64_t shared_rows, int64_t shared_k_stride_n,
                                 int64_t shared_v_stride_n, const int32_t* cu_shared, const int32_t* cu_group, int num_groups, const float* slopes, int batch, int num_q_heads, int num_kv_heads, int head_dim,
                                 int dtype, float sm_scale, float softcap, int window, int64_t max_len, int64_t max_shared, void* o, float* lse, void* scratch,
                                 int64_t scratch_bytes, void* stream_) {
    int64_t need = 0;
    int rc = fsa_biased_decode_bytes(batch, num_q_heads, num_kv_heads, head_dim, num_groups, max_len, max_shared, window, &need);
    if (rc) return rc;
    if (dtype != FSA_DTYPE_BF16 && dtype != FSA_DTYPE_FP16) return FSA_ERR_BAD_ARG;
    if (!(sm_scale > 0.f) || !(softcap >= 0.f)) return FSA_ERR_BAD_ARG;
    if (batch == 0) return FSA_OK;
    const bool has_shared = num_groups > 0 && shared_rows > 0;
    const int64_t packed = (int64_t)num_kv_heads * head_dim;
    if (!q || !k || !v || !seq_len || !seq_row0 || !o || !lse || !scratch || kv_rows <= 0) return FSA_ERR_BAD_ARG;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || ((uintptr_t)scratch & 31)) return FSA_ERR_BAD_ARG;
    if ((k_stride_n % 8) || (v_stride_n % 8) || k_stride_n < packed || v_stride_n < packed || kv_rows >= ((int64_t)1 << 31)) return FSA_ERR_BAD_ARG;
    if (has_shared && (!shared_k || !shared_v || !cu_shared || !cu_group || !aligned16(shared_k) || !aligned16(shared_v) || (shared_k_stride_n % 8) ||
                       (shared_v_stride_n % 8) || shared_k_stride_n < packed || shared_v_stride_n < packed))
        return FSA_ERR_BAD_ARG;
    if (shared_rows >= kMaxTokens || batch >= kMaxTokens || num_groups >= kMaxTokens) return FSA_ERR_UNSUPPORTED;
    if (scratch_bytes < need) return FSA_ERR_WORKSPACE;
    const int B = batch, Hq = num_q_heads, Hk = num_kv_heads, D = head_dim, G = Hq / Hk, TPT = (kTileRows / G) & ~3;
    const DecodeCut cut(B, Hk, G, TPT, has_shared ? num_groups : 0, max_len, max_shared, window);
    if ((int64_t)B * Hk * cut.parts * cut.nown >= ((int64_t)1 << 31) || cut.nown > (1 << 20)) return FSA_ERR_UNSUPPORTED;
    (void)cudaGetLastError();
    if ((rc = ensure_context())) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    const int64_t rows = (int64_t)B * Hq;
    const int P = cut.partials();
    float* o_part = (float*)scratch;
    float2* ml = (float2*)((char*)scratch + align_up(rows * P * D * 4, 256));
    ScoreMod mod = {};
    const int which = (softcap > 0.f ? kModCap : 0) | (slopes ? kModBias : 0);
    if (softcap > 0.f && !set_cap(&mod, sm_scale, softcap)) return FSA_ERR_BAD_ARG;
    mod.slopes = slopes;
    cudaError_t e;
    BiasedDecodeParams p = {};
    p.q = q; p.seq_len = seq_len; p.row0 = seq_row0;
    p.B = B; p.Hq = Hq; p.Hk = Hk; p.G = G; p.parts = cut.parts; p.window = window; p.chunk = cut.own; p.nchunk = cut.nown; p.P = P; p.p0 = cut.nshared;
    p.scale_log2 = sm_scale * kLog2e; p.mod = mod; p.o_part = o_part; p.ml = ml;
    if ((e = biased_status_word(&p.status)) != cudaSuccess) return cuda_failed(e);
    CUtensorMap kmap, vmap;
    if ((rc = make_tile_map(&kmap, k, dtype, kv_rows, packed, k_stride_n, kBdKT))) return rc;
    if ((rc = make_tile_map(&vmap, v, dtype, kv_rows, packed, v_stride_n, kBdKT))) return rc;
    const bool bf16 = dtype == FSA_DTYPE_BF16;
    if (D == 128) e = bf16 ? launch_bd_which<128, __nv_bfloat16>(which, p, kmap, vmap, stream) : launch_bd_which<128, __half>(which, p, kmap, vmap, stream);
    else e = bf16 ? launch_bd_which<64, __nv_bfloat16>(which, p, kmap, vmap, stream) : launch_bd_which<64, __half>(which, p, kmap, vmap, stream);
    if (e != cudaSuccess) return cuda_failed(e);
    // (beside the own rows' kernel: neither needs anything of the other)
    if (has_shared) {
        BiasedFwdLaunch l = {};
        if ((rc = make_tile_map_3d_box(&l.q, q, dtype, D, B, Hq, (int64_t)Hq * D, D, TPT, G))) return rc;
        if ((rc = make_tile_map(&l.k, shared_k, dtype, shared_rows, packed, shared_k_stride_n, kBiasedBK))) return rc;
        if ((rc = make_tile_map(&l.v, shared_v, dtype, shared_rows, packed, shared_v_stride_n, kBiasedBK))) return rc;
        BiasedFwdParams& r = l.p;
        r.cu_q = cu_group; r.cu_k = cu_shared;
        r.N = B; r.Nk = shared_rows; r.B = num_groups; r.Hq = Hq; r.Hk = Hk; r.G = G; r.TPT = TPT;
        r.scale_log2 = sm_scale * kLog2e;
        r.status = p.status;
        l.mod = mod;
        l.seq_len = seq_len; l.window = window;
        l.o_part = o_part; l.ml = ml; l.P = P; l.nchunk = cut.nshared; l.chunk = cut.tiles;
        e = launch_biased_fwd(D, dtype, which, true, l, cut.mtiles, stream);
        if (e != cudaSuccess) return cuda_failed(e);
    }
    e = launch_biased_merge(D, dtype, BiasedMerge{o_part, ml, rows, Hq, P, cut.nshared, cu_group, num_groups, o, lse, Hq, 1}, stream);
    return e == cudaSuccess ? FSA_OK : cuda_failed(e);
}
