// Shared by the range-attention backward's kernels (range_bwd_dkdv.cu) and their callers (fsa_api.cu, sel_bwd.cu).
#pragma once
#include "sel_launch.cuh"

namespace fsa {

inline int range_kv_items() { return 8 * sm_count(); }       // work items (all heads) that the plan aims at
constexpr int kRkMinTiles = 8;          // shortest stretch that a K/V tile's tokens are cut into, in row tiles

struct RangeKvPlan {
    const int32_t* cu_q;
    const int32_t* cu_k;
    const int32_t* kv_lo;
    const int32_t* kv_hi;
    int64_t N, Nk;
    int B, Hk, TPT, max_tiles;
    int D;
    int aim;            // range_kv_items()
    int* counts;        // [0] items, [1] tiles cut into several items, [2] items that have been taken (biased_bwd_dkdv.cu)
    int4* tiles;        // [max_tiles] first K/V row, rows, first and last token that see one of them
    int4* items;        // tile, first row tile of its stretch, row tiles, slab (-1: written in place)
    int4* multi;        // first K/V row, rows, first slab, slabs
};

// Sizes of the plan and the slabs: ceil(n / C) <= 2 n / C for a tile that is cut, so the cut tiles have at most 2 aim / Hk items.
inline int64_t range_kv_max_tiles(const SelShape& s) { return (s.Nk + kTileRows - 1) / kTileRows + s.B; }
inline int64_t range_kv_max_cut(const SelShape& s, int64_t aim = range_kv_items()) {
    const int64_t row_tiles = range_kv_max_tiles(s) * ((s.N + s.TPT - 1) / s.TPT);
    const int64_t a = 2 * aim / s.Hk + 1, b = 2 * row_tiles / kRkMinTiles + 1;
    return a < b ? a : b;
}
inline int64_t range_kv_plan_bytes(const SelShape& s, int64_t aim = range_kv_items()) { return 256 + 16 * (3 * range_kv_max_tiles(s) + range_kv_max_cut(s, aim)); }
inline int64_t range_kv_slab_bytes(const SelShape& s, int64_t aim = range_kv_items()) { return range_kv_max_cut(s, aim) * s.Hk * (2 * 128 * (int64_t)s.D * 4); }

// Work items from the stretches (one CTA of T threads): a tile of n row tiles becomes ceil(n / C) items of about equal length, C the
// smallest length that leaves about p.aim items (times heads), and at least kRkMinTiles: below that an item's epilogue weighs
// more than an idle SM.
template <int T>
__device__ __forceinline__ void plan_items(const RangeKvPlan& p) {
    __shared__ int wa[32], wb[32], wc[32];      // (of the T / 32 warps)
    __shared__ long long total;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto row_tiles = [&](const int4& t) { return t.w >= 0 ? (t.w - t.z + p.TPT) / p.TPT : 0; };
    if (tid == 0) total = 0;
    __syncthreads();
    int mine = 0;
    for (int i = tid; i < p.max_tiles; i += T) mine += row_tiles(p.tiles[i]);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) atomicAdd(reinterpret_cast<unsigned long long*>(&total), (unsigned long long)mine);
    __syncthreads();
    const int C = max(kRkMinTiles, (int)((total * p.Hk + p.aim - 1) / p.aim));
    int items = 0, slabs = 0, multi = 0;              // so far
    for (int base = 0; base < p.max_tiles; base += T) {
        const int i = base + tid;
        const int4 t = i < p.max_tiles ? p.tiles[i] : make_int4(0, 0, 0, -1);
        const int n = row_tiles(t);
        const int nch = t.y > 0 ? max(1, (n + C - 1) / C) : 0;
        const int a = nch, b = nch > 1 ? nch : 0, c = nch > 1;
        int sa = a, sb = b, sc = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int ta = __shfl_up_sync(0xffffffffu, sa, o), tb = __shfl_up_sync(0xffffffffu, sb, o), tc = __shfl_up_sync(0xffffffffu, sc, o);
            if (lane >= o) { sa += ta; sb += tb; sc += tc; }
        }
        if (lane == 31) { wa[warp] = sa; wb[warp] = sb; wc[warp] = sc; }
        __syncthreads();
        const int va = lane < T / 32 ? wa[lane] : 0, vb = lane < T / 32 ? wb[lane] : 0, vc = lane < T / 32 ? wc[lane] : 0;
        const int first = items + __reduce_add_sync(0xffffffffu, lane < warp ? va : 0) + sa - a;
        const int slab = slabs + __reduce_add_sync(0xffffffffu, lane < warp ? vb : 0) + sb - b;
        const int list = multi + __reduce_add_sync(0xffffffffu, lane < warp ? vc : 0) + sc - c;
        for (int j = 0; j < nch; ++j) {
            const int r0 = (int)((int64_t)n * j / nch), r1 = (int)((int64_t)n * (j + 1) / nch);
            p.items[first + j] = make_int4(i, r0, r1 - r0, nch > 1 ? slab + j : -1);
        }
        if (nch > 1) p.multi[list] = make_int4(t.x, t.y, slab, nch);
        items += __reduce_add_sync(0xffffffffu, va);
        slabs += __reduce_add_sync(0xffffffffu, vb);
        multi += __reduce_add_sync(0xffffffffu, vc);
        __syncthreads();
    }
    if (tid == 0) { p.counts[0] = items; p.counts[1] = multi; p.counts[2] = 0; }
}

cudaError_t launch_range_bwd_plan(const RangeKvPlan& p, const SelBwdArgs& a, int* status, cudaStream_t stream);
// The stretches alone, as part of a chain of dependent launches; leaves the status word alone.
cudaError_t launch_range_key_tiles(const RangeKvPlan& p, const SelBwdArgs& a, cudaStream_t stream);
// dk / dv rows of the K/V tiles that were cut, as part of such a chain; head_dim 64 or 128
cudaError_t launch_range_dkdv_reduce(int dtype, const RangeKvPlan& p, const float* slabs, void* dk, void* dv, int sms, cudaStream_t stream);
cudaError_t launch_range_bwd_dkdv(int dtype, const RangeKvPlan& p, const SelBwdArgs& a, const SelShape& s, const CUtensorMap& kmap,
                                  const CUtensorMap& vmap, int* status, cudaStream_t stream);

}  // namespace fsa
