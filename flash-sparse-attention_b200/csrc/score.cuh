// Attention scores that are not the plain product: capped by a tanh and / or biased by distance,
//   s = scale q.k;   s = cap tanh(s / cap);   s = s - slope_h |t - j|        (t, j: places of the token and the key)
// and what the kernels of range attention need besides.  A kernel's MOD says what it is compiled with; 0 is the plain product.
#pragma once
#include "sm100_prims.cuh"

namespace fsa {

constexpr int kModCap = 1;       // tanh cap
constexpr int kModBias = 2;      // distance bias
constexpr int kModGuard = 4;     // rows that nobody sees (padding, rows behind a sequence) may hold anything, NaN included
constexpr int kModSplit = 8;     // K/V rows cut into chunks, unnormalised partial results (forward)
constexpr int kModScore = kModCap | kModBias;

struct ScoreMod {
    float x_scale;              // scale / cap: from a product to the argument of the tanh
    float cap_log2;             // cap log2(e): from the tanh to a score in log2 units
    const float* slopes;        // [Hq]
    const int32_t* pos;         // [N] place of every token, as a K/V row
    const int32_t* key_ids;     // [Nk] documents of the K/V rows, negative: padding; or null
    int ahead;                  // tokens may see keys behind their own place
};

template <bool ON> struct Flag { static constexpr bool on = ON; };      // (what a generic lambda is compiled for)

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// tanh(x) = 1 - 2 / (1 + e^2x) for any x (k = 2 log2(e) times what v is to be multiplied with): off by some 2e-7, which a cap of 50
// makes 1e-5 of a score.  tanh.approx would take one special-function step instead of two, but is off by 5e-4 of the score.
__device__ __forceinline__ float tanh_any(float v, float k) { return fmaf(-2.f, rcp_approx(1.f + ex2_approx(v * k)), 1.f); }

// v <- tanh(x_scale v), N scores of a row (all lanes of a warp call it).  The special-function unit gives 16 results a cycle and SM, and the
// softmax needs one for each score already; with two more the capped forward would be bound by it, three times as long as its products.
// Where no |x| of the warp's 32 rows is above 3/4 (scores below 37 at a cap of 50), tanh(x) = x p(x^2) with p of degree 4: the
// polynomial that is nearest to tanh(x) / x on [0, 9/16] in relative error, 6e-7 (fitted on Chebyshev points); two scores an instruction.
constexpr float kTanhNear = 0.75f;
template <int N>
__device__ __forceinline__ void cap_scores(uint32_t (&v)[N], float x_scale) {
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; i += 2) {        // (a NaN stays out of a maximum: it is masked, or makes the row NaN either way)
        a[0] = fmaxf(a[0], fabsf(__uint_as_float(v[i])));
        a[1] = fmaxf(a[1], fabsf(__uint_as_float(v[i + 1])));
    }
    if (__all_sync(0xffffffffu, fmaxf(a[0], a[1]) * x_scale <= kTanhNear)) {
        const uint64_t xs = f32x2(x_scale, x_scale), c0 = f32x2(0.999999463558197f, 0.999999463558197f),
                       c1 = f32x2(-0.3332825005054474f, -0.3332825005054474f), c2 = f32x2(0.13258983194828033f, 0.13258983194828033f),
                       c3 = f32x2(-0.050056297332048416f, -0.050056297332048416f), c4 = f32x2(0.012929627671837807f, 0.012929627671837807f);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint64_t x = mul_f32x2(f32x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), xs), u = mul_f32x2(x, x);
            const float2 t = f32x2_get(mul_f32x2(x, fma_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(c4, u, c3), u, c2), u, c1), u, c0)));
            v[i] = __float_as_uint(t.x);
            v[i + 1] = __float_as_uint(t.y);
        }
    } else {
        const float k = 2.f * kLog2e * x_scale;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __float_as_uint(tanh_any(__uint_as_float(v[i]), k));
    }
}

// v <- scale v - slope |rel - i|, N scores of a row against keys i = 0, 1, ... of a tile; rel: the token's place among them.  both (the
// same for the warp): a key that some row sees may lie behind its token.
template <int N>
__device__ __forceinline__ void bias_scores(uint32_t (&v)[N], float scale, float slope, float rel, bool both) {
    const uint64_t s2 = f32x2(scale, scale);
    if (!both) {
        const float base = -slope * rel;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 s = f32x2_get(fma_f32x2(f32x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), s2,
                                                 f32x2(fmaf(slope, (float)i, base), fmaf(slope, (float)(i + 1), base))));
            v[i] = __float_as_uint(s.x);
            v[i + 1] = __float_as_uint(s.y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __float_as_uint(fmaf(__uint_as_float(v[i]), scale, -slope * fabsf(rel - (float)i)));
    }
}

}  // namespace fsa
