// Attention scores that are not the plain product: capped by a tanh and / or biased by distance,
//   s = scale q.k;   s = cap tanh(s / cap);   s = s - slope_h |t - j|        (t, j: places of the token and the key)
// and what the kernels of range attention need besides.  A kernel's MOD says what it is compiled with; 0 is the plain product.
#pragma once
#include <cfloat>

#include "sm100_prims.cuh"

namespace fsa {

constexpr int kModCap = 1;       // tanh cap
constexpr int kModBias = 2;      // distance bias
constexpr int kModSplit = 4;     // K/V rows cut into chunks, unnormalised partial results (forward)

struct ScoreMod {
    float x_scale;              // scale / cap: from a product to the argument of the tanh
    float near_v;               // products up to this size have the tanh v (near[0] + near[1] v^2 + ...)
    float near[4];
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

// tanh(x) = 1 - 2 / (1 + e^2x) (k = 2 log2(e) times what v is to be multiplied with): off by some 2e-7, whatever the value: for |x| above 3/4, where that is
// 3e-7 of it (a cap of 50 makes 1e-5 of a score).  tanh.approx would take one special-function step instead of two, but is off by 5e-4 of the score.
__device__ __forceinline__ float tanh_far(float v, float k) { return fmaf(-2.f, rcp_approx(1.f + ex2_approx(v * k)), 1.f); }

// tanh_near: of two values no larger than 3/4; cap_scores: v <- tanh(x_scale v), N scores of a row (all lanes of a warp
// call it; whether some |v| of the lanes that count was above near_v).  The special-function unit gives 16 results a cycle and SM, and the
// softmax needs one for each score already; with two more the capped forward would be bound by it, three times as long as its products.
// Where no |x| of the warp's 32 rows is above 3/4 (scores below 37 at a cap of 50), tanh(x) = x p(x^2) with p of degree 4: the
// polynomial that is nearest to tanh(x) / x on [0, 9/16] in relative error, 6e-7 (fitted on Chebyshev points); two scores an instruction.  In other
// warps every score takes the form for its size: the other one's error, times a cap far above a small score, can be as large as the score.
constexpr float kTanhNear = 0.75f;
__device__ __forceinline__ uint64_t tanh_near(uint64_t x) {
    constexpr float c[5] = {0.999999463558197f, -0.3332825005054474f, 0.13258983194828033f, -0.050056297332048416f, 0.012929627671837807f};
    const uint64_t u = mul_f32x2(x, x);
    uint64_t p = f32x2(c[4], c[4]);
#pragma unroll
    for (int i = 3; i >= 0; --i) p = fma_f32x2(p, u, f32x2(c[i], c[i]));
    return mul_f32x2(x, p);
}
template <int N>
__device__ __forceinline__ bool cap_scores(uint32_t (&v)[N], float x_scale, float near_v, bool counts = true) {
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; i += 4) {        // (a NaN stays out of a maximum: it is masked, or makes the row NaN either way)
        a[0] = max3_abs(a[0], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        a[1] = max3_abs(a[1], __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
    }
    const float most = fmaxf(a[0], a[1]);
    if (__all_sync(0xffffffffu, most * x_scale <= kTanhNear)) {
        const uint64_t xs = f32x2(x_scale, x_scale);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 t = f32x2_get(tanh_near(mul_f32x2(f32x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), xs)));
            v[i] = __float_as_uint(t.x);
            v[i + 1] = __float_as_uint(t.y);
        }
    } else {
        const uint64_t xs = f32x2(x_scale, x_scale);
        const float k = 2.f * kLog2e * x_scale;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float a = __uint_as_float(v[i]), b = __uint_as_float(v[i + 1]);
            const float2 x = f32x2_get(mul_f32x2(f32x2(a, b), xs)), t = f32x2_get(tanh_near(f32x2(x.x, x.y)));
            v[i] = __float_as_uint(fabsf(x.x) <= kTanhNear ? t.x : tanh_far(a, k));
            v[i + 1] = __float_as_uint(fabsf(x.y) <= kTanhNear ? t.y : tanh_far(b, k));
        }
    }
    return __any_sync(0xffffffffu, counts && most > near_v);
}

// Of products no larger than near_v, half a cap: tanh(x_scale v) = v p(v^2), p of degree 3 with the scale in its coefficients (host: near_coefficients);
// 6e-7 of the value as well.  f: what every coefficient is multiplied with.
struct NearTanh {
    uint64_t c[4];
    __device__ __forceinline__ NearTanh(const ScoreMod& m, float f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = f32x2(m.near[i] * f, m.near[i] * f);
    }
    // the factor of v
    __device__ __forceinline__ uint64_t slope(uint64_t v) const {
        const uint64_t w = mul_f32x2(v, v);
        return fma_f32x2(fma_f32x2(fma_f32x2(c[3], w, c[2]), w, c[1]), w, c[0]);
    }
};
inline void near_coefficients(ScoreMod* m) {
    // nearest to tanh(x) / x on x^2 in [0, 1/4] in relative error.  Scales whose powers leave the normal numbers do without.
    constexpr double c[4] = {0.999999463558197, -0.33326318860054016, 0.13190296292304993, -0.04440222308039665};
    const double x = m->x_scale;
    m->near_v = 0.f;
    if (!(x >= 1e-4 && x <= 1e4)) return;
    m->near_v = (float)(0.5 / x);
    double pow = x;
    for (int i = 0; i < 4; ++i, pow *= x * x) m->near[i] = (float)(c[i] * pow);
}
// The cap's numbers; false where they leave the normal ones.
inline bool set_cap(ScoreMod* m, float sm_scale, float softcap) {
    m->x_scale = sm_scale / softcap;
    m->cap_log2 = softcap * kLog2e;
    near_coefficients(m);
    return m->x_scale >= FLT_MIN && m->x_scale <= FLT_MAX / 4 && m->cap_log2 >= FLT_MIN && m->cap_log2 <= FLT_MAX;
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
