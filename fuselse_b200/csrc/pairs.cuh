// Folds on pairs of fp32 values (sm_100a): add, mul and fma of two values in one
// instruction, and the three-operand maximum.  A fold of K values costs K/2 max,
// K/2 subtractions, K/2 multiplications, K exponentials and K/2 additions, where
// the one-value form (ms_fold) issues 5 K: the folds over 16-bit logits and over
// accumulator tiles are bound by instruction issue and the exponential unit.
// The difference to the maximum is taken first, as in ms_fold, so that logits of
// any magnitude keep their terms in range.
#pragma once

#include "common.cuh"

namespace fl {

using f32x2 = uint64_t;

__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// ex2((v - M) * scale) of a pair, with neg_m = (-M, -M) and scale2 = (scale, scale).
__device__ __forceinline__ float2 exp_pair(f32x2 v, f32x2 neg_m, f32x2 scale2) {
    const float2 t = unpair(mul2(add2(v, neg_m), scale2));
    return make_float2(ex2(t.x), ex2(t.y));
}

// Largest of K values and m, NaN if any is (K even).
template <int K>
__device__ __forceinline__ float max_of(float m, const float* v) {
    float a = m, b = -INFINITY;
#pragma unroll
    for (int i = 0; i < K; i += 4) {
        a = max3_nan(a, v[i], v[i + 1]);
        if (i + 2 < K) b = max3_nan(b, v[i + 2], v[i + 3]);
    }
    return max_nan(a, b);
}

// Folds K values into (m, s), s = sum exp2((x - safe(m)) * scale), given M, the
// largest of them and m.
template <int K>
__device__ __forceinline__ void fold_pairs(float& m, float& s, const float* v, float M, float scale) {
    const float Ms = safe_max(M);
    const f32x2 neg_m = pair(-Ms, -Ms), scale2 = pair(scale, scale);
    f32x2 a = pair(s * ex2((m - Ms) * scale), 0.0f), b = pair(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < K; i += 4) {
        const float2 e = exp_pair(pair(v[i], v[i + 1]), neg_m, scale2);
        a = add2(a, pair(e.x, e.y));
        if (i + 2 < K) {
            const float2 f = exp_pair(pair(v[i + 2], v[i + 3]), neg_m, scale2);
            b = add2(b, pair(f.x, f.y));
        }
    }
    const float2 t = unpair(add2(a, b));
    s = t.x + t.y;
    m = M;
}

// Merge of (m2, s2) into (m, s) under the same scale.
__device__ __forceinline__ void ms_merge_scaled(float& m, float& s, float m2, float s2, float scale) {
    const float M = max_nan(m, m2);
    const float Ms = safe_max(M);
    s = s * ex2((m - Ms) * scale) + s2 * ex2((m2 - Ms) * scale);
    m = M;
}

}  // namespace fl
