// expert_mm.cuh -- what the translation units of the grouped and fused
// products share: the call's operands, the row groups and the activations.
#pragma once

#include "common.cuh"

namespace jlb {
namespace emm {

// One product y[p] = act(x[src(p)] W[e] + b[e]) + r[p], p in group e.
struct Product {
    int dtype, base, act;
    int w_order;                       // JLB_ROW_MAJOR: element (k, n) at k*ldw + n
    int64_t E, S, T, K, N;             // experts, output rows, rows of x, inner and output widths
    const int32_t *rowptr;             // E + 1; null with E == 1: all S rows are one group
    const int32_t *rows;               // S: the row of x of each output row; null: the row itself
    const void *x;
    int64_t ldx;
    const void *w;
    int64_t ldw, w_stride;             // leading dimension, elements from one expert to the next
    const void *bias;                  // E x N, or null
    int64_t ldb;
    const void *res;                   // S x N, or null
    int64_t ldr;
    void *z;                           // S x N: the product before act, or null
    int64_t ldz;
    void *y;
    int64_t ldy;
};

// dw[e] = sum over p in group e of x[src(p)]^T dz[p] (K x N each).
struct Gradient {
    int dtype, base;
    int w_order;                       // layout of dw
    int64_t E, S, T, K, N;
    const int32_t *rowptr;
    const int32_t *rows;
    const void *x;
    int64_t ldx;
    const void *dz;
    int64_t lddz;
    void *dw;
    int64_t lddw, dw_stride;
};

// The tensor-core kernels (expert_mm_tc.cu), bf16 operands of 16-byte aligned
// rows, or F32 ones as three planes of bf16: the workspace of their split
// tiles, and the launch; -1 when the driver refuses a tensor map.
size_t tc_product_workspace(const Product &P);
int tc_product(cudaStream_t st, const Product &P, void *ws);
size_t tc_gradient_workspace(const Gradient &G);
int tc_gradient(cudaStream_t st, const Gradient &G, void *ws);

// A stream over the weights for a few rows a group (expert_mm_skinny.cu), any
// type, order and alignment.
bool skinny_ok(const Product &P);
int skinny_product(cudaStream_t st, const Product &P);

// Rows [lo, hi) of group e, kept inside [0, S] whatever rowptr holds.
__device__ __forceinline__ void group_rows(const int32_t *__restrict__ rowptr, int base, int64_t S,
                                           int64_t e, int &lo, int &hi) {
    if (!rowptr) {
        lo = 0;
        hi = (int)S;
        return;
    }
    lo = __ldg(rowptr + e) - base;
    hi = __ldg(rowptr + e + 1) - base;
    lo = lo < 0 ? 0 : lo > S ? (int)S : lo;
    hi = hi < lo ? lo : hi > S ? (int)S : hi;
}

// Whether group e's row range is one that group_rows had to correct.
__device__ __forceinline__ bool group_bad(const int32_t *__restrict__ rowptr, int base, int64_t S,
                                          int64_t e) {
    if (!rowptr) return false;
    const int lo = __ldg(rowptr + e) - base, hi = __ldg(rowptr + e + 1) - base;
    return lo < 0 || hi < lo || hi > S || (e == 0 && lo != 0);
}

// ------------------------------------------------------------ activations
// relu keeps NaN.  silu = z / (1 + e^-z); gelu = z Phi(z).  For BF16 results the
// exponential and the quotients are cheaper; relative to the result, silu's and
// gelu's errors stay below 1e-4 down to z = -10 (the exponential's grows with its
// argument), and the rounding to 8 bits is 2^-8.  silu is 0 where e^-z or its sum leaves the
// quotient's range, below z = -87.3 (BF16) and -88.7 (F32): there its size is
// under 1.1e-36.

// Phi(z), the normal distribution's lower tail, and e = exp(-z^2 / 2) on the way.
// For z < 0, Phi = (a1 t + a2 t^2 + ..) e with t = 1 / (1 + p |z|), and 1 - Phi(-z)
// above: a tail is computed as it is, because (1 + erf) / 2 cancels (below z =
// -5.5 nothing of it is left in fp32).  The a's make the largest relative error
// over -14 <= z <= 0 least for their p (reweighted least squares, p by search):
// 4.2e-6 with six for BF16, 9.4e-8 with eight for F32.  Beyond that the
// error is the exponential's, whose argument's rounding grows with z^2.
// Measured against erfc in 64 bits, z of deviation 2: F32 1.1e-6 at most and
// 8e-8 on average.  8192 x 256 x 16384, where gelu's cost shows: BF16 191 us, F32
// 575 (687 with a rounded reciprocal, 750 with erfcf, 548 with the erff that
// cancels).
template <bool FAST>
__device__ __forceinline__ float phi(float z, float &e) {
    const float s = z * z;
    float q;
    if (FAST) {
        const float t = __fdividef(1.0f, fmaf(0.309f, fabsf(z), 1.0f));
        e = __expf(-0.5f * s);
        q = fmaf(-0.0747226672f, t, 0.185119432f);
        q = fmaf(q, t, 0.0114483713f);
        q = fmaf(q, t, 0.135001994f);
        q = fmaf(q, t, 0.119659127f);
        q = fmaf(q, t, 0.123491637f) * t * e;
    } else {
        const float t = __fdividef(1.0f, fmaf(0.305f, fabsf(z), 1.0f));
        e = expf(-0.5f * s);
        q = fmaf(0.0366991245f, t, -0.152988045f);
        q = fmaf(q, t, 0.185716456f);
        q = fmaf(q, t, -0.0379764289f);
        q = fmaf(q, t, 0.121021474f);
        q = fmaf(q, t, 0.103420926f);
        q = fmaf(q, t, 0.122466808f);
        q = fmaf(q, t, 0.121639733f) * t * e;
    }
    return z < 0.0f ? q : 1.0f - q;
}

// act's last product and the residual's sum are rounded separately (mul_rn,
// add_rn): contracted in one caller and not in another they would give a call
// with the pre-activation kept other bits than one without.
template <typename T>
__device__ __forceinline__ float act_value(float z, int act) {
    constexpr bool fast = sizeof(T) == 2;
    switch (act) {
        case JLB_ACT_RELU: return z < 0.0f ? 0.0f : z;
        case JLB_ACT_SILU: return fast ? __fdividef(z, 1.0f + __expf(-z)) : z / (1.0f + expf(-z));
        case JLB_ACT_GELU: {
            float e;
            return mul_rn(z, phi<fast>(z, e));
        }
        default: return z;
    }
}

template <typename T>
__device__ __forceinline__ float act_slope(float z, int act) {
    constexpr bool fast = sizeof(T) == 2;
    switch (act) {
        case JLB_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case JLB_ACT_SILU: {
            const float s = fast ? __fdividef(1.0f, 1.0f + __expf(-z)) : 1.0f / (1.0f + expf(-z));
            return s * (1.0f + z * (1.0f - s));
        }
        case JLB_ACT_GELU: {
            float e;
            const float p = phi<fast>(z, e);
            return fmaf(z * 0.39894228040143268f, e, p);
        }
        default: return 1.0f;
    }
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

}  // namespace emm
}  // namespace jlb
