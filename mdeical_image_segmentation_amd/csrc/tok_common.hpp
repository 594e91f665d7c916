// Shared by the token operators (layernorm.hip, tok_gemm*.hip, token_ops.hip): unaligned 16-byte accesses, the activations and their derivatives.
#pragma once
#include "common.hpp"

// 8 consecutive elements <-> 8 floats.  Rows may start at any element (odd widths), so the 16-byte pieces are only element-aligned: the memcpy form compiles to one
// global_{load,store}_dwordx4, which takes any alignment in global memory.
template <typename T> __device__ __forceinline__ u32x4 tok_ld16(const T* p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
template <typename T> __device__ __forceinline__ void tok_st16(T* p, const u32x4& v) { __builtin_memcpy(p, &v, 16); }

template <typename T> __device__ __forceinline__ void tok_ld8(const T* p, float* f) {
    constexpr int EPC = Tr<T>::EPC;
#pragma unroll
    for (int i = 0; i < 8; i += EPC) unpack_chunk<T>(tok_ld16(p + i), f + i);
}
template <typename T> __device__ __forceinline__ void tok_st8(T* p, const float* f) {
    constexpr int EPC = Tr<T>::EPC;
#pragma unroll
    for (int i = 0; i < 8; i += EPC) tok_st16(p + i, pack_chunk<T>(f + i));
}
// ... the first n of them only (n < 8: the ragged end of a row)
template <typename T> __device__ __forceinline__ void tok_ldn(const T* p, float* f, int n) {
    if (n >= 8) return tok_ld8<T>(p, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? ld_elem<T>(p + i) : 0.f;
}
template <typename T> __device__ __forceinline__ void tok_stn(T* p, const float* f, int n) {
    if (n >= 8) return tok_st8<T>(p, f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) st_elem<T>(p + i, f[i]);
}

// ---- activations.  PRECISE (f32 operands): the library's expf and a divide; bf16 operands: the hardware's exp2 / reciprocal (relative error ~1e-6 against 2^-9 of the result's
// own rounding).  gelu_tanh(z) = z/2 (1 + tanh(s)) is evaluated as z sigmoid(2 s): the same function without the cancellation of 1 + tanh at negative z. ----
template <bool PRECISE> __device__ __forceinline__ float tok_sigmoid(float z) {
    if constexpr (PRECISE) return 1.f / (1.f + expf(-z));
    else return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
constexpr float TOK_GT_C = 1.5957691216057308f;          // 2 sqrt(2 / pi)
constexpr float TOK_GT_K = 0.044715f;

// f and, with D, f' of one activation at 8 places; a NaN stays one
template <bool PRECISE, bool D> __device__ __forceinline__ void tok_act8(int act, float* z, float* d) {
    switch (act) {
        case MIS_ACT_RELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (D) d[i] = z[i] > 0.f ? 1.f : 0.f;
                z[i] = z[i] < 0.f ? 0.f : z[i];
            }
            break;
        case MIS_ACT_GELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = z[i];
                float c, e;
                if constexpr (PRECISE) {
                    e = D ? expf(-0.5f * x * x) : 0.f;
                    c = 0.5f * (1.f + erff(x * 0.70710678118654752f));
                } else {
                    // Abramowitz & Stegun 7.1.26: erfc(|x| / sqrt 2) = poly(t) exp(-x^2 / 2), |error| <= 1.5e-7 - a third of erff's instructions, and the exponential is the derivative's
                    // (log2 e and 1/2 are in the constants: the bf16 epilogue of a large product is these instructions: 8192 x 2048 x 8192 236 us, 214 without an activation)
                    e = __builtin_amdgcn_exp2f(-0.72134752044448170f * (x * x));
                    const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * 0.70710678118654752f * fabsf(x));
                    const float q = e * (t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f)))));
                    c = x < 0.f ? q : 1.f - q;
                }
                if constexpr (D) d[i] = c + x * (0.3989422804014327f * e);
                z[i] = x * c;
            }
            break;
        case MIS_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = z[i], x2 = x * x, s = tok_sigmoid<PRECISE>(TOK_GT_C * x * (1.f + TOK_GT_K * x2));
                if constexpr (D) {
                    const float t = s * (1.f - s);
                    d[i] = t == 0.f ? s : s + x * t * (TOK_GT_C * (1.f + 3.f * TOK_GT_K * x2));          // (t = 0 far out, where x2 may be infinite)
                }
                z[i] = x * s;
            }
            break;
        case MIS_ACT_SILU:
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = tok_sigmoid<PRECISE>(z[i]);
                z[i] *= s;
                if constexpr (D) d[i] = fmaf(z[i], 1.f - s, s);
            }
            break;
        case MIS_ACT_SIGMOID:
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = tok_sigmoid<PRECISE>(z[i]);
                if constexpr (D) d[i] = s * (1.f - s);
                z[i] = s;
            }
            break;
        default:
            if constexpr (D) {
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = 1.f;
            }
            break;
    }
}

constexpr long long TOK_BLOCKS = 1ll << 24;          // blocks of 256 threads: a grid holds fewer than 2^32 work-items, and HIP cuts a larger one without an error
static inline size_t tok_align(size_t n) { return (n + 255) & ~(size_t)255; }
static inline bool tok_act_ok(int act) { return act >= MIS_ACT_NONE && act <= MIS_ACT_SIGMOID; }
// out0[n] = sum over the nrow rows of p0[row][n], out1 the same of p1 (either out may be null), in a fixed order; nrow = 0: zeros (token_ops.hip)
int tok_column_sums(const float* p0, const float* p1, long long nrow, long long N, float* out0, float* out1, hipStream_t stream);
