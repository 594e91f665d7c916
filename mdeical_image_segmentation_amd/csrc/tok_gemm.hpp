// The matrix products of the token operators: C[m][n] = sum_k A(m, k) B(n, k) with an epilogue.  Each operand lies in memory with k or with its own index contiguous, so one kernel
// serves x W^T (k, k), dz W (k, n) and dz^T x (m, n) without a transposed copy.
#pragma once
#include "tok_common.hpp"

struct TgOperand {
    const void* p;          // element (i, k): p[i * ld + k] (k contiguous) or p[k * ld + i]
    const void* p2;         // second tensor of a pair: the columns of the "up" projection (EPI gated), or the k >= split of (gate | up) weights
    long long ld;
    long long split;
};
enum { TG_LINEAR = 0, TG_GATED = 1 };
struct TgArgs {
    TgOperand a, b;
    long long M, N, K;      // gated: N = columns of h; the products have 2 N
    int act;
    const float* bias;      // [N] or null
    const float* bias2;     // gated: of the up projection
    const void* res;        // linear: added after the activation, or null
    long long ldres;
    void* y;                // [M][N]; rows m >= msplit go to y2
    void* y2;
    long long ldy, msplit;
    float* z;               // pre-activation(s) kept for the backward pass, [M][N] f32, or null
    float* z2;
    long long ldz;
};
// dtype MIS_F32 | MIS_BF16; a_mn / b_mn: 1 = the operand's own index is contiguous (else k); epi TG_*.  Enqueues on `stream`.
int tg_launch(int dtype, int a_mn, int b_mn, int epi, const TgArgs& a, hipStream_t stream);
