// The matrix products of the token operators: C[m][n] = sum_k A(m, k) B(n, k) with an epilogue.  Each operand lies in memory with k or with its own index contiguous, so one kernel
// serves x W^T (k, k), dz W (k, n) and dz^T x (m, n) without a transposed copy.
#pragma once
#include "tok_common.hpp"

// A product may run over two ranges of k (dx = dg Wg + du Wu: range 0 on p, range 1 on p2, K long each) or be two products of one shape (dWg = dg^T x, dWu = du^T x: batch 1 reads p2 and
// writes y2).  The gated forward product takes the rows of the "up" projection from b.p2; cut along k it is two products of one shape, joined where their parts are added.
struct TgOperand {
    const void* p;          // element (i, k): p[i * ld + k] (k contiguous) or p[k * ld + i]
    const void* p2;
    long long ld;
    bool padded;            // rows end on a whole 16-byte chunk whose surplus is readable, and zero where it lies along k
};
enum { TG_LINEAR = 0, TG_GATED = 1, TG_STORE = 2, TG_SLAB = 3 };          // epilogues: forward products; a rounded store (gradients); an f32 slab of one part of k (internal)
struct TgArgs {
    TgOperand a, b;
    long long M, N, K;      // gated: N = columns of h; the products have 2 N
    int ranges, batches;    // 1 or 2
    int act;
    const float* bias;      // [N] or null
    const float* bias2;     // gated: of the up projection
    const void* res;        // linear: added after the activation, or null
    long long ldres;
    void* y;                // [M][N]
    void* y2;
    long long ldy;
    float* kept;            // [M][N] pre-activations for the backward pass (gated: kept of gate, kept2 of up), or null
    float* kept2;
};
// dtype MIS_F32 | MIS_BF16; a_mn / b_mn: 1 = the operand's own index is contiguous (else k); epi TG_LINEAR, TG_GATED or TG_STORE.  Enqueues on `stream`.  A product may be cut along
// k: its parts go to `slab` (tg_slab_bytes; null: a forward product is not cut) and are added in their order.
// later (TG_STORE): the sum of the parts, if there are any, is not enqueued but left there for tg_sums - a backward pass adds those of both its products in one launch.
struct TgSum {
    TgArgs a;
    const float* slab;      // null: nothing to add
    int splits;
    long long runs;         // runs of 8 columns
};
int tg_launch(int dtype, int a_mn, int b_mn, int epi, const TgArgs& a, float* slab, hipStream_t stream, TgSum* later = nullptr);
int tg_sums(int dtype, const TgSum& s, const TgSum& t, hipStream_t stream);
size_t tg_slab_bytes(int dtype, int epi, long long M, long long N, long long K, int ranges, int batches);
