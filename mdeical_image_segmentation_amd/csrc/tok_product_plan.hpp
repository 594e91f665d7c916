// How a token product is cut, and the launchers of tok_product_*.hip
#pragma once
#include "tok_gemm.hpp"

// where a work item lies
struct TpItem {
    int bt, sp;             // batch, part of k
    long long m0, n0;
};
struct TpPlan {
    int tm, tn;             // tiles of a product
    int splits;             // parts of the k steps (TG_SLAB, else 1)
    int spr;                // steps of one range
    int sps;                // steps of one part
    int items;              // batches * splits * tm * tn
    float* slab;            // TG_SLAB: [batch][part][M][N] f32
};

int tok_product_bf16_256(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
int tok_product_bf16_128(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
int tok_product_bf16_128_any(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
int tok_product_bf16_64(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
int tok_product_bf16_64_any(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
int tok_product_f32_128(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
int tok_product_f32_128_any(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
int tok_product_f32_64(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
int tok_product_f32_64_any(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream);
// forward products of at most 32 rows (tok_skinny.hip)
int tok_product_skinny(int dtype, int epi, const TgArgs& a, bool aligned, hipStream_t stream);
