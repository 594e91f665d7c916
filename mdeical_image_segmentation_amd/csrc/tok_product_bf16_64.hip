// bf16 token products, 64 x 64 tiles, 16-byte aligned operands of whole chunks (tok_product.hpp)
#include "tok_product.hpp"

int tok_product_bf16_64(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream) { return tp_pick<__bf16, 2, true>(a_mn, b_mn, epi, a, pl, stream); }
