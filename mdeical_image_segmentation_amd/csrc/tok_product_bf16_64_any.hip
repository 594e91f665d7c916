// bf16 token products, 64 x 64 tiles, operands at any element address (tok_product.hpp)
#include "tok_product.hpp"

int tok_product_bf16_64_any(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream) { return tp_pick<__bf16, 2, false>(a_mn, b_mn, epi, a, pl, stream); }
