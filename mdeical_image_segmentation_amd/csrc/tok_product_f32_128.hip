// f32 token products, 128 x 128 tiles, 16-byte aligned operands of whole chunks (tok_product.hpp)
#include "tok_product.hpp"

int tok_product_f32_128(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream) { return tp_pick<float, 4, true>(a_mn, b_mn, epi, a, pl, stream); }
