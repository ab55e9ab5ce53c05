// Attention over packed documents on f32 (products on v_mfma_f32_32x32x2_f32).
#define PACKED_T float
#include "k_packed.inc"
