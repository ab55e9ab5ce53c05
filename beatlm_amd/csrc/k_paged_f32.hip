// Attention over pages of keys: f32.
#define PAGED_T float
#include "k_paged.inc"
