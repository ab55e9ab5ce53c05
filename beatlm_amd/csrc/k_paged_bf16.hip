// Attention over pages of keys: bf16.
#define PAGED_T __bf16
#include "k_paged.inc"
