// Attention over pages of keys: f16.
#define PAGED_T _Float16
#include "k_paged.inc"
