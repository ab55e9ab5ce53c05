// Attention over packed documents on bf16.
#define PACKED_T __bf16
#include "k_packed.inc"
