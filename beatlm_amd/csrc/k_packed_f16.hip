// Attention over packed documents on f16.
#define PACKED_T _Float16
#include "k_packed.inc"
