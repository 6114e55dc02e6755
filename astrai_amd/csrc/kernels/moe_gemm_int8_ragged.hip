// The 8-bit products for rows that are no whole number of 128-byte K steps (the
// chunks past a row's end are staged from zeros) or outputs whose rows are no whole
// number of 16-byte stores: the kernels of moe_gemm_int8.hip under namespace
// ragged, as a code object of its own.
#define ASTRAI_MOE_RAGGED_K 1
#include "moe_gemm_int8.hip"
