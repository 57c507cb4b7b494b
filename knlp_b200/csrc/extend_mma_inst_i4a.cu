// Tensor-core extend attention: instantiation for one pair of plane modes.
#include "extend_mma.cuh"

KNLP_EXTEND_PAIR(KNLP_KV_INT4_ASYM, KNLP_KV_INT4_ASYM)
