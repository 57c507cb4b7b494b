// Tensor-core extend attention: instantiation for one pair of plane modes.
#include "extend_mma.cuh"

KNLP_EXTEND_PAIR(kRaw, KNLP_KV_INT8_G32)
