// Tensor-core extend attention: instantiation for one pair of plane modes.
#include "extend_launch.cuh"

KNLP_EXTEND_PAIR(kRaw, KNLP_KV_INT4_ASYM)
