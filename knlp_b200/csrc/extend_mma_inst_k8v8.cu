// Tensor-core extend attention: instantiation for one pair of plane modes.
#include "extend_launch.cuh"

KNLP_EXTEND_PAIR(KNLP_KV_INT8_G32, KNLP_KV_INT8_G32)
