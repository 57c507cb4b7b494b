// One cached row as fp32, for the stride-generic kernels: a lane owns EPL consecutive elements.
#pragma once

#include "common.cuh"

namespace knlp {

template <int EPL>
__device__ __forceinline__ void load_row(const Plane& p, const uint8_t* crow, const __half* srow,
                                         const __half* zrow, int lane, float out[EPL]) {
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    const int g = e >> 5;
    if (p.mode == KNLP_KV_F16) {  // unquantized K (kfp16_* decodes, reference :1076-1083)
      out[i] = __half2float(reinterpret_cast<const __half*>(crow)[e]);
      continue;
    }
    if (p.mode == KNLP_KV_BF16) {
      out[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(crow)[e]);
      continue;
    }
    const float s = __half2float(srow[g]);
    if (p.mode == KNLP_KV_INT8_G32) {
      out[i] = static_cast<float>(static_cast<int8_t>(crow[e])) * s;
    } else {
      const unsigned b = crow[e >> 1];
      const float c = static_cast<float>((e & 1) ? (b >> 4) : (b & 0xFu));
      if (p.mode == KNLP_KV_INT4_ASYM) {
        out[i] = c * s + __half2float(zrow[g]);
      } else {
        out[i] = (c - 8.0f) * s;
      }
    }
  }
}

}  // namespace knlp
