// Activations of the products' epilogues (codes: enum Act in kernels.h).
#pragma once
#include "kernels.h"

namespace gonn {
namespace {

// The epilogues keep their accumulators in registers, so their loops are fully unrolled:
// 32 to 128 copies of whatever the activation inlines.  With expf / tanhf inlined in every
// copy the epilogue's code no longer fits the instruction cache, and even a ReLU, which
// only branches past them, took 11 us longer per launch (512 x 1024 x 1024: 27 against
// 16 us).  The transcendental activations are therefore one out-of-line function.
__device__ __noinline__ float apply_act_transcendental(float v, int act) {
  switch (act) {
    case ACT_SIGMOID: return 1.0f / (1.0f + expf(-v));
    case ACT_TANH: return tanhf(v);
    default: return 0.5f * v * (1.0f + tanhf(0.7978845608f * (v + 0.044715f * v * v * v)));  // ACT_GELU
  }
}
__device__ __forceinline__ float apply_act(float v, int act, float param) {
  if (act == ACT_RELU) return fmaxf(v, 0.0f);
  if (act == ACT_LEAKY) return v > 0.0f ? v : v * param;
  if (act == ACT_SIGMOID || act == ACT_TANH || act == ACT_GELU) return apply_act_transcendental(v, act);
  return v;
}

}  // namespace
}  // namespace gonn
