// Element types of the policy-side kernels (categorical.hip, grad_clip.hip): float, bfloat16 and half in memory, float in registers.
#pragma once
#include "mdp_device.hpp"

namespace mdp {

struct bf16 { uint16_t bits; };
struct f16 { _Float16 v; };

MDP_DEV float to_f32(float x) { return x; }
MDP_DEV float to_f32(bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }
MDP_DEV float to_f32(f16 x) { return (float)x.v; }

// one rounding, to nearest even; a NaN stays one
MDP_DEV void from_f32(float x, float& y) { y = x; }
MDP_DEV void from_f32(float x, f16& y) { y.v = (_Float16)x; }
MDP_DEV void from_f32(float x, bf16& y) {
    const uint32_t u = __float_as_uint(x);
    y.bits = x != x ? (uint16_t)((u >> 16) | 0x40u) : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

}  // namespace mdp
