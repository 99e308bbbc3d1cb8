// Element types of the policy-side kernels (categorical.hip, grad_clip.hip): float, bfloat16 and half in memory, float in registers.
#pragma once
#include "mdp_device.hpp"
#include <type_traits>

namespace mdp {

struct bf16 { uint16_t bits; };
struct f16 { _Float16 v; };

MDP_DEV float to_f32(float x) { return x; }
MDP_DEV float to_f32(bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }
MDP_DEV float to_f32(f16 x) { return (float)x.v; }

// one rounding, to nearest even; a NaN stays one (v_cvt_pk_bf16_f32 for bfloat16)
MDP_DEV void from_f32(float x, float& y) { y = x; }
MDP_DEV void from_f32(float x, f16& y) { y.v = (_Float16)x; }
MDP_DEV void from_f32(float x, bf16& y) { y.bits = __builtin_bit_cast(uint16_t, (__bf16)x); }

// 16 bytes of elements, the unit of vector loads and stores
template <typename T>
struct Chunk {
    static constexpr int N = 16 / sizeof(T);
    uint4 raw;
    MDP_DEV float at(int e) const {
        const uint32_t w = e * (int)sizeof(T) / 4 == 0 ? raw.x : e * (int)sizeof(T) / 4 == 1 ? raw.y : e * (int)sizeof(T) / 4 == 2 ? raw.z : raw.w;
        return unpack((T*)nullptr, w, e);
    }
    MDP_DEV static Chunk lowest() {                    // -inf in every place
        const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, f16>::value ? 0xfc00fc00u : 0xff80ff80u;
        return Chunk{uint4{w, w, w, w}};
    }
    MDP_DEV static Chunk of(const float (&v)[N]) {
        Chunk c;
        uint32_t w[4];
        for (int k = 0; k < 4; ++k) w[k] = pack((T*)nullptr, v, k);
        c.raw = uint4{w[0], w[1], w[2], w[3]};
        return c;
    }

private:
    MDP_DEV static float unpack(float*, uint32_t w, int) { return __uint_as_float(w); }
    MDP_DEV static float unpack(bf16*, uint32_t w, int e) { return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16); }
    MDP_DEV static float unpack(f16*, uint32_t w, int e) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? w >> 16 : w & 0xffffu));
    }
    MDP_DEV static uint32_t pack(float*, const float (&v)[N], int k) { return __float_as_uint(v[k]); }
    MDP_DEV static uint32_t pack(bf16*, const float (&v)[N], int k) {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        pair q;
        q[0] = (__bf16)v[2 * k];
        q[1] = (__bf16)v[2 * k + 1];
        return __builtin_bit_cast(uint32_t, q);
    }
    MDP_DEV static uint32_t pack(f16*, const float (&v)[N], int k) {
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        pair q;
        q[0] = (_Float16)v[2 * k];
        q[1] = (_Float16)v[2 * k + 1];
        return __builtin_bit_cast(uint32_t, q);
    }
};

}  // namespace mdp
