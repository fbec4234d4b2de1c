// softcap.cuh -- the softcap to f32 accuracy, for the heads' epilogues.
#pragma once

#include <cuda_runtime.h>

#include "common.cuh"

namespace z2 {

namespace {

// cap * tanh(l / cap) of N values: an odd polynomial (Taylor to y^11) below |y| = 0.35,
// where its remainder is under 2e-8 of the value, and cap - 2 cap / (exp(2 y) + 1) above,
// whose rounding (a few 2^-24 of cap) is small against the value there.  Where all of the
// warp's values are small, as an output head's mostly are, only the polynomial is
// computed, two values to an instruction.
template <int N>
__device__ __forceinline__ void softcap_exact(float (&l)[N], float cap)
{
    const float inv_cap = 1.0f / cap;
    float most = fabsf(l[0]);
#pragma unroll
    for (int i = 1; i < N; i++) most = fmaxf(most, fabsf(l[i]));
    const bool tiny = __all_sync(kFull, most * inv_cap < 0.35f);
    const float k2 = 2.0f * 1.4426950408889634f * inv_cap;
    auto both = [](float x) { return make_float2(x, x); };
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 x = make_float2(l[i], l[i + 1]), y = __fmul2_rn(x, both(inv_cap)), z = __fmul2_rn(y, y);
        float2 p = __ffma2_rn(z, both(-1382.0f / 155925.0f), both(62.0f / 2835.0f));
        p = __ffma2_rn(z, p, both(-17.0f / 315.0f));
        p = __ffma2_rn(z, p, both(2.0f / 15.0f));
        p = __ffma2_rn(z, p, both(-1.0f / 3.0f));
        p = __ffma2_rn(__fmul2_rn(x, z), p, x);
        if (!tiny) {
            float e0, e1, r0, r1;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(x.x * k2));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(x.y * k2));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(e0 + 1.0f));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(e1 + 1.0f));
            if (!(fabsf(y.x) < 0.35f)) p.x = fmaf(-2.0f * cap, r0, cap);
            if (!(fabsf(y.y) < 0.35f)) p.y = fmaf(-2.0f * cap, r1, cap);
        }
        l[i] = p.x;
        l[i + 1] = p.y;
    }
}

}  // namespace

}  // namespace z2
