// Rotary positions: device code shared by the rotary kernel and the paged
// cache's append kernel.
//
// A head's first `rot` elements are rot/2 pairs; pair p of a token at
// position n turns by n * inv_freq[p] radians:
//   (a, b) -> (a cos - b sin, a sin + b cos) * amplitude
// with a, b at p and p + rot/2 (half layout) or 2p and 2p + 1 (interleaved).
// Elements behind `rot` pass through.
//
// Angles of far positions: n * inv_freq is taken in 64 bits in units of whole
// turns and reduced to [-1/2, 1/2] there (at n = 2^30 its error is below
// 1e-7 of a turn; in 32 bits it would be whole turns), and only the remainder
// goes to sincospif in 32 bits.
//
// A unit is 4 pairs = 8 elements, the work of one thread on one row: two
// 8-byte accesses at off0 and off1.  rot is a multiple of 8, so a unit is
// either turned as a whole or passed through as a whole.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace fkvdev {

struct Turn {
    float c[4], s[4];
};

struct RotaryUnit {
    int off0, off1;   // element offsets of the unit's two groups of 4
    bool turned;
};

__device__ __forceinline__ RotaryUnit rotary_unit(int u, int half, bool interleaved) {
    RotaryUnit r;
    r.turned = 4 * u < half;
    const bool split = r.turned && !interleaved;
    r.off0 = split ? 4 * u : 8 * u;
    r.off1 = split ? half + 4 * u : 8 * u + 4;
    return r;
}

// turns per position of the unit's 4 pairs
__device__ __forceinline__ void rotary_rates(const double* __restrict__ inv_freq, int u,
                                             double (&rate)[4]) {
    constexpr double kInv2Pi = 0.15915494309189533577;
#pragma unroll
    for (int i = 0; i < 4; ++i) rate[i] = inv_freq[4 * u + i] * kInv2Pi;
}

__device__ __forceinline__ Turn rotary_turn(const double (&rate)[4], int64_t pos, float amplitude,
                                            float sign) {
    Turn t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double turns = (double)pos * rate[i];
        const float frac = (float)(turns - rint(turns));
        float s, c;
        sincospif(2.f * frac, &s, &c);
        t.c[i] = c * amplitude;
        t.s[i] = s * amplitude * sign;
    }
    return t;
}

// x[0..3] are the elements at off0, x[4..7] those at off1
__device__ __forceinline__ void rotary_apply(float (&x)[8], const Turn& t, bool interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int ia = interleaved ? 2 * i : i, ib = interleaved ? 2 * i + 1 : 4 + i;
        const float a = x[ia], b = x[ib];
        x[ia] = fmaf(a, t.c[i], -b * t.s[i]);
        x[ib] = fmaf(a, t.s[i], b * t.c[i]);
    }
}

// 16-bit elements <-> 32 bits
template <bool BF>
__device__ __forceinline__ void unpack2(uint32_t u, float* x) {
    if (BF) {
        x[0] = __uint_as_float(u << 16);
        x[1] = __uint_as_float(u & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
        x[0] = f.x;
        x[1] = f.y;
    }
}

template <bool BF>
__device__ __forceinline__ void unpack4(uint2 w, float* x) {
    unpack2<BF>(w.x, x);
    unpack2<BF>(w.y, x + 2);
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}

template <bool BF>
__device__ __forceinline__ uint2 pack4(const float* x) {
    return make_uint2(pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]));
}

}  // namespace fkvdev
