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
// A block takes a few tokens: it first puts the sines and cosines of their
// pairs into shared memory, one pair per thread, then goes over all rows
// (heads) of the tokens.  A unit is 4 pairs = 8 elements, the work of one
// thread on one row: at off0 and off1, 4 elements each.  rot is a multiple of
// 8, so a unit is either turned as a whole or passed through as a whole.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace fkvdev {

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

// tokens of a block, a power of two: enough for some 450 rows, as long as that
// leaves kMinBlocks blocks (us with 4 / 8 / 16 tokens: 16K tokens of 40 heads of
// 128 57.9 / 55.5 / -, 28.7K of 4 + 4 + 28, fp8 - / 83.8 / 86.1)
constexpr int kMinBlocks = 148 * 8, kMostTokens = 16, kBlockRows = 450;
inline int tokens_per_block(int64_t tokens, int rows) {
    int p = 1;
    while (p < kMostTokens && 2 * p * rows <= kBlockRows && tokens / (2 * p) >= kMinBlocks) p *= 2;
    return p;
}

// grids of up to so many blocks are launched beside their predecessor
constexpr int kEarlyBlocks = 148 * 4;

// rows that a thread has in flight: loads come first, since the compiler may
// not move them over the stores of rows that could be the same memory
constexpr int kRowsAtOnce = 4;

// cosine and sine (times amplitude) of pair p at position pos (inv_freq without
// __restrict__, which allows loads through the read-only cache: an early launch's
// inputs may still be written while it waits)
__device__ __forceinline__ void rotary_pair(const double* inv_freq, int p, int64_t pos,
                                            float amplitude, float& c, float& s) {
    constexpr double kInv2Pi = 0.15915494309189533577;
    const double turns = (double)pos * (inv_freq[p] * kInv2Pi);
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    c *= amplitude;
    s *= amplitude;
}

// x[0..3] are the elements at off0, x[4..7] those at off1; c, s of 4 pairs
__device__ __forceinline__ void rotary_apply(float (&x)[8], const float4 c4, const float4 s4, bool interleaved) {
    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int ia = interleaved ? 2 * i : i, ib = interleaved ? 2 * i + 1 : 4 + i;
        const float a = x[ia], b = x[ib];
        x[ia] = fmaf(a, c[i], -b * s[i]);
        x[ib] = fmaf(a, s[i], b * c[i]);
    }
}

// A unit of a row of 16-bit elements.  W16: one 16-byte access (its two groups
// are neighbours and rows are 16-byte aligned), otherwise two of 8.
template <bool W16>
__device__ __forceinline__ void load_unit(const uint16_t* row, const RotaryUnit& u, uint2 (&w)[2]) {
    if (W16) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + u.off0);
        w[0] = make_uint2(x.x, x.y);
        w[1] = make_uint2(x.z, x.w);
    } else {
        w[0] = *reinterpret_cast<const uint2*>(row + u.off0);
        w[1] = *reinterpret_cast<const uint2*>(row + u.off1);
    }
}
template <bool W16>
__device__ __forceinline__ void store_unit(uint16_t* row, const RotaryUnit& u, const uint2 (&w)[2]) {
    if (W16) {
        *reinterpret_cast<uint4*>(row + u.off0) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
    } else {
        *reinterpret_cast<uint2*>(row + u.off0) = w[0];
        *reinterpret_cast<uint2*>(row + u.off1) = w[1];
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

// the unit turned, in its 16-bit form
template <bool BF>
__device__ __forceinline__ void turn_unit(uint2 (&w)[2], const float4 c, const float4 s, bool interleaved) {
    float x[8];
    unpack4<BF>(w[0], x);
    unpack4<BF>(w[1], x + 4);
    rotary_apply(x, c, s, interleaved);
    w[0] = pack4<BF>(x);
    w[1] = pack4<BF>(x + 4);
}

// Rows of one token, heads h, h + step, ...: turned or passed through, or zeros
// where !live
template <bool BF, bool IL, bool W16>
__device__ __forceinline__ void rotary_rows(const uint16_t* src, int64_t src_head, uint16_t* dst, int64_t dst_head,
                                            int h, int step, int heads, const RotaryUnit& ru, const float4 c,
                                            const float4 s, bool live) {
    src += h * src_head;
    dst += h * dst_head;
    const int64_t ds = step * src_head, dd = step * dst_head;
    for (; h < heads; h += kRowsAtOnce * step) {
        uint2 w[kRowsAtOnce][2];
#pragma unroll
        for (int j = 0; j < kRowsAtOnce; ++j) {
            w[j][0] = w[j][1] = make_uint2(0, 0);
            if (live && h + j * step < heads) load_unit<W16>(src + j * ds, ru, w[j]);
        }
#pragma unroll
        for (int j = 0; j < kRowsAtOnce; ++j) {
            if (h + j * step >= heads) break;
            if (ru.turned && live) turn_unit<BF>(w[j], c, s, IL);
            store_unit<W16>(dst + j * dd, ru, w[j]);
        }
        src += kRowsAtOnce * ds;
        dst += kRowsAtOnce * dd;
    }
}

}  // namespace fkvdev
