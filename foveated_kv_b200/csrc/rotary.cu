// Rotary positions of queries and keys in one launch (no counterpart in the
// reference, whose models rotate before they call it).
#include <algorithm>
#include <climits>

#include "fkv_common.h"
#include "rotary.cuh"

using namespace fkvdev;

namespace {

constexpr int kThreads = 128;

struct RotaryArgs {
    const uint16_t* q;
    const uint16_t* k;
    uint16_t* q_out;
    uint16_t* k_out;
    int64_t qs[3], ks[3], qos[3], kos[3];   // strides of (batch, token, head), elements
    const void* pos;
    int64_t ps[2];                          // strides of (batch, token)
    const double* inv_freq;
    int S, Hq, Hk, D, half;
    float amplitude, sign;
};

// One block per token (and slice of the heads): thread = (unit u, row r); the
// unit's sines are computed once and used for every head of its rows.
template <bool BF, bool IL, bool POS64>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
    const int upr = a.D >> 3;
    const int rows = kThreads / upr;
    const int r = threadIdx.x / upr, u = threadIdx.x - r * upr;
    if (r >= rows) return;
    const int64_t tok = blockIdx.x;
    const int64_t b = tok / a.S, s = tok - b * a.S;
    const RotaryUnit ru = rotary_unit(u, a.half, IL);
    Turn t;
    if (ru.turned) {
        const int64_t pi = b * a.ps[0] + s * a.ps[1];
        const int64_t pos = POS64 ? reinterpret_cast<const int64_t*>(a.pos)[pi]
                                  : (int64_t) reinterpret_cast<const int32_t*>(a.pos)[pi];
        double rate[4];
        rotary_rates(a.inv_freq, u, rate);
        t = rotary_turn(rate, pos, a.amplitude, a.sign);
    }
    const uint16_t* q = a.q + b * a.qs[0] + s * a.qs[1];
    const uint16_t* k = a.k + b * a.ks[0] + s * a.ks[1];
    uint16_t* qo = a.q_out + b * a.qos[0] + s * a.qos[1];
    uint16_t* ko = a.k_out + b * a.kos[0] + s * a.kos[1];
    const int H = a.Hq + a.Hk;
    for (int h = blockIdx.y * rows + r; h < H; h += gridDim.y * rows) {
        const bool isq = h < a.Hq;
        const uint16_t* src = isq ? q + h * a.qs[2] : k + (h - a.Hq) * a.ks[2];
        uint16_t* dst = isq ? qo + h * a.qos[2] : ko + (h - a.Hq) * a.kos[2];
        const uint2 w0 = *reinterpret_cast<const uint2*>(src + ru.off0);
        const uint2 w1 = *reinterpret_cast<const uint2*>(src + ru.off1);
        if (!ru.turned) {
            *reinterpret_cast<uint2*>(dst + ru.off0) = w0;
            *reinterpret_cast<uint2*>(dst + ru.off1) = w1;
            continue;
        }
        float x[8];
        unpack4<BF>(w0, x);
        unpack4<BF>(w1, x + 4);
        rotary_apply(x, t, IL);
        *reinterpret_cast<uint2*>(dst + ru.off0) = pack4<BF>(x);
        *reinterpret_cast<uint2*>(dst + ru.off1) = pack4<BF>(x + 4);
    }
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }

}  // namespace

extern "C" int fkv_rotary(const FkvRotaryShape* sh, const uint16_t* q, const uint16_t* k,
                          const void* positions, const double* inv_freq, uint16_t* q_out,
                          uint16_t* k_out, void* stream) {
    FKV_REQUIRE(sh != nullptr, FKV_ERR_INVALID, "fkv_rotary: shape is NULL");
    FKV_REQUIRE(sh->B >= 0 && sh->S >= 0 && sh->Hq >= 0 && sh->Hk >= 0, FKV_ERR_INVALID,
                "fkv_rotary: negative size (B=%d S=%d Hq=%d Hk=%d)", sh->B, sh->S, sh->Hq, sh->Hk);
    FKV_REQUIRE(sh->D >= 8 && sh->D <= 1024 && sh->D % 8 == 0, FKV_ERR_UNSUPPORTED,
                "fkv_rotary: head dim %d is not a multiple of 8 up to 1024", sh->D);
    FKV_REQUIRE(sh->rot >= 8 && sh->rot <= sh->D && sh->rot % 8 == 0, FKV_ERR_UNSUPPORTED,
                "fkv_rotary: rotated part %d is not a multiple of 8 within the head dim %d",
                sh->rot, sh->D);
    const int64_t tokens = (int64_t)sh->B * sh->S;
    FKV_REQUIRE(tokens <= INT_MAX, FKV_ERR_UNSUPPORTED, "fkv_rotary: %lld tokens exceed the grid",
                (long long)tokens);
    if (tokens == 0 || sh->Hq + sh->Hk == 0) return FKV_OK;
    FKV_REQUIRE(positions && inv_freq && (sh->Hq == 0 || (q && q_out)) &&
                    (sh->Hk == 0 || (k && k_out)),
                FKV_ERR_INVALID, "fkv_rotary: NULL pointer");
    RotaryArgs a;
    const int64_t* st[4] = {sh->q_stride, sh->k_stride, sh->q_out_stride, sh->k_out_stride};
    int64_t* to[4] = {a.qs, a.ks, a.qos, a.kos};
    const void* ptr[4] = {q, k, q_out, k_out};
    for (int i = 0; i < 4; ++i) {
        if (((i & 1) ? sh->Hk : sh->Hq) == 0) {
            to[i][0] = to[i][1] = to[i][2] = 0;
            continue;
        }
        FKV_REQUIRE(aligned8(ptr[i]), FKV_ERR_INVALID, "fkv_rotary: tensor not 8-byte aligned");
        for (int j = 0; j < 3; ++j) {
            FKV_REQUIRE(st[i][j] % 4 == 0, FKV_ERR_INVALID,
                        "fkv_rotary: stride %lld is not a multiple of 4 elements",
                        (long long)st[i][j]);
            to[i][j] = st[i][j];
        }
    }
    a.q = q;
    a.k = k;
    a.q_out = q_out;
    a.k_out = k_out;
    a.pos = positions;
    a.ps[0] = sh->pos_stride[0];
    a.ps[1] = sh->pos_stride[1];
    a.inv_freq = inv_freq;
    a.S = sh->S;
    a.Hq = sh->Hq;
    a.Hk = sh->Hk;
    a.D = sh->D;
    a.half = sh->rot / 2;
    a.amplitude = sh->amplitude;
    a.sign = sh->inverse ? -1.f : 1.f;
    const int rows = kThreads / (sh->D / 8);
    const int passes = (sh->Hq + sh->Hk + rows - 1) / rows;
    // few tokens: their heads are spread over more blocks
    const int gy = (int)std::min<int64_t>(passes, std::max<int64_t>(1, 592 / tokens));
    const dim3 grid((unsigned)tokens, (unsigned)gy);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int mode = (sh->bf16 ? 4 : 0) | (sh->interleaved ? 2 : 0) | (sh->pos64 ? 1 : 0);
    switch (mode) {
        case 0: rotary_kernel<false, false, false><<<grid, kThreads, 0, s>>>(a); break;
        case 1: rotary_kernel<false, false, true><<<grid, kThreads, 0, s>>>(a); break;
        case 2: rotary_kernel<false, true, false><<<grid, kThreads, 0, s>>>(a); break;
        case 3: rotary_kernel<false, true, true><<<grid, kThreads, 0, s>>>(a); break;
        case 4: rotary_kernel<true, false, false><<<grid, kThreads, 0, s>>>(a); break;
        case 5: rotary_kernel<true, false, true><<<grid, kThreads, 0, s>>>(a); break;
        case 6: rotary_kernel<true, true, false><<<grid, kThreads, 0, s>>>(a); break;
        default: rotary_kernel<true, true, true><<<grid, kThreads, 0, s>>>(a); break;
    }
    FKV_LAUNCH_CHECK();
    return FKV_OK;
}
