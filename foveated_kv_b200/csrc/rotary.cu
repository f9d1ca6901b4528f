// Rotary positions of queries and keys in one launch (no counterpart in the
// reference, whose models rotate before they call it).
#include <algorithm>
#include <climits>

#include "fkv_common.h"
#include "paged.cuh"
#include "rotary.cuh"

using namespace fkvdev;

namespace {

constexpr int kThreads = 256;
constexpr int kMostPairs = 4096;   // of a block: 32 KB of sines and cosines

struct RotaryArgs {
    const uint16_t* q;
    const uint16_t* k;
    uint16_t* q_out;
    uint16_t* k_out;
    int64_t qs[3], ks[3], qos[3], kos[3];   // strides of (batch, token, head), elements
    const void* pos;
    int64_t ps[2];                          // strides of (batch, token)
    const double* inv_freq;
    int64_t tokens;
    int S, Hq, Hk, D, half, per_block;
    float amplitude;
    float sign;                             // of the sines: -1 turns back
};

template <bool BF, bool IL, bool W16>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a, bool pos64) {
    extern __shared__ __align__(16) float turns[];       // cosines, sines: [per_block][half] each
    const int upr = a.D >> 3, rows = kThreads / upr;
    const int r = threadIdx.x / upr, u = threadIdx.x - r * upr;
    const int64_t tok0 = (int64_t)blockIdx.x * a.per_block;
    const int n = (int)min((int64_t)a.per_block, a.tokens - tok0);
    float* cosines = turns;
    float* sines = turns + a.per_block * a.half;
    await_predecessor();
    for (int i = threadIdx.x; i < n * a.half; i += kThreads) {
        const int k = i / a.half;
        const int64_t b = (tok0 + k) / a.S, s = tok0 + k - b * a.S, at = b * a.ps[0] + s * a.ps[1];
        const int64_t pos = pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at]
                                  : (int64_t) reinterpret_cast<const int32_t*>(a.pos)[at];
        float c, sn;
        rotary_pair(a.inv_freq, i - k * a.half, pos, a.amplitude, c, sn);
        cosines[i] = c;
        sines[i] = sn * a.sign;
    }
    __syncthreads();
    // a thread stays with one token: its sines in registers, heads in steps
    const int group = rows / a.per_block;                // rows of a token at a time
    const int k = r % a.per_block, h = blockIdx.y * group + r / a.per_block;
    if (r >= group * a.per_block || k >= n) return;
    const RotaryUnit ru = rotary_unit(u, a.half, IL);
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f), sn = c;
    if (ru.turned) {
        c = *reinterpret_cast<const float4*>(cosines + k * a.half + 4 * u);
        sn = *reinterpret_cast<const float4*>(sines + k * a.half + 4 * u);
    }
    const int64_t b = a.S == a.tokens ? 0 : (tok0 + k) / a.S, s = tok0 + k - b * a.S;
    const int step = gridDim.y * group;
    rotary_rows<BF, IL, W16>(a.q + b * a.qs[0] + s * a.qs[1], a.qs[2], a.q_out + b * a.qos[0] + s * a.qos[1], a.qos[2], h,
                             step, a.Hq, ru, c, sn, true);
    rotary_rows<BF, IL, W16>(a.k + b * a.ks[0] + s * a.ks[1], a.ks[2], a.k_out + b * a.kos[0] + s * a.kos[1], a.kos[2], h,
                             step, a.Hk, ru, c, sn, true);
}

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
    FKV_REQUIRE((int64_t)sh->Hq + sh->Hk <= 8192, FKV_ERR_UNSUPPORTED, "fkv_rotary: %d + %d heads are too many",
                sh->Hq, sh->Hk);
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
    bool wide = sh->interleaved != 0;
    for (int i = 0; i < 4; ++i) {
        if (((i & 1) ? sh->Hk : sh->Hq) == 0) {
            to[i][0] = to[i][1] = to[i][2] = 0;
            continue;
        }
        FKV_REQUIRE((reinterpret_cast<uintptr_t>(ptr[i]) & 7) == 0, FKV_ERR_INVALID,
                    "fkv_rotary: tensor not 8-byte aligned");
        wide = wide && (reinterpret_cast<uintptr_t>(ptr[i]) & 15) == 0;
        for (int j = 0; j < 3; ++j) {
            FKV_REQUIRE(st[i][j] % 4 == 0, FKV_ERR_INVALID,
                        "fkv_rotary: stride %lld is not a multiple of 4 elements",
                        (long long)st[i][j]);
            to[i][j] = st[i][j];
            wide = wide && st[i][j] % 8 == 0;
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
    a.tokens = tokens;
    a.S = sh->S;
    a.Hq = sh->Hq;
    a.Hk = sh->Hk;
    a.D = sh->D;
    a.half = sh->rot / 2;
    a.amplitude = sh->amplitude;
    a.sign = sh->inverse ? -1.f : 1.f;
    const int rows = kThreads / (sh->D / 8);
    const int passes = (std::max(sh->Hq, sh->Hk) + rows - 1) / rows;
    a.per_block = tokens_per_block(tokens, sh->Hq + sh->Hk);
    // a row of each token at a time, and sines within the limit
    while (a.per_block * a.half > kMostPairs || a.per_block > rows) a.per_block /= 2;
    // few tokens: their heads are spread over more blocks
    const int gy = (int)std::min<int64_t>(passes, std::max<int64_t>(1, 592 / tokens));
    const dim3 grid((unsigned)((tokens + a.per_block - 1) / a.per_block), (unsigned)gy);
    const size_t smem = (size_t)a.per_block * a.half * 2 * sizeof(float);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool p64 = sh->pos64 != 0;
    const bool early = (int64_t)grid.x * grid.y <= kEarlyBlocks;
    auto run = [&](void (*k)(RotaryArgs, bool)) {
        return fkv::launch_beside(k, grid, kThreads, smem, s, early, a, p64);
    };
    cudaError_t e;
    switch ((sh->bf16 ? 4 : 0) | (sh->interleaved ? 2 : 0) | (wide ? 1 : 0)) {
        case 0: e = run(rotary_kernel<false, false, false>); break;
        case 2: e = run(rotary_kernel<false, true, false>); break;
        case 3: e = run(rotary_kernel<false, true, true>); break;
        case 4: e = run(rotary_kernel<true, false, false>); break;
        case 6: e = run(rotary_kernel<true, true, false>); break;
        default: e = run(rotary_kernel<true, true, true>); break;
    }
    FKV_CUDA_CHECK(e);
    return FKV_OK;
}
