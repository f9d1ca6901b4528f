// Paged key-value cache: writing new tokens (with rotary positions and 8-bit
// quantisation on the way) and reading sequences back (no counterpart in the
// reference, whose cache holds whole sequences of one length).
//
// Pages are (n_pages, Hk, page, D); the table names the page of tokens
// [j * page, (j + 1) * page) of a sequence.  8-bit rows are E4M3 codes times
// one f32 scale per (token, kv head):
//   most  = max(|x|, 2^-100) over the row (NaN if any is)
//   scale = most / 448,  code = e4m3(x * (448 / most)), to nearest even
// so a row with an infinity or a NaN reads back as NaN throughout.
#include <algorithm>
#include <climits>

#include <cuda_fp8.h>

#include "fkv_common.h"
#include "paged.cuh"
#include "rotary.cuh"

using namespace fkvdev;

namespace {

constexpr int kThreads = 128;
constexpr float kRowFloor = 7.888609052210118e-31f;   // 2^-100

struct AppendArgs {
    FkvPagedCache c;
    const uint16_t *k, *v, *q;
    uint16_t* q_out;
    int64_t ks[3], vs[3], qs[3], qos[3];   // strides of (sequence, token, head), elements
    const int32_t* cu_new;
    const double* inv_freq;
    int n_uniform, Hq, half, pshift;
    float amplitude;
};

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// One block per new token (and slice of its rows): Hk key rows, Hk value rows
// and Hq query rows, each taken by D/8 lanes of one warp.
template <int D, bool BF, bool FP8, bool IL>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int LPR = D / 8, ROWS = kThreads / LPR;
    const int u = threadIdx.x % LPR, r = threadIdx.x / LPR;
    const int t = blockIdx.x;
    // sequence and position of token t
    int b, i, n;
    bool used = true;
    if (a.cu_new == nullptr) {
        n = a.n_uniform;
        b = t / n;
        i = t - b * n;
    } else {
        int lo = 0, hi = a.c.B;               // last b with cu_new[b] <= t
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.cu_new[mid] <= t) lo = mid; else hi = mid - 1;
        }
        b = lo;
        used = b < a.c.B && t >= a.cu_new[b];
        b = min(b, a.c.B - 1);
        n = a.cu_new[b + 1] - a.cu_new[b];
        i = t - a.cu_new[b];
    }
    const int len = a.c.lens[b];
    used = used && (a.cu_new != nullptr || len != 0);   // an empty slot of a fixed batch
    const int64_t pos = (int64_t)len - n + i;
    int pid = -1;
    if (used) {
        if (pos < 0 || pos >= ((int64_t)a.c.width << a.pshift)) {
            paged_report(a.c.status, FKV_PAGED_BAD_POSITION);
        } else {
            pid = a.c.table[(int64_t)b * a.c.table_stride + (pos >> a.pshift)];
            if ((unsigned)pid >= (unsigned)a.c.n_pages) {
                paged_report(a.c.status, FKV_PAGED_BAD_PAGE);
                pid = -1;
            }
        }
    }
    const bool live = pid >= 0;
    const RotaryUnit ru = rotary_unit(u, a.half, IL);
    Turn turn;
    if (live && ru.turned) {
        double rate[4];
        rotary_rates(a.inv_freq, u, rate);
        turn = rotary_turn(rate, pos, a.amplitude, 1.f);
    }
    // strides: a uniform batch is (sequence, token, head); packed rows are (token, head)
    const int64_t sb = a.cu_new ? 0 : b, st = a.cu_new ? t : i;
    const uint16_t* krow = a.k + sb * a.ks[0] + st * a.ks[1];
    const uint16_t* vrow = a.v + sb * a.vs[0] + st * a.vs[1];
    const uint16_t* qrow = a.q + sb * a.qs[0] + st * a.qs[1];
    uint16_t* qout = a.q_out + sb * a.qos[0] + st * a.qos[1];
    const int Hk = a.c.Hk, H = 2 * Hk + a.Hq;
    const int prow = (int)(pos & ((1 << a.pshift) - 1));
    for (int base = blockIdx.y * ROWS; base < H; base += gridDim.y * ROWS) {
        const int h = base + r;
        const bool isq = h >= 2 * Hk, isv = h >= Hk && !isq;
        const int hh = isq ? h - 2 * Hk : isv ? h - Hk : h;
        const bool have = live && h < H;
        uint2 w0 = make_uint2(0, 0), w1 = make_uint2(0, 0);
        if (have) {
            const uint16_t* src = isq ? qrow + hh * a.qs[2] : isv ? vrow + hh * a.vs[2] : krow + hh * a.ks[2];
            w0 = *reinterpret_cast<const uint2*>(src + ru.off0);
            w1 = *reinterpret_cast<const uint2*>(src + ru.off1);
        }
        float x[8];
        unpack4<BF>(w0, x);
        unpack4<BF>(w1, x + 4);
        if (ru.turned && !isv && have) {
            rotary_apply(x, turn, IL);
            w0 = pack4<BF>(x);
            w1 = pack4<BF>(x + 4);
        }
        if (isq) {
            if (h < H) {                       // zeros behind the last sequence
                uint16_t* dst = qout + hh * a.qos[2];
                *reinterpret_cast<uint2*>(dst + ru.off0) = w0;
                *reinterpret_cast<uint2*>(dst + ru.off1) = w1;
            }
        }
        const int64_t line = (((int64_t)pid * Hk + hh) << a.pshift) + prow;
        if (FP8) {
            // the largest magnitude by its bits: a NaN is above infinity and stays
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1)
                top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            float most = __uint_as_float(top);
            most = most < kRowFloor ? kRowFloor : most;
            if (have && !isq) {
                const float inv = 448.f / most;
                uint8_t* dst = reinterpret_cast<uint8_t*>(isv ? a.c.v_pages : a.c.k_pages) + line * D;
                *reinterpret_cast<uint32_t*>(dst + ru.off0) =
                    e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
                *reinterpret_cast<uint32_t*>(dst + ru.off1) =
                    e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
                if (u == 0) (isv ? a.c.v_scale : a.c.k_scale)[line] = most / 448.f;
            }
        } else if (have && !isq) {
            uint16_t* dst = reinterpret_cast<uint16_t*>(isv ? a.c.v_pages : a.c.k_pages) + line * D;
            *reinterpret_cast<uint2*>(dst + ru.off0) = w0;
            *reinterpret_cast<uint2*>(dst + ru.off1) = w1;
        }
    }
}

struct ReadArgs {
    FkvPagedCache c;
    uint16_t *k, *v;
    int max_len, n_chunks, pshift;
};

constexpr int kReadTokens = 64;   // tokens of one (sequence, kv head) per block

// 8 stored elements -> 8 16-bit elements
template <bool BF, bool FP8>
__device__ __forceinline__ uint4 read8(const void* pages, const float* scale, int64_t line, int D, int e) {
    if (!FP8)
        return *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(pages) + line * D + e);
    const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(pages) + line * D + e);
    const float s = scale[line];
    uint32_t o[4];
    const uint32_t u[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
            (__nv_fp8x2_storage_t)((u[i >> 1] >> ((i & 1) * 16)) & 0xFFFFu), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        o[i] = pack2<BF>(f.x * s, f.y * s);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int D, bool BF, bool FP8>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadArgs a) {
    constexpr int LPR = D / 8, ROWS = kThreads / LPR;
    const int u = threadIdx.x % LPR, r = threadIdx.x / LPR;
    const int64_t bh = blockIdx.x / a.n_chunks;
    const int chunk = (int)(blockIdx.x - bh * a.n_chunks);
    const int b = (int)(bh / a.c.Hk), h = (int)(bh - (int64_t)b * a.c.Hk);
    const int64_t reach = (int64_t)a.c.width << a.pshift;
    const int len = a.c.lens[b];
    if (len > reach && u == 0 && r == 0 && chunk == 0 && h == 0)
        paged_report(a.c.status, FKV_PAGED_BAD_POSITION);
    const int n = (int)(len < reach ? len : reach);
#pragma unroll
    for (int j = 0; j < kReadTokens / ROWS; ++j) {
        const int tok = chunk * kReadTokens + j * ROWS + r;
        if (tok >= a.max_len) return;
        uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
        if (tok < n) {
            const int pid = a.c.table[(int64_t)b * a.c.table_stride + (tok >> a.pshift)];
            if ((unsigned)pid < (unsigned)a.c.n_pages) {
                const int64_t line = (((int64_t)pid * a.c.Hk + h) << a.pshift) + (tok & ((1 << a.pshift) - 1));
                kw = read8<BF, FP8>(a.c.k_pages, a.c.k_scale, line, D, u * 8);
                vw = read8<BF, FP8>(a.c.v_pages, a.c.v_scale, line, D, u * 8);
            } else if (u == 0) {
                paged_report(a.c.status, FKV_PAGED_BAD_PAGE);
            }
        }
        const int64_t o = (bh * a.max_len + tok) * D + u * 8;
        *reinterpret_cast<uint4*>(a.k + o) = kw;
        *reinterpret_cast<uint4*>(a.v + o) = vw;
    }
}

template <int D>
void launch_append(const AppendArgs& a, dim3 grid, bool il, cudaStream_t s) {
    const int mode = (a.c.bf16 ? 4 : 0) | (a.c.fp8 ? 2 : 0) | (il ? 1 : 0);
    switch (mode) {
        case 0: append_kernel<D, false, false, false><<<grid, kThreads, 0, s>>>(a); break;
        case 1: append_kernel<D, false, false, true><<<grid, kThreads, 0, s>>>(a); break;
        case 2: append_kernel<D, false, true, false><<<grid, kThreads, 0, s>>>(a); break;
        case 3: append_kernel<D, false, true, true><<<grid, kThreads, 0, s>>>(a); break;
        case 4: append_kernel<D, true, false, false><<<grid, kThreads, 0, s>>>(a); break;
        case 5: append_kernel<D, true, false, true><<<grid, kThreads, 0, s>>>(a); break;
        case 6: append_kernel<D, true, true, false><<<grid, kThreads, 0, s>>>(a); break;
        default: append_kernel<D, true, true, true><<<grid, kThreads, 0, s>>>(a); break;
    }
}

template <int D>
void launch_read(const ReadArgs& a, unsigned grid, cudaStream_t s) {
    if (a.c.fp8) {
        if (a.c.bf16) read_kernel<D, true, true><<<grid, kThreads, 0, s>>>(a);
        else read_kernel<D, false, true><<<grid, kThreads, 0, s>>>(a);
    } else {
        if (a.c.bf16) read_kernel<D, true, false><<<grid, kThreads, 0, s>>>(a);
        else read_kernel<D, false, false><<<grid, kThreads, 0, s>>>(a);
    }
}

}  // namespace

namespace fkv {

int paged_check(const FkvPagedCache* c, const char* who, int* pshift) {
    FKV_REQUIRE(c != nullptr, FKV_ERR_INVALID, "%s: cache is NULL", who);
    FKV_REQUIRE(c->D == 64 || c->D == 128 || c->D == 256, FKV_ERR_UNSUPPORTED,
                "%s: head dim %d unsupported (64, 128 or 256)", who, c->D);
    FKV_REQUIRE(c->page >= 8 && c->page <= 256 && (c->page & (c->page - 1)) == 0,
                FKV_ERR_UNSUPPORTED, "%s: page size %d is not a power of two from 8 to 256", who,
                c->page);
    FKV_REQUIRE(c->B >= 0 && c->Hk >= 1 && c->n_pages >= 0 && c->width >= 0 && c->table_stride >= c->width,
                FKV_ERR_INVALID, "%s: bad size (B=%d Hk=%d pages=%d table width=%d stride=%d)", who, c->B,
                c->Hk, c->n_pages, c->width, c->table_stride);
    int sh = 0;
    while ((1 << sh) < c->page) ++sh;
    *pshift = sh;
    FKV_REQUIRE(((int64_t)c->width << sh) <= INT_MAX, FKV_ERR_UNSUPPORTED,
                "%s: table reaches %lld tokens a sequence", who, (long long)c->width << sh);
    if (c->B == 0) return FKV_OK;
    FKV_REQUIRE(c->lens && (c->width == 0 || c->table) && (c->n_pages == 0 || (c->k_pages && c->v_pages)),
                FKV_ERR_INVALID, "%s: NULL pointer", who);
    FKV_REQUIRE(!c->fp8 || c->n_pages == 0 || (c->k_scale && c->v_scale), FKV_ERR_INVALID,
                "%s: 8-bit pages need k_scale and v_scale", who);
    FKV_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_pages) | reinterpret_cast<uintptr_t>(c->v_pages)) & 15) == 0,
                FKV_ERR_INVALID, "%s: pages not 16-byte aligned", who);
    return FKV_OK;
}

}  // namespace fkv

extern "C" int fkv_paged_append(const FkvPagedCache* c, const FkvPagedNew* n, void* stream) {
    int pshift = 0;
    const int rc = fkv::paged_check(c, "fkv_paged_append", &pshift);
    if (rc != FKV_OK) return rc;
    FKV_REQUIRE(n != nullptr, FKV_ERR_INVALID, "fkv_paged_append: new tokens are NULL");
    FKV_REQUIRE(n->T >= 0 && n->Hq >= 0 && n->n_uniform >= 0, FKV_ERR_INVALID,
                "fkv_paged_append: negative size (T=%d Hq=%d n=%d)", n->T, n->Hq, n->n_uniform);
    FKV_REQUIRE(n->rot == 0 || (n->rot >= 8 && n->rot <= c->D && n->rot % 8 == 0), FKV_ERR_UNSUPPORTED,
                "fkv_paged_append: rotated part %d is not a multiple of 8 within the head dim %d", n->rot, c->D);
    FKV_REQUIRE(n->cu_new != nullptr || (int64_t)n->n_uniform * c->B == n->T, FKV_ERR_INVALID,
                "fkv_paged_append: %d tokens are not %d for each of %d sequences", n->T, n->n_uniform, c->B);
    FKV_REQUIRE(n->Hq == 0 || n->rot != 0, FKV_ERR_INVALID, "fkv_paged_append: queries without a rotation");
    if (n->T == 0 || c->B == 0) return FKV_OK;
    FKV_REQUIRE(n->k && n->v && (n->Hq == 0 || (n->q && n->q_out)) && (n->rot == 0 || n->inv_freq),
                FKV_ERR_INVALID, "fkv_paged_append: NULL pointer");
    AppendArgs a;
    a.c = *c;
    const int64_t* st[4] = {n->k_stride, n->v_stride, n->q_stride, n->q_out_stride};
    int64_t* to[4] = {a.ks, a.vs, a.qs, a.qos};
    const void* ptr[4] = {n->k, n->v, n->q, n->q_out};
    for (int i = 0; i < 4; ++i) {
        if (i >= 2 && n->Hq == 0) {
            to[i][0] = to[i][1] = to[i][2] = 0;
            continue;
        }
        FKV_REQUIRE((reinterpret_cast<uintptr_t>(ptr[i]) & 7) == 0, FKV_ERR_INVALID,
                    "fkv_paged_append: tensor not 8-byte aligned");
        for (int j = 0; j < 3; ++j) {
            FKV_REQUIRE(st[i][j] % 4 == 0, FKV_ERR_INVALID,
                        "fkv_paged_append: stride %lld is not a multiple of 4 elements", (long long)st[i][j]);
            to[i][j] = st[i][j];
        }
    }
    a.k = n->k;
    a.v = n->v;
    a.q = n->q;
    a.q_out = n->q_out;
    a.cu_new = n->cu_new;
    a.inv_freq = n->inv_freq;
    a.n_uniform = n->n_uniform;
    a.Hq = n->Hq;
    a.half = n->rot / 2;
    a.pshift = pshift;
    a.amplitude = n->amplitude;
    const int rows = kThreads / (c->D / 8);
    const int passes = (2 * c->Hk + n->Hq + rows - 1) / rows;
    const int gy = std::min(passes, std::max(1, 592 / n->T));   // few tokens: rows over more blocks
    const dim3 grid(n->T, gy);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool il = n->interleaved != 0;
    if (c->D == 64) launch_append<64>(a, grid, il, s);
    else if (c->D == 128) launch_append<128>(a, grid, il, s);
    else launch_append<256>(a, grid, il, s);
    FKV_LAUNCH_CHECK();
    return FKV_OK;
}

extern "C" int fkv_paged_read(const FkvPagedCache* c, int32_t max_len, uint16_t* k, uint16_t* v, void* stream) {
    int pshift = 0;
    const int rc = fkv::paged_check(c, "fkv_paged_read", &pshift);
    if (rc != FKV_OK) return rc;
    FKV_REQUIRE(max_len >= 0, FKV_ERR_INVALID, "fkv_paged_read: max_len %d", max_len);
    if (c->B == 0 || max_len == 0) return FKV_OK;
    FKV_REQUIRE(k && v, FKV_ERR_INVALID, "fkv_paged_read: NULL pointer");
    FKV_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0, FKV_ERR_INVALID,
                "fkv_paged_read: outputs not 16-byte aligned");
    ReadArgs a;
    a.c = *c;
    a.k = k;
    a.v = v;
    a.max_len = max_len;
    a.n_chunks = (int)(((int64_t)max_len + kReadTokens - 1) / kReadTokens);
    a.pshift = pshift;
    const int64_t blocks = (int64_t)c->B * c->Hk * a.n_chunks;
    FKV_REQUIRE(blocks <= INT_MAX, FKV_ERR_UNSUPPORTED, "fkv_paged_read: %lld blocks exceed the grid",
                (long long)blocks);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (c->D == 64) launch_read<64>(a, (unsigned)blocks, s);
    else if (c->D == 128) launch_read<128>(a, (unsigned)blocks, s);
    else launch_read<256>(a, (unsigned)blocks, s);
    FKV_LAUNCH_CHECK();
    return FKV_OK;
}
