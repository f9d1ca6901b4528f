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
#include <type_traits>

#include <cuda_fp8.h>

#include "fkv_common.h"
#include "paged.cuh"
#include "rotary.cuh"

using namespace fkvdev;

namespace {

constexpr int kThreads = 256;
constexpr float kRowFloor = 7.888609052210118e-31f;   // 2^-100

struct AppendArgs {
    FkvPagedCache c;
    const uint16_t *k, *v, *q;
    uint16_t* q_out;
    int64_t ks[3], vs[3], qs[3], qos[3];   // strides of (sequence, token, head), elements
    const int32_t* cu_new;
    const double* inv_freq;
    int T, per_block, n_uniform, Hq, half, pshift;
    float amplitude;
};

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// Where a new token is read and stored.
struct Place {
    int64_t k, v, q, q_out;   // element offsets of its rows
    int64_t line;             // its row of head 0 in the pages; < 0: it is not stored
    int64_t pos;
};
__device__ __forceinline__ Place place_of(const AppendArgs& a, int t) {
    Place p;
    int n, b, i;
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
        used = lo < a.c.B && t >= a.cu_new[lo];
        b = min(lo, a.c.B - 1);
        n = a.cu_new[b + 1] - a.cu_new[b];
        i = t - a.cu_new[b];
    }
    const int len = a.c.lens[b];
    used = used && (a.cu_new != nullptr || len != 0);   // an empty slot of a fixed batch
    p.pos = (int64_t)len - n + i;
    p.line = -1;
    if (used) {
        if (p.pos < 0 || p.pos >= ((int64_t)a.c.width << a.pshift)) {
            paged_report(a.c.status, FKV_PAGED_BAD_POSITION);
        } else {
            const int pid = a.c.table[(int64_t)b * a.c.table_stride + (p.pos >> a.pshift)];
            if ((unsigned)pid >= (unsigned)a.c.n_pages)
                paged_report(a.c.status, FKV_PAGED_BAD_PAGE);
            else
                p.line = (((int64_t)pid * a.c.Hk) << a.pshift) + (p.pos & ((1 << a.pshift) - 1));
        }
    }
    // a uniform batch has strides of (sequence, token, head), packed rows of (token, head)
    const int64_t sb = a.cu_new ? 0 : b, st = a.cu_new ? t : i;
    p.k = sb * a.ks[0] + st * a.ks[1];
    p.v = sb * a.vs[0] + st * a.vs[1];
    p.q = sb * a.qs[0] + st * a.qs[1];
    p.q_out = sb * a.qos[0] + st * a.qos[1];
    return p;
}

// A block takes up to 16 new tokens (or a slice of one's rows): D/8 lanes of a
// warp to a row, first the tokens' 2 Hk key and value rows, then their Hq
// query rows.
template <int D, bool BF, bool FP8, bool IL, bool W16>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int LPR = D / 8, ROWS = kThreads / LPR;
    extern __shared__ __align__(16) float turns[];       // cosines, sines: [per_block][half] each
    __shared__ Place places[kMostTokens];
    const int u = threadIdx.x % LPR, r = threadIdx.x / LPR;
    const int tok0 = blockIdx.x * a.per_block, count = min(a.per_block, a.T - tok0);
    await_predecessor();
    if (threadIdx.x < count) places[threadIdx.x] = place_of(a, tok0 + threadIdx.x);
    __syncthreads();
    float* cosines = turns;
    float* sines = turns + a.per_block * a.half;
    if (a.half) {
        for (int i = threadIdx.x; i < count * a.half; i += kThreads) {
            const int k = i / a.half;
            if (places[k].line >= 0)
                rotary_pair(a.inv_freq, i - k * a.half, places[k].pos, a.amplitude, cosines[i], sines[i]);
        }
        __syncthreads();
    }
    // a thread stays with one token: its place and sines in registers, heads in
    // steps.  All lanes of a warp take the same number of steps (the shuffles).
    const int group = ROWS / a.per_block;                // rows of a token at a time
    const int k = r % a.per_block, h0 = blockIdx.y * group + r / a.per_block, step = gridDim.y * group;
    const bool mine = r < group * a.per_block && k < count;
    const Place p = places[mine ? k : 0];
    const bool live = mine && p.line >= 0;
    const RotaryUnit ru = rotary_unit(u, a.half, IL);
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f), s = c;
    if (ru.turned && live) {
        c = *reinterpret_cast<const float4*>(cosines + k * a.half + 4 * u);
        s = *reinterpret_cast<const float4*>(sines + k * a.half + 4 * u);
    }
    const int Hk = a.c.Hk;
    constexpr int NH = 2;    // heads with their rows in flight (32K tokens of 8 kv heads, fp8: 119 us, one at a time 127)
    for (int i = 0; i < Hk; i += NH * step) {
        uint2 w[2 * NH][2] = {};                         // their keys and values
#pragma unroll
        for (int e = 0; e < NH; ++e) {
            const int h = i + e * step + h0;
            if (live && h < Hk) {
                load_unit<W16>(a.k + p.k + h * a.ks[2], ru, w[2 * e]);
                load_unit<W16>(a.v + p.v + h * a.vs[2], ru, w[2 * e + 1]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2 * NH; ++j) {
            if (i + (j >> 1) * step >= Hk) break;        // no such head for any thread
            const bool isk = (j & 1) == 0;
            const int h = i + (j >> 1) * step + h0;
            const bool have = live && h < Hk;
            const int64_t line = p.line + ((int64_t)h << a.pshift);
            void* pages = isk ? a.c.k_pages : a.c.v_pages;
            if (FP8) {
                float x[8];
                unpack4<BF>(w[j][0], x);
                unpack4<BF>(w[j][1], x + 4);
                if (isk && ru.turned) rotary_apply(x, c, s, IL);
                // the largest magnitude by its bits: a NaN is above infinity and stays
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                float most = __uint_as_float(top);
                most = most < kRowFloor ? kRowFloor : most;
                if (have) {
                    const float inv = 448.f / most;
                    const uint32_t lo = e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
                    const uint32_t hi = e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
                    uint8_t* dst = reinterpret_cast<uint8_t*>(pages) + line * D;
                    if (W16) {
                        *reinterpret_cast<uint2*>(dst + ru.off0) = make_uint2(lo, hi);
                    } else {
                        *reinterpret_cast<uint32_t*>(dst + ru.off0) = lo;
                        *reinterpret_cast<uint32_t*>(dst + ru.off1) = hi;
                    }
                    if (u == 0) (isk ? a.c.k_scale : a.c.v_scale)[line] = most / 448.f;
                }
            } else if (have) {
                if (isk && ru.turned) turn_unit<BF>(w[j], c, s, IL);
                store_unit<W16>(reinterpret_cast<uint16_t*>(pages) + line * D, ru, w[j]);
            }
        }
    }
    if (mine)                                            // zeros where a token is not stored
        rotary_rows<BF, IL, W16>(a.q + p.q, a.qs[2], a.q_out + p.q_out, a.qos[2], h0, step, a.Hq, ru, c, s, live);
}

struct ReadArgs {
    FkvPagedCache c;
    uint16_t *k, *v;
    int max_len, n_chunks, pshift;
};

constexpr int kReadTokens = 64;   // tokens of one (sequence, kv head) per block

// 8 codes -> 16-bit elements
template <bool BF>
__device__ __forceinline__ uint4 widen(const uint2 w, float s) {
    const uint32_t u[2] = {w.x, w.y};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
            (__nv_fp8x2_storage_t)((u[i >> 1] >> ((i & 1) * 16)) & 0xFFFFu), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        r[i] = pack2<BF>(f.x * s, f.y * s);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// A block reads 64 tokens of one (sequence, kv head), a thread 8 elements of a
// row at a time, so that a warp's stores fill whole sectors (16 codes and two
// stores a thread: 24.4 us for 16K tokens), with the loads of several rows of
// K and V in flight together.
template <int D, bool BF, bool FP8>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadArgs a) {
    constexpr int LPR = D / 8, ROWS = kThreads / LPR, MOST = FP8 ? 8 : 4;
    constexpr int AT_ONCE = kReadTokens / ROWS < MOST ? kReadTokens / ROWS : MOST;
    using Piece = std::conditional_t<FP8, uint2, uint4>;
    const int u = threadIdx.x % LPR, r = threadIdx.x / LPR;
    const int64_t bh = blockIdx.x / a.n_chunks;
    const int chunk = (int)(blockIdx.x - bh * a.n_chunks);
    const int b = (int)(bh / a.c.Hk), h = (int)(bh - (int64_t)b * a.c.Hk);
    const int64_t reach = (int64_t)a.c.width << a.pshift;
    const int len = a.c.lens[b];
    if ((len < 0 || len > reach) && threadIdx.x == 0 && chunk == 0 && h == 0)
        paged_report(a.c.status, FKV_PAGED_BAD_POSITION);
    const int n = (int)min((int64_t)min(len, a.max_len), reach);
    const int32_t* tab = a.c.table + (int64_t)b * a.c.table_stride;
#pragma unroll 1
    for (int j0 = 0; j0 < kReadTokens / ROWS; j0 += AT_ONCE) {
        const int tok0 = chunk * kReadTokens + j0 * ROWS + r;
        int64_t line[AT_ONCE];
        Piece kw[AT_ONCE], vw[AT_ONCE];
        float ks[AT_ONCE], vs[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int tok = tok0 + j * ROWS;
            line[j] = -1;
            if (tok < n) {
                const int pid = tab[tok >> a.pshift];
                if ((unsigned)pid < (unsigned)a.c.n_pages)
                    line[j] = (((int64_t)pid * a.c.Hk + h) << a.pshift) + (tok & ((1 << a.pshift) - 1));
                else if (u == 0)
                    paged_report(a.c.status, FKV_PAGED_BAD_PAGE);
            }
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            kw[j] = vw[j] = Piece{};
            ks[j] = vs[j] = 0.f;
            if (line[j] >= 0) {
                const int64_t at = line[j] * LPR + u;
                kw[j] = reinterpret_cast<const Piece*>(a.c.k_pages)[at];
                vw[j] = reinterpret_cast<const Piece*>(a.c.v_pages)[at];
                if (FP8) {
                    ks[j] = a.c.k_scale[line[j]];
                    vs[j] = a.c.v_scale[line[j]];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int tok = tok0 + j * ROWS;
            if (tok >= a.max_len) continue;
            const int64_t o = (bh * a.max_len + tok) * LPR + u;
            if constexpr (FP8) {
                reinterpret_cast<uint4*>(a.k)[o] = widen<BF>(kw[j], ks[j]);
                reinterpret_cast<uint4*>(a.v)[o] = widen<BF>(vw[j], vs[j]);
            } else {
                reinterpret_cast<uint4*>(a.k)[o] = kw[j];
                reinterpret_cast<uint4*>(a.v)[o] = vw[j];
            }
        }
    }
}

template <int D, bool BF, bool FP8>
cudaError_t launch_append(const AppendArgs& a, dim3 grid, size_t smem, bool il, bool wide, cudaStream_t s) {
    const bool early = (int64_t)grid.x * grid.y <= kEarlyBlocks;
    if (wide) return fkv::launch_beside(append_kernel<D, BF, FP8, true, true>, grid, kThreads, smem, s, early, a);
    if (il) return fkv::launch_beside(append_kernel<D, BF, FP8, true, false>, grid, kThreads, smem, s, early, a);
    return fkv::launch_beside(append_kernel<D, BF, FP8, false, false>, grid, kThreads, smem, s, early, a);
}

template <int D>
cudaError_t launch_append(const AppendArgs& a, dim3 grid, size_t smem, bool il, bool wide, cudaStream_t s) {
    if (a.c.bf16)
        return a.c.fp8 ? launch_append<D, true, true>(a, grid, smem, il, wide, s)
                       : launch_append<D, true, false>(a, grid, smem, il, wide, s);
    return a.c.fp8 ? launch_append<D, false, true>(a, grid, smem, il, wide, s)
                   : launch_append<D, false, false>(a, grid, smem, il, wide, s);
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
    FKV_REQUIRE(((int64_t)c->width << sh) <= 1 << 30, FKV_ERR_UNSUPPORTED,
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
    FKV_REQUIRE(c->Hk <= 4096 && n->Hq <= 8192, FKV_ERR_UNSUPPORTED, "fkv_paged_append: %d / %d heads are too many",
                c->Hk, n->Hq);
    if (n->T == 0) return FKV_OK;
    FKV_REQUIRE(n->k && n->v && (n->Hq == 0 || (n->q && n->q_out)) && (n->rot == 0 || n->inv_freq),
                FKV_ERR_INVALID, "fkv_paged_append: NULL pointer");
    AppendArgs a;
    a.c = *c;
    const int64_t* st[4] = {n->k_stride, n->v_stride, n->q_stride, n->q_out_stride};
    int64_t* to[4] = {a.ks, a.vs, a.qs, a.qos};
    const void* ptr[4] = {n->k, n->v, n->q, n->q_out};
    bool wide = n->rot == 0 || n->interleaved != 0;      // a unit is 16 bytes in a row
    for (int i = 0; i < 4; ++i) {
        if (i >= 2 && n->Hq == 0) {
            to[i][0] = to[i][1] = to[i][2] = 0;
            continue;
        }
        FKV_REQUIRE((reinterpret_cast<uintptr_t>(ptr[i]) & 7) == 0, FKV_ERR_INVALID,
                    "fkv_paged_append: tensor not 8-byte aligned");
        wide = wide && (reinterpret_cast<uintptr_t>(ptr[i]) & 15) == 0;
        for (int j = 0; j < 3; ++j) {
            FKV_REQUIRE(st[i][j] % 4 == 0, FKV_ERR_INVALID,
                        "fkv_paged_append: stride %lld is not a multiple of 4 elements", (long long)st[i][j]);
            to[i][j] = st[i][j];
            wide = wide && st[i][j] % 8 == 0;
        }
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (c->B == 0) {             // packed rows of no sequence: padding, whose queries are zeros
        const int64_t tok = a.qos[1], head = a.qos[2];
        const size_t row = c->D * sizeof(uint16_t);
        const bool packed = head == c->D;        // a token's heads in a row
        for (int h = 0; h < (packed ? std::min(n->Hq, 1) : n->Hq); ++h) {
            const size_t width = packed ? n->Hq * row : row;
            const size_t pitch = n->T > 1 ? (size_t)tok * sizeof(uint16_t) : width;
            FKV_CUDA_CHECK(cudaMemset2DAsync(n->q_out + h * head, pitch, 0, width, n->T, s));
        }
        return FKV_OK;
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
    a.T = n->T;
    const int rows = kThreads / (c->D / 8);
    const int passes = (std::max(c->Hk, n->Hq) + rows - 1) / rows;
    // few tokens: their rows are spread over more blocks
    a.per_block = std::min(tokens_per_block(n->T, 2 * c->Hk + n->Hq), rows);
    const dim3 grid((n->T - 1) / a.per_block + 1, std::min(passes, std::max(1, 592 / n->T)));
    const size_t smem = (size_t)a.per_block * a.half * 2 * sizeof(float);
    const bool il = n->interleaved != 0;
    FKV_CUDA_CHECK(c->D == 64    ? launch_append<64>(a, grid, smem, il, wide, s)
                   : c->D == 128 ? launch_append<128>(a, grid, smem, il, wide, s)
                                 : launch_append<256>(a, grid, smem, il, wide, s));
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
