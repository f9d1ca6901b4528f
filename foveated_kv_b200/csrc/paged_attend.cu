// Attention of one new token per sequence over the paged cache, split over
// the cache's length and joined (no counterpart in the reference, whose fused
// decode wants every sequence of a batch to have one length).
//
//   out[h] = sum_n p_n v_n / sum_n p_n,  p_n = exp(scale q[h].k_n - m),
//   n over the last `window` (or all) tokens of the sequence that have a page;
//   a sequence without such tokens gives zeros and a log-sum-exp of -inf, one
//   whose scores are all -inf NaN (0 / 0) and -inf.
//
// Work split.  A stream is one (sequence, kv head, group of up to 16 query
// heads); its tokens are cut into units of 64 or 128.  The units of all
// streams, in order, are dealt to the CTAs of one wave in equal contiguous
// runs (or falling ones, see Deal), so every CTA reads the same number of bytes
// whatever the lengths are (the lengths stay on the device: each CTA sums them
// up itself).  A CTA that holds a whole stream writes its output; a piece of
// one is left as a record (maximum, sum, unnormalised output) that a second,
// dependent launch joins.  Short streams that have an SM each stay whole.
// No atomics and no counters: records and descriptors are written before they
// are read in every call, so the workspace needs no initialisation, and two
// calls share nothing.
//
// Tile.  One warp takes 16 or 32 tokens at a time, each lane in 16-byte pieces in
// the order in which the tensor core wants them (row = lane / 4 = g, quad =
// lane % 4 = t):
//   S^T (16 tok x 8 heads)  = K (16 x D) . Q^T      lane: rows g, g + 8 of K
//   O^T (D x 8 heads)      += V^T (D x 16) . P^T    lane: rows 2t, 2t+1, 2t+8, 2t+9 of V
// The products' inner order is free, so the 16-byte pieces of K pair with the
// same pieces of Q; V rows pair up by byte permutes; P^T comes from S^T by an
// 8x8 transpose across lanes.  mma.sync, not tcgen05: with up to 8 heads a
// tile the products are 13 % of the tensor pipe's time, and every byte is used
// once, so the bound is memory.
//
// Loads.  16-bit pages go straight from global memory to registers, K of the
// next tile in flight during the softmax and V, V during the next K (1 x 64K of
// 8 kv heads, f16: 50.9 us, through shared memory 53.1; 33 ragged windows 46 /
// 55).  8-bit pages need twice the instructions a byte, and registers could not
// hide them: they go by 16-byte asynchronous copies through two buffers a warp
// in shared memory (64 x 32K: 531 us direct, 502 through buffers).
//
// 8-bit rows: codes become f16 exactly.  A key's scale multiplies its score.
// A value's scale joins the exponent: w_n = exp2(x_n + log2 s_n - M) with a
// running maximum M of its own, so w never passes the range of f16 however
// large or small the scales are, and the result is (sum w_n c_n) 2^(M-m) / l.
#include <algorithm>
#include <atomic>
#include <climits>
#include <mutex>

#include <cuda_fp8.h>

#include "decode_common.cuh"
#include "fkv_common.h"
#include "paged.cuh"
#include "rotary.cuh"

using namespace fkvdev;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr uint32_t kFull = 0xFFFFFFFFu;
enum { F16 = 0, BF16 = 1, FP8 = 2 };  // what the pages hold

// A running maximum may lag kLazy log2 units behind the scores.  Weights that
// enter the tensor core as f16 (beside f16 and 8-bit pages) are held times
// 2^kLift, up to 2^15 with the lag, and so is their sum: f16 holds them to half
// of 2^-24, which is 2^-36 of the largest weight.  Unlifted, 2^-25 of it, many
// small weights together were lost (500 tokens at 2^-25 of one whose value is
// zero: a quarter of the output); it costs up to 1.3 % (8 x 64K fp8, 16 heads a
// group: 72.4 -> 73.5 us).  bf16 has the range of f32, and its values need the room.
template <int KIND>
constexpr float kLift = KIND == BF16 ? 0.f : 11.f;
template <int KIND>
constexpr float kLazy = KIND == BF16 ? 8.f : 4.f;

struct AttendArgs {
    FkvPagedCache c;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    float* rec_o;      // (2 per CTA, HP heads, D)
    float4* rec_s;     // (2 per CTA, HP heads): m, M, l, 1 if it attended any token
    int4* desc;        // first output row, heads, pieces (0: nothing to join), first record
    int Hq, G, HT, pshift, window, per_stream, wave, waves;
    float sl2;         // scale * log2(e)
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^(a - b) where b is a maximum over a: 0 for an empty side
__device__ __forceinline__ float ratio2(float a, float b) { return a == -INFINITY ? 0.f : ex2(a - b); }

// natural log of l 2^(m - lift); +inf where a score is (the weights are NaN then)
__device__ __forceinline__ float log_sum(float m, float l, float lift) {
    return m == INFINITY ? m : (m + (log2f(l) - lift)) * 0.6931471805599453f;
}

// (not .nc: an early launch's data may be written while the grid already waits)
__device__ __forceinline__ uint4 ldg16(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// the next 16-bit numbers below a and b that leave a positive remainder (0 for 0):
// remainders in (0, 2^-7] of the weight for bf16, [2^-10, 2^-9] for f16
template <bool BF>
__device__ __forceinline__ uint32_t pack2_below(float a, float b) {
    constexpr float f = BF ? 1.f - 0x1p-23f : 1.f - 0x1p-10f;
    uint32_t r;
    if (BF) asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b * f), "f"(a * f));
    else asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b * f), "f"(a * f));
    return r;
}
template <bool BF>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
    if (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Which units a CTA takes: equal shares, or, for 8-bit pages and much work,
// falling ones, 90 % to the first wave of CTAs and the rest to CTAs that start
// as others end; with more work 80 %, 13 % and the rest.  With equal shares of
// 8-bit pages some SMs finished 15 % after the mean (1M tokens: mean 305 us,
// last 370), while a CTA costs a start and a record (1 / 2 / 3 waves, us: 1 x
// 128K fp8, 18 units a CTA: 56.0 / 60.6 / 64.9; 1 x 256K, 37 units: 104 / 99 /
// 104; 1 x 512K, 74: 193 / 180 / 183; 64 x 32K, 221: 552 / 507 / 501).  16-bit
// pages gain nothing (64 x 4K f16, 54 units: 129 / 132 / 135; 64 x 16K, 222:
// 474 / 476 / 475).  The shares go by the CTA's number alone, so pieces and
// results do not depend on who was faster.
constexpr int kMostWaves = 3;
constexpr int kUnits2 = 24, kUnits3 = 100;   // units a CTA from which 2 and 3 waves pay
struct Deal {
    int wave, total, r[kMostWaves];
    Deal() = default;
    __device__ Deal(int total_, int wave_, int waves) : wave(wave_), total(total_) {
        if (waves == 1) {
            r[0] = (total + wave - 1) / wave;
            r[1] = r[2] = 0;
            return;
        }
        const int each = total / wave;
        waves = min(waves, each < kUnits2 ? 1 : each < kUnits3 ? 2 : 3);
        int left = total;
#pragma unroll
        for (int k = 0; k < kMostWaves; ++k) {
            const int share = waves == 2 ? 90 : k == 0 ? 80 : 13;
            r[k] = k >= waves ? 0 : k == waves - 1 ? (left + wave - 1) / wave : max(1, (int)((int64_t)each * share / 100));
            left = max(0, left - wave * r[k]);
        }
    }
    // units [u0, u1) of a CTA
    __device__ void range(int cta, int& u0, int& u1) const {
        if (r[1] == 0) {
            u0 = (int)min((int64_t)r[0] * cta, (int64_t)total);
            u1 = min(u0 + r[0], total);
        } else {
            u0 = begin(cta);
            u1 = begin(cta + 1);
        }
    }
    __device__ int begin(int cta) const {        // first unit of a CTA, at most `total`
        int64_t u = 0;
#pragma unroll
        for (int k = 0; k < kMostWaves; ++k) {
            const int n = min(cta, wave);
            u += (int64_t)n * r[k];
            cta -= n;
        }
        return (int)min(u, (int64_t)total);
    }
    __device__ int cta_of(int unit) const {      // the CTA that takes a unit below `total`
        int cta = 0;
#pragma unroll
        for (int k = 0; k < kMostWaves; ++k) {
            const int64_t n = (int64_t)wave * r[k];
            if (unit < n) return cta + unit / r[k];
            unit -= (int)n;
            cta += wave;
        }
        return cta;
    }
};

template <int D, int KIND>
struct Geo {
    static constexpr int ES = KIND == FP8 ? 1 : 2;            // bytes of a stored element
    static constexpr int RB = D * ES;                         // bytes of a row
    static constexpr int TG = RB >= 256 ? 1 : 2;              // 16-token groups of one warp's tile
    static constexpr int UNIT = kWarps * 16 * TG;             // tokens of one CTA step
    static constexpr int KC = RB / 64;                        // 16-byte pieces of a key row per lane
    static constexpr int KE = 16 / ES;                        // elements of a piece
    static constexpr int KS = KE / 4;                         // tensor-core steps of a piece
    static constexpr int VB = RB >= 128 ? 16 : 8;             // bytes of a value piece
    static constexpr int VC = RB / (8 * VB);                  // value pieces per lane and token
    static constexpr int VW = VB / 4;                         // words of a value piece
    static constexpr int VE = VB / ES;                        // elements of a value piece
    static constexpr int MT = D / 16;                         // 16-row tiles of O^T
    static constexpr int CP = RB / 32;                        // 512-byte copies of a 16-token group
    static constexpr bool DIRECT = KIND != FP8;               // straight to registers
    // one warp's buffer: 16 TG rows of K, of V, their scales, and which of its
    // 8-token groups have a page
    static constexpr int ROWS = 16 * TG;
    static constexpr int OFF_V = ROWS * RB;
    static constexpr int OFF_S = 2 * OFF_V;
    static constexpr int OFF_L = OFF_S + (KIND == FP8 ? ROWS * 8 : 0);
    static constexpr int BUF = OFF_L + 16;
    static constexpr int BUFS = 2;
};

// Rows sit in shared memory in 128-byte lines whose 16-byte pieces are
// permuted by the row, so that the lanes of a tensor-core fragment (8 rows of
// K, or 4 rows and 2 pieces of V, at a time) touch all banks.
template <int RB>
__device__ __forceinline__ constexpr int piece_at(int row, int piece) {
    if (RB >= 128) return row * RB + (piece >> 3) * 128 + (((piece & 7) ^ (row & 7)) << 4);
    const int line = row >> 1;
    return line * 128 + ((((row & 1) * 4 + piece) ^ ((line & 3) * 2)) << 4);
}
// token (of 8) that row i of a fragment stands for
template <int RB>
__device__ __forceinline__ constexpr int token_of(int i) {
    return RB >= 128 && (i & 1) ? ((i - 1) ^ 4) + 1 : i;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// zeros where !ok
__device__ __forceinline__ void copy16_if(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4_if(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts4(uint32_t a, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

// CTAs per SM that a kernel's registers are held to
template <int D, int HP>
constexpr int kPerSm = D == 256 || HP == 16 ? 2 : 3;

// Units of work of sequence b: tokens [lo, len), cut from lo rounded down to 16.
__device__ __forceinline__ void seq_range(const AttendArgs& a, int b, int& lo, int& len) {
    const int reach = a.c.width << a.pshift;
    len = a.c.lens[b];
    if ((unsigned)len > (unsigned)reach) {       // or below zero
        paged_report(a.c.status, FKV_PAGED_BAD_POSITION);
        len = len < 0 ? 0 : reach;
    }
    lo = a.window > 0 ? max(0, len - a.window) : 0;
}
template <int UNIT>
__device__ __forceinline__ int seq_units(int lo, int len) {
    return len <= lo ? 0 : (len - (lo & ~15) + UNIT - 1) / UNIT;
}

// the warps' results of one piece of a stream; shares its memory with the buffers
template <int D, int HP>
struct Join {
    float o[kWarps][HP][D + 2];
    float m[kWarps][HP], M[kWarps][HP], l[kWarps][HP];
    int any[kWarps];     // a token was there
};

template <int D, int HP, int KIND>
constexpr size_t smem_bytes() {
    const size_t r = Geo<D, KIND>::DIRECT ? 0 : (size_t)kWarps * Geo<D, KIND>::BUFS * Geo<D, KIND>::BUF;
    return r > sizeof(Join<D, HP>) ? r : sizeof(Join<D, HP>);
}

// HP query heads a CTA, in NT tiles of 8 columns: 8 a tile, or, of up to 4, one
// in every other column, so that a lane has one head's scores and not the
// scores of one that does not exist beside them (16 x 1K f16, 4 heads a group:
// 17.7 -> 16.9 us).
template <int D, int HP, int KIND>
__global__ void __launch_bounds__(kThreads, kPerSm<D, HP>) attend_kernel(const __grid_constant__ AttendArgs a) {
    using GG = Geo<D, KIND>;
    constexpr int TG = GG::TG, UNIT = GG::UNIT, KC = GG::KC, KS = GG::KS, VC = GG::VC, VW = GG::VW, MT = GG::MT;
    constexpr int RB = GG::RB;
    constexpr bool DIRECT = GG::DIRECT;
    constexpr int NT = HP == 16 ? 2 : 1, NI = HP == 4 ? 1 : 2;   // tiles; heads of a lane in one
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Join<D, HP>& sm = *reinterpret_cast<Join<D, HP>*>(smem_raw);
    __shared__ int sh_scan[kWarps], sh_b, sh_prefix;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int B = a.c.B, HS = a.c.Hk * a.HT;
    const bool bf = KIND == BF16 || (KIND == FP8 && a.c.bf16);
    await_predecessor();
    // this lane's places in a buffer: fragment rows g of K, rows 2t and 2t + 1 of V
    const uint32_t bufs = smem_u32(smem_raw) + warp * (GG::BUFS * GG::BUF);
    const int tok_k = DIRECT ? g : token_of<RB>(g);
    const uint32_t at_k0 = piece_at<RB>(tok_k, t), at_k1 = RB >= 128 ? piece_at<RB>(tok_k, t + 4) : 0;
    uint32_t at_c[GG::CP / 2], at_v[2];      // 512-byte copies of 8 rows
#pragma unroll
    for (int i = 0; i < GG::CP / 2; ++i) at_c[i] = piece_at<RB>(i * (512 / RB) + lane / (RB / 16), lane % (RB / 16));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int tok = token_of<RB>(2 * t + j);
        at_v[j] = GG::OFF_V + (GG::VB == 16 ? piece_at<RB>(tok, g) : piece_at<RB>(tok, g >> 1) + (g & 1) * 8);
    }

    // ---- this CTA's run of units ------------------------------------------------------------
    Deal deal;
    int u0, u1, b = 0, prefix = 0;
    if (a.desc == nullptr) {               // a CTA per stream
        int lo, len;
        b = blockIdx.x / HS;
        seq_range(a, b, lo, len);
        const int n = seq_units<UNIT>(lo, len);
        u0 = (blockIdx.x - b * HS) * n;
        u1 = u0 + n;
    } else if (B == 1) {                   // nothing to sum up
        int lo, len;
        seq_range(a, 0, lo, len);
        deal = Deal(seq_units<UNIT>(lo, len) * HS, a.wave, a.waves);
        deal.range(blockIdx.x, u0, u1);
    } else {
        const int per = (B + kThreads - 1) / kThreads;
        int mine = 0;
        for (int b = tid * per; b < min(B, (tid + 1) * per); ++b) {
            int lo, len;
            seq_range(a, b, lo, len);
            mine += seq_units<UNIT>(lo, len);
        }
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) sh_scan[warp] = incl;
        __syncthreads();
        int before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            before += w < warp ? sh_scan[w] : 0;
            total += sh_scan[w];
        }
        total *= HS;
        const int excl = before + incl - mine;
        deal = Deal(total, a.wave, a.waves);
        deal.range(blockIdx.x, u0, u1);
        if (u0 < u1 && u0 >= excl * HS && u0 < (excl + mine) * HS) {
            int b = tid * per, p = excl;
            while (b + 1 < B) {
                int lo, len;
                seq_range(a, b, lo, len);
                const int n = seq_units<UNIT>(lo, len);
                if (u0 < (p + n) * HS) break;
                p += n;
                ++b;
            }
            sh_b = b;
            sh_prefix = p;
        }
    }
    // sequences without tokens
    for (int b = blockIdx.x; b < B; b += gridDim.x) {
        int lo, len;
        seq_range(a, b, lo, len);
        if (len > lo) continue;
        for (int i = tid; i < a.Hq * D / 2; i += kThreads)
            reinterpret_cast<uint32_t*>(a.out)[(int64_t)b * a.Hq * D / 2 + i] = 0;
        if (a.lse)
            for (int i = tid; i < a.Hq; i += kThreads) a.lse[(int64_t)b * a.Hq + i] = -INFINITY;
        if (a.per_stream)
            for (int i = tid; i < HS; i += kThreads) a.desc[b * HS + i] = make_int4(0, 0, 0, 0);
    }
    if (a.desc != nullptr && !a.per_stream && tid == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    if (u0 >= u1) return;
    if (a.desc != nullptr && B > 1) {
        __syncthreads();
        b = sh_b;
        prefix = sh_prefix;
    }

    for (int u = u0; u < u1 && b < B;) {
        int lo, len;
        seq_range(a, b, lo, len);
        const int nu = seq_units<UNIT>(lo, len);
        if (u >= (prefix + nu) * HS) {       // past this sequence (or it is empty)
            prefix += nu;
            ++b;
            continue;
        }
        const int rel = u - prefix * HS, stream = rel / nu, chunk = rel - stream * nu;
        const int hk = a.HT == 1 ? stream : stream / a.HT, ht = stream - hk * a.HT;
        const int s_begin = u - chunk, s_end = s_begin + nu;       // the stream's units
        const int chunk_end = min(nu, chunk + (u1 - u));
        const int base = lo & ~15;
        const int t_begin = base + chunk * UNIT, t_end = min(len, base + chunk_end * UNIT);
        const int h0 = hk * a.G + ht * HP, nh = min(HP, a.G - ht * HP);
        const int64_t row0 = (int64_t)b * a.Hq + h0;

        // the lane's pieces of query row g: those of a key row, as 16-bit elements
        constexpr int QW = KC * KS / 2;
        uint4 qw[NT][QW];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < QW; ++i) {
                qw[nt][i] = make_uint4(0, 0, 0, 0);
                const int at = (t + 4 * (i / (KS / 2))) * GG::KE + 8 * (i % (KS / 2));
                const int h = HP == 4 ? g >> 1 : nt * 8 + g;
                if ((HP != 4 || (g & 1) == 0) && h < nh) qw[nt][i] = ldg16(a.q + (row0 + h) * D + at);
            }

        // row of the 8-token group `lane` of the tile at token t0 (~0: nothing to read)
        const int32_t* tab = a.c.table + (int64_t)b * a.c.table_stride;
        auto group_of = [&](int t0) {
            const int tok = t0 + 8 * lane;
            uint32_t line = ~0u;
            if (lane < 2 * TG && tok < t_end && tok + 7 >= lo) {
                const int pid = tab[tok >> a.pshift];
                if ((unsigned)pid >= (unsigned)a.c.n_pages)
                    paged_report(a.c.status, FKV_PAGED_BAD_PAGE);
                else
                    line = (((uint32_t)pid * a.c.Hk + hk) << a.pshift) + (tok & ((1 << a.pshift) - 1));
            }
            return line;
        };
        // start the copies of the tile at t0 into `buf`; rows outside [lo, t_end)
        // become zeros.  The last word says which 8-token groups have a page,
        // or kFull where every row is there.
        auto fetch = [&](uint32_t buf, int t0, uint32_t lines) {
            if (t0 < t_end) {
                uint32_t have = __ballot_sync(0xffffffffu, lines != ~0u);
                const bool full = t0 >= lo && t0 + GG::ROWS <= t_end && have == (1u << 2 * TG) - 1;
                have = full ? kFull : have;
#pragma unroll
                for (int k = 0; k < 2 * TG; ++k) {
                    const uint32_t line = __shfl_sync(0xffffffffu, lines, k);
                    const uint64_t at = (uint64_t)(line != ~0u ? line : 0) * RB + lane * 16;
                    const unsigned char* ks = reinterpret_cast<const unsigned char*>(a.c.k_pages) + at;
                    const unsigned char* vs = reinterpret_cast<const unsigned char*>(a.c.v_pages) + at;
                    const uint32_t to = buf + 8 * k * RB;
                    if (full) {
#pragma unroll
                        for (int i = 0; i < GG::CP / 2; ++i) {
                            copy16(to + at_c[i], ks + i * 512);
                            copy16(to + at_c[i] + GG::OFF_V, vs + i * 512);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < GG::CP / 2; ++i) {
                            const int tok = t0 + 8 * k + i * (512 / RB) + lane / (RB / 16);
                            const bool ok = line != ~0u && tok >= lo && tok < t_end;
                            copy16_if(to + at_c[i], ks + i * 512, ok);
                            copy16_if(to + at_c[i] + GG::OFF_V, vs + i * 512, ok);
                        }
                    }
                }
                if (KIND == FP8) {                        // one token's pair of scales per lane
                    const uint32_t line = __shfl_sync(0xffffffffu, lines, (lane >> 3) & (2 * TG - 1));
                    const int tok = t0 + lane;
                    const bool ok = line != ~0u && tok >= lo && tok < t_end;
                    const uint64_t at = ok ? (uint64_t)line + (lane & 7) : 0;
                    if (lane < GG::ROWS) {
                        copy4_if(buf + GG::OFF_S + lane * 8, a.c.k_scale + at, ok);
                        copy4_if(buf + GG::OFF_S + lane * 8 + 4, a.c.v_scale + at, ok);
                    }
                }
                if (lane == 0) sts4(buf + GG::OFF_L, have);
            }
            copies_commit();
        };

        // DIRECT: the lane's pieces of the tile at t0, rows g of K and 2t, 2t + 1 of
        // V of every 8-token group; rows outside [lo, t_end) become zeros
        uint4 kr[TG][2][KC], vr[TG][4][VC];
        // rows g to attend, a bit for each 8-token group; the sign stays once any tile
        // had one (a flag of its own spilled registers)
        uint32_t live = 0;
        auto is_full = [&](int t0, uint32_t lines) {
            return __all_sync(0xffffffffu, lines != ~0u || lane >= 2 * TG) && t0 >= lo && t0 + GG::ROWS <= t_end;
        };
        auto load_k = [&](int t0, uint32_t lines) {
            const bool full = is_full(t0, lines);
            live = full ? ~0u : live & 0x80000000u;
#pragma unroll
            for (int k = 0; k < 2 * TG; ++k) {
                const uint32_t line = __shfl_sync(0xffffffffu, lines, k);
                const unsigned char* src = reinterpret_cast<const unsigned char*>(a.c.k_pages) +
                                           ((uint64_t)line * RB + g * RB + 16 * t);
                if (full) {
#pragma unroll
                    for (int cc = 0; cc < KC; ++cc) kr[k >> 1][k & 1][cc] = ldg16(src + 64 * cc);
                } else {
                    const int tok = t0 + 8 * k + g;
                    const bool ok = line != ~0u && tok >= lo && tok < t_end;
                    if (ok) live |= 0x80000000u | 1u << k;
#pragma unroll
                    for (int cc = 0; cc < KC; ++cc) {
                        kr[k >> 1][k & 1][cc] = make_uint4(0, 0, 0, 0);
                        if (ok) kr[k >> 1][k & 1][cc] = ldg16(src + 64 * cc);
                    }
                }
            }
        };
        auto load_v = [&](int t0, uint32_t lines) {
            const bool full = is_full(t0, lines);
#pragma unroll
            for (int k = 0; k < 2 * TG; ++k) {
                const uint32_t line = __shfl_sync(0xffffffffu, lines, k);
                const unsigned char* src = reinterpret_cast<const unsigned char*>(a.c.v_pages) +
                                           ((uint64_t)line * RB + 2 * t * RB + GG::VB * g);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int tok = t0 + 8 * k + 2 * t + j;
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        uint4& x = vr[k >> 1][2 * (k & 1) + j][c];
                        if (full) {
                            x = ldg16(src + j * RB + 8 * GG::VB * c);
                        } else {
                            x = make_uint4(0, 0, 0, 0);
                            if (line != ~0u && tok >= lo && tok < t_end) x = ldg16(src + j * RB + 8 * GG::VB * c);
                        }
                    }
                }
            }
        };

        int t0 = t_begin + warp * 16 * TG;
        uint32_t buf = 0;      // offset of the tile's buffer
        uint32_t lines = group_of(t0);
        bool seen = false;
        if constexpr (DIRECT) {
            load_k(t0, lines);
            load_v(t0, lines);
        } else {
            fetch(bufs, t0, lines);
        }
        lines = group_of(t0 + UNIT);

        // ---- queries as B fragments, in the order of the key pieces ---------------------------
        uint32_t qf[NT][KC][KS][2];
        float qs[NT][2];      // score factor of heads 2t, 2t + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            qs[nt][0] = qs[nt][1] = a.sl2;
            // f16 holds a bf16 query exactly once its largest magnitude is moved
            // to [2^14, 2^15) (what falls below 2^-24 there is 2^-38 of that
            // magnitude); the power of two goes to the score factor
            float f = 1.f;
            if (KIND == FP8 && bf) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < QW; ++i) {
                    const uint32_t ww[4] = {qw[nt][i].x, qw[nt][i].y, qw[nt][i].z, qw[nt][i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = max(top, max((ww[j] << 16) & 0x7FFF0000u, ww[j] & 0x7FFF0000u));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // exponent of the largest magnitude; infinities and NaN stay as they are
                const int e = top >= 0x7F800000u ? 14 : max((int)(top >> 23) - 127, -100);
                f = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
                const float back = __uint_as_float((uint32_t)(127 - 14 + e) << 23) * a.sl2;
                qs[nt][0] = __shfl_sync(0xffffffffu, back, 8 * t);
                qs[nt][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
            }
#pragma unroll
            for (int i = 0; i < QW; ++i) {
                uint32_t ww[4] = {qw[nt][i].x, qw[nt][i].y, qw[nt][i].z, qw[nt][i].w};
                if (KIND == FP8 && bf) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        ww[j] = pack2<false>(__uint_as_float(ww[j] << 16) * f, __uint_as_float(ww[j] & 0xFFFF0000u) * f);
                }
                // 8 elements = 2 tensor-core steps
                const int cc = i / (KS / 2), st = 2 * (i % (KS / 2));
                qf[nt][cc][st][0] = ww[0];
                qf[nt][cc][st][1] = ww[1];
                qf[nt][cc][st + 1][0] = ww[2];
                qf[nt][cc][st + 1][1] = ww[3];
            }
        }

        // ---- online softmax state ---------------------------------------------------------------
        float o[NT][MT][4];
        float m[NT][2], M[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
            m[nt][0] = m[nt][1] = M[nt][0] = M[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }

        for (; t0 < t_end; t0 += UNIT) {
            const uint32_t lines_next = group_of(t0 + 2 * UNIT);
            if constexpr (!DIRECT) {
                copies_wait<0>();
                __syncwarp();
                fetch(bufs + (GG::BUF - buf), t0 + UNIT, lines);
            }
            const uint32_t cur = bufs + buf;
            buf = GG::BUF - buf;
            // scores
            float x[TG][NT][4];
#pragma unroll
            for (int tg = 0; tg < TG; ++tg)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) x[tg][nt][0] = x[tg][nt][1] = x[tg][nt][2] = x[tg][nt][3] = 0.f;
#pragma unroll
            for (int tg = 0; tg < TG; ++tg)
#pragma unroll
                for (int cc = 0; cc < KC; ++cc) {
                    uint4 k0, k1;
                    if constexpr (DIRECT) {
                        k0 = kr[tg][0][cc];
                        k1 = kr[tg][1][cc];
                    } else {
                        const uint32_t at = cur + 16 * tg * RB + (cc & 1 ? at_k1 : at_k0) + (cc >> 1) * 128;
                        k0 = lds16(at);
                        k1 = lds16(at + 8 * RB);
                    }
                    const uint32_t r0[4] = {k0.x, k0.y, k0.z, k0.w};
                    const uint32_t r1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                    for (int st = 0; st < KS; ++st) {
                        uint32_t a0, a1, a2, a3;
                        if (KIND == FP8) {
                            e4m3x4_to_h2x2(r0[st], a0, a2);
                            e4m3x4_to_h2x2(r1[st], a1, a3);
                        } else {
                            a0 = r0[2 * (st & 1)];
                            a1 = r1[2 * (st & 1)];
                            a2 = r0[2 * (st & 1) + 1];
                            a3 = r1[2 * (st & 1) + 1];
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma<KIND == BF16>(x[tg][nt], a0, a1, a2, a3, qf[nt][cc][st][0], qf[nt][cc][st][1]);
                    }
                }
            float av[TG][2];      // log2 of the values' scales
            float top[NT][2], topw[NT][2];
            uint32_t have = live;
            if constexpr (!DIRECT) {
                have = lds4(cur + GG::OFF_L);
                seen |= have != 0;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = topw[nt][0] = topw[nt][1] = -INFINITY;
#pragma unroll
            for (int tg = 0; tg < TG; ++tg)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int row = 16 * tg + 8 * hf + tok_k;
                    float kscale = 1.f;
                    if (KIND == FP8) {
                        const uint2 w = lds8(cur + GG::OFF_S + row * 8);
                        kscale = __uint_as_float(w.x);
                        av[tg][hf] = lg2(__uint_as_float(w.y));
                    }
                    const bool ok = DIRECT ? (have >> (2 * tg + hf)) & 1
                                           : have == kFull || (((have >> (2 * tg + hf)) & 1) && t0 + row >= lo && t0 + row < t_end);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            float& s = x[tg][nt][2 * hf + i];
                            s *= KIND == FP8 ? qs[nt][i] * kscale : qs[nt][i];
                            if (!ok) s = -INFINITY;
                            top[nt][i] = fmaxf(top[nt][i], s);
                            if (KIND == FP8) topw[nt][i] = fmaxf(topw[nt][i], s + av[tg][hf]);
                        }
                }
            if constexpr (DIRECT) load_k(t0 + UNIT, lines);
            // raise the running maxima when a score passes them by more than kLazy
            bool up = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    up |= top[nt][i] > m[nt][i] + kLazy<KIND>;
                    if (KIND == FP8) up |= topw[nt][i] > M[nt][i] + kLazy<KIND>;
                }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        float y = top[nt][i], z = topw[nt][i];
#pragma unroll
                        for (int s = 4; s < 32; s <<= 1) {
                            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, s));
                            if (KIND == FP8) z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, s));
                        }
                        y = fmaxf(y, m[nt][i]);
                        const float al = ratio2(m[nt][i], y);
                        float aw = al;
                        m[nt][i] = y;
                        l[nt][i] *= al;
                        if (KIND == FP8) {
                            z = fmaxf(z, M[nt][i]);
                            aw = ratio2(M[nt][i], z);
                            M[nt][i] = z;
                        }
#pragma unroll
                        for (int k = 0; k < MT; ++k) {
                            o[nt][k][i] *= aw;
                            o[nt][k][2 + i] *= aw;
                        }
                    }
            }
            // weights, transposed to B fragments; beside 16-bit pages in two parts:
            // one part alone would add an error as large as the output's own
            // rounding (8 bits of bf16: larger), and the second product is free
            // (1 x 128K f16: 96.4 us with one, 95.9 with two).  8-bit pages take
            // one f16 part, 2^-12 of a weight against the codes' 2^-4: with two,
            // 64 x 32K goes from 507 to 516 us, 592 to 617 under the power cap.
            // The first part is cut off below the weight, so that both are
            // positive and an infinite value gives an infinity, not the NaN of
            // inf - inf (f16: for weights from 2^-25 of the largest; under that
            // the second part may be zero)
            uint32_t pf[TG][NT][2], pl[TG][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                auto base = [](float x) { return (x == -INFINITY ? 0.f : x) - kLift<KIND>; };
                const float m0 = base(m[nt][0]), m1 = base(m[nt][1]), M0 = base(M[nt][0]), M1 = base(M[nt][1]);
#pragma unroll
                for (int tg = 0; tg < TG; ++tg)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const float x0 = x[tg][nt][2 * hf], x1 = x[tg][nt][2 * hf + 1];
                        const float p0 = ex2(x0 - m0), p1 = NI == 2 ? ex2(x1 - m1) : 0.f;
                        l[nt][0] += p0;
                        if (NI == 2) l[nt][1] += p1;
                        float w0 = p0, w1 = p1;
                        if (KIND == FP8) {
                            w0 = ex2(x0 + av[tg][hf] - M0);
                            if (NI == 2) w1 = ex2(x1 + av[tg][hf] - M1);
                        }
                        if (KIND == FP8) {
                            pf[tg][nt][hf] = transpose8x8(pack2<false>(w0, w1));
                        } else {
                            const uint32_t hi = pack2_below<KIND == BF16>(w0, w1);
                            float r[2];
                            unpack2<KIND == BF16>(hi, r);
                            pf[tg][nt][hf] = transpose8x8(hi);
                            pl[tg][nt][hf] = transpose8x8(pack2<KIND == BF16>(w0 - r[0], w1 - r[1]));
                        }
                    }
            }
            // values
#pragma unroll
            for (int tg = 0; tg < TG; ++tg)
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    // tokens (rows of the fragment) 2t, 2t + 1, 2t + 8, 2t + 9
                    uint32_t v0[4], v1[4], v2[4], v3[4];
                    const uint32_t at = cur + 16 * tg * RB + c * 128;
                    if (VW == 4) {
                        uint4 x0, x1, x2, x3;
                        if constexpr (DIRECT) {
                            x0 = vr[tg][0][c], x1 = vr[tg][1][c], x2 = vr[tg][2][c], x3 = vr[tg][3][c];
                        } else {
                            x0 = lds16(at + at_v[0]), x1 = lds16(at + at_v[1]);
                            x2 = lds16(at + at_v[0] + 8 * RB), x3 = lds16(at + at_v[1] + 8 * RB);
                        }
                        v0[0] = x0.x, v0[1] = x0.y, v0[2] = x0.z, v0[3] = x0.w;
                        v1[0] = x1.x, v1[1] = x1.y, v1[2] = x1.z, v1[3] = x1.w;
                        v2[0] = x2.x, v2[1] = x2.y, v2[2] = x2.z, v2[3] = x2.w;
                        v3[0] = x3.x, v3[1] = x3.y, v3[2] = x3.z, v3[3] = x3.w;
                    } else {
                        const uint2 x0 = lds8(at + at_v[0]), x1 = lds8(at + at_v[1]);
                        const uint2 x2 = lds8(at + at_v[0] + 8 * RB), x3 = lds8(at + at_v[1] + 8 * RB);
                        v0[0] = x0.x, v0[1] = x0.y, v1[0] = x1.x, v1[1] = x1.y;
                        v2[0] = x2.x, v2[1] = x2.y, v3[0] = x3.x, v3[1] = x3.y;
                    }
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        if (KIND == FP8) {
                            uint32_t f[2][4];      // [tokens 2t, 2t+1 | 2t+8, 2t+9][element of the word]
                            e4m3x4_to_h2x2(prmt(v0[w], v1[w], 0x5140), f[0][0], f[0][1]);
                            e4m3x4_to_h2x2(prmt(v0[w], v1[w], 0x7362), f[0][2], f[0][3]);
                            e4m3x4_to_h2x2(prmt(v2[w], v3[w], 0x5140), f[1][0], f[1][1]);
                            e4m3x4_to_h2x2(prmt(v2[w], v3[w], 0x7362), f[1][2], f[1][3]);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int i = 0; i < 2; ++i)
                                    mma<false>(o[nt][(c * VW + w) * 2 + i], f[0][2 * i], f[0][2 * i + 1], f[1][2 * i],
                                               f[1][2 * i + 1], pf[tg][nt][0], pf[tg][nt][1]);
                        } else {
                            const uint32_t a0 = prmt(v0[w], v1[w], 0x5410), a1 = prmt(v0[w], v1[w], 0x7632);
                            const uint32_t a2 = prmt(v2[w], v3[w], 0x5410), a3 = prmt(v2[w], v3[w], 0x7632);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma<KIND == BF16>(o[nt][c * VW + w], a0, a1, a2, a3, pf[tg][nt][0], pf[tg][nt][1]);
                                mma<KIND == BF16>(o[nt][c * VW + w], a0, a1, a2, a3, pl[tg][nt][0], pl[tg][nt][1]);
                            }
                        }
                    }
                }
            if constexpr (DIRECT) load_v(t0 + UNIT, lines);
            lines = lines_next;
        }

        // ---- join the warps -----------------------------------------------------------------------
        copies_wait<0>();
        const bool any = __any_sync(0xffffffffu, DIRECT ? live >> 31 : seen);
        __syncthreads();                 // the buffers' memory changes hands
        if (lane == 0) sm.any[warp] = any;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int h = HP == 4 ? t : nt * 8 + 2 * t + i;
                float s = l[nt][i];
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
                if (g == 0) {
                    sm.m[warp][h] = m[nt][i];
                    sm.M[warp][h] = KIND == FP8 ? M[nt][i] : m[nt][i];
                    sm.l[warp][h] = s;
                }
#pragma unroll
                for (int k = 0; k < MT; ++k) {
                    // row tile k covers elements d, d + 1 of this lane's piece
                    const int d = (k / (GG::VE / 2)) * 8 * GG::VE + g * GG::VE + 2 * (k % (GG::VE / 2));
                    *reinterpret_cast<float2*>(&sm.o[warp][h][d]) = make_float2(o[nt][k][i], o[nt][k][2 + i]);
                }
            }
        __syncthreads();
        const bool whole = chunk == 0 && chunk_end == nu;
        int attended = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) attended |= sm.any[w];
        const int slot = 2 * blockIdx.x + (u == u0 ? 0 : 1);
        for (int i = tid; i < nh * (D / 2); i += kThreads) {
            const int h = i / (D / 2), d = 2 * (i - h * (D / 2));
            float mm = -INFINITY, MM = -INFINITY, ll = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                mm = fmaxf(mm, sm.m[w][h]);
                MM = fmaxf(MM, sm.M[w][h]);
            }
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                ll += sm.l[w][h] * (sm.m[w][h] == -INFINITY ? 1.f : ex2(sm.m[w][h] - mm));
                const float f = sm.M[w][h] == -INFINITY ? 1.f : ex2(sm.M[w][h] - MM);
                y0 += sm.o[w][h][d] * f;
                y1 += sm.o[w][h][d + 1] * f;
            }
            if (whole) {
                // all scores -inf: l = 0 and the quotient is NaN, as the formula's;
                // no token at all: zeros
                const float f = (KIND == FP8 && MM != -INFINITY && mm != -INFINITY ? ex2(MM - mm) : 1.f) /
                                (attended ? ll : 1.f);
                y0 *= f;
                y1 *= f;
                const int64_t at = (row0 + h) * D + d;
                *reinterpret_cast<uint32_t*>(a.out + at) = bf ? pack2<true>(y0, y1) : pack2<false>(y0, y1);
                if (a.lse && d == 0) a.lse[row0 + h] = log_sum(mm, ll, kLift<KIND>);
            } else {
                const int64_t at = (int64_t)slot * HP + h;
                *reinterpret_cast<float2*>(a.rec_o + at * D + d) = make_float2(y0, y1);
                if (d == 0) a.rec_s[at] = make_float4(mm, MM, ll, attended ? 1.f : 0.f);
            }
        }
        if (a.desc && chunk == 0 && tid == 0) {
            // the CTA that holds a stream's first unit says how to join it
            // (never past the last CTA's records, even if a length grew under way)
            const int pieces = whole ? 0 : min(deal.cta_of(s_end - 1), (int)gridDim.x - 1) - (int)blockIdx.x + 1;
            const int4 d = make_int4((int)row0, nh, pieces, slot);
            if (a.per_stream) a.desc[b * HS + stream] = d;
            else if (!whole) a.desc[blockIdx.x] = d;
        }
        u += chunk_end - chunk;
        __syncthreads();
    }
}

constexpr int kJoinMost = 512;       // threads of a joining block, at most

// Joins the pieces of one split stream for one head: piece 0 is record
// `first`, piece j > 0 the first record of the j-th CTA after it.  A warp
// takes 32 pieces at a time, a lane the maxima of one and D / 32 elements of
// every row; the rows' loads go out before the weights are known.  Up to 8
// pieces are one warp's work, without a barrier; more are dealt to all warps
// of the block, whose sums meet in shared memory.  (One chain of rescaled sums
// took 121 us for 278 pieces; with block-wide weights 16 sequences of 2K took
// 5 us longer than this.)
template <int D>
__global__ void __launch_bounds__(kJoinMost) join_kernel(const __grid_constant__ AttendArgs a, int HP, bool fp8) {
    constexpr int VE = D / 32, BATCH = 8;
    __shared__ float so[kJoinMost / 32][D];
    __shared__ float ss[kJoinMost / 32][4];
    await_predecessor();
    const int4 ds = a.desc[blockIdx.x];
    const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (ds.z == 0 || h >= ds.y) return;
    const bool alone = ds.z <= 8;
    if (alone && warp > 0) return;
    const int warps = alone ? 1 : blockDim.x >> 5;
    const int cta = ds.w >> 1, mine = (ds.z - warp + warps - 1) / warps;
    auto record = [&](int i) {
        const int j = warp + i * warps;
        return (int64_t)(j == 0 ? ds.w : 2 * (cta + j)) * HP + h;
    };
    struct alignas(4 * (VE < 4 ? VE : 4)) Row {
        float v[VE];
    };
    float m = -INFINITY, M = -INFINITY, l = 0.f, any = 0.f, o[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) o[e] = 0.f;
    for (int i0 = 0; i0 < mine; i0 += 32) {
        const int n = min(32, mine - i0);
        float4 s = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
        if (lane < n) s = a.rec_s[record(i0 + lane)];
        Row r[BATCH];
        auto load = [&](int i1) {
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
                if (i1 + i < n) r[i] = *reinterpret_cast<const Row*>(a.rec_o + record(i0 + i1 + i) * D + lane * VE);
        };
        load(0);
        float mn = s.x, Mn = s.y;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) {
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, k));
            Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, k));
        }
        mn = fmaxf(m, mn);
        Mn = fmaxf(M, Mn);
        const float fl = m == -INFINITY ? 1.f : ex2(m - mn), fo = M == -INFINITY ? 1.f : ex2(M - Mn);
        l = l * fl + s.z * (s.x == -INFINITY ? 1.f : ex2(s.x - mn));
        any = fmaxf(any, s.w);
        const float w = s.y == -INFINITY ? 1.f : ex2(s.y - Mn);
#pragma unroll
        for (int e = 0; e < VE; ++e) o[e] *= fo;
        for (int i1 = 0; i1 < n; i1 += BATCH) {
            if (i1) load(i1);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, i1 + i);
                if (i1 + i < n) {
#pragma unroll
                    for (int e = 0; e < VE; ++e) o[e] = fmaf(r[i].v[e], wi, o[e]);
                }
            }
        }
        m = mn;
        M = Mn;
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
    any = __any_sync(0xffffffffu, any != 0.f) ? 1.f : 0.f;
    if (!alone) {
#pragma unroll
        for (int e = 0; e < VE; ++e) so[warp][lane * VE + e] = o[e];
        if (lane == 0) {
            ss[warp][0] = m;
            ss[warp][1] = M;
            ss[warp][2] = l;
            ss[warp][3] = any;
        }
        __syncthreads();
        if (warp > 0) return;
        float mm = -INFINITY, MM = -INFINITY, ll = 0.f;
        for (int w = 0; w < warps; ++w) {
            mm = fmaxf(mm, ss[w][0]);
            MM = fmaxf(MM, ss[w][1]);
            any = fmaxf(any, ss[w][3]);
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) o[e] = 0.f;
        for (int w = 0; w < warps; ++w) {
            ll += ss[w][2] * (ss[w][0] == -INFINITY ? 1.f : ex2(ss[w][0] - mm));
            const float x = ss[w][1] == -INFINITY ? 1.f : ex2(ss[w][1] - MM);
#pragma unroll
            for (int e = 0; e < VE; ++e) o[e] = fmaf(so[w][lane * VE + e], x, o[e]);
        }
        m = mm;
        M = MM;
        l = ll;
    }
    const float f = (fp8 && M != -INFINITY && m != -INFINITY ? ex2(M - m) : 1.f) / (any != 0.f ? l : 1.f);
    uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + (int64_t)(ds.x + h) * D) + lane * (VE / 2);
#pragma unroll
    for (int e = 0; e < VE; e += 2)
        dst[e / 2] = a.c.bf16 ? pack2<true>(o[e] * f, o[e + 1] * f) : pack2<false>(o[e] * f, o[e + 1] * f);
    if (a.lse && lane == 0) a.lse[ds.x + h] = log_sum(m, l, fp8 || !a.c.bf16 ? kLift<F16> : kLift<BF16>);
}

// Streams of up to so many units stay whole, a CTA each: no records, no second
// launch, and no CTA that starts on one short stream after another.  A few
// streams (us whole / split, 2 kv heads of 64): 256 tokens 5.2 / 6.6, 384 6.3 /
// 6.6, 512 7.2 / 6.6.  More streams than SMs (sequences of up to 500 tokens, 8
// kv heads of 128, f16): 24 of them 13.7 / 15.7, 64 22.0 / 28.5 (all of 500:
// 34.0 / 30.2), 128 34.8 / 48.0; up to 1000 tokens, 16 units: 64 35.5 / 37.3
// (60.2 / 49.6).  Four waves of streams balance by themselves: 256 of up to
// 1000 tokens 102 / 110.
constexpr int kWholeFew = 4, kWholeUnits = 9, kWholeMany = 16;

struct Plan {
    int hp, ht, unit, wave, waves, ctas, streams;
    bool split, per_stream;
    size_t bytes, off_s, off_d;
};

using Kernel = void (*)(const AttendArgs);

template <int D, int HP, int KIND>
void entry(Kernel& k, size_t& smem) {
    k = attend_kernel<D, HP, KIND>;
    smem = smem_bytes<D, HP, KIND>();
}

template <int D, int HP>
void entry_h(int kind, Kernel& k, size_t& smem) {
    switch (kind) {
        case F16: entry<D, HP, F16>(k, smem); break;
        case BF16: entry<D, HP, BF16>(k, smem); break;
        default: entry<D, HP, FP8>(k, smem); break;
    }
}

template <int D>
void entry_d(int hp, int kind, Kernel& k, size_t& smem) {
    if (hp == 4) entry_h<D, 4>(kind, k, smem);
    else if (hp == 8) entry_h<D, 8>(kind, k, smem);
    else if constexpr (D != 256) entry_h<D, 16>(kind, k, smem);
}

int kind_of(const FkvPagedCache* c) { return c->fp8 ? FP8 : c->bf16 ? BF16 : F16; }

// SMs of the current device (148 where there is none, for sizing)
int sm_count() {
    static std::atomic<int> memo[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return 148;
    }
    if ((n = memo[dev].load(std::memory_order_relaxed)) != 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        return 148;
    }
    memo[dev].store(n, std::memory_order_relaxed);
    return n;
}

// The kernels' shared memory limit is raised on their first use on a device.
int raise_smem(Kernel k, size_t smem) {
    static std::mutex mu;
    static struct { Kernel k; int dev; } memo[1024];
    static int used = 0;
    int dev = 0;
    FKV_CUDA_CHECK(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < used; ++i)
        if (memo[i].k == k && memo[i].dev == dev) return FKV_OK;
    FKV_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (used < 1024) memo[used++] = {k, dev};
    return FKV_OK;
}

// query heads of a group that a CTA takes together (16 heads' accumulators of 256
// do not fit the registers)
int heads_of(int G, int D) { return G <= 4 ? 4 : G <= 8 || D == 256 ? 8 : 16; }

int make_plan(const FkvPagedCache* c, int Hq, int pshift, Plan* p) {
    const int G = Hq / c->Hk;
    p->hp = heads_of(G, c->D);
    p->ht = (G + p->hp - 1) / p->hp;
    const int es = c->fp8 ? 1 : 2;
    p->unit = kWarps * 16 * (c->D * es >= 256 ? 1 : 2);      // Geo::UNIT
    const int64_t reach = (int64_t)c->width << pshift;
    const int64_t units = (reach + 15 + p->unit - 1) / p->unit;
    const int64_t streams = (int64_t)c->B * c->Hk * p->ht;
    FKV_REQUIRE(streams * std::max<int64_t>(units, 1) < INT_MAX / 2 && (int64_t)c->B * Hq < INT_MAX,
                FKV_ERR_UNSUPPORTED, "fkv_paged_attend: %lld streams of %lld tokens are too many",
                (long long)streams, (long long)reach);
    p->streams = (int)streams;
    const int per_sm = c->D == 256 || p->hp == 16 ? 2 : 3;      // kPerSm
    const int ctas = per_sm * sm_count();
    const int64_t most = std::max<int64_t>(1, streams * std::max<int64_t>(units, 1));
    p->split = units > (streams >= 4 * (int64_t)ctas ? kWholeMany : streams > sm_count() ? kWholeUnits : kWholeFew);
    p->wave = p->split ? (int)std::min<int64_t>(ctas, most) : std::max(p->streams, 1);
    p->waves = !p->split || !c->fp8 || most < (int64_t)ctas * kUnits2 ? 1 : most < (int64_t)ctas * kUnits3 ? 2 : 3;
    p->ctas = p->wave * p->waves;
    p->per_stream = p->split && p->streams <= p->ctas;
    const size_t recs = 2 * (size_t)p->ctas * p->hp;
    p->off_s = recs * c->D * sizeof(float);
    p->off_d = p->off_s + recs * sizeof(float4);
    p->bytes = p->split ? p->off_d + (size_t)std::max(p->ctas, 1) * sizeof(int4) : 0;
    return FKV_OK;
}

}  // namespace

extern "C" size_t fkv_paged_attend_workspace_bytes(const FkvPagedCache* c, int32_t Hq) {
    int pshift = 0;
    Plan p;
    FkvPagedCache s;
    if (c == nullptr) return 0;
    s = *c;
    if (s.D != 64 && s.D != 128 && s.D != 256) return 0;
    if (s.page < 8 || s.page > 256 || (s.page & (s.page - 1)) || s.Hk < 1 || s.B < 0 || s.width < 0) return 0;
    while ((1 << pshift) < s.page) ++pshift;
    if (Hq < 1 || Hq % s.Hk != 0 || ((int64_t)s.width << pshift) > 1 << 30) return 0;
    return make_plan(&s, Hq, pshift, &p) == FKV_OK ? p.bytes : 0;
}

extern "C" int fkv_paged_attend(const FkvPagedCache* c, int32_t Hq, float scale, int32_t window,
                                const uint16_t* q, uint16_t* out, float* lse, void* workspace,
                                size_t workspace_bytes, void* stream) {
    int pshift = 0;
    int rc = fkv::paged_check(c, "fkv_paged_attend", &pshift);
    if (rc != FKV_OK) return rc;
    FKV_REQUIRE(Hq >= 1 && Hq % c->Hk == 0, FKV_ERR_INVALID,
                "fkv_paged_attend: Hq=%d is not a multiple of Hk=%d", Hq, c->Hk);
    FKV_REQUIRE(window >= 0, FKV_ERR_INVALID, "fkv_paged_attend: window %d", window);
    if (c->B == 0) return FKV_OK;
    FKV_REQUIRE(q && out, FKV_ERR_INVALID, "fkv_paged_attend: NULL pointer");
    FKV_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0, FKV_ERR_INVALID,
                "fkv_paged_attend: q / out not 16-byte aligned");
    const int G = Hq / c->Hk, hp = heads_of(G, c->D);
    Kernel k = nullptr;
    size_t smem = 0;
    if (c->D == 64) entry_d<64>(hp, kind_of(c), k, smem);
    else if (c->D == 128) entry_d<128>(hp, kind_of(c), k, smem);
    else entry_d<256>(hp, kind_of(c), k, smem);
    // a row's number is kept in 32 bits (2^32 rows of 64 bytes are more than the device holds)
    FKV_REQUIRE(((int64_t)c->n_pages * c->Hk << pshift) < 0xFFFFFFFFll, FKV_ERR_UNSUPPORTED,
                "fkv_paged_attend: %d pages of %d x %d rows are too many", c->n_pages, c->Hk, c->page);
    Plan p;
    rc = make_plan(c, Hq, pshift, &p);
    if (rc != FKV_OK) return rc;
    rc = raise_smem(k, smem);
    if (rc != FKV_OK) return rc;
    FKV_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes), FKV_ERR_INVALID,
                "fkv_paged_attend: workspace of %zu bytes, %zu needed", workspace_bytes, p.bytes);
    FKV_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, FKV_ERR_INVALID,
                "fkv_paged_attend: workspace not 16-byte aligned");
    AttendArgs a;
    a.c = *c;
    if (c->n_pages == 0) {        // copies of no bytes still name an address
        a.c.k_pages = a.c.v_pages = const_cast<uint16_t*>(q);
        a.c.k_scale = a.c.v_scale = reinterpret_cast<float*>(const_cast<uint16_t*>(q));
    }
    a.q = q;
    a.out = out;
    a.lse = lse;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    a.rec_o = p.split ? reinterpret_cast<float*>(ws) : nullptr;
    a.rec_s = p.split ? reinterpret_cast<float4*>(ws + p.off_s) : nullptr;
    a.desc = p.split ? reinterpret_cast<int4*>(ws + p.off_d) : nullptr;
    a.Hq = Hq;
    a.G = G;
    a.HT = p.ht;
    a.pshift = pshift;
    a.window = window;
    a.per_stream = p.per_stream;
    a.wave = p.wave;
    a.waves = p.waves;
    a.sl2 = scale * 1.4426950408889634f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // launched early only where the grid leaves room beside its predecessor:
    // 8.4 -> 7.3 us for 1K tokens, but 508 -> 526 for 64 x 32K, whose CTAs then
    // settled unevenly beside the last joining blocks
    FKV_CUDA_CHECK(fkv::launch_beside(k, dim3(p.ctas), kThreads, smem, s, p.ctas <= sm_count(), a));
    if (!p.split) return FKV_OK;
    const dim3 grid(p.per_stream ? p.streams : p.ctas, std::min(G, hp));
    // many streams have few pieces each; blocks for many would wait for room
    // (16 sequences of 2K, 4 pieces a stream: 29.7 us with 512 threads, 25.6 with 128)
    const int threads = p.ctas <= 8 * p.streams ? 128 : kJoinMost;
    const bool fp8 = c->fp8 != 0;
    FKV_CUDA_CHECK(c->D == 64    ? fkv::launch_beside(join_kernel<64>, grid, threads, 0, s, true, a, hp, fp8)
                   : c->D == 128 ? fkv::launch_beside(join_kernel<128>, grid, threads, 0, s, true, a, hp, fp8)
                                 : fkv::launch_beside(join_kernel<256>, grid, threads, 0, s, true, a, hp, fp8));
    return FKV_OK;
}
