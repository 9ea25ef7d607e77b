// Shared pieces of the paged-cache kernels (trx_paged.cu, trx_paged_tc.cu): the launch arguments, the
// sequences' geometry, and the division of the attention work among CTAs.
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "trx_common.cuh"
#include "trx_internal.h"

namespace trx {

constexpr int kPagedMaxSeq = 1024;  // sequences of one plan (the kernels keep a prefix of them in shared memory)

// The pools as [8 slots][slot of 8][64 dims of a head][dim], one box a page's (or a tile's part of it) slots of
// one kv head: a single copy lays them as groups of 8 slots, in each group the head's 64-dim blocks of 8 rows
// x 128 bytes.  (A box per 64 dims cost 80 cycles of the producer each: 1,300 for a tile of head dim 256 in
// pages of 16.)  The queries (16-bit ones of the tcgen05 kernel) as [rows][n_kv][rep][head_dim].
struct PgMaps {
    CUtensorMap k, v, q;
};

template <int HD>
inline bool pg_encode_pools(PgMaps &maps, const PgAttnArgs &A, uint32_t box_rows) {
    const uint64_t pitch = (uint64_t)A.Hkv * HD * 2, groups = ((uint64_t)A.n_pages << A.page_shift) / 8;
    const uint64_t dims[4] = {64, 8, (uint64_t)A.Hkv * HD / 64, groups}, strides[3] = {pitch, 128, 8 * pitch};
    const uint32_t box[4] = {64, 8, HD / 64, box_rows / 8};
    return encode_map_16bit_4d(&maps.k, A.kp, dims, strides, box) && encode_map_16bit_4d(&maps.v, A.vp, dims, strides, box);
}

__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void load_box4(uint32_t dst, const void *map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// Bounded wait on an mbarrier phase by the SM's own clock (2^29 cycles, about 0.3 s; then
// TRX_DEV_TIMEOUT).
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, uint32_t *err) {
    if (mbar_try_wait_s(bar, parity)) return true;
    const long long t0 = clock64();
    do {
#pragma unroll 1
        for (int i = 0; i < 16; ++i)
            if (mbar_try_wait_s(bar, parity)) return true;
    } while (clock64() - t0 < (1ll << 29));
    if (err && (threadIdx.x & 31) == 0) atomicOr(err, TRX_DEV_TIMEOUT);
    return false;
}

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename CT> struct PgIsBf16 { static constexpr bool value = false; };
template <> struct PgIsBf16<__nv_bfloat16> { static constexpr bool value = true; };

// Softmax weights that are split into two fp16 parts are scaled by 2^15 first (their sum too, so the quotient is the
// same).  The parts' last place is 2^-24 at the least, so they keep 2^-22 of a scaled weight down to 2^-3 and are within
// 2^-25 below.  The largest is 2^15, or in the tcgen05 kernel, whose maxima are whole numbers rounded up, above 2^14:
// 2^-22 of a weight down to 2^-17 of the row's largest, and 2^-39 of the largest below, where unscaled ones would keep
// 2^-25: too little where the largest weight meets values near 0.
constexpr float kSplitBits = 15.f, kSplitScale = 32768.f;
// Single fp16 weights are scaled too: by 2^15 in the mma.sync kernel, by 2^7 in the tcgen05 kernel, whose weights reach
// 2^8 before.  They keep 2^-11 of themselves down to 2^-29 (2^-21) of the row's largest, and 2^-40 (2^-32) of the
// largest below, where unscaled ones would lose bits from 2^-14 on and vanish at 2^-25.  bf16 ones have the range.
template <typename CT>
constexpr float kHalfBits = PgIsBf16<CT>::value ? 0.f : 7.f;

// One sequence of an attention launch: its new rows [row0, row0 + n) at positions [p0, p0 + n).
struct PgSeq {
    int row0, n, p0;
};

// The sequence's rows and positions, or n = 0 for one whose offsets or length are out of range
// (bad is then set; nothing outside the buffers is read or written for it).
__device__ __forceinline__ PgSeq pg_seq(const PgAttnArgs &A, int b, bool &bad) {
    PgSeq S{};
    const int c0 = A.cu[b], c1 = A.cu[b + 1], len = A.lens[b];
    // Compared before it is subtracted: no difference of what passes leaves 32 bits.
    if (c0 < 0 || c1 < c0 || c1 > A.max_rows || c1 - c0 > A.max_new || len < c1 - c0 ||
        (c1 > c0 && (long long)len > (long long)A.max_pages << A.page_shift)) {
        bad = true;
        return S;
    }
    S.row0 = c0;
    S.n = c1 - c0;
    S.p0 = len - S.n;
    return S;
}

// The key tiles (KT positions each) that query tile t of a sequence reads: tile index i < ns is the
// i-th sink tile, the rest are the tiles from w0 on.
struct PgRange {
    int ns, w0, cnt;
    __device__ __forceinline__ int tile(int i) const { return i < ns ? i : w0 + i - ns; }
};

__device__ __forceinline__ PgRange pg_range(const PgAttnArgs &A, const PgSeq &S, int t) {
    const int lo = S.p0 + t * A.tq, hi = S.p0 + min(S.n, (t + 1) * A.tq) - 1;
    PgRange R;
    R.w0 = A.window ? max(0, lo - A.window + 1) >> A.kt_shift : 0;
    R.ns = A.window ? min((A.sinks + (1 << A.kt_shift) - 1) >> A.kt_shift, R.w0) : 0;
    R.cnt = R.ns + (hi >> A.kt_shift) - R.w0 + 1;
    return R;
}

// Division of the work.  The (query tile, kv head, key tile) units of all sequences form one line,
// query tile major, key tile minor; G CTAs take N / G units each in order (the first N % G one more).
// An item is one (query tile, kv head); a CTA's range cuts it into pieces.  An item in one piece is
// finished by its CTA; the pieces of a cut item go to scratch as (max, sum, unnormalised output) and the
// CTA that arrives last joins them in the order of the CTAs, so that the result does not depend on
// timing.  Every CTA finds its own range by scanning the sequences' lengths: no launch in front, and
// nothing of the lengths has to be known on the host.
struct PgSched {
    long long N, per;          // units in all, and of every CTA
    int G, rem;                // CTAs that take part; the first rem have one unit more
    long long u0, u1;          // this CTA's units
    int b, t, kh, i;           // its first unit: sequence, query tile, kv head, index among the item's key tiles
};

struct PgSchedSmem {
    int qpre[kPagedMaxSeq + 1];  // query tiles of the sequences before b
    long long wsum[33];
    PgSched S;
    int bad;
};

// 64-bit quotient by the 32-bit one where it suffices.
__device__ __forceinline__ long long pg_div(long long a, long long b) {
    return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

// Block-wide exclusive sum of v (blockDim a multiple of 32, at most 1024 threads); total in *tot.
__device__ __forceinline__ long long pg_block_scan(long long v, long long *wsum, long long *tot) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    if (warp == 0) {
        long long w = lane < nw ? wsum[lane] : 0;
        const long long w0 = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        if (lane < nw) wsum[lane] = w - w0;
        if (lane == 31) wsum[32] = w;
    }
    __syncthreads();
    const long long r = wsum[warp] + x - v;
    *tot = wsum[32];
    __syncthreads();
    return r;
}

// The sequence that query tile q belongs to.
__device__ __forceinline__ int pg_find(const int *qpre, int nseq, int q) {
    int lo = 0, hi = nseq;  // qpre[lo] <= q < qpre[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (qpre[mid] <= q) lo = mid; else hi = mid;
    }
    return lo;
}

// This CTA's range of N units (min_units: CTAs take part as long as each gets this many).
__device__ __forceinline__ void pg_share(PgSched &S, long long N, int min_units) {
    const long long gmax = pg_div(N + min_units - 1, min_units);
    S.N = N;
    S.G = (int)(gmax < (long long)gridDim.x ? gmax : (long long)gridDim.x);
    S.per = S.G ? pg_div(N, S.G) : 0;
    S.rem = (int)(N - S.per * S.G);
    const int c = (int)blockIdx.x;
    S.u0 = c * S.per + min(c, S.rem);
    S.u1 = c < S.G ? S.u0 + S.per + (c < S.rem ? 1 : 0) : S.u0;
}

// The CTA that owns unit x.
__device__ __forceinline__ int pg_owner(const PgSched &S, long long x) {
    const long long big = (S.per + 1) * S.rem;
    return (int)(x < big ? pg_div(x, S.per + 1) : S.rem + pg_div(x - big, S.per));
}

// Units of query tile q, its sequence b and place t there.
__device__ __forceinline__ long long pg_units(const PgAttnArgs &A, const int *qpre, int q, int &b, int &t, PgRange &R) {
    bool ignore = false;
    b = pg_find(qpre, A.nseq, q);
    t = q - qpre[b];
    R = pg_range(A, pg_seq(A, b, ignore), t);
    return (long long)R.cnt * A.Hkv;
}

__device__ __forceinline__ void pg_first(PgSched &S, long long at, int b, int t, int cnt) {
    const long long d = S.u0 - at, kh = pg_div(d, cnt);
    S.b = b;
    S.t = t;
    S.kh = (int)kh;
    S.i = (int)(d - kh * cnt);
}

// Every thread of the block: fills sm.S (see PgSched).  Up to 32 sequences with up to 32 query tiles (a
// decode step) are one warp's work; else the block scans.
__device__ __forceinline__ void pg_schedule(const PgAttnArgs &A, PgSchedSmem &sm, int min_units, uint32_t *err) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31;
    if (A.nseq <= 32) {
        if (tid < 32) {
            bool bad = false;
            PgSeq seq{};
            if (lane < A.nseq) seq = pg_seq(A, lane, bad);
            const int q = (seq.n + A.tq - 1) / A.tq;
            if (__any_sync(0xffffffffu, bad) && lane == 0 && blockIdx.x == 0) atomicOr(err, TRX_DEV_RANGE);
            const bool single = !__any_sync(0xffffffffu, q > 1);  // at most one query tile each: a lane has its own
            int x = q;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            sm.qpre[lane + 1] = x;  // beyond nseq: the total again
            if (lane == 0) sm.qpre[0] = 0;
            __syncwarp();
            const int NQ = sm.qpre[32];
            if (NQ <= 32) {
                int b = 0, t = 0;
                PgRange R{};
                long long u = 0;
                if (single) {
                    b = lane;
                    if (q) {
                        R = pg_range(A, seq, 0);
                        u = (long long)R.cnt * A.Hkv;
                    }
                } else if (lane < NQ) {
                    u = pg_units(A, sm.qpre, lane, b, t, R);
                }
                long long v = u;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long y = __shfl_up_sync(0xffffffffu, v, o);
                    if (lane >= o) v += y;
                }
                PgSched S;
                pg_share(S, __shfl_sync(0xffffffffu, v, 31), min_units);
                if (lane == 0) sm.S = S;
                __syncwarp();
                if (S.u0 < S.u1 && v - u <= S.u0 && S.u0 < v) pg_first(sm.S, v - u, b, t, R.cnt);
            }
        }
        __syncthreads();
        if (sm.qpre[32] <= 32) return;
    } else {
        if (tid == 0) sm.bad = 0;
        __syncthreads();
        long long carry = 0;
        bool bad = false;
        for (int b0 = 0; b0 < A.nseq; b0 += nt) {
            const int b = b0 + tid;
            int q = 0;
            if (b < A.nseq) q = (pg_seq(A, b, bad).n + A.tq - 1) / A.tq;
            long long tot;
            const long long ex = pg_block_scan(q, sm.wsum, &tot);
            if (b < A.nseq) sm.qpre[b] = (int)(carry + ex);
            carry += tot;
        }
        if (tid == 0) sm.qpre[A.nseq] = (int)carry;
        if (bad) sm.bad = 1;
        __syncthreads();
        if (tid == 0 && sm.bad && blockIdx.x == 0) atomicOr(err, TRX_DEV_RANGE);
    }
    const int NQ = sm.qpre[A.nseq];
    int b = 0, t = 0;
    PgRange R{};
    long long u = 0, at = 0, N = 0;  // of this thread's query tile in the last round
    for (int q0 = 0; q0 < NQ; q0 += nt) {
        long long tot;
        u = q0 + tid < NQ ? pg_units(A, sm.qpre, q0 + tid, b, t, R) : 0;
        at = N + pg_block_scan(u, sm.wsum, &tot);
        N += tot;
    }
    if (tid == 0) pg_share(sm.S, N, min_units);
    __syncthreads();
    const long long u0 = sm.S.u0;
    if (u0 < sm.S.u1) {
        if (NQ <= nt) {
            if (at <= u0 && u0 < at + u) pg_first(sm.S, at, b, t, R.cnt);
        } else {
            long long base = 0;
            for (int q0 = 0; q0 < NQ && base <= u0; q0 += nt) {
                long long tot;
                u = q0 + tid < NQ ? pg_units(A, sm.qpre, q0 + tid, b, t, R) : 0;
                at = base + pg_block_scan(u, sm.wsum, &tot);
                if (at <= u0 && u0 < at + u) pg_first(sm.S, at, b, t, R.cnt);
                base += tot;
            }
        }
    }
    __syncthreads();
}

// A role's walk along its CTA's pieces.
struct PgWalk {
    PgSeq q;
    PgRange R;
    int b, t, kh, i0, i1;    // this piece: key tiles i0..i1-1 of the item's R.cnt
    long long u, u1;         // units before the end of this piece, the end of the range

    __device__ __forceinline__ void load(const PgAttnArgs &A) {
        bool ignore = false;
        q = pg_seq(A, b, ignore);
        R = pg_range(A, q, t);
    }
    __device__ __forceinline__ void cut() {
        const long long left = u1 - u;
        i1 = (int)(left < R.cnt - i0 ? i0 + left : R.cnt);
        u += i1 - i0;
    }
    // false: the CTA has no units.
    __device__ __forceinline__ bool start(const PgAttnArgs &A, const PgSched &S) {
        if (S.u0 >= S.u1) return false;
        b = S.b;
        t = S.t;
        kh = S.kh;
        i0 = S.i;
        u = S.u0;
        u1 = S.u1;
        load(A);
        cut();
        return true;
    }
    __device__ __forceinline__ bool next(const PgAttnArgs &A) {
        if (u >= u1) return false;
        i0 = 0;
        if (++kh == A.Hkv) {
            kh = 0;
            if (++t * A.tq >= q.n) {
                t = 0;
                bool ignore = false;
                do { ++b; } while (b < A.nseq && pg_seq(A, b, ignore).n == 0);
                if (b >= A.nseq) return false;
            }
            load(A);
        }
        cut();
        return true;
    }
    __device__ __forceinline__ bool whole() const { return i0 == 0 && i1 == R.cnt; }
    __device__ __forceinline__ int rows(const PgAttnArgs &A) const { return min(q.n - t * A.tq, A.tq) * A.rep; }
};

// Is key position k hidden from the query at position p?
__device__ __forceinline__ bool pg_hidden(int k, int p, int window, int sinks) {
    return k > p || (window && p - k >= window && k >= sinks);
}

template <typename CT> struct PgCvt;
template <> struct PgCvt<__half> {
    static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        uint32_t u;
        memcpy(&u, &h, 4);
        return u;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        __half2 h;
        memcpy(&h, &u, 4);
        return __half22float2(h);
    }
};
template <> struct PgCvt<__nv_bfloat16> {
    static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        uint32_t u;
        memcpy(&u, &h, 4);
        return u;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        __nv_bfloat162 h;
        memcpy(&h, &u, 4);
        return __bfloat1622float2(h);
    }
};

}  // namespace trx
