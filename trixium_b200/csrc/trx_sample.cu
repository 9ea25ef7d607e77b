// Sampling of one token per row of logits (sm_100a): temperature, top-k, top-p and min-p from given
// random numbers, in one launch.
//
// Order: descending by logit, ties by index.  Weights w = exp((x - max) / T), held as integers of steps
// 2^-S (S = 62 - ceil(log2 V), at most 50), each within 2^-30 of itself, so that every sum is exact
// whatever its order: the borders of top-p and of the draw do not move with the division of the work.
// (32-bit sums will not do: with 152k tokens they are off by more than many tokens' whole share.)
//
// A row is held by a cluster of C thread blocks, its logits in their shared memory (a row too long for that
// is read again in every pass); distributed shared memory joins the blocks' parts:
//  1. max (and with it the greedy token) and min.
//  2. top-k / top-p: counts over 512 equal steps of max - x, down to where weights round to 0.  Equal steps
//     order the tokens like their logits and spread them better than the bits of a float would.
//  3. top-k: the step with the k-th token follows from the counts.  If few tokens lie up to it (at most
//     kList), block 0 takes them over, ranks them, cuts at k, p and min-p, and draws.  Otherwise the step
//     is narrowed by histograms over the keys' bits until one key is left: the cut is that key and how many of
//     its ties (in index order) are kept.
//     top-p over more than that: the steps' counts and mean places tell, to a fraction of a step, where the
//     nucleus ends; one pass then sums exactly the weights of the row, above that step and in it, and
//     collects the step's tokens, which block 0 ranks (or the step is narrowed, if they are too many).  Should
//     the end lie in a neighbouring step after all, the pass is repeated there.
//  4. Unless block 0 has drawn: the draw over the whole row: each warp sums its contiguous part, the
//     parts' prefix tells which warp holds the token, and that warp sums its part again, a lane at a time.
// Bound by the arithmetic of the weights (about 50 instructions each, twice 32 bits of sum) and of the counts, and
// by the cluster's barriers: in a graph one row of 151,936 takes 17 us, 32 of them 51 us (54 to 65 from Python, by their
// settings; 19 MB, the bytes alone 3 us), 333 rows of 32,003 68 us.  A cluster per row keeps the row on chip between
// its three to five passes.
#include <cfloat>
#include <cstdint>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "trx_common.cuh"
#include "trx_internal.h"

namespace trx {
namespace {
namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreadsS = 512;
constexpr int kWarpsS = kThreadsS / 32;
constexpr int kBins = kThreadsS;  // a thread has one
constexpr int kList = 1024;
constexpr int kMaxCluster = 16;
constexpr size_t kCacheMax = 80 * 1024;  // a block's part of the row: two blocks fit an SM

// Order-preserving bits of a float.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float val_of(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // key_of(-inf)

template <typename T> __device__ __forceinline__ float load_f(const T *p);
template <> __device__ __forceinline__ float load_f<float>(const float *p) { return *p; }
template <> __device__ __forceinline__ float load_f<__half>(const __half *p) { return __half2float(*p); }
template <> __device__ __forceinline__ float load_f<__nv_bfloat16>(const __nv_bfloat16 *p) {
    return __bfloat162float(*p);
}

struct SmemS {
    uint2 tab[32];                   // 2^(i / 32) in steps of 2^-31: as a whole number, as a float
    uint32_t cnt[kBins];             // this block's histogram
    uint32_t mlo[kBins], mhi[kBins]; // its weights, 64 bits in two words; in step 2 mlo: the places within a step
    uint32_t tcnt[kBins];            // the cluster's histogram (every block forms it)
    u64 tmass[kBins];
    u64 list[kList], sorted[kList];  // block 0: gathered tokens (key << 32 | ~index)
    u64 best[kMaxCluster];           // every block's max, for the whole cluster
    uint32_t lo[kMaxCluster], hi[kMaxCluster];
    u64 sum[kMaxCluster][3];         // every block's weight: the row's, above a step, in it
    u64 wmass[kMaxCluster * kWarpsS];
    uint32_t wties[kMaxCluster * kWarpsS];
    u64 red[kWarpsS + 1], part[kWarpsS][3];
    double redd[kWarpsS + 1];
    uint32_t redu[kWarpsS + 1];
    int owner;
    uint32_t nlist, found, got, nall, base;  // nall: block 0, tokens handed over
    u64 base_cnt, base_mass;
    double est[kBins + 1];           // estimated running weight before a step
    uint32_t cut_key, cut_ties;
};

// Weight function of a row: round(2^((x - max) k) * 2^S) with k = log2(e) / T, in 32-bit operations only (64-bit
// floats took three times as long).  t = 32 (x - max) k as a sum of two floats: x - max with its exact
// rounding error, times k as two floats.  2^(t / 32) = 2^n * 2^(i / 32) * (1 + q), t = 32 n + i + r with |r| <= 1/2:
// 2^(i / 32) from the table in steps of 2^-31, q = 2^(r / 32) - 1 = y + y^2 / 2 + y^3 / 6 + y^4 / 24 with
// y = r ln2 / 32 <= 0.011 (the next term is below 2^-39), rounded at 2^-24 of itself: 2^-30 of the weight.
struct Weigh {
    float mx, kh, kl, lowest;  // 32 k in two floats; t below lowest rounds to 0
    u64 minw;                  // min_p * 2^S, rounded up
    int S;
    const uint2 *tab;
    __device__ __forceinline__ u64 operator()(float x) const {
        const float d = x - mx, c = d - x, dl = (x - (d - c)) - (mx + c);
        const float p = d * kh, t = fmaxf(p, lowest);  // lowest also for x = -inf
        const float tl = fmaf(d, kh, -p) + fmaf(d, kl, dl * kh);
        const float magic = 12582912.f, big = t + magic;  // the nearest whole number in its low bits
        const int n = __float_as_int(big) - __float_as_int(magic);
        const float r = (t - (big - magic)) + tl;
        const float y = r * (float)(0.6931471805599453 / 32);
        const float q = fmaf(y * y, fmaf(y, fmaf(y, 1.f / 24, 1.f / 6), 0.5f), y);
        const uint2 e = tab[n & 31];
        const uint32_t m = e.x + (uint32_t)__float2int_rn(q * __uint_as_float(e.y));
        const u64 w = ((u64)m << 31) >> (62 - S - (n >> 5));
        return x == mx ? 1ull << S : (p > lowest ? w : 0);
    }
    __device__ __forceinline__ bool enough(u64 w) const { return w >= minw; }
};

// Block-wide inclusive sums; every thread gets its own, and the total.
template <typename T>
__device__ __forceinline__ T block_incl(T v, T *red, T *tot) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    if (lane == 31) red[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const T w0 = lane < kWarpsS ? red[lane] : 0;
        T w = w0;
#pragma unroll
        for (int o = 1; o < kWarpsS; o <<= 1) {
            const T y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        if (lane < kWarpsS) red[lane] = w - w0;
        if (lane == kWarpsS - 1) red[kWarpsS] = w;
    }
    __syncthreads();
    v += red[warp];
    *tot = red[kWarpsS];
    __syncthreads();
    return v;
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ void add_mass(SmemS &sm, int b, u64 w) {
    const uint32_t lo = (uint32_t)w, old = atomicAdd(&sm.mlo[b], lo);
    const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
    if (hi) atomicAdd(&sm.mhi[b], hi);
}

template <typename T, bool CACHED>
__global__ void __launch_bounds__(kThreadsS, 2) sample_kernel(SampleArgs A, int S) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SmemS &sm = *reinterpret_cast<SmemS *>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / C, V = A.V;
    pdl_trigger();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // waited for before the first remote store
    if (tid < 32) {
        const double v = exp2((double)tid / 32) * 2147483648.0;
        sm.tab[tid] = make_uint2((uint32_t)(v + 0.5), __float_as_uint((float)v));
    }
    pdl_wait();
    const T *const x = reinterpret_cast<const T *>(A.x) + row * A.ld;
    // Temperatures below 2^-100 count as that (NaN as 0): 32 log2(e) / T and steps of T stay finite, and weights
    // change only where logits differ by less than 2^-94.
    const float t_in = A.temp[row], temp = t_in > 0.f ? fmaxf(t_in, 0x1p-100f) : 0.f;
    const float u = A.u[row], topp = A.top_p[row];
    const int k = A.top_k[row];
    // This warp's contiguous part, a multiple of 32 tokens; its e-th step of 32.
    const int part = ((V + C * kWarpsS - 1) / (C * kWarpsS) + 31) / 32 * 32;
    const int w0 = min(V, (rank * kWarpsS + warp) * part), w1 = min(V, w0 + part);
    float *const cache = reinterpret_cast<float *>(smem_raw + sizeof(SmemS)) + warp * part - w0;
    auto fetch = [&](int i) {  // NaN counts as -inf; -0 and 0 are equal (and one key)
        return __fadd_rn(fmaxf(load_f(x + i), -INFINITY), 0.f);
    };
    // 1. Max (the first of equal ones), min.
    float vmax = -INFINITY, vmin = INFINITY;
    int imax = 0x7fffffff;
    for (int i0 = w0 + lane; i0 < w0 + part; i0 += 32 * 20) {  // twenty loads in flight
        float v[20];
#pragma unroll
        for (int e = 0; e < 20; ++e) v[e] = i0 + 32 * e < w1 ? fetch(i0 + 32 * e) : -INFINITY;
#pragma unroll
        for (int e = 0; e < 20; ++e) {
            const int i = i0 + 32 * e;
            if (i < w0 + part) {
                if constexpr (CACHED) cache[i] = v[e];
                if (v[e] > vmax) {
                    vmax = v[e];
                    imax = i;
                }
                if (v[e] != -INFINITY) vmin = fminf(vmin, v[e]);
            }
        }
    }
    // f(index, logit) for every token of this thread (places behind the row: -inf), in index order by warp; a
    // thread reads only what it stored.
    auto each = [&](auto &&f) {
#pragma unroll 4
        for (int i = w0 + lane; i < w0 + part; i += 32) {
            if constexpr (CACHED)
                f(i, cache[i]);
            else
                f(i, i < w1 ? fetch(i) : -INFINITY);
        }
    };
    // The same four at a time: f(index of the first, logits), the next 32 tokens further on each.  Sums of weights
    // go this way: without branches between them four weights are worked on together.
    auto each4 = [&](auto &&f) {
        for (int i = w0 + lane; i < w0 + part; i += 128) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = i + 32 * e;
                if constexpr (CACHED)
                    v[e] = j < w0 + part ? cache[j] : -INFINITY;
                else
                    v[e] = j < w1 ? fetch(j) : -INFINITY;
            }
            f(i, v);
        }
    };
    {
        u64 best = ((u64)key_of(vmax) << 32) | (0xffffffffu - (uint32_t)imax);
        uint32_t lo = key_of(vmin);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const u64 b = __shfl_xor_sync(0xffffffffu, best, o);
            best = b > best ? b : best;
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        if (lane == 0) {
            sm.red[warp] = best;
            sm.redu[warp] = lo;
        }
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every block has started
        __syncthreads();
        if (warp == 0) {
            best = lane < kWarpsS ? sm.red[lane] : 0;
            lo = __reduce_min_sync(0xffffffffu, lane < kWarpsS ? sm.redu[lane] : 0xffffffffu);
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const u64 b = __shfl_xor_sync(0xffffffffu, best, o);
                best = b > best ? b : best;
            }
            if (lane < C) {
                *cluster.map_shared_rank(&sm.best[rank], lane) = best;
                *cluster.map_shared_rank(&sm.lo[rank], lane) = lo;
            }
        }
    }
    if (tid == 0) sm.got = sm.nall = 0;
    cluster.sync();
    u64 best = sm.best[0];
    uint32_t klo = sm.lo[0];
    for (int r = 1; r < C; ++r) {
        best = sm.best[r] > best ? sm.best[r] : best;
        klo = min(klo, sm.lo[r]);
    }
    const uint32_t kmax = (uint32_t)(best >> 32);
    const bool none = kmax <= kKeyNegInf, greedy = temp == 0.f || k == 1 || topp <= 0.f;
    const float minp = A.min_p[row];
    if (none || (greedy && (temp == 0.f || minp <= 1.f))) {
        if (rank == 0 && tid == 0) A.tokens[row] = none ? -1 : (int)(0xffffffffu - (uint32_t)best);
        return;
    }
    Weigh W;
    W.mx = val_of(kmax);
    const double k32 = 32 * 1.4426950408889634 / (double)temp;
    W.kh = (float)k32;
    W.kl = (float)(k32 - (double)W.kh);
    W.lowest = -32.f * (float)S;  // shifts stay below 64
    W.S = S;
    W.minw = minp <= 0.f ? 0 : (minp <= 1.f ? (u64)ceil((double)minp * (double)(1ull << S)) : ~0ull);
    W.tab = sm.tab;
    const bool need_k = k > 0 && k < V, need_p = topp < 1.f;
    uint32_t thr = 0;           // kept: keys above thr, and the first `ties` with key thr
    uint32_t ties = 0xffffffffu;
    if (need_k || need_p) {
        // 2. Counts over max - x.
        const float span = fminf(36.f * temp, W.mx - val_of(klo));
        // The last step ends short of kBins, so that only what rounds to no weight (or an infinity) is beyond.
        // Of spans so small that this would overflow (logits next to 0) the steps fill the first places only.
        const float step = span > 0.f && span < INFINITY ? fminf((kBins - 0.5f) / span, FLT_MAX) : 0.f;
        auto place = [&](float v) {  // in steps; kBins: beyond
            const float d = v == W.mx ? 0.f : W.mx - v;
            return fminf(d * step, (float)kBins);
        };
        auto bin_of = [&](float v) { return (int)place(v); };
        bool joined = false;
        auto clear = [&] {
            if (joined) cluster.sync();  // the other blocks have read the last one
            joined = false;
            sm.cnt[tid] = sm.mlo[tid] = sm.mhi[tid] = 0u;
            __syncthreads();
        };
        // The blocks' histograms into tcnt, tmass.
        auto join = [&] {
            cluster.sync();
            uint32_t n = 0;
            u64 m = 0;
            for (int r = 0; r < C; ++r) {
                const SmemS *const o = cluster.map_shared_rank(&sm, r);
                n += o->cnt[tid];
                if (need_p) m += ((u64)o->mhi[tid] << 32) + o->mlo[tid];
            }
            sm.tcnt[tid] = n;
            sm.tmass[tid] = m;
            joined = true;
        };
        // The first step whose running count reaches n, or whose running weight reaches target
        // (by_mass), with the count and weight before it (base_cnt, base_mass) and the count up to it (nlist);
        // kBins: none.  (A thread reads its own tcnt and tmass.)
        auto cross = [&](bool by_mass, u64 n, double target, u64 bc, u64 bm) {
            u64 tot;
            const u64 own = by_mass ? sm.tmass[tid] : sm.tcnt[tid], base = by_mass ? bm : bc;
            const u64 inc = base + block_incl<u64>(own, sm.red, &tot);
            if (tid == 0) sm.found = kBins;
            __syncthreads();
            if (by_mass ? (double)inc >= target : inc >= n) atomicMin(&sm.found, (uint32_t)tid);
            __syncthreads();
            const int f = (int)sm.found;
            if (f == tid) {
                sm.base_cnt = by_mass ? 0 : inc - own;
                sm.base_mass = by_mass ? inc - own : 0;
                sm.nlist = (uint32_t)inc;
            }
            __syncthreads();
            return f;
        };
        // Tokens of this block that are set aside in a pass, then handed to block 0's list (at most kList in all;
        // nall counts them all).
        u64 *const mine = rank ? sm.list : sm.sorted;
        auto set_aside = [&](int i, float v) {
            const uint32_t at = atomicAdd(&sm.got, 1u);
            if (at < kList) mine[at] = ((u64)key_of(v) << 32) | (0xffffffffu - (uint32_t)i);
        };
        auto hand_over = [&] {
            __syncthreads();
            SmemS *const s0 = cluster.map_shared_rank(&sm, 0);
            const int got = min((int)sm.got, kList);
            if (tid == 0) sm.base = atomicAdd(&s0->nall, sm.got);
            __syncthreads();
            for (int j = tid; j < got; j += kThreadsS)
                if (sm.base + j < kList) s0->list[sm.base + j] = mine[j];
        };
        // Block 0: its list in order into sorted; returns the number.
        auto rank_list = [&] {
            const int n = min((int)sm.nall, kList), n2 = (n + 1) & ~1;
            if (tid == 0 && n < n2) sm.list[n] = 0;
            __syncthreads();
            const ulonglong2 *const l2 = reinterpret_cast<const ulonglong2 *>(sm.list);
            for (int j = tid; j < n; j += kThreadsS) {
                const u64 e = sm.list[j];
                int r = 0;
#pragma unroll 4
                for (int q = 0; q < n2 / 2; ++q) {
                    const ulonglong2 o = l2[q];
                    r += (o.x > e) + (o.y > e);
                }
                sm.sorted[r] = e;
            }
            __syncthreads();
            return n;
        };
        // The key in which step b is cut: by histograms over the bits of its keys.  bc, bm: counts and
        // weights before the step, on return before that key.
        auto narrow = [&](int b, bool by_mass, double target, u64 &bc, u64 &bm) {
            uint32_t kl = 0xffffffffu, kh = 0;
            each([&](int i, float v) {
                if (v != -INFINITY && bin_of(v) == b) {
                    kl = min(kl, key_of(v));
                    kh = max(kh, key_of(v));
                }
            });
            kl = __reduce_min_sync(0xffffffffu, kl);
            kh = __reduce_max_sync(0xffffffffu, kh);
            __syncthreads();
            if (lane == 0) {
                sm.redu[warp] = kl;
                sm.red[warp] = kh;
            }
            __syncthreads();
            if (warp == 0) {
                kl = __reduce_min_sync(0xffffffffu, lane < kWarpsS ? sm.redu[lane] : 0xffffffffu);
                kh = __reduce_max_sync(0xffffffffu, lane < kWarpsS ? (uint32_t)sm.red[lane] : 0u);
                if (lane < C) {
                    *cluster.map_shared_rank(&sm.lo[rank], lane) = kl;
                    *cluster.map_shared_rank(&sm.hi[rank], lane) = kh;
                }
            }
            cluster.sync();
            joined = false;  // behind a barrier: the last histogram has been read
            kl = sm.lo[0];
            kh = sm.hi[0];
            for (int r = 1; r < C; ++r) {
                kl = min(kl, sm.lo[r]);
                kh = max(kh, sm.hi[r]);
            }
            for (;;) {
                int shift = 0;
                while (((kh - kl) >> shift) >= (uint32_t)kBins) ++shift;
                clear();
                each([&](int i, float v) {
                    const uint32_t key = key_of(v);
                    if (key < kl || key > kh) return;
                    const int bb = (int)((kh - key) >> shift);
                    atomicAdd(&sm.cnt[bb], 1u);
                    if (by_mass) {
                        const u64 w = W(v);
                        if (w) add_mass(sm, bb, w);
                    }
                });
                join();
                const uint32_t f = (uint32_t)cross(by_mass, (u64)k, target, bc, bm);
                bc = sm.base_cnt;
                bm = sm.base_mass;
                kh -= f << shift;
                if (shift == 0) return kh;
                const uint32_t width = (1u << shift) - 1u;
                if (kh - kl > width) kl = kh - width;
            }
        };

        clear();
        each([&](int i, float v) {
            const float at = place(v);
            const int b = (int)at;
            if (b >= kBins) return;
            atomicAdd(&sm.cnt[b], 1u);
            if (need_p) atomicAdd(&sm.mlo[b], (uint32_t)((at - (float)b) * 4096.f));
        });
        join();
        int bin_k = kBins;
        if (need_k) bin_k = cross(false, (u64)k, 0.0, 0, 0);
        if (bin_k < kBins && sm.nlist <= kList) {
            // 3. The first k are among few tokens: block 0 finishes the row.
            each4([&](int i, const float (&v)[4]) {
                unsigned in = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) in |= (v[e] != -INFINITY && bin_of(v[e]) <= bin_k ? 1u : 0u) << e;
                for (; in; in &= in - 1) {
                    const int e = __ffs(in) - 1;
                    set_aside(i + 32 * e, e < 2 ? (e ? v[1] : v[0]) : (e > 2 ? v[3] : v[2]));
                }
            });
            hand_over();
            cluster.sync();
            if (rank) return;
            const int n = rank_list(), nk = min(n, k);
            // Two consecutive ranks per thread.
            u64 e[2], w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = 2 * tid + h;
                e[h] = r < nk ? sm.sorted[r] : 0;
                w[h] = r < nk ? W(val_of((uint32_t)(e[h] >> 32))) : 0;
            }
            u64 sk;
            const u64 inc = block_incl<u64>(w[0] + w[1], sm.red, &sk);
            const double target = (double)topp * (double)sk;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u64 before = inc - (h ? 0 : w[0]) - w[1];
                if ((need_p && 2 * tid + h && (double)before >= target) || !W.enough(w[h])) e[h] = 0;
            }
            if (!e[0]) w[0] = 0;
            if (!e[1]) w[1] = 0;
            u64 tot;
            block_incl<u64>(w[0] + w[1], sm.red, &tot);
            // The draw: the first in index order whose running weight passes u * tot.
            u64 goal = (u64)((double)u * (double)tot);
            goal = tot && goal >= tot ? tot - 1 : goal;
            __syncthreads();
            // list: indices, sorted: weights; kept ones are a prefix of the order.
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (2 * tid + h < n) {
                    sm.sorted[2 * tid + h] = w[h];
                    sm.list[2 * tid + h] = w[h] ? 0xffffffffu - (uint32_t)e[h] : 0xffffffffffffffffull;
                }
            const int kept = __syncthreads_count(w[0] != 0) + __syncthreads_count(w[1] != 0);
            if (tid == 0) sm.found = 0xffffffffu;
            __syncthreads();
            for (int j = tid; j < kept; j += kThreadsS) {
                const u64 me = sm.list[j];
                u64 run = 0;
#pragma unroll 4
                for (int q = 0; q < kept; ++q) run += sm.list[q] <= me ? sm.sorted[q] : 0;
                if (run > goal) atomicMin(&sm.found, (uint32_t)me);
            }
            __syncthreads();
            if (tid == 0) A.tokens[row] = (int)sm.found;
            return;
        }
        // The estimate of top-p, from the same counts (before a narrowing replaces them): the running weight
        // before every step, a step's weight as its count at its mean place.
        double est_all = 0.0;
        int guess = kBins;
        if (need_p) {
            const uint32_t n = sm.tcnt[tid];
            const double at = n ? tid + (double)sm.tmass[tid] / (4096.0 * n) : 0.0;
            const double est = n ? n * (step > 0.f ? exp(-at / ((double)step * (double)temp)) : 1.0) : 0.0;
            double tot;
            const double inc = block_incl<double>(est, sm.redd, &tot);
            sm.est[tid + 1] = inc;
            if (tid == 0) sm.est[0] = 0.0;
            __syncthreads();
            est_all = tot;
            if (bin_k < kBins) {  // the first k only: a part of step bin_k
                const double part = (double)(k - (long long)sm.base_cnt) / (double)sm.tcnt[bin_k];
                est_all = sm.est[bin_k] + part * (sm.est[bin_k + 1] - sm.est[bin_k]);
            }
            if (tid == 0) sm.found = kBins - 1;
            __syncthreads();
            if (inc >= (double)topp * est_all) atomicMin(&sm.found, (uint32_t)tid);
            __syncthreads();
            guess = (int)sm.found;
            __syncthreads();
        }
        if (bin_k < kBins) {
            u64 bc = sm.base_cnt, bm = 0;
            thr = narrow(bin_k, false, 0.0, bc, bm);
            ties = (uint32_t)((u64)k - bc);
        }
        if (need_p) {
            const u64 wk = thr ? (u64)ties * W(val_of(thr)) : 0;  // of the ties at the k-th token's key
            u64 all, above, in;
            double target;
            for (int tries = 0;; ++tries) {
                // Exactly: the weight kept by k, above the step, in the step; and the step's tokens.
                if (tid == 0) sm.got = 0;
                __syncthreads();
                u64 sa = 0, sb = 0, sc = 0;
                each4([&](int i, const float (&v)[4]) {
                    unsigned in = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int b = bin_of(v[e]);
                        const u64 w = W(v[e]);
                        sa += key_of(v[e]) > thr ? w : 0;
                        sb += b < guess ? w : 0;
                        sc += b == guess ? w : 0;
                        in |= (b == guess && v[e] != -INFINITY ? 1u : 0u) << e;
                    }
                    for (; in; in &= in - 1) {
                        const int e = __ffs(in) - 1;
                        set_aside(i + 32 * e, e < 2 ? (e ? v[1] : v[0]) : (e > 2 ? v[3] : v[2]));
                    }
                });
                sa = warp_sum(sa);
                sb = warp_sum(sb);
                sc = warp_sum(sc);
                __syncthreads();
                if (lane == 0) {
                    sm.part[warp][0] = sa;
                    sm.part[warp][1] = sb;
                    sm.part[warp][2] = sc;
                }
                __syncthreads();
                if (warp == 0) {
                    for (int q = 0; q < 3; ++q) {
                        const u64 v = warp_sum(lane < kWarpsS ? sm.part[lane][q] : 0);
                        if (lane < C) *cluster.map_shared_rank(&sm.sum[rank][q], lane) = v;
                    }
                }
                hand_over();
                cluster.sync();
                joined = false;
                all = wk;
                above = in = 0;
                for (int r = 0; r < C; ++r) {
                    all += sm.sum[r][0];
                    above += sm.sum[r][1];
                    in += sm.sum[r][2];
                }
                target = (double)topp * (double)all;
                int next = guess;
                if (guess && (double)above >= target) --next;
                else if (guess < kBins - 1 && (double)(above + in) < target) ++next;
                if (next == guess || tries >= 2 * kBins) break;
                guess = next;
                cluster.sync();  // the sums have been read
                if (tid == 0) sm.nall = 0;
                cluster.sync();
            }
            uint32_t key, nties;
            if (*cluster.map_shared_rank(&sm.nall, 0) <= kList) {
                if (rank == 0) {
                    const int n = rank_list();
                    u64 e[2], w[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = 2 * tid + h;
                        e[h] = r < n ? sm.sorted[r] : 0;
                        w[h] = r < n ? W(val_of((uint32_t)(e[h] >> 32))) : 0;
                    }
                    u64 tot;
                    const u64 inc = above + block_incl<u64>(w[0] + w[1], sm.red, &tot);
                    if (tid == 0) sm.found = sm.nlist = 0;
                    __syncthreads();
                    // The last rank before which the running weight is below the target.
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const u64 before = inc - (h ? 0 : w[0]) - w[1];
                        if (e[h] && (double)before < target) atomicMax(&sm.found, (uint32_t)(2 * tid + h));
                    }
                    __syncthreads();
                    const uint32_t last = sm.found, lk = (uint32_t)(sm.sorted[last] >> 32);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (2 * tid + h <= (int)last && (uint32_t)(e[h] >> 32) == lk) atomicAdd(&sm.nlist, 1u);
                    __syncthreads();
                    if (tid < C) {
                        SmemS *const o = cluster.map_shared_rank(&sm, tid);
                        o->cut_key = lk;
                        o->cut_ties = sm.nlist;
                    }
                }
                cluster.sync();
                key = sm.cut_key;
                nties = sm.cut_ties;
            } else {
                u64 bc = 0, bm = above;
                key = narrow(guess, true, target, bc, bm);
                // Ties before which the running weight is still below the target.
                const u64 wt = W(val_of(key));
                const double left = target - (double)bm;
                nties = wt ? (left <= 0.0 ? 1u : (uint32_t)fmin(ceil(left / (double)wt), 4294967295.0)) : 0xffffffffu;
                nties = nties ? nties : 1u;
            }
            if (key > thr) {
                thr = key;
                ties = nties;
            } else if (key == thr) {
                ties = min(ties, nties);
            }
        }
    }
    // 4. The draw over the row.
    u64 mass = 0;
    uint32_t nt = 0;
    each4([&](int, const float (&v)[4]) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            any |= key_of(v[e]) > thr;
            nt += key_of(v[e]) == thr && v[e] != -INFINITY ? 1u : 0u;
        }
        if (any) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u64 w = W(v[e]);
                mass += key_of(v[e]) > thr && W.enough(w) ? w : 0;
            }
        }
    });
    mass = warp_sum(mass);
    nt = __reduce_add_sync(0xffffffffu, nt);
    if (lane < C) {
        SmemS *const o = cluster.map_shared_rank(&sm, lane);
        o->wmass[rank * kWarpsS + warp] = mass;
        o->wties[rank * kWarpsS + warp] = nt;
    }
    cluster.sync();
    u64 wt = thr ? W(val_of(thr)) : 0;
    if (!W.enough(wt)) wt = 0;
    // Before and up to each warp's part; one thread per part of the cluster.
    const int parts = C * kWarpsS;
    const u64 tn = tid < parts ? sm.wties[tid] : 0;
    u64 all_t, tot;
    const u64 it = block_incl<u64>(tn, sm.red, &all_t);
    const u64 et = it - tn;
    const u64 keep = et >= ties ? 0 : min((u64)ties - et, tn);
    const u64 mine = tid < parts ? sm.wmass[tid] + keep * wt : 0;
    const u64 im = block_incl<u64>(mine, sm.red, &tot);
    u64 goal = (u64)((double)u * (double)tot);
    goal = tot && goal >= tot ? tot - 1 : goal;
    if (tid == 0) sm.owner = -1;
    __syncthreads();
    if (mine && im > goal && im - mine <= goal) {
        sm.owner = tid;
        sm.base_mass = im - mine;
        sm.base_cnt = et;
    }
    __syncthreads();
    const int owner = sm.owner;
    if (owner < 0) {
        if (rank == 0 && tid == 0) A.tokens[row] = -1;
        return;
    }
    if (owner / kWarpsS != rank || owner % kWarpsS != warp) return;
    // A lane sums a 32nd of the part, in index order by lane; the lane that holds the token follows from the
    // sums, and all look for it in that lane's share.  (Scans of 32 tokens at a time along the whole part took
    // 15,000 cycles.)
    u64 run = sm.base_mass, seen = sm.base_cnt;
    const int share = part / 32;
    auto at = [&](int i) {
        if constexpr (CACHED) return cache[i];
        return i < w1 ? fetch(i) : -INFINITY;
    };
    u64 s = 0;
    uint32_t n = 0;
#pragma unroll 4
    for (int i = w0 + lane * share; i < w0 + (lane + 1) * share; ++i) {
        const float v = at(i);
        const uint32_t key = key_of(v);
        const u64 w = W(v);
        s += key > thr && W.enough(w) ? w : 0;
        n += key == thr && v != -INFINITY ? 1u : 0u;
    }
    auto scan = [&](u64 v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += y;
        }
        return v;
    };
    const u64 before = seen + scan(n) - n;
    s += (before >= ties ? 0 : min((u64)ties - before, (u64)n)) * wt;
    const u64 upto = run + scan(s);
    const int holder = __ffs(__ballot_sync(0xffffffffu, upto > goal)) - 1;
    if (holder < 0) return;  // (the part's own sum is past the goal)
    run = __shfl_sync(0xffffffffu, upto - s, holder);
    seen = __shfl_sync(0xffffffffu, before, holder);
    const int i0 = w0 + holder * share;
    for (int j = 0; j < share; j += 32) {
        const int i = i0 + j + lane;
        const float v = j + lane < share ? at(i) : -INFINITY;
        const uint32_t key = key_of(v);
        const bool tie = key == thr && v != -INFINITY;
        const unsigned bal = __ballot_sync(0xffffffffu, tie);
        u64 w = 0;
        if (key > thr) {
            w = W(v);
            if (!W.enough(w)) w = 0;
        } else if (tie && seen + __popc(bal & ((1u << lane) - 1u)) < ties) {
            w = wt;
        }
        const u64 e = scan(w);
        const unsigned hit = __ballot_sync(0xffffffffu, run + e > goal);
        if (hit) {
            if (lane == __ffs(hit) - 1) A.tokens[row] = i;
            return;
        }
        run += __shfl_sync(0xffffffffu, e, 31);
        seen += __popc(bal);
    }
}

template <typename T, bool CACHED>
cudaError_t launch_e(const SampleArgs &A, int S, int C, size_t cache, cudaStream_t st) {
    static DevBits configured{0};
    cudaError_t e = once_per_device(configured, [] {
        const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, CACHED>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(sample_kernel<T, CACHED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                           (int)(sizeof(SmemS) + kCacheMax));
    });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)A.nrows * C);
    cfg.blockDim = dim3(kThreadsS);
    cfg.dynamicSmemBytes = sizeof(SmemS) + cache;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, sample_kernel<T, CACHED>, A, S);
}

template <typename T>
trx_status launch_t(const SampleArgs &A, cudaStream_t st) {
    int bits = 0;
    while ((1 << bits) < A.V) ++bits;
    const int S = 62 - bits < 50 ? 62 - bits : 50;
    // Blocks per row: a power of two that fills the SMs (two blocks each), none with less than two tokens per
    // thread; more for a row that would not fit the blocks' shared memory otherwise.
    auto bytes = [&](int C) {  // of a block's part of the row
        return (size_t)((A.V + C * kWarpsS - 1) / (C * kWarpsS) + 31) / 32 * 32 * kWarpsS * 4;
    };
    // Sixteen blocks (not 8) only while they leave half of the SMs free: 2 rows of 151,936 take 11.6 us (16.6), 3 of
    // 600,001 45 us (71), but 9 rows 22.8 us (20.4).
    const int most = A.nrows * kMaxCluster * 2 <= device_sms() ? kMaxCluster : 8;
    int C = 1;
    while (C < most && A.V > C * 2 * kThreadsS && ((long long)A.nrows * C < device_sms() || bytes(C) > kCacheMax))
        C *= 2;
    return note_cuda(bytes(C) <= kCacheMax ? launch_e<T, true>(A, S, C, bytes(C), st) : launch_e<T, false>(A, S, C, 0, st));
}

}  // namespace

trx_status launch_sample_rows(const SampleArgs &A, int type, cudaStream_t st) {
    if (type == TRX_TYPE_F32) return launch_t<float>(A, st);
    return type == TRX_TYPE_F16 ? launch_t<__half>(A, st) : launch_t<__nv_bfloat16>(A, st);
}

}  // namespace trx
