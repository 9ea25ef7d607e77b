// Sampling of one token per row of logits (sm_100a): temperature, top-k, top-p and min-p from given
// random numbers, in one launch.
//
// Order: descending by logit, ties by index.  Weights w = exp((x - max) / T), held as integers
// round(w * 2^S) (S = 62 - ceil(log2 V), at most 50), so that every sum is exact whatever its order:
// the borders of top-p and of the draw do not move with the division of the work.  The exponent and
// exp are in 64 bits: with 152k tokens a 32-bit sum is off by more than many tokens' whole share.
//
// A row is held by a cluster of C thread blocks (distributed shared memory joins their parts):
//  1. max (and with it the greedy token) and min.
//  2. top-k / top-p: a histogram over 2048 equal steps of max - x (counts, and weights for top-p).
//     Equal steps order the tokens like their logits, and spread them better than the bits of a float
//     would.  Block 0 finds the step in which the k-th token, or the last of the nucleus, lies.
//  3a. Few tokens up to that step (at most kList): they are gathered in block 0, which ranks them, cuts
//     at k, p and min-p, and draws.
//  3b. Otherwise the step is narrowed by histograms over the keys' bits until one key is left: the cut
//     is that key and how many of its ties (in index order) are kept.
//  4. (3b, or no top-k and top-p) The draw over the whole row: each warp sums its contiguous part, the
//     parts' prefix tells which warp holds the token, and that warp scans its part again.
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

constexpr int kThreadsS = 1024;
constexpr int kWarpsS = kThreadsS / 32;
constexpr int kBins = 2048;
constexpr int kList = 2048;
constexpr int kMaxCluster = 8;

// Order-preserving bits of a float (NaN counts as -inf).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x != x ? -INFINITY : x);
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
    uint32_t cnt[kBins];             // this block's histogram
    uint32_t mlo[kBins], mhi[kBins]; // its weights, 64 bits in two words
    uint32_t tcnt[kBins];            // block 0: the cluster's histogram
    u64 tmass[kBins];
    u64 list[kList], sorted[kList];  // block 0: gathered tokens (key << 32 | ~index)
    u64 best[kMaxCluster];           // every block's max, for the whole cluster
    uint32_t lo[kMaxCluster], hi[kMaxCluster];
    u64 wmass[kMaxCluster * kWarpsS];
    uint32_t wties[kMaxCluster * kWarpsS];
    u64 red[kWarpsS + 1];
    uint32_t redu[kWarpsS + 1];
    // Block 0's findings, copied to every block.
    int bin_k, bin_p, mode;
    uint32_t key, nlist, found;
    u64 base_cnt, base_mass, total;
};

// Weight function of a row.
struct Weigh {
    float mx;
    double inv, minp, scale;  // 1 / T, 2^S
    __device__ __forceinline__ u64 operator()(float x) const {
        double w;
        if (x == mx)
            w = 1.0;
        else if (x == -INFINITY)
            w = 0.0;
        else
            w = exp(((double)x - (double)mx) * inv);
        return (u64)__double2ull_rn(w * scale);
    }
    __device__ __forceinline__ bool enough(u64 w) const { return (double)w >= minp * scale; }
};

// Block-wide inclusive sums of (count, mass); every thread gets its own.
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
        const T w0 = red[lane];
        T w = w0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const T y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        red[lane] = w - w0;
        if (lane == 31) red[32] = w;
    }
    __syncthreads();
    v += red[warp];
    *tot = red[32];
    __syncthreads();
    return v;
}

__device__ __forceinline__ void add_mass(SmemS &sm, int b, u64 w) {
    const uint32_t lo = (uint32_t)w, old = atomicAdd(&sm.mlo[b], lo);
    const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
    if (hi) atomicAdd(&sm.mhi[b], hi);
}

template <typename T>
__global__ void __launch_bounds__(kThreadsS, 1) sample_kernel(SampleArgs A, int S) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SmemS &sm = *reinterpret_cast<SmemS *>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / C, V = A.V;
    pdl_trigger();
    pdl_wait();
    const T *const x = reinterpret_cast<const T *>(A.x) + row * A.ld;
    const float temp = A.temp[row], u = A.u[row], topp = A.top_p[row];
    const int k = A.top_k[row];
    // This warp's contiguous part, a multiple of 32 tokens.
    const int part = ((V + C * kWarpsS - 1) / (C * kWarpsS) + 31) / 32 * 32;
    const int w0 = min(V, (rank * kWarpsS + warp) * part), w1 = min(V, w0 + part);

    // 1. Max, min.
    u64 best = 0;
    uint32_t lo = 0xffffffffu;
    for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t key = key_of(load_f(x + i));
        const u64 b = ((u64)key << 32) | (0xffffffffu - (uint32_t)i);
        best = b > best ? b : best;
        if (key > kKeyNegInf && key < lo) lo = key;
    }
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
    cluster.sync();  // every block has started; red complete
    if (warp == 0) {
        best = sm.red[lane];
        lo = __reduce_min_sync(0xffffffffu, sm.redu[lane]);
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
    cluster.sync();
    best = sm.best[0];
    lo = sm.lo[0];
    for (int r = 1; r < C; ++r) {
        best = sm.best[r] > best ? sm.best[r] : best;
        lo = min(lo, sm.lo[r]);
    }
    const uint32_t kmax = (uint32_t)(best >> 32);
    const bool none = kmax <= kKeyNegInf, greedy = !(temp > 0.f) || k == 1;
    Weigh W;
    W.mx = val_of(kmax);
    W.inv = 1.0 / (double)temp;
    W.scale = (double)(1ull << S);
    W.minp = (double)A.min_p[row];
    if (none || (greedy && (!(temp > 0.f) || W.minp <= 1.0))) {
        if (rank == 0 && tid == 0) A.tokens[row] = none ? -1 : (int)(0xffffffffu - (uint32_t)best);
        return;
    }
    const bool need_k = k > 0 && k < V, need_p = topp < 1.f;
    uint32_t thr = 0;           // kept: keys above thr, and the first `ties` with key thr
    uint32_t ties = 0xffffffffu;
    if (need_k || need_p) {
        // 2. Histogram over max - x.
        const float span = fminf(36.f * temp, W.mx - val_of(lo));
        const bool by_temp = span == 36.f * temp;  // then the last step holds only weights that round to 0
        const float step = span > 0.f && span < INFINITY ? 2047.5f / span : 0.f;
        auto bin_of = [&](float v) {
            const float d = v == W.mx ? 0.f : W.mx - v;
            return (int)fminf(d * step, (float)(kBins - 1));
        };
        auto clear = [&] {
            for (int i = tid; i < kBins; i += kThreadsS) sm.cnt[i] = sm.mlo[i] = sm.mhi[i] = 0u;
            __syncthreads();
        };
        // The blocks' histograms into block 0's tcnt, tmass.
        auto join = [&] {
            cluster.sync();
            SmemS *const s0 = cluster.map_shared_rank(&sm, 0);
            for (int i = rank * (kBins / C) + tid; i < (rank + 1) * (kBins / C); i += kThreadsS) {
                uint32_t n = 0;
                u64 m = 0;
                for (int r = 0; r < C; ++r) {
                    const SmemS *const o = cluster.map_shared_rank(&sm, r);
                    n += o->cnt[i];
                    m += ((u64)o->mhi[i] << 32) + o->mlo[i];
                }
                s0->tcnt[i] = n;
                s0->tmass[i] = m;
            }
            cluster.sync();
        };
        // Block 0: the first step whose running count reaches n, or whose running weight reaches
        // target (by_mass), with the count and weight before it: bin, base_cnt, base_mass.
        auto cross = [&](bool by_mass, u64 n, double target, u64 bc, u64 bm) {
            u64 tc, tm;
            const uint32_t c0 = sm.tcnt[2 * tid], c1 = sm.tcnt[2 * tid + 1];
            const u64 m0 = sm.tmass[2 * tid], m1 = sm.tmass[2 * tid + 1];
            const u64 ic = bc + block_incl<u64>((u64)c0 + c1, sm.red, &tc);
            const u64 im = bm + block_incl<u64>(m0 + m1, sm.red, &tm);
            const u64 ec = ic - c0 - c1, em = im - m0 - m1;
            if (tid == 0) sm.found = kBins;
            __syncthreads();
            const bool h0 = by_mass ? (double)(em + m0) >= target : ec + c0 >= n;
            const bool h1 = by_mass ? (double)im >= target : ic >= n;
            if (h1) atomicMin(&sm.found, (uint32_t)(h0 ? 2 * tid : 2 * tid + 1));
            __syncthreads();
            if (sm.found / 2 == (uint32_t)tid) {
                const bool second = sm.found & 1;
                sm.base_cnt = second ? ec + c0 : ec;
                sm.base_mass = second ? em + m0 : em;
                sm.nlist = second ? (uint32_t)ic : (uint32_t)(ec + c0);
            }
            __syncthreads();
            return (int)sm.found;
        };
        clear();
        for (int i = w0 + lane; i < w1; i += 32) {
            const float v = val_of(key_of(load_f(x + i)));
            const int b = bin_of(v);
            atomicAdd(&sm.cnt[b], 1u);
            if (need_p) {
                const u64 w = W(v);
                if (w) add_mass(sm, b, w);
            }
        }
        join();
        if (rank == 0) {
            // mode 0: keep everything (by k and p), 1: gather the steps up to bin_k, 2: narrow.
            u64 s = 0;
            if (need_p) {
                u64 t;
                block_incl<u64>(sm.tmass[2 * tid] + sm.tmass[2 * tid + 1], sm.red, &t);
                s = t;
            }
            const int bk = need_k ? cross(false, (u64)k, 0.0, 0, 0) : kBins;
            const bool all_k = !need_k || bk >= kBins || (by_temp && bk == kBins - 1);
            int bp = kBins;
            if (all_k && need_p) bp = cross(true, 0, (double)topp * (double)s, 0, 0);
            const bool all_p = !need_p || (all_k && (bp >= kBins || (by_temp && bp == kBins - 1)));
            if (tid == 0) {
                sm.mode = all_k && all_p ? 0 : (sm.nlist <= kList ? 1 : 2);
                sm.bin_k = all_k ? -1 : bk;
                sm.bin_p = all_k ? bp : -1;
                sm.total = s;
                sm.found = 0;
            }
            __syncthreads();
            if (tid < C && tid) {
                SmemS *const o = cluster.map_shared_rank(&sm, tid);
                o->mode = sm.mode;
                o->bin_k = sm.bin_k;
                o->bin_p = sm.bin_p;
                o->total = sm.total;
            }
        }
        cluster.sync();
        const int mode = sm.mode, bin_k = sm.bin_k, bin_p = sm.bin_p;
        if (mode == 1) {
            // 3a. The tokens up to the cut's step, in block 0.
            SmemS *const s0 = cluster.map_shared_rank(&sm, 0);
            const int cut = bin_k >= 0 ? bin_k : bin_p;
            for (int i0 = w0; i0 < w1; i0 += 32) {
                const int i = i0 + lane;
                uint32_t key = 0;
                bool in = false;
                if (i < w1) {
                    key = key_of(load_f(x + i));
                    in = bin_of(val_of(key)) <= cut;
                }
                const unsigned bal = __ballot_sync(0xffffffffu, in);
                if (!bal) continue;
                uint32_t at = 0;
                if (lane == 0) at = atomicAdd(&s0->found, (uint32_t)__popc(bal));
                at = __shfl_sync(0xffffffffu, at, 0) + __popc(bal & ((1u << lane) - 1u));
                if (in && at < kList) s0->list[at] = ((u64)key << 32) | (0xffffffffu - (uint32_t)i);
            }
            cluster.sync();
            if (rank) return;
            const int n = min((int)sm.found, kList);
            for (int j = tid; j < n; j += kThreadsS) {
                const u64 e = sm.list[j];
                int r = 0;
                for (int q = 0; q < n; ++q) r += sm.list[q] > e;
                sm.sorted[r] = e;
            }
            __syncthreads();
            const int nk = need_k && bin_k >= 0 ? min(n, k) : n;
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
            const double target = (double)topp * (double)(bin_k >= 0 ? sk : sm.total);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u64 before = inc - w[1] - (h ? 0 : w[0]);
                if ((need_p && !(2 * tid + h == 0) && (double)before >= target) || !W.enough(w[h])) w[h] = 0;
            }
            u64 tot;
            block_incl<u64>(w[0] + w[1], sm.red, &tot);
            // The draw: the first in index order whose running weight passes u * tot.
            u64 goal = (u64)((double)u * (double)tot);
            goal = tot && goal >= tot ? tot - 1 : goal;
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (2 * tid + h < n) {
                    sm.sorted[2 * tid + h] = w[h];
                    sm.list[2 * tid + h] = w[h] ? 0xffffffffu - (uint32_t)e[h] : 0xffffffffffffffffull;
                }
            if (tid == 0) sm.found = 0xffffffffu;
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (2 * tid + h >= n || !w[h]) continue;
                const u64 me = sm.list[2 * tid + h];
                u64 run = 0;
                for (int q = 0; q < n; ++q) run += sm.list[q] <= me ? sm.sorted[q] : 0;
                if (run > goal) atomicMin(&sm.found, (uint32_t)me);
            }
            __syncthreads();
            if (tid == 0) A.tokens[row] = (int)sm.found;
            return;
        }
        if (mode == 2) {
            // 3b. Narrow the step of the cut: first for k, then (with the weight of the first k as the
            // whole) for p.
            u64 whole = sm.total;
            for (int pass = 0; pass < 2; ++pass) {
                const bool by_mass = pass == 1;
                if (by_mass ? !need_p : bin_k < 0) continue;
                const double target = (double)topp * (double)whole;
                u64 bc = 0, bm = 0;  // block 0: counts and weights before the range
                int b = by_mass ? bin_p : bin_k;
                if (by_mass && b < 0) {
                    // k was narrowed first: the step of p among the row's steps again.
                    clear();
                    for (int i = w0 + lane; i < w1; i += 32) {
                        const float v = val_of(key_of(load_f(x + i)));
                        const u64 w = W(v);
                        const int bb = bin_of(v);
                        atomicAdd(&sm.cnt[bb], 1u);
                        if (w) add_mass(sm, bb, w);
                    }
                    join();
                    if (rank == 0) {
                        const int f = cross(true, 0, target, 0, 0);
                        if (tid < C) cluster.map_shared_rank(&sm, tid)->bin_p = f;
                    }
                    cluster.sync();
                    b = sm.bin_p;
                    if (b >= kBins) continue;
                }
                if (rank == 0) {
                    // The step's base, from the row's steps (tcnt and tmass still hold them).
                    cross(by_mass, (u64)k, target, 0, 0);
                    bc = sm.base_cnt;
                    bm = sm.base_mass;
                }
                // The keys of the step.
                uint32_t kl = 0xffffffffu, kh = 0;
                for (int i = w0 + lane; i < w1; i += 32) {
                    const uint32_t key = key_of(load_f(x + i));
                    if (bin_of(val_of(key)) == b) {
                        kl = min(kl, key);
                        kh = max(kh, key);
                    }
                }
                kl = __reduce_min_sync(0xffffffffu, kl);
                kh = __reduce_max_sync(0xffffffffu, kh);
                __syncthreads();
                if (lane == 0) {
                    sm.redu[warp] = kl;
                    sm.red[warp] = kh;
                }
                __syncthreads();
                if (warp == 0) {
                    kl = __reduce_min_sync(0xffffffffu, sm.redu[lane]);
                    kh = __reduce_max_sync(0xffffffffu, (uint32_t)sm.red[lane]);
                    if (lane < C) {
                        *cluster.map_shared_rank(&sm.lo[rank], lane) = kl;
                        *cluster.map_shared_rank(&sm.hi[rank], lane) = kh;
                    }
                }
                cluster.sync();
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
                    for (int i = w0 + lane; i < w1; i += 32) {
                        const uint32_t key = key_of(load_f(x + i));
                        if (key < kl || key > kh) continue;
                        const int bb = (int)((kh - key) >> shift);
                        atomicAdd(&sm.cnt[bb], 1u);
                        if (need_p) {
                            const u64 w = W(val_of(key));
                            if (w) add_mass(sm, bb, w);
                        }
                    }
                    join();
                    if (rank == 0) {
                        const int f = cross(by_mass, (u64)k, target, bc, bm);
                        bc = sm.base_cnt;
                        bm = sm.base_mass;
                        if (tid < C) {
                            SmemS *const o = cluster.map_shared_rank(&sm, tid);
                            o->key = (uint32_t)f;
                            o->base_cnt = bc;
                            o->base_mass = bm;
                        }
                    }
                    cluster.sync();
                    const uint32_t f = sm.key;
                    kh -= f << shift;
                    if (shift == 0) break;
                    const uint32_t width = (1u << shift) - 1u;
                    if (kh - kl > width) kl = kh - width;
                }
                const u64 wt = W(val_of(kh));
                if (!by_mass) {
                    thr = kh;
                    ties = (uint32_t)((u64)k - sm.base_cnt);
                    whole = sm.base_mass + (u64)ties * wt;
                } else {
                    // Ties before which the running weight is still below the target.
                    uint32_t n = 0xffffffffu;
                    if (wt) {
                        const double left = target - (double)sm.base_mass;
                        n = left <= 0.0 ? 1u : (uint32_t)ceil(left / (double)wt);
                        n = n ? n : 1u;
                    }
                    if (kh > thr) {
                        thr = kh;
                        ties = n;
                    } else if (kh == thr) {
                        ties = min(ties, n);
                    }
                }
                cluster.sync();  // sm.key, base_* are read before the next pass writes them
            }
        }
    }
    // 4. The draw over the row.
    u64 mass = 0;
    uint32_t nt = 0;
    for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t key = key_of(load_f(x + i));
        if (key > thr) {
            const u64 w = W(val_of(key));
            if (W.enough(w)) mass += w;
        } else if (key == thr) {
            ++nt;
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
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
    if (tid == 0) sm.mode = -1;
    __syncthreads();
    if (mine && im > goal && im - mine <= goal) {
        sm.mode = tid;
        sm.base_mass = im - mine;
        sm.base_cnt = et;
    }
    __syncthreads();
    const int owner = sm.mode;
    if (owner < 0) {
        if (rank == 0 && tid == 0) A.tokens[row] = -1;
        return;
    }
    if (owner / kWarpsS != rank || owner % kWarpsS != warp) return;
    u64 run = sm.base_mass, seen = sm.base_cnt;
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t key = i < w1 ? key_of(load_f(x + i)) : 0u;
        const bool tie = i < w1 && key == thr;
        const unsigned bal = __ballot_sync(0xffffffffu, tie);
        u64 w = 0;
        if (i < w1 && key > thr) {
            w = W(val_of(key));
            if (!W.enough(w)) w = 0;
        } else if (tie && seen + __popc(bal & ((1u << lane) - 1u)) < ties) {
            w = wt;
        }
        u64 s = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, run + s > goal);
        if (hit) {
            if (lane == __ffs(hit) - 1) A.tokens[row] = i;
            return;
        }
        run += __shfl_sync(0xffffffffu, s, 31);
        seen += __popc(bal);
    }
}

template <typename T>
trx_status launch_t(const SampleArgs &A, cudaStream_t st) {
    static DevBits configured{0};
    cudaError_t e = once_per_device(configured, [] {
        return cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SmemS));
    });
    if (e != cudaSuccess) return note_cuda(e);
    int bits = 0;
    while ((1 << bits) < A.V) ++bits;
    const int S = 62 - bits < 50 ? 62 - bits : 50;
    // Blocks per row: a power of two that fills the SMs, none with less than two tokens per thread.
    int C = 1;
    while (C < kMaxCluster && (long long)A.nrows * C * 2 <= device_sms() * 2 && A.V > C * 2 * kThreadsS) C *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)A.nrows * C);
    cfg.blockDim = dim3(kThreadsS);
    cfg.dynamicSmemBytes = sizeof(SmemS);
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
    return note_cuda(cudaLaunchKernelEx(&cfg, sample_kernel<T>, A, S));
}

}  // namespace

trx_status launch_sample_rows(const SampleArgs &A, int type, cudaStream_t st) {
    if (type == TRX_TYPE_F32) return launch_t<float>(A, st);
    return type == TRX_TYPE_F16 ? launch_t<__half>(A, st) : launch_t<__nv_bfloat16>(A, st);
}

}  // namespace trx
