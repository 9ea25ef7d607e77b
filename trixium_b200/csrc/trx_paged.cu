// The paged KV cache of a server's step (sm_100a): the plan (block tables, slots and row offsets from
// the sequences' lengths), the release of finished sequences' pages, the append of the new keys and
// values, and attention over the pages for few query rows per kv head (decode).  The attention of
// prompt chunks is in trx_paged_tc.cu.
#include <cstdint>
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "trx_paged.cuh"

namespace trx {
namespace {
namespace cg = cooperative_groups;

// Plan ---------------------------------------------------------------------------------------------
// have = ceil(cached / P), need = ceil((cached + new) / P) for a sequence with new rows.  Two prefix
// sums over the sequences place everything: the rows give cu, the pages taken (need - have) give each
// sequence its part of the free stack.  Both run as one 64-bit sum (rows in the low 33 bits).  The
// kernel is latency: a few hundred bytes in, at most some hundred KB out.  One thread block, or a
// cluster of up to 8 when there are many rows to write; every block of the cluster repeats the sums,
// and the cluster barrier between the last read of the lengths and the first write lets lens and
// n_free be the inputs' own buffers.  In a graph 32 decoding sequences take 3.3 us (a launch and four dependent
// loads), 256 sequences with 23,700 rows 5.4; called from Python both take the host's 6.5.
constexpr int kPlanThreads = 1024;
constexpr int kPlanRowBits = 33;

__device__ __forceinline__ int pages_of(int positions, int shift) {
    return (int)(((unsigned)positions + (1u << shift) - 1u) >> shift);
}

struct PlanSmem {
    int cu[kPagedMaxSeq + 1];
    int pg[kPagedMaxSeq + 1];  // pages taken by the sequences before
    int cached[kPagedMaxSeq];
    long long wsum[33];
    int bad;
};

__device__ __forceinline__ int find_le(const int *a, int n, int v) {  // a[i] <= v < a[i + 1]
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads)
    paged_plan_kernel(const trx_pages P, int shift, const int *cached, const int *fresh, const int *free_pages,
                      uint32_t free_cap, const int *n_free, uint32_t *err) {
    __shared__ PlanSmem sm;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, nseq = (int)P.nseq;
    const int crank = (int)cluster.block_rank(), nthr = (int)cluster.num_blocks() * kPlanThreads;
    const bool writer = crank == 0;
    pdl_trigger();
    if (tid == 0) sm.bad = 0;
    pdl_wait();
    __syncthreads();
    const int nf = *n_free;
    int c = 0, n = 0, have = 0, need = 0;
    if (tid < nseq) {
        c = cached[tid];
        n = fresh[tid];
        if (c < 0 || n < 0 || n > (int)P.max_rows || (long long)c + n > (long long)P.max_pages << shift) {
            sm.bad = TRX_DEV_RANGE;
            n = 0;
        } else {
            have = pages_of(c, shift);
            need = n ? pages_of(c + n, shift) : have;
        }
        sm.cached[tid] = c;
    }
    long long tot;
    const long long ex = pg_block_scan((long long)n + ((long long)(need - have) << kPlanRowBits), sm.wsum, &tot);
    const long long rows = tot & ((1ll << kPlanRowBits) - 1), taken = tot >> kPlanRowBits;
    if (tid < nseq) {
        sm.cu[tid] = (int)(ex & ((1ll << kPlanRowBits) - 1));
        sm.pg[tid] = (int)(ex >> kPlanRowBits);
    }
    int bad = sm.bad;
    if (nf < 0 || (uint32_t)nf > min(P.n_pages, free_cap) || rows > (long long)P.max_rows) bad |= TRX_DEV_RANGE;
    if (!bad && taken > nf) bad = TRX_DEV_PAGES;
    if (tid == 0) {
        sm.cu[nseq] = bad ? 0 : (int)rows;
        sm.pg[nseq] = bad ? 0 : (int)taken;
    }
    cluster.sync();  // all inputs read, the prefixes complete
    if (writer) {
        if (tid < nseq) {
            P.cu[tid] = bad ? 0 : sm.cu[tid];
            P.lens[tid] = bad ? c : c + n;
            P.last[tid] = bad || n == 0 ? 0 : sm.cu[tid] + n - 1;
        }
        if (tid == 0) {
            P.cu[nseq] = bad ? 0 : (int)rows;
            *P.n_free = bad ? nf : nf - (int)taken;
            if (bad) atomicOr(err, (unsigned)bad);
        }
    }
    if (bad) return;
    const int g = crank * kPlanThreads + tid;
    for (int r = g; r < (int)rows; r += nthr) {
        const int b = find_le(sm.cu, nseq, r);
        const int cb = sm.cached[b], p = cb + r - sm.cu[b];
        const int hb = pages_of(cb, shift), j = p >> shift;
        int id;
        if (j < hb)
            id = P.tables[(size_t)b * P.max_pages + j];
        else
            id = free_pages[nf - 1 - (sm.pg[b] + j - hb)];
        int slot = -1;
        if ((unsigned)id < P.n_pages)
            slot = (id << shift) + (p & ((1 << shift) - 1));
        else
            atomicOr(err, TRX_DEV_RANGE);
        P.slots[r] = slot;
        P.pos[r] = p;
    }
    for (int i = g; i < (int)taken; i += nthr) {
        const int b = find_le(sm.pg, nseq, i);
        P.tables[(size_t)b * P.max_pages + pages_of(sm.cached[b], shift) + i - sm.pg[b]] = free_pages[nf - 1 - i];
    }
}

__global__ void __launch_bounds__(kPlanThreads)
    paged_release_kernel(const trx_pages P, int shift, const int *done, int *lens, int *free_pages, int *n_free,
                         uint32_t *err) {
    __shared__ PlanSmem sm;
    const int tid = threadIdx.x, nseq = (int)P.nseq;
    pdl_trigger();
    if (tid == 0) sm.bad = 0;
    pdl_wait();
    __syncthreads();
    const int nf = *n_free;
    int cnt = 0;
    if (tid < nseq && done[tid]) {
        const int len = lens[tid];
        if (len < 0 || (long long)len > (long long)P.max_pages << shift)
            sm.bad = 1;
        else
            cnt = pages_of(len, shift);
    }
    long long tot;
    const long long ex = pg_block_scan(cnt, sm.wsum, &tot);
    if (tid < nseq) sm.pg[tid] = (int)ex;
    if (tid == 0) sm.pg[nseq] = (int)tot;
    if (nf < 0 || (long long)nf + tot > (long long)P.n_pages) sm.bad = 1;
    __syncthreads();
    if (!sm.bad)
        for (int i = tid; i < (int)tot; i += kPlanThreads) {
            const int b = find_le(sm.pg, nseq, i);
            if ((unsigned)P.tables[(size_t)b * P.max_pages + i - sm.pg[b]] >= P.n_pages) sm.bad = 1;
        }
    __syncthreads();
    if (sm.bad) {
        if (tid == 0) atomicOr(err, TRX_DEV_RANGE);
        return;
    }
    for (int i = tid; i < (int)tot; i += kPlanThreads) {
        const int b = find_le(sm.pg, nseq, i);
        int *t = P.tables + (size_t)b * P.max_pages + i - sm.pg[b];
        free_pages[nf + i] = *t;
        *t = -1;
    }
    if (tid < nseq && done[tid]) lens[tid] = 0;
    if (tid == 0) *n_free = nf + (int)tot;
}

// Append -------------------------------------------------------------------------------------------
// A unit is 8 elements of a head: for u < half / 4 the pairs 4u..4u+3 and half+4u.. that the rotation
// mixes, else 8 consecutive dims behind the rotated ones; hd / 8 neighbouring lanes hold a head, so the
// norm is a shuffle over them and a rotation needs no exchange.  A block takes one row and a share of
// its heads (y): its first loads go out, and meanwhile one thread per pair computes the row's cosines
// and sines, which all heads share, into shared memory; then each head's loads go out a head ahead.
// HBM-bound for chunks: 4 bytes in and 2 (or 4) out per element.  2,602 rows of 24 + 2 x 4 gated heads of
// 256 take 26 us in a graph (27 from Python), 5.0 TB/s; one head's loads at a time, behind the table, and the norms'
// weights kept in registers (4 blocks per SM for 5) took 32.  Few rows are latency: 16 of 48 heads of 128 take 2.6 us
// in a graph (11.5 from Python).
constexpr int kAppThreads = 256;

template <typename T> __device__ __forceinline__ void store4(T *p, float4 v) {
    const uint2 u = make_uint2(PgCvt<T>::pack(v.x, v.y), PgCvt<T>::pack(v.z, v.w));
    *reinterpret_cast<uint2 *>(p) = u;
}
template <> __device__ __forceinline__ void store4<float>(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }

__device__ __forceinline__ float4 mul4(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
__device__ __forceinline__ float4 mul4(float4 a, float4 b) {
    return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w);
}
__device__ __forceinline__ float dot4(float4 a) { return a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w; }

template <typename CT, typename QT, int HD>
__global__ void __launch_bounds__(kAppThreads, 5) paged_append_kernel(PgAppendArgs A, uint32_t *err) {
    constexpr int UPH = HD / 8;               // lanes (units) per head
    constexpr int HPB = kAppThreads / UPH;    // heads a block takes at a time
    __shared__ __align__(16) float cs[HD / 2], sn[HD / 2];
    const int tid = threadIdx.x, u = tid % UPH;
    pdl_trigger();
    const bool rot = u < A.half / 4;
    const int d0 = rot ? 4 * u : 2 * A.half + 8 * (u - A.half / 4), d1 = rot ? A.half + 4 * u : d0 + 4;
    const int heads = A.H + 2 * A.Hkv;
    pdl_wait();
    int rows = A.cu[A.nseq];
    if (rows > A.max_rows || rows < 0) {
        if (tid == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(err, TRX_DEV_RANGE);
        rows = rows < 0 ? 0 : A.max_rows;
    }
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const int slot = A.slots[row], pos = A.pos[row];
        const bool live = (unsigned)slot < (unsigned)A.n_slots;
        if (!live && tid == 0 && blockIdx.y == 0) atomicOr(err, TRX_DEV_RANGE);
        // Whole groups of UPH lanes share a head; heads past the end do nothing but the shuffles.
        auto load = [&](int h, float4 &a, float4 &b) {
            const float *src = h < A.H ? A.q + row * A.q_ld + (long long)h * HD * (A.gated ? 2 : 1)
                                       : (h < A.H + A.Hkv ? A.k + row * A.k_ld + (long long)(h - A.H) * HD
                                                          : A.v + row * A.v_ld + (long long)(h - A.H - A.Hkv) * HD);
            a = b = make_float4(0.f, 0.f, 0.f, 0.f);
            if (h < heads) {
                a = *reinterpret_cast<const float4 *>(src + d0);
                b = *reinterpret_cast<const float4 *>(src + d1);
            }
        };
        int h = blockIdx.y * HPB + tid / UPH;
        float4 a, b, wa, wb;  // a head's elements, and the norm's weights (in L1 after the first row)
        auto weights = [&](int h) {
            const float *w = h < A.H ? A.qn : A.kn;
            wa = __ldg(reinterpret_cast<const float4 *>(w + d0));
            wb = __ldg(reinterpret_cast<const float4 *>(w + d1));
        };
        load(h, a, b);
        weights(h);
        __syncthreads();  // the previous row's table is done with
        if (tid < A.half) {
            const float ang = __fmul_rn((float)pos, __ldg(A.freq + tid));
            sincosf(ang, &sn[tid], &cs[tid]);
        }
        __syncthreads();
        for (; h < (heads + HPB - 1) / HPB * HPB; h += gridDim.y * HPB) {
            const bool on = h < heads, is_q = h < A.H, is_k = !is_q && h < A.H + A.Hkv;
            float4 na, nb;  // the next head's, meanwhile
            load(h + gridDim.y * HPB, na, nb);
            float ss = dot4(a) + dot4(b);
#pragma unroll
            for (int o = UPH / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (on && (is_q || is_k)) {
                const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)HD), A.eps)));
                a = mul4(mul4(a, r), wa);
                b = mul4(mul4(b, r), wb);
                if (rot) {
                    const float4 c = *reinterpret_cast<const float4 *>(cs + 4 * u);
                    const float4 s = *reinterpret_cast<const float4 *>(sn + 4 * u);
                    const float4 x = a, y = b;
                    a = make_float4(x.x * c.x - y.x * s.x, x.y * c.y - y.y * s.y, x.z * c.z - y.z * s.z,
                                    x.w * c.w - y.w * s.w);
                    b = make_float4(x.x * s.x + y.x * c.x, x.y * s.y + y.y * c.y, x.z * s.z + y.z * c.z,
                                    x.w * s.w + y.w * c.w);
                }
            }
            if (on && is_q) {
                QT *dst = reinterpret_cast<QT *>(A.q_out) + ((size_t)row * A.H + h) * HD;
                store4<QT>(dst + d0, a);
                store4<QT>(dst + d1, b);
            } else if (on && live) {
                const int kh = is_k ? h - A.H : h - A.H - A.Hkv;
                CT *dst = reinterpret_cast<CT *>(is_k ? A.kp : A.vp) + ((size_t)slot * A.Hkv + kh) * HD;
                store4<CT>(dst + d0, a);
                store4<CT>(dst + d1, b);
            }
            a = na;
            b = nb;
            weights(h + gridDim.y * HPB);
        }
    }
}

// Attention, few query rows ------------------------------------------------------------------------
// A CTA walks its pieces (PgSched) in tiles of 64 key positions. Rows of the products are the query rows
// of one (query tile, kv head): 16 / rep tokens x rep heads, padded to 16.
//  * warp 4, the producer: key tiles by TMA (boxes of one page, or the tile's part of it, see PgMaps;
//    lanes 0-15 K, 16-31 V) through a ring, and each piece's query rows into one of two
//    places, all ahead of the work.
//  * warps 0-3: 16 positions each of every tile: S = Q K^T and O += P V on mma.sync m16n8k16 with fp32
//    accumulation, the softmax online per warp (running maximum and sum per row). At the end of a piece
//    the four are joined in a fixed order.
// fp32 queries: Q and P enter as two fp16 parts each (x = hi + lo), so that products keep 2^-22.
// Bound by the K/V stream: rep tokens' work per byte is far below the tensor cores' rate even with 16 rows
// padded, so the ring (64 to 192 KB per SM in flight) and short ends of pieces are what matters.
// In a graph 3 sequences, 371 MB of fp16 K and V (16 query, 8 kv heads of 128, fp32 queries), take 70 us (76 with
// changing inputs from Python), 5.3 TB/s; 16 sequences of 900 tokens, 63 MB, 18.2 us (22.9), of which the stream is 10: the
// rest is the start (schedule, tables, first tiles) and the joins of cut items.
constexpr int kDecThreads = 160;
constexpr int kDecWarps = 4;
constexpr int kDecTile = 64;

template <int HD, bool SPLIT>
struct DecSmem {
    static constexpr int ST = HD == 64 ? 4 : 3;          // ring stages
    static constexpr int TB = kDecTile * HD * 2;         // bytes of a K or V tile
    static constexpr int QB = SPLIT && HD >= 128 ? 1 : 2;  // places for a piece's query rows
    unsigned char kv[ST][2][TB];
    unsigned char q[QB][SPLIT ? 2 : 1][16 * HD * 2];
    union {
        PgSchedSmem sched;
        float o[kDecWarps][4][HD];                       // four rows of every warp's O
    };
    float wm[kDecWarps][16], wl[kDecWarps][16];
    uint64_t full[ST], freed[ST], qfull[2], qfreed[2], join;
    volatile uint32_t dead;
    int last;
};

template <typename CT>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// Byte offset of 16-byte piece c of row r of a tile: groups of 8 rows, in each the 64-dim blocks of 8 rows x
// 128 bytes, pieces permuted within the 128 bytes by the row (the swizzle).
template <int HD>
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
    return (uint32_t)((r >> 3) * (HD * 16) + (c >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <typename QT>
__device__ __forceinline__ void put_out(const PgAttnArgs &A, int hd, int row, int h, int d, float o) {
    if (A.gate) {
        const float g = A.gate[row * A.gate_ld + (long long)h * 2 * hd + hd + d];
        o = __fdiv_rn(o, 1.0f + expf(-g));
    }
    QT *dst = reinterpret_cast<QT *>(A.out) + ((size_t)row * A.H + h) * hd + d;
    if constexpr (sizeof(QT) == 4)
        *dst = o;
    else
        *dst = PgCvt<QT>::from(o);
}

template <typename CT, typename QT, int HD>
__global__ void __launch_bounds__(kDecThreads, HD == 256 ? 1 : 2)
    attn_paged_kernel(const __grid_constant__ PgMaps maps, const __grid_constant__ PgAttnArgs A, uint32_t *err) {
    constexpr bool SPLIT = sizeof(QT) == 4;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    using Smem = DecSmem<HD, SPLIT>;
    constexpr int ST = Smem::ST, TB = Smem::TB, QB = Smem::QB;
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    pdl_trigger();
    if (smem_u32(smem_raw) & 1023u) {  // the swizzled tiles need 1024-byte places
        pdl_wait();
        if (tid == 0) atomicOr(err, TRX_DEV_INTERNAL);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.freed[i], kDecWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.qfull[i], 1);
            mbar_init(&sm.qfreed[i], kDecWarps);
        }
        mbar_init(&sm.join, kDecWarps);
        sm.dead = 0u;
        mbar_fence_init();
        tma_prefetch_map(&maps.k);
        tma_prefetch_map(&maps.v);
    }
    pdl_wait();
    pg_schedule(A, sm.sched, 2, err);  // barriers inside: the set-up above is visible behind it
    const PgSched S = sm.sched.S;
    __syncthreads();
    PgWalk W;
    if (!W.start(A, S)) return;
    const uint32_t full = smem_u32(sm.full), freed = smem_u32(sm.freed), qfull = smem_u32(sm.qfull),
                   qfreed = smem_u32(sm.qfreed), joinb = smem_u32(&sm.join);
    auto wait = [&](uint32_t bar, uint32_t parity) {
        const bool ok = __all_sync(0xffffffffu, wait_phase(bar, parity & 1u, err));
        if (!ok) sm.dead = 1u;
        return ok;
    };
    if (warp == kDecWarps) {
        // Producer.
        const int br = min(1 << A.page_shift, kDecTile), boxes = kDecTile / br;  // rows of a box, boxes of a tile
        const int bi = lane & 15;
        static_assert(kDecTile / 16 <= 16, "a lane has one box");
        const int beyond = A.n_pages << A.page_shift;  // a row outside the maps: zeros
        const int my_pos = bi * br;
        const uint32_t my_dst = smem_u32(sm.kv) + (uint32_t)((lane >> 4) * TB + my_pos * HD * 2);
        const CUtensorMap *const map = lane < 16 ? &maps.k : &maps.v;
        const bool mine = bi < boxes;
        // This lane's table entry of tile it of a piece (-1 behind the sequence's end); looked at only when the box
        // is sent, so that the load's time is not waited for.
        auto pos_of = [&](const PgWalk &P, int it) { return P.R.tile(it) * kDecTile + my_pos; };
        auto id_of = [&](const PgWalk &P, int it) {
            const int p = pos_of(P, it);
            return mine && p < P.q.p0 + P.q.n ? __ldg(A.tables + (long long)P.b * A.max_pages + (p >> A.page_shift)) : -1;
        };
        int j = 0, piece = 0, it = W.i0;
        bool ok = true;
        int id = id_of(W, it);
        for (;;) {
            // The table is read a tile ahead.
            PgWalk N = W;
            int nit = it + 1;
            const bool more = nit < W.i1 || N.next(A);
            if (nit == W.i1) nit = N.i0;
            const int nid = more ? id_of(N, nit) : 0;
            const int st = j % ST;
            ok = !sm.dead && (j < ST || wait(freed + 8u * st, (uint32_t)(j / ST - 1)));
            if (!ok) break;
            if (lane == 0) mbar_expect_tx_s(full + 8u * st, 2u * TB);
            int row = beyond;
            if ((unsigned)id < (unsigned)A.n_pages)
                row = (id << A.page_shift) + (pos_of(W, it) & ((1 << A.page_shift) - 1));
            else if (mine && pos_of(W, it) < W.q.p0 + W.q.n)
                atomicOr(err, TRX_DEV_RANGE);
            __syncwarp();
            if (mine) load_box4(my_dst + (uint32_t)(st * 2 * TB), map, 0, 0, W.kh * (HD / 64), row / 8, full + 8u * st);
            __syncwarp();
            if (it == W.i0) {  // a new piece: its query rows, zeros behind them
                const int qb = piece % QB;
                ok = piece < QB || wait(qfreed + 8u * qb, (uint32_t)(piece / QB - 1));
                if (!ok) break;
                const int rows = W.rows(A), row0 = W.q.row0 + W.t * A.tq;
                // Rows behind the last keep what was there: every position is hidden from them.
                const QT *const src = reinterpret_cast<const QT *>(A.q) + ((long long)row0 * A.H + W.kh * A.rep) * HD;
                const int inv = (65536 + A.rep - 1) / A.rep;  // r / rep = r * inv >> 16 for r < 16
                constexpr int B = 4;                          // loads of a lane in flight
                for (int i0 = lane; i0 < rows * (HD / 8); i0 += 32 * B) {
                    uint4 x[B], y[SPLIT ? B : 1];
#pragma unroll
                    for (int e = 0; e < B; ++e) {
                        const int i = i0 + 32 * e, r = i / (HD / 8), tk = r * inv >> 16;
                        const QT *p = src + (long long)(tk * A.H + r - tk * A.rep) * HD + (i % (HD / 8)) * 8;
                        if (r < rows) {
                            x[e] = *reinterpret_cast<const uint4 *>(p);
                            if constexpr (SPLIT) y[e] = *reinterpret_cast<const uint4 *>(p + 4);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < B; ++e) {
                        const int i = i0 + 32 * e, r = i / (HD / 8);
                        if (r >= rows) break;
                        const uint32_t off = tile_off<HD>(r, i % (HD / 8));
                        if constexpr (SPLIT) {
                            const uint32_t f[8] = {x[e].x, x[e].y, x[e].z, x[e].w, y[e].x, y[e].y, y[e].z, y[e].w};
                            uint32_t hw[4], lw[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float f0 = __uint_as_float(f[2 * k]), f1 = __uint_as_float(f[2 * k + 1]);
                                hw[k] = PgCvt<CT>::pack(f0, f1);
                                const float2 h = PgCvt<CT>::unpack(hw[k]);
                                lw[k] = PgCvt<CT>::pack(f0 - h.x, f1 - h.y);
                            }
                            *reinterpret_cast<uint4 *>(&sm.q[qb][0][off]) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
                            *reinterpret_cast<uint4 *>(&sm.q[qb][SPLIT ? 1 : 0][off]) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
                        } else {
                            *reinterpret_cast<uint4 *>(&sm.q[qb][0][off]) = x[e];
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) arrive(qfull + 8u * qb);
                ++piece;
            }
            ++j;
            if (!more) break;
            W = N;
            it = nit;
            id = nid;
        }
        if (!ok) {
            // Whatever was issued has landed before the block leaves (bounded; the timeout is recorded).
            sm.dead = 1u;
            for (int st = 0; st < ST; ++st)
                for (int ph = 0; ph < 2; ++ph) wait_phase(full + 8u * st, ph, nullptr);
        }
        return;
    }
    uint32_t joined = 0;
    auto join = [&] {  // the four warps (bounded, unlike a block barrier)
        __syncwarp();
        if (lane == 0) arrive(joinb);
        return wait(joinb, joined++);
    };
    int j = 0, piece = 0;
    bool ok = true, more = true;
    while (ok && more) {
        const int rows = W.rows(A), len = W.q.p0 + W.q.n;
        const int row0 = W.q.row0 + W.t * A.tq, tok_pos = W.q.p0 + W.t * A.tq;
        const uint32_t qs = smem_u32(sm.q[piece % QB][0]);
        if (!wait(qfull + 8u * (piece % QB), (uint32_t)(piece / QB))) break;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        float o[HD / 8][4];
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        // Positions of rows g and g + 8 (-1 behind the last: everything hidden).
        const int qp[2] = {g < rows ? tok_pos + g / A.rep : -1, g + 8 < rows ? tok_pos + (g + 8) / A.rep : -1};
        for (int it = W.i0; it < W.i1; ++it, ++j) {
            const int st = j % ST;
            ok = wait(full + 8u * st, (uint32_t)(j / ST));
            if (!ok) break;
            const int k0 = W.R.tile(it) * kDecTile + warp * 16;
            const uint32_t ks = smem_u32(sm.kv[st][0]), vs = ks + TB;
            float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
            float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};  // the low parts' sums
            const int arow = (lane & 7) + ((lane >> 3) & 1) * 8, acol = lane >> 4;
            const int brow = warp * 16 + (lane & 7) + (lane >> 4) * 8, bcol = (lane >> 3) & 1;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                uint32_t a[4], b[4];
                ldsm4(qs + tile_off<HD>(arow, 2 * k + acol), a);
                ldsm4(ks + tile_off<HD>(brow, 2 * k + bcol), b);
                mma_16816<CT>(s0, a, b[0], b[1]);
                mma_16816<CT>(s1, a, b[2], b[3]);
                if constexpr (SPLIT) {
                    ldsm4(qs + 16 * HD * 2 + tile_off<HD>(arow, 2 * k + acol), a);
                    mma_16816<CT>(t0, a, b[0], b[1]);
                    mma_16816<CT>(t1, a, b[2], b[3]);
                }
            }
            if constexpr (SPLIT) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s0[e] += t0[e];
                    s1[e] += t1[e];
                }
            }
            // This warp's rows of V behind the sequence's end: zeros (0 times what lies there would not be 0
            // if it is not finite).
            if (k0 + 16 > len) {
                const int z0 = max(0, len - k0);
                for (int i = lane; i < (16 - z0) * (HD / 8); i += 32)
                    *reinterpret_cast<uint4 *>(&sm.kv[st][1][tile_off<HD>(warp * 16 + z0 + i / (HD / 8), i % (HD / 8))]) =
                        make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async();  // before the copy that refills the slot
                __syncwarp();
            }
            // Row g: s0[0], s0[1] at positions k0 + 2c, + 1, s1[0], s1[1] at k0 + 8 + 2c; row g + 8: [2], [3].
            uint32_t ph[4], pl[4];
            float alpha[2];
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                float x[4] = {s0[2 * rr], s0[2 * rr + 1], s1[2 * rr], s1[2 * rr + 1]};
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int kp = k0 + 2 * c + (e & 1) + (e >> 1) * 8;
                    x[e] = pg_hidden(kp, qp[rr], A.window, A.sinks) ? -INFINITY : x[e] * A.scale_log2;
                    mx = fmaxf(mx, x[e]);
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[rr], mx), ms = mn == -INFINITY ? 0.f : mn;
                const float al = ex2f(m[rr] - ms);
                float p[4], sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = ex2f(x[e] - ms);
                    if constexpr (!PgIsBf16<CT>::value) p[e] *= kSplitScale;  // at most 2^15 in one part or two
                    sum += p[e];
                }
                l[rr] = l[rr] * al + sum;
                m[rr] = mn;
                alpha[rr] = al;
                ph[rr] = PgCvt<CT>::pack(p[0], p[1]);
                ph[2 + rr] = PgCvt<CT>::pack(p[2], p[3]);
                if constexpr (SPLIT) {
                    const float2 h0 = PgCvt<CT>::unpack(ph[rr]), h1 = PgCvt<CT>::unpack(ph[2 + rr]);
                    pl[rr] = PgCvt<CT>::pack(p[0] - h0.x, p[1] - h0.y);
                    pl[2 + rr] = PgCvt<CT>::pack(p[2] - h1.x, p[3] - h1.y);
                }
            }
            const int vrow = warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, vcol = lane >> 4;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
                uint32_t b[4];
                ldsm4t(vs + tile_off<HD>(vrow, 2 * i + vcol), b);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float(&d)[4] = o[2 * i + h];
                    if constexpr (SPLIT) {
                        // The tensor core cuts its sums off instead of rounding them: over hundreds of tiles
                        // that adds up (1.8e-6 against 0.4e-6 at 30,000 positions), so each tile's product
                        // is summed alone and added by a rounded FMA.
                        float t[4] = {0.f, 0.f, 0.f, 0.f};
                        mma_16816<CT>(t, pl, b[2 * h], b[2 * h + 1]);
                        mma_16816<CT>(t, ph, b[2 * h], b[2 * h + 1]);
                        d[0] = fmaf(d[0], alpha[0], t[0]);
                        d[1] = fmaf(d[1], alpha[0], t[1]);
                        d[2] = fmaf(d[2], alpha[1], t[2]);
                        d[3] = fmaf(d[3], alpha[1], t[3]);
                    } else {
                        d[0] *= alpha[0];
                        d[1] *= alpha[0];
                        d[2] *= alpha[1];
                        d[3] *= alpha[1];
                        mma_16816<CT>(d, ph, b[2 * h], b[2 * h + 1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) arrive(freed + 8u * st);
        }
        if (!ok) break;
        if (lane == 0) arrive(qfreed + 8u * (piece % QB));
        ++piece;
        // The warps' parts of the piece, joined in their order, four rows at a time.  (A row sees its own position, so
        // its sum is never 0 unless its query is not finite: the quotient is then NaN, as by the formula.)
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 1);
            l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 2);
            if (c == 0) {
                sm.wm[warp][g + 8 * rr] = m[rr];
                sm.wl[warp][g + 8 * rr] = l[rr];
            }
        }
        const bool whole = W.whole();
        const long long item0 = W.u - W.i1, item1 = item0 + W.R.cnt;
        const int kh = W.kh;
        int c0 = 0, c1 = 0;
        if (!whole) {
            c0 = pg_owner(S, item0);
            c1 = pg_owner(S, item1 - 1);
        }
        constexpr size_t kPart = 16 * (HD + 2);  // a cut piece in scratch: maxima, sums, then O by row (16-byte places)
        auto slot_of = [&](int cc) { return A.part + kPart * (2 * (size_t)cc + (cc == c0 ? 1 : 0)); };
        float *const part = slot_of(blockIdx.x);
        for (int r0 = 0; ok && r0 < rows; r0 += 4) {
            // Lanes of rows r0..r0+3: g or g + 8.
            const int rr = r0 >= 8 ? 1 : 0, lr = g + 8 * rr - r0;
            if (lr >= 0 && lr < 4) {
#pragma unroll
                for (int i = 0; i < HD / 8; ++i)
                    *reinterpret_cast<float2 *>(&sm.o[warp][lr][8 * i + 2 * c]) =
                        rr ? make_float2(o[i][2], o[i][3]) : make_float2(o[i][0], o[i][1]);
            }
            ok = join();
            if (!ok) break;
            const int nr = min(4, rows - r0);
            for (int i = tid; i < nr * HD; i += 32 * kDecWarps) {
                const int r = i / HD, d = i - r * HD, R = r0 + r, tk = R / A.rep;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sm.wm[w][R]);
                const float Ms = M == -INFINITY ? 0.f : M;
                float L = 0.f, acc = 0.f;
#pragma unroll
                for (int w = 0; w < kDecWarps; ++w) {
                    const float e = ex2f(sm.wm[w][R] - Ms);
                    L = fmaf(e, sm.wl[w][R], L);
                    acc = fmaf(e, sm.o[w][r][d], acc);
                }
                if (whole) {
                    put_out<QT>(A, HD, row0 + tk, kh * A.rep + R - tk * A.rep, d, __fdiv_rn(acc, L));
                } else {
                    part[32 + R * HD + d] = acc;
                    if (d == 0) {
                        part[R] = M;
                        part[16 + R] = L;
                    }
                }
            }
            ok = join();
        }
        if (!ok) break;
        if (!whole) {
            // The last CTA to arrive joins the pieces in CTA order.
            __threadfence();
            ok = join();
            if (!ok) break;
            if (tid == 0) sm.last = atomicAdd(A.cnt + c0, 1u) == (unsigned)(c1 - c0);
            ok = join();
            if (!ok) break;
            if (sm.last) {
                __threadfence();
                // Four dims of a row per thread; the pieces of a round all in flight.
                for (int i = 4 * tid; i < rows * HD; i += 4 * 32 * kDecWarps) {
                    const int r = i / HD, d = i - r * HD, tk = r / A.rep;
                    float M = -INFINITY, L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
                    for (int cc = c0; cc <= c1; cc += 4) {
                        float pm[4], pl[4];
                        float4 po[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float *p = slot_of(min(cc + e, c1));
                            pm[e] = cc + e <= c1 ? __ldcg(p + r) : -INFINITY;
                            pl[e] = __ldcg(p + 16 + r);
                            po[e] = __ldcg(reinterpret_cast<const float4 *>(p + 32 + i));
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float Mn = fmaxf(M, pm[e]), Ms = Mn == -INFINITY ? 0.f : Mn;
                            const float f = ex2f(M - Ms), w = ex2f(pm[e] - Ms);
                            M = Mn;
                            L = fmaf(w, pl[e], L * f);
                            acc[0] = fmaf(w, po[e].x, acc[0] * f);
                            acc[1] = fmaf(w, po[e].y, acc[1] * f);
                            acc[2] = fmaf(w, po[e].z, acc[2] * f);
                            acc[3] = fmaf(w, po[e].w, acc[3] * f);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        put_out<QT>(A, HD, row0 + tk, kh * A.rep + r - tk * A.rep, d + e, __fdiv_rn(acc[e], L));
                }
                if (tid == 0) A.cnt[c0] = 0u;
            }
        }
        more = W.next(A);
    }
    if (!ok) sm.dead = 1u;
}

template <typename CT, typename QT, int HD>
trx_status launch_dec(PgAttnArgs A, size_t part_cap, int cnt_cap, uint32_t *err, cudaStream_t st) {
    constexpr size_t smem = sizeof(DecSmem<HD, sizeof(QT) == 4>);
    static_assert(smem <= (HD == 256 ? 232448 : 115712), "one CTA (head dim 256) or two per SM");
    static DevBits configured{0};
    const cudaError_t e = once_per_device(configured, [] {
        return cudaFuncSetAttribute(attn_paged_kernel<CT, QT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    });
    if (e != cudaSuccess) return note_cuda(e);
    A.tq = 16 / A.rep;
    A.kt_shift = 6;
    PgMaps maps;
    if (!pg_encode_pools<HD>(maps, A, 1u << (A.page_shift < 6 ? A.page_shift : 6))) return TRX_ERR_CUDA;
    const int grid = device_sms() * (HD == 256 ? 1 : 2);
    if ((size_t)grid * 2 * 16 * (HD + 2) > part_cap || grid > cnt_cap) return TRX_ERR_UNSUPPORTED;
    return note_cuda(launch_kernel(attn_paged_kernel<CT, QT, HD>, dim3(grid), dim3(kDecThreads), smem, st, maps, A, err));
}

template <typename CT, typename QT>
trx_status launch_dec_hd(const PgAttnArgs &A, int hd, size_t part_cap, int cnt_cap, uint32_t *err, cudaStream_t st) {
    switch (hd) {
        case 64: return launch_dec<CT, QT, 64>(A, part_cap, cnt_cap, err, st);
        case 128: return launch_dec<CT, QT, 128>(A, part_cap, cnt_cap, err, st);
        default: return launch_dec<CT, QT, 256>(A, part_cap, cnt_cap, err, st);
    }
}

template <typename CT, typename QT>
trx_status launch_app_hd(const PgAppendArgs &A, uint32_t *err, cudaStream_t st) {
    // Blocks per row: enough to give every SM a block when there are few rows.
    const int hpb = kAppThreads / (A.hd / 8), most = (A.H + 2 * A.Hkv + hpb - 1) / hpb;
    int ny = (2 * device_sms() + A.max_rows - 1) / A.max_rows;
    ny = ny < 1 ? 1 : (ny > most ? most : ny);
    const int nx = A.max_rows < 65536 ? A.max_rows : 65536;
    const dim3 grid(nx, ny), block(kAppThreads);
    switch (A.hd) {
        case 64: return note_cuda(launch_kernel(paged_append_kernel<CT, QT, 64>, grid, block, 0, st, A, err));
        case 128: return note_cuda(launch_kernel(paged_append_kernel<CT, QT, 128>, grid, block, 0, st, A, err));
        default: return note_cuda(launch_kernel(paged_append_kernel<CT, QT, 256>, grid, block, 0, st, A, err));
    }
}

int shift_of(uint32_t page) {
    int s = 0;
    while ((1u << s) < page) ++s;
    return s;
}

}  // namespace

trx_status launch_paged_plan(const trx_pages &P, const int *cached, const int *fresh, const int *free_pages,
                             uint32_t free_cap, const int *n_free, uint32_t *err, cudaStream_t st) {
    // Blocks: one per 2048 rows, at most a portable cluster.
    int nb = 1;
    while (nb < 8 && (uint32_t)nb * 2048 < P.max_rows) nb *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(nb);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = nb;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return note_cuda(cudaLaunchKernelEx(&cfg, paged_plan_kernel, P, shift_of(P.page), cached, fresh, free_pages, free_cap,
                                        n_free, err));
}

trx_status launch_paged_release(const trx_pages &P, const int *done, int *lens, int *free_pages, int *n_free,
                                uint32_t *err, cudaStream_t st) {
    return note_cuda(launch_kernel(paged_release_kernel, dim3(1), dim3(kPlanThreads), 0, st, P, shift_of(P.page), done,
                                   lens, free_pages, n_free, err));
}

trx_status launch_paged_append(const PgAppendArgs &A, int cache_type, int q_type, uint32_t *err, cudaStream_t st) {
    if (cache_type == TRX_TYPE_F16)
        return q_type == TRX_TYPE_F32 ? launch_app_hd<__half, float>(A, err, st) : launch_app_hd<__half, __half>(A, err, st);
    return q_type == TRX_TYPE_F32 ? launch_app_hd<__nv_bfloat16, float>(A, err, st)
                                  : launch_app_hd<__nv_bfloat16, __nv_bfloat16>(A, err, st);
}

trx_status launch_attn_paged(const PgAttnArgs &A, int hd, int cache_type, int q_type, size_t part_cap, int cnt_cap,
                             uint32_t *err, cudaStream_t st) {
    // More query rows per kv head than the 16 of one mma.sync tile: the tcgen05 kernel, whose 128-row tiles would
    // be mostly padding below.  In a graph 16 sequences of 900 tokens, 4 (or 16) rows per kv head, take 18.5 (24.2) us
    // here, 24.6 (24.7) there; 3 sequences of 30,000 tokens, fp32 queries: 70 us here, 109 there.
    if ((long long)A.max_new * A.rep > 16) return launch_attn_paged_tc(A, hd, cache_type, q_type, part_cap, cnt_cap, err, st);
    if (cache_type == TRX_TYPE_BF16)
        return launch_dec_hd<__nv_bfloat16, __nv_bfloat16>(A, hd, part_cap, cnt_cap, err, st);
    return q_type == TRX_TYPE_F32 ? launch_dec_hd<__half, float>(A, hd, part_cap, cnt_cap, err, st)
                                  : launch_dec_hd<__half, __half>(A, hd, part_cap, cnt_cap, err, st);
}

}  // namespace trx
