// Attention of prompt chunks over a paged KV cache on the 5th-generation tensor cores (sm_100a
// tcgen05, kind::f16): the same computation as attn_paged_kernel (trx_paged.cu), for sequences with
// more than 16 query rows per kv head.
//
// Work: a query tile is 128 rows of one kv head, (token, head of the group) pairs in order: 128 / rep
// tokens x rep heads (padded).  A CTA walks its pieces (PgSched): key tiles of KT positions of one
// (query tile, kv head).  Per key tile S = Q K^T (M = 128, N = KT), the softmax in 32 bits, O += P V
// (M = 128, N = head dim).  Warp roles:
//  * warps 0-3: one query row per thread (its TMEM lane).  They put an fp32 query tile into shared memory (a
//    16-bit one comes by TMA), read S from tensor memory, keep the row's maximum and sum, write P (16 bits) over
//    S as the A operand of the second product, and finish the piece.  O is rescaled only when a row's maximum has grown by
//    more than 2^8 over the one in use: P then stays below 2^8 (fp16: 2^15, see kHalfBits), exact in any 16-bit
//    float's exponent.
//  * warp 4: the producer.  A key tile is gathered by TMA boxes of one page (or the tile's part of it, see
//    PgMaps); places behind the sequence's end come from outside the map, as zeros.
//  * warps 5 and 6: issue the MMAs of the first and of the second product, each from one elected lane. Two
//    warps, since one's instructions between two MMAs (waits, commits) take as long as the MMAs.
// fp32 queries: Q = hi + lo and P = hi + lo in fp16 (P and its sum times 2^15, see kSplitScale), two MMAs per
// product, so products keep 2^-22; each tile's P V is added to an O in registers (head dim 256: tensor memory)
// by the softmax warps.
// V is read as the N-major B operand of the second product straight from its row-major tile; the rows
// of a sequence's last page behind its end are overwritten with zeros first (0 times what lies there
// would not be 0 if it is not finite).
//
// Two S buffers: the next tile's S is computed while this one's softmax runs.  Head dims 64 and 128 run
// two CTAs per SM (at most 113 KB of shared memory, 256 TMEM columns each), head dim 256 and fp32 queries
// one.
//
// What bounds it (launches in a row or in a graph; tensor pipe and cycles by ncu):
//  - 16-bit heads of 128: the products and the power they draw.  2,048 rows of 32 heads behind 6,001 positions: 231 us,
//    1,020 TFLOP/s, in short runs, 276 us in long ones.  1,032 cycles a tile of 128 x 64, its MMAs' math 512 (pipe at
//    50 %): S, 64 keys wide, reads 6 KB of shared memory (48 cycles) for 32 cycles of math, so 640 at least.
//  - fp32 queries: the softmax warps, one per scheduler.  4,096 rows of 16 heads, a window of 1,024: 137 to 141 us,
//    3,750 cycles a tile, ends of pieces included, its MMAs 1,024 (27 %).
//  - heads of 256: the ends of pieces, and K and V from L2 (64 KB a tile).  1,137 rows of 24 gated heads, 9 sequences:
//    101 us, 3,470 cycles a tile, its MMAs 1,024 (30 %); 32 bytes a cycle and SM from L2 over the whole launch.
#include <algorithm>
#include <cstdint>
#include <cstring>
#include <cuda.h>
#include <cuda_runtime.h>

#include "trx_paged.cuh"

namespace trx {
namespace {

constexpr int kTcThreads = 256;
constexpr int kTcRows = 128;  // query rows of a tile: the MMA's M, the TMEM lanes

template <int HD, bool SPLIT>
struct TcCfg {
    static constexpr int KT = 64, KT_SHIFT = 6;                   // key positions of a tile
    static constexpr int NS = 2;                                  // S buffers (the barriers' pairs)
    static constexpr int KST = SPLIT && HD == 256 ? 1 : 2;       // K and V tiles in shared memory
    static constexpr int CTAS = SPLIT || HD == 256 ? 1 : 2;      // per SM
    // Tensor memory.  16-bit: O [HD], S [2][KT].  Split: a tile's P V [NACC][NW], S [2][KT], and for head
    // dim 256, whose O does not fit the registers, O [256] in front.
    static constexpr bool REGO = SPLIT && HD <= 128;             // O in registers
    static constexpr int NACC = REGO ? 2 : 1, NW = SPLIT && HD == 256 ? 128 : HD, NCH = HD / NW;
    static constexpr int AOFF = SPLIT && !REGO ? HD : 0, SOFF = AOFF + NACC * NW;
    static constexpr int TMEM = SOFF + NS * KT <= 256 ? 256 : 512;
    static constexpr int QBYTES = kTcRows * HD * 2, TBYTES = KT * HD * 2;
    static constexpr int QOFF = 0, KOFF = QBYTES * (SPLIT ? 2 : 1), VOFF = KOFF + KST * TBYTES,
                         END = VOFF + KST * TBYTES;  // multiples of 1024
    // Gates through shared memory (a ring of three pieces of 16 dims per row, behind the tail) where there is
    // room for it: head dim 256 with 16-bit queries.
    static constexpr bool RING = !SPLIT && HD == 256;
    static constexpr int GBYTES = RING ? 3 * kTcRows * 64 : 0;
    static_assert(SOFF + NS * KT <= 512 && TMEM * CTAS <= 512, "tensor memory holds O and every S");
};

struct TcBars {
    // Tile j of the CTA is phase j / KST of barrier j % KST, or phase j / 2 of barrier j % 2.
    uint64_t kfull[2], vfull[2];   // the K, V tile has landed
    uint64_t sfull[2];             // Q K^T is complete: S is there, the K tile is free
    uint64_t pready[2];            // P is in the place of S (4 warps)
    uint64_t odone[2];             // P V is complete: O, the V tile and the S buffer are free
    uint64_t cdone[2], ofree[2];   // split: part n of P V is complete; it has been added to O (4 warps)
    uint64_t qready;               // the query tile is in shared memory (split: 4 warps; else by TMA)
    uint64_t fin[2];               // every MMA of warps 5 and 6
    uint32_t tmem;
    volatile uint32_t dead;        // a wait ran out somewhere in the block
};

struct TcTail {  // behind the tiles
    TcBars bars;
    PgSchedSmem sched;
};
static_assert(sizeof(TcTail) % 16 == 0 && TcCfg<256, false>::END + sizeof(TcTail) + TcCfg<256, false>::GBYTES <= 232448,
              "the gates' ring is aligned and fits");

__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// K-major operand tile, 128-byte swizzle: rows of 64 16-bit elements in groups of 8 (1024 bytes), `group` bytes
// apart.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t a, uint32_t group) {
    return (uint64_t)((a >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) | ((uint64_t)(group >> 4) << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
// N-major operand tile, 128-byte swizzle: 64 N elements contiguous, K rows 128 bytes apart in groups of 8,
// `group` bytes apart, the next 64 N elements `block` bytes on.
__device__ __forceinline__ uint64_t desc_nmajor(uint32_t a, uint32_t group, uint32_t block) {
    return (uint64_t)((a >> 4) & 0x3FFFu) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(group >> 4) << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
// Instruction descriptor of kind::f16: D fp32, A and B fp16 (0) or bf16 (1), B N-major if bn, N, M = 128.
template <typename CT>
__device__ __forceinline__ uint32_t idesc_f16(int n, bool bn) {
    constexpr uint32_t t = PgIsBf16<CT>::value ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | ((bn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kTcRows >> 4) << 24);
}

// Four MMAs (64 of K) issued by one elected lane of the converged warp (all lanes execute; operands are
// warp-uniform).  A and B from shared memory, K-major: a step of 16 elements is 32 bytes.
__device__ __forceinline__ void mma_ss4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p, e, t;\n .reg .b64 a1, a2, a3, b1, b2, b3;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n"
        " add.s64 a1, %1, 2;\n add.s64 a2, %1, 4;\n add.s64 a3, %1, 6;\n"
        " add.s64 b1, %2, 2;\n add.s64 b2, %2, 4;\n add.s64 b3, %2, 6;\n"
        " elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((int)acc)
        : "memory");
}
// A from tensor memory at columns a0..a3, B N-major: a step of 16 rows is two groups.
template <int HD>
__device__ __forceinline__ void mma_ts4(uint32_t d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint64_t b,
                                        uint32_t idesc, bool acc) {
    constexpr int step = 2 * (HD / 64) * 1024 / 16;
    asm volatile(
        "{\n .reg .pred p, e, t;\n .reg .b64 b1, b2, b3;\n setp.ne.b32 p, %7, 0;\n setp.eq.b32 t, 0, 0;\n"
        " add.s64 b1, %5, %8;\n add.s64 b2, %5, %9;\n add.s64 b3, %5, %10;\n"
        " elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %5, %6, p;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%2], b1, %6, t;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%3], b2, %6, t;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%4], b3, %6, t;\n}\n" ::"r"(d),
        "r"(a0), "r"(a1), "r"(a2), "r"(a3), "l"(b), "r"(idesc), "r"((int)acc), "n"(step), "n"(2 * step), "n"(3 * step)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile(
        "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar)
        : "memory");
}
// Tensor memory, one lane per thread, 32 (or 16) consecutive columns.
__device__ __forceinline__ void tm_ld32(uint32_t a, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t a, const uint32_t (&o)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
        "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]), "r"(o[8]), "r"(o[9]),
        "r"(o[10]), "r"(o[11]), "r"(o[12]), "r"(o[13]), "r"(o[14]), "r"(o[15]), "r"(o[16]), "r"(o[17]), "r"(o[18]),
        "r"(o[19]), "r"(o[20]), "r"(o[21]), "r"(o[22]), "r"(o[23]), "r"(o[24]), "r"(o[25]), "r"(o[26]), "r"(o[27]),
        "r"(o[28]), "r"(o[29]), "r"(o[30]), "r"(o[31])
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t a, const uint32_t (&o)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(a),
        "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]), "r"(o[8]), "r"(o[9]),
        "r"(o[10]), "r"(o[11]), "r"(o[12]), "r"(o[13]), "r"(o[14]), "r"(o[15])
        : "memory");
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The gates of a piece on their way to a warp's ring: 16 dims of its 32 rows at a time, each row's 64 bytes read
// by four lanes together, kept swizzled so that a lane per row reads them without conflicts.  With loads by the
// thread of a row at the time of use (32 lines per access, one round trip per 32 dims) 1,137 rows of 24 gated heads of
// 256 took 114 us, this way 101.
struct GateRing {
    uint32_t at;       // shared address of the warp's ring
    long long row0;    // the piece's first row and head, its rows
    int head0, rows;
    int next, slot;    // the next 16 dims to be sent for; the slot of the next to be used
    __device__ __forceinline__ void send(const PgAttnArgs &A, int hd, int s) {
        const int lane = threadIdx.x & 31, inv = (65536 + A.rep - 1) / A.rep;
        if (16 * next < hd) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int wr = 8 * i + (lane >> 2), r = (threadIdx.x & ~31) + wr, tok = r * inv >> 16, u = lane & 3;
                const float *g = A.gate + (row0 + tok) * A.gate_ld + (long long)(head0 + r - tok * A.rep) * 2 * hd + hd +
                                 16 * next + 4 * u;
                if (r < rows)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + s * (kTcRows * 64) + wr * 64 +
                                                                                   ((u ^ (wr >> 1 & 3)) << 4)),
                                 "l"(g)
                                 : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ++next;
    }
    __device__ __forceinline__ void drain() const { asm volatile("cp.async.wait_all;" ::: "memory"); }
    // The first three of a piece; what an unfinished piece left on its way lands first.
    __device__ __forceinline__ void start(const PgAttnArgs &A, int hd) {
        drain();
        __syncwarp();
        next = slot = 0;
        for (int s = 0; s < 3; ++s) send(A, hd, s);
    }
    // The next 16 gates of this lane's row; another 16 dims are sent for.
    __device__ __forceinline__ void take(const PgAttnArgs &A, int hd, float4 (&g)[4]) {
        const int lane = threadIdx.x & 31;
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 4; ++u)
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(g[u].x), "=f"(g[u].y), "=f"(g[u].z), "=f"(g[u].w)
                         : "r"(at + slot * (kTcRows * 64) + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4))
                         : "memory");
        __syncwarp();
        send(A, hd, slot);
        slot = slot == 2 ? 0 : slot + 1;
    }
};

// 32 outputs of one row (row < 0: none; every lane of the warp takes part), dims d..d+31.
template <typename QT, bool RING>
__device__ __forceinline__ void put32(const PgAttnArgs &A, GateRing &G, int hd, int row, int h, int d, float (&o)[32]) {
    if (A.gate) {
        const float4 *gp = nullptr;
        if constexpr (!RING)
            gp = reinterpret_cast<const float4 *>(A.gate + (row < 0 ? 0 : row) * A.gate_ld + (long long)h * 2 * hd + hd + d);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float4 g[4];
            if constexpr (RING) {
                G.take(A, hd, g);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) g[i] = gp[4 * n + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float *const v = &o[16 * n + 4 * i];
                v[0] = __fdividef(v[0], 1.0f + expf(-g[i].x));
                v[1] = __fdividef(v[1], 1.0f + expf(-g[i].y));
                v[2] = __fdividef(v[2], 1.0f + expf(-g[i].z));
                v[3] = __fdividef(v[3], 1.0f + expf(-g[i].w));
            }
        }
    }
    if (row < 0) return;
    QT *dst = reinterpret_cast<QT *>(A.out) + ((size_t)row * A.H + h) * hd + d;
    if constexpr (sizeof(QT) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            reinterpret_cast<float4 *>(dst)[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            reinterpret_cast<uint4 *>(dst)[i] =
                make_uint4(PgCvt<QT>::pack(o[8 * i], o[8 * i + 1]), PgCvt<QT>::pack(o[8 * i + 2], o[8 * i + 3]),
                           PgCvt<QT>::pack(o[8 * i + 4], o[8 * i + 5]), PgCvt<QT>::pack(o[8 * i + 6], o[8 * i + 7]));
    }
}

// The fp32 query tile into shared memory as two fp16 parts (K-major, 128-byte swizzle), zeros behind its rows;
// sixteen 16-byte loads of a thread in flight at a time.
template <typename CT, typename QT, int HD>
__device__ __forceinline__ void load_query(const PgAttnArgs &A, unsigned char *smem, int r, int rows, int row0, int head0) {
    using C = TcCfg<HD, true>;
    constexpr int PPR = HD / 8, B = 8;            // pieces of 8 elements per row, of a batch
    const int inv = (65536 + A.rep - 1) / A.rep;  // qr / rep = qr * inv >> 16 for qr < 128, rep <= 16
    const int c = r % PPR;
    const uint32_t coff = (uint32_t)((c / 8) * (kTcRows * 128));
    const QT *const src = reinterpret_cast<const QT *>(A.q) + ((long long)row0 * A.H + head0) * HD + c * 8;
#pragma unroll 1
    for (int i0 = 0; i0 < PPR; i0 += B) {
        uint4 x[B], y[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int qr = (i0 + b) * (kTcRows / PPR) + r / PPR, tk = qr * inv >> 16;
            const QT *p = src + (long long)(tk * A.H + qr - tk * A.rep) * HD;
            x[b] = y[b] = make_uint4(0u, 0u, 0u, 0u);
            if (qr < rows) {
                x[b] = *reinterpret_cast<const uint4 *>(p);
                y[b] = *reinterpret_cast<const uint4 *>(p + 4);
            }
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int qr = (i0 + b) * (kTcRows / PPR) + r / PPR;
            unsigned char *const dst = smem + C::QOFF + coff + qr * 128 + (((c % 8) ^ (qr & 7)) << 4);
            const uint32_t f[8] = {x[b].x, x[b].y, x[b].z, x[b].w, y[b].x, y[b].y, y[b].z, y[b].w};
            uint32_t hw[4], lw[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float f0 = __uint_as_float(f[2 * e]), f1 = __uint_as_float(f[2 * e + 1]);
                hw[e] = PgCvt<CT>::pack(f0, f1);
                const float2 h = PgCvt<CT>::unpack(hw[e]);
                lw[e] = PgCvt<CT>::pack(f0 - h.x, f1 - h.y);
            }
            *reinterpret_cast<uint4 *>(dst) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
            *reinterpret_cast<uint4 *>(dst + C::QBYTES) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
        }
    }
}

// A row's output from its O, 32 dims at a time from get (row < 0: none; every lane of the warp takes part).
// REG: get reads registers, so the loops are unrolled.
template <typename QT, int HD, bool REG, bool RING, typename Get>
__device__ __forceinline__ void finish_whole(const PgAttnArgs &A, GateRing &G, Get &&get, float l, int row, int head) {
    if (!__any_sync(0xffffffffu, row >= 0)) return;
    const float inv = __fdiv_rn(1.0f, l);  // l = 0 or NaN: a query that is not finite; its outputs are NaN
#pragma unroll (REG ? HD / 32 : 1)
    for (int c = 0; c < HD / 32; ++c) {
        uint32_t v[32];
        get(c, v);
        float o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(v[e]) * inv;
        put32<QT, RING>(A, G, HD, row, head, 32 * c, o);
    }
}

// A cut item: this piece's rows to scratch, [HD / 4][128 rows] of four dims, then the maxima and sums; the
// last to arrive joins the pieces in the order of the CTAs (its own still from get).  The warps
// arrive and join on their own, 32 rows each.
template <typename QT, int HD, bool REG, bool RING, typename Get>
__device__ __forceinline__ void finish_cut(const PgAttnArgs &A, const PgSched &S, GateRing &G, Get &&get, long long item0,
                                           long long item1, float m, float l, int row, int head) {
    constexpr size_t kPart = kTcRows * (HD + 2);
    if (!__any_sync(0xffffffffu, row >= 0)) return;  // none of this warp's rows exist (the same in every piece)
    const int r = threadIdx.x, lane = r & 31, me = (int)blockIdx.x;
    const int c0 = pg_owner(S, item0), c1 = pg_owner(S, item1 - 1);
    unsigned *const cnt = A.cnt + 4 * c0 + (r >> 5);
    auto slot_of = [&](int cc) { return A.part + kPart * (2 * (size_t)cc + (cc == c0 ? 1 : 0)); };
    {
        float *const mine = slot_of(me);
#pragma unroll (REG ? HD / 32 : 1)
        for (int c = 0; c < HD / 32; ++c) {
            uint32_t v[32];
            get(c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                reinterpret_cast<uint4 *>(mine)[(8 * c + e) * kTcRows + r] =
                    make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
        }
        mine[kTcRows * HD + r] = m;
        mine[kTcRows * (HD + 1) + r] = l;
        __threadfence();
        __syncwarp();
        unsigned seen = 0;
        if (lane == 0) seen = atomicAdd(cnt, 1u);
        seen = __shfl_sync(0xffffffffu, seen, 0);
        if (seen != (unsigned)(c1 - c0)) return;
    }
    __threadfence();
    // The pieces' maxima and sums, four pieces' loads at a time.
    float M = -INFINITY, L = 0.f;
    for (int cc = c0; cc <= c1; cc += 4) {
        float pm[4], pl[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float *p = slot_of(min(cc + e, c1)) + kTcRows * HD + r;
            pm[e] = cc + e <= c1 ? __ldcg(p) : -INFINITY;
            pl[e] = __ldcg(p + kTcRows);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float Mn = fmaxf(M, pm[e]), Mz = Mn == -INFINITY ? 0.f : Mn;
            L = fmaf(ex2f(pm[e] - Mz), pl[e], L * ex2f(M - Mz));
            M = Mn;
        }
    }
    const float Ms = M == -INFINITY ? 0.f : M;
    const float inv = __fdiv_rn(1.0f, L);
    constexpr int GC = HD == 256 ? 2 : 1;  // 32 dims at a time, or 64: loads in flight
#pragma unroll (REG ? HD / 32 : 1)
    for (int c = 0; c < HD / 32; c += GC) {
        float o[GC][32];
#pragma unroll
        for (int g = 0; g < GC; ++g)
#pragma unroll
            for (int e = 0; e < 32; ++e) o[g][e] = 0.f;
#pragma unroll 1
        for (int cc = c0; cc <= c1; ++cc) {
            uint32_t v[GC][32];
            float w;
            if (cc == me) {
#pragma unroll
                for (int g = 0; g < GC; ++g) get(c + g, v[g]);
                w = ex2f(m - Ms);
            } else {
                const float *p = slot_of(cc);
                w = __ldcg(p + kTcRows * HD + r);
#pragma unroll
                for (int g = 0; g < GC; ++g)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint4 x = __ldcg(reinterpret_cast<const uint4 *>(p) + (8 * (c + g) + e) * kTcRows + r);
                        v[g][4 * e] = x.x;
                        v[g][4 * e + 1] = x.y;
                        v[g][4 * e + 2] = x.z;
                        v[g][4 * e + 3] = x.w;
                    }
                w = ex2f(w - Ms);
            }
#pragma unroll
            for (int g = 0; g < GC; ++g)
#pragma unroll
                for (int e = 0; e < 32; ++e) o[g][e] = fmaf(w, __uint_as_float(v[g][e]), o[g][e]);
        }
#pragma unroll
        for (int g = 0; g < GC; ++g) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[g][e] *= inv;
            put32<QT, RING>(A, G, HD, row, head, 32 * (c + g), o[g]);
        }
    }
    __syncwarp();
    if (lane == 0) *cnt = 0u;
}

// A tile's weights where scores lie beyond kFar (in powers of 2).  One FMA gives a weight's exponent elsewhere, and
// m was rounded to 32 bits: from there on that is no longer a small common factor of the row's weights, but 2^16 and
// more, or 2^-64.  So the products are rounded as m was, the largest to m itself.  A function, reading the row of S
// again (visible: k <= hi and (k >= lo or k < sk)): in the loop this cost 12 % of a long chunk with fp32 queries; this
// way the question costs 1 to 2.5 % (2,048 rows behind 6,001 positions in fp16: 231 us in short runs, 226 without;
// differences of scores instead of products for every tile: 243).
constexpr float kFar = 0x1p20f;
template <typename CT, bool SPLIT>
__device__ __noinline__ float far_weights(const PgAttnArgs &A, uint32_t ts, bool far, float m, int hi, int k0) {
    const float scale = A.scale_log2, bits = SPLIT ? kSplitBits : 0.f, nm = m == -INFINITY ? 0.f : bits - m;
    const int lo = A.window ? hi - A.window + 1 : -1, sk = A.sinks - k0;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
        uint32_t v[32], ph[16];
        // Column 32 c of S is read before anything is written there.
        tm_ld32(ts + 32 * c, v);
        tm_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const int k = 32 * c + e;
            const float x = k > hi || (k < lo && k >= sk) ? -INFINITY : __uint_as_float(v[e]);
            const float near = fmaf(x, scale, nm);
            const float p = ex2f(far ? __fadd_rn(__fsub_rn(__fmul_rn(x, scale), m), bits) : near);
            v[e] = __float_as_uint(p);
            sum[e & 3] += p;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) ph[e] = PgCvt<CT>::pack(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
        if constexpr (SPLIT) {
            tm_st16(ts + 32 * c, ph);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float2 b = PgCvt<CT>::unpack(ph[e]);
                ph[e] = PgCvt<CT>::pack(__uint_as_float(v[2 * e]) - b.x, __uint_as_float(v[2 * e + 1]) - b.y);
            }
            tm_st16(ts + 32 * c + 16, ph);
        } else {
            tm_st16(ts + 16 * c, ph);
        }
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <typename CT, typename QT, int HD>
__global__ void __launch_bounds__(kTcThreads, HD == 256 || sizeof(QT) == 4 ? 1 : 2)
    attn_paged_tc_kernel(const __grid_constant__ PgMaps maps, const __grid_constant__ PgAttnArgs A, uint32_t *err) {
    constexpr bool SPLIT = sizeof(QT) == 4;
    using C = TcCfg<HD, SPLIT>;
    constexpr int KT = C::KT, NS = C::NS, KST = C::KST;
    extern __shared__ __align__(1024) unsigned char smem[];
    TcTail &tail = *reinterpret_cast<TcTail *>(smem + C::END);
    TcBars &bars = tail.bars;
    PgSchedSmem &sched = tail.sched;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = smem_u32(smem);
    if (sbase & 1023u) {  // the swizzled tiles need 1024-byte places
        pdl_wait();
        if (tid == 0) atomicOr(err, TRX_DEV_INTERNAL);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.kfull[i], 1);
            mbar_init(&bars.vfull[i], 1);
            mbar_init(&bars.sfull[i], 1);
            mbar_init(&bars.pready[i], 4);
            mbar_init(&bars.odone[i], 1);
            mbar_init(&bars.cdone[i], 1);
            mbar_init(&bars.ofree[i], 4);
        }
        mbar_init(&bars.qready, SPLIT ? 4 : 1);
        mbar_init(&bars.fin[0], 1);
        mbar_init(&bars.fin[1], 1);
        bars.dead = 0u;
        mbar_fence_init();
        tma_prefetch_map(&maps.k);
        tma_prefetch_map(&maps.v);
        if (!SPLIT) tma_prefetch_map(&maps.q);
    }
    pdl_wait();
    // Tensor memory is taken only now that the kernel in front has ended, and the kernel behind is let in
    // only once it is taken: a neighbour that allocates before it waits could otherwise hold what this
    // one needs while it waits for this one.
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)),
                     "r"(C::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    pg_schedule(A, sched, 4, err);  // barriers inside: the allocation and the barriers' set-up are visible behind it
    tc_after();
    pdl_trigger();
    const uint32_t tmem = bars.tmem;
    const PgSched &S = sched.S;
    const uint32_t kfull = smem_u32(bars.kfull), vfull = smem_u32(bars.vfull), sfull = smem_u32(bars.sfull),
                   pready = smem_u32(bars.pready), odone = smem_u32(bars.odone), cdone = smem_u32(C::NCH == 1 ? bars.odone : bars.cdone),
                   ofree = smem_u32(bars.ofree), qready = smem_u32(&bars.qready),
                   fin = smem_u32(bars.fin);
    // Every lane of a warp waits; false for all of them if any wait ran out.
    auto wait = [&](uint32_t bar, uint32_t parity) {
        const bool ok = __all_sync(0xffffffffu, wait_phase(bar, parity & 1u, err));
        if (!ok) bars.dead = 1u;
        return ok;
    };
    // Tile j's phase of a pair of barriers.
    auto wait2 = [&](uint32_t bar, int j) { return wait(bar + 8u * (j & 1), (uint32_t)(j >> 1)); };
    PgWalk W;
    const bool any = W.start(A, S);
    if (any && warp == 4) {
        // Producer.
        const int br = min(1 << A.page_shift, KT), boxes = KT / br;  // rows of a box, boxes of a tile
        const int beyond = A.n_pages << A.page_shift;  // a row outside the maps: zeros
        static_assert(KT / 16 <= 32, "a lane has one box");
        const int my_pos = lane * br;
        const uint32_t my_dst = sbase + (uint32_t)(my_pos * HD * 2);
        int it = W.i0;
        bool more = true;
        // Of the walk's next tile: this lane's page (its table entry, or -1 behind the sequence's end; used only
        // when the box is sent, so that the load's time is not waited for), place in it, and kv head.
        struct Box {
            int id, at, kh;
            bool in;
        };
        auto next_box = [&](Box &B) {
            const int p = W.R.tile(it) * KT + my_pos;
            B.in = lane < boxes && p < W.q.p0 + W.q.n;
            B.id = B.in ? __ldg(A.tables + (long long)W.b * A.max_pages + (p >> A.page_shift)) : -1;
            B.at = p & ((1 << A.page_shift) - 1);
            B.kh = W.kh;
            if (++it == W.i1) {
                more = W.next(A);
                it = W.i0;
            }
        };
        auto row_of = [&](const Box &B) {
            if ((unsigned)B.id < (unsigned)A.n_pages) return (B.id << A.page_shift) + B.at;
            if (B.in) atomicOr(err, TRX_DEV_RANGE);
            return beyond;
        };
        auto issue = [&](int j, int off, const CUtensorMap *map, uint32_t full, int row, int kh) {
            const int st = j % KST;
            if (lane == 0) mbar_expect_tx_s(full + 8u * st, (uint32_t)C::TBYTES);
            __syncwarp();
            if (lane < boxes)
                load_box4(my_dst + (uint32_t)(off + st * C::TBYTES), map, 0, 0, kh * (HD / 64), row / 8, full + 8u * st);
            __syncwarp();
        };
        // K runs a tile ahead of V (its place is free earlier), and the table is read a tile ahead of that.
        Box box, nbox{};
        next_box(box);
        int vrow = 0, vkh = 0;
        bool ok = true, tile = true;
        for (int j = 0; ok; ++j) {
            int row = 0;
            const bool next = tile && more;
            if (next) next_box(nbox);
            if (bars.dead) ok = false;
            if (ok && tile) {
                ok = j < KST || wait2(sfull, j - KST);
                row = row_of(box);
                if (ok) issue(j, C::KOFF, &maps.k, kfull, row, box.kh);
            }
            if (ok && j) {
                ok = j - 1 < KST || wait2(odone, j - 1 - KST);
                if (ok) issue(j - 1, C::VOFF, &maps.v, vfull, vrow, vkh);
            }
            if (!tile) break;
            vrow = row;
            vkh = box.kh;
            box = nbox;
            tile = next;
        }
        if (!ok) {
            // Whatever was issued has landed before the block leaves (bounded; the timeout is recorded).
            bars.dead = 1u;
            for (int kind = 0; kind < 2; ++kind)
                for (int st = 0; st < KST; ++st)
                    for (int ph = 0; ph < 2; ++ph) wait_phase((kind ? vfull : kfull) + 8u * st, ph, nullptr);
        }
    } else if (any && warp == 5) {
        // S = Q K^T of every tile, as soon as its K tile and its S buffer allow.
        const uint32_t idq = idesc_f16<CT>(KT, false);
        const uint64_t qdesc = desc_kmajor(sbase + C::QOFF, 1024), kdesc = desc_kmajor(sbase + C::KOFF, HD / 64 * 1024);
        int j = 0;
        uint32_t piece = 0;
        bool ok = true, more = true;
        while (ok && more) {
            if constexpr (!SPLIT) {
                // The piece's query tile (rows of other sequences or zeros behind its own, whose results are not
                // used), once the MMAs that read the one before are complete.
                ok = j == 0 || wait2(sfull, j - 1);
                if (!ok) break;
                if (lane == 0) mbar_expect_tx_s(qready, (uint32_t)(A.tq * A.rep * HD * 2));
                __syncwarp();
                if (lane < HD / 64)
                    load_box4(sbase + C::QOFF + (uint32_t)(lane * kTcRows * 128), &maps.q, 64 * lane, 0, W.kh,
                              W.q.row0 + W.t * A.tq, qready);
                __syncwarp();
            }
            ok = wait(qready, piece++);
            for (int n = W.i1 - W.i0; ok && n; --n, ++j) {
                const int st = j % KST;
                ok = wait(kfull + 8u * st, (uint32_t)(j / KST)) && (j < NS || wait2(odone, j - NS));
                if (!ok) break;
                tc_after();
                const uint32_t d = tmem + C::SOFF + (uint32_t)((j % NS) * KT);
                const uint64_t kb = kdesc + (uint64_t)((st * C::TBYTES) >> 4);
#pragma unroll
                for (int part = SPLIT ? 1 : 0; part >= 0; --part)  // the small part first: the sums are cut off, not rounded
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c)
                        mma_ss4(d, qdesc + ((part * C::QBYTES + c * kTcRows * 128) >> 4), kb + ((c * 1024) >> 4), idq,
                                (SPLIT && part == 0) || c);
                commit(sfull + 8u * (j % NS));
            }
            if (ok) more = W.next(A);
        }
        if (!SPLIT && !ok)  // a query tile on its way has landed
            for (int ph = 0; ph < 2; ++ph) wait_phase(qready, ph, nullptr);
        commit(fin);  // every MMA is complete before the tensor memory is given back
        wait_phase(fin, 0u, nullptr);
    } else if (any && warp == 6) {
        // O += P V.
        const uint32_t idv = idesc_f16<CT>(C::NW, true);
        const uint64_t vdesc = desc_nmajor(sbase + C::VOFF, HD / 64 * 1024, 1024);
        int j = 0;
        bool ok = true, more = true;
        while (ok && more) {
            bool first = true;
            for (int n = W.i1 - W.i0; ok && n; --n, ++j) {
                const int st = j % KST;
                ok = wait(vfull + 8u * st, (uint32_t)(j / KST)) && wait2(pready, j);
                if (!ok) break;
                tc_after();
                const uint32_t p = tmem + C::SOFF + (uint32_t)((j % NS) * KT);
                const uint64_t vb = vdesc + (uint64_t)((st * C::TBYTES) >> 4);
                if constexpr (SPLIT) {
                    // 16 columns of high parts, 16 of low parts, for each 32 positions; alone, not onto O.
                    for (int q = 0; ok && q < C::NCH; ++q) {
                        const int n = j * C::NCH + q;
                        ok = n < C::NACC || wait2(ofree, n - C::NACC);
                        if (!ok) break;
                        tc_after();
                        const uint32_t d = tmem + C::AOFF + (uint32_t)((n % C::NACC) * C::NW);
                        const uint64_t qb = vb + (uint64_t)((q * (C::NW / 64) * 1024) >> 4);
                        mma_ts4<HD>(d, p + 16, p + 24, p + 48, p + 56, qb, idv, false);
                        mma_ts4<HD>(d, p, p + 8, p + 32, p + 40, qb, idv, true);
                        if constexpr (C::NCH > 1) commit(cdone + 8u * (n & 1));
                    }
                } else {
                    mma_ts4<HD>(tmem, p, p + 8, p + 16, p + 24, vb, idv, !first);
                }
                commit(odone + 8u * (j & 1));
                first = false;
            }
            if (ok) more = W.next(A);
        }
        commit(fin + 8u);
        wait_phase(fin + 8u, 0u, nullptr);
    } else if (any && warp < 4) {
        // Softmax: query row tid of the piece's tile.
        const int r = tid;
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        int j = 0;
        bool ok = true;
        // The walk's query tile; every MMA that read the one before is complete (its S was waited for).
        auto fetch = [&] {  // split: warp 5 brings 16-bit queries
            if constexpr (SPLIT) {
                load_query<CT, QT, HD>(A, smem, r, W.rows(A), W.q.row0 + W.t * A.tq, W.kh * A.rep);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) arrive(qready);
            }
        };
        // Split: part n of P V (dims q NW..) onto O scaled by f.  The tensor cores cut their sums off instead of
        // rounding them, which over the tiles of a row adds up to 2.6e-6 of the output (17 tiles of 64); so
        // a tile is summed alone and joined by a rounded FMA.
        float o[C::REGO ? HD : 1];
        auto fold = [&](int n, int q, float f, bool first) {
            if (!wait2(cdone, n)) return false;
            tc_after();
            const uint32_t ta = tmem + lanes + C::AOFF + (uint32_t)((n % C::NACC) * C::NW);
#pragma unroll
            for (int c = 0; c < C::NW / 32; ++c) {
                uint32_t w[32];
                tm_ld32(ta + 32 * c, w);
                if constexpr (C::REGO) {
                    tm_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[32 * c + e] = fmaf(o[32 * c + e], f, __uint_as_float(w[e]));
                } else {
                    const uint32_t to = tmem + lanes + (uint32_t)(q * C::NW + 32 * c);
                    if (!first) {
                        uint32_t x[32];
                        tm_ld32(to, x);
                        tm_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            w[e] = __float_as_uint(fmaf(__uint_as_float(x[e]), f, __uint_as_float(w[e])));
                    } else {
                        tm_wait_ld();
                    }
                    tm_st32(to, w);
                }
            }
            if constexpr (!C::REGO) tm_wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0) arrive(ofree + 8u * (n & 1));
            return true;
        };
        // 32 dims of this row's O.
        auto get = [&](int c, uint32_t (&w)[32]) {
            if constexpr (C::REGO) {
#pragma unroll
                for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(o[32 * c + e]);
            } else {
                tm_ld32(tmem + lanes + 32 * c, w);
                tm_wait_ld();
            }
        };
        GateRing G;
        if (C::RING) G.at = smem_u32(smem + C::END + sizeof(TcTail)) + warp * (32 * 64);
        fetch();
        for (bool more = true; ok && more;) {
            const int rows = W.rows(A), len = W.q.p0 + W.q.n;
            const int pos0 = W.q.p0 + W.t * A.tq;
            const int tok = r / A.rep, head = W.kh * A.rep + r - tok * A.rep;
            const int qpos = r < rows ? pos0 + tok : -1;
            const int pmax = pos0 + (rows - 1) / A.rep;  // the tile's last position; pos0 its first
            if (C::RING && A.gate) {
                G.row0 = W.q.row0 + W.t * A.tq;
                G.head0 = W.kh * A.rep;
                G.rows = rows;
                G.start(A, HD);
            }
            float m = -INFINITY, l = 0.f, fold_f = 0.f;
#pragma unroll
            for (int e = 0; e < (C::REGO ? HD : 1); ++e) o[e] = 0.f;
            const int j0 = j;
            for (int it = W.i0; it < W.i1; ++it, ++j) {
                const int k0 = W.R.tile(it) * KT;
                const uint32_t ts = tmem + lanes + C::SOFF + (uint32_t)((j % NS) * KT);
                // Nothing of the tile is hidden from any row.
                const bool open = k0 + KT - 1 <= pos0 &&
                                  (!A.window || pmax - k0 < A.window || k0 + KT <= A.sinks);
                if (!wait2(sfull, j)) {
                    ok = false;
                    break;
                }
                tc_after();
                uint32_t v[KT];  // the row of S
                tm_ld32(ts, *reinterpret_cast<uint32_t(*)[32]>(v));
                tm_ld32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
                tm_wait_ld();
                if (!open) {  // visible: e <= hi and (e >= lo or e < sk)
                    const int hi = qpos - k0, lo = A.window ? hi - A.window + 1 : -1, sk = A.sinks - k0;
#pragma unroll
                    for (int e = 0; e < KT; ++e)
                        if (e > hi || (e < lo && e >= sk)) v[e] = 0xff800000u;
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < KT; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(v[e]));
                float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                mx *= A.scale_log2;
                if (r >= rows) mx = -INFINITY;
                float f = 1.f;
                const bool far = fabsf(mx) >= kFar && mx != -INFINITY;
                bool any_far = false;  // of the warp's rows (asked together with what else is rare)
                if constexpr (SPLIT) {  // O = O f + P V, tile by tile
                    const float mo = m;
                    m = fmaxf(m, ceilf(mx));  // a whole number: 15 - m below is exact, and f a power of two
                    f = m == -INFINITY ? 0.f : ex2f(mo - m);
                    l *= f;
                    any_far = __any_sync(0xffffffffu, far);
                } else if (j == j0) {
                    m = mx - kHalfBits<CT>;  // the reference of O, l and the weights
                    any_far = __any_sync(0xffffffffu, far);
                } else {
                    const bool grow = mx - m > 8.f + kHalfBits<CT>;  // (m + 8 would round to m for large scores)
                    if (__any_sync(0xffffffffu, grow || far)) {
                        any_far = __any_sync(0xffffffffu, far);
                        if (!wait2(odone, j - 1)) {
                            ok = false;
                            break;
                        }
                        tc_after();
                        // A row without a maximum so far has O = 0 and l = 0.
                        const float ref = mx - kHalfBits<CT>;
                        f = grow && m != -INFINITY ? ex2f(m - ref) : 1.f;
                        if (grow) m = ref;
                        l *= f;
#pragma unroll 1
                        for (int c = 0; c < HD / 32; ++c) {
                            uint32_t w[32];
                            tm_ld32(tmem + lanes + 32 * c, w);
                            tm_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
                            tm_st32(tmem + lanes + 32 * c, w);
                        }
                        tm_wait_st();
                    }
                }
                const float nm = m == -INFINITY ? 0.f : (SPLIT ? kSplitBits - m : -m);
                if (any_far) {
                    l += far_weights<CT, SPLIT>(A, ts, far, m, qpos - k0, k0);
                } else {
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < KT / 32; ++c) {
                        uint32_t ph[16];
#pragma unroll
                        for (int e = 32 * c; e < 32 * c + 32; ++e) {
                            const float p = ex2f(fmaf(__uint_as_float(v[e]), A.scale_log2, nm));
                            v[e] = __float_as_uint(p);
                            sum[e & 3] += p;
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            ph[e] = PgCvt<CT>::pack(__uint_as_float(v[32 * c + 2 * e]), __uint_as_float(v[32 * c + 2 * e + 1]));
                        if constexpr (SPLIT) {
                            tm_st16(ts + 32 * c, ph);
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float2 b = PgCvt<CT>::unpack(ph[e]);
                                ph[e] = PgCvt<CT>::pack(__uint_as_float(v[32 * c + 2 * e]) - b.x,
                                                        __uint_as_float(v[32 * c + 2 * e + 1]) - b.y);
                            }
                            tm_st16(ts + 32 * c + 16, ph);
                        } else {
                            tm_st16(ts + 16 * c, ph);
                        }
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                }
                if (k0 + KT > len) {  // the rows of V behind the sequence's end
                    if (!wait(vfull + 8u * (j % KST), (uint32_t)(j / KST))) {
                        ok = false;
                        break;
                    }
                    unsigned char *vt = smem + C::VOFF + (j % KST) * C::TBYTES;
                    for (int i = r; i < (KT - (len - k0)) * (HD / 8); i += kTcRows) {
                        const int vr = len - k0 + i / (HD / 8), c = i % (HD / 8);
                        *reinterpret_cast<uint4 *>(vt + (vr / 8) * (HD * 16) + (c / 8) * 1024 + (vr % 8) * 128 + (c % 8) * 16) =
                            make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async();
                }
                tm_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) arrive(pready + 8u * (j % NS));
                if constexpr (SPLIT) {
                    if constexpr (C::REGO) {  // the tile before, while this one's P V runs
                        ok = j == j0 || fold(j - 1, 0, fold_f, false);
                        fold_f = f;
                    } else {
                        for (int q = 0; ok && q < C::NCH; ++q) ok = fold(j * C::NCH + q, q, f, j == j0);
                    }
                    if (!ok) break;
                }
            }
            if (!ok) break;
            // The next piece's query tile before this one is finished: its first S are computed meanwhile.
            const bool whole = W.whole();
            const int row = r < rows ? W.q.row0 + W.t * A.tq + tok : -1;
            const long long item0 = W.u - W.i1, item1 = item0 + W.R.cnt;
            more = W.next(A);
            if (more) fetch();
            if constexpr (C::REGO)
                ok = fold(j - 1, 0, fold_f, false);
            else
                ok = wait2(odone, j - 1);
            if (!ok) break;
            tc_after();
            if (whole)
                finish_whole<QT, HD, C::REGO, C::RING>(A, G, get, l, row, head);
            else
                finish_cut<QT, HD, C::REGO, C::RING>(A, S, G, get, item0, item1, m, l, row, head);
            tc_before();
        }
        if (C::RING && A.gate) G.drain();
        if (!ok) bars.dead = 1u;
    }
    tc_before();
    __syncthreads();
    if (warp == 5) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM) : "memory");
    }
}

template <typename CT, typename QT, int HD>
trx_status launch_tc(PgAttnArgs A, size_t part_cap, int cnt_cap, uint32_t *err, cudaStream_t st) {
    using C = TcCfg<HD, sizeof(QT) == 4>;
    static DevBits configured{0};
    const cudaError_t e = once_per_device(configured, [] {
        return cudaFuncSetAttribute(attn_paged_tc_kernel<CT, QT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)(C::END + sizeof(TcTail) + C::GBYTES));
    });
    if (e != cudaSuccess) return note_cuda(e);
    A.tq = kTcRows / A.rep;
    A.kt_shift = C::KT_SHIFT;
    PgMaps maps;
    if (!pg_encode_pools<HD>(maps, A, (uint32_t)std::min(1 << A.page_shift, C::KT))) return TRX_ERR_CUDA;
    if (sizeof(QT) == 2) {
        const uint64_t dims[4] = {HD, (uint64_t)A.rep, (uint64_t)A.Hkv, (uint64_t)A.max_rows};
        const uint64_t strides[3] = {HD * 2ull, (uint64_t)A.rep * HD * 2, (uint64_t)A.H * HD * 2};
        const uint32_t box[4] = {64, (uint32_t)A.rep, 1, (uint32_t)A.tq};
        if (!encode_map_16bit_4d(&maps.q, A.q, dims, strides, box)) return TRX_ERR_CUDA;
    }
    const int grid = device_sms() * C::CTAS;
    if ((size_t)grid * 2 * kTcRows * (HD + 2) > part_cap || 4 * grid > cnt_cap) return TRX_ERR_UNSUPPORTED;
    return note_cuda(launch_kernel(attn_paged_tc_kernel<CT, QT, HD>, dim3(grid), dim3(kTcThreads), C::END + sizeof(TcTail) + C::GBYTES, st,
                                   maps, A, err));
}

template <typename CT, typename QT>
trx_status launch_tc_hd(const PgAttnArgs &A, int hd, size_t part_cap, int cnt_cap, uint32_t *err, cudaStream_t st) {
    switch (hd) {
        case 64: return launch_tc<CT, QT, 64>(A, part_cap, cnt_cap, err, st);
        case 128: return launch_tc<CT, QT, 128>(A, part_cap, cnt_cap, err, st);
        default: return launch_tc<CT, QT, 256>(A, part_cap, cnt_cap, err, st);
    }
}

}  // namespace

trx_status launch_attn_paged_tc(const PgAttnArgs &A, int hd, int cache_type, int q_type, size_t part_cap, int cnt_cap,
                                uint32_t *err, cudaStream_t st) {
    if (cache_type == TRX_TYPE_BF16)
        return launch_tc_hd<__nv_bfloat16, __nv_bfloat16>(A, hd, part_cap, cnt_cap, err, st);
    return q_type == TRX_TYPE_F32 ? launch_tc_hd<__half, float>(A, hd, part_cap, cnt_cap, err, st)
                                  : launch_tc_hd<__half, __half>(A, hd, part_cap, cnt_cap, err, st);
}

}  // namespace trx
