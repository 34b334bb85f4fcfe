// Fifth-generation tensor core path of the gated delta rule: mbarriers with bounded waits, tcgen05 wrappers, and the
// arithmetic of a chunk that is prepared (gates, M, P) while others carry the state through the chunk before it.
#pragma once

#include "delta_common.cuh"

namespace ascan {

// ---- barriers --------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("{ .reg .b64 t; mbarrier.arrive.shared::cta.b64 t, [%0]; }" :: "r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

// Every wait ends: after WAIT_TRIES the CTA is given up (`dead`, in shared memory), from then on no wait of the CTA
// waits, the kernel runs to its end on whatever is in its buffers, leaves its copies time to land, and the host reads
// the status word.
constexpr uint32_t WAIT_TRIES = 1u << 21;
struct Waiter {
    volatile int *dead;
    int *status;           // pinned host memory
    __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity) const {
        uint32_t left = WAIT_TRIES;
#pragma unroll 1
        while (!mbar_try(bar, parity)) {
            if (*dead) return;
            if (--left == 0) {
                *dead = 1;
                if (status) *reinterpret_cast<volatile int *>(status) = 1;
            }
        }
    }
    // All lanes together: they may leave the loop one by one, and what follows (ldmatrix, tcgen05.ld) needs the whole warp.
    __device__ __forceinline__ void warp(uint32_t bar, uint32_t parity) const {
        (*this)(bar, parity);
        __syncwarp();
    }
};

// Before a CTA ends: one that was given up may have copies in flight, which end by themselves within microseconds.
__device__ __forceinline__ void drain(volatile const int *dead) {
    if (*dead)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

template <int ID, int THREADS>
__device__ __forceinline__ void group_sync() {
    asm volatile("bar.sync %0, %1;" :: "n"(ID), "n"(THREADS) : "memory");
}

// ---- tcgen05 ---------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// A thread's reads of a tile have ended, before it says that the next copy may write over it.  An arrival alone does not wait for
// loads of the generic proxy that are still queued behind the tensor cores' operands: sums of such reads came out of the next
// tile's values in most runs, d_log_gates off by up to a sixth of the largest, until this stood before the arrival.
__device__ __forceinline__ void give_back_reads() { fence_async_proxy(); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}

// Operand tiles in shared memory: rows of 128 bytes (64 bf16), 16-byte pieces permuted by the row (tile_off<8>), which
// is the 128-byte swizzle; rows lie 8 to 1024 bytes.  Tiles of more columns are several such blocks.  K along the row
// ("K-major"): sbo = 1024.  K down the rows ("MN-major"): lbo = distance of the blocks of 64 columns, sbo = 1024.
// Shared addresses lie below 2^18, so bytes / 16 may be added to the low word.
constexpr uint32_t TILE_HIGH = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t tile_low(uint32_t addr, uint32_t lbo = 16) { return addr >> 4 | lbo >> 4 << 16; }
// fp32 accumulators, bf16 operands, 128 rows
__host__ __device__ constexpr uint32_t mma_desc(int n, bool b_mn_major, bool negate_a = false, bool a_mn_major = false) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (negate_a ? 1u << 13 : 0) | (a_mn_major ? 1u << 15 : 0) | (b_mn_major ? 1u << 16 : 0) |
           uint32_t(n / 8) << 17 | uint32_t(128 / 16) << 24;
}
// One thread of the warp.  The compiler knows that what runs under it is one thread's and keeps the operands of a product in
// uniform registers: 35 clocks to the next product of 64 columns, against 150 under `lane == 0`.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{ .reg .pred q; elect.sync _|q, 0xffffffff; selp.u32 %0, 1, 0, q; }" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, bool add) {     // A in tensor memory
    asm volatile("{ .reg .pred p; .reg .b64 b; mov.b64 b, {%2, %5}; setp.ne.u32 p, %4, 0;"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p; }"
                 :: "r"(d), "r"(a), "r"(b), "r"(desc), "r"(uint32_t(add)), "n"(TILE_HIGH) : "memory");
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, bool add) {
    asm volatile("{ .reg .pred p; .reg .b64 a, b; mov.b64 a, {%1, %5}; mov.b64 b, {%2, %5}; setp.ne.u32 p, %4, 0;"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p; }"
                 :: "r"(d), "r"(a), "r"(b), "r"(desc), "r"(uint32_t(add)), "n"(TILE_HIGH) : "memory");
}

// 32 (16) columns of the warp's 32 lanes; a thread holds its lane's
#define ASCAN_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define ASCAN_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t a) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
                 "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : ASCAN_R8(r, 0), ASCAN_R8(r, 8), ASCAN_R8(r, 16), ASCAN_R8(r, 24) : "r"(a));
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], uint32_t a) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : ASCAN_R8(r, 0), ASCAN_R8(r, 8) : "r"(a));
}
__device__ __forceinline__ void tmem_ld8(uint32_t (&r)[8], uint32_t a) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : ASCAN_R8(r, 0) : "r"(a));
}
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" :: "r"(a), ASCAN_I8(r, 0) : "memory");
}

// ---- two floats at a time (first in the low half) ----------------------------------------------------------------------

typedef unsigned long long f2;
__device__ __forceinline__ f2 two(float x, float y) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ f2 two_bits(uint32_t x, uint32_t y) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
    return r;
}
__device__ __forceinline__ float2 apart(f2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint32_t pack_f2(f2 v) {
    const float2 x = apart(v);
    return pack2(x.x, x.y);
}
__device__ __forceinline__ void split_f2(f2 v, uint32_t &hi, uint32_t &lo) {
    hi = pack_f2(v);
    lo = pack_f2(fma2(two_bits(hi << 16, hi & 0xffff0000u), two(-1.f, -1.f), v));
}

// ---- tiles by TMA ----------------------------------------------------------------------------------------------------

__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("{ .reg .b64 t; mbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1; }" :: "r"(bar), "r"(bytes) : "memory");
}
// (column, head, token, batch) box of a tensor map; the column is 0 or a multiple of 64: 16-byte aligned
__device__ __forceinline__ void tma_load(uint32_t dst, const void *map, int col, int head, int tok, int b, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 :: "r"(dst), "l"(map), "r"(col), "r"(head), "r"(tok), "r"(b), "r"(bar) : "memory");
}

// A box of 64 tokens x 128 columns back; rows behind the array are left out.
__device__ __forceinline__ void tma_store(const void *map, uint32_t src, int col, int head, int tok, int b) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];"
                 :: "l"(map), "r"(col), "r"(head), "r"(tok), "r"(b), "r"(src) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ---- preparing a chunk -----------------------------------------------------------------------------------------------
//
// 128 threads.  K K^T and Q K^T of the chunk come from one product of 128 rows ([K; Q]) in tensor memory, a row a
// thread.  Here L carries the factor beta on its columns (forward) or rows (backward), and with it M: N = M diag(beta) =
// L' (I + L')^{-1} for L' = L diag(beta), or diag(beta) M likewise.  By halves: for the lower left block between two
// finished ones,
//     N21 = (I - N22) L'21 (I - N11),
// from 4 x 4 (substitution) to 8 and 16 in fp32, to 32 and 64 on warp matrix instructions with two-term operands
// (2^-16, as N itself is handed on).

constexpr int PITCH = 68;                        // floats a row of M
constexpr int M_BYTES = 64 * PITCH * 4;          // 17 KB: also the place of M's two tiles
enum : int { SC_OUT = SC_ARRAYS, SC_GAMC_BETA, SC_SHARED };      // in shared memory also scale * gam and Gam_C * beta
struct GateShared {                              // of one chunk
    float sc[SC_SHARED * 64];
    float w[2][2][64];                           // for token j in a block of 16: e^{G_end - G_j}, and e^{G_first - G_j};
                                                 // [1]: times beta_j
    int direct[4];                               // blocks whose decay leaves the range of the second
};

// 16 x 16 blocks of fp32 in shared memory (PITCH floats a row): to = from - A B over `steps` blocks of A's columns and B's
// rows.  One warp.
__device__ __forceinline__ void block_product(float *to, const float *from, const float *A, const float *B, int steps) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t2 = 2 * (lane & 3);
    float c[2][2][4];                            // two sums a tile, so that products need not wait for one another
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 x = *reinterpret_cast<const float2 *>(from + (g + 8 * h) * PITCH + 8 * n + t2);
            c[0][n][2 * h] = x.x;
            c[0][n][2 * h + 1] = x.y;
            c[1][n][2 * h] = c[1][n][2 * h + 1] = 0.f;
        }
#pragma unroll 1
    for (int k = 0; k < steps; ++k, A += 16, B += 16 * PITCH) {
        uint32_t a[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = (j >> 1) * 8 + t2;
            const float2 x = *reinterpret_cast<const float2 *>(A + (g + (j & 1) * 8) * PITCH + col);
            split2(-x.x, -x.y, a[0][j], a[1][j]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            uint32_t b[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float *x = B + (j * 8 + t2) * PITCH + 8 * n + g;
                split2(x[0], x[PITCH], b[0][j], b[1][j]);
            }
            mma(c[0][n], a[0], b[0][0], b[0][1]);
            mma(c[1][n], a[1], b[0][0], b[0][1]);
            mma(c[1][n], a[0], b[1][0], b[1][1]);
        }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2 *>(to + (g + 8 * h) * PITCH + 8 * n + t2) =
                make_float2(c[0][n][2 * h] + c[1][n][2 * h], c[0][n][2 * h + 1] + c[1][n][2 * h + 1]);
}

// Running sum of the chunk's log gates in 64 bits and what follows from it; one warp, `sc` in shared memory.
__device__ __forceinline__ void chunk_gates(const float (&g)[2], const float (&beta)[2], float scale, GateShared &gs, int lane) {
    float *sc = gs.sc;
    double sum[2];
    int reset[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        reset[j] = g[j] <= -104.f;               // e^g is zero in fp32
        sum[j] = reset[j] ? 0.0 : double(g[j]);
    }
    double s = sum[0] + sum[1];
    int r = reset[0] + reset[1];
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const double sp = __shfl_up_sync(~0u, s, d);
        const int rp = __shfl_up_sync(~0u, r, d);
        if (lane >= d) { s += sp; r += rp; }
    }
    const double G0 = s - sum[1];                // of token 2 lane; s is that of 2 lane + 1
    const int R0 = r - reset[1];
    const double last = __shfl_sync(~0u, s, 31), end = __shfl_sync(~0u, s, lane | 7), first = __shfl_sync(~0u, G0, lane & ~7);
    const int all = __shfl_sync(~0u, r, 31), r_end = __shfl_sync(~0u, r, lane | 7), r_first = __shfl_sync(~0u, R0, lane & ~7);
    bool plain = r_first == r_end;
#pragma unroll 1
    for (int j = 0; j < 2; ++j) {
        const int i = 2 * lane + j;
        const double G = j ? s : G0;
        const int R = j ? r : R0;
        const float hi = float(G), gam = R == 0 ? expf(hi) : 0.f, back = float(first - G);
        sc[SC_GAM * 64 + i] = gam;
        sc[SC_OUT * 64 + i] = scale * gam;
        const float be = j ? beta[1] : beta[0], gam_c = R == all ? expf(float(last - G)) : 0.f;
        sc[SC_GAMC * 64 + i] = gam_c;
        sc[SC_GAMC_BETA * 64 + i] = gam_c * be;
        sc[SC_BETA * 64 + i] = be;
        sc[SC_GHI * 64 + i] = hi;
        sc[SC_GLO * 64 + i] = float(G - double(hi));
        sc[SC_RESET * 64 + i] = float(R);
        const float to_end = R == r_end ? expf(float(end - G)) : 0.f, to_first = expf(back);
        gs.w[0][0][i] = to_end;
        gs.w[0][1][i] = to_first;
        gs.w[1][0][i] = to_end * be;
        gs.w[1][1][i] = to_first * be;
        plain = plain && fabsf(back) <= 60.f;
    }
    const unsigned ok = __ballot_sync(~0u, plain);
    if (lane < 4) gs.direct[lane] = (ok >> (8 * lane) & 255u) != 255u;
}

// Row i of a product in tensor memory times Gam, block by block of 16 tokens.  Behind block bj,
// Gam_ij = e^{G_i - G_end} e^{G_end - G_j}; inside i's own block the first token takes the place of the end, unless the decay
// in the block is so strong (or a gate zero) that these factors leave fp32: then one exponential an element.
__device__ __forceinline__ void row_factors(float (&f)[4][128], float factor, const GateShared &gs, int i, int tid) {
    const float *sc = gs.sc;
    const int bi = i >> 4;
#pragma unroll 1
    for (int bj = 0; bj < 4; ++bj) {
        const int ref = bj == bi ? 16 * bj : 16 * bj + 15;
        f[bj][tid] = bj > bi ? 0.f : factor * decay_between(sc[SC_GHI * 64 + i], sc[SC_GLO * 64 + i], sc[SC_RESET * 64 + i],
                                                            sc[SC_GHI * 64 + ref], sc[SC_GLO * 64 + ref], sc[SC_RESET * 64 + ref]);
    }
}
// put(bj, x) gets 16 values of block bj, times beta of their tokens where `columns`.  A warp has the rows of two blocks and
// skips what lies above both.  Where `mask`, values above the diagonal (which stays) are zero; else they are anything.
template <class PUT>
__device__ __forceinline__ void decayed_row(uint32_t tmem, const float (&f)[4][128], float factor, bool columns, bool mask,
                                            const GateShared &gs, int i, int tid, PUT put) {
    const float *sc = gs.sc;
    const int bi = i >> 4, b1 = i >> 5 << 1 | 1;         // b1: the warp's last own block
#pragma unroll 1
    for (int bj = 0; bj <= b1; ++bj) {
        uint32_t r[16];
        tmem_ld16(r, tmem + 16 * bj);
        const float *w = gs.w[columns][bj == bi] + 16 * bj;
        const f2 ff = two(f[bj][tid], f[bj][tid]);
        float x[16];
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const ulonglong2 w4 = *reinterpret_cast<const ulonglong2 *>(w + j);
            const float2 a = apart(mul2(mul2(w4.x, ff), two_bits(r[j], r[j + 1])));
            const float2 b = apart(mul2(mul2(w4.y, ff), two_bits(r[j + 2], r[j + 3])));
            x[j] = a.x; x[j + 1] = a.y; x[j + 2] = b.x; x[j + 3] = b.y;
        }
        if (bj == bi && gs.direct[bj]) {
#pragma unroll 1
            for (int j = 0; j < 16; ++j) {
                const int t = 16 * bj + j;
                const float d = factor * (columns ? sc[SC_BETA * 64 + t] : 1.f) *
                    decay_between(sc[SC_GHI * 64 + i], sc[SC_GLO * 64 + i], sc[SC_RESET * 64 + i], sc[SC_GHI * 64 + t], sc[SC_GLO * 64 + t],
                                  sc[SC_RESET * 64 + t]);
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (k == j) x[k] = d * __uint_as_float(r[k]);
            }
        }
        if (mask && bj >= b1 - 1)
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = 16 * bj + j <= i ? x[j] : 0.f;
        put(bj, x);
    }
}

// From L (shared, fp32, 64 rows of PITCH) to N = L (I + L)^{-1} as two bf16 tiles, hi and lo, in its place; all 128 threads,
// SYNC a barrier of theirs.  What lies above L's diagonal is not read; the upper right quarter is scratch.
template <class SYNC>
__device__ __forceinline__ void make_m(float *m, int tid, SYNC sync) {
    const int lane = tid & 31, warp = tid >> 5;
    const auto block = [&](int r, int col) { return m + 16 * r * PITCH + 16 * col; };
    {   // a diagonal block a warp: 4 x 4 blocks by substitution, then two steps of the same kind as below
        float *d = block(warp, warp), *t = block(warp >> 1, 2 + (warp & 1));
        if (lane < 16) {
            const int c = lane & 3;
            float *x = d + (lane >> 2) * 4 * (PITCH + 1);
            const float l21 = x[2 * PITCH + 1], l31 = x[3 * PITCH + 1], l32 = x[3 * PITCH + 2];
            const float m1 = c < 1 ? x[PITCH + c] : 0.f;
            const float m2 = (c < 2 ? x[2 * PITCH + c] : 0.f) - l21 * m1;
            const float m3 = (c < 3 ? x[3 * PITCH + c] : 0.f) - l31 * m1 - l32 * m2;
            __syncwarp(0xffff);
            x[c] = 0.f;
            x[PITCH + c] = m1;
            x[2 * PITCH + c] = m2;
            x[3 * PITCH + c] = m3;
        }
        __syncwarp();
        {
            const int r = lane >> 2 & 3, c = lane & 3, o = (lane >> 4) * 8;
            float *low = d + (o + 4) * PITCH + o;
            float y = low[r * PITCH + c];
            const float4 a = *reinterpret_cast<const float4 *>(low + r * PITCH);
            const float *x = d + o * PITCH + o + c;
            y -= a.x * x[0] + a.y * x[PITCH] + a.z * x[2 * PITCH] + a.w * x[3 * PITCH];
            t[(o + r) * PITCH + c] = y;
            __syncwarp();
            const float4 b = *reinterpret_cast<const float4 *>(low + r * PITCH + 4);
            const float *z = t + o * PITCH + c;
            y -= b.x * z[0] + b.y * z[PITCH] + b.z * z[2 * PITCH] + b.w * z[3 * PITCH];
            low[r * PITCH + c] = y;
            d[(o + r) * PITCH + o + 4 + c] = 0.f;
        }
        __syncwarp();
        {
            const int r = lane >> 2, c = 2 * (lane & 3);
            float *low = d + 8 * PITCH;
            float2 y = *reinterpret_cast<const float2 *>(low + r * PITCH + c);
            const auto subtract = [&](const float *row, const float *x) {
#pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    const float4 a = *reinterpret_cast<const float4 *>(row + k);
                    const float a4[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 v = *reinterpret_cast<const float2 *>(x + (k + j) * PITCH + c);
                        y.x -= a4[j] * v.x;
                        y.y -= a4[j] * v.y;
                    }
                }
            };
            subtract(low + r * PITCH, d);
            *reinterpret_cast<float2 *>(t + r * PITCH + c) = y;
            __syncwarp();
            subtract(low + r * PITCH + 8, t);
            *reinterpret_cast<float2 *>(low + r * PITCH + c) = y;
            *reinterpret_cast<float2 *>(d + r * PITCH + 8 + c) = make_float2(0.f, 0.f);
        }
    }
    sync();
    // Steps 0 and 1, blocks of 32: pair (0, 1) on warp 0, (2, 3) on warp 1, the first product through the block above the
    // diagonal.  Steps 2 and 3, the whole, 32 x 32 by 32: a block a warp, the first product through the upper right quarter
    // (M11 and M22 are lower triangular).  A loop, so that the four share their instructions: the cache for those is small.
    const int r = warp >> 1, q = warp & 1;
#pragma unroll 1
    for (int step = 0; step < 4; ++step) {
        const int low = step < 2 ? 2 * warp + 1 : 2 + r, left = step < 2 ? 2 * warp : q;         // block of M21
        const int up = step < 2 ? 2 * warp : r, right = step < 2 ? 2 * warp + 1 : 2 + q;         // and the one above
        const bool first = !(step & 1);
        if (step >= 2 || warp < 2)
            block_product(first ? block(up, right) : block(low, left), first ? block(low, left) : block(up, right),
                          first ? block(low, left) : step < 2 ? block(low, low) : block(low, 2),
                          first ? block(left, left) : step < 2 ? block(up, right) : block(0, right),
                          step < 2 ? 1 : first ? 2 - q : 1 + r);
        sync();
    }
    const int row = tid >> 1, half = tid & 1;
    float4 v[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) v[p] = *reinterpret_cast<const float4 *>(m + row * PITCH + 32 * half + 4 * p);
    sync();
    unsigned char *tiles = reinterpret_cast<unsigned char *>(m);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int col = 32 * half + 8 * p;
        const float x[8] = {v[2 * p].x, v[2 * p].y, v[2 * p].z, v[2 * p].w, v[2 * p + 1].x, v[2 * p + 1].y, v[2 * p + 1].z, v[2 * p + 1].w};
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            split2(x[2 * j], x[2 * j + 1], h[j], l[j]);
        *reinterpret_cast<uint4 *>(tiles + tile_off<8>(row, col >> 3)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(tiles + 8192 + tile_off<8>(row, col >> 3)) = make_uint4(l[0], l[1], l[2], l[3]);
    }
}

}  // namespace ascan
