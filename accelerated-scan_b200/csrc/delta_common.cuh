// Device helpers of the gated delta rule kernels: warp matrix instructions on bf16 fragments, two-term splitting
// of fp32 operands, swizzled shared-memory tiles, the chunk table.
#pragma once

#include <cuda_fp16.h>

#include "delta.h"

namespace ascan {

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void stsm4(uint32_t a, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};"
                 :: "r"(a), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool real) {
    const int n = real ? 16 : 0;      // nothing is read and 16 zero bytes are written where `real` is false
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}

// Two floats as packed bf16 (first in the low half), rounded to nearest: 2^-8 relative.
__device__ __forceinline__ uint32_t pack2(float x0, float x1) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x1), "f"(x0));
    return r;
}
__device__ __forceinline__ float low_half(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float high_half(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }
// x = hi + lo with both in bf16: what is left is at most 2^-16 of x.
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    hi = pack2(x0, x1);
    lo = pack2(x0 - low_half(hi), x1 - high_half(hi));
}

// Byte offset of 16-byte piece `ch` of row `row` in a tile with NCH pieces a row: pieces are permuted by the row so
// that the eight rows a matrix load takes at one piece lie in different banks.
template <int NCH>
__device__ __forceinline__ uint32_t tile_off(int row, int ch) {
    return static_cast<uint32_t>(row * NCH + (ch ^ (NCH >= 8 ? row & 7 : (row * NCH / 8) & (NCH - 1)))) << 4;
}

// Lane addresses of the four 8x8 matrices of one load.  (r0, c0): corner, c0 in 16-byte pieces.
template <int NCH>   // B operand from X[n][k] (16 n, 16 k): {b0, b1} of n..n+7 and of n+8..n+15
__device__ __forceinline__ uint32_t addr_bn(uint32_t base, int r0, int c0, int lane) {
    const int m = lane >> 3;
    return base + tile_off<NCH>(r0 + (m >> 1) * 8 + (lane & 7), c0 + (m & 1));
}
template <int NCH>   // B operand from X[k][n], transposed load
__device__ __forceinline__ uint32_t addr_bt(uint32_t base, int k0, int c0, int lane) {
    const int m = lane >> 3;
    return base + tile_off<NCH>(k0 + (m & 1) * 8 + (lane & 7), c0 + (m >> 1));
}
template <int NCH>   // A operand from X[row][k]
__device__ __forceinline__ uint32_t addr_an(uint32_t base, int r0, int c0, int lane) {
    const int m = lane >> 3;
    return base + tile_off<NCH>(r0 + (m & 1) * 8 + (lane & 7), c0 + (m >> 1));
}
template <int NCH>   // A operand from X[k][row], transposed load
__device__ __forceinline__ uint32_t addr_at(uint32_t base, int k0, int c0, int lane) {
    const int m = lane >> 3;
    return base + tile_off<NCH>(k0 + (m >> 1) * 8 + (lane & 7), c0 + (m & 1));
}

// 64 rows of a tile with NCH pieces a row; rows >= rows and pieces >= pieces become zero.
template <int NCH>
__device__ __forceinline__ void load_tile(uint32_t dst, const bf16 *src, int64_t row_stride, int rows, int pieces, int tid,
                                          int threads, int all_rows = 64) {
    for (int i = tid; i < all_rows * NCH; i += threads) {
        const int r = i / NCH, c = i % NCH;
        const bool real = r < rows && c < pieces;
        cp16(dst + tile_off<NCH>(r, c), real ? src + r * row_stride + c * 8 : src, real);
    }
}

__device__ __forceinline__ float load_as_float(const void *p, int dtype, int64_t i) {
    if (dtype == ASCAN_F32) return static_cast<const float *>(p)[i];
    if (dtype == ASCAN_BF16) return __bfloat162float(static_cast<const bf16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store_from_float(void *p, int dtype, int64_t i, float x) {
    if (dtype == ASCAN_F32) static_cast<float *>(p)[i] = x;
    else if (dtype == ASCAN_BF16) static_cast<bf16 *>(p)[i] = __float2bfloat16_rn(x);
    else static_cast<__half *>(p)[i] = __float2half_rn(x);
}

// Sequence boundaries are read on the device and clamped into [0, T]: whatever they hold, no access leaves the arrays.
__device__ __forceinline__ int64_t seq_start(const DeltaParams &p, int n) {
    const int64_t s = p.starts64 ? static_cast<const int64_t *>(p.starts)[n] : static_cast<const int32_t *>(p.starts)[n];
    return s < 0 ? 0 : (s > p.T ? p.T : s);
}

struct Sequence {
    int64_t t0, len;     // first token in the batch row, length
    int64_t b;           // batch row
    int slot0, chunks;   // its chunks hold the slots slot0 .. slot0 + chunks - 1
};

__device__ __forceinline__ Sequence get_sequence(const DeltaParams &p, int n) {
    Sequence s;
    if (!p.packed) {
        s.t0 = 0;
        s.len = p.T;
        s.b = n;
        s.slot0 = n * p.chunks;
    } else {
        s.t0 = seq_start(p, n);
        const int64_t end = seq_start(p, n + 1);
        s.len = end > s.t0 ? end - s.t0 : 0;
        s.b = 0;
        s.slot0 = static_cast<int>(s.t0 / DELTA_CHUNK) + n;     // no two sequences share a slot: a sequence has at most
    }                                                           // end/64 - start/64 + 1 chunks
    s.chunks = static_cast<int>((s.len + DELTA_CHUNK - 1) / DELTA_CHUNK);
    return s;
}

struct Chunk {
    int64_t t0, b;
    int rows;            // tokens of the chunk; 0 for a slot that no chunk uses
};

__device__ __forceinline__ Chunk get_chunk(const DeltaParams &p, int slot) {
    int n;
    if (!p.packed) {
        n = slot / p.chunks;
    } else {             // the last sequence whose first slot is not behind this one
        int lo = 0, hi = p.n_seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (static_cast<int>(seq_start(p, mid) / DELTA_CHUNK) + mid <= slot) lo = mid;
            else hi = mid - 1;
        }
        n = lo;
    }
    const Sequence s = get_sequence(p, n);
    const int c = slot - s.slot0;
    Chunk r;
    r.b = s.b;
    r.t0 = s.t0 + static_cast<int64_t>(c) * DELTA_CHUNK;
    const int64_t left = (c < 0 || c >= s.chunks) ? 0 : s.len - static_cast<int64_t>(c) * DELTA_CHUNK;
    r.rows = static_cast<int>(left > DELTA_CHUNK ? DELTA_CHUNK : left);
    return r;
}

// e^{G_i - G_j} for tokens of one chunk; 0 where a zero gate lies between them.
__device__ __forceinline__ float decay_between(float ghi_i, float glo_i, float r_i, float ghi_j, float glo_j, float r_j) {
    return r_i == r_j ? expf((ghi_i - ghi_j) + (glo_i - glo_j)) : 0.f;
}

}  // namespace ascan
