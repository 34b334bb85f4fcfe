// What the forward and the backward sweep of the gated delta rule share: a warp's 16 columns of results, which lie
// transposed in its accumulators, on their way to memory.
#pragma once

#include "delta_common.cuh"

namespace ascan {

// rows of 16 columns (v0 ..) of a warp's 64 x 16 result that lies transposed in accumulators: out (any type)
template <int NT>
__device__ __forceinline__ void stage_transposed(uint32_t stg, unsigned char *stg_p, const float (&c)[8][4], int lane) {
    if (NT == 1) {           // bf16, [piece][token] of 16 bytes
#pragma unroll
        for (int np = 0; np < 4; ++np) {
            const int m = lane >> 3;     // matrices: (tokens 16 np, piece 0), (.., piece 1), (tokens + 8, 0), (.., 1)
            const uint32_t a = stg + ((m & 1) * 64 + 16 * np + (m >> 1) * 8 + (lane & 7)) * 16;
            stsm4t(a, pack2(c[2 * np][0], c[2 * np][1]), pack2(c[2 * np][2], c[2 * np][3]),
                   pack2(c[2 * np + 1][0], c[2 * np + 1][1]), pack2(c[2 * np + 1][2], c[2 * np + 1][3]));
        }
    } else {                 // fp32, [v / 4][token] of 16 bytes
        float *f = reinterpret_cast<float *>(stg_p);
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int v = (lane >> 2) + (j >> 1) * 8, t = 8 * n + 2 * (lane & 3) + (j & 1);
                f[((v >> 2) * 64 + t) * 4 + (v & 3)] = c[n][j];
            }
    }
}

// ... to a (token, v) array of the storage type; rows tokens, columns v0 .. of V
template <int NT>
__device__ __forceinline__ void flush_out(const unsigned char *stg, void *dst, int dtype, int64_t base, int64_t row_stride, int rows,
                                          int v0, int V, int lane) {
    for (int i = lane; i < 128; i += 32) {
        const int t = i >> 1, pc = i & 1, v = v0 + pc * 8;
        if (t >= rows || v >= V) continue;
        const int64_t at = base + t * row_stride + v;
        if (NT == 1) {
            const uint4 x = *reinterpret_cast<const uint4 *>(stg + (pc * 64 + t) * 16);
            bf16 *o = static_cast<bf16 *>(dst) + at;
            if (V % 8 == 0) {
                *reinterpret_cast<uint4 *>(o) = x;
            } else {
                const bf16 *s = reinterpret_cast<const bf16 *>(&x);
                for (int j = 0; j < 8 && v + j < V; ++j) o[j] = s[j];
            }
        } else {
            const float *f = reinterpret_cast<const float *>(stg);
            for (int j = 0; j < 8 && v + j < V; ++j) store_from_float(dst, dtype, at + j, f[((2 * pc + (j >> 2)) * 64 + t) * 4 + (j & 3)]);
        }
    }
}

// the warp's 16 x KP accumulators (of the state, or KP = 64 tokens of e or z) to bf16 planes [plane][Vp][KP], through the
// staging area
template <int KP, int NT>
__device__ __forceinline__ void save_state(uint32_t stg, const unsigned char *stg_p, const float (&s)[KP / 8][4], bf16 *dst, int v0,
                                           int Vp, int lane) {
    constexpr int NCH = KP / 8;
#pragma unroll
    for (int pl = 0; pl < NT; ++pl) {
        __syncwarp();
#pragma unroll
        for (int kk = 0; kk < KP / 16; ++kk) {
            uint32_t r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {      // (v 0-7, k), (v 8-15, k), (v 0-7, k + 8), (v 8-15, k + 8)
                uint32_t hi, lo;
                split2(s[2 * kk + (j >> 1)][2 * (j & 1)], s[2 * kk + (j >> 1)][2 * (j & 1) + 1], hi, lo);
                r[j] = pl == 0 ? hi : lo;
            }
            stsm4(addr_an<NCH>(stg, 0, 2 * kk, lane), r[0], r[1], r[2], r[3]);
        }
        __syncwarp();
        for (int i = lane; i < 16 * NCH; i += 32) {
            const int r = i / NCH, c = i % NCH;
            if (v0 + r < Vp)
                *reinterpret_cast<uint4 *>(dst + int64_t(pl) * Vp * KP + (v0 + r) * KP + c * 8) =
                    *reinterpret_cast<const uint4 *>(stg_p + tile_off<NCH>(r, c));
        }
    }
    __syncwarp();
}

// Warps of a CTA: eight share one copy of the chunk's tiles where shared memory holds their own ones as well; fewer
// while that would leave SMs without a CTA.
static inline int sweep_warps(const DeltaParams &p, int sm_count, size_t (*bytes)(int)) {
    const int64_t slices = (p.Vp + 15) / 16, chains = int64_t(p.n_seqs) * p.H;
    int w = 8;
    while (w > 1 && (bytes(w) > 227 * 1024 || w / 2 >= slices || chains * ((slices + w - 1) / w) < sm_count)) w /= 2;
    return w;
}

}  // namespace ascan
