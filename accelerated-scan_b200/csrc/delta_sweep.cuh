// What the forward and the backward sweep of the gated delta rule share: a warp's 16 columns of results, which lie
// transposed in its accumulators, on their way to memory.
#pragma once

#include "delta_common.cuh"

namespace ascan {

// rows of 16 columns (v0 ..) of a warp's 64 x 16 result that lies transposed in accumulators: out (any type)
__device__ __forceinline__ void stage_transposed(uint32_t stg, unsigned char *stg_p, const float (&c)[8][4], int lane) {
    // fp32, [v / 4][token] of 16 bytes
    float *f = reinterpret_cast<float *>(stg_p);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int v = (lane >> 2) + (j >> 1) * 8, t = 8 * n + 2 * (lane & 3) + (j & 1);
            f[((v >> 2) * 64 + t) * 4 + (v & 3)] = c[n][j];
        }
}

// ... to a (token, v) array of the storage type; rows tokens, columns v0 .. of V
__device__ __forceinline__ void flush_out(const unsigned char *stg, void *dst, int dtype, int64_t base, int64_t row_stride, int rows,
                                          int v0, int V, int lane) {
    for (int i = lane; i < 128; i += 32) {
        const int t = i >> 1, pc = i & 1, v = v0 + pc * 8;
        if (t >= rows || v >= V) continue;
        const int64_t at = base + t * row_stride + v;
        const float *f = reinterpret_cast<const float *>(stg) + (2 * pc * 64 + t) * 4;
        const float4 x = *reinterpret_cast<const float4 *>(f), y = *reinterpret_cast<const float4 *>(f + 256);
        if (V % 8) {
            const float e[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (v + j < V) store_from_float(dst, dtype, at + j, e[j]);
        } else if (dtype == ASCAN_F32) {
            float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(dst) + at);
            o[0] = x;
            o[1] = y;
        } else {
            alignas(16) const __half2 h[4] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w), __floats2half2_rn(y.x, y.y), __floats2half2_rn(y.z, y.w)};
            *reinterpret_cast<uint4 *>(static_cast<__half *>(dst) + at) = *reinterpret_cast<const uint4 *>(h);
        }
    }
}

// the warp's 16 x KP accumulators (of the state, or KP = 64 tokens of e or z) to bf16 planes [plane][Vp][KP], through the
// staging area
template <int KP>
__device__ __forceinline__ void save_state(uint32_t stg, const unsigned char *stg_p, const float (&s)[KP / 8][4], bf16 *dst, int v0,
                                           int Vp, int lane) {
    constexpr int NCH = KP / 8;
#pragma unroll
    for (int pl = 0; pl < 2; ++pl) {
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

// Warps of a CTA that carry columns: eight share one copy of the chunk's tiles where shared memory holds their own ones as
// well; fewer while that would leave SMs without a CTA.  All eight load: with one warp for its own tiles, 100 KB a chunk
// and 200 copies a thread, loading took half of the time (1000 fp32 tokens, 8 heads of 128 x 64: 247 us a sweep, now 132).
constexpr int SWEEP_THREADS = 256;
__device__ __forceinline__ void sweep_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

static inline int sweep_warps(const DeltaParams &p, int sm_count, size_t (*bytes)(int)) {
    const int64_t slices = (p.Vp + 15) / 16, chains = int64_t(p.n_seqs) * p.H;
    int w = 8;
    while (w > 1 && (bytes(w) > 227 * 1024 || w / 2 >= slices || chains * ((slices + w - 1) / w) < sm_count)) w /= 2;
    return w;
}

}  // namespace ascan
