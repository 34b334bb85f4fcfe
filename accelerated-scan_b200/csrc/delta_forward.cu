// Gated delta rule: packing into bf16 planes, the per-chunk matrices, the forward sweep over the chunks.
#include "delta_sweep.cuh"

namespace ascan {

// ---- packing: any strides and type to rows of bf16 planes, zero-padded to a multiple of eight ------------------------

struct PackParams {
    const void *src;
    bf16 *dst;
    int64_t plane, sb, st, sh, T, rows;
    int32_t dtype, heads, d, dp;
};

// hi + lo holds an fp16 exactly (11 bits in 8 + 8) and an fp32 to 2^-16 of itself; bf16 fills one plane.
__global__ void delta_pack_kernel(PackParams p) {
    const int pieces = p.dp / 8;
    const int64_t total = p.rows * pieces;
    for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
        const int64_t row = i / pieces;
        const int c = static_cast<int>(i % pieces) * 8;
        const int h = static_cast<int>(row % p.heads);
        const int64_t bt = row / p.heads, t = bt % p.T, b = bt / p.T;
        const int64_t at = b * p.sb + t * p.st + h * p.sh;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = c + j < p.d ? load_as_float(p.src, p.dtype, at + c + j) : 0.f;
        uint4 hi, lo;
        split2(x[0], x[1], hi.x, lo.x);
        split2(x[2], x[3], hi.y, lo.y);
        split2(x[4], x[5], hi.z, lo.z);
        split2(x[6], x[7], hi.w, lo.w);
        *reinterpret_cast<uint4 *>(p.dst + row * p.dp + c) = hi;
        if (p.plane) *reinterpret_cast<uint4 *>(p.dst + p.plane + row * p.dp + c) = lo;
    }
}

int delta_launch_pack(const void *src, int dtype, const int64_t *strides, int64_t batch, int64_t T, int heads, int d, int dp,
                      bf16 *dst, int64_t plane, cudaStream_t st) {
    PackParams p = {src, dst, plane, strides[0], strides[1], strides[2], T, batch * T * heads, dtype, heads, d, dp};
    const int64_t blocks = (p.rows * (dp / 8) + 255) / 256;
    if (blocks == 0) return ASCAN_OK;
    delta_pack_kernel<<<static_cast<unsigned>(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

// ---- per-chunk matrices ----------------------------------------------------------------------------------------------
//
// One CTA of four warps per chunk and key head; K K^T and Q K^T are shared by the value heads of the group.  M solves
// (I + L diag(beta)) M = L: 16 x 16 diagonal blocks are inverted by substitution in fp32, the rest is four block rows
// in turn, all in fp32 (powers of L, as a series would need them, grow like binomial coefficients).  K K^T and Q K^T take all
// four term products: out and d_log_gates feel them most.  1000 fp32 tokens, 8 heads, K = 128: 32 us, bound by the
// substitutions' latency.

constexpr int PREP_PITCH = 68;     // floats; rows stay 16-byte aligned

template <int KP>
constexpr size_t prep_smem() {
    return size_t(4) * 64 * KP * 2 + 2 * 64 * PREP_PITCH * 4 + 4 * 16 * 20 * 4 + SC_ARRAYS * 64 * 4;
}

template <int KP>
__global__ void __launch_bounds__(128) delta_prep_kernel(DeltaParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int NCH = KP / 8, TILE = 64 * KP * 2;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slot = blockIdx.x, hk = blockIdx.y, group = p.H / p.Hk;
    const Chunk ch = get_chunk(p, slot);
    if (ch.rows == 0) return;
    const uint32_t sk = smem_addr(smem), sq = sk + 2 * TILE;
    float *sL = reinterpret_cast<float *>(smem + 4 * TILE), *sA = sL + 64 * PREP_PITCH, *sD = sA + 64 * PREP_PITCH;
    float *ssc = sD + 4 * 16 * 20;

    for (int pl = 0; pl < 2; ++pl) {
        load_tile<NCH>(sk + pl * TILE, p.k.p + pl * p.k.plane + ch.b * p.k.sb + ch.t0 * p.k.st + hk * p.k.sh, p.k.st, ch.rows,
                       p.Kp / 8, tid, 128);
        load_tile<NCH>(sq + pl * TILE, p.q.p + pl * p.q.plane + ch.b * p.q.sb + ch.t0 * p.q.st + hk * p.q.sh, p.q.st, ch.rows,
                       p.Kp / 8, tid, 128);
    }
    cp_commit();
    cp_wait<0>();
    __syncthreads();

    // rows 16 warp .. + 15 against the 16 (warp + 1) first tokens
    float kk[8][4] = {}, qk[8][4] = {};
#pragma unroll
    for (int s = 0; s < KP / 16; ++s) {
        uint32_t ak[2][4], aq[2][4];
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {
            ldsm4(ak[pl], addr_an<NCH>(sk + pl * TILE, 16 * warp, 2 * s, lane));
            ldsm4(aq[pl], addr_an<NCH>(sq + pl * TILE, 16 * warp, 2 * s, lane));
        }
#pragma unroll
        for (int np = 0; np < 4; ++np) {
            if (np > warp) break;
#pragma unroll
            for (int pl = 0; pl < 2; ++pl) {
                uint32_t b[4];
                ldsm4(b, addr_bn<NCH>(sk + pl * TILE, 16 * np, 2 * s, lane));
#pragma unroll
                for (int pa = 0; pa < 2; ++pa) {
                    mma(kk[2 * np], ak[pa], b[0], b[1]);
                    mma(kk[2 * np + 1], ak[pa], b[2], b[3]);
                    mma(qk[2 * np], aq[pa], b[0], b[1]);
                    mma(qk[2 * np + 1], aq[pa], b[2], b[3]);
                }
            }
        }
    }

    for (int hh = 0; hh < group; ++hh) {
        const int h = hk * group + hh;
        const int64_t at = int64_t(slot) * p.H + h;
        if (warp == 0) {     // running sum of the log gates in 64 bits, kept as two floats; zero gates are counted instead
            double sum[2];
            int reset[2];
            float beta[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int i = 2 * lane + j;
                float g = 0.f;
                beta[j] = 0.f;
                if (i < ch.rows) {
                    g = load_as_float(p.g, p.g_dtype, ch.b * p.g_s[0] + (ch.t0 + i) * p.g_s[1] + h * p.g_s[2]);
                    beta[j] = load_as_float(p.b, p.b_dtype, ch.b * p.b_s[0] + (ch.t0 + i) * p.b_s[1] + h * p.b_s[2]);
                }
                reset[j] = g <= -104.f;            // e^g is zero in fp32
                sum[j] = reset[j] ? 0.0 : double(g);
            }
            double s = sum[0] + sum[1];
            int r = reset[0] + reset[1];
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const double sp = __shfl_up_sync(~0u, s, d);
                const int rp = __shfl_up_sync(~0u, r, d);
                if (lane >= d) { s += sp; r += rp; }
            }
            const double last = __shfl_sync(~0u, s, 31);
            const int all = __shfl_sync(~0u, r, 31);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int i = 2 * lane + j;
                const double G = j ? s : s - sum[1];
                const int R = j ? r : r - reset[1];
                const float hi = float(G);
                ssc[SC_GAM * 64 + i] = R == 0 ? expf(hi) : 0.f;
                ssc[SC_GAMC * 64 + i] = R == all ? expf(float(last - G)) : 0.f;
                ssc[SC_BETA * 64 + i] = beta[j];
                ssc[SC_GHI * 64 + i] = hi;
                ssc[SC_GLO * 64 + i] = float(G - double(hi));
                ssc[SC_RESET * 64 + i] = float(R);
            }
        }
        __syncthreads();
        for (int i = tid; i < SC_ARRAYS * 64; i += 128) p.sc[at * SC_ARRAYS * 64 + i] = ssc[i];
        bf16 *gP = p.P + at * 2 * 4096;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            if (n > 2 * warp + 1) break;
            const int j = 8 * n + 2 * (lane & 3);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int i = 16 * warp + (lane >> 2) + 8 * half;
                float d[2];
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    d[c] = j + c <= i ? decay_between(ssc[SC_GHI * 64 + i], ssc[SC_GLO * 64 + i], ssc[SC_RESET * 64 + i],
                                                      ssc[SC_GHI * 64 + j + c], ssc[SC_GLO * 64 + j + c],
                                                      ssc[SC_RESET * 64 + j + c]) : 0.f;
                float2 l, a;
                l.x = j < i ? d[0] * kk[n][2 * half] : 0.f;
                l.y = j + 1 < i ? d[1] * kk[n][2 * half + 1] : 0.f;
                a.x = l.x * ssc[SC_BETA * 64 + j];
                a.y = l.y * ssc[SC_BETA * 64 + j + 1];
                *reinterpret_cast<float2 *>(sL + i * PREP_PITCH + j) = l;
                *reinterpret_cast<float2 *>(sA + i * PREP_PITCH + j) = a;
                uint32_t hi, lo;
                split2(j <= i ? p.scale * d[0] * qk[n][2 * half] : 0.f,
                       j + 1 <= i ? p.scale * d[1] * qk[n][2 * half + 1] : 0.f, hi, lo);
                *reinterpret_cast<uint32_t *>(gP + i * 64 + j) = hi;
                *reinterpret_cast<uint32_t *>(gP + 4096 + i * 64 + j) = lo;
            }
        }
        __syncthreads();
        if (tid < 64) {      // inverse of I + A on the diagonal blocks: one column a thread
            const int b = tid >> 4, c = tid & 15;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float acc = i == c ? 1.f : 0.f;
#pragma unroll
                for (int j = 0; j < i; ++j) acc -= sA[(16 * b + i) * PREP_PITCH + 16 * b + j] * x[j];
                x[i] = acc;
                sD[(b * 16 + i) * 20 + c] = acc;
            }
        }
        __syncthreads();
        // block rows: M_b = D_b (L_b - sum_{d<b} A_bd M_d), in place of L
        const int c = tid & 63, r0 = (tid >> 6) * 8;
        for (int b = 0; b < 4; ++b) {
            float acc[8];
            const bool live = c < 16 * (b + 1);
            if (live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = sL[(16 * b + r0 + i) * PREP_PITCH + c];
                for (int k = c & ~15; k < 16 * b; k += 4) {       // M is lower triangular
                    float m[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) m[j] = sL[(k + j) * PREP_PITCH + c];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float4 a = *reinterpret_cast<const float4 *>(sA + (16 * b + r0 + i) * PREP_PITCH + k);
                        acc[i] -= a.x * m[0] + a.y * m[1] + a.z * m[2] + a.w * m[3];
                    }
                }
            }
            __syncthreads();
            if (live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) sL[(16 * b + r0 + i) * PREP_PITCH + c] = acc[i];
            }
            __syncthreads();
            if (live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    float m[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) m[j] = sL[(16 * b + k + j) * PREP_PITCH + c];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float4 a = *reinterpret_cast<const float4 *>(sD + (b * 16 + r0 + i) * 20 + k);
                        acc[i] += a.x * m[0] + a.y * m[1] + a.z * m[2] + a.w * m[3];
                    }
                }
            }
            __syncthreads();
            if (live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) sL[(16 * b + r0 + i) * PREP_PITCH + c] = acc[i];
            }
            __syncthreads();
        }
        bf16 *gM = p.M + at * 2 * 4096;
        for (int i = tid; i < 64 * 8; i += 128) {
            const int r = i >> 3, cc = (i & 7) * 8;
            if (cc > (r | 15)) continue;         // 16 x 16 blocks above the diagonal are never read
            const float *m = sL + r * PREP_PITCH + cc;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = cc + j < r ? m[j] : 0.f;
            uint4 hi, lo;
            split2(x[0], x[1], hi.x, lo.x);
            split2(x[2], x[3], hi.y, lo.y);
            split2(x[4], x[5], hi.z, lo.z);
            split2(x[6], x[7], hi.w, lo.w);
            *reinterpret_cast<uint4 *>(gM + r * 64 + cc) = hi;
            *reinterpret_cast<uint4 *>(gM + 4096 + r * 64 + cc) = lo;
        }
        __syncthreads();
    }
}

template <int KP>
static int launch_prep(const DeltaParams &p, cudaStream_t st) {
    const size_t smem = prep_smem<KP>();
    if (cudaFuncSetAttribute(delta_prep_kernel<KP>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
        return ASCAN_ERR_LAUNCH;
    delta_prep_kernel<KP><<<dim3(p.slots, p.Hk), 128, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

int delta_launch_prep(const DeltaParams &p, cudaStream_t st) {
    if (p.slots == 0) return ASCAN_OK;
    return p.Kp <= 64 ? launch_prep<64>(p, st) : launch_prep<128>(p, st);
}

// ---- forward sweep ---------------------------------------------------------------------------------------------------
//
// The columns of S are independent of each other, so a warp carries 16 of them through a whole sequence by itself, as
// the transposed state S^T (16 x K) in the accumulators of its matrix instructions: accumulators of one product are,
// register by register, the A operand of the next, and S^T K^T -> x^T -> e^T -> S^T runs without shared memory or a
// barrier between the products.  The chunk's K, Q, M, P are shared by the warps of a CTA and double-buffered.
//
// For fp16 and fp32 inputs, which are two bf16 planes each (bf16 ones have a sweep of their own): every operand is two terms,
// hi + lo, off by at most 2^-16 of itself, and a product takes the three largest of the four term products, P u all four.
// fp32 results are 5.7e-6 off so, fp16 ones half an ulp.  A third term would halve the rate again and does not fit: K and Q
// of two chunks take 128 of the 227 KB at K = 128.
//
// Bound by the chain of a chunk in one warp, not by memory or the matrix pipe: 1000 fp32 tokens, 8 heads of 128 x 64 take
// 132 us (8.3 us a chunk, of which the warp's matrix instructions are about 3).

template <int KP>
struct SweepLayout {
    static constexpr int TILE = 64 * KP * 2;
    static constexpr int K = 0, Q = 2 * TILE, M = 4 * TILE, P = M + 2 * 8192, SC = P + 2 * 8192;
    static constexpr int V = SC + SC_ARRAYS * 256;
    static constexpr int V_WARP = 2 * 64 * 32;             // [plane][piece][64] of 16 bytes
    static constexpr int STAGING = 32 * KP > 4096 ? 32 * KP : 4096;
    static constexpr size_t bytes(int warps) { return 2 * (size_t(V) + size_t(warps) * V_WARP) + size_t(warps) * STAGING; }
};

template <int KP>
__device__ __forceinline__ void sweep_load(const DeltaParams &p, uint32_t base, const Sequence &sq, int c, int h, int hk, int v0_cta,
                                           int warps, int tid, int threads) {
    typedef SweepLayout<KP> L;
    const int64_t t0 = sq.t0 + int64_t(c) * 64, left = sq.len - int64_t(c) * 64;
    const int rows = static_cast<int>(left < 64 ? left : 64);
    const int64_t at = int64_t(sq.slot0 + c) * p.H + h;
#pragma unroll
    for (int pl = 0; pl < 2; ++pl) {
        load_tile<KP / 8>(base + L::K + pl * L::TILE, p.k.p + pl * p.k.plane + sq.b * p.k.sb + t0 * p.k.st + hk * p.k.sh, p.k.st,
                          rows, p.Kp / 8, tid, threads);
        load_tile<KP / 8>(base + L::Q + pl * L::TILE, p.q.p + pl * p.q.plane + sq.b * p.q.sb + t0 * p.q.st + hk * p.q.sh, p.q.st,
                          rows, p.Kp / 8, tid, threads);
        load_tile<8>(base + L::P + pl * 8192, p.P + (at * 2 + pl) * 4096, 64, 64, 8, tid, threads);
        const bf16 *v = p.v.p + pl * p.v.plane + sq.b * p.v.sb + t0 * p.v.st + h * p.v.sh;
        for (int i = tid; i < warps * 128; i += threads) {
            const int pc = i % (2 * warps), t = i / (2 * warps), col = v0_cta + pc * 8;
            const bool real = t < rows && col < p.Vp;
            cp16(base + L::V + (pc >> 1) * L::V_WARP + ((pl * 2 + (pc & 1)) * 64 + t) * 16,
                 real ? v + t * p.v.st + col : v, real);
        }
    }
    load_tile<8>(base + L::M, p.M + at * 2 * 4096, 64, 64, 8, tid, threads);
    load_tile<8>(base + L::M + 8192, p.M + (at * 2 + 1) * 4096, 64, 64, 8, tid, threads);
    for (int i = tid; i < SC_ARRAYS * 16; i += threads) cp16(base + L::SC + i * 16, p.sc + at * SC_ARRAYS * 64 + i * 4, true);
}

template <int KP, bool SAVE>
__global__ void __launch_bounds__(256, 1) delta_sweep_kernel(DeltaParams p, int warps) {
    extern __shared__ __align__(128) unsigned char smem[];
    typedef SweepLayout<KP> L;
    constexpr int NCH = KP / 8, KT = KP / 8;
    constexpr int threads = SWEEP_THREADS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t2 = 2 * (lane & 3);
    const int cta_cols = 16 * warps, slices = (p.Vp + cta_cols - 1) / cta_cols;
    const int slice = blockIdx.x % slices;
    const int h = (blockIdx.x / slices) % p.H, n_seq = blockIdx.x / slices / p.H;
    const int hk = h / (p.H / p.Hk), v0_cta = slice * cta_cols, v0 = v0_cta + 16 * warp;
    const Sequence sq = get_sequence(p, n_seq);
    const uint32_t base = smem_addr(smem), stage_bytes = L::V + warps * L::V_WARP;
    unsigned char *stg_p = smem + 2 * stage_bytes + warp * L::STAGING;
    const uint32_t stg = base + 2 * stage_bytes + warp * L::STAGING;

    float s[KT][4];
    const int64_t state_at = (int64_t(n_seq) * p.H + h) * p.K * p.V;
#pragma unroll
    for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = 8 * n + t2 + (j & 1), v = v0 + g + (j >> 1) * 8;
            s[n][j] = p.s0 && warp < warps && k < p.K && v < p.V ? p.s0[state_at + int64_t(k) * p.V + v] : 0.f;
        }

    if (sq.chunks > 0) {
        sweep_load<KP>(p, base, sq, 0, h, hk, v0_cta, warps, tid, threads);
        cp_commit();
    }
    for (int c = 0; c < sq.chunks; ++c) {
        if (c + 1 < sq.chunks) sweep_load<KP>(p, base + ((c + 1) & 1) * stage_bytes, sq, c + 1, h, hk, v0_cta, warps, tid, threads);
        cp_commit();
        cp_wait<1>();
        sweep_sync();
        if (warp >= warps) {           // loads only
            sweep_sync();
            continue;
        }
        const uint32_t st = base + (c & 1) * stage_bytes;
        const float *sc = reinterpret_cast<const float *>(smem + (c & 1) * stage_bytes + L::SC);
        const int64_t at = int64_t(sq.slot0 + c) * p.H + h;
        const int64_t left = sq.len - int64_t(c) * 64;
        const int rows = static_cast<int>(left < 64 ? left : 64);
        if (SAVE) save_state<KP>(stg, stg_p, s, p.S + at * 2 * p.Vp * KP, v0, p.Vp, lane);

        float x[8][4] = {}, o[8][4] = {};
#pragma unroll
        for (int kk = 0; kk < KP / 16; ++kk) {
            uint32_t a[2][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                split2(s[2 * kk + (j >> 1)][2 * (j & 1)], s[2 * kk + (j >> 1)][2 * (j & 1) + 1], a[0][j], a[1][j]);
#pragma unroll
            for (int np = 0; np < 4; ++np) {
                uint32_t b[4];
                ldsm4(b, addr_bn<NCH>(st + L::K, 16 * np, 2 * kk, lane));
                mma(x[2 * np], a[0], b[0], b[1]);
                mma(x[2 * np + 1], a[0], b[2], b[3]);
                mma(x[2 * np], a[1], b[0], b[1]);
                mma(x[2 * np + 1], a[1], b[2], b[3]);
                ldsm4(b, addr_bn<NCH>(st + L::K + L::TILE, 16 * np, 2 * kk, lane));
                mma(x[2 * np], a[0], b[0], b[1]);
                mma(x[2 * np + 1], a[0], b[2], b[3]);
                ldsm4(b, addr_bn<NCH>(st + L::Q, 16 * np, 2 * kk, lane));
                mma(o[2 * np], a[0], b[0], b[1]);
                mma(o[2 * np + 1], a[0], b[2], b[3]);
                mma(o[2 * np], a[1], b[0], b[1]);
                mma(o[2 * np + 1], a[1], b[2], b[3]);
                ldsm4(b, addr_bn<NCH>(st + L::Q + L::TILE, 16 * np, 2 * kk, lane));
                mma(o[2 * np], a[0], b[0], b[1]);
                mma(o[2 * np + 1], a[0], b[2], b[3]);
            }
        }
        // x = V - gam (K S0);  out so far scale gam (Q S0)
#pragma unroll
        for (int np = 0; np < 4; ++np) {
            float v[2][4] = {};
#pragma unroll
            for (int pl = 0; pl < 2; ++pl) {
                uint32_t r[4];
                const int m = lane >> 3;
                ldsm4t(r, st + L::V + warp * L::V_WARP + ((pl * 2 + (m & 1)) * 64 + 16 * np + (m >> 1) * 8 + (lane & 7)) * 16);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    v[j][0] += low_half(r[2 * j]);
                    v[j][1] += high_half(r[2 * j]);
                    v[j][2] += low_half(r[2 * j + 1]);
                    v[j][3] += high_half(r[2 * j + 1]);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 gam = *reinterpret_cast<const float2 *>(sc + SC_GAM * 64 + 16 * np + 8 * j + t2);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float ga = i & 1 ? gam.y : gam.x;
                    x[2 * np + j][i] = v[j][i] - ga * x[2 * np + j][i];
                    o[2 * np + j][i] *= p.scale * ga;
                }
            }
        }
        // e = x - M (beta x), in place: block kk changes later blocks and, last of all, itself
#pragma unroll
        for (int kk = 3; kk >= 0; --kk) {
            uint32_t a[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 be = *reinterpret_cast<const float2 *>(sc + SC_BETA * 64 + 16 * kk + 8 * j + t2);
                split2(-be.x * x[2 * kk + j][0], -be.y * x[2 * kk + j][1], a[0][2 * j], a[1][2 * j]);
                split2(-be.x * x[2 * kk + j][2], -be.y * x[2 * kk + j][3], a[0][2 * j + 1], a[1][2 * j + 1]);
            }
#pragma unroll
            for (int np = kk; np < 4; ++np) {
                uint32_t b[4];
                ldsm4(b, addr_bn<8>(st + L::M, 16 * np, 2 * kk, lane));
                mma(x[2 * np], a[0], b[0], b[1]);
                mma(x[2 * np + 1], a[0], b[2], b[3]);
                mma(x[2 * np], a[1], b[0], b[1]);
                mma(x[2 * np + 1], a[1], b[2], b[3]);
                ldsm4(b, addr_bn<8>(st + L::M + 8192, 16 * np, 2 * kk, lane));
                mma(x[2 * np], a[0], b[0], b[1]);
                mma(x[2 * np + 1], a[0], b[2], b[3]);
            }
        }
        if (SAVE) save_state<64>(stg, stg_p, x, p.e + at * 2 * 64 * p.Vp, v0, p.Vp, lane);
        const float gam_c = sc[SC_GAM * 64 + 63];
#pragma unroll
        for (int n = 0; n < KT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] *= gam_c;
        // out += P u;  S = gam_C S + K^T (Gam_C u)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uint32_t au[2][4], as[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 be = *reinterpret_cast<const float2 *>(sc + SC_BETA * 64 + 16 * kk + 8 * j + t2);
                const float2 gc = *reinterpret_cast<const float2 *>(sc + SC_GAMC * 64 + 16 * kk + 8 * j + t2);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float u0 = be.x * x[2 * kk + j][2 * i], u1 = be.y * x[2 * kk + j][2 * i + 1];
                    split2(u0, u1, au[0][2 * j + i], au[1][2 * j + i]);
                    split2(gc.x * u0, gc.y * u1, as[0][2 * j + i], as[1][2 * j + i]);
                }
            }
#pragma unroll
            for (int np = kk; np < 4; ++np) {
                uint32_t b[4];
                ldsm4(b, addr_bn<8>(st + L::P, 16 * np, 2 * kk, lane));
                mma(o[2 * np], au[0], b[0], b[1]);
                mma(o[2 * np + 1], au[0], b[2], b[3]);
                mma(o[2 * np], au[1], b[0], b[1]);
                mma(o[2 * np + 1], au[1], b[2], b[3]);
                ldsm4(b, addr_bn<8>(st + L::P + 8192, 16 * np, 2 * kk, lane));
                mma(o[2 * np], au[0], b[0], b[1]);
                mma(o[2 * np + 1], au[0], b[2], b[3]);
                mma(o[2 * np], au[1], b[0], b[1]);
                mma(o[2 * np + 1], au[1], b[2], b[3]);
            }
#pragma unroll
            for (int np = 0; np < KP / 16; ++np) {
                uint32_t b[4];
                ldsm4t(b, addr_bt<NCH>(st + L::K, 16 * kk, 2 * np, lane));
                mma(s[2 * np], as[0], b[0], b[1]);
                mma(s[2 * np + 1], as[0], b[2], b[3]);
                mma(s[2 * np], as[1], b[0], b[1]);
                mma(s[2 * np + 1], as[1], b[2], b[3]);
                ldsm4t(b, addr_bt<NCH>(st + L::K + L::TILE, 16 * kk, 2 * np, lane));
                mma(s[2 * np], as[0], b[0], b[1]);
                mma(s[2 * np + 1], as[0], b[2], b[3]);
            }
        }
        stage_transposed(stg, stg_p, o, lane);
        __syncwarp();
        const int64_t t0 = sq.t0 + int64_t(c) * 64;
        flush_out(stg_p, p.out, p.dtype, ((sq.b * p.T + t0) * p.H + h) * int64_t(p.V), int64_t(p.H) * p.V, rows, v0, p.V, lane);
        sweep_sync();
    }
    cp_wait<0>();
#pragma unroll
    for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = 8 * n + t2 + (j & 1), v = v0 + g + (j >> 1) * 8;
            if (warp < warps && k < p.K && v < p.V) p.s1[state_at + int64_t(k) * p.V + v] = s[n][j];
        }
    if (p.packed && (n_seq == 0 || n_seq == p.n_seqs - 1)) {      // tokens of no sequence: zeros
        const int64_t front = n_seq == 0 ? sq.t0 : 0, back = n_seq == p.n_seqs - 1 ? sq.t0 + sq.len : p.T;
        const int64_t rows = front + (p.T - back);
        for (int64_t i = tid; i < rows * cta_cols; i += threads) {
            const int64_t r = i / cta_cols;
            const int v = v0_cta + static_cast<int>(i % cta_cols);
            if (v < p.V) store_from_float(p.out, p.dtype, ((r < front ? r : back + (r - front)) * p.H + h) * p.V + v, 0.f);
        }
    }
}

template <int KP, bool SAVE>
static int launch_sweep(const DeltaParams &p, int sm_count, cudaStream_t st) {
    const int warps = sweep_warps(p, sm_count, SweepLayout<KP>::bytes);
    const size_t smem = SweepLayout<KP>::bytes(warps);
    const int64_t grid = int64_t(p.n_seqs) * p.H * ((p.Vp + 16 * warps - 1) / (16 * warps));
    if (grid > 0x7fffffff) return ASCAN_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(delta_sweep_kernel<KP, SAVE>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
        return ASCAN_ERR_LAUNCH;
    delta_sweep_kernel<KP, SAVE><<<unsigned(grid), SWEEP_THREADS, smem, st>>>(p, warps);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

int delta_launch_sweep(const DeltaParams &p, bool save, int sm_count, cudaStream_t st) {
    if (p.Kp <= 64) return save ? launch_sweep<64, true>(p, sm_count, st) : launch_sweep<64, false>(p, sm_count, st);
    return save ? launch_sweep<128, true>(p, sm_count, st) : launch_sweep<128, false>(p, sm_count, st);
}

}  // namespace ascan
