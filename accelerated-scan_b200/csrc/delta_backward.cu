// Gated delta rule, backward.  With d_out (times scale inside P and Q's factor) and the gradient dS1 of the state
// behind a chunk:
//     du = P^T d_out + Gam_C (K dS1);   z = du - M^T (beta du);   y = beta z
//     dV = y;   dbeta = e . z;   dS0 = gam_C dS1 + Q^T (scale gam d_out) - K^T (gam y)
//     D = scale Gam * lower(d_out u^T);   F = -Gam * strictly lower(y u^T)
//     dQ = scale gam (d_out S0^T) + D K
//     dK = [-gam (y S0^T) + F K] + [Gam_C (u dS1^T) + D^T Q + F^T K]  = read + write
//     dG = q . dQ + k . (read - write), and <S1, dS1> on the last token;   dg = sum of dG from the token to the chunk's end
// A sweep from the last chunk to the first produces dS1 and z of every chunk; a second kernel does the rest of a
// chunk by itself.
#include "delta_sweep.cuh"

namespace ascan {

// ---- backward sweep: as the forward one, on the transposed gradient of the state --------------------------------------

template <int KP>
struct BackLayout {
    static constexpr int TILE = 64 * KP * 2;
    static constexpr int K = 0, Q = 2 * TILE, M = 4 * TILE, P = M + 2 * 8192, SC = P + 2 * 8192;
    static constexpr int DO = SC + SC_ARRAYS * 256;
    static constexpr int DO_WARP = 2 * 64 * 32;
    static constexpr int STAGING = 32 * KP > 4096 ? 32 * KP : 4096;
    static constexpr size_t bytes(int warps) { return 2 * (size_t(DO) + size_t(warps) * DO_WARP) + size_t(warps) * STAGING; }
};

template <int KP>
__device__ __forceinline__ void back_load(const DeltaParams &p, uint32_t base, const Sequence &sq, int c, int h, int hk, int v0_cta,
                                          int warps, int tid, int threads) {
    typedef BackLayout<KP> L;
    const int64_t t0 = sq.t0 + int64_t(c) * 64, left = sq.len - int64_t(c) * 64;
    const int rows = static_cast<int>(left < 64 ? left : 64);
    const int64_t at = int64_t(sq.slot0 + c) * p.H + h;
#pragma unroll
    for (int pl = 0; pl < 2; ++pl) {
        load_tile<KP / 8>(base + L::K + pl * L::TILE, p.k.p + pl * p.k.plane + sq.b * p.k.sb + t0 * p.k.st + hk * p.k.sh, p.k.st,
                          rows, p.Kp / 8, tid, threads);
        load_tile<KP / 8>(base + L::Q + pl * L::TILE, p.q.p + pl * p.q.plane + sq.b * p.q.sb + t0 * p.q.st + hk * p.q.sh, p.q.st,
                          rows, p.Kp / 8, tid, threads);
        const bf16 *v = p.d_out.p + pl * p.d_out.plane + sq.b * p.d_out.sb + t0 * p.d_out.st + h * p.d_out.sh;
        for (int i = tid; i < warps * 128; i += threads) {
            const int pc = i % (2 * warps), t = i / (2 * warps), col = v0_cta + pc * 8;
            const bool real = t < rows && col < p.Vp;
            cp16(base + L::DO + (pc >> 1) * L::DO_WARP + ((pl * 2 + (pc & 1)) * 64 + t) * 16,
                 real ? v + t * p.d_out.st + col : v, real);
        }
    }
    for (int pl = 0; pl < 2; ++pl) {
        load_tile<8>(base + L::M + pl * 8192, p.M + (at * 2 + pl) * 4096, 64, 64, 8, tid, threads);
        load_tile<8>(base + L::P + pl * 8192, p.P + (at * 2 + pl) * 4096, 64, 64, 8, tid, threads);
    }
    for (int i = tid; i < SC_ARRAYS * 16; i += threads) cp16(base + L::SC + i * 16, p.sc + at * SC_ARRAYS * 64 + i * 4, true);
}

template <int KP>
__global__ void __launch_bounds__(256, 1) delta_back_sweep_kernel(DeltaParams p, int warps) {
    extern __shared__ __align__(128) unsigned char smem[];
    typedef BackLayout<KP> L;
    constexpr int NCH = KP / 8, KT = KP / 8;
    constexpr int threads = SWEEP_THREADS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t2 = 2 * (lane & 3);
    const int cta_cols = 16 * warps, slices = (p.Vp + cta_cols - 1) / cta_cols;
    const int slice = blockIdx.x % slices;
    const int h = (blockIdx.x / slices) % p.H, n_seq = blockIdx.x / slices / p.H;
    const int hk = h / (p.H / p.Hk), v0_cta = slice * cta_cols, v0 = v0_cta + 16 * warp;
    const Sequence sq = get_sequence(p, n_seq);
    const uint32_t base = smem_addr(smem), stage_bytes = L::DO + warps * L::DO_WARP;
    unsigned char *stg_p = smem + 2 * stage_bytes + warp * L::STAGING;
    const uint32_t stg = base + 2 * stage_bytes + warp * L::STAGING;

    float s[KT][4];
    const int64_t state_at = (int64_t(n_seq) * p.H + h) * p.K * p.V;
#pragma unroll
    for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = 8 * n + t2 + (j & 1), v = v0 + g + (j >> 1) * 8;
            s[n][j] = p.d_s1 && warp < warps && k < p.K && v < p.V ? p.d_s1[state_at + int64_t(k) * p.V + v] : 0.f;
        }

    if (sq.chunks > 0) {
        back_load<KP>(p, base, sq, sq.chunks - 1, h, hk, v0_cta, warps, tid, threads);
        cp_commit();
    }
    for (int c = sq.chunks - 1, turn = 0; c >= 0; --c, turn ^= 1) {
        if (c > 0) back_load<KP>(p, base + (turn ^ 1) * stage_bytes, sq, c - 1, h, hk, v0_cta, warps, tid, threads);
        cp_commit();
        cp_wait<1>();
        sweep_sync();
        if (warp >= warps) {           // loads only
            sweep_sync();
            continue;
        }
        const uint32_t st = base + turn * stage_bytes;
        const float *sc = reinterpret_cast<const float *>(smem + turn * stage_bytes + L::SC);
        const int64_t at = int64_t(sq.slot0 + c) * p.H + h;
        save_state<KP>(stg, stg_p, s, p.dS + at * 2 * p.Vp * KP, v0, p.Vp, lane);

        float d[8][4] = {};
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
                mma(d[2 * np], a[0], b[0], b[1]);
                mma(d[2 * np + 1], a[0], b[2], b[3]);
                mma(d[2 * np], a[1], b[0], b[1]);
                mma(d[2 * np + 1], a[1], b[2], b[3]);
                ldsm4(b, addr_bn<NCH>(st + L::K + L::TILE, 16 * np, 2 * kk, lane));
                mma(d[2 * np], a[0], b[0], b[1]);
                mma(d[2 * np + 1], a[0], b[2], b[3]);
            }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float2 gc = *reinterpret_cast<const float2 *>(sc + SC_GAMC * 64 + 8 * n + t2);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[n][i] *= i & 1 ? gc.y : gc.x;
        }
        const float gam_c = sc[SC_GAM * 64 + 63];
#pragma unroll
        for (int n = 0; n < KT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] *= gam_c;
        // du += P^T d_out, and dS += Q^T (scale gam d_out)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uint32_t a[2][4], as[2][4];
#pragma unroll
            for (int pl = 0; pl < 2; ++pl) {
                const int m = lane >> 3;
                ldsm4t(a[pl], st + L::DO + warp * L::DO_WARP + ((pl * 2 + (m & 1)) * 64 + 16 * kk + (m >> 1) * 8 + (lane & 7)) * 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 gam = *reinterpret_cast<const float2 *>(sc + SC_GAM * 64 + 16 * kk + 8 * (j >> 1) + t2);
                float x0 = low_half(a[0][j]), x1 = high_half(a[0][j]);
                x0 += low_half(a[1][j]);
                x1 += high_half(a[1][j]);
                split2(p.scale * gam.x * x0, p.scale * gam.y * x1, as[0][j], as[1][j]);
            }
#pragma unroll
            for (int np = 0; np <= kk; ++np) {
                uint32_t b[4];
                ldsm4t(b, addr_bt<8>(st + L::P, 16 * kk, 2 * np, lane));
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    mma(d[2 * np], a[pl], b[0], b[1]);
                    mma(d[2 * np + 1], a[pl], b[2], b[3]);
                }
                ldsm4t(b, addr_bt<8>(st + L::P + 8192, 16 * kk, 2 * np, lane));
                mma(d[2 * np], a[0], b[0], b[1]);
                mma(d[2 * np + 1], a[0], b[2], b[3]);
            }
#pragma unroll
            for (int np = 0; np < KP / 16; ++np) {
                uint32_t b[4];
                ldsm4t(b, addr_bt<NCH>(st + L::Q, 16 * kk, 2 * np, lane));
                mma(s[2 * np], as[0], b[0], b[1]);
                mma(s[2 * np + 1], as[0], b[2], b[3]);
                mma(s[2 * np], as[1], b[0], b[1]);
                mma(s[2 * np + 1], as[1], b[2], b[3]);
                ldsm4t(b, addr_bt<NCH>(st + L::Q + L::TILE, 16 * kk, 2 * np, lane));
                mma(s[2 * np], as[0], b[0], b[1]);
                mma(s[2 * np + 1], as[0], b[2], b[3]);
            }
        }
        // z = du - M^T (beta du), in place: block kk changes earlier blocks and itself
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uint32_t a[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 be = *reinterpret_cast<const float2 *>(sc + SC_BETA * 64 + 16 * kk + 8 * j + t2);
                split2(-be.x * d[2 * kk + j][0], -be.y * d[2 * kk + j][1], a[0][2 * j], a[1][2 * j]);
                split2(-be.x * d[2 * kk + j][2], -be.y * d[2 * kk + j][3], a[0][2 * j + 1], a[1][2 * j + 1]);
            }
#pragma unroll
            for (int np = 0; np <= kk; ++np) {
                uint32_t b[4];
                ldsm4t(b, addr_bt<8>(st + L::M, 16 * kk, 2 * np, lane));
                mma(d[2 * np], a[0], b[0], b[1]);
                mma(d[2 * np + 1], a[0], b[2], b[3]);
                mma(d[2 * np], a[1], b[0], b[1]);
                mma(d[2 * np + 1], a[1], b[2], b[3]);
                ldsm4t(b, addr_bt<8>(st + L::M + 8192, 16 * kk, 2 * np, lane));
                mma(d[2 * np], a[0], b[0], b[1]);
                mma(d[2 * np + 1], a[0], b[2], b[3]);
            }
        }
        save_state<64>(stg, stg_p, d, p.z + at * 2 * 64 * p.Vp, v0, p.Vp, lane);
        // y = beta z = dV
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float2 be = *reinterpret_cast<const float2 *>(sc + SC_BETA * 64 + 8 * n + t2);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[n][i] *= i & 1 ? be.y : be.x;
        }
        stage_transposed(stg, stg_p, d, lane);
        __syncwarp();
        const int64_t tok = sq.t0 + int64_t(c) * 64, left = sq.len - int64_t(c) * 64;
        flush_out(stg_p, p.d_v, p.dtype, ((sq.b * p.T + tok) * p.H + h) * int64_t(p.V), int64_t(p.H) * p.V,
                      static_cast<int>(left < 64 ? left : 64), v0, p.V, lane);
        // dS -= K^T (gam y)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uint32_t as[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 ga = *reinterpret_cast<const float2 *>(sc + SC_GAM * 64 + 16 * kk + 8 * j + t2);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    split2(-ga.x * d[2 * kk + j][2 * i], -ga.y * d[2 * kk + j][2 * i + 1], as[0][2 * j + i], as[1][2 * j + i]);
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
        sweep_sync();
    }
    cp_wait<0>();
    if (p.d_s0 && warp < warps) {
#pragma unroll
        for (int n = 0; n < KT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 8 * n + t2 + (j & 1), v = v0 + g + (j >> 1) * 8;
                if (k < p.K && v < p.V) p.d_s0[state_at + int64_t(k) * p.V + v] = s[n][j];
            }
    }
}

template <int KP>
static int launch_back_sweep(const DeltaParams &p, int sm_count, cudaStream_t st) {
    const int warps = sweep_warps(p, sm_count, BackLayout<KP>::bytes);
    const size_t smem = BackLayout<KP>::bytes(warps);
    const int64_t grid = int64_t(p.n_seqs) * p.H * ((p.Vp + 16 * warps - 1) / (16 * warps));
    if (grid > 0x7fffffff) return ASCAN_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(delta_back_sweep_kernel<KP>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
        return ASCAN_ERR_LAUNCH;
    delta_back_sweep_kernel<KP><<<unsigned(grid), SWEEP_THREADS, smem, st>>>(p, warps);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

int delta_launch_back_sweep(const DeltaParams &p, int sm_count, cudaStream_t st) {
    return p.Kp <= 64 ? launch_back_sweep<64>(p, sm_count, st) : launch_back_sweep<128>(p, sm_count, st);
}

// ---- gradients of a chunk --------------------------------------------------------------------------------------------
//
// For fp16 and fp32 inputs.  One CTA of eight warps per chunk and key head; the value heads of the group follow one another
// and their dQ, dK are summed in registers, in a fixed order.  V is walked in slabs of 32 columns (d_out, e, z, S0, dS1 of
// the slab, double-buffered); a warp holds 16 tokens x half of K of dQ, dK read and dK write.  Two terms an operand as in the
// sweeps.  1000 fp32 tokens, 8 heads of 128 x 64: 21 us for 44 MB, one turn of the grid, bound by its latency.

template <int KP>
struct GradLayout {
    static constexpr int TILE = 64 * KP * 2;
    static constexpr int VS = 32;                              // columns of a slab
    static constexpr int VCH = VS / 8;
    static constexpr int TOK = 64 * VS * 2, STATE = VS * KP * 2;
    static constexpr int SLAB = 2 * (3 * TOK + 2 * STATE);
    static constexpr int K = 0, Q = 2 * TILE, D = 4 * TILE, F = D + 2 * 8192, SLABS = F + 2 * 8192;
    static constexpr int SC = SLABS + 2 * SLAB, RED = SC + SC_ARRAYS * 256, BYTES = RED + (192 + 256 + 256) * 4;
    // inside a slab; e and z lie transposed, VS rows of 64 tokens
    static constexpr int DO = 0, E = 2 * TOK, Z = 4 * TOK, S = 6 * TOK, DS = S + 2 * STATE;
};

template <int KP>
__device__ __forceinline__ void grad_load(const DeltaParams &p, uint32_t base, const Chunk &ch, int64_t at, int h, int v0, int tid) {
    typedef GradLayout<KP> L;
    const int left = p.Vp - v0, pieces = (left < L::VS ? left : L::VS) / 8, rows = left < L::VS ? left : L::VS;
#pragma unroll
    for (int pl = 0; pl < 2; ++pl) {
        load_tile<L::VCH>(base + L::DO + pl * L::TOK, p.d_out.p + pl * p.d_out.plane + ch.b * p.d_out.sb + ch.t0 * p.d_out.st +
                          h * p.d_out.sh + v0, p.d_out.st, ch.rows, pieces, tid, 256);
        load_tile<8>(base + L::E + pl * L::TOK, p.e + ((at * 2 + pl) * p.Vp + v0) * 64, 64, rows, 8, tid, 256, L::VS);
        load_tile<8>(base + L::Z + pl * L::TOK, p.z + ((at * 2 + pl) * p.Vp + v0) * 64, 64, rows, 8, tid, 256, L::VS);
        load_tile<KP / 8>(base + L::S + pl * L::STATE, p.S + ((at * 2 + pl) * p.Vp + v0) * KP, KP, rows, KP / 8, tid, 256, L::VS);
        load_tile<KP / 8>(base + L::DS + pl * L::STATE, p.dS + ((at * 2 + pl) * p.Vp + v0) * KP, KP, rows, KP / 8, tid, 256, L::VS);
    }
}

__device__ __forceinline__ void read8(const unsigned char *tile, int plane_bytes, uint32_t off, float (&x)[8]) {
    const uint4 r = *reinterpret_cast<const uint4 *>(tile + off);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = low_half(w[j]);
        x[2 * j + 1] = high_half(w[j]);
    }
    const uint4 l = *reinterpret_cast<const uint4 *>(tile + plane_bytes + off);
    const uint32_t u[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] += low_half(u[j]);
        x[2 * j + 1] += high_half(u[j]);
    }
}

// two neighbouring elements of a K tile
template <int KP>
__device__ __forceinline__ float2 read_pair(const unsigned char *tile, int row, int col) {
    const uint32_t off = tile_off<KP / 8>(row, col >> 3) + (col & 7) * 2;
    const uint32_t r = *reinterpret_cast<const uint32_t *>(tile + off);
    float2 x = make_float2(low_half(r), high_half(r));
    const uint32_t l = *reinterpret_cast<const uint32_t *>(tile + 64 * KP * 2 + off);
    x.x += low_half(l);
    x.y += high_half(l);
    return x;
}

__device__ __forceinline__ void store_pair(void *dst, int dtype, int64_t at, int col, int cols, float x0, float x1, bool even) {
    if (col >= cols) return;
    if (even) {            // rows start at even elements, cols is even
        if (dtype == ASCAN_F16) *reinterpret_cast<__half2 *>(static_cast<__half *>(dst) + at + col) = __floats2half2_rn(x0, x1);
        else *reinterpret_cast<float2 *>(static_cast<float *>(dst) + at + col) = make_float2(x0, x1);
    } else {
        store_from_float(dst, dtype, at + col, x0);
        if (col + 1 < cols) store_from_float(dst, dtype, at + col + 1, x1);
    }
}

// C (16 x 8 NTILES) += A[pa] B[pb] over the kept term products; A fragments given, B from a tile by transposed loads
template <int NTILES, int NCH>
__device__ __forceinline__ void mma_bt(float (&c)[NTILES][4], const uint32_t (&a)[2][4], uint32_t tile, int plane, int k0, int c0,
                                       int lane) {
#pragma unroll
    for (int np = 0; np < NTILES / 2; ++np)
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {
            uint32_t b[4];
            ldsm4t(b, addr_bt<NCH>(tile + pl * plane, k0, c0 + 2 * np, lane));
#pragma unroll
            for (int pa = 0; pa + pl < 2; ++pa) {
                mma(c[2 * np], a[pa], b[0], b[1]);
                mma(c[2 * np + 1], a[pa], b[2], b[3]);
            }
        }
}

template <int KP, bool GROUPED>
__global__ void __launch_bounds__(256, 1) delta_grads_kernel(DeltaParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    typedef GradLayout<KP> L;
    constexpr int NCH = KP / 8, KT = KP / 16;          // KT: tiles of eight columns a warp holds
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wr = warp >> 1, wc = warp & 1;
    const int g = lane >> 2, t2 = 2 * (lane & 3);
    const int slot = blockIdx.x, hk = blockIdx.y, group = p.H / p.Hk;
    const Chunk ch = get_chunk(p, slot);
    if (ch.rows == 0) return;
    const uint32_t base = smem_addr(smem);
    float *ssc = reinterpret_cast<float *>(smem + L::SC), *red = reinterpret_cast<float *>(smem + L::RED);

#pragma unroll
    for (int pl = 0; pl < 2; ++pl) {
        load_tile<NCH>(base + L::K + pl * L::TILE, p.k.p + pl * p.k.plane + ch.b * p.k.sb + ch.t0 * p.k.st + hk * p.k.sh, p.k.st,
                       ch.rows, p.Kp / 8, tid, 256);
        load_tile<NCH>(base + L::Q + pl * L::TILE, p.q.p + pl * p.q.plane + ch.b * p.q.sb + ch.t0 * p.q.st + hk * p.q.sh, p.q.st,
                       ch.rows, p.Kp / 8, tid, 256);
    }
    const int slabs = (p.Vp + L::VS - 1) / L::VS, turns = group * slabs;
    grad_load<KP>(p, base + L::SLABS, ch, int64_t(slot) * p.H + hk * group, hk * group, 0, tid);
    cp_commit();

    float rq[GROUPED ? KT : 1][4] = {}, rk[GROUPED ? KT : 1][4] = {};
    float dq[KT][4], dr[KT][4], dw[KT][4], dp[4][4], df[4][4];
    float dot_s = 0.f, dbeta = 0.f;
    for (int turn = 0; turn < turns; ++turn) {
        const int hh = turn / slabs, slab = turn % slabs, h = hk * group + hh, v0 = slab * L::VS;
        const int64_t at = int64_t(slot) * p.H + h;
        if (turn + 1 < turns) {
            const int h1 = hk * group + (turn + 1) / slabs;
            grad_load<KP>(p, base + L::SLABS + ((turn + 1) & 1) * L::SLAB, ch, int64_t(slot) * p.H + h1, h1,
                              (turn + 1) % slabs * L::VS, tid);
        }
        cp_commit();
        if (slab == 0) {
            for (int i = tid; i < SC_ARRAYS * 64; i += 256) ssc[i] = p.sc[at * SC_ARRAYS * 64 + i];
#pragma unroll
            for (int n = 0; n < KT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) dq[n][j] = dr[n][j] = dw[n][j] = 0.f;
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) dp[n][j] = df[n][j] = 0.f;
            dot_s = dbeta = 0.f;
        }
        cp_wait<1>();
        __syncthreads();
        const uint32_t sb = base + L::SLABS + (turn & 1) * L::SLAB;
        const unsigned char *sp = smem + L::SLABS + (turn & 1) * L::SLAB;
#pragma unroll
        for (int kk = 0; kk < L::VS / 16; ++kk) {
            uint32_t ao[2][4], ae[2][4], az[2][4];
#pragma unroll
            for (int pl = 0; pl < 2; ++pl) {
                ldsm4(ao[pl], addr_an<L::VCH>(sb + L::DO + pl * L::TOK, 16 * wr, 2 * kk, lane));
                ldsm4t(ae[pl], addr_at<8>(sb + L::E + pl * L::TOK, 16 * kk, 2 * wr, lane));
                ldsm4t(az[pl], addr_at<8>(sb + L::Z + pl * L::TOK, 16 * kk, 2 * wr, lane));
            }
#pragma unroll
            for (int np = 0; np < KT / 2; ++np)
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    uint32_t b[4];
                    ldsm4t(b, addr_bt<NCH>(sb + L::S + pl * L::STATE, 16 * kk, wc * KT + 2 * np, lane));
#pragma unroll
                    for (int pa = 0; pa + pl < 2; ++pa) {
                        mma(dq[2 * np], ao[pa], b[0], b[1]);
                        mma(dq[2 * np + 1], ao[pa], b[2], b[3]);
                        mma(dr[2 * np], az[pa], b[0], b[1]);
                        mma(dr[2 * np + 1], az[pa], b[2], b[3]);
                    }
                    ldsm4t(b, addr_bt<NCH>(sb + L::DS + pl * L::STATE, 16 * kk, wc * KT + 2 * np, lane));
#pragma unroll
                    for (int pa = 0; pa + pl < 2; ++pa) {
                        mma(dw[2 * np], ae[pa], b[0], b[1]);
                        mma(dw[2 * np + 1], ae[pa], b[2], b[3]);
                    }
                }
#pragma unroll
            for (int np = 0; np < 2; ++np) {
                if (2 * wc + np > wr) break;                 // above the diagonal
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    uint32_t b[4];
                    ldsm4t(b, addr_bt<8>(sb + L::E + pl * L::TOK, 16 * kk, 4 * wc + 2 * np, lane));
#pragma unroll
                    for (int pa = 0; pa < 2; ++pa) {
                        mma(dp[2 * np], ao[pa], b[0], b[1]);
                        mma(dp[2 * np + 1], ao[pa], b[2], b[3]);
                        mma(df[2 * np], az[pa], b[0], b[1]);
                        mma(df[2 * np + 1], az[pa], b[2], b[3]);
                    }
                }
            }
        }
        {   // dbeta = e . z: four threads a token, a quarter of the slab each;  <S0, dS1>: every thread
            const int t = tid & 63, part = tid >> 6;
            for (int i = 0; i < L::VS / 4; ++i) {
                const uint32_t o = tile_off<8>(part * (L::VS / 4) + i, t >> 3) + (t & 7) * 2;
                float e = __bfloat162float(*reinterpret_cast<const bf16 *>(sp + L::E + o));
                float z = __bfloat162float(*reinterpret_cast<const bf16 *>(sp + L::Z + o));
                e += __bfloat162float(*reinterpret_cast<const bf16 *>(sp + L::E + L::TOK + o));
                z += __bfloat162float(*reinterpret_cast<const bf16 *>(sp + L::Z + L::TOK + o));
                dbeta += e * z;
            }
            for (int i = tid; i < L::VS * NCH; i += 256) {
                float a[8], b[8];
                read8(sp + L::S, L::STATE, uint32_t(i) * 16, a);
                read8(sp + L::DS, L::STATE, uint32_t(i) * 16, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) dot_s += a[j] * b[j];
            }
        }
        if (slab == slabs - 1) {
            const int i0 = 16 * wr + g;
            // D and F to shared memory; row factors; W_ij = D_ij (q_i . k_j) = beta_j (d_out_i . e_j) P_ij
            float dot[2] = {};
            const bf16 *gP = p.P + at * 2 * 4096;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int j = 32 * wc + 8 * n + t2;
                float col[2] = {};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = i0 + 8 * half;
                    float d[2] = {}, f[2] = {};
                    if (j <= i) {
                        const uint32_t ph = *reinterpret_cast<const uint32_t *>(gP + i * 64 + j);
                        const uint32_t pl = *reinterpret_cast<const uint32_t *>(gP + 4096 + i * 64 + j);
                        const float pp[2] = {low_half(ph) + low_half(pl), high_half(ph) + high_half(pl)};
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float be = ssc[SC_BETA * 64 + j + c];
                            const float dec = be * decay_between(ssc[SC_GHI * 64 + i], ssc[SC_GLO * 64 + i], ssc[SC_RESET * 64 + i],
                                ssc[SC_GHI * 64 + j + c], ssc[SC_GLO * 64 + j + c], ssc[SC_RESET * 64 + j + c]);
                            if (j + c <= i) d[c] = p.scale * dec * dp[n][2 * half + c];
                            if (j + c < i) f[c] = -ssc[SC_BETA * 64 + i] * dec * df[n][2 * half + c];
                            const float w = j + c < i ? be * dp[n][2 * half + c] * pp[c] : 0.f;
                            dot[half] += w;
                            col[c] += w;
                        }
                    }
                    uint32_t hi, lo;
                    const uint32_t off = tile_off<8>(i, j >> 3) + (j & 7) * 2;
                    split2(d[0], d[1], hi, lo);
                    *reinterpret_cast<uint32_t *>(smem + L::D + off) = hi;
                    *reinterpret_cast<uint32_t *>(smem + L::D + 8192 + off) = lo;
                    split2(f[0], f[1], hi, lo);
                    *reinterpret_cast<uint32_t *>(smem + L::F + off) = hi;
                    *reinterpret_cast<uint32_t *>(smem + L::F + 8192 + off) = lo;
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int m = 4; m < 32; m *= 2) col[c] += __shfl_xor_sync(~0u, col[c], m);
                    if (g == 0) red[448 + wr * 64 + j + c] = col[c];
                }
            }
            float w_dot[2] = {};
#pragma unroll
            for (int n = 0; n < KT; ++n)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = i0 + 8 * half;
                    const float gam = ssc[SC_GAM * 64 + i], be = ssc[SC_BETA * 64 + i], gc = ssc[SC_GAMC * 64 + i];
                    const float2 k = read_pair<KP>(smem + L::K, i, (wc * KT + n) * 8 + t2);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        dq[n][2 * half + c] *= p.scale * gam;
                        dr[n][2 * half + c] *= -gam * be;
                        dw[n][2 * half + c] *= gc * be;
                    }
                    w_dot[half] += k.x * dw[n][2 * half] + k.y * dw[n][2 * half + 1];
                }
            dot_s = dot_s * ssc[SC_GAM * 64 + 63] + w_dot[0] + w_dot[1];        // to <S1, dS1>
            __syncthreads();
            // F's products, the sums over K, then D's: in dG_i = sum_j W_ij - sum_j W_ji and what stands beside it, most of the two
            // sums cancels from token to token, so both are taken of the same W and not of D's products (two-term products in
            // their place leave fp32 gates 1.3e-5 off)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                uint32_t a[2][4];
                if (kk <= wr) {
#pragma unroll
                    for (int pl = 0; pl < 2; ++pl) ldsm4(a[pl], addr_an<8>(base + L::F + pl * 8192, 16 * wr, 2 * kk, lane));
                    mma_bt<KT, NCH>(dr, a, base + L::K, L::TILE, 16 * kk, wc * KT, lane);
                }
                if (kk >= wr) {
#pragma unroll
                    for (int pl = 0; pl < 2; ++pl) ldsm4t(a[pl], addr_at<8>(base + L::F + pl * 8192, 16 * kk, 2 * wr, lane));
                    mma_bt<KT, NCH>(dw, a, base + L::K, L::TILE, 16 * kk, wc * KT, lane);
                }
            }
#pragma unroll
            for (int n = 0; n < KT; ++n)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = i0 + 8 * half, col = (wc * KT + n) * 8 + t2;
                    const float2 k = read_pair<KP>(smem + L::K, i, col), q = read_pair<KP>(smem + L::Q, i, col);
                    dot[half] += q.x * dq[n][2 * half] + q.y * dq[n][2 * half + 1];
                    dot[half] += k.x * (dr[n][2 * half] - dw[n][2 * half]) + k.y * (dr[n][2 * half + 1] - dw[n][2 * half + 1]);
                }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                uint32_t a[2][4];
                if (kk <= wr) {
#pragma unroll
                    for (int pl = 0; pl < 2; ++pl) ldsm4(a[pl], addr_an<8>(base + L::D + pl * 8192, 16 * wr, 2 * kk, lane));
                    mma_bt<KT, NCH>(dq, a, base + L::K, L::TILE, 16 * kk, wc * KT, lane);
                }
                if (kk >= wr) {
#pragma unroll
                    for (int pl = 0; pl < 2; ++pl) ldsm4t(a[pl], addr_at<8>(base + L::D + pl * 8192, 16 * kk, 2 * wr, lane));
                    mma_bt<KT, NCH>(dw, a, base + L::Q, L::TILE, 16 * kk, wc * KT, lane);
                }
            }
            if (GROUPED) {
#pragma unroll
                for (int n = 0; n < KT; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        rq[GROUPED ? n : 0][c] += dq[n][c];
                        rk[GROUPED ? n : 0][c] += dr[n][c] + dw[n][c];
                    }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                dot[half] += __shfl_xor_sync(~0u, dot[half], 1);
                dot[half] += __shfl_xor_sync(~0u, dot[half], 2);
                if ((lane & 3) == 0) red[wc * 64 + i0 + 8 * half] = dot[half];
            }
#pragma unroll
            for (int d = 16; d; d /= 2) dot_s += __shfl_xor_sync(~0u, dot_s, d);
            if (lane == 0) red[128 + warp] = dot_s;
            red[192 + tid] = dbeta;
            const int64_t row = ch.b * p.T + ch.t0;
            __syncthreads();
            if (tid >= 64 && tid - 64 < ch.rows) {
                const float *r = red + 128 + tid;
                store_from_float(p.d_b, p.b_dtype, (row + tid - 64) * p.H + h, (r[0] + r[64]) + (r[128] + r[192]));
            }
            if (warp == 0) {            // sums of dG from each token to the end; the state's share stands on the last one
                float x[2], tail = 0.f;
#pragma unroll
                for (int w = 0; w < 8; ++w) tail += red[128 + w];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float *r = red + 2 * lane + j, *w = r + 448;
                    x[j] = (r[0] + r[64]) - ((w[0] + w[64]) + (w[128] + w[192]));
                }
                float s = x[0] + x[1];
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const float o = __shfl_down_sync(~0u, s, d);
                    if (lane + d < 32) s += o;
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int i = 2 * lane + j;
                    const float before = i == 0 ? 0.f : ssc[SC_RESET * 64 + i - 1];
                    const float dg = ssc[SC_RESET * 64 + i] != before ? 0.f : tail + (j ? s - x[0] : s);
                    if (i < ch.rows) store_from_float(p.d_g, p.g_dtype, (row + i) * p.H + h, dg);
                }
            }
        }
        __syncthreads();
    }
    cp_wait<0>();
#pragma unroll
    for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = 16 * wr + g + 8 * half, col = (wc * KT + n) * 8 + t2;
            if (i >= ch.rows) continue;
            const int64_t o = ((ch.b * p.T + ch.t0 + i) * p.Hk + hk) * p.K;
            if (GROUPED) {
                constexpr int G = GROUPED ? 1 : 0;
                store_pair(p.d_q, p.dtype, o, col, p.K, rq[G * n][2 * half], rq[G * n][2 * half + 1], p.K % 2 == 0);
                store_pair(p.d_k, p.dtype, o, col, p.K, rk[G * n][2 * half], rk[G * n][2 * half + 1], p.K % 2 == 0);
            } else {
                store_pair(p.d_q, p.dtype, o, col, p.K, dq[n][2 * half], dq[n][2 * half + 1], p.K % 2 == 0);
                store_pair(p.d_k, p.dtype, o, col, p.K, dr[n][2 * half] + dw[n][2 * half], dr[n][2 * half + 1] + dw[n][2 * half + 1],
                           p.K % 2 == 0);
            }
        }
}

// Gradients of tokens that lie in no sequence of a packed row are zero.
__global__ void delta_zero_outside_kernel(DeltaParams p) {
    const int64_t front = seq_start(p, 0), back = seq_start(p, p.n_seqs), rows = front + (p.T - back);
    const int64_t nq = int64_t(p.Hk) * p.K, nv = int64_t(p.H) * p.V;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int64_t t = r < front ? r : back + (r - front);
        for (int64_t i = threadIdx.x; i < nq; i += blockDim.x) {
            store_from_float(p.d_q, p.dtype, t * nq + i, 0.f);
            store_from_float(p.d_k, p.dtype, t * nq + i, 0.f);
        }
        for (int64_t i = threadIdx.x; i < nv; i += blockDim.x) store_from_float(p.d_v, p.dtype, t * nv + i, 0.f);
        for (int64_t i = threadIdx.x; i < p.H; i += blockDim.x) {
            store_from_float(p.d_g, p.g_dtype, t * p.H + i, 0.f);
            store_from_float(p.d_b, p.b_dtype, t * p.H + i, 0.f);
        }
    }
}

template <int KP, bool GROUPED>
static int launch_grads(const DeltaParams &p, cudaStream_t st) {
    const int smem = GradLayout<KP>::BYTES;
    if (cudaFuncSetAttribute(delta_grads_kernel<KP, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return ASCAN_ERR_LAUNCH;
    delta_grads_kernel<KP, GROUPED><<<dim3(p.slots, p.Hk), 256, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

int delta_launch_zero_outside(const DeltaParams &p, cudaStream_t st) {
    if (!p.packed) return ASCAN_OK;
    delta_zero_outside_kernel<<<64, 256, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

int delta_launch_grads(const DeltaParams &p, cudaStream_t st) {
    if (p.slots == 0) return ASCAN_OK;
    if (p.Kp <= 64) return p.H == p.Hk ? launch_grads<64, false>(p, st) : launch_grads<64, true>(p, st);
    return p.H == p.Hk ? launch_grads<128, false>(p, st) : launch_grads<128, true>(p, st);
}

}  // namespace ascan
