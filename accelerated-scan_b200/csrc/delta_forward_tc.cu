// Gated delta rule, forward sweep on tcgen05: bf16 inputs, one CTA a sequence, head and 128 columns of V.
//
// The state is held transposed: rows of tensor memory and threads are columns of V, so that all products of a chunk
//     x = V^T - gam (S^T K^T);   e = x - x (M beta)^T;   dS^T = (Gam_C u) K;   out = scale gam (S^T Q^T) + u P^T
// have 128 rows, and their left operands come from tensor memory, where the threads that computed them (256: two for each
// row, half of the columns each) put them as bf16 terms.  The fp32 state itself stays in those threads' registers.  Terms
// are chosen as in the warp-level sweep: two for whatever reaches the state; for out alone S and P are one, u is two (of the
// three, S matters least: out was 2.9e-3 off with one term each, 2.4e-3 so, 1.7e-3 of it its own rounding).
//
// Two more groups of four warps prepare M and P, each of every other chunk, up to two chunks ahead; one warp loads the
// tiles (three stages), one runs the gates' sums and one issues.  Products that the state does not wait for (Q, P, the next
// chunk's K K^T) are issued behind those that it does, so that they run while the 256 threads convert.
//
// What bounds it is the chain of a chunk, about 8000 clocks: five products, each followed by a conversion of the result into
// the next one's operand (6500 clocks of the 256 threads' work and waits), and beside it the preparation of M, 11000 to
// 13000 clocks a chunk over two groups.  Sequences times heads give the parallelism, so memory waits: 4 x 16384 tokens, 32
// heads of 128 x 128 take 1075 us (1.6 GB, 1.5 TB/s; the same on warp matrix instructions 3344 us), nine packed prompts of
// 8192 tokens in all 165 to 300 us (the longest has 1830 to 4000, and its turn comes first or later), 4 x 4096 tokens of 16
// heads 267 us, with what the backward needs 383 us.
#include "delta_tc_roles.cuh"

namespace ascan {

struct TcForward {           // columns of tensor memory
    static constexpr int S = 0, X = 128, BX = 192, D2 = 256, O1 = 320, O2 = 384;
};
enum : int { B_X = B_OWN, B_D2, B_S, B_O, B_AS, B_BX, B_U, B_UO, B_OREAD };

template <int KP, bool SAVE>
__global__ void __launch_bounds__(TC_THREADS, 1) delta_sweep_tc_kernel(const __grid_constant__ DeltaParams p,
                                                                       const __grid_constant__ TcMaps maps) {
    extern __shared__ unsigned char smem_raw[];
    typedef TcLayout<KP, false> L;
    typedef TcForward F;
    constexpr int HK = KP / 2;                         // columns of the state a thread holds
    const TcBlock k = tc_begin<L>(p, smem_raw, blockIdx.x, 4, 5);
    const Sequence &sq = k.sq;
    unsigned char *smem = k.smem;
    const uint32_t base = k.base, tmem = k.tmem;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = k.h, v0 = k.v0, n_seq = k.n_seq;
    const int64_t state_at = (int64_t(n_seq) * p.H + h) * p.K * p.V;

    if (warp < 8) {
        // ---- the state: thread (row v, half of K; half of the tokens)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        const int v = (warp & 3) * 32 + lane, part = warp >> 2;
        const bool real = v0 + v < p.V;
        const uint32_t t0 = tmem + (uint32_t((warp & 3) * 32) << 16);
        f2 s[HK / 2];
#pragma unroll
        for (int i = 0; i < HK / 2; ++i) {
            const int col = part * HK + 2 * i;
            const float *at = p.s0 + state_at + int64_t(col) * p.V + v0 + v;
            s[i] = two(p.s0 && real && col < p.K ? at[0] : 0.f, p.s0 && real && col + 1 < p.K ? at[p.V] : 0.f);
        }
        // where a chunk's state starts for the backward
        const auto kept = [&](int c) {
            return SAVE && v0 + v < p.Vp ? p.S + (int64_t(sq.slot0 + c) * p.H + h) * p.Vp * KP + (v0 + v) * KP + part * HK : nullptr;
        };
        if (sq.chunks > 0) {
            put_state<HK>(s, t0 + F::S + part * HK, kept(0));
            hand_over(k, B_AS);
        }
        for (int c = 0; c < sq.chunks; ++c) {
            const int stage = c % 3;
            const float *sc = reinterpret_cast<const GateShared *>(smem + L::SC)[stage].sc + part * 32;
            const auto scalars = [&](int which, int i) { return *reinterpret_cast<const ulonglong2 *>(sc + which * 64 + i); };
            unsigned char *vt = smem + stage * L::STAGE + L::KQ_BYTES + part * 32 * 256 + v * 2;
            k.wait.warp(k.bar(B_TILE + stage), (c / 3) & 1);
            k.wait.warp(k.bar(B_GATES + stage), (c / 3) & 1);
            k.wait.warp(k.bar(B_PREP + (c & 1)), (c >> 1) & 1);
            f2 x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x[i] = two_bits(uint32_t(*reinterpret_cast<const uint16_t *>(vt + 2 * i * 256)) << 16,
                                uint32_t(*reinterpret_cast<const uint16_t *>(vt + (2 * i + 1) * 256)) << 16);
            k.wait.warp(k.bar(B_X), c & 1);
            tc_fence_after();
            uint32_t r[32];
            tmem_ld32(r, t0 + F::X + 32 * part);
            tc_wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int i = 8 * q + j;
                    const ulonglong2 ga = scalars(SC_GAM, 2 * i);
                    x[i] = fma2(ga.x, two_bits(r[2 * i], r[2 * i + 1]), x[i]);
                    x[i + 1] = fma2(ga.y, two_bits(r[2 * i + 2], r[2 * i + 3]), x[i + 1]);
                    split_f2(x[i], hi[j], lo[j]);
                    split_f2(x[i + 1], hi[j + 1], lo[j + 1]);
                }
                tmem_st8(t0 + F::BX + 16 * part + 8 * q, hi);
                tmem_st8(t0 + F::BX + 32 + 16 * part + 8 * q, lo);
            }
            hand_over(k, B_BX);
            k.wait.warp(k.bar(B_D2), c & 1);
            tc_fence_after();
            tmem_ld32(r, t0 + F::D2 + 32 * part);
            tc_wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int i = 8 * q + j;
                    const ulonglong2 gb = scalars(SC_GAMC_BETA, 2 * i);
                    x[i] = add2(x[i], two_bits(r[2 * i], r[2 * i + 1]));
                    x[i + 1] = add2(x[i + 1], two_bits(r[2 * i + 2], r[2 * i + 3]));
                    split_f2(mul2(gb.x, x[i]), hi[j], lo[j]);
                    split_f2(mul2(gb.y, x[i + 1]), hi[j + 1], lo[j + 1]);
                }
                tmem_st8(t0 + F::X + 16 * part + 8 * q, hi);
                tmem_st8(t0 + F::X + 32 + 16 * part + 8 * q, lo);
            }
            hand_over(k, B_U);
            // u for out, while the state's product runs
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const ulonglong2 be = scalars(SC_BETA, 16 * q + 2 * j);
                    split_f2(mul2(be.x, x[8 * q + j]), hi[j], lo[j]);
                    split_f2(mul2(be.y, x[8 * q + j + 1]), hi[j + 1], lo[j + 1]);
                }
                tmem_st8(t0 + F::BX + 16 * part + 8 * q, hi);
                tmem_st8(t0 + F::BX + 32 + 16 * part + 8 * q, lo);
            }
            hand_over(k, B_UO);
            const float gam_c = sc[SC_GAM * 64 + 63 - part * 32];
            const f2 gam_c2 = two(gam_c, gam_c);
            k.wait.warp(k.bar(B_S), c & 1);
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < HK / 32; ++q) {
                tmem_ld32(r, t0 + F::S + part * HK + 32 * q);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) s[16 * q + i] = fma2(gam_c2, s[16 * q + i], two_bits(r[2 * i], r[2 * i + 1]));
            }
            if (c + 1 < sq.chunks) {
                put_state<HK>(s, t0 + F::S + part * HK, kept(c + 1));
                hand_over(k, B_AS);
            }
            if (SAVE && v0 + v < p.Vp)
                keep_tokens(x, p.e + ((int64_t(sq.slot0 + c) * p.H + h) * 2 * p.Vp + v0 + v) * 64 + 32 * part, int64_t(p.Vp) * 64);
            k.wait.warp(k.bar(B_O), c & 1);
            tc_fence_after();
            uint32_t r2[32];
            tmem_ld32(r, t0 + F::O1 + 32 * part);
            tmem_ld32(r2, t0 + F::O2 + 32 * part);
            tc_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(k.bar(B_OREAD));
#pragma unroll
            for (int i = 0; i < 16; i += 2) {         // out takes the place of V in shared memory
                const ulonglong2 ga = scalars(SC_OUT, 2 * i);
                const uint32_t a = pack_f2(fma2(ga.x, two_bits(r[2 * i], r[2 * i + 1]), two_bits(r2[2 * i], r2[2 * i + 1])));
                const uint32_t b = pack_f2(fma2(ga.y, two_bits(r[2 * i + 2], r[2 * i + 3]), two_bits(r2[2 * i + 2], r2[2 * i + 3])));
                *reinterpret_cast<uint16_t *>(vt + 2 * i * 256) = static_cast<uint16_t>(a);
                *reinterpret_cast<uint16_t *>(vt + (2 * i + 1) * 256) = static_cast<uint16_t>(a >> 16);
                *reinterpret_cast<uint16_t *>(vt + (2 * i + 2) * 256) = static_cast<uint16_t>(b);
                *reinterpret_cast<uint16_t *>(vt + (2 * i + 3) * 256) = static_cast<uint16_t>(b >> 16);
            }
            const int64_t left = sq.len - int64_t(c) * 64;
            // One copy takes the tile to memory; it leaves out rows behind the array, but not those of a next sequence.
            const bool by_copy = maps.store && (left >= 64 || sq.t0 + sq.len == p.T);
            fence_async_proxy();                  // before this copy reads the tile, or the next chunk's copies write over it
            group_sync<1, 256>();
            if (by_copy) {
                if (tid == 0) {
                    tma_store(&maps.out, base + stage * L::STAGE + L::KQ_BYTES, v0, h, static_cast<int>(sq.t0 + int64_t(c) * 64),
                              static_cast<int>(sq.b));
                    tma_store_read();
                }
            } else {
                const int64_t row0 = sq.b * p.T + sq.t0 + int64_t(c) * 64;
                const unsigned char *ot = smem + stage * L::STAGE + L::KQ_BYTES;
#pragma unroll 1
                for (int i = tid; i < 64 * 128; i += 256) {
                    const int t = i >> 7, col = v0 + (i & 127);
                    if (t < left && col < p.V)
                        static_cast<bf16 *>(p.out)[((row0 + t) * p.H + h) * p.V + col] =
                            *reinterpret_cast<const bf16 *>(ot + t * 256 + (i & 127) * 2);
                }
                give_back_reads();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(k.bar(B_FREE + stage));
        }
        if (tid == 0) tma_store_done();
#pragma unroll
        for (int i = 0; i < HK / 2; ++i) {
            const int col = part * HK + 2 * i;
            const float2 x = apart(s[i]);
            float *to = p.s1 + state_at + int64_t(col) * p.V + v0 + v;
            if (real && col < p.K) to[0] = x.x;
            if (real && col + 1 < p.K) to[p.V] = x.y;
        }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        prepare_chunks<L, false>(p, k);
    } else if (warp == 16) {
        // ---- issue
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (elect_one()) {
            const auto kq = [](int step, int row) { return ((step >> 2) * 16384 + (step & 3) * 32 + row * 128) >> 4; };
            TileRing<L> ring;
            ring.begin(k);
#pragma unroll 1
            for (int c = 0; c < sq.chunks; ++c) {
                const int stage = ring.stage;
                const uint32_t tile = base + stage * L::STAGE, rows = tile_low(tile), down = tile_low(tile, 16384);
                k.wait(k.bar(B_AS), c & 1);
                tc_fence_after();
#pragma unroll
                for (int lo = 0; lo < 2; ++lo)
#pragma unroll
                    for (int s = 0; s < KP / 16; ++s)
                        tc_mma_ts(tmem + F::X, state_term<HK>(tmem + F::S, s, lo), rows + kq(s, 0), mma_desc(64, false, true), lo + s > 0);      // -K S
                tc_commit(k.bar(B_X));
                if (c > 0) k.wait(k.bar(B_OREAD), (c - 1) & 1);
                tc_fence_after();
#pragma unroll
                for (int s = 0; s < KP / 16; ++s)
                    tc_mma_ts(tmem + F::O1, state_term<HK>(tmem + F::S, s, 0), rows + kq(s, 64), mma_desc(64, false), s > 0);
                const uint32_t m = tile_low(base + L::M + (c & 1) * M_BYTES), pt = tile_low(base + L::P + stage * L::P_BYTES);
                k.wait(k.bar(B_PREP + (c & 1)), (c >> 1) & 1);
                k.wait(k.bar(B_BX), c & 1);
                tc_fence_after();
                // tokens 16 t .. of x reach the tokens from 16 t on only
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t desc = mma_desc(64 - 16 * t, false, true), d = tmem + F::D2 + 16 * t, at = (16 * t * 128 + 32 * t) >> 4;
                    tc_mma_ts(d, tmem + F::BX + 8 * t, m + at, desc, t > 0);
                    tc_mma_ts(d, tmem + F::BX + 32 + 8 * t, m + at, desc, true);
                    tc_mma_ts(d, tmem + F::BX + 8 * t, m + (8192 >> 4) + at, desc, true);
                }
                tc_commit(k.bar(B_D2));
                ring.m_read(k, c);
                k.wait(k.bar(B_U), c & 1);
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo)
                        tc_mma_ts(tmem + F::S, tmem + F::X + 32 * lo + 8 * t, down + kq(0, 16 * t), mma_desc(KP, true), t + lo > 0);
                tc_commit(k.bar(B_S));
                k.wait(k.bar(B_UO), c & 1);
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo)
                        tc_mma_ts(tmem + F::O2 + 16 * t, tmem + F::BX + 32 * lo + 8 * t, pt + ((16 * t * 128 + 32 * t) >> 4),
                                  mma_desc(64 - 16 * t, false), t + lo > 0);
                tc_commit(k.bar(B_O));
                ring.next(k);
            }
        }
    } else if (warp == 17) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        load_tiles<L, false, false>(p, k, maps);
    } else if (warp == 18) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        run_gates<L, false, SAVE>(p, k);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    }
    if (p.packed && (n_seq == 0 || n_seq == p.n_seqs - 1)) {      // tokens of no sequence: zeros
        const int64_t front = n_seq == 0 ? sq.t0 : 0, back = n_seq == p.n_seqs - 1 ? sq.t0 + sq.len : p.T;
        const int64_t rows = front + (p.T - back);
        for (int64_t i = tid; i < rows * 128; i += TC_THREADS) {
            const int64_t r = i / 128;
            const int v = v0 + static_cast<int>(i % 128);
            if (v < p.V) static_cast<bf16 *>(p.out)[((r < front ? r : back + (r - front)) * p.H + h) * p.V + v] = __float2bfloat16_rn(0.f);
        }
    }
    tc_end(k);
}

template <int KP, bool SAVE>
static int launch_sweep_tc(const DeltaParams &p, const TcMaps &maps, cudaStream_t st) {
    const int64_t grid = int64_t(p.n_seqs) * p.H * ((p.Vp + 127) / 128);
    const int smem = TcLayout<KP, false>::BYTES;
    if (grid > 0x7fffffff) return ASCAN_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(delta_sweep_tc_kernel<KP, SAVE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return ASCAN_ERR_LAUNCH;
    delta_sweep_tc_kernel<KP, SAVE><<<unsigned(grid), TC_THREADS, smem, st>>>(p, maps);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

int delta_launch_sweep_tc(const DeltaParams &p, bool save, cudaStream_t st) {
    TcMaps maps;
    int rc;
    if ((rc = make_map(&maps.k, p.k, p, p.Kp, p.Hk, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_map(&maps.q, p.q, p, p.Kp, p.Hk, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_map(&maps.v, p.v, p, p.Vp, p.H, 128, false)) != ASCAN_OK) return rc;
    if ((rc = make_store_map(&maps, p.out, p, false)) != ASCAN_OK) return rc;
    if (p.Kp <= 64) return save ? launch_sweep_tc<64, true>(p, maps, st) : launch_sweep_tc<64, false>(p, maps, st);
    return save ? launch_sweep_tc<128, true>(p, maps, st) : launch_sweep_tc<128, false>(p, maps, st);
}

}  // namespace ascan
