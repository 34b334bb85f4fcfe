// Gated delta rule, backward sweep on tcgen05, from the last chunk to the first: as the forward one, on the transposed gradient
// of the state.  Per chunk
//     du = Gam_C (dS^T K^T) + d_out^T P;   z = du - du (beta M);   y = beta z = dV
//     dS^T = gam_C dS^T + (scale gam d_out)^T Q - (gam y)^T K
// d_out^T P takes d_out from shared memory as it is (rows of the product lie along the tile's rows); it and
// (scale gam d_out)^T Q do not wait for the state and run while the threads convert.  dS1 and z go to memory for the gradients
// of the chunk, which other CTAs of the same launch compute meanwhile.  M and P are prepared again: reading them back would be 32 KB a chunk and head, and the groups that prepare
// would idle.  Bound as the forward sweep is; 4 x 4096 tokens, 16 heads of 128 x 128: 413 us by itself,
// and 480 with the gradients beside it, whose 266 us by themselves would else come behind.
#include "delta_grads_tc.cuh"

namespace ascan {

struct TcBackward {          // columns of tensor memory; A1 lies in D2's place, A2 in D1's
    static constexpr int S = 0, D1 = 128, D2 = 192, DU = 256, D3 = 320;
};
enum : int { B_D1 = B_OWN, B_D2, B_D3, B_S, B_AS, B_DU, B_A1, B_YZ };

template <int KP>
__device__ __forceinline__ void back_sweep(const DeltaParams &p, const TcMaps &maps, unsigned char *smem_raw, int block) {
    typedef TcLayout<KP, true> L;
    typedef TcBackward F;
    constexpr int HK = KP / 2;                         // columns of the state a thread holds
    const TcBlock k = tc_begin<L>(p, smem_raw, block, 4, 4);
    const Sequence &sq = k.sq;
    unsigned char *smem = k.smem;
    const uint32_t base = k.base, tmem = k.tmem;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = k.h, v0 = k.v0;
    const int64_t state_at = (int64_t(k.n_seq) * p.H + h) * p.K * p.V;

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
            const float *at = p.d_s1 + state_at + int64_t(col) * p.V + v0 + v;
            s[i] = two(p.d_s1 && real && col < p.K ? at[0] : 0.f, p.d_s1 && real && col + 1 < p.K ? at[p.V] : 0.f);
        }
        const auto kept = [&](int c) {
            return v0 + v < p.Vp ? p.dS + (int64_t(sq.slot0 + c) * p.H + h) * p.Vp * KP + (v0 + v) * KP + part * HK : nullptr;
        };
        if (sq.chunks > 0) {
            put_state<HK>(s, t0 + F::S + part * HK, kept(sq.chunks - 1));
            hand_over(k, B_AS);
        }
#pragma unroll 1
        for (int turn = 0; turn < sq.chunks; ++turn) {
            const int stage = turn % 3, c = sq.chunks - 1 - turn;
            const float *sc = reinterpret_cast<const GateShared *>(smem + L::SC)[stage].sc + part * 32;
            const auto scalars = [&](int which, int i) { return *reinterpret_cast<const ulonglong2 *>(sc + which * 64 + i); };
            // this thread's column of the tile of d_out, and later of dV: row t, piece (v % 64) / 8 of a swizzled block
            unsigned char *col = smem + stage * L::STAGE + L::KQ_BYTES + (v >> 6) * 8192 + part * 32 * 128 + (v & 7) * 2;
            const auto element = [&](int t) { return reinterpret_cast<uint16_t *>(col + t * 128 + (((v >> 3 & 7) ^ (t & 7)) << 4)); };
            k.wait.warp(k.bar(B_TILE + stage), (turn / 3) & 1);
            k.wait.warp(k.bar(B_GATES + stage), (turn / 3) & 1);
            k.wait.warp(k.bar(B_D2), turn & 1);
            k.wait.warp(k.bar(B_D1), turn & 1);
            tc_fence_after();
            f2 x[16];
            {
                uint32_t r[32];
                tmem_ld32(r, t0 + F::D2 + 32 * part);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = two_bits(r[2 * i], r[2 * i + 1]);
            }
            uint32_t r[32];
            tmem_ld32(r, t0 + F::D1 + 32 * part);
            tc_wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int i = 8 * q + j;
                    const ulonglong2 gc = scalars(SC_GAMC, 2 * i);
                    x[i] = fma2(gc.x, two_bits(r[2 * i], r[2 * i + 1]), x[i]);
                    x[i + 1] = fma2(gc.y, two_bits(r[2 * i + 2], r[2 * i + 3]), x[i + 1]);
                    split_f2(x[i], hi[j], lo[j]);
                    split_f2(x[i + 1], hi[j + 1], lo[j + 1]);
                }
                tmem_st8(t0 + F::DU + 16 * part + 8 * q, hi);
                tmem_st8(t0 + F::DU + 32 + 16 * part + 8 * q, lo);
            }
            hand_over(k, B_DU);
            // A1 = scale gam d_out, into the columns of D2 that this warp itself has read
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int t = 16 * q + 2 * j;
                    const ulonglong2 ga = scalars(SC_OUT, t);
                    split_f2(mul2(ga.x, two_bits(uint32_t(*element(t)) << 16, uint32_t(*element(t + 1)) << 16)), hi[j], lo[j]);
                    split_f2(mul2(ga.y, two_bits(uint32_t(*element(t + 2)) << 16, uint32_t(*element(t + 3)) << 16)), hi[j + 1], lo[j + 1]);
                }
                tmem_st8(t0 + F::D2 + 32 * part + 8 * q, hi);
                tmem_st8(t0 + F::D2 + 32 * part + 16 + 8 * q, lo);
            }
            hand_over(k, B_A1);
            k.wait.warp(k.bar(B_D3), turn & 1);
            tc_fence_after();
            tmem_ld32(r, t0 + F::D3 + 32 * part);
            tc_wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int i = 8 * q + j;
                    const ulonglong2 be = scalars(SC_BETA, 2 * i), ga = scalars(SC_GAM, 2 * i);
                    x[i] = add2(x[i], two_bits(r[2 * i], r[2 * i + 1]));
                    x[i + 1] = add2(x[i + 1], two_bits(r[2 * i + 2], r[2 * i + 3]));
                    split_f2(mul2(ga.x, mul2(be.x, x[i])), hi[j], lo[j]);
                    split_f2(mul2(ga.y, mul2(be.y, x[i + 1])), hi[j + 1], lo[j + 1]);
                }
                tmem_st8(t0 + F::D1 + 16 * part + 8 * q, hi);
                tmem_st8(t0 + F::D1 + 32 + 16 * part + 8 * q, lo);
            }
            hand_over(k, B_YZ);
            if (v0 + v < p.Vp)
                keep_tokens(x, p.z + ((int64_t(sq.slot0 + c) * p.H + h) * 2 * p.Vp + v0 + v) * 64 + 32 * part, int64_t(p.Vp) * 64);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {        // dV in the place of d_out, which nobody needs any more
                const ulonglong2 be = scalars(SC_BETA, 2 * i);
                const uint32_t y = pack_f2(mul2(be.x, x[i])), w = pack_f2(mul2(be.y, x[i + 1]));
                *element(2 * i) = static_cast<uint16_t>(y);
                *element(2 * i + 1) = static_cast<uint16_t>(y >> 16);
                *element(2 * i + 2) = static_cast<uint16_t>(w);
                *element(2 * i + 3) = static_cast<uint16_t>(w >> 16);
            }
            const int64_t left = sq.len - int64_t(c) * 64;
            const bool by_copy = maps.store && (left >= 64 || sq.t0 + sq.len == p.T);        // as in the forward sweep
            fence_async_proxy();
            group_sync<1, 256>();
            const uint32_t tile = base + stage * L::STAGE + L::KQ_BYTES;
            if (by_copy) {
                if (tid == 0) {
                    const int tok = static_cast<int>(sq.t0 + int64_t(c) * 64);
                    tma_store(&maps.out, tile, v0, h, tok, static_cast<int>(sq.b));
                    if (v0 + 64 < p.V) tma_store(&maps.out, tile + 8192, v0 + 64, h, tok, static_cast<int>(sq.b));
                }
            } else {
                const int64_t row0 = sq.b * p.T + sq.t0 + int64_t(c) * 64;
                const unsigned char *tp = smem + stage * L::STAGE + L::KQ_BYTES;
#pragma unroll 1
                for (int i = tid; i < 64 * 128; i += 256) {
                    const int t = i >> 7, u = i & 127;
                    if (t < left && v0 + u < p.V)
                        static_cast<bf16 *>(p.d_v)[((row0 + t) * p.H + h) * p.V + v0 + u] = *reinterpret_cast<const bf16 *>(
                            tp + (u >> 6) * 8192 + t * 128 + (((u >> 3 & 7) ^ (t & 7)) << 4) + (u & 7) * 2);
                }
                give_back_reads();
            }
            const float gam_c = sc[SC_GAM * 64 + 63 - part * 32];
            const f2 gam_c2 = two(gam_c, gam_c);
            k.wait.warp(k.bar(B_S), turn & 1);
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < HK / 32; ++q) {
                tmem_ld32(r, t0 + F::S + part * HK + 32 * q);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) s[16 * q + i] = fma2(gam_c2, s[16 * q + i], two_bits(r[2 * i], r[2 * i + 1]));
            }
            if (c > 0) {
                put_state<HK>(s, t0 + F::S + part * HK, kept(c - 1));
                hand_over(k, B_AS);
            }
            if (tid == 0) tma_store_read();
            __syncwarp();
            if (lane == 0) mbar_arrive(k.bar(B_FREE + stage));
        }
        if (tid == 0) tma_store_done();
        if (p.d_s0) {
#pragma unroll
            for (int i = 0; i < HK / 2; ++i) {
                const int col = part * HK + 2 * i;
                const float2 x = apart(s[i]);
                float *to = p.d_s0 + state_at + int64_t(col) * p.V + v0 + v;
                if (real && col < p.K) to[0] = x.x;
                if (real && col + 1 < p.K) to[p.V] = x.y;
            }
        }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        prepare_chunks<L, true>(p, k);
    } else if (warp == 16) {
        // ---- issue
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (elect_one()) {
            const auto kq = [](int step, int row) { return ((step >> 2) * 16384 + (step & 3) * 32 + row * 128) >> 4; };
            TileRing<L> ring;
            ring.begin(k);
#pragma unroll 1
            for (int turn = 0; turn < sq.chunks; ++turn) {
                const uint32_t tile = base + ring.stage * L::STAGE, rows = tile_low(tile), down = tile_low(tile, 16384);
                const uint32_t m = tile_low(base + L::M + (turn & 1) * M_BYTES), pt = tile_low(base + L::P + (turn & 1) * L::P_BYTES);
                const uint32_t d_out = tile_low(tile + L::KQ_BYTES, 8192);
                // tokens 16 t .. 16 t + 15 reach the tokens up to 16 t + 15 only; the last ones come first and write all
                k.wait(k.bar(B_PREP + (turn & 1)), (turn >> 1) & 1);
                if (turn > 0) k.wait(k.bar(B_S), (turn - 1) & 1);          // A1's reader has ended
                tc_fence_after();
#pragma unroll
                for (int t = 3; t >= 0; --t)
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo)
                        tc_mma_ss(tmem + F::D2, d_out + ((2048 * t) >> 4), pt + ((8192 * lo + 2048 * t) >> 4),
                                  mma_desc(16 * (t + 1), true, false, true), t < 3 || lo > 0);
                tc_commit(k.bar(B_D2));
                k.wait(k.bar(B_AS), turn & 1);
                tc_fence_after();
#pragma unroll
                for (int lo = 0; lo < 2; ++lo)
#pragma unroll
                    for (int s = 0; s < KP / 16; ++s)
                        tc_mma_ts(tmem + F::D1, state_term<HK>(tmem + F::S, s, lo), rows + kq(s, 0), mma_desc(64, false), lo + s > 0);
                tc_commit(k.bar(B_D1));
                k.wait(k.bar(B_DU), turn & 1);
                tc_fence_after();
#pragma unroll
                for (int t = 3; t >= 0; --t) {
                    const uint32_t desc = mma_desc(16 * (t + 1), true, true), at = (2048 * t) >> 4;
                    tc_mma_ts(tmem + F::D3, tmem + F::DU + 8 * t, m + at, desc, t < 3);
                    tc_mma_ts(tmem + F::D3, tmem + F::DU + 32 + 8 * t, m + at, desc, true);
                    tc_mma_ts(tmem + F::D3, tmem + F::DU + 8 * t, m + (8192 >> 4) + at, desc, true);
                }
                tc_commit(k.bar(B_D3));
                ring.m_read(k, turn);
                k.wait(k.bar(B_A1), turn & 1);
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo)
                        tc_mma_ts(tmem + F::S, tmem + F::D2 + 32 * (t >> 1) + 8 * (t & 1) + 16 * lo, down + kq(0, 64 + 16 * t), mma_desc(KP, true),
                                  t + lo > 0);
                k.wait(k.bar(B_YZ), turn & 1);
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo)
                        tc_mma_ts(tmem + F::S, tmem + F::D1 + 32 * lo + 8 * t, down + kq(0, 16 * t), mma_desc(KP, true, true), true);
                tc_commit(k.bar(B_S));
                ring.next(k);
            }
        }
    } else if (warp == 17) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        load_tiles<L, true, true>(p, k, maps);
    } else if (warp == 18) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        run_gates<L, true, false>(p, k);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    }
    tc_end(k);
}

// The sweep and the gradients of the chunks that it has finished, in one launch: the first `sweeps` CTAs to start sweep, so a
// CTA that waits for a sweep waits for one that runs.  One sweep needs one SM a head and sequence, and leaves the others idle.
template <int KP, bool GROUPED>
__global__ void __launch_bounds__(TC_THREADS, 1) delta_backward_tc_kernel(const __grid_constant__ DeltaParams p, const __grid_constant__ TcMaps maps,
                                                                          const __grid_constant__ GradMaps grad_maps, int sweeps) {
    extern __shared__ unsigned char smem_raw[];
    volatile int *ticket = reinterpret_cast<volatile int *>(smem_raw);
    if (threadIdx.x == 0) *ticket = atomicAdd(p.done, 1);
    __syncthreads();
    const int role = *ticket;
    __syncthreads();
    if (role < sweeps) back_sweep<KP>(p, maps, smem_raw, role);
    else chunk_gradients<GROUPED>(p, grad_maps, smem_raw);
}

template <int KP, bool GROUPED>
static int launch_backward_tc(const DeltaParams &p, const TcMaps &maps, const GradMaps &grad_maps, int sm_count, cudaStream_t st) {
    const int64_t sweeps = int64_t(p.n_seqs) * p.H * ((p.Vp + 127) / 128), items = int64_t(p.slots) * p.Hk;
    const int64_t others = items < sm_count ? items : sm_count;
    if (sweeps + others > 0x7fffffff) return ASCAN_ERR_UNSUPPORTED;
    const int smem = TcLayout<KP, true>::BYTES > TcGrads::BYTES ? TcLayout<KP, true>::BYTES : TcGrads::BYTES;
    const auto kernel = delta_backward_tc_kernel<KP, GROUPED>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return ASCAN_ERR_LAUNCH;
    if (cudaMemsetAsync(p.done, 0, (2 + size_t(p.slots) * p.H) * sizeof(int), st) != cudaSuccess) return ASCAN_ERR_LAUNCH;
    kernel<<<unsigned(sweeps + others), TC_THREADS, smem, st>>>(p, maps, grad_maps, static_cast<int>(sweeps));
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

int delta_launch_backward_tc(const DeltaParams &p, int sm_count, cudaStream_t st) {
    TcMaps maps;
    GradMaps grad_maps;
    int rc;
    if ((rc = make_map(&maps.k, p.k, p, p.Kp, p.Hk, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_map(&maps.q, p.q, p, p.Kp, p.Hk, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_map(&maps.v, p.d_out, p, p.Vp, p.H, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_store_map(&maps, p.d_v, p, true)) != ASCAN_OK) return rc;
    if ((rc = make_grad_maps(&grad_maps, p)) != ASCAN_OK) return rc;
    const bool grouped = p.H != p.Hk;
    if (p.Kp <= 64) return grouped ? launch_backward_tc<64, true>(p, maps, grad_maps, sm_count, st) : launch_backward_tc<64, false>(p, maps, grad_maps, sm_count, st);
    return grouped ? launch_backward_tc<128, true>(p, maps, grad_maps, sm_count, st) : launch_backward_tc<128, false>(p, maps, grad_maps, sm_count, st);
}

}  // namespace ascan
