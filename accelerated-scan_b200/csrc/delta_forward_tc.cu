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
// tiles (three stages), one runs the gates' sums and one issues.  Products that the
// state does not wait for (Q, P, the next chunk's K K^T) are issued behind those that it does, so that they run while the
// 256 threads convert.
#include <cuda.h>

#include "delta_tc.cuh"

namespace ascan {

struct TcMaps {
    CUtensorMap k, q, v, out;
    bool store;                // out can be written by copies: rows start on 16 bytes
};

// (column, head, token, batch) of planes; a box is `cols` columns of 64 tokens.  What lies outside of the array reads as zero.
static int make_map(CUtensorMap *map, const Planes &x, const DeltaParams &p, int d, int heads, int cols, bool swizzled) {
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                               const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (!encode) return ASCAN_ERR_DEVICE;
    *map = CUtensorMap{};
    if (p.T == 0) return ASCAN_OK;                      // nothing will be loaded
    // a dimension of one element has any stride: take the dense one
    const cuuint64_t dims[4] = {cuuint64_t(d), cuuint64_t(heads), cuuint64_t(p.T), cuuint64_t(p.batch)};
    const cuuint64_t strides[3] = {cuuint64_t(heads > 1 ? x.sh : d) * 2, cuuint64_t(p.T > 1 ? x.st : int64_t(heads) * d) * 2,
                                   cuuint64_t(p.batch > 1 ? x.sb : p.T * heads * d) * 2};
    const cuuint32_t box[4] = {cuuint32_t(cols), 1, 64, 1}, unit[4] = {1, 1, 1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16 *>(x.p), dims, strides, box, unit,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

// The next chunk's log gates and rates, two tokens a lane, held as they are until they are needed: a conversion would wait
// for them.
struct GateLoader {
    uint32_t g[2], b[2];
    static __device__ __forceinline__ uint32_t raw(const void *p, int dtype, int64_t i) {
        return dtype == ASCAN_F32 ? static_cast<const uint32_t *>(p)[i] : static_cast<const uint16_t *>(p)[i];
    }
    static __device__ __forceinline__ float value(uint32_t x, int dtype) {
        if (dtype == ASCAN_F32) return __uint_as_float(x);
        return dtype == ASCAN_BF16 ? __uint_as_float(x << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(x)));
    }
    __device__ __forceinline__ void load(const DeltaParams &p, const Sequence &sq, int c, int h, int lane) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t i = int64_t(c) * 64 + 2 * lane + j, tok = sq.t0 + i;
            g[j] = b[j] = 0;
            if (i < sq.len) {
                g[j] = raw(p.g, p.g_dtype, sq.b * p.g_s[0] + tok * p.g_s[1] + h * p.g_s[2]);
                b[j] = raw(p.b, p.b_dtype, sq.b * p.b_s[0] + tok * p.b_s[1] + h * p.b_s[2]);
            }
        }
    }
    __device__ __forceinline__ void get(const DeltaParams &p, float (&gv)[2], float (&bv)[2]) const {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            gv[j] = value(g[j], p.g_dtype);
            bv[j] = value(b[j], p.b_dtype);
        }
    }
};

template <int KP>
struct TcForward {
    static constexpr int HALVES = KP / 64, KQ_BYTES = HALVES * 16384, V_BYTES = 64 * 256, STAGE = KQ_BYTES + V_BYTES;
    static constexpr int MP = 3 * STAGE, P = M_BYTES, MP_BYTES = M_BYTES + 8192;       // M (hi, lo), P
    static constexpr int SC = MP + 2 * MP_BYTES, PREP = SC + 3 * sizeof(GateShared);
    static constexpr int BARS = PREP + 2 * 4 * 128 * 4, BYTES = BARS + 256 + 1024;      // and 1024 to align the start
    // columns of tensor memory
    static constexpr int S = 0, X = 128, BX = 192, D2 = 256, O1 = 320, O2 = 384, KK = 448;
};
enum : int { B_TILE = 0, B_PREP = 3, B_GATES = 5, B_KK = 8, B_MP = 10, B_X = 12, B_D2, B_S, B_O, B_AS, B_BX, B_U, B_UO, B_OREAD, B_KREAD, B_FREE, B_TAIL = B_FREE + 3, B_COUNT };

constexpr int TC_THREADS = 20 * 32;
// Registers a thread: 96 at launch; 152 * 256 + 64 * 256 + 48 * 128 = 96 * 640


template <int KP, bool SAVE>
__global__ void __launch_bounds__(TC_THREADS, 1) delta_sweep_tc_kernel(const __grid_constant__ DeltaParams p,
                                                                       const __grid_constant__ TcMaps maps) {
    extern __shared__ unsigned char smem_raw[];
    typedef TcForward<KP> L;
    constexpr int HK = KP / 2;                         // columns of the state a thread holds
    unsigned char *smem = smem_raw + (-smem_addr(smem_raw) & 1023);
    const uint32_t base = smem_addr(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slices = (p.Vp + 127) / 128, slice = blockIdx.x % slices, h = (blockIdx.x / slices) % p.H, n_seq = blockIdx.x / slices / p.H;
    const int hk = h / (p.H / p.Hk), v0 = slice * 128;
    const Sequence sq = get_sequence(p, n_seq);
    const uint32_t bars = base + L::BARS;
    const auto bar = [&](int i) { return bars + 8 * i; };
    volatile int *dead = reinterpret_cast<volatile int *>(smem + L::BARS + 8 * B_COUNT);
    const uint32_t tmem_slot = bars + 8 * B_COUNT + 8;
    const Waiter wait = {dead, p.status};

    if (tid == 0) {
        *dead = 0;
        for (int i = 0; i < B_COUNT; ++i)
            mbar_init(bar(i), i < B_PREP ? 1 : i < B_GATES ? 128 : i < B_AS ? 1 : i < B_KREAD ? 8 : i < B_FREE ? 4 : i < B_TAIL ? 9 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_proxy();
    }
    if (warp == 16) tmem_alloc(tmem_slot, 512);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::BARS + 8 * B_COUNT + 8);
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
            const int k = part * HK + 2 * i;
            const float *at = p.s0 + state_at + int64_t(k) * p.V + v0 + v;
            s[i] = two(p.s0 && real && k < p.K ? at[0] : 0.f, p.s0 && real && k + 1 < p.K ? at[p.V] : 0.f);
        }
        const auto hand_over = [&](int b) {          // what this warp stored to tensor memory is there
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(b));
        };
        const auto put_state = [&](int c) {          // S as two terms to tensor memory, the first one to the backward's store
#pragma unroll
            for (int q = 0; q < HK / 16; ++q) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) split_f2(s[8 * q + i], hi[i], lo[i]);
                tmem_st8(t0 + L::S + part * HK + 8 * q, hi);
                tmem_st8(t0 + L::S + part * HK + HK / 2 + 8 * q, lo);
                if (SAVE && c < sq.chunks && v0 + v < p.Vp) {
                    uint4 *o = reinterpret_cast<uint4 *>(p.S + (int64_t(sq.slot0 + c) * p.H + h) * p.Vp * KP + (v0 + v) * KP +
                                                         part * HK + 16 * q);
                    o[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    o[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                }
            }
        };
        if (sq.chunks > 0) {
            put_state(0);
            hand_over(B_AS);
        }
        for (int c = 0; c < sq.chunks; ++c) {
            const int stage = c % 3;
            const float *sc = reinterpret_cast<const GateShared *>(smem + L::SC)[stage].sc + part * 32;
            const auto scalars = [&](int which, int i) { return *reinterpret_cast<const ulonglong2 *>(sc + which * 64 + i); };
            unsigned char *vt = smem + stage * L::STAGE + L::KQ_BYTES + part * 32 * 256 + v * 2;
            wait(bar(B_TILE + stage), (c / 3) & 1);
            wait(bar(B_GATES + stage), (c / 3) & 1);
            wait(bar(B_PREP + (c & 1)), (c >> 1) & 1);
            f2 x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x[i] = two_bits(uint32_t(*reinterpret_cast<const uint16_t *>(vt + 2 * i * 256)) << 16,
                                uint32_t(*reinterpret_cast<const uint16_t *>(vt + (2 * i + 1) * 256)) << 16);
            wait(bar(B_X), c & 1);
            tc_fence_after();
            uint32_t r[32];
            tmem_ld32(r, t0 + L::X + 32 * part);
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
                tmem_st8(t0 + L::BX + 16 * part + 8 * q, hi);
                tmem_st8(t0 + L::BX + 32 + 16 * part + 8 * q, lo);
            }
            hand_over(B_BX);
            wait(bar(B_D2), c & 1);
            tc_fence_after();
            tmem_ld32(r, t0 + L::D2 + 32 * part);
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
                tmem_st8(t0 + L::X + 16 * part + 8 * q, hi);
                tmem_st8(t0 + L::X + 32 + 16 * part + 8 * q, lo);
            }
            hand_over(B_U);
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
                tmem_st8(t0 + L::BX + 16 * part + 8 * q, hi);
                tmem_st8(t0 + L::BX + 32 + 16 * part + 8 * q, lo);
            }
            hand_over(B_UO);
            const int64_t at = int64_t(sq.slot0 + c) * p.H + h;
            if (SAVE && v0 + v < p.Vp) {
                uint4 *o = reinterpret_cast<uint4 *>(p.e + (at * p.Vp + v0 + v) * 64 + 32 * part);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[i] = make_uint4(pack_f2(x[4 * i]), pack_f2(x[4 * i + 1]), pack_f2(x[4 * i + 2]), pack_f2(x[4 * i + 3]));
            }
            const float gam_c = sc[SC_GAM * 64 + 63 - part * 32];
            const f2 gam_c2 = two(gam_c, gam_c);
            wait(bar(B_S), c & 1);
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < HK / 32; ++q) {
                tmem_ld32(r, t0 + L::S + part * HK + 32 * q);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) s[16 * q + i] = fma2(gam_c2, s[16 * q + i], two_bits(r[2 * i], r[2 * i + 1]));
            }
            if (c + 1 < sq.chunks) {
                put_state(c + 1);
                hand_over(B_AS);
            }
            wait(bar(B_O), c & 1);
            tc_fence_after();
            uint32_t r2[32];
            tmem_ld32(r, t0 + L::O1 + 32 * part);
            tmem_ld32(r2, t0 + L::O2 + 32 * part);
            tc_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_OREAD));
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
            if (by_copy) fence_async_proxy();
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
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_FREE + stage));
        }
        if (tid == 0) tma_store_done();
#pragma unroll
        for (int i = 0; i < HK / 2; ++i) {
            const int k = part * HK + 2 * i;
            const float2 x = apart(s[i]);
            float *to = p.s1 + state_at + int64_t(k) * p.V + v0 + v;
            if (real && k < p.K) to[0] = x.x;
            if (real && k + 1 < p.K) to[p.V] = x.y;
        }
    } else if (warp < 16) {
        // ---- M and P: every other chunk to each of two groups, up to two chunks ahead
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        const int t = tid & 127, pw = warp & 3, team = warp >> 2 & 1;
        unsigned char *mp = smem + L::MP + team * L::MP_BYTES;
        float *m = reinterpret_cast<float *>(mp);
        auto &f = reinterpret_cast<float (*)[4][128]>(smem + L::PREP)[team];
        const auto sync = [&] { asm volatile("bar.sync %0, 128;" :: "r"(2 + team) : "memory"); };
#pragma unroll 1
        for (int c = team; c < sq.chunks; c += 2) {
            const GateShared &gs = reinterpret_cast<const GateShared *>(smem + L::SC)[c % 3];
            wait(bar(B_GATES + c % 3), (c / 3) & 1);
            const int i = t & 63;
            const uint32_t row = tmem + (uint32_t(pw * 32) << 16) + L::KK;
            const bool l_row = t < 64;
            const float factor = l_row ? 1.f : p.scale;
            row_factors(f, factor, gs, i, t);
            if (c >= 2) wait(bar(B_MP + team), ((c - 2) >> 1) & 1);
            wait(bar(B_KK + team), (c >> 1) & 1);
            tc_fence_after();
            decayed_row(row, f, factor, l_row, !l_row, gs, i, t, [&](int bj, const float (&x)[16]) {
                if (l_row) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                        *reinterpret_cast<float4 *>(m + i * PITCH + 16 * bj + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                } else {
#pragma unroll
                    for (int pc = 0; pc < 2; ++pc)
                        *reinterpret_cast<uint4 *>(mp + L::P + tile_off<8>(i, 2 * bj + pc)) =
                            make_uint4(pack2(x[8 * pc], x[8 * pc + 1]), pack2(x[8 * pc + 2], x[8 * pc + 3]),
                                       pack2(x[8 * pc + 4], x[8 * pc + 5]), pack2(x[8 * pc + 6], x[8 * pc + 7]));
                }
            });
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_KREAD));
            sync();
            make_m(m, t, sync);
            fence_async_proxy();
            mbar_arrive(bar(B_PREP + team));
        }
    } else if (warp == 17) {
        // ---- tiles
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        for (int c = 0; c < sq.chunks; ++c) {
            if (c >= 3) wait(bar(B_FREE + c % 3), ((c - 3) / 3) & 1);
            const int tok = static_cast<int>(sq.t0 + int64_t(c) * 64);
            const int64_t left = sq.len - int64_t(c) * 64;
            const uint32_t st = base + (c % 3) * L::STAGE;
            // Behind the end of the row the copies bring zeros; behind a sequence that ends inside the row they bring the next
            // one's tokens, which are replaced by zeros here before anyone sees the tile.
            const bool tail = left < 64 && sq.t0 + sq.len < p.T;
            const uint32_t b = bar(tail ? B_TAIL : B_TILE + c % 3);
            if (lane == 0) {
                mbar_expect(b, L::STAGE);
#pragma unroll
                for (int half = 0; half < L::HALVES; ++half) {
                    tma_load(st + half * 16384, &maps.k, 64 * half, hk, tok, static_cast<int>(sq.b), b);
                    tma_load(st + half * 16384 + 8192, &maps.q, 64 * half, hk, tok, static_cast<int>(sq.b), b);
                }
                tma_load(st + L::KQ_BYTES, &maps.v, v0, h, tok, static_cast<int>(sq.b), b);
            }
            if (tail) {                              // once a sequence, its last chunk
                wait(b, 0);
                const uint4 zero = make_uint4(0, 0, 0, 0);
                unsigned char *sp = smem + (c % 3) * L::STAGE;
                for (int i = lane; i < (64 - static_cast<int>(left)) * 16; i += 32) {
                    const int r = static_cast<int>(left) + i / 16, pc = i % 16;
                    if (pc < 8 * L::HALVES) {
                        *reinterpret_cast<uint4 *>(sp + (pc >> 3) * 16384 + r * 128 + (pc & 7) * 16) = zero;
                        *reinterpret_cast<uint4 *>(sp + (pc >> 3) * 16384 + (64 + r) * 128 + (pc & 7) * 16) = zero;
                    }
                    *reinterpret_cast<uint4 *>(sp + L::KQ_BYTES + r * 256 + pc * 16) = zero;
                }
                fence_async_proxy();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_TILE + c % 3));
            }
        }
    } else if (warp == 16) {
        // ---- issue
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (elect_one()) {
            // 16 columns of K of S in tensor memory
            const auto state_term = [&](int step, int lo) {
                const int k = 16 * step, part = k / HK;
                return tmem + L::S + part * HK + (k - part * HK) / 2 + lo * HK / 2;
            };
            const auto kq = [](int step, int row) { return ((step >> 2) * 16384 + (step & 3) * 32 + row * 128) >> 4; };
            const auto issue_kk = [&](uint32_t tile, int team) {
#pragma unroll
                for (int s = 0; s < KP / 16; ++s)
                    tc_mma_ss(tmem + L::KK, tile_low(tile) + kq(s, 0), tile_low(tile) + kq(s, 0), mma_desc(64, false), s > 0);
                tc_commit(bar(B_KK + team));
            };
            int stage = 0, ahead = 2;                // ahead: stage of the chunk after the next
            uint32_t ahead_turn = 0;                 // how often it was filled before
            for (int c = 0; c < 2 && c < sq.chunks; ++c) {
                wait(bar(B_TILE + c), 0);
                if (c > 0) wait(bar(B_KREAD), 0);
                tc_fence_after();
                issue_kk(base + c * L::STAGE, c);
            }
#pragma unroll 1
            for (int c = 0; c < sq.chunks; ++c) {
                const uint32_t tile = base + stage * L::STAGE, rows = tile_low(tile), down = tile_low(tile, 16384);
                wait(bar(B_AS), c & 1);
                tc_fence_after();
#pragma unroll
                for (int lo = 0; lo < 2; ++lo)
#pragma unroll
                    for (int s = 0; s < KP / 16; ++s)
                        tc_mma_ts(tmem + L::X, state_term(s, lo), rows + kq(s, 0), mma_desc(64, false, true), lo + s > 0);      // -K S
                tc_commit(bar(B_X));
                if (c > 0) wait(bar(B_OREAD), (c - 1) & 1);
                tc_fence_after();
#pragma unroll
                for (int s = 0; s < KP / 16; ++s)
                    tc_mma_ts(tmem + L::O1, state_term(s, 0), rows + kq(s, 64), mma_desc(64, false), s > 0);
                const uint32_t mp = base + L::MP + (c & 1) * L::MP_BYTES, m = tile_low(mp);
                wait(bar(B_PREP + (c & 1)), (c >> 1) & 1);
                wait(bar(B_BX), c & 1);
                tc_fence_after();
                // tokens 16 t .. of x reach the tokens from 16 t on only
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t desc = mma_desc(64 - 16 * t, false, true), d = tmem + L::D2 + 16 * t, at = (16 * t * 128 + 32 * t) >> 4;
                    tc_mma_ts(d, tmem + L::BX + 8 * t, m + at, desc, t > 0);
                    tc_mma_ts(d, tmem + L::BX + 32 + 8 * t, m + at, desc, true);
                    tc_mma_ts(d, tmem + L::BX + 8 * t, m + (8192 >> 4) + at, desc, true);
                }
                tc_commit(bar(B_D2));
                wait(bar(B_U), c & 1);
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo)
                        tc_mma_ts(tmem + L::S, tmem + L::X + 32 * lo + 8 * t, down + kq(0, 16 * t), mma_desc(KP, true), t + lo > 0);
                tc_commit(bar(B_S));
                wait(bar(B_UO), c & 1);
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo)
                        tc_mma_ts(tmem + L::O2 + 16 * t, tmem + L::BX + 32 * lo + 8 * t, m + ((L::P + 16 * t * 128 + 32 * t) >> 4),
                                  mma_desc(64 - 16 * t, false), t + lo > 0);
                tc_commit(bar(B_O));
                tc_commit(bar(B_MP + (c & 1)));
                tc_commit(bar(B_FREE + stage));
                if (c + 2 < sq.chunks) {
                    wait(bar(B_TILE + ahead), ahead_turn & 1);
                    wait(bar(B_KREAD), (c + 1) & 1);
                    tc_fence_after();
                    issue_kk(base + ahead * L::STAGE, c & 1);
                }
                if (++ahead == 3) {
                    ahead = 0;
                    ++ahead_turn;
                }
                if (++stage == 3) stage = 0;
            }
        }
    } else if (warp == 18) {
        // ---- gates, as far ahead as there is room
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        GateLoader gates;
        gates.load(p, sq, 0, h, lane);
        for (int c = 0; c < sq.chunks; ++c) {
            GateShared &gs = reinterpret_cast<GateShared *>(smem + L::SC)[c % 3];
            float g[2], be[2];
            gates.get(p, g, be);
            if (c + 1 < sq.chunks) gates.load(p, sq, c + 1, h, lane);
            if (c >= 3) wait(bar(B_FREE + c % 3), ((c - 3) / 3) & 1);
            chunk_gates(g, be, p.scale, gs, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_GATES + c % 3));
            if (SAVE)
                for (int i = lane; i < SC_ARRAYS * 64; i += 32) p.sc[(int64_t(sq.slot0 + c) * p.H + h) * SC_ARRAYS * 64 + i] = gs.sc[i];
        }
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
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 16) tmem_dealloc(tmem, 512);
}

template <int KP, bool SAVE>
static int launch_sweep_tc(const DeltaParams &p, const TcMaps &maps, cudaStream_t st) {
    const int64_t grid = int64_t(p.n_seqs) * p.H * ((p.Vp + 127) / 128);
    if (grid > 0x7fffffff) return ASCAN_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(delta_sweep_tc_kernel<KP, SAVE>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcForward<KP>::BYTES) !=
        cudaSuccess)
        return ASCAN_ERR_LAUNCH;
    delta_sweep_tc_kernel<KP, SAVE><<<unsigned(grid), TC_THREADS, TcForward<KP>::BYTES, st>>>(p, maps);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

int delta_launch_sweep_tc(const DeltaParams &p, bool save, cudaStream_t st) {
    TcMaps maps;
    int rc;
    if ((rc = make_map(&maps.k, p.k, p, p.Kp, p.Hk, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_map(&maps.q, p.q, p, p.Kp, p.Hk, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_map(&maps.v, p.v, p, p.Vp, p.H, 128, false)) != ASCAN_OK) return rc;
    maps.store = p.V % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
    if (maps.store) {
        const int64_t row = int64_t(p.H) * p.V;
        const Planes out = {static_cast<const __nv_bfloat16 *>(p.out), 0, p.T * row, row, p.V};
        if ((rc = make_map(&maps.out, out, p, p.V, p.H, 128, false)) != ASCAN_OK) return rc;
    }
    if (p.Kp <= 64) return save ? launch_sweep_tc<64, true>(p, maps, st) : launch_sweep_tc<64, false>(p, maps, st);
    return save ? launch_sweep_tc<128, true>(p, maps, st) : launch_sweep_tc<128, false>(p, maps, st);
}

}  // namespace ascan
