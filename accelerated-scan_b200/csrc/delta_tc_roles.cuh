// What the forward and the backward sweep on tcgen05 have in common: the warps beside the ones that carry the state.
#pragma once

#include <cuda.h>

#include "delta_tc.cuh"

namespace ascan {

struct TcMaps {
    CUtensorMap k, q, v, out;  // v: values, or the gradient of out; out: out, or the gradient of values
    bool store;                // out can be written by copies: rows start on 16 bytes
};

// (column, head, token, batch) of planes, in boxes of `cols` columns, `box_heads` heads and `tokens` tokens.  What lies outside
// of the array reads as zero.
static inline int make_box_map(CUtensorMap *map, const Planes &x, const DeltaParams &p, int d, int heads, int cols, int box_heads,
                               int tokens, bool swizzled) {
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
    const cuuint32_t box[4] = {cuuint32_t(cols), cuuint32_t(box_heads), cuuint32_t(tokens), 1}, unit[4] = {1, 1, 1, 1};
    const auto run = [&] {
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16 *>(x.p), dims, strides, box, unit,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult rc = run();
    if (rc == CUDA_ERROR_INVALID_CONTEXT) {             // a thread that has not used its device yet, as autograd's may be
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return ASCAN_ERR_DEVICE;
        rc = run();
    }
    return rc == CUDA_SUCCESS ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}
static inline int make_map(CUtensorMap *map, const Planes &x, const DeltaParams &p, int d, int heads, int cols, bool swizzled) {
    return make_box_map(map, x, p, d, heads, cols, 1, 64, swizzled);
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


// (token, v) arrays of the output type that copies can write
static inline int make_store_map(TcMaps *maps, void *dst, const DeltaParams &p, bool swizzled) {
    maps->store = p.V % 8 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
    if (!maps->store) return ASCAN_OK;
    const int64_t row = int64_t(p.H) * p.V;
    const Planes out = {static_cast<const __nv_bfloat16 *>(dst), 0, p.T * row, row, p.V};
    return make_map(&maps->out, out, p, p.V, p.H, swizzled ? 64 : 128, swizzled);
}

// Shared memory: three stages of tiles ([K; Q] as 128 rows, one block of 64 columns or two; V or d_out), two buffers of M, two
// or three of P, three of the gates.  The forward reads a chunk's P last, so P has a third buffer there: the next preparation
// but one then waits for M's reader only.  The backward reads P first.
template <int KP, bool BACK>
struct TcLayout {
    static constexpr int HALVES = KP / 64, KQ_BYTES = HALVES * 16384, V_BYTES = 64 * 256, STAGE = KQ_BYTES + V_BYTES;
    static constexpr int M = 3 * STAGE, P = M + 2 * M_BYTES, P_BYTES = (BACK ? 2 : 1) * 8192, P_BUFFERS = BACK ? 2 : 3;
    static constexpr int SC = P + P_BUFFERS * P_BYTES, PREP = SC + 3 * sizeof(GateShared);
    static constexpr int BARS = PREP + 2 * 4 * 128 * 4, BYTES = BARS + 256 + 1024;               // and 1024 to align the start
    static constexpr int KK = 448;           // columns of tensor memory of [K; Q] K^T
};
static_assert(TcLayout<128, false>::BYTES <= 227 * 1024 && TcLayout<128, true>::BYTES <= 227 * 1024, "shared memory");

// Barriers: filled tiles, prepared chunks, gates; commits of K K^T and of M's reader; K K^T read; tile free
// (the commit of its last product and eight warps); a sequence's last tile.  From B_OWN on each kernel's.
enum : int { B_TILE = 0, B_PREP = 3, B_GATES = 5, B_KK = 8, B_MP = 10, B_KREAD = 12, B_FREE = 13, B_TAIL = 16, B_OWN = 17 };

constexpr int TC_THREADS = 20 * 32;
// Registers a thread: 96 at launch; 152 * 256 (state) + 64 * 256 (preparation) + 48 * 128 (the others) = 96 * 640

struct TcBlock {             // what every role starts from
    unsigned char *smem;
    uint32_t base, bars, tmem;
    Waiter wait;
    Sequence sq;
    int h, hk, n_seq, v0;
    __device__ __forceinline__ uint32_t bar(int i) const { return bars + 8 * i; }
};

// block: which sequence, head and 128 columns of V.  commits: barriers from B_OWN on that one commit completes; the next `warps` ones take eight warps
template <class L>
__device__ __forceinline__ TcBlock tc_begin(const DeltaParams &p, unsigned char *raw, int block, int commits, int warps) {
    TcBlock k;
    k.smem = raw + (-smem_addr(raw) & 1023);
    k.base = smem_addr(k.smem);
    k.bars = k.base + L::BARS;
    const int slices = (p.Vp + 127) / 128, count = B_OWN + commits + warps;
    k.v0 = block % slices * 128;
    k.h = block / slices % p.H;
    k.n_seq = block / slices / p.H;
    k.hk = k.h / (p.H / p.Hk);
    k.sq = get_sequence(p, k.n_seq);
    volatile int *dead = reinterpret_cast<volatile int *>(k.smem + L::BARS + 8 * count);
    k.wait = Waiter{dead, p.status};
    if (threadIdx.x == 0) {
        *dead = 0;
        for (int i = 0; i < count; ++i)
            mbar_init(k.bar(i), i >= B_PREP && i < B_GATES ? 128 : i == B_KREAD ? 4 : i >= B_FREE && i < B_TAIL ? 9 :
                                i >= B_OWN + commits ? 8 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_proxy();
    }
    if (threadIdx.x >> 5 == 16) tmem_alloc(k.bar(count + 1), 512);
    __syncthreads();
    tc_fence_after();
    k.tmem = *reinterpret_cast<volatile uint32_t *>(k.smem + L::BARS + 8 * (count + 1));
    return k;
}

__device__ __forceinline__ void tc_end(const TcBlock &k) {
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    drain(k.wait.dead);
    if (threadIdx.x >> 5 == 16) tmem_dealloc(k.tmem, 512);
}

// M and P: every other chunk to each of two groups of four warps, up to two chunks ahead.  `turn` counts chunks in the order
// of the sweep.  Forward: M diag(beta), P in one term; backward: diag(beta) M, P in two.
template <class L, bool BACK>
__device__ __forceinline__ void prepare_chunks(const DeltaParams &p, const TcBlock &k) {
    const int t = threadIdx.x & 127, lane = t & 31, pw = t >> 5, team = threadIdx.x >> 7 & 1;
    float *m = reinterpret_cast<float *>(k.smem + L::M + team * M_BYTES);
    auto &f = reinterpret_cast<float (*)[4][128]>(k.smem + L::PREP)[team];
    const auto sync = [&] { asm volatile("bar.sync %0, 128;" :: "r"(2 + team) : "memory"); };
    const int i = t & 63;
    const uint32_t row = k.tmem + (uint32_t(pw * 32) << 16) + L::KK;
    const bool l_row = t < 64;
#pragma unroll 1
    for (int turn = team; turn < k.sq.chunks; turn += 2) {
        const GateShared &gs = reinterpret_cast<const GateShared *>(k.smem + L::SC)[turn % 3];
        k.wait.warp(k.bar(B_GATES + turn % 3), (turn / 3) & 1);
        unsigned char *pt = k.smem + L::P + turn % L::P_BUFFERS * L::P_BYTES;      // three: free when this chunk's gates were written
        const float factor = !l_row ? p.scale : BACK ? gs.sc[SC_BETA * 64 + i] : 1.f;
        row_factors(f, factor, gs, i, t);
        if (turn >= 2) k.wait.warp(k.bar(B_MP + team), ((turn - 2) >> 1) & 1);
        k.wait.warp(k.bar(B_KK + team), (turn >> 1) & 1);
        tc_fence_after();
        decayed_row(row, f, factor, !BACK && l_row, !l_row, gs, i, t, [&](int bj, const float (&x)[16]) {
            if (l_row) {
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                    *reinterpret_cast<float4 *>(m + i * PITCH + 16 * bj + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
            } else {
#pragma unroll
                for (int pc = 0; pc < 2; ++pc) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (BACK) split2(x[8 * pc + 2 * j], x[8 * pc + 2 * j + 1], hi[j], lo[j]);
                        else hi[j] = pack2(x[8 * pc + 2 * j], x[8 * pc + 2 * j + 1]);
                    }
                    *reinterpret_cast<uint4 *>(pt + tile_off<8>(i, 2 * bj + pc)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (BACK)
                        *reinterpret_cast<uint4 *>(pt + 8192 + tile_off<8>(i, 2 * bj + pc)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
        });
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(k.bar(B_KREAD));
        sync();
        make_m(m, t, sync);
        fence_async_proxy();
        mbar_arrive(k.bar(B_PREP + team));
    }
}

// Tiles of a chunk, up to three in flight; one warp.  V_HALVES: V's tile is two swizzled blocks of 64 columns, else 64 rows
// of 256 bytes.
template <class L, bool BACK, bool V_HALVES>
__device__ __forceinline__ void load_tiles(const DeltaParams &p, const TcBlock &k, const TcMaps &maps) {
    const int lane = threadIdx.x & 31, b0 = static_cast<int>(k.sq.b);
    // Backward: a chunk whose tiles are free has written z and dS1; the CTAs that wait for them are told.
    const auto publish = [&](int turn) {
        if (lane == 0) {
            __threadfence();
            atomicAdd(p.done + 2 + (k.sq.slot0 + k.sq.chunks - 1 - turn) * p.H + k.h, 1);
        }
        __syncwarp();
    };
#pragma unroll 1
    for (int turn = 0; turn < k.sq.chunks; ++turn) {
        const int c = BACK ? k.sq.chunks - 1 - turn : turn, stage = turn % 3;
        if (turn >= 3) k.wait(k.bar(B_FREE + stage), ((turn - 3) / 3) & 1);
        const int tok = static_cast<int>(k.sq.t0 + int64_t(c) * 64);
        const int64_t left = k.sq.len - int64_t(c) * 64;
        const uint32_t st = k.base + stage * L::STAGE;
        // Behind the end of the row the copies bring zeros; behind a sequence that ends inside the row they bring the next
        // one's tokens, which are replaced by zeros here before anyone sees the tile.
        const bool tail = left < 64 && k.sq.t0 + k.sq.len < p.T;
        const uint32_t b = k.bar(tail ? B_TAIL : B_TILE + stage);
        if (lane == 0) {
            mbar_expect(b, L::STAGE);
#pragma unroll
            for (int half = 0; half < L::HALVES; ++half) {
                tma_load(st + half * 16384, &maps.k, 64 * half, k.hk, tok, b0, b);
                tma_load(st + half * 16384 + 8192, &maps.q, 64 * half, k.hk, tok, b0, b);
            }
            tma_load(st + L::KQ_BYTES, &maps.v, k.v0, k.h, tok, b0, b);
            if (V_HALVES) tma_load(st + L::KQ_BYTES + 8192, &maps.v, k.v0 + 64, k.h, tok, b0, b);
        }
        if (tail) {                              // once a sequence, its last chunk
            k.wait(b, 0);
            const uint4 zero = make_uint4(0, 0, 0, 0);
            unsigned char *sp = k.smem + stage * L::STAGE;
            for (int i = lane; i < (64 - static_cast<int>(left)) * 16; i += 32) {
                const int r = static_cast<int>(left) + i / 16, pc = i % 16;
                if (pc < 8 * L::HALVES) {
                    *reinterpret_cast<uint4 *>(sp + (pc >> 3) * 16384 + r * 128 + (pc & 7) * 16) = zero;
                    *reinterpret_cast<uint4 *>(sp + (pc >> 3) * 16384 + (64 + r) * 128 + (pc & 7) * 16) = zero;
                }
                *reinterpret_cast<uint4 *>(sp + L::KQ_BYTES + (V_HALVES ? (pc >> 3) * 8192 + r * 128 + (pc & 7) * 16 : r * 256 + pc * 16)) = zero;
            }
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(k.bar(B_TILE + stage));
        }
        if (BACK && turn >= 3) publish(turn - 3);
    }
    if (BACK)
#pragma unroll 1
        for (int turn = k.sq.chunks < 3 ? 0 : k.sq.chunks - 3; turn < k.sq.chunks; ++turn) {
            k.wait(k.bar(B_FREE + turn % 3), (turn / 3) & 1);
            publish(turn);
        }
}

// Gates, as far ahead as there is room; one warp.  KEEP: also to memory, for the gradients of the chunk.
template <class L, bool BACK, bool KEEP>
__device__ __forceinline__ void run_gates(const DeltaParams &p, const TcBlock &k) {
    const int lane = threadIdx.x & 31;
    const auto chunk = [&](int turn) { return BACK ? k.sq.chunks - 1 - turn : turn; };
    GateLoader gates;
    if (k.sq.chunks > 0) gates.load(p, k.sq, chunk(0), k.h, lane);
#pragma unroll 1
    for (int turn = 0; turn < k.sq.chunks; ++turn) {
        GateShared &gs = reinterpret_cast<GateShared *>(k.smem + L::SC)[turn % 3];
        float g[2], be[2];
        gates.get(p, g, be);
        if (turn + 1 < k.sq.chunks) gates.load(p, k.sq, chunk(turn + 1), k.h, lane);
        if (turn >= 3) k.wait(k.bar(B_FREE + turn % 3), ((turn - 3) / 3) & 1);
        chunk_gates(g, be, p.scale, gs, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(k.bar(B_GATES + turn % 3));
        if (KEEP)
            for (int i = lane; i < SC_ARRAYS * 64; i += 32)
                p.sc[(int64_t(k.sq.slot0 + chunk(turn)) * p.H + k.h) * SC_ARRAYS * 64 + i] = gs.sc[i];
    }
}

// [K; Q] K^T of a tile
template <class L>
__device__ __forceinline__ void issue_kk(const TcBlock &k, int stage, int team) {
    const uint32_t tile = tile_low(k.base + stage * L::STAGE);
#pragma unroll
    for (int s = 0; s < 4 * L::HALVES; ++s) {
        const uint32_t at = tile + (((s >> 2) * 16384 + (s & 3) * 32) >> 4);
        tc_mma_ss(k.tmem + L::KK, at, at, mma_desc(64, false), s > 0);
    }
    tc_commit(k.bar(B_KK + team));
}

// The issuing thread's view of the ring: stages in turn, and K K^T two chunks ahead
template <class L>
struct TileRing {
    int stage = 0, ahead = 2;
    uint32_t ahead_turn = 0;                 // how often that stage was filled before
    __device__ __forceinline__ void begin(const TcBlock &k) {
        for (int c = 0; c < 2 && c < k.sq.chunks; ++c) {
            k.wait(k.bar(B_TILE + c), 0);
            if (c > 0) k.wait(k.bar(B_KREAD), 0);
            tc_fence_after();
            issue_kk<L>(k, c, c);
        }
    }
    // Where M's reader has been issued: the group that prepared this chunk is free for the next but one.
    __device__ __forceinline__ void m_read(const TcBlock &k, int turn) {
        tc_commit(k.bar(B_MP + (turn & 1)));
        if (turn + 2 < k.sq.chunks) {
            k.wait(k.bar(B_TILE + ahead), ahead_turn & 1);
            k.wait(k.bar(B_KREAD), (turn + 1) & 1);
            tc_fence_after();
            issue_kk<L>(k, ahead, turn & 1);
        }
        if (++ahead == 3) {
            ahead = 0;
            ++ahead_turn;
        }
    }
    __device__ __forceinline__ void next(const TcBlock &k) {
        tc_commit(k.bar(B_FREE + stage));
        if (++stage == 3) stage = 0;
    }
};

// What a warp stored to tensor memory is there
__device__ __forceinline__ void hand_over(const TcBlock &k, int b) {
    tc_wait_st();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(k.bar(b));
}

// 32 bytes, a whole sector at once (4 x 4096 tokens, 16 heads of 128 x 128, forward and backward sweep: 383 and 413 us; with
// 16 bytes a store, and e and z stored before the next product's operand is handed over, 439 and 469)
__device__ __forceinline__ void store_sector(bf16 *to, const uint32_t (&r)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// A thread's part of the (transposed) state, HK of K's columns, as two terms to tensor memory at `at`; the first one also to
// memory where keep.
template <int HK>
__device__ __forceinline__ void put_state(const f2 (&s)[HK / 2], uint32_t at, bf16 *keep) {
#pragma unroll
    for (int q = 0; q < HK / 16; ++q) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split_f2(s[8 * q + i], hi[i], lo[i]);
        tmem_st8(at + 8 * q, hi);
        tmem_st8(at + HK / 2 + 8 * q, lo);
        if (keep) store_sector(keep + 16 * q, hi);
    }
}
// A thread's 32 tokens of e or z, as two terms in two planes `plane` elements apart
__device__ __forceinline__ void keep_tokens(const f2 (&x)[16], bf16 *to, int64_t plane) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split_f2(x[8 * q + i], hi[i], lo[i]);
        store_sector(to + 16 * q, hi);
        store_sector(to + plane + 16 * q, lo);
    }
}
// 16 columns of the state as an operand
template <int HK>
__device__ __forceinline__ uint32_t state_term(uint32_t at, int step, int lo) {
    const int k = 16 * step, part = k / HK;
    return at + part * HK + (k - part * HK) / 2 + lo * HK / 2;
}

}  // namespace ascan
