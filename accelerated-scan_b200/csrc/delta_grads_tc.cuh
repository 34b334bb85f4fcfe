// Gated delta rule, gradients of a chunk on tcgen05, for bf16.  What delta_backward.cu computes after the sweep,
// with every product transposed to 128 rows of K:
//     dQ^T  = scale gam (S0 d_out^T) + K^T D^T                    D^T[j][i] = scale Gam_ij beta_j (e_j . d_out_i),   i >= j
//     read^T  = -gam beta (S0 z^T)   + K^T F^T                    F[i][j] = -Gam_ij beta_i beta_j (z_i . e_j),       i > j
//     write^T = Gam_C beta (dS1 e^T) + Q^T D + K^T F              dbeta_i = z_i . e_i, on F's diagonal
// All left operands lie in shared memory as they come ([v][k] states, [token][k] keys), D and F serve once by their rows and
// once by their columns.  D, F, e and z are two bf16 terms, the states one: the gradients are off by little more than their own
// rounding (1.7e-3; with one-term e and z 2.4e-3 for dQ and dK and 2.9e-3 for dbeta, one-term D and F too 2.9e-3).
//
// A persistent CTA walks over (chunk, key head) and the value heads of each; V comes in slabs of 64 through a ring of two, so
// that copies go on while D, F and the sums are worked on.  16 warps: thread (row, quarter of the columns) holds 16 values of
// every product.  What bounds it is the chain of an item, products - D, F - products - sums - stores, which one CTA an SM cannot
// hide: 4 x 4096 tokens, 16 heads of 128 x 128 took 266 us for 600 MB (2.3 TB/s) as a kernel of its own; on mma.sync 397, and
// with 8 warps, <S0, dS1> re-read from memory and an exponential an element of D and F 486.  It runs beside the sweep, on the
// SMs that the sweep leaves and on all of them behind it: the two take 480 us, not 679; with the chunks dealt out in advance
// over the SMs that do not sweep 590.
#pragma once

#include "delta_tc_roles.cuh"

namespace ascan {

struct GradMaps {
    CUtensorMap k, q, d_out, e, z, S, dS;
};

// Of a head's tokens: the gates' sums, and what the rows and columns of the products are multiplied by.  In blocks of 16 tokens
// (first, end: a block's first and last one): FROM = e^{G_t - G_first}, BACK = its inverse, TO = e^{G_end - G_t}.
enum : int { GR_GHI = 0, GR_GLO, GR_RESET, GR_BETA, GR_Q, GR_READ, GR_WRITE, GR_FROM, GR_BACK, GR_TO, GR_ARRAYS };

struct TcGrads {
    static constexpr int TOK = 8192, STATE = 16384;                               // a slab's [64][64] and [64 v][128 k]
    static constexpr int DO = 0, E = TOK, E_LO = 3 * TOK, S = 5 * TOK, DS = S + STATE, SLAB = DS + STATE;    // z behind e
    static constexpr int KQ = 2 * SLAB, KQ_BYTES = 32768, Z = E + TOK, Z_LO = E_LO + TOK;       // K: two halves of 8 KB, then Q
    static constexpr int D = KQ + KQ_BYTES, F = D + 2 * 8192;                 // hi, lo; later dQ and dK on their way out
    static constexpr int SC = D + 4 * 8192, RED = SC + GR_ARRAYS * 256, BARS = RED + 1024 + 128, BYTES = BARS + 256 + 1024;
    // columns of tensor memory
    static constexpr int DQ1 = 0, DR1 = 64, DW1 = 128, DP = 192, F0 = 256, DQ2 = 320, DR2 = 384, DW2 = 448;
};
static_assert(TcGrads::BYTES <= 227 * 1024, "shared memory");
enum : int { G_SLAB = 0, G_KQ = 2, G_ACC, G_OUT, G_TAIL, G_DF, G_READ, G_KQ_FREE, G_SLAB_FREE, G_ITEM = G_SLAB_FREE + 2, G_COUNT = G_ITEM + 2 };

constexpr int GRADS_WARPS = 16, GRADS_COMPUTE = 32 * GRADS_WARPS;      // and one that copies, one that issues

// Until the sweep has finished a chunk of a head, in all its slices of V: dS1 and z are in memory then, and what the copies
// read is what was written.  One thread.  A sweep takes about six microseconds a chunk: the limit
// allows a second and sixty a chunk.
__device__ __forceinline__ void wait_for_sweep(const DeltaParams &p, int at, const Waiter &wait) {
    const int slices = (p.Vp + 127) / 128;
    int64_t left = (int64_t(1) << 21) + 2 * p.T;
    int seen;
    while (true) {
        asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(seen) : "l"(p.done + 2 + at) : "memory");
        if (seen >= slices || *wait.dead) break;
        if (--left == 0) {
            *wait.dead = 1;
            if (wait.status) *reinterpret_cast<volatile int *>(wait.status) = 1;
        }
        __nanosleep(500);
    }
    asm volatile("fence.proxy.async.global;" ::: "memory");
}

// CTAs take chunks from a counter, in the order in which the sweep finishes them: CTAs that start when the sweeps end share what
// is left.  The copying warp takes them, the others read them from a ring of two (an item's place is written again when K and
// Q of the item behind it have been waited for, which all of them have finished then).
template <bool GROUPED>
__device__ __forceinline__ void chunk_gradients(const DeltaParams &p, const GradMaps &maps, unsigned char *smem_raw) {
    typedef TcGrads L;
    unsigned char *smem = smem_raw + (-smem_addr(smem_raw) & 1023);
    const uint32_t base = smem_addr(smem), bars = base + L::BARS;
    const auto bar = [&](int i) { return bars + 8 * i; };
    volatile int *dead = reinterpret_cast<volatile int *>(smem + L::BARS + 8 * G_COUNT);
    volatile int *ring = dead + 4, *current = dead + 6;          // behind dead and the address of tensor memory
    const Waiter wait = {dead, p.status};
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = p.H / p.Hk, slabs = (p.Vp + 63) / 64;
    const int items = p.slots * p.Hk;
    const auto slot_of = [&](int item) {
        const int i = item / p.Hk;
        return p.packed ? p.slots - 1 - i : i % p.n_seqs * p.chunks + p.chunks - 1 - i / p.n_seqs;
    };
    if (tid == 0) {
        *dead = 0;
        for (int i = 0; i < G_COUNT; ++i) mbar_init(bar(i), i < G_DF || i >= G_ITEM ? 1 : i < G_SLAB_FREE ? GRADS_WARPS : GRADS_WARPS + 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_proxy();
    }
    if (warp == GRADS_WARPS + 1) tmem_alloc(bar(G_COUNT + 1), 512);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::BARS + 8 * (G_COUNT + 1));

    if (warp < GRADS_WARPS) {
        const int part = warp >> 2, row = (warp & 3) * 32 + lane;         // row of tensor memory; quarter of the columns
        const uint32_t t0 = tmem + (uint32_t((warp & 3) * 32) << 16) + 16 * part;
        float *sg = reinterpret_cast<float *>(smem + L::SC), *red = reinterpret_cast<float *>(smem + L::RED);
        const auto sync = [] { group_sync<1, GRADS_COMPUTE>(); };
        int n_item = 0;
        uint32_t n_head = 0, n_slab = 0;
#pragma unroll 1
        while (true) {
            if (tid == 0) {                    // one thread says whether there is another item: all see the same
                wait(bar(G_ITEM + (n_item & 1)), (n_item >> 1) & 1);
                *current = *dead ? -1 : ring[n_item & 1];
            }
            sync();
            const int item = *current;
            if (item < 0) break;
            const int slot = slot_of(item), hk = item % p.Hk;
            const Chunk ch = get_chunk(p, slot);
            const int64_t tok0 = ch.b * p.T + ch.t0;
            const unsigned char *kq = smem + L::KQ + (row >> 6) * 8192 + (row & 7) * 2;
            const auto key = [&](int t, int q) {                           // K (Q) of token t, this thread's column
                return __uint_as_float(uint32_t(*reinterpret_cast<const uint16_t *>(
                    kq + q * 16384 + t * 128 + (((row >> 3 & 7) ^ (t & 7)) << 4))) << 16);
            };
            float rq[GROUPED ? 16 : 1] = {}, rk[GROUPED ? 16 : 1] = {};
#pragma unroll 1
            for (int hh = 0; hh < group; ++hh, ++n_head) {
                const int h = hk * group + hh;
                const float *sc = p.sc + (int64_t(slot) * p.H + h) * SC_ARRAYS * 64;
                sync();
                int *direct = reinterpret_cast<int *>(red + 256 + 16);
                if (tid < 64) {
                    const int t = tid, first = t & ~15, end = t | 15;
                    const float ghi = sc[SC_GHI * 64 + t], glo = sc[SC_GLO * 64 + t], res = sc[SC_RESET * 64 + t];
                    const float beta = sc[SC_BETA * 64 + t], gam = sc[SC_GAM * 64 + t], gam_c = sc[SC_GAMC * 64 + t];
                    const float from = (ghi - sc[SC_GHI * 64 + first]) + (glo - sc[SC_GLO * 64 + first]);
                    const float to = (sc[SC_GHI * 64 + end] - ghi) + (sc[SC_GLO * 64 + end] - glo);
                    sg[GR_GHI * 64 + t] = ghi;
                    sg[GR_GLO * 64 + t] = glo;
                    sg[GR_RESET * 64 + t] = res;
                    sg[GR_BETA * 64 + t] = beta;
                    sg[GR_Q * 64 + t] = p.scale * gam;
                    sg[GR_READ * 64 + t] = -gam * beta;
                    sg[GR_WRITE * 64 + t] = gam_c * beta;
                    sg[GR_FROM * 64 + t] = res == sc[SC_RESET * 64 + first] ? expf(from) : 0.f;
                    sg[GR_BACK * 64 + t] = expf(-from);
                    sg[GR_TO * 64 + t] = res == sc[SC_RESET * 64 + end] ? expf(to) : 0.f;
                    // blocks whose factors would leave fp32, or with a zero gate inside: an exponential an element
                    const bool plain = fabsf(from) <= 60.f && res == sc[SC_RESET * 64 + first];
                    const unsigned ok = __ballot_sync(~0u, plain);
                    if ((lane & 15) == 0) direct[t >> 4] = ((ok >> (lane & 16)) & 0xffffu) != 0xffffu;
                }
                const float gam_c = sc[SC_GAM * 64 + 63];
                // <S0, dS1>: 16 products a thread and slab, by plain loads (480 us a launch; as a diagonal of warp products 489)
                float dot_s = 0.f;
#pragma unroll 1
                for (int s = 0; s < slabs; ++s, ++n_slab) {
                    wait.warp(bar(G_SLAB + (n_slab & 1)), (n_slab >> 1) & 1);
                    // both lie alike: the same 16 bytes of each half of either
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const unsigned char *at = smem + (n_slab & 1) * L::SLAB + half * 8192 + tid * 16;
                        const uint4 x = *reinterpret_cast<const uint4 *>(at + L::S), y = *reinterpret_cast<const uint4 *>(at + L::DS);
                        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) dot_s += low_half(xs[j]) * low_half(ys[j]) + high_half(xs[j]) * high_half(ys[j]);
                    }
                    give_back_reads();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(G_SLAB_FREE + (n_slab & 1)));
                }
                dot_s *= gam_c;
                sync();
                wait.warp(bar(G_ACC), n_head & 1);
                tc_fence_after();
                // D^T (rows j, this quarter of i) on rows 0 - 63, F (rows i, this quarter of j) on rows 64 - 127
                {
                    const int me = row & 63, mine = me >> 4;
                    const bool d_row = row < 64;
                    const float beta = sg[GR_BETA * 64 + me];
                    uint32_t r[16];
                    tmem_ld16(r, t0 + (d_row ? L::DP : L::F0));
                    // behind the own block the factor of the row and block, inside it that of the row
                    const int ref = d_row ? 16 * part : 16 * part + 15;
                    const float *w = sg + (d_row ? GR_FROM : part == mine ? GR_BACK : GR_TO) * 64 + 16 * part;
                    float f = 0.f;
                    if (part == mine) {
                        f = sg[(d_row ? GR_BACK : GR_FROM) * 64 + me];
                    } else if (d_row ? part > mine : part < mine) {
                        const float g = (sg[GR_GHI * 64 + me] - sg[GR_GHI * 64 + ref]) + (sg[GR_GLO * 64 + me] - sg[GR_GLO * 64 + ref]);
                        f = sg[GR_RESET * 64 + me] == sg[GR_RESET * 64 + ref] ? expf(d_row ? -g : g) : 0.f;
                    }
                    f *= d_row ? p.scale * beta : -beta;
                    tc_wait_ld();
                    float x[16];
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 w4 = *reinterpret_cast<const float4 *>(w + j);
                        float4 b4 = make_float4(1.f, 1.f, 1.f, 1.f);
                        if (!d_row) b4 = *reinterpret_cast<const float4 *>(sg + GR_BETA * 64 + 16 * part + j);
                        x[j] = f * w4.x * b4.x; x[j + 1] = f * w4.y * b4.y; x[j + 2] = f * w4.z * b4.z; x[j + 3] = f * w4.w * b4.w;
                    }
                    if (part == mine && direct[part]) {
#pragma unroll 1
                        for (int j = 0; j < 16; ++j) {
                            const int c = 16 * part + j;
                            const float g = (sg[GR_GHI * 64 + me] - sg[GR_GHI * 64 + c]) + (sg[GR_GLO * 64 + me] - sg[GR_GLO * 64 + c]);
                            const float e = sg[GR_RESET * 64 + me] == sg[GR_RESET * 64 + c] ? expf(d_row ? -g : g) : 0.f;
                            const float y = e * (d_row ? p.scale * beta : -beta * sg[GR_BETA * 64 + c]);
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                if (k == j) x[k] = y;
                        }
                    }
                    const int low = d_row ? me : 0, high = d_row ? ch.rows : me;         // columns that count
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int c = 16 * part + j;
                        if (!d_row && c == me && me < ch.rows)
                            store_from_float(p.d_b, p.b_dtype, (tok0 + me) * p.H + h, __uint_as_float(r[j]));
                        x[j] = c >= low && c < high ? x[j] * __uint_as_float(r[j]) : 0.f;
                    }
                    unsigned char *tile = smem + (d_row ? L::D : L::F);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) split2(x[8 * q + 2 * j], x[8 * q + 2 * j + 1], hi[j], lo[j]);
                        *reinterpret_cast<uint4 *>(tile + tile_off<8>(me, 2 * part + q)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(tile + 8192 + tile_off<8>(me, 2 * part + q)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                tc_fence_before();
                fence_async_proxy();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(G_DF));
                if (hh == 0) wait.warp(bar(G_KQ), n_item & 1);
                wait.warp(bar(G_OUT), n_head & 1);
                tc_fence_after();
                float dot[16];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t a[8], b[8], c[8], d[8], e[8], f[8];
                    const int c0 = 16 * part + 8 * q;
                    tmem_ld8(a, t0 + L::DQ1 + 8 * q);
                    tmem_ld8(b, t0 + L::DQ2 + 8 * q);
                    tmem_ld8(c, t0 + L::DR1 + 8 * q);
                    tmem_ld8(d, t0 + L::DR2 + 8 * q);
                    tmem_ld8(e, t0 + L::DW1 + 8 * q);
                    tmem_ld8(f, t0 + L::DW2 + 8 * q);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        const float4 fq = *reinterpret_cast<const float4 *>(sg + GR_Q * 64 + c0 + i);
                        const float4 fr = *reinterpret_cast<const float4 *>(sg + GR_READ * 64 + c0 + i);
                        const float4 fw = *reinterpret_cast<const float4 *>(sg + GR_WRITE * 64 + c0 + i);
                        const float q4[4] = {fq.x, fq.y, fq.z, fq.w}, r4[4] = {fr.x, fr.y, fr.z, fr.w}, w4[4] = {fw.x, fw.y, fw.z, fw.w};
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const int j = i + m;
                            const float kv = key(c0 + j, 0), qv = key(c0 + j, 1);
                            float dq = q4[m] * __uint_as_float(a[j]) + __uint_as_float(b[j]);
                            const float dr = r4[m] * __uint_as_float(c[j]) + __uint_as_float(d[j]);
                            const float w1 = w4[m] * __uint_as_float(e[j]), dw = w1 + __uint_as_float(f[j]);
                            float dk = dr + dw;
                            dot_s += kv * w1;
                            dot[8 * q + j] = qv * dq + kv * (dr - dw);
                            if (GROUPED) {
                                constexpr int G = GROUPED ? 1 : 0;
                                dq = rq[G * (8 * q + j)] += dq;
                                dk = rk[G * (8 * q + j)] += dk;
                            }
                            if (!GROUPED || hh == group - 1) {             // the last head's products have read D and F
                                *reinterpret_cast<bf16 *>(smem + L::D + (c0 + j) * 256 + row * 2) = __float2bfloat16_rn(dq);
                                *reinterpret_cast<bf16 *>(smem + L::F + (c0 + j) * 256 + row * 2) = __float2bfloat16_rn(dk);
                            }
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(G_READ));
                // sums over K: 16 columns over 32 lanes, half of them handed over at a time; lanes 2 c and 2 c + 1 keep column c
#pragma unroll
                for (int d = 16; d > 1; d /= 2)
#pragma unroll
                    for (int j = 0; j < d / 2; ++j) {
                        const bool upper = lane & d;
                        const float give = upper ? dot[j] : dot[j + d / 2], keep = upper ? dot[j + d / 2] : dot[j];
                        dot[j] = keep + __shfl_xor_sync(~0u, give, d);
                    }
                dot[0] += __shfl_xor_sync(~0u, dot[0], 1);
                if (!(lane & 1)) red[(warp & 3) * 64 + 16 * part + (lane >> 1)] = dot[0];
#pragma unroll
                for (int d = 16; d; d /= 2) dot_s += __shfl_xor_sync(~0u, dot_s, d);
                if (lane == 0) red[256 + warp] = dot_s;
                sync();
                if (warp == 0) {            // sums of dG from each token to the end; the state's share stands on the last one
                    float x[2], tail = 0.f;
#pragma unroll
                    for (int w = 0; w < GRADS_WARPS; ++w) tail += red[256 + w];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int i = 2 * lane + j;
                        x[j] = i < ch.rows ? (red[i] + red[64 + i]) + (red[128 + i] + red[192 + i]) : 0.f;
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
                        const float before = i == 0 ? 0.f : sg[GR_RESET * 64 + i - 1];
                        const float dg = sg[GR_RESET * 64 + i] != before ? 0.f : tail + (j ? s - x[0] : s);
                        if (i < ch.rows) store_from_float(p.d_g, p.g_dtype, (tok0 + i) * p.H + h, dg);
                    }
                }
            }
            give_back_reads();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(G_KQ_FREE));
            ++n_item;
            // dQ and dK of the key head (the barrier before the sums has seen all their columns)
            for (int i = tid; i < 2 * 64 * 16; i += GRADS_COMPUTE) {
                const int which = i >> 10, t = i >> 4 & 63, col = (i & 15) * 8;
                if (t >= ch.rows || col >= p.K) continue;
                const uint4 v = *reinterpret_cast<const uint4 *>(smem + (which ? L::F : L::D) + t * 256 + col * 2);
                bf16 *o = static_cast<bf16 *>(which ? p.d_k : p.d_q) + ((tok0 + t) * p.Hk + hk) * p.K + col;
                if (p.K % 8 == 0) {
                    *reinterpret_cast<uint4 *>(o) = v;
                } else {
                    const bf16 *e = reinterpret_cast<const bf16 *>(&v);
                    for (int j = 0; j < 8 && col + j < p.K; ++j) o[j] = e[j];
                }
            }
        }
    } else if (warp == GRADS_WARPS) {
        // ---- copies
        int n_item = 0, n_tail = 0;
        uint32_t n_slab = 0;
        while (true) {
            int item = 0;
            if (lane == 0) item = *dead ? items : atomicAdd(p.done + 1, 1);
            item = __shfl_sync(~0u, item, 0);
            const bool more = item < items;
            const int slot = more ? slot_of(item) : 0, hk = item % p.Hk;
            const Chunk ch = get_chunk(p, slot);
            if (more && ch.rows == 0) continue;
            if (lane == 0) {
                ring[n_item & 1] = more ? item : -1;
                mbar_arrive(bar(G_ITEM + (n_item & 1)));
            }
            if (!more) break;
            const int tok = static_cast<int>(ch.t0), b0 = static_cast<int>(ch.b);
            for (int hh = 0; hh < group; ++hh) {
                const int h = hk * group + hh, at = slot * p.H + h;
                if (lane == 0) wait_for_sweep(p, at, wait);
                __syncwarp();
                for (int s = 0; s < slabs; ++s, ++n_slab) {
                    const int st = n_slab & 1;
                    if (n_slab >= 2) wait(bar(G_SLAB_FREE + st), ((n_slab - 2) >> 1) & 1);
                    if (lane == 0) {
                        const uint32_t d = base + st * L::SLAB, f = bar(G_SLAB + st);
                        mbar_expect(f, L::SLAB);
                        tma_load(d + L::DO, &maps.d_out, 64 * s, h, tok, b0, f);
#pragma unroll
                        for (int pl = 0; pl < 2; ++pl) {
                            tma_load(d + L::E + pl * (L::E_LO - L::E), &maps.e, 0, 64 * s, 2 * at + pl, 0, f);
                            tma_load(d + L::Z + pl * (L::E_LO - L::E), &maps.z, 0, 64 * s, 2 * at + pl, 0, f);
                        }
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            tma_load(d + L::S + half * 8192, &maps.S, 64 * half, 64 * s, at, 0, f);
                            tma_load(d + L::DS + half * 8192, &maps.dS, 64 * half, 64 * s, at, 0, f);
                        }
                    }
                    __syncwarp();
                }
                if (hh > 0) continue;
                // K and Q, once the item before has been finished.  Rows behind a sequence that ends inside the packed row are
                // the next one's: zeros in their place (K and Q only: of d_out's they reach columns that are not used)
                const bool tail = ch.rows < 64 && ch.t0 + ch.rows < p.T;
                if (n_item > 0) wait(bar(G_KQ_FREE), (n_item - 1) & 1);
                const uint32_t b = bar(tail ? G_TAIL : G_KQ), dst = base + L::KQ;
                if (lane == 0) {
                    mbar_expect(b, L::KQ_BYTES);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        tma_load(dst + half * 8192, &maps.k, 64 * half, hk, tok, b0, b);
                        tma_load(dst + 16384 + half * 8192, &maps.q, 64 * half, hk, tok, b0, b);
                    }
                }
                if (tail) {
                    wait(b, n_tail++ & 1);
                    for (int i = lane; i < (64 - ch.rows) * 32; i += 32)
                        *reinterpret_cast<uint4 *>(smem + L::KQ + (i >> 3 & 3) * 8192 + (ch.rows + i / 32) * 128 + (i & 7) * 16) =
                            make_uint4(0, 0, 0, 0);
                    fence_async_proxy();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(G_KQ));
                }
                ++n_item;
            }
        }
    } else if (warp == GRADS_WARPS + 1 && elect_one()) {
        // ---- issue.  Left operands: columns along the rows of their tiles, blocks of 64 columns 8 KB apart.  Right ones: `along`
        // a tile's rows (32 bytes a step of 16) or down them (2048).
        constexpr uint32_t ALONG = mma_desc(64, false, false, true), DOWN = mma_desc(64, true, false, true);
        const auto product = [&](uint32_t d, uint32_t a, uint32_t b, bool along, bool add) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                tc_mma_ss(tmem + d, tile_low(a, 8192) + (2048 * t >> 4), tile_low(b) + ((along ? 32 : 2048) * t >> 4), along ? ALONG : DOWN, add || t > 0);
        };
        int n_item = 0;
        uint32_t n_slab = 0, n_head = 0;
        while (true) {
            wait(bar(G_ITEM + (n_item & 1)), (n_item >> 1) & 1);
            if (*dead || ring[n_item & 1] < 0) break;
            const uint32_t keys = base + L::KQ, queries = keys + 16384;
            for (int hh = 0; hh < group; ++hh, ++n_head) {
                // what D and F are made of does not wait until the head before has been read; the rest does.  Both slabs of a V
                // up to 128 stay for that; of a longer one each slab is finished in its turn.
                const auto early = [&](uint32_t n, bool add) {
                    const uint32_t d = base + (n & 1) * L::SLAB;
                    wait(bar(G_SLAB + (n & 1)), (n >> 1) & 1);
                    tc_fence_after();
                    product(L::DP, d + L::E, d + L::DO, true, add);                 // [e; z] d_out^T: rows of e
                    product(L::DP, d + L::E_LO, d + L::DO, true, true);
                    product(L::F0, d + L::E, d + L::E, false, add);                 // [e; z] e^T: rows of z
                    product(L::F0, d + L::E_LO, d + L::E, false, true);
                    product(L::F0, d + L::E, d + L::E_LO, false, true);
                };
                const auto second = [&](uint32_t n, bool add) {
                    const uint32_t d = base + (n & 1) * L::SLAB;
                    product(L::DQ1, d + L::S, d + L::DO, true, add);
                    product(L::DR1, d + L::S, d + L::Z, false, add);
                    product(L::DR1, d + L::S, d + L::Z_LO, false, true);
                    product(L::DW1, d + L::DS, d + L::E, false, add);
                    product(L::DW1, d + L::DS, d + L::E_LO, false, true);
                    tc_commit(bar(G_SLAB_FREE + (n & 1)));
                };
                const auto read_before = [&] {
                    if (n_head > 0) wait(bar(G_READ), (n_head - 1) & 1);
                    tc_fence_after();
                };
                if (slabs <= 2) {
                    for (int s = 0; s < slabs; ++s) early(n_slab + s, s > 0);
                    tc_commit(bar(G_ACC));
                    read_before();
                    for (int s = 0; s < slabs; ++s) second(n_slab + s, s > 0);
                } else {
                    read_before();
                    for (int s = 0; s < slabs; ++s) {
                        early(n_slab + s, s > 0);
                        second(n_slab + s, s > 0);
                    }
                    tc_commit(bar(G_ACC));
                }
                n_slab += slabs;
                if (hh == 0) wait(bar(G_KQ), n_item & 1);
                wait(bar(G_DF), n_head & 1);
                tc_fence_after();
#pragma unroll
                for (int lo = 0; lo < 2; ++lo) {
                    product(L::DQ2, keys, base + L::D + lo * 8192, false, lo > 0);
                    product(L::DR2, keys, base + L::F + lo * 8192, true, lo > 0);
                    product(L::DW2, queries, base + L::D + lo * 8192, true, lo > 0);
                    product(L::DW2, keys, base + L::F + lo * 8192, false, true);
                }
                tc_commit(bar(G_OUT));
            }
            ++n_item;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    drain(dead);
    if (warp == GRADS_WARPS + 1) tmem_dealloc(tmem, 512);
}

// rows of `cols` bf16 in [outer][Vp][cols] scratch, in boxes of 64 x 64
static int scratch_map(CUtensorMap *map, const bf16 *x, const DeltaParams &p, int cols, int planes) {
    DeltaParams q = p;                       // (column, row, slot and head and plane, -)
    q.T = int64_t(p.slots) * p.H * planes;
    q.batch = 1;
    const Planes pl = {x, 0, 0, int64_t(p.Vp) * cols, cols};
    return make_box_map(map, pl, q, cols, p.Vp, 64, 64, 1, true);
}

static int make_grad_maps(GradMaps *maps, const DeltaParams &p) {
    int rc;
    if ((rc = make_map(&maps->k, p.k, p, p.Kp, p.Hk, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_map(&maps->q, p.q, p, p.Kp, p.Hk, 64, true)) != ASCAN_OK) return rc;
    if ((rc = make_map(&maps->d_out, p.d_out, p, p.Vp, p.H, 64, true)) != ASCAN_OK) return rc;
    if ((rc = scratch_map(&maps->e, p.e, p, 64, 2)) != ASCAN_OK) return rc;
    if ((rc = scratch_map(&maps->z, p.z, p, 64, 2)) != ASCAN_OK) return rc;
    if ((rc = scratch_map(&maps->S, p.S, p, p.Kp <= 64 ? 64 : 128, 1)) != ASCAN_OK) return rc;
    if ((rc = scratch_map(&maps->dS, p.dS, p, p.Kp <= 64 ? 64 : 128, 1)) != ASCAN_OK) return rc;
    return ASCAN_OK;
}

}  // namespace ascan
