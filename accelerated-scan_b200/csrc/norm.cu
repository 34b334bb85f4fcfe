// Norms before and after a block, with its gate and residual scale, in one pass over the rows:
//     n = x rsqrt(mean x^2 + eps) post_weight          (x itself without post_weight)
//     h = residual + scale act(gate) n
//     y = h rsqrt(mean h^2 + eps) pre_weight
// and its gradients.  Everything is bound by memory: the forward reads x, residual and gate and writes h and y, the
// backward reads x, residual, gate and the two gradients and writes three; a row stays in registers between its
// reductions.  The backward recomputes h from the inputs (the same bytes as reading a saved one), so that no sum sees a
// rounded h.  A thread holds eight elements (sixteen in the forward of long rows), 16 bytes at a time;
// G threads share a row, and a CTA keeps the weights, and in the backward the weights' gradients, in registers over all
// its rows.  Sums of the weights' gradients over CTAs are a second launch, in a fixed order.
//
// Measured, bf16: 32768 rows of 4096 with all parts, forward, 276 us (1.34 GB, 4.9 TB/s; 6.55 are a plain copy's); 262144
// heads of 128 with a gate, forward 52 us and backward 85 us (201 and 335 MB, 3.9 TB/s).  Backward with all parts, 2.15 GB each:
// 32768 rows of 4096 823 us, 16384 of 8192 1716 us; in fp32, 16384 of 4096, 471 us.  What is missing is issue slots and warps to
// hide latencies: 2.7 of 4 instructions a clock at 35 % of the warps (rows of 128), 2.0 to 2.2 at 25 % (long rows), where fixed
// latencies, shared loads and barriers stall about equally; conversions, gates and the rows' reductions are most of the work.
#include <atomic>

#include "delta_tc.cuh"

namespace ascan {

struct NormParams {
    int64_t rows, x_s, r_s, g_s, dh_s, dy_s;        // rows; elements from row to row
    int32_t D, w_dtype, act, groups;                // groups: threads of a row, G
    float eps, scale_value;
    const void *x, *residual, *gate, *post_w, *scale, *pre_w;
    void *hidden, *normed;
    const void *d_hidden, *d_normed;
    void *d_x, *d_residual, *d_gate;
    float *partial;                                 // [grid][2][D]: post and scale (below), pre
    int32_t stages;                                 // of the copies' ring; 0: plain loads
    int *status;                                    // nullable: set when a wait for a copy expired
};

constexpr int NORM_THREADS = 1024, NORM_MAX_D = 8 * NORM_THREADS;
constexpr int NORM_NARROW = 512;                    // threads up to which the backward keeps all it needs in registers

enum : int { LEAN, MIDDLE, WIDE_ROWS };
enum : int { ACT_NONE = 0, ACT_SIGMOID = 1, ACT_SILU = 2 };

template <class T> struct Elem;
template <> struct Elem<float> {
    static constexpr int VEC = 4;
    static __device__ void unpack(uint4 r, float *x) {
        x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
    }
    static __device__ uint4 pack(const float *x) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    static __device__ float get(float v) { return v; }
    static __device__ float put(float v) { return v; }
};
template <> struct Elem<bf16> {
    static constexpr int VEC = 8;
    static __device__ void unpack(uint4 r, float *x) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = low_half(w[i]); x[2 * i + 1] = high_half(w[i]); }
    }
    static __device__ uint4 pack(const float *x) {
        return make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
    }
    static __device__ float get(bf16 v) { return __bfloat162float(v); }
    static __device__ bf16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
    static constexpr int VEC = 8;
    static __device__ void unpack(uint4 r, float *x) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
    static __device__ uint4 pack(const float *x) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ float get(__half v) { return __half2float(v); }
    static __device__ __half put(float v) { return __float2half_rn(v); }
};

// Where a thread's E elements lie in a row: pieces of 16 bytes, G pieces apart, or every G-th element (not ALIGNED).
template <class T, bool ALIGNED>
__device__ __forceinline__ int element(int i, int gt, int G) {
    constexpr int VEC = Elem<T>::VEC;
    return ALIGNED ? (i / VEC * G + gt) * VEC + i % VEC : gt + i * G;
}

template <class T, bool ALIGNED, int E>
__device__ __forceinline__ void load_row(const void *src, int64_t at, int gt, int G, int D, float (&x)[E]) {
    const T *s = static_cast<const T *>(src) + at;
    if (ALIGNED) {
        constexpr int VEC = Elem<T>::VEC;
#pragma unroll
        for (int i = 0; i < E; i += VEC) {
            uint4 r = make_uint4(0, 0, 0, 0);
            const int e = element<T, true>(i, gt, G);
            if (e < D) r = __ldcs(reinterpret_cast<const uint4 *>(s + e));
            Elem<T>::unpack(r, x + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = gt + i * G < D ? Elem<T>::get(s[gt + i * G]) : 0.f;
    }
}

template <class T, bool ALIGNED, int E>
__device__ __forceinline__ void store_row(void *dst, int64_t at, int gt, int G, int D, const float (&x)[E]) {
    T *s = static_cast<T *>(dst) + at;
    if (ALIGNED) {
        constexpr int VEC = Elem<T>::VEC;
#pragma unroll
        for (int i = 0; i < E; i += VEC) {
            const int e = element<T, true>(i, gt, G);
            if (e < D) *reinterpret_cast<uint4 *>(s + e) = Elem<T>::pack(x + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (gt + i * G < D) s[gt + i * G] = Elem<T>::put(x[i]);
    }
}

// Rows by bulk copies: a ring of `stages` buffers, each the rows that the CTA works on at once (`slots`) of every input, so
// that the next rows are under way while these are reduced: with plain loads a CTA asks for nothing between its first
// barrier and its last store.  One thread issues; rows that lie dense are one copy an input.  32768 rows of 4096, bf16: 508 us
// with plain loads, 278 so (lighter gates and sixteen elements a thread are in it too).
template <class T, int INPUTS>
struct RowRing {
    const NormParams &p;
    const void *src[INPUTS];
    int64_t stride[INPUTS];
    int slots, stage = 0, turn = 0;
    uint32_t base, bars, bytes;          // bytes: of an input in a buffer
    unsigned char *mem;
    volatile int *dead;
    int64_t next;                        // first row that has not been asked for

    __device__ __forceinline__ RowRing(const NormParams &params, unsigned char *smem, uint64_t *bar, int *gave_up, int slots_)
        : p(params), slots(slots_), bars(smem_addr(bar)), mem(smem), dead(gave_up) {
        base = smem_addr(smem);
        bytes = uint32_t(slots) * p.D * sizeof(T);
        next = int64_t(blockIdx.x) * slots;
    }
    __device__ __forceinline__ void init() {
        if (threadIdx.x == 0) {
            *dead = 0;
            for (int i = 0; i < p.stages; ++i) mbar_init(bars + 8 * i, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_async_proxy();
        }
        __syncthreads();
        if (threadIdx.x == 0)
            for (int i = 0; i < p.stages; ++i) issue(i);
    }
    __device__ __forceinline__ void copy(uint32_t dst, const void *from, uint32_t n, uint32_t bar) {
        asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     :: "r"(dst), "l"(from), "r"(n), "r"(bar) : "memory");
    }
    __device__ __forceinline__ void issue(int s) {       // one thread
        if (next >= p.rows) return;
        const int rows = static_cast<int>(p.rows - next < slots ? p.rows - next : slots);
        uint32_t total = 0;
#pragma unroll
        for (int i = 0; i < INPUTS; ++i) total += src[i] ? rows * p.D * uint32_t(sizeof(T)) : 0;
        mbar_expect(bars + 8 * s, total);
#pragma unroll
        for (int i = 0; i < INPUTS; ++i) {
            if (!src[i]) continue;
            const T *from = static_cast<const T *>(src[i]) + next * stride[i];
            const uint32_t dst = base + (s * INPUTS + i) * bytes;
            if (stride[i] == p.D || rows == 1) {
                copy(dst, from, rows * p.D * uint32_t(sizeof(T)), bars + 8 * s);
            } else {
                for (int r = 0; r < rows; ++r)
                    copy(dst + r * p.D * uint32_t(sizeof(T)), from + r * stride[i], p.D * uint32_t(sizeof(T)), bars + 8 * s);
            }
        }
        next += int64_t(gridDim.x) * slots;
    }
    __device__ __forceinline__ void arrive() {           // the rows of this turn are in their buffer
        const Waiter wait = {dead, p.status};
        wait(bars + 8 * stage, turn & 1);
    }
    template <int E>
    __device__ __forceinline__ void read(int i, int slot, int gt, int G, float (&x)[E]) const {
        const T *s = reinterpret_cast<const T *>(mem + (size_t(stage) * INPUTS + i) * bytes) + slot * p.D;
        constexpr int VEC = Elem<T>::VEC;
#pragma unroll
        for (int j = 0; j < E; j += VEC) {
            uint4 r = make_uint4(0, 0, 0, 0);
            const int e = element<T, true>(j, gt, G);
            if (e < p.D) r = *reinterpret_cast<const uint4 *>(s + e);
            Elem<T>::unpack(r, x + j);
        }
    }
    __device__ __forceinline__ void release() {          // everybody has read: ask for the rows that come here next
        give_back_reads();
        __syncthreads();
        if (threadIdx.x == 0) issue(stage);
        if (++stage == p.stages) {
            stage = 0;
            ++turn;
        }
    }
};

template <class T, bool ALIGNED, int E>
__device__ __forceinline__ void load_weight(const void *w, int dtype, int gt, int G, int D, float missing, float (&x)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int e = element<T, ALIGNED>(i, gt, G);
        x[i] = w && e < D ? load_as_float(w, dtype, e) : missing;
    }
}

// Sum over the G threads of a row: lanes by shuffles (G <= 32: a power of two), warps through shared memory.  Two
// halves of `red` are used in turn, so one barrier a reduction suffices.
struct RowSum {
    float *red;
    int lanes, first, warps, turn;       // lanes of a warp in one sum; the row's first warp and their number (0: one warp)
    __device__ __forceinline__ RowSum(float *shared, int G) : red(shared), lanes(G < 32 ? G : 32), warps(G > 32 ? G / 32 : 0), turn(0) {
        first = warps ? int(threadIdx.x >> 5) / warps * warps : 0;
    }
    template <int N>
    __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
        for (int d = 16; d; d /= 2)
            if (d < lanes)
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] += __shfl_xor_sync(~0u, v[j], d);
        if (warps == 0) return;
        float *r = red + turn * 2 * 32;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int j = 0; j < N; ++j) r[j * 32 + (threadIdx.x >> 5)] = v[j];
        __syncthreads();
        r += first;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float s = 0.f;
            if ((warps & 7) == 0) {
                for (int w = 0; w < warps; w += 8) {
                    const float4 a = *reinterpret_cast<const float4 *>(r + j * 32 + w), b = *reinterpret_cast<const float4 *>(r + j * 32 + w + 4);
                    s += ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
                }
            } else {
                for (int w = 0; w < warps; ++w) s += r[j * 32 + w];
            }
            v[j] = s;
        }
    }
};

// The gates' values in place of the gates, and their slopes: s c with c = 1 or z, and s ((1 - s) c + 0 or 1).
// s = 1 / (1 + 2^t), t = -z log2 e, by the two approximations (2^-22 and 2^-23 of the result): two slow instructions an element,
// where the exact exponential and division took half of a kernel's time.  Past |z| = 88 it is 0 and 1.  1 - s, which would cancel
// where a gate is open, is s 2^t.
// t is off by its rounding and that of log2 e, |t| 2^-23, and 2^t by as much of itself: 2^-16 at |z| = 80.  For results of 16 bits
// that is little beside their own 2^-9 and 2^-12.  FINE, for fp32: what t is off goes onto 2^t as a factor, and the gate is within
// 10 2^-24, the slope within 24 2^-24 of its terms.
template <bool SLOPE, bool FINE, int E>
__device__ __forceinline__ void open_gates(float (&z)[E], float (&slope)[E], int act) {
    if (act == ACT_NONE) {
#pragma unroll
        for (int i = 0; i < E; ++i) slope[i] = 1.f;
        return;
    }
    constexpr float LOG2E = 1.4426950408889634f, LOG2E_LO = 1.92596299112661746e-8f, LN2 = 0.693147180559945309f;
    const bool silu = act == ACT_SILU;
    const float one = silu ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float t = z[i] * -LOG2E;
        float e, s;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
        if (FINE) {
            const float off = fmaf(z[i], -LOG2E_LO, fmaf(z[i], -LOG2E, -t));
            e = fabsf(z[i]) < 88.f ? fmaf(e, LN2 * off, e) : e;              // beyond, 2^t is infinite or nothing beside 1
        }
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
        const float c = silu ? z[i] : 1.f;
        if (SLOPE) slope[i] = s * fmaf(s * fminf(e, 3.402823466e38f), c, one);
        z[i] = s * c;
    }
}

// E = 8: up to 256 threads, three CTAs an SM; E = 16, for long rows: a thread's work outside of its elements (addresses,
// barriers, reductions) was half of all at eight.
template <class T, bool ALIGNED, bool RING, int E>
__global__ void __launch_bounds__(E == 8 ? 256 : 512, E == 8 ? 3 : 1) norm_forward_kernel(const __grid_constant__ NormParams p) {
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ __align__(16) float red[2 * 2 * 32];
    __shared__ uint64_t bar[8];
    __shared__ int gave_up;
    const int G = p.groups, slots = blockDim.x / G, gt = threadIdx.x % G, slot = threadIdx.x / G;
    const float inv_d = 1.f / float(p.D);
    RowSum row_sum(red, G);
    RowRing<T, 3> ring(p, dynamic, bar, &gave_up, slots);
    if (RING) {
        ring.src[0] = p.x; ring.src[1] = p.residual; ring.src[2] = p.gate;
        ring.stride[0] = p.x_s; ring.stride[1] = p.r_s; ring.stride[2] = p.g_s;
        ring.init();
    }
    float w[E], qw[E];                                // w: scale and post_weight in one
    load_weight<T, ALIGNED>(p.post_w, p.w_dtype, gt, G, p.D, 1.f, w);
    load_weight<T, ALIGNED>(p.scale, p.w_dtype, gt, G, p.D, p.scale_value, qw);
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] *= qw[i];
    load_weight<T, ALIGNED>(p.pre_w, p.w_dtype, gt, G, p.D, 1.f, qw);
    for (int64_t first = int64_t(blockIdx.x) * slots; first < p.rows; first += int64_t(gridDim.x) * slots) {
        const int64_t row = first + slot;
        const bool live = row < p.rows;
        float x[E] = {}, r[E] = {}, z[E] = {};
        if (RING) {
            ring.arrive();
            if (live) {
                ring.read(0, slot, gt, G, x);
                if (p.residual) ring.read(1, slot, gt, G, r);
                if (p.gate) ring.read(2, slot, gt, G, z);
            }
            ring.release();
        } else if (live) {
            load_row<T, ALIGNED>(p.x, row * p.x_s, gt, G, p.D, x);
            if (p.residual) load_row<T, ALIGNED>(p.residual, row * p.r_s, gt, G, p.D, r);
            if (p.gate) load_row<T, ALIGNED>(p.gate, row * p.g_s, gt, G, p.D, z);
        }
        float rx = 1.f;
        if (p.post_w) {
            float s[1] = {};
#pragma unroll
            for (int i = 0; i < E; ++i) s[0] += x[i] * x[i];
            row_sum(s);
            rx = rsqrtf(s[0] * inv_d + p.eps);
        }
        if (p.gate) {
            float none[E];
            open_gates<false, sizeof(T) == 4>(z, none, p.act);
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] += w[i] * (z[i] * (x[i] * rx));
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] += w[i] * (x[i] * rx);
        }
        if (live) store_row<T, ALIGNED>(p.hidden, row * p.D, gt, G, p.D, r);
        if (p.pre_w) {
            float s[1] = {};
#pragma unroll
            for (int i = 0; i < E; ++i) s[0] += r[i] * r[i];
            row_sum(s);
            const float rh = rsqrtf(s[0] * inv_d + p.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] *= rh * qw[i];
            if (live) store_row<T, ALIGNED>(p.normed, row * p.D, gt, G, p.D, r);
        }
    }
    if (RING) drain(&gave_up);
}

// With x' the normed x, z the gate's value and dh the gradient of h: sum over rows of dh z x' is the gradient of post_weight but
// for the factor scale, and that of scale but for the factor post_weight, so one sum serves both, and one product of the two
// weights the rest.  WIDE: rows whose threads have only 64 registers each.  The weights are read where they are used (from the L1 cache) and
// their gradients are summed in shared memory, by the thread that owns the element.  It spills 240 to 400 bytes a thread all the
// same, and beside the sums no ring of 16-bit rows of 8192 fits: 16384 x 8192 waits for memory (1.3 TB/s), twice the time
// that the same elements take in rows of 4096.
template <class T, bool ALIGNED, int FORM, bool RING>
__global__ void __launch_bounds__(FORM == LEAN ? 256 : FORM == WIDE_ROWS ? NORM_THREADS : NORM_NARROW, FORM == LEAN ? 3 : 1) norm_backward_kernel(const __grid_constant__ NormParams p) {
    extern __shared__ __align__(128) unsigned char dynamic[];
    float *sums = reinterpret_cast<float *>(dynamic);     // [slots][2][D] when rows share a CTA; WIDE: [2][EPT][threads]
    __shared__ __align__(16) float red[2 * 2 * 32];
    __shared__ uint64_t bar[8];
    __shared__ int gave_up;
    constexpr int EPT = 8;
    constexpr bool WIDE = FORM == WIDE_ROWS, PRE = FORM != LEAN;
    const int G = p.groups, slots = blockDim.x / G, gt = threadIdx.x % G, slot = threadIdx.x / G;
    const float inv_d = 1.f / float(p.D);
    RowSum row_sum(red, G);
    float w[EPT], qw[EPT], d_w[WIDE || !PRE ? 1 : 2][EPT] = {};         // w: scale and post_weight in one
    const auto load_w = [&] {
        load_weight<T, ALIGNED>(p.post_w, p.w_dtype, gt, G, p.D, 1.f, w);
        load_weight<T, ALIGNED>(p.scale, p.w_dtype, gt, G, p.D, p.scale_value, qw);
#pragma unroll
        for (int i = 0; i < EPT; ++i) w[i] *= qw[i];
    };
    if (!WIDE) {
        load_w();
        if (PRE) load_weight<T, ALIGNED>(p.pre_w, p.w_dtype, gt, G, p.D, 1.f, qw);
    } else if (p.partial) {
        for (int i = 0; i < 2 * EPT; ++i) sums[i * blockDim.x + threadIdx.x] = 0.f;
    }
    // the ring lies behind the sums where these are kept from the start, and in their place else
    RowRing<T, PRE ? 5 : 3> ring(p, dynamic + (WIDE && p.partial ? 2 * EPT * blockDim.x * 4 : 0), bar, &gave_up, slots);
    if (RING) {
        ring.src[0] = p.x; ring.src[1] = p.gate; ring.src[2] = p.d_hidden;
        ring.stride[0] = p.x_s; ring.stride[1] = p.g_s; ring.stride[2] = p.dh_s;
        if (PRE) {
            ring.src[PRE ? 3 : 0] = p.d_normed ? p.residual : nullptr; ring.src[PRE ? 4 : 0] = p.d_normed;
            ring.stride[PRE ? 3 : 0] = p.r_s; ring.stride[PRE ? 4 : 0] = p.dy_s;
        }
        ring.init();
    }
    const auto add = [&](int which, int i, float x) {     // post and scale, pre
        if (!WIDE) d_w[WIDE || !PRE ? 0 : which][i] += x;
        else if (p.partial) sums[(which * EPT + i) * blockDim.x + threadIdx.x] += x;
    };
    for (int64_t first = int64_t(blockIdx.x) * slots; first < p.rows; first += int64_t(gridDim.x) * slots) {
        const int64_t row = first + slot;
        const bool live = row < p.rows;
        float x[EPT] = {}, h[EPT] = {}, z[EPT] = {}, dh[EPT] = {}, dy[EPT] = {};
        if (RING) {
            ring.arrive();
            if (live) {
                ring.read(0, slot, gt, G, x);
                if (p.gate) ring.read(1, slot, gt, G, z);
                if (p.d_hidden) ring.read(2, slot, gt, G, dh);
                if (PRE && p.d_normed) {
                    if (p.residual) ring.read(3, slot, gt, G, h);
                    ring.read(4, slot, gt, G, dy);
                }
            }
            ring.release();
        } else if (live) {
            load_row<T, ALIGNED>(p.x, row * p.x_s, gt, G, p.D, x);
            if (p.gate) load_row<T, ALIGNED>(p.gate, row * p.g_s, gt, G, p.D, z);
            if (p.d_hidden) load_row<T, ALIGNED>(p.d_hidden, row * p.dh_s, gt, G, p.D, dh);
            if (PRE && p.d_normed) {
                if (p.residual) load_row<T, ALIGNED>(p.residual, row * p.r_s, gt, G, p.D, h);
                load_row<T, ALIGNED>(p.d_normed, row * p.dy_s, gt, G, p.D, dy);
            }
        }
        float rx = 1.f;
        if (p.post_w) {
            float s[1] = {};
#pragma unroll
            for (int i = 0; i < EPT; ++i) s[0] += x[i] * x[i];
            row_sum(s);
            rx = rsqrtf(s[0] * inv_d + p.eps);
        }
        float slope[EPT];
        if (p.gate) {
            open_gates<true, sizeof(T) == 4>(z, slope, p.act);                            // from here on the gate's value
        } else {
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                z[i] = 1.f;
                slope[i] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < EPT; ++i) x[i] *= rx;                         // ... and the normed x
        if (WIDE) load_w();
        if (PRE && p.d_normed) {
#pragma unroll
            for (int i = 0; i < EPT; ++i) h[i] += w[i] * (z[i] * x[i]);
            if (WIDE) load_weight<T, ALIGNED>(p.pre_w, p.w_dtype, gt, G, p.D, 1.f, qw);
            float s[2] = {};
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                s[0] += h[i] * h[i];
                s[1] += dy[i] * qw[i] * h[i];
            }
            row_sum(s);
            const float rh = rsqrtf(s[0] * inv_d + p.eps), c = s[1] * rh * rh * inv_d;
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                add(1, i, dy[i] * (h[i] * rh));
                dh[i] += rh * (dy[i] * qw[i] - h[i] * c);
            }
        }
        if (p.d_residual && live) store_row<T, ALIGNED>(p.d_residual, row * p.D, gt, G, p.D, dh);
        if (WIDE && p.d_normed) load_w();
        float s[1] = {};
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            slope[i] *= dh[i] * (x[i] * w[i]);                            // gradient of the gate
            dh[i] *= z[i];
            const float a = dh[i] * x[i];
            add(0, i, a);
            dh[i] *= w[i];                                                // gradient of the normed x
            s[0] += a * w[i];
        }
        if (p.d_gate && live) store_row<T, ALIGNED>(p.d_gate, row * p.D, gt, G, p.D, slope);
        if (p.post_w) {
            row_sum(s);
            const float c = s[0] * inv_d;
#pragma unroll
            for (int i = 0; i < EPT; ++i) dh[i] = rx * (dh[i] - x[i] * c);
        }
        if (live) store_row<T, ALIGNED>(p.d_x, row * p.D, gt, G, p.D, dh);
    }
    if (RING) drain(&gave_up);
    if (!p.partial) return;
    if (RING && slots > 1) __syncthreads();               // the sums take the ring's place
    float *to = p.partial + int64_t(blockIdx.x) * 2 * p.D;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const int e = element<T, ALIGNED>(i, gt, G);
        if (e >= p.D) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float v = WIDE ? sums[(j * EPT + i) * blockDim.x + threadIdx.x] : j == 0 || PRE ? d_w[WIDE || !PRE ? 0 : j][i] : 0.f;
            if (slots > 1) sums[(slot * 2 + j) * p.D + e] = v;
            else to[j * p.D + e] = v;
        }
    }
    if (slots > 1) {                                      // never WIDE
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * p.D; i += blockDim.x) {
            float s = 0.f;
            for (int k = 0; k < slots; ++k) s += sums[k * 2 * p.D + i];
            to[i] = s;
        }
    }
}

// Weights' gradients from the CTAs' sums: 32 columns by 32 threads a CTA, CTAs' sums added in a fixed order.
__global__ void __launch_bounds__(1024) norm_weights_kernel(const __grid_constant__ NormParams p, int parts, void *d_post, void *d_scale,
                                                            void *d_pre) {
    __shared__ float s[32][33];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, col = blockIdx.x * 32 + cx, which = blockIdx.y;
    if (which == 0 ? !d_post && !d_scale : !d_pre) return;
    float a = 0.f;
    if (col < p.D)
        for (int r = ry; r < parts; r += 32) a += p.partial[(int64_t(r) * 2 + which) * p.D + col];
    s[ry][cx] = a;
    __syncthreads();
    if (ry == 0 && col < p.D) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) t += s[r][cx];
        if (which == 1) store_from_float(d_pre, p.w_dtype, col, t);
        else {
            if (d_post) store_from_float(d_post, p.w_dtype, col, t * (p.scale ? load_as_float(p.scale, p.w_dtype, col) : p.scale_value));
            if (d_scale) store_from_float(d_scale, p.w_dtype, col, t * (p.post_w ? load_as_float(p.post_w, p.w_dtype, col) : 1.f));
        }
    }
}

// Threads of a row: E elements each; below a warp a power of two, so that several rows share one.
static void norm_shape(int D, int E, int *groups, int *threads) {
    int need = (D + E - 1) / E, g = 1;
    if (need <= 32) {
        while (g < need) g *= 2;
    } else {
        g = (need + 31) / 32 * 32;
    }
    *groups = g;
    *threads = g >= 256 ? g : 256 / g * g;
}

// CTAs: what the SMs hold at once by registers (128 a thread, 80 in the forward of short rows); every CTA walks rows with
// its weights in registers.
static int norm_grid(int64_t rows, int groups, int threads, int sms, bool short_forward) {
    const int64_t slots = threads / groups, need = (rows + slots - 1) / slots;
    const int per_sm = (short_forward ? 768 : 512) / threads;
    const int64_t most = int64_t(sms) * (per_sm > 1 ? per_sm : 1);
    return static_cast<int>(need < most ? need : most);
}

static int norm_device(int *sms) {
    static std::atomic<int> counts[64];
    int dev = 0, n = 0, major = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ASCAN_ERR_DEVICE;
    if (dev >= 0 && dev < 64 && (n = counts[dev].load(std::memory_order_relaxed)) > 0) {
        *sms = n;
        return ASCAN_OK;
    }
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return ASCAN_ERR_DEVICE;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) return ASCAN_ERR_DEVICE;
    if (major != 10 || n < 1) return ASCAN_ERR_DEVICE;
    if (dev >= 0 && dev < 64) counts[dev].store(n, std::memory_order_relaxed);
    *sms = n;
    return ASCAN_OK;
}

// The backward without a gradient of `normed` needs neither residual nor the weights and sums of the second norm: 80 registers
// a thread and, for rows of one CTA of 256 threads, three CTAs an SM (262144
// heads of 128, bf16: 85 us, 101 in the general form).
static bool lean(const NormParams &p) { return !p.d_normed && p.D <= 1024; }

// Stages of the ring: at most four, in what two CTAs of an SM share (the long rows' kernels, one or two CTAs an SM) or
// three; none where two do not fit, or where no CTA comes to a second turn.  `kept`: bytes of the sums that live beside it.
static int ring_stages(const NormParams &p, int inputs, int slots, int grid, bool short_forward, size_t size, size_t kept) {
    const size_t buffer = size_t(inputs) * slots * p.D * size, room = short_forward ? 68 * 1024 : 104 * 1024;
    if (p.rows <= int64_t(grid) * slots) return 0;
    int n = 4;
    while (n > 1 && kept + n * buffer > room) --n;
    if (n == 1 && !short_forward && kept + 2 * buffer <= 216 * 1024) n = 2;
    return n > 1 ? n : 0;
}

template <class K>
static int launch_norm(K kernel, const NormParams &p, int grid, int threads, size_t smem, cudaStream_t st) {
    if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
        return ASCAN_ERR_LAUNCH;
    kernel<<<grid, threads, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

template <class T, bool ALIGNED, int FORM>
static int launch_back(NormParams p, int grid, int threads, cudaStream_t st) {
    constexpr bool WIDE = FORM == WIDE_ROWS;
    const int slots = threads / p.groups;
    size_t sums = 0;
    if (p.partial) sums = WIDE ? size_t(2) * 8 * threads * 4 : slots > 1 ? size_t(slots) * 2 * p.D * 4 : 0;   // at most 64 KB
    p.stages = ALIGNED ? ring_stages(p, FORM == LEAN ? 3 : 5, slots, grid, FORM == LEAN, sizeof(T), WIDE ? sums : 0) : 0;
    const size_t ring = size_t(p.stages) * (FORM == LEAN ? 3 : 5) * slots * p.D * sizeof(T);
    const size_t smem = WIDE ? sums + ring : sums > ring ? sums : ring;
    if (ALIGNED && p.stages) return launch_norm(norm_backward_kernel<T, ALIGNED, FORM, ALIGNED>, p, grid, threads, smem, st);
    return launch_norm(norm_backward_kernel<T, ALIGNED, FORM, false>, p, grid, threads, smem, st);
}

template <class T, bool ALIGNED, int E>
static int launch_fore(NormParams p, int grid, int threads, cudaStream_t st) {
    const int slots = threads / p.groups;
    p.stages = ALIGNED ? ring_stages(p, 3, slots, grid, E == 8, sizeof(T), 0) : 0;
    const size_t smem = size_t(p.stages) * 3 * slots * p.D * sizeof(T);
    if (ALIGNED && p.stages) return launch_norm(norm_forward_kernel<T, ALIGNED, ALIGNED, E>, p, grid, threads, smem, st);
    return launch_norm(norm_forward_kernel<T, ALIGNED, false, E>, p, grid, threads, smem, st);
}

template <class T>
static int launch_type(const NormParams &p, int grid, int threads, bool aligned, bool backward, cudaStream_t st) {
    if (backward) {
        if (threads > NORM_NARROW)
            return aligned ? launch_back<T, true, WIDE_ROWS>(p, grid, threads, st) : launch_back<T, false, WIDE_ROWS>(p, grid, threads, st);
        if (lean(p)) return aligned ? launch_back<T, true, LEAN>(p, grid, threads, st) : launch_back<T, false, LEAN>(p, grid, threads, st);
        return aligned ? launch_back<T, true, MIDDLE>(p, grid, threads, st) : launch_back<T, false, MIDDLE>(p, grid, threads, st);
    }
    if (p.D > 1024) return aligned ? launch_fore<T, true, 16>(p, grid, threads, st) : launch_fore<T, false, 16>(p, grid, threads, st);
    return aligned ? launch_fore<T, true, 8>(p, grid, threads, st) : launch_fore<T, false, 8>(p, grid, threads, st);
}

static int launch_norm_by_type(const NormParams &p, int dtype, int grid, int threads, bool aligned, bool backward, cudaStream_t st) {
    if (dtype == ASCAN_F32) return launch_type<float>(p, grid, threads, aligned, backward, st);
    if (dtype == ASCAN_BF16) return launch_type<bf16>(p, grid, threads, aligned, backward, st);
    return launch_type<__half>(p, grid, threads, aligned, backward, st);
}

static int norm_fill(const ascan_norm *a, NormParams &p, bool *aligned) {
    if (!a || a->rows < 0 || a->dim < 1 || a->activation < 0 || a->activation > 2) return ASCAN_ERR_INVALID_ARG;
    if (!(a->dtype == ASCAN_F32 || a->dtype == ASCAN_BF16 || a->dtype == ASCAN_F16)) return ASCAN_ERR_INVALID_ARG;
    if (!(a->weights_dtype == a->dtype || a->weights_dtype == ASCAN_F32)) return ASCAN_ERR_INVALID_ARG;
    if (a->dim > NORM_MAX_D) return ASCAN_ERR_UNSUPPORTED;
    p.rows = a->rows;
    p.D = a->dim;
    p.x_s = a->x_stride;
    p.r_s = a->residual_stride;
    p.g_s = a->gate_stride;
    p.w_dtype = a->weights_dtype;
    p.act = a->activation;
    p.eps = a->eps;
    p.scale_value = a->scale_value;
    p.x = a->x;
    p.residual = a->residual;
    p.gate = a->gate;
    p.post_w = a->post_weight;
    p.scale = a->scale;
    p.pre_w = a->pre_weight;
    p.status = a->status;
    const int vec = a->dtype == ASCAN_F32 ? 4 : 8;
    const auto ok = [&](const void *q, int64_t s) { return !q || ((reinterpret_cast<uintptr_t>(q) & 15) == 0 && s % vec == 0); };
    *aligned = a->dim % vec == 0 && ok(p.x, p.x_s) && ok(p.residual, p.r_s) && ok(p.gate, p.g_s);
    return ASCAN_OK;
}

static bool on16(const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

}  // namespace ascan

using namespace ascan;

extern "C" {

int ascan_norm_forward(const ascan_norm *a, void *hidden, void *normed, void *stream) {
    NormParams p = {};
    bool aligned = false;
    int rc = norm_fill(a, p, &aligned);
    if (rc != ASCAN_OK) return rc;
    if (a->rows == 0) return ASCAN_OK;
    if (!p.x || !hidden || (p.pre_w && !normed)) return ASCAN_ERR_INVALID_ARG;
    p.hidden = hidden;
    p.normed = normed;
    aligned = aligned && on16(hidden) && on16(normed);
    int sms = 0, threads;
    if ((rc = norm_device(&sms)) != ASCAN_OK) return rc;
    norm_shape(p.D, p.D > 1024 ? 16 : 8, &p.groups, &threads);
    return launch_norm_by_type(p, a->dtype, norm_grid(p.rows, p.groups, threads, sms, p.D <= 1024), threads, aligned, false,
                       static_cast<cudaStream_t>(stream));
}

size_t ascan_norm_backward_bytes(const ascan_norm *a) {
    NormParams p = {};
    bool aligned = false;
    int sms = 148, threads;
    if (norm_fill(a, p, &aligned) != ASCAN_OK) return 0;
    if (norm_device(&sms) != ASCAN_OK) {
        cudaGetLastError();
        sms = 148;          // no device to ask: size for a full B200
    }
    norm_shape(p.D, 8, &p.groups, &threads);
    return size_t(norm_grid(p.rows, p.groups, threads, sms, p.D <= 1024)) * 2 * p.D * 4;
}

int ascan_norm_backward(const ascan_norm *a, const void *d_hidden, int64_t d_hidden_stride, const void *d_normed, int64_t d_normed_stride,
                        void *d_x, void *d_residual, void *d_gate, void *d_post_weight, void *d_scale, void *d_pre_weight, void *ws,
                        size_t ws_bytes, void *stream) {
    NormParams p = {};
    bool aligned = false;
    int rc = norm_fill(a, p, &aligned);
    if (rc != ASCAN_OK) return rc;
    if (a->rows > 0 && (!p.x || !d_x || (d_normed && !p.pre_w))) return ASCAN_ERR_INVALID_ARG;
    const bool weights = d_post_weight || d_scale || d_pre_weight;
    if (weights && a->rows > 0 && (!ws || !on16(ws) || ws_bytes < ascan_norm_backward_bytes(a))) return ASCAN_ERR_WORKSPACE;
    p.d_hidden = d_hidden;
    p.d_normed = d_normed;
    p.dh_s = d_hidden_stride;
    p.dy_s = d_normed_stride;
    p.d_x = d_x;
    p.d_residual = d_residual;
    p.d_gate = d_gate;
    p.partial = weights ? static_cast<float *>(ws) : nullptr;
    const int vec = a->dtype == ASCAN_F32 ? 4 : 8;
    aligned = aligned && on16(d_hidden) && on16(d_normed) && on16(d_x) && on16(d_residual) && on16(d_gate) &&
              (!d_hidden || d_hidden_stride % vec == 0) && (!d_normed || d_normed_stride % vec == 0);
    int sms = 0, threads;
    if ((rc = norm_device(&sms)) != ASCAN_OK) return rc;
    norm_shape(p.D, 8, &p.groups, &threads);
    const int grid = norm_grid(p.rows, p.groups, threads, sms, lean(p));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.rows > 0 && (rc = launch_norm_by_type(p, a->dtype, grid, threads, aligned, true, st)) != ASCAN_OK) return rc;
    if (weights) {         // without rows: zeros
        norm_weights_kernel<<<dim3((p.D + 31) / 32, 2), 1024, 0, st>>>(p, p.rows > 0 ? grid : 0, d_post_weight, d_scale, d_pre_weight);
        if (cudaGetLastError() != cudaSuccess) return ASCAN_ERR_LAUNCH;
    }
    return ASCAN_OK;
}

}  // extern "C"
