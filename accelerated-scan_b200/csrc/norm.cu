// Norms before and after a block, with its gate and residual scale, in one pass over the rows:
//     n = x rsqrt(mean x^2 + eps) post_weight          (x itself without post_weight)
//     h = residual + scale act(gate) n
//     y = h rsqrt(mean h^2 + eps) pre_weight
// and its gradients.  Everything is bound by memory: the forward reads x, residual and gate and writes h and y, the
// backward reads x, residual, gate and the two gradients and writes three; a row stays in registers between its
// reductions.  The backward recomputes h from the inputs (the same bytes as reading a saved one), so that no sum sees a
// rounded h.  A thread holds eight neighbouring elements, 16 bytes at a time;
// G threads share a row, and a CTA keeps the weights, and in the backward the weights' gradients, in registers over all
// its rows.  Sums of the weights' gradients over CTAs are a second launch, in a fixed order.
#include <atomic>

#include "delta_common.cuh"

namespace ascan {

struct NormParams {
    int64_t rows, x_s, r_s, g_s, dh_s, dy_s;        // rows; elements from row to row
    int32_t D, w_dtype, act, groups;                // groups: threads of a row, G
    float eps, scale_value;
    const void *x, *residual, *gate, *post_w, *scale, *pre_w;
    void *hidden, *normed;
    const void *d_hidden, *d_normed;
    void *d_x, *d_residual, *d_gate;
    float *partial;                                 // [grid][3][D]: post, scale, pre
};

constexpr int EPT = 8;                              // elements a thread holds
constexpr int NORM_THREADS = 1024, NORM_MAX_D = EPT * NORM_THREADS;
constexpr int NORM_NARROW = 512;                    // threads up to which the backward keeps all it needs in registers

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

// Where a thread's elements lie in a row: EPT neighbours (ALIGNED), or every G-th element.
template <bool ALIGNED>
__device__ __forceinline__ int element(int i, int gt, int G) { return ALIGNED ? gt * EPT + i : gt + i * G; }

template <class T, bool ALIGNED>
__device__ __forceinline__ void load_row(const void *src, int64_t at, int gt, int G, int D, float (&x)[EPT]) {
    const T *s = static_cast<const T *>(src) + at;
    if (ALIGNED) {
        constexpr int VEC = Elem<T>::VEC;
#pragma unroll
        for (int i = 0; i < EPT; i += VEC) {
            uint4 r = make_uint4(0, 0, 0, 0);
            if (gt * EPT + i < D) r = __ldcs(reinterpret_cast<const uint4 *>(s + gt * EPT + i));
            Elem<T>::unpack(r, x + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < EPT; ++i) x[i] = gt + i * G < D ? Elem<T>::get(s[gt + i * G]) : 0.f;
    }
}

template <class T, bool ALIGNED>
__device__ __forceinline__ void store_row(void *dst, int64_t at, int gt, int G, int D, const float (&x)[EPT]) {
    T *s = static_cast<T *>(dst) + at;
    if (ALIGNED) {
        constexpr int VEC = Elem<T>::VEC;
#pragma unroll
        for (int i = 0; i < EPT; i += VEC)
            if (gt * EPT + i < D) *reinterpret_cast<uint4 *>(s + gt * EPT + i) = Elem<T>::pack(x + i);
    } else {
#pragma unroll
        for (int i = 0; i < EPT; ++i)
            if (gt + i * G < D) s[gt + i * G] = Elem<T>::put(x[i]);
    }
}

template <bool ALIGNED>
__device__ __forceinline__ void load_weight(const void *w, int dtype, int gt, int G, int D, float missing, float (&x)[EPT]) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const int e = element<ALIGNED>(i, gt, G);
        x[i] = w && e < D ? load_as_float(w, dtype, e) : missing;
    }
}

// Sum over the G threads of a row: lanes by shuffles (G <= 32: a power of two), warps through shared memory.  Two
// halves of `red` are used in turn, so one barrier a reduction suffices.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int G, int warps, float *red, int &turn) {
    const int top = G < 32 ? G : 32;
#pragma unroll
    for (int j = 0; j < N; ++j)
        for (int d = top / 2; d; d /= 2) v[j] += __shfl_xor_sync(~0u, v[j], d);
    if (G <= 32) return;
    const int warp = threadIdx.x >> 5, first = warp / (G / 32) * (G / 32);
    float *r = red + turn * 2 * 32;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int j = 0; j < N; ++j) r[j * 32 + warp] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float s = 0.f;
        for (int w = 0; w < G / 32; ++w) s += r[j * 32 + first + w];
        v[j] = s;
    }
}

__device__ __forceinline__ float gate_value(float z, int act, float &slope) {
    if (act == ACT_NONE) {
        slope = 1.f;
        return z;
    }
    const float s = 1.f / (1.f + expf(-z));
    if (act == ACT_SIGMOID) {
        slope = s * (1.f - s);
        return s;
    }
    slope = s * (1.f + z * (1.f - s));
    return z * s;
}

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(NORM_THREADS) norm_forward_kernel(NormParams p) {
    __shared__ float red[2 * 2 * 32];
    const int G = p.groups, slots = blockDim.x / G, gt = threadIdx.x % G, slot = threadIdx.x / G;
    const float inv_d = 1.f / float(p.D);
    int turn = 0;
    float pw[EPT], sc[EPT], qw[EPT];
    load_weight<ALIGNED>(p.post_w, p.w_dtype, gt, G, p.D, 1.f, pw);
    load_weight<ALIGNED>(p.scale, p.w_dtype, gt, G, p.D, p.scale_value, sc);
    load_weight<ALIGNED>(p.pre_w, p.w_dtype, gt, G, p.D, 1.f, qw);
    for (int64_t first = int64_t(blockIdx.x) * slots; first < p.rows; first += int64_t(gridDim.x) * slots) {
        const int64_t row = first + slot;
        const bool live = row < p.rows;
        float x[EPT] = {}, r[EPT] = {}, z[EPT] = {};
        if (live) {
            load_row<T, ALIGNED>(p.x, row * p.x_s, gt, G, p.D, x);
            if (p.residual) load_row<T, ALIGNED>(p.residual, row * p.r_s, gt, G, p.D, r);
            if (p.gate) load_row<T, ALIGNED>(p.gate, row * p.g_s, gt, G, p.D, z);
        }
        float rx = 1.f;
        if (p.post_w) {
            float s[1] = {};
#pragma unroll
            for (int i = 0; i < EPT; ++i) s[0] += x[i] * x[i];
            row_sum(s, G, blockDim.x / 32, red, turn);
            rx = rsqrtf(s[0] * inv_d + p.eps);
        }
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            float slope, a = 1.f;
            if (p.gate) a = gate_value(z[i], p.act, slope);
            r[i] += sc[i] * (a * (x[i] * rx * pw[i]));
        }
        if (live) store_row<T, ALIGNED>(p.hidden, row * p.D, gt, G, p.D, r);
        if (p.pre_w) {
            float s[1] = {};
#pragma unroll
            for (int i = 0; i < EPT; ++i) s[0] += r[i] * r[i];
            row_sum(s, G, blockDim.x / 32, red, turn);
            const float rh = rsqrtf(s[0] * inv_d + p.eps);
#pragma unroll
            for (int i = 0; i < EPT; ++i) r[i] *= rh * qw[i];
            if (live) store_row<T, ALIGNED>(p.normed, row * p.D, gt, G, p.D, r);
        }
    }
}

// WIDE: rows whose threads have only 64 registers each.  The weights are read where they are used (from the L1 cache) and
// their gradients are summed in shared memory, by the thread that owns the element.
template <class T, bool ALIGNED, bool WIDE>
__global__ void __launch_bounds__(WIDE ? NORM_THREADS : NORM_NARROW) norm_backward_kernel(NormParams p) {
    extern __shared__ float sums[];                       // [slots][3][D] when rows share a CTA; WIDE: [3][EPT][threads]
    __shared__ float red[2 * 2 * 32];
    const int G = p.groups, slots = blockDim.x / G, gt = threadIdx.x % G, slot = threadIdx.x / G;
    const float inv_d = 1.f / float(p.D);
    int turn = 0;
    float pw[EPT], sc[EPT], qw[EPT], d_w[WIDE ? 1 : 3][EPT] = {};
    if (!WIDE) {
        load_weight<ALIGNED>(p.post_w, p.w_dtype, gt, G, p.D, 1.f, pw);
        load_weight<ALIGNED>(p.scale, p.w_dtype, gt, G, p.D, p.scale_value, sc);
        load_weight<ALIGNED>(p.pre_w, p.w_dtype, gt, G, p.D, 1.f, qw);
    } else if (p.partial) {
        for (int i = 0; i < 3 * EPT; ++i) sums[i * blockDim.x + threadIdx.x] = 0.f;
    }
    const auto add = [&](int which, int i, float x) {     // post, scale, pre
        if (!WIDE) d_w[WIDE ? 0 : which][i] += x;
        else if (p.partial) sums[(which * EPT + i) * blockDim.x + threadIdx.x] += x;
    };
    for (int64_t first = int64_t(blockIdx.x) * slots; first < p.rows; first += int64_t(gridDim.x) * slots) {
        const int64_t row = first + slot;
        const bool live = row < p.rows;
        float x[EPT] = {}, h[EPT] = {}, z[EPT] = {}, dh[EPT] = {}, dy[EPT] = {};
        if (live) {
            load_row<T, ALIGNED>(p.x, row * p.x_s, gt, G, p.D, x);
            if (p.residual) load_row<T, ALIGNED>(p.residual, row * p.r_s, gt, G, p.D, h);
            if (p.gate) load_row<T, ALIGNED>(p.gate, row * p.g_s, gt, G, p.D, z);
            if (p.d_hidden) load_row<T, ALIGNED>(p.d_hidden, row * p.dh_s, gt, G, p.D, dh);
            if (p.d_normed) load_row<T, ALIGNED>(p.d_normed, row * p.dy_s, gt, G, p.D, dy);
        }
        float rx = 1.f;
        if (p.post_w) {
            float s[1] = {};
#pragma unroll
            for (int i = 0; i < EPT; ++i) s[0] += x[i] * x[i];
            row_sum(s, G, blockDim.x / 32, red, turn);
            rx = rsqrtf(s[0] * inv_d + p.eps);
        }
        if (WIDE) {
            load_weight<ALIGNED>(p.post_w, p.w_dtype, gt, G, p.D, 1.f, pw);
            load_weight<ALIGNED>(p.scale, p.w_dtype, gt, G, p.D, p.scale_value, sc);
        }
        float slope[EPT];
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            slope[i] = 0.f;
            z[i] = p.gate ? gate_value(z[i], p.act, slope[i]) : 1.f;      // from here on the gate's value
            x[i] *= rx;                                                   // ... and the normed x
            h[i] += sc[i] * (z[i] * (x[i] * pw[i]));
        }
        if (p.d_normed) {
            if (WIDE) load_weight<ALIGNED>(p.pre_w, p.w_dtype, gt, G, p.D, 1.f, qw);
            float s[2] = {};
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                s[0] += h[i] * h[i];
                s[1] += dy[i] * qw[i] * h[i];
            }
            row_sum(s, G, blockDim.x / 32, red, turn);
            const float rh = rsqrtf(s[0] * inv_d + p.eps), c = s[1] * rh * rh * inv_d;
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                add(2, i, dy[i] * (h[i] * rh));
                dh[i] += rh * (dy[i] * qw[i] - h[i] * c);
            }
        }
        if (p.d_residual && live) store_row<T, ALIGNED>(p.d_residual, row * p.D, gt, G, p.D, dh);
        if (WIDE) {
            load_weight<ALIGNED>(p.post_w, p.w_dtype, gt, G, p.D, 1.f, pw);
            load_weight<ALIGNED>(p.scale, p.w_dtype, gt, G, p.D, p.scale_value, sc);
        }
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const float n = x[i] * pw[i];
            add(1, i, dh[i] * (z[i] * n));
            slope[i] *= dh[i] * sc[i] * n;                                // gradient of the gate
            dh[i] *= sc[i] * z[i];                                        // gradient of n
        }
        if (p.d_gate && live) store_row<T, ALIGNED>(p.d_gate, row * p.D, gt, G, p.D, slope);
        if (p.post_w) {
            float s[1] = {};
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                add(0, i, dh[i] * x[i]);
                dh[i] *= pw[i];
                s[0] += dh[i] * x[i];
            }
            row_sum(s, G, blockDim.x / 32, red, turn);
            const float c = s[0] * inv_d;
#pragma unroll
            for (int i = 0; i < EPT; ++i) dh[i] = rx * (dh[i] - x[i] * c);
        }
        if (live) store_row<T, ALIGNED>(p.d_x, row * p.D, gt, G, p.D, dh);
    }
    if (!p.partial) return;
    float *to = p.partial + int64_t(blockIdx.x) * 3 * p.D;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const int e = element<ALIGNED>(i, gt, G);
        if (e >= p.D) continue;
#pragma unroll
        for (int w = 0; w < 3; ++w) {
            const float v = WIDE ? sums[(w * EPT + i) * blockDim.x + threadIdx.x] : d_w[WIDE ? 0 : w][i];
            if (slots > 1) sums[(slot * 3 + w) * p.D + e] = v;
            else to[w * p.D + e] = v;
        }
    }
    if (slots > 1) {                                      // never WIDE
        __syncthreads();
        for (int i = threadIdx.x; i < 3 * p.D; i += blockDim.x) {
            float s = 0.f;
            for (int k = 0; k < slots; ++k) s += sums[k * 3 * p.D + i];
            to[i] = s;
        }
    }
}

// Weights' gradients from the CTAs' sums: 32 columns by 32 threads a CTA, CTAs' sums added in a fixed order.
__global__ void __launch_bounds__(1024) norm_weights_kernel(const float *partial, int parts, int D, int w_dtype, void *d_post, void *d_scale,
                                                            void *d_pre) {
    __shared__ float s[32][33];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, col = blockIdx.x * 32 + cx, which = blockIdx.y;
    void *dst = which == 0 ? d_post : which == 1 ? d_scale : d_pre;
    if (!dst) return;
    float a = 0.f;
    if (col < D)
        for (int r = ry; r < parts; r += 32) a += partial[(int64_t(r) * 3 + which) * D + col];
    s[ry][cx] = a;
    __syncthreads();
    if (ry == 0 && col < D) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) t += s[r][cx];
        store_from_float(dst, w_dtype, col, t);
    }
}

// Threads of a row: eight elements each; below a warp a power of two, so that several rows share one.
static void norm_shape(int D, int *groups, int *threads) {
    int need = (D + EPT - 1) / EPT, g = 1;
    if (need <= 32) {
        while (g < need) g *= 2;
    } else {
        g = (need + 31) / 32 * 32;
    }
    *groups = g;
    *threads = g >= 256 ? g : 256 / g * g;
}

// CTAs: what the SMs hold at once by registers (128 a thread in the backward, 64 in the forward); every CTA walks rows
// with its weights in registers.
static int norm_grid(int64_t rows, int groups, int threads, int sms, bool backward) {
    const int64_t slots = threads / groups, need = (rows + slots - 1) / slots;
    const int per_sm = (backward ? NORM_NARROW : 1024) / threads;
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

template <class T, bool ALIGNED, bool WIDE>
static int launch_norm_back(const NormParams &p, int grid, int threads, cudaStream_t st) {
    const int slots = threads / p.groups;
    size_t smem = 0;
    if (p.partial) smem = WIDE ? size_t(3) * EPT * threads * 4 : slots > 1 ? size_t(slots) * 3 * p.D * 4 : 0;   // at most 96 KB
    if (WIDE && cudaFuncSetAttribute(norm_backward_kernel<T, ALIGNED, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     3 * EPT * NORM_THREADS * 4) != cudaSuccess)
        return ASCAN_ERR_LAUNCH;
    norm_backward_kernel<T, ALIGNED, WIDE><<<grid, threads, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

template <class T, bool ALIGNED>
static int launch_norm_kernel(const NormParams &p, int grid, int threads, bool backward, cudaStream_t st) {
    if (backward)
        return threads > NORM_NARROW ? launch_norm_back<T, ALIGNED, true>(p, grid, threads, st)
                                     : launch_norm_back<T, ALIGNED, false>(p, grid, threads, st);
    norm_forward_kernel<T, ALIGNED><<<grid, threads, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

template <class T>
static int launch_norm_type(const NormParams &p, int grid, int threads, bool aligned, bool backward, cudaStream_t st) {
    return aligned ? launch_norm_kernel<T, true>(p, grid, threads, backward, st)
                   : launch_norm_kernel<T, false>(p, grid, threads, backward, st);
}

static int launch_norm(const NormParams &p, int dtype, int grid, int threads, bool aligned, bool backward, cudaStream_t st) {
    if (dtype == ASCAN_F32) return launch_norm_type<float>(p, grid, threads, aligned, backward, st);
    if (dtype == ASCAN_BF16) return launch_norm_type<bf16>(p, grid, threads, aligned, backward, st);
    return launch_norm_type<__half>(p, grid, threads, aligned, backward, st);
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
    norm_shape(p.D, &p.groups, &threads);
    return launch_norm(p, a->dtype, norm_grid(p.rows, p.groups, threads, sms, false), threads, aligned, false,
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
    norm_shape(p.D, &p.groups, &threads);
    return size_t(norm_grid(p.rows, p.groups, threads, sms, true)) * 3 * p.D * 4;
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
    norm_shape(p.D, &p.groups, &threads);
    const int grid = norm_grid(p.rows, p.groups, threads, sms, true);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.rows > 0 && (rc = launch_norm(p, a->dtype, grid, threads, aligned, true, st)) != ASCAN_OK) return rc;
    if (weights) {         // without rows: zeros
        norm_weights_kernel<<<dim3((p.D + 31) / 32, 3), 1024, 0, st>>>(p.partial, p.rows > 0 ? grid : 0, p.D, p.w_dtype, d_post_weight,
                                                                       d_scale, d_pre_weight);
        if (cudaGetLastError() != cudaSuccess) return ASCAN_ERR_LAUNCH;
    }
    return ASCAN_OK;
}

}  // extern "C"
