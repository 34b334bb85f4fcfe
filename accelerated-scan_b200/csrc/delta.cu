// extern "C" entry points of the gated delta rule (declared in include/ascan_b200.h): argument checks, scratch layout,
// launches; and the kernel of single tokens.
#include <atomic>

#include "delta_tc.cuh"

namespace ascan {

static int delta_sm_count(int *out) {
    static std::atomic<int> counts[64];
    int dev = 0, n = 0, major = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ASCAN_ERR_DEVICE;
    if (dev >= 0 && dev < 64 && (n = counts[dev].load(std::memory_order_relaxed)) > 0) {
        *out = n;
        return ASCAN_OK;
    }
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return ASCAN_ERR_DEVICE;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) return ASCAN_ERR_DEVICE;
    if (major != 10 || n < 1) return ASCAN_ERR_DEVICE;
    if (dev >= 0 && dev < 64) counts[dev].store(n, std::memory_order_relaxed);
    *out = n;
    return ASCAN_OK;
}

static bool real_dtype(int d) { return d == ASCAN_F32 || d == ASCAN_BF16 || d == ASCAN_F16; }
static int round_up8(int x) { return (x + 7) & ~7; }

static int check_shape(const ascan_delta *a) {
    if (!a) return ASCAN_ERR_INVALID_ARG;
    if (a->batch < 0 || a->seqlen < 0 || a->heads < 1 || a->heads_k < 1 || a->heads % a->heads_k != 0) return ASCAN_ERR_INVALID_ARG;
    if (a->k_dim < 1 || a->v_dim < 1 || !real_dtype(a->dtype)) return ASCAN_ERR_INVALID_ARG;
    if (!(a->log_gates_dtype == a->dtype || a->log_gates_dtype == ASCAN_F32)) return ASCAN_ERR_INVALID_ARG;
    if (!(a->betas_dtype == a->dtype || a->betas_dtype == ASCAN_F32)) return ASCAN_ERR_INVALID_ARG;
    if (a->n_seqs < 0 || (a->n_seqs > 0 && a->batch != 1)) return ASCAN_ERR_INVALID_ARG;
    if (a->k_dim > 128 || a->v_dim > 1024 || a->heads > 65535) return ASCAN_ERR_UNSUPPORTED;
    const int64_t slots = a->n_seqs ? a->seqlen / DELTA_CHUNK + a->n_seqs : a->batch * ((a->seqlen + 63) / DELTA_CHUNK);
    const int64_t chains = (a->n_seqs ? a->n_seqs : a->batch) * int64_t(a->heads) * ((a->v_dim + 15) / 16);
    if (slots > 0x3fffffff / a->heads || chains > 0x7fffffff || a->seqlen > (int64_t(1) << 30)) return ASCAN_ERR_UNSUPPORTED;
    return ASCAN_OK;
}

static int terms(int dtype) { return dtype == ASCAN_BF16 ? 1 : 2; }

// bf16 rows that 16-byte copies and tensor maps can take as they are
static bool is_plane(const ascan_delta *a, const void *p, const int64_t *s, int heads, int d) {
    if (a->dtype != ASCAN_BF16 || d % 8 != 0 || (reinterpret_cast<uintptr_t>(p) & 15)) return false;
    const int64_t sizes[3] = {a->batch, a->seqlen, heads};
    for (int i = 0; i < 3; ++i)
        if (s[i] % 8 != 0 || (sizes[i] > 1 && (s[i] <= 0 || s[i] >= int64_t(1) << 38))) return false;
    return true;
}

struct Bump {          // 256-byte aligned pieces of one buffer
    unsigned char *base;
    size_t used = 0;
    template <class T>
    T *take(int64_t n) {
        unsigned char *p = base ? base + used : nullptr;
        used += (size_t(n) * sizeof(T) + 255) & ~size_t(255);
        return reinterpret_cast<T *>(p);
    }
};

struct PackJob {
    const void *src;
    const int64_t *strides;
    int heads, d, dp;
    Planes *to;
    int64_t plane;
};

static Planes user_plane(const void *p, const int64_t *s) {
    return Planes{static_cast<const __nv_bfloat16 *>(p), 0, s[0], s[1], s[2]};
}

static void take_copy(const ascan_delta *a, int heads, int d, Planes *to, Bump &bump) {
    const int dp = round_up8(d);
    const int64_t plane = a->batch * a->seqlen * heads * dp;
    __nv_bfloat16 *dst = bump.take<__nv_bfloat16>(plane * terms(a->dtype));
    *to = Planes{dst, terms(a->dtype) == 2 ? plane : 0, a->seqlen * heads * dp, int64_t(heads) * dp, dp};
}

static void plan_pack(const ascan_delta *a, const void *src, const int64_t *strides, int heads, int d, Planes *to, Bump &bump,
                      PackJob *jobs, int *n) {
    if (is_plane(a, src, strides, heads, d)) {
        *to = user_plane(src, strides);
        return;
    }
    take_copy(a, heads, d, to, bump);
    jobs[(*n)++] = PackJob{src, strides, heads, d, round_up8(d), to, a->batch * a->seqlen * heads * round_up8(d)};
}

static int run_packs(const ascan_delta *a, const PackJob *jobs, int n, cudaStream_t st) {
    for (int i = 0; i < n; ++i) {
        const PackJob &j = jobs[i];
        int rc = delta_launch_pack(j.src, a->dtype, j.strides, a->batch, a->seqlen, j.heads, j.d, j.dp,
                                   const_cast<__nv_bfloat16 *>(j.to->p), j.to->plane, st);
        if (rc != ASCAN_OK) return rc;
    }
    return ASCAN_OK;
}

static void take_chunks(DeltaParams &p, Bump &bump) {
    const int64_t each = int64_t(p.slots) * p.H;
    p.M = bump.take<__nv_bfloat16>(each * 2 * 4096);
    p.P = bump.take<__nv_bfloat16>(each * 2 * 4096);
}

static void fill(const ascan_delta *a, DeltaParams &p) {
    p.batch = a->batch;
    p.T = a->seqlen;
    p.packed = a->n_seqs > 0;
    p.n_seqs = p.packed ? a->n_seqs : int32_t(a->batch);
    p.starts = a->seq_starts;
    p.starts64 = a->seq_starts_64;
    p.chunks = int32_t((a->seqlen + 63) / DELTA_CHUNK);
    p.slots = p.packed ? int32_t(a->seqlen / DELTA_CHUNK + a->n_seqs) : int32_t(a->batch * p.chunks);
    p.Hk = a->heads_k;
    p.H = a->heads;
    p.K = a->k_dim;
    p.V = a->v_dim;
    p.Kp = round_up8(a->k_dim);
    p.Vp = round_up8(a->v_dim);
    p.dtype = a->dtype;
    p.g_dtype = a->log_gates_dtype;
    p.b_dtype = a->betas_dtype;
    p.scale = a->scale;
    p.g = a->log_gates;
    p.b = a->betas;
    for (int i = 0; i < 3; ++i) {
        p.g_s[i] = a->log_gates_stride[i];
        p.b_s[i] = a->betas_stride[i];
    }
    p.s0 = a->initial_state;
    p.status = a->status;
}

// What the backward reads again comes first, at places that only sizes and types decide: the inputs may come to the backward
// with other strides, and then other ones of them are planes of their own.
static void take_kept(const ascan_delta *a, DeltaParams &p, Bump &bump, bool keep) {
    const int64_t each = int64_t(p.slots) * p.H;
    p.sc = bump.take<float>(each * SC_ARRAYS * 64);
    if (keep) {
        const int nt = terms(a->dtype), kp = p.Kp <= 64 ? 64 : 128;
        p.S = bump.take<__nv_bfloat16>(each * nt * p.Vp * kp);
        p.e = bump.take<__nv_bfloat16>(each * 2 * 64 * p.Vp);
    }
}

struct Input {
    const void *src;
    const int64_t *strides;
    int heads, d;
    Planes *to;
};
static void list_inputs(const ascan_delta *a, DeltaParams &p, Input (&in)[3]) {
    in[0] = Input{a->queries, a->queries_stride, a->heads_k, a->k_dim, &p.q};
    in[1] = Input{a->keys, a->keys_stride, a->heads_k, a->k_dim, &p.k};
    in[2] = Input{a->values, a->values_stride, a->heads, a->v_dim, &p.v};
}
static void plan_inputs(const ascan_delta *a, DeltaParams &p, Bump &bump, PackJob *jobs, int *n) {
    Input in[3];
    list_inputs(a, p, in);
    for (const Input &x : in) plan_pack(a, x.src, x.strides, x.heads, x.d, x.to, bump, jobs, n);
}
// The backward's: copies that the forward has left behind what it kept, new ones of what it read as it was and is no plane now.
static void plan_inputs_again(const ascan_delta *a, DeltaParams &p, Bump &kept, Bump &bump, PackJob *jobs, int *n) {
    Input in[3];
    list_inputs(a, p, in);
    for (int i = 0; i < 3; ++i) {
        if (a->kept_packed >> i & 1) take_copy(a, in[i].heads, in[i].d, in[i].to, kept);
        else plan_pack(a, in[i].src, in[i].strides, in[i].heads, in[i].d, in[i].to, bump, jobs, n);
    }
}

static bool tensor_core_path(const ascan_delta *a) { return a->dtype == ASCAN_BF16; }

static void fill_back(const ascan_delta *a, DeltaParams &p, Bump &bump, const void *d_out, const int64_t *d_out_stride, PackJob *jobs,
                      int *n_jobs) {
    const int64_t each = int64_t(p.slots) * p.H;
    const int nt = terms(a->dtype), kp = p.Kp <= 64 ? 64 : 128;
    p.dS = bump.take<__nv_bfloat16>(each * nt * p.Vp * kp);
    p.z = bump.take<__nv_bfloat16>(each * 2 * 64 * p.Vp);
    if (tensor_core_path(a)) p.done = bump.take<int>(2 + each);
    else take_chunks(p, bump);
    plan_pack(a, d_out, d_out_stride, a->heads, a->v_dim, &p.d_out, bump, jobs, n_jobs);
}

// ---- one token -------------------------------------------------------------------------------------------------------
//
// x = S'^T k and y = S'^T q are both sums over the old state, and S^T q = y + (k . q) u, so the state is read once, kept
// in registers across one reduction, and written once: 8 bytes per state element are all the traffic there is.  A CTA
// of 256 threads takes 32 columns; a thread holds up to 4 rows of 4 columns (VEC = 4) or 16 rows of one column.  32 states of
// 128 x 128 (one request): 3.9 us, the latency of a read, a reduction and a write.

struct StepParams {
    const void *q, *k, *v, *g, *b;
    int64_t q_s[2], k_s[2], v_s[2], g_s[2], b_s[2];       // row of the batch, head
    float *state;
    int64_t slot_stride, pool;
    const void *slots;
    int32_t slots64, batch, Hk, H, K, V, dtype, g_dtype, b_dtype;
    float scale;
    void *out;
};

__device__ __forceinline__ int64_t read_slot(const StepParams &p, int b) {
    if (!p.slots) return b;
    return p.slots64 ? static_cast<const int64_t *>(p.slots)[b] : static_cast<const int32_t *>(p.slots)[b];
}

template <int VEC>
__global__ void __launch_bounds__(256) delta_step_kernel(StepParams p) {
    constexpr int LANES = 32 / VEC, GROUPS = 256 / LANES, ROWS = 128 / GROUPS;      // ROWS of K a thread holds
    __shared__ float sk[128], sq[128], part[8][2][32], skq[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slices = (p.V + 31) / 32, slice = blockIdx.x % slices, h = blockIdx.x / slices % p.H;
    const int b = blockIdx.x / slices / p.H, hk = h / (p.H / p.Hk);
    const int v0 = slice * 32 + (tid % LANES) * VEC, r0 = tid / LANES;
    const int64_t slot = read_slot(p, b);
    const bool inside = slot >= 0 && slot < p.pool;
    float *state = p.state + (inside ? slot : 0) * p.slot_stride + int64_t(h) * p.K * p.V;

    float s[ROWS][VEC];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int k = r0 + i * GROUPS;
        if (VEC == 4) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (inside && k < p.K && v0 < p.V) x = __ldcs(reinterpret_cast<const float4 *>(state + int64_t(k) * p.V + v0));
            s[i][VEC - 1] = x.w;
            s[i][VEC / 2] = x.z;
            s[i][VEC / 4] = x.y;
            s[i][0] = x.x;
        } else {
            s[i][0] = inside && k < p.K && v0 < p.V ? __ldcs(state + int64_t(k) * p.V + v0) : 0.f;
        }
    }
    bool again = false;             // an earlier row of the batch has this slot
    if (p.slots && inside)
        for (int i = tid; i < b; i += 256) again |= read_slot(p, i) == slot;
    float kq = 0.f;
    if (tid < 128) {
        const float kv = tid < p.K ? load_as_float(p.k, p.dtype, b * p.k_s[0] + hk * p.k_s[1] + tid) : 0.f;
        const float qv = tid < p.K ? load_as_float(p.q, p.dtype, b * p.q_s[0] + hk * p.q_s[1] + tid) : 0.f;
        sk[tid] = kv;
        sq[tid] = qv;
        kq = kv * qv;
    }
#pragma unroll
    for (int d = 16; d; d /= 2) kq += __shfl_xor_sync(~0u, kq, d);
    if (lane == 0) skq[warp] = kq;
    const float decay = expf(load_as_float(p.g, p.g_dtype, b * p.g_s[0] + h * p.g_s[1]));
    const float beta = load_as_float(p.b, p.b_dtype, b * p.b_s[0] + h * p.b_s[1]);
    again = __syncthreads_or(again);
    const bool live = inside && !again;

    float x[VEC] = {}, y[VEC] = {};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int k = r0 + i * GROUPS;
        const float kv = sk[k], qv = sq[k];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            s[i][j] *= decay;
            x[j] += kv * s[i][j];
            y[j] += qv * s[i][j];
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
#pragma unroll
        for (int d = LANES; d < 32; d *= 2) {
            x[j] += __shfl_xor_sync(~0u, x[j], d);
            y[j] += __shfl_xor_sync(~0u, y[j], d);
        }
        if (lane < LANES) {
            part[warp][0][lane * VEC + j] = x[j];
            part[warp][1][lane * VEC + j] = y[j];
        }
    }
    __syncthreads();
    const float dot = (skq[0] + skq[1]) + (skq[2] + skq[3]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int col = (tid % LANES) * VEC + j;
        float xs = 0.f, ys = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            xs += part[w][0][col];
            ys += part[w][1][col];
        }
        const int v = v0 + j;
        const float val = v < p.V ? load_as_float(p.v, p.dtype, b * p.v_s[0] + h * p.v_s[1] + v) : 0.f;
        const float u = beta * (val - xs);
        x[j] = u;
        if (r0 == 0 && v < p.V) {
            // a padded row (slot < 0) answers zeros; a slot behind the pool or taken by an earlier row answers NaN
            const float o = live ? p.scale * (ys + dot * u) : (slot < 0 ? 0.f : __int_as_float(0x7fc00000));
            store_from_float(p.out, p.dtype, (int64_t(b) * p.H + h) * p.V + v, o);
        }
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int k = r0 + i * GROUPS;
        if (k >= p.K || v0 >= p.V) continue;
        const float kv = sk[k];
        if (VEC == 4) {
            const float4 o = make_float4(s[i][0] + kv * x[0], s[i][VEC / 4] + kv * x[VEC / 4], s[i][VEC / 2] + kv * x[VEC / 2],
                                         s[i][VEC - 1] + kv * x[VEC - 1]);
            __stcs(reinterpret_cast<float4 *>(state + int64_t(k) * p.V + v0), o);
        } else {
            __stcs(state + int64_t(k) * p.V + v0, s[i][0] + kv * x[0]);
        }
    }
}

// The same for many rows: a head's K x V state is one dense block, so a persistent CTA takes it by one bulk copy into a
// ring of shared-memory buffers, updates it there and sends it back by another, while the next ones arrive and the next
// token's vectors are on their way to registers.  The kernel above asks for nothing while it reduces.  A warp takes 32
// columns and every 4 N-th row, four rows at a time.  128 requests of 32 heads of 128 x 128: 97 us, 5.5 TB/s of state
// (0.84 of what a plain copy reaches).
constexpr int STEP_THREADS = 512, STEP_MAX_STAGES = 6, STEP_MAX_BATCH = 1024;

struct StepRing {
    int32_t stages, items;           // items: rows of the batch times heads
    uint32_t bytes;                  // of a state
    int *status;
};

__device__ __forceinline__ uint32_t load_raw(const void *p, int dtype, int64_t i) {
    return dtype == ASCAN_F32 ? static_cast<const uint32_t *>(p)[i] : static_cast<const uint16_t *>(p)[i];
}
__device__ __forceinline__ float raw_value(uint32_t x, int dtype) {
    if (dtype == ASCAN_F32) return __uint_as_float(x);
    return dtype == ASCAN_BF16 ? __uint_as_float(x << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(x)));
}

__global__ void __launch_bounds__(STEP_THREADS, 1) delta_step_ring_kernel(const __grid_constant__ StepParams p, StepRing ring) {
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ float sk[128], sq[128], part_dot[4];
    __shared__ __align__(16) float sums[2][16][32];      // [x, y][warp][column of its 32]
    __shared__ uint64_t bars[STEP_MAX_STAGES];
    __shared__ int slots[STEP_MAX_BATCH];                // -1: padded; -2: no such slot, or an earlier row has it
    __shared__ int dead_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nv = p.V / 4, blocks = (nv + 7) / 8, block = warp % blocks, teams = 16 / blocks, team = warp / blocks;
    const int cv = block * 8 + (lane & 7), row0 = team * 4 + (lane >> 3), rows = teams * 4;
    const bool works = team < teams && cv < nv;
    const uint32_t base = smem_addr(dynamic), bar0 = smem_addr(bars);
    const Waiter wait = {&dead_flag, ring.status};
    if (tid == 0) {
        dead_flag = 0;
        for (int i = 0; i < ring.stages; ++i) mbar_init(bar0 + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_proxy();
    }
    for (int b = tid; b < p.batch; b += STEP_THREADS) {
        const int64_t slot = read_slot(p, b);
        slots[b] = slot < 0 ? -1 : slot >= p.pool ? -2 : static_cast<int>(slot);
    }
    __syncthreads();
    int taken[STEP_MAX_BATCH / STEP_THREADS] = {};
#pragma unroll
    for (int j = 0; j < STEP_MAX_BATCH / STEP_THREADS; ++j) {
        const int b = tid + j * STEP_THREADS;
        if (p.slots && b < p.batch && slots[b] >= 0)
            for (int i = 0; i < b; ++i) taken[j] |= slots[i] == slots[b];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < STEP_MAX_BATCH / STEP_THREADS; ++j)
        if (taken[j]) slots[tid + j * STEP_THREADS] = -2;
    __syncthreads();

    const auto state_of = [&](int item) { return p.state + slots[item / p.H] * p.slot_stride + int64_t(item % p.H) * p.K * p.V; };
    const auto ask = [&](int item, int stage) {          // one thread
        const uint32_t bar = bar0 + 8 * stage;
        if (slots[item / p.H] < 0) {
            mbar_arrive(bar);
            return;
        }
        mbar_expect(bar, ring.bytes);
        asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     :: "r"(base + stage * ring.bytes), "l"(state_of(item)), "r"(ring.bytes), "r"(bar) : "memory");
    };
    uint32_t rk = 0, rq = 0, rv[4] = {}, rg = 0, rb = 0;
    const auto fetch = [&](int item) {                   // a token's vectors, as they are: a conversion would wait for them
        const int b = item / p.H, h = item % p.H, hk = h / (p.H / p.Hk);
        if (tid < p.K) {
            rk = load_raw(p.k, p.dtype, b * p.k_s[0] + hk * p.k_s[1] + tid);
            rq = load_raw(p.q, p.dtype, b * p.q_s[0] + hk * p.q_s[1] + tid);
        }
        rg = load_raw(p.g, p.g_dtype, b * p.g_s[0] + h * p.g_s[1]);
        rb = load_raw(p.b, p.b_dtype, b * p.b_s[0] + h * p.b_s[1]);
        if (works)
#pragma unroll
            for (int j = 0; j < 4; ++j) rv[j] = load_raw(p.v, p.dtype, b * p.v_s[0] + h * p.v_s[1] + 4 * cv + j);
    };
    // one buffer less than there are is asked for ahead: the last one's way back ends while the next item is worked on
    const int ahead = ring.stages - 1;
    if (tid == 0)
        for (int i = 0; i < ahead; ++i)
            if (int(blockIdx.x) + i * int(gridDim.x) < ring.items) ask(blockIdx.x + i * gridDim.x, i);
    if (int(blockIdx.x) < ring.items) fetch(blockIdx.x);
    int stage = 0, turn = 0;
    for (int item = blockIdx.x; item < ring.items; item += gridDim.x) {
        const int b = item / p.H, h = item % p.H, slot = slots[b];
        if (tid < 128) {
            const float kv = tid < p.K ? raw_value(rk, p.dtype) : 0.f, qv = tid < p.K ? raw_value(rq, p.dtype) : 0.f;
            sk[tid] = kv;
            sq[tid] = qv;
            float kq = kv * qv;
#pragma unroll
            for (int d = 16; d; d /= 2) kq += __shfl_xor_sync(~0u, kq, d);
            if (lane == 0) part_dot[warp] = kq;
        }
        const float decay = expf(raw_value(rg, p.g_dtype)), beta = raw_value(rb, p.b_dtype);
        float val[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) val[j] = raw_value(rv[j], p.dtype);
        if (item + int64_t(gridDim.x) < ring.items) fetch(item + gridDim.x);
        __syncthreads();
        wait(bar0 + 8 * stage, turn & 1);
        float4 *s = reinterpret_cast<float4 *>(dynamic + stage * ring.bytes) + cv;
        float x[4] = {}, y[4] = {};
        if (slot >= 0 && works) {
#pragma unroll 4
            for (int k = row0; k < p.K; k += rows) {
                const float4 v = s[k * nv];
                const float kv = sk[k], qv = sq[k];
                x[0] += kv * v.x; x[1] += kv * v.y; x[2] += kv * v.z; x[3] += kv * v.w;
                y[0] += qv * v.x; y[1] += qv * v.y; y[2] += qv * v.z; y[3] += qv * v.w;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] += __shfl_xor_sync(~0u, x[j], 8);
            y[j] += __shfl_xor_sync(~0u, y[j], 8);
            x[j] += __shfl_xor_sync(~0u, x[j], 16);
            y[j] += __shfl_xor_sync(~0u, y[j], 16);
        }
        if (lane < 8) {
            *reinterpret_cast<float4 *>(&sums[0][warp][4 * lane]) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(&sums[1][warp][4 * lane]) = make_float4(y[0], y[1], y[2], y[3]);
        }
        __syncthreads();
        if (slot >= 0 && works) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = y[j] = 0.f;
            for (int i = 0; i < teams; ++i) {
                const float4 a = *reinterpret_cast<const float4 *>(&sums[0][i * blocks + block][4 * (lane & 7)]);
                x[0] += a.x; x[1] += a.y; x[2] += a.z; x[3] += a.w;
            }
            float u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = beta * (val[j] - decay * x[j]);
            if (row0 == 0) {
                for (int i = 0; i < teams; ++i) {
                    const float4 a = *reinterpret_cast<const float4 *>(&sums[1][i * blocks + block][4 * (lane & 7)]);
                    y[0] += a.x; y[1] += a.y; y[2] += a.z; y[3] += a.w;
                }
                const float dot = (part_dot[0] + part_dot[1]) + (part_dot[2] + part_dot[3]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    store_from_float(p.out, p.dtype, (int64_t(b) * p.H + h) * p.V + 4 * cv + j, p.scale * (decay * y[j] + dot * u[j]));
            }
#pragma unroll 4
            for (int k = row0; k < p.K; k += rows) {
                float4 v = s[k * nv];
                const float kv = sk[k];
                v.x = decay * v.x + kv * u[0]; v.y = decay * v.y + kv * u[1]; v.z = decay * v.z + kv * u[2]; v.w = decay * v.w + kv * u[3];
                s[k * nv] = v;
            }
            fence_async_proxy();
        } else if (slot < 0 && works && row0 == 0) {         // as in the kernel above
            const float o = slot == -1 ? 0.f : __int_as_float(0x7fc00000);
#pragma unroll
            for (int j = 0; j < 4; ++j) store_from_float(p.out, p.dtype, (int64_t(b) * p.H + h) * p.V + 4 * cv + j, o);
        }
        __syncthreads();
        if (tid == 0) {
            if (slot >= 0)
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                             :: "l"(state_of(item)), "r"(base + stage * ring.bytes), "r"(ring.bytes) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");      // the item before this one has left its buffer
            const int64_t next = int64_t(item) + int64_t(ahead) * gridDim.x;
            if (next < ring.items) ask(static_cast<int>(next), stage == 0 ? ring.stages - 1 : stage - 1);
        }
        if (++stage == ring.stages) {
            stage = 0;
            ++turn;
        }
    }
    if (tid == 0) tma_store_done();
    drain(&dead_flag);
}

}  // namespace ascan

using namespace ascan;

extern "C" {

size_t ascan_delta_forward_bytes(const ascan_delta *a, int keep) {
    if (check_shape(a) != ASCAN_OK) return 0;
    DeltaParams p = {};
    Bump bump{nullptr};
    PackJob jobs[4];
    int n = 0;
    fill(a, p);
    take_kept(a, p, bump, keep != 0);
    plan_inputs(a, p, bump, jobs, &n);
    if (!tensor_core_path(a)) take_chunks(p, bump);
    return bump.used + 256;
}

size_t ascan_delta_backward_bytes(const ascan_delta *a, const void *d_out, const int64_t *d_out_stride) {
    if (check_shape(a) != ASCAN_OK || !d_out_stride) return 0;
    DeltaParams p = {};
    Bump bump{nullptr}, none{nullptr};
    PackJob jobs[8];
    int n = 0;
    fill(a, p);
    fill_back(a, p, bump, d_out, d_out_stride, jobs, &n);
    plan_inputs_again(a, p, none, bump, jobs, &n);
    return bump.used + 256;
}

int ascan_delta_packed(const ascan_delta *a) {
    if (check_shape(a) != ASCAN_OK) return 0;
    DeltaParams p = {};
    Input in[3];
    list_inputs(a, p, in);
    int packed = 0;
    for (int i = 0; i < 3; ++i) packed |= is_plane(a, in[i].src, in[i].strides, in[i].heads, in[i].d) ? 0 : 1 << i;
    return packed;
}

static int check_pointers(const ascan_delta *a) {
    if (a->batch * a->seqlen > 0 && !(a->queries && a->keys && a->values && a->log_gates && a->betas)) return ASCAN_ERR_INVALID_ARG;
    if (a->n_seqs > 0 && !a->seq_starts) return ASCAN_ERR_INVALID_ARG;
    return ASCAN_OK;
}

int ascan_delta_forward(const ascan_delta *a, void *out, float *final_state, int keep, void *ws, size_t ws_bytes, void *stream) {
    int rc = check_shape(a);
    if (rc != ASCAN_OK || (rc = check_pointers(a)) != ASCAN_OK) return rc;
    if (a->batch == 0) return ASCAN_OK;
    if (!final_state || (a->seqlen > 0 && !out)) return ASCAN_ERR_INVALID_ARG;
    if (!ws || (reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < ascan_delta_forward_bytes(a, keep)) return ASCAN_ERR_WORKSPACE;
    int sms = 0;
    if ((rc = delta_sm_count(&sms)) != ASCAN_OK) return rc;
    DeltaParams p = {};
    Bump bump{static_cast<unsigned char *>(ws)};
    PackJob jobs[4];
    int n = 0;
    fill(a, p);
    take_kept(a, p, bump, keep != 0);
    plan_inputs(a, p, bump, jobs, &n);
    if (!tensor_core_path(a)) take_chunks(p, bump);
    p.out = out;
    p.s1 = final_state;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if ((rc = run_packs(a, jobs, n, st)) != ASCAN_OK) return rc;
    if (tensor_core_path(a)) return delta_launch_sweep_tc(p, keep != 0, st);
    if ((rc = delta_launch_prep(p, st)) != ASCAN_OK) return rc;
    return delta_launch_sweep(p, keep != 0, sms, st);
}

int ascan_delta_backward(const ascan_delta *a, const void *d_out, const int64_t *d_out_stride, const float *d_final_state,
                         void *d_queries, void *d_keys, void *d_values, void *d_log_gates, void *d_betas, float *d_initial_state,
                         void *kept, size_t kept_bytes, void *ws, size_t ws_bytes, void *stream) {
    int rc = check_shape(a);
    if (rc != ASCAN_OK || (rc = check_pointers(a)) != ASCAN_OK) return rc;
    if (a->batch == 0) return ASCAN_OK;
    if (!d_out_stride) return ASCAN_ERR_INVALID_ARG;
    if (a->seqlen > 0 && !(d_out && d_queries && d_keys && d_values && d_log_gates && d_betas)) return ASCAN_ERR_INVALID_ARG;
    if (!kept || (reinterpret_cast<uintptr_t>(kept) & 255)) return ASCAN_ERR_WORKSPACE;
    if (!ws || (reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < ascan_delta_backward_bytes(a, d_out, d_out_stride))
        return ASCAN_ERR_WORKSPACE;
    int sms = 0;
    if ((rc = delta_sm_count(&sms)) != ASCAN_OK) return rc;
    DeltaParams p = {};
    Bump saved{static_cast<unsigned char *>(kept)}, bump{static_cast<unsigned char *>(ws)};
    PackJob jobs[8];
    int n = 0;
    fill(a, p);
    take_kept(a, p, saved, true);
    fill_back(a, p, bump, d_out, d_out_stride, jobs, &n);
    plan_inputs_again(a, p, saved, bump, jobs, &n);
    if (kept_bytes < saved.used) return ASCAN_ERR_WORKSPACE;
    p.d_s1 = d_final_state;
    p.d_s0 = d_initial_state;
    p.d_q = d_queries;
    p.d_k = d_keys;
    p.d_v = d_values;
    p.d_g = d_log_gates;
    p.d_b = d_betas;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if ((rc = run_packs(a, jobs, n, st)) != ASCAN_OK) return rc;
    if ((rc = delta_launch_zero_outside(p, st)) != ASCAN_OK) return rc;
    if (tensor_core_path(a)) return delta_launch_backward_tc(p, sms, st);
    if ((rc = delta_launch_prep(p, st)) != ASCAN_OK) return rc;
    if ((rc = delta_launch_back_sweep(p, sms, st)) != ASCAN_OK) return rc;
    return delta_launch_grads(p, st);
}

int ascan_delta_step(const ascan_delta_token *a, void *out, float *state, int64_t pool, int64_t slot_stride, const void *slots,
                     int slots_64, void *stream) {
    if (!a || a->batch < 0 || a->heads < 1 || a->heads_k < 1 || a->heads % a->heads_k != 0 || a->k_dim < 1 || a->v_dim < 1 ||
        !real_dtype(a->dtype) || pool < 0)
        return ASCAN_ERR_INVALID_ARG;
    if (!(a->log_gates_dtype == a->dtype || a->log_gates_dtype == ASCAN_F32)) return ASCAN_ERR_INVALID_ARG;
    if (!(a->betas_dtype == a->dtype || a->betas_dtype == ASCAN_F32)) return ASCAN_ERR_INVALID_ARG;
    if (a->k_dim > 128) return ASCAN_ERR_UNSUPPORTED;
    if (a->batch == 0) return ASCAN_OK;
    if (!a->queries || !a->keys || !a->values || !a->log_gates || !a->betas || !out || (!state && pool > 0)) return ASCAN_ERR_INVALID_ARG;
    if (!slots && pool < a->batch) return ASCAN_ERR_INVALID_ARG;
    const int64_t inner = int64_t(a->heads) * a->k_dim * a->v_dim;
    if (slot_stride < inner) return ASCAN_ERR_INVALID_ARG;
    const int64_t grid = a->batch * a->heads * ((int64_t(a->v_dim) + 31) / 32);
    if (grid > 0x7fffffff || a->batch > 0x7fffffff) return ASCAN_ERR_UNSUPPORTED;
    StepParams p = {};
    p.q = a->queries; p.k = a->keys; p.v = a->values; p.g = a->log_gates; p.b = a->betas;
    for (int i = 0; i < 2; ++i) {
        p.q_s[i] = a->queries_stride[i];
        p.k_s[i] = a->keys_stride[i];
        p.v_s[i] = a->values_stride[i];
        p.g_s[i] = a->log_gates_stride[i];
        p.b_s[i] = a->betas_stride[i];
    }
    p.state = state;
    p.slot_stride = slot_stride;
    p.pool = pool;
    p.slots = slots;
    p.slots64 = slots_64;
    p.batch = int32_t(a->batch);
    p.Hk = a->heads_k; p.H = a->heads; p.K = a->k_dim; p.V = a->v_dim;
    p.dtype = a->dtype; p.g_dtype = a->log_gates_dtype; p.b_dtype = a->betas_dtype;
    p.scale = a->scale;
    p.out = out;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // 16-byte accesses need rows of the state that start on 16 bytes; the ring needs states of which three fit into shared
    // memory.  Its price is a state's, that of the other kernel a CTA's, one per 32 columns: it pays from three CTAs a state
    // and three states an SM on.  us, ring and split: 4096 states of 128 x 128 98 and 130, 640 of them 22.8 and 24.1, 448 18.1
    // and 17.4, 128 8.1 and 6.9; 4096 of 64 x 256 96 and 221, of 128 x 96 91 and 100, of 128 x 64 87 and 67.
    const bool aligned = p.V % 4 == 0 && slot_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0;
    int sms = 0;
    const int rc = delta_sm_count(&sms);
    if (rc != ASCAN_OK) return rc;
    const int64_t items = a->batch * a->heads, bytes = int64_t(p.K) * p.V * 4;
    if (aligned && p.V <= 512 && bytes <= 65536 && a->batch <= STEP_MAX_BATCH && pool <= 0x7fffffff && p.V > 64 && items >= 3 * sms) {
        int stages = static_cast<int>(200 * 1024 / bytes);
        if (stages > STEP_MAX_STAGES) stages = STEP_MAX_STAGES;
        const StepRing ring = {stages, static_cast<int32_t>(items), static_cast<uint32_t>(bytes), a->status};
        const int smem = static_cast<int>(stages * bytes);
        if (cudaFuncSetAttribute(delta_step_ring_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess)
            return ASCAN_ERR_LAUNCH;
        delta_step_ring_kernel<<<sms, STEP_THREADS, smem, st>>>(p, ring);
    } else if (aligned)
        delta_step_kernel<4><<<unsigned(grid), 256, 0, st>>>(p);
    else
        delta_step_kernel<1><<<unsigned(grid), 256, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? ASCAN_OK : ASCAN_ERR_LAUNCH;
}

}  // extern "C"
