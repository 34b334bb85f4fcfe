// Gated delta rule: problem description shared by the host entry points and the kernels.
//
// Per sequence and head a K x V state S (fp32) is carried from token to token:
//     S' = e^g S;   e = v - S'^T k;   u = beta e;   S = S' + k u^T;   out = scale S^T q.
// Sequences are cut into chunks of 64 tokens.  With G the running sum of g in a chunk, gam_i = e^{G_i},
// Gam_ij = e^{G_i - G_j}, L = strictly lower part of Gam * K K^T and M = L (I + diag(beta) L)^{-1}:
//     x = V - gam (K S0);   e = x - M (beta x);   u = beta e
//     out = scale gam (Q S0) + P u,   P = scale * lower part of Gam * Q K^T
//     S1 = gam_C S0 + K^T (Gam_C u)
// M carries no factor beta on either side, so nothing is divided by beta and beta = 0 is an ordinary value.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/ascan_b200.h"

namespace ascan {

constexpr int DELTA_CHUNK = 64;
// per chunk and head: gam, Gam_C, beta, the running sum of g as two floats, zero gates so far
enum : int { SC_GAM = 0, SC_GAMC = 1, SC_BETA = 2, SC_GHI = 3, SC_GLO = 4, SC_RESET = 5, SC_ARRAYS = 6 };

// A (batch, token, head, d) array as one or two bf16 planes whose sum is the value: what the matrix
// instructions read.  bf16 inputs with 16-byte aligned rows are their own plane.
struct Planes {
    const __nv_bfloat16 *p;
    int64_t plane, sb, st, sh;      // elements from one plane / batch row / token / head to the next
};

struct DeltaParams {
    int64_t batch, T;
    int32_t n_seqs, packed, starts64, slots;     // packed: batch == 1, n_seqs sequences given by starts
    int32_t chunks;                              // chunks of a row when not packed
    int32_t Hk, H, K, V, Kp, Vp;                 // Kp, Vp: extents of the planes' rows (multiples of 8)
    int32_t dtype, g_dtype, b_dtype;
    float scale;
    const void *starts;
    Planes q, k, v, d_out;
    const void *g, *b;
    int64_t g_s[3], b_s[3];
    const float *s0;
    void *out;
    float *s1;
    // scratch
    __nv_bfloat16 *M, *P;            // [slot][H][2][64][64]
    float *sc;                       // [slot][H][SC_ARRAYS][64]
    __nv_bfloat16 *S, *e;            // saved for the backward: [slot][H][terms][Vp][KP] (bf16: one term) and [slot][H][2][Vp][64]
    // backward
    __nv_bfloat16 *dS, *z;           // as S and e
    int *done;                       // two tickets, and [slot][H]: slices of V that the sweep has finished
    const float *d_s1;
    float *d_s0;
    void *d_q, *d_k, *d_v, *d_g, *d_b;
    int *status;                     // nullable, host memory: set when a bounded wait expired
};

int delta_launch_pack(const void *src, int dtype, const int64_t *strides, int64_t batch, int64_t T, int heads, int d,
                      int dp, __nv_bfloat16 *dst, int64_t plane, cudaStream_t st);
int delta_launch_prep(const DeltaParams &p, cudaStream_t st);
int delta_launch_sweep(const DeltaParams &p, bool save, int sm_count, cudaStream_t st);
int delta_launch_sweep_tc(const DeltaParams &p, bool save, cudaStream_t st);
int delta_launch_backward_tc(const DeltaParams &p, int sm_count, cudaStream_t st);
int delta_launch_back_sweep(const DeltaParams &p, int sm_count, cudaStream_t st);
int delta_launch_zero_outside(const DeltaParams &p, cudaStream_t st);
int delta_launch_grads(const DeltaParams &p, cudaStream_t st);

}  // namespace ascan
