// Norms around a block, shared by blocknorm.hip (forward) and blocknorm_bwd.hip:
//     x' = residual_scale x + branch_scale g N1(y),    h = N2(x')
// N = RMSNorm (t r w, r = 1 / sqrt(mean t^2 + eps)) or LayerNorm ((t - m) r w + b).  Bound: HBM bytes -- x, y in and x', h out once
// forward (x, y, dx', dh in and dx, dy out backward), everything between in registers.
//
// One row belongs to TPR threads, each with NV vectors of V channels: 16 lanes at <= 128 channels, a wave up to 1024, 256 threads
// up to 4096, 512 up to 8192 (V = 8, 16-byte loads); channel counts that are no multiple of 8, and pointers that are not 16-byte
// aligned, take V = 1.  A workgroup has R such row groups and walks its rows with the weights in registers.
#pragma once
#include "token_common.h"

struct NormArgs {
    const void *x, *y;
    const float *w1, *b1, *w2, *b2;      // post / pre weights and biases, or null
    const void* gate;                    // [T / gate_rows][C] or null
    int gate_f32;                        // gate type: fp32, else y's
    long long gate_rows;                 // tokens that share a row of the gate
    float bs, rs, eps;
    long long T;
    int C, rows_per_wg;
    void *xo, *h;                        // forward outputs (xo null without y, h null without w2)
    float* stats;                        // [T][4]: m1, r1, m2, r2 (forward: written, or null; backward: read)
    const void *dxo, *dh;                // backward inputs (either may be null)
    void *dx, *dy;
    float* part;                         // backward: [workgroup][sums][C] partial column sums
    int want;                            // backward: bit q = sum q is written (w1, b1, w2, b2, gate)
    void* dgate;                         // backward, gate of every token: its gradient, in the gate's type
};

// sums over the TPR threads of a row group.  TPR > 64: one barrier a call, two LDS slots in turn (the barrier of call n + 1 is after
// every thread's read of call n, so call n + 2 may reuse its slot).
template <int TPR, int R, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* lds, int& slot) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o, 64);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        float* s = lds + slot * (R * W * 2);
        slot ^= 1;
        const int g = threadIdx.x / TPR, w = (threadIdx.x % TPR) / 64;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) s[(g * W + w) * 2 + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) t += s[(g * W + i) * 2 + k];
            v[k] = t;
        }
    }
}

#define NORM_TYPES(TABLE, LAUNCH)                                                                         \
    do {                                                                                                  \
        if (x_type == TCVOM_TYPE_F32 && y_type == TCVOM_TYPE_F32) TABLE(float, float, LAUNCH);            \
        else if (x_type == TCVOM_TYPE_F32 && y_type == TCVOM_TYPE_BF16) TABLE(float, __bf16, LAUNCH);     \
        else if (x_type == TCVOM_TYPE_F32 && y_type == TCVOM_TYPE_F16) TABLE(float, _Float16, LAUNCH);    \
        else if (x_type == TCVOM_TYPE_BF16) TABLE(__bf16, __bf16, LAUNCH);                                \
        else TABLE(_Float16, _Float16, LAUNCH);                                                           \
    } while (0)

static inline bool norm_types_ok(int x_type, int y_type) {
    return (x_type == y_type && x_type >= TCVOM_TYPE_F32 && x_type <= TCVOM_TYPE_F16) ||
           (x_type == TCVOM_TYPE_F32 && (y_type == TCVOM_TYPE_BF16 || y_type == TCVOM_TYPE_F16));
}

