// Norms around a block, shared by blocknorm.hip (forward) and blocknorm_bwd.hip:
//     x' = residual_scale x + branch_scale g N1(y),    h = N2(x')
// N = RMSNorm (t r w, r = 1 / sqrt(mean t^2 + eps)) or LayerNorm ((t - m) r w + b).  Bound: HBM bytes -- x, y in and x', h out once
// forward (x, y, dx', dh in and dx, dy out backward), everything between in registers.  8192 rows of 4096, bf16: forward 50 us = 5.3 TB/s,
// backward 80 us = 5.0 TB/s + 4.0 us for the column sums (a copy reaches 5.1), all fp32: 100 and 166 us, the same rates; 8160 rows of 512, fp32 x
// and bf16 y: 13 us = 3.8 TB/s and 17 us = 4.4 TB/s + 5.2 us; 4 rows of 4096: 3.9 us, a launch.  Channels just above a step of the launch tables
// leave lanes idle: 131072 rows of 128 bf16 24 and 37 us (5.6 TB/s), of 136 52 and 74 us (2.8), of 256 75 and 82 us (3.6 and 4.9); 32768 rows of 512
// 24 and 37 us, of 520 28 and 49 us (4.9 and 4.2).
//
// One row belongs to TPR threads, each with NV vectors of 8 channels: 16 lanes at <= 128 channels, up to 512 threads at 8192.  A
// workgroup has R such row groups and walks its rows with the weights in registers.  TAIL: the channels are no multiple of 8; rows
// then start at any address, which 16-byte accesses allow, and the last vector of a row is moved element by element.
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

constexpr int V = 8;                     // channels a vector
// vector at channel c of a row of C channels at p, zeros past the end
template <class T, bool TAIL>
__device__ __forceinline__ typename RawVec<T, V>::type row_load(const T* p, int c, int C) {
    return !TAIL || c + V <= C ? load_raw<T, V>(p + c) : load_first<T, V>(p + c, C - c);
}
template <class T, bool TAIL>
__device__ __forceinline__ void row_load_f(const T* p, int c, int C, float (&f)[V]) { raw_to_float<T, V>(row_load<T, TAIL>(p, c, C), f); }
template <class T, bool TAIL>
__device__ __forceinline__ void row_store(T* p, int c, int C, const float (&f)[V]) {
    if (!TAIL || c + V <= C) store_vec<T, V>(p + c, f);
    else store_first<T, V>(p + c, f, C - c);
}

// sums over 16 lanes and over a wave, in every lane, on the vector unit (a shuffle through LDS takes over 100 cycles a stage, and a row of
// the backward waits for 12 of them)
__device__ __forceinline__ float row_sum(float v) {
    v += H16_DPP(v, 0xB1);                  // lane ^ 1
    v += H16_DPP(v, 0x4E);                  // lane ^ 2
    v += H16_DPP(v, 0x124);                 // row_ror:4
    return v + H16_DPP(v, 0x128);           // row_ror:8
}
__device__ __forceinline__ float full_sum(float v) {
    v = row_sum(v);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// sums over the TPR threads of a row group.  TPR > 64: one barrier a call, two LDS slots in turn (the barrier of call n + 1 is after
// every thread's read of call n, so call n + 2 may reuse its slot).
template <int TPR, int R, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* lds, int& slot) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = TPR == 16 ? row_sum(v[k]) : full_sum(v[k]);
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

// element types and the form of a launch table
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

