// Forward of the norms around a block (blocknorm.h), reached through tcvom_block_norm_fwd.
#include "blocknorm.h"

template <class TX, class TY, int TPR, int R, int NV, bool TAIL, bool LAYER>
__global__ __launch_bounds__(TPR * R) void block_norm_fwd_kernel(NormArgs a) {
    __shared__ float lds[TPR > 64 ? 4 * R * (TPR / 64) : 1];
    int slot = 0;
    const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const int C = a.C;
    const float inv = 1.f / (float)C;
    const bool has_y = a.y != nullptr, post = a.w1 != nullptr, pre = a.w2 != nullptr;
    float w1[NV][V], b1[NV][V], w2[NV][V], b2[NV][V], gt[NV][V];
    bool in[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int c = (n * TPR + lane) * V;
        in[n] = c < C;
#pragma unroll
        for (int j = 0; j < V; ++j) { w1[n][j] = !TAIL || c + j < C ? 1.f : 0.f; b1[n][j] = 0.f; w2[n][j] = 1.f; b2[n][j] = 0.f; gt[n][j] = 1.f; }
        if (!in[n]) continue;
        if (post) row_load_f<float, TAIL>(a.w1, c, C, w1[n]);
        if (LAYER && post && a.b1) row_load_f<float, TAIL>(a.b1, c, C, b1[n]);
        if (pre) row_load_f<float, TAIL>(a.w2, c, C, w2[n]);
        if (LAYER && pre && a.b2) row_load_f<float, TAIL>(a.b2, c, C, b2[n]);
    }
    long long grow = -1;
    const long long r0 = (long long)blockIdx.x * a.rows_per_wg;
    for (int k = 0; k < a.rows_per_wg; k += R) {             // every thread runs every round: the reductions hold barriers
        const long long row = r0 + k + g;
        const bool live = k + g < a.rows_per_wg && row < a.T;
        float x[NV][V], y[NV][V];
        const long long base = row * C;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * TPR + lane) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) x[n][j] = y[n][j] = 0.f;
            if (live && in[n]) {
                row_load_f<TX, TAIL>((const TX*)a.x + base, c, C, x[n]);
                if (has_y) row_load_f<TY, TAIL>((const TY*)a.y + base, c, C, y[n]);
            }
        }
        if (a.gate && live && row / a.gate_rows != grow) {
            grow = row / a.gate_rows;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int c = (n * TPR + lane) * V;
                if (!in[n]) continue;
                if (a.gate_f32) row_load_f<float, TAIL>((const float*)a.gate + grow * C, c, C, gt[n]);
                else row_load_f<TY, TAIL>((const TY*)a.gate + grow * C, c, C, gt[n]);
            }
        }
        float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
        auto moments = [&](const float (&t)[NV][V], float& m, float& r) {
            float s[1] = {0.f};
            if (LAYER) {
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int j = 0; j < V; ++j) s[0] += t[n][j];
                group_sum<TPR, R, 1>(s, lds, slot);
                m = s[0] * inv;
                s[0] = 0.f;
            }
#pragma unroll
            for (int n = 0; n < NV; ++n)
                if (in[n])
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float d = t[n][j] - (LAYER ? m : 0.f);
                        if (!(TAIL && LAYER) || (n * TPR + lane) * V + j < C) s[0] += d * d;
                    }
            group_sum<TPR, R, 1>(s, lds, slot);
            r = 1.f / sqrtf(s[0] * inv + a.eps);
        };
        if (has_y) {
            if (post) moments(y, m1, r1);
#pragma unroll
            for (int n = 0; n < NV; ++n)
                if (in[n])
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        // (an absent post norm is one of weight 1 on rows of mean 0 and deviation 1)
                        const float z = (LAYER ? y[n][j] - m1 : y[n][j]) * r1;
                        const float t = LAYER ? fmaf(z, w1[n][j], b1[n][j]) : z * w1[n][j];
                        x[n][j] = fmaf(a.bs * gt[n][j], t, a.rs * x[n][j]);
                    }
        }
        if (pre) moments(x, m2, r2);
        if (!live) continue;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * TPR + lane) * V;
            if (!in[n]) continue;
            if (has_y) row_store<TX, TAIL>((TX*)a.xo + base, c, C, x[n]);
            if (pre) {
                float h[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float z = (LAYER ? x[n][j] - m2 : x[n][j]) * r2;
                    h[j] = LAYER ? fmaf(z, w2[n][j], b2[n][j]) : z * w2[n][j];
                }
                row_store<TY, TAIL>((TY*)a.h + base, c, C, h);
            }
        }
        if (a.stats && lane == 0) *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(m1, r1, m2, r2);
    }
}

// threads by channels (see blocknorm.h)
#define FWD_TABLE(TX, TY, LAUNCH)                      \
    do {                                               \
        if (C <= 128) LAUNCH(TX, TY, 16, 16, 1);       \
        else if (C <= 512) LAUNCH(TX, TY, 64, 4, 1);   \
        else if (C <= 1024) LAUNCH(TX, TY, 64, 4, 2);  \
        else if (C <= 2048) LAUNCH(TX, TY, 256, 1, 1); \
        else if (C <= 4096) LAUNCH(TX, TY, 256, 1, 2); \
        else LAUNCH(TX, TY, 512, 1, 2);                \
    } while (0)

extern "C" int tcvom_block_norm_fwd(const void* x, const void* y, const float* post_weight, const float* post_bias, const void* gate,
                                    int32_t gate_f32, int64_t gate_rows, const float* pre_weight, const float* pre_bias, float branch_scale,
                                    float residual_scale, float eps, int32_t layer, void* x_out, void* h, float* stats, int64_t T, int32_t C,
                                    int32_t x_type, int32_t y_type, void* stream) {
    TCVOM_CHECK_ARG((x || T == 0) && T >= 0 && C > 0 && C <= TCVOM_MAX_NORM_CHANNELS, "block_norm_fwd: T=%lld C=%d (1..%d)", (long long)T, C,
                    TCVOM_MAX_NORM_CHANNELS);
    TCVOM_CHECK_ARG(norm_types_ok(x_type, y_type), "block_norm_fwd: types %d, %d", x_type, y_type);
    if (T == 0) return 0;
    TCVOM_CHECK_ARG(y ? x_out != nullptr : !post_weight && !gate && pre_weight, "block_norm_fwd: outputs / weights do not match y");
    TCVOM_CHECK_ARG(!pre_weight || h, "block_norm_fwd: null h");
    TCVOM_CHECK_ARG(layer || (!post_bias && !pre_bias), "block_norm_fwd: a bias belongs to LayerNorm");
    TCVOM_CHECK_ARG(!gate || (gate_rows > 0 && T % gate_rows == 0), "block_norm_fwd: %lld tokens a gate row", (long long)gate_rows);
    TCVOM_CHECK_ARG(T < (1LL << 31), "block_norm_fwd: %lld tokens", (long long)T);
    NormArgs a = {};
    a.x = x; a.y = y; a.w1 = post_weight; a.b1 = post_bias; a.w2 = pre_weight; a.b2 = pre_bias;
    a.gate = gate; a.gate_f32 = gate_f32; a.gate_rows = gate_rows > 0 ? gate_rows : 1;
    a.bs = branch_scale; a.rs = residual_scale; a.eps = eps; a.T = T; a.C = C;
    a.xo = x_out; a.h = h; a.stats = stats;
    const hipStream_t st = (hipStream_t)stream;
#define FWD_LAUNCH(TX, TY, TPR, R, NV, TAIL)                                                                                   \
    do {                                                                                                                      \
        if (layer) hipLaunchKernelGGL((block_norm_fwd_kernel<TX, TY, TPR, R, NV, TAIL, true>), grid, dim3(TPR * R), 0, st, a);  \
        else hipLaunchKernelGGL((block_norm_fwd_kernel<TX, TY, TPR, R, NV, TAIL, false>), grid, dim3(TPR * R), 0, st, a);       \
    } while (0)
#define FWD(TX, TY, TPR, R, NV)                                           \
    do {                                                                  \
        const int wgs = 256 * (2048 / (TPR * R));                         \
        a.rows_per_wg = cdiv(cdiv(T, R), wgs) * R;                        \
        const dim3 grid(cdiv(T, a.rows_per_wg));                          \
        if (C % V) FWD_LAUNCH(TX, TY, TPR, R, NV, true);                  \
        else FWD_LAUNCH(TX, TY, TPR, R, NV, false);                       \
    } while (0)
    NORM_TYPES(FWD_TABLE, FWD);
#undef FWD
#undef FWD_LAUNCH
    TCVOM_LAUNCH_CHECK("block_norm_fwd");
    return 0;
}
