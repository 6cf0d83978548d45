// Forward of the norms around a block (blocknorm.h), reached through tcvom_block_norm_fwd.
#include "blocknorm.h"

template <class TX, class TY, int V, int TPR, int R, int NV, bool LAYER>
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
        for (int j = 0; j < V; ++j) { w1[n][j] = 1.f; b1[n][j] = 0.f; w2[n][j] = 1.f; b2[n][j] = 0.f; gt[n][j] = 1.f; }
        if (!in[n]) continue;
        if (post) load_vec<float, V>(a.w1 + c, w1[n]);
        if (LAYER && post && a.b1) load_vec<float, V>(a.b1 + c, b1[n]);
        if (pre) load_vec<float, V>(a.w2 + c, w2[n]);
        if (LAYER && pre && a.b2) load_vec<float, V>(a.b2 + c, b2[n]);
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
                load_vec<TX, V>((const TX*)a.x + base + c, x[n]);
                if (has_y) load_vec<TY, V>((const TY*)a.y + base + c, y[n]);
            }
        }
        if (a.gate && live && row / a.gate_rows != grow) {
            grow = row / a.gate_rows;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int c = (n * TPR + lane) * V;
                if (!in[n]) continue;
                if (a.gate_f32) load_vec<float, V>((const float*)a.gate + grow * C + c, gt[n]);
                else load_vec<TY, V>((const TY*)a.gate + grow * C + c, gt[n]);
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
                    for (int j = 0; j < V; ++j) { const float d = t[n][j] - (LAYER ? m : 0.f); s[0] += d * d; }
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
                        const float t = post ? (y[n][j] - m1) * r1 * w1[n][j] + b1[n][j] : y[n][j];
                        x[n][j] = a.rs * x[n][j] + a.bs * gt[n][j] * t;
                    }
        }
        if (pre) moments(x, m2, r2);
        if (!live) continue;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * TPR + lane) * V;
            if (!in[n]) continue;
            if (has_y) store_vec<TX, V>((TX*)a.xo + base + c, x[n]);
            if (pre) {
                float h[V];
#pragma unroll
                for (int j = 0; j < V; ++j) h[j] = (x[n][j] - m2) * r2 * w2[n][j] + b2[n][j];
                store_vec<TY, V>((TY*)a.h + base + c, h);
            }
        }
        if (a.stats && lane == 0) *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(m1, r1, m2, r2);
    }
}

// vector width by alignment, threads by channels (see blocknorm.h)
#define FWD_TABLE(TX, TY, LAUNCH)                                      \
    do {                                                               \
        if (vec) {                                                     \
            if (C <= 128) LAUNCH(TX, TY, 8, 16, 16, 1);                \
            else if (C <= 512) LAUNCH(TX, TY, 8, 64, 4, 1);            \
            else if (C <= 1024) LAUNCH(TX, TY, 8, 64, 4, 2);           \
            else if (C <= 2048) LAUNCH(TX, TY, 8, 256, 1, 1);          \
            else if (C <= 4096) LAUNCH(TX, TY, 8, 256, 1, 2);          \
            else LAUNCH(TX, TY, 8, 512, 1, 2);                         \
        } else {                                                       \
            if (C <= 512) LAUNCH(TX, TY, 1, 64, 4, 8);                 \
            else if (C <= 4096) LAUNCH(TX, TY, 1, 256, 1, 16);         \
            else LAUNCH(TX, TY, 1, 512, 1, 16);                        \
        }                                                              \
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
    const bool vec = C % 8 == 0 && aligned16(x) && aligned16(y) && aligned16(post_weight) && aligned16(post_bias) && aligned16(gate) &&
                     aligned16(pre_weight) && aligned16(pre_bias) && aligned16(x_out) && aligned16(h);
    const hipStream_t st = (hipStream_t)stream;
#define FWD(TX, TY, V, TPR, R, NV)                                                                                      \
    do {                                                                                                                \
        const int wgs = 256 * (2048 / (TPR * R));                                                                       \
        a.rows_per_wg = cdiv(cdiv(T, R), wgs) * R;                                                                      \
        const dim3 grid(cdiv(T, a.rows_per_wg));                                                                        \
        if (layer) hipLaunchKernelGGL((block_norm_fwd_kernel<TX, TY, V, TPR, R, NV, true>), grid, dim3(TPR * R), 0, st, a);  \
        else hipLaunchKernelGGL((block_norm_fwd_kernel<TX, TY, V, TPR, R, NV, false>), grid, dim3(TPR * R), 0, st, a);       \
    } while (0)
    NORM_TYPES(FWD_TABLE, FWD);
#undef FWD
    TCVOM_LAUNCH_CHECK("block_norm_fwd");
    return 0;
}
