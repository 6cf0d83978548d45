// Backward of the norms around a block (blocknorm.h), reached through tcvom_block_norm_bwd.
//   a   = dh w2                       dX = dx' + r2 (a - [mean a] - xhat mean(a xhat))          ([..]: LayerNorm only)
//   dx  = rs dX                       dn = bs g dX,   dg = bs n dX,   n = N1(y)
//   e   = dn w1                       dy = r1 (e - [mean e] - yhat mean(e yhat))
//   dw1 = sum dn yhat, db1 = sum dn, dw2 = sum dh xhat, db2 = sum dh over the tokens
// x' is formed again in 32 bits from x and y (the same bytes as reading the rounded x', none of its rounding); the row statistics come
// from the forward.  Column sums: a workgroup keeps its channels' sums in registers over its rows, adds its row groups through LDS
// and writes one partial row; a second kernel adds the partial rows in a fixed order (no atomics: equal calls give equal bits).
#include "blocknorm.h"

enum { SUM_W1 = 0, SUM_B1, SUM_W2, SUM_B2, SUM_G, SUMS };

// FULL: y, dx' and dh are all there and the channels a multiple of 8.  The loads of a row are then the same ones on every path (a row or
// channel past the end reads the last one again), so that the compiler can count those in flight and wait for a row's own only; between
// branches it waits for all (8192 rows of 4096, bf16: 90 us without, 82 us with, at that step).
template <class TX, class TY, int TPR, int R, int NV, bool TAIL, bool LAYER, bool FULL>
__global__ __launch_bounds__(TPR * R, 2) void block_norm_bwd_kernel(NormArgs a) {
    constexpr int RED = TPR > 64 ? 4 * R * (TPR / 64) : 1;
    constexpr int COLS = R > 1 ? TPR * R * V : 1;
    __shared__ float lds[RED];
    __shared__ float cols[COLS];
    int slot = 0;
    const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const int C = a.C;
    const float inv = 1.f / (float)C;
    const bool has_y = FULL || a.y != nullptr, post = a.w1 != nullptr, pre = FULL || (a.w2 != nullptr && a.dh != nullptr);
    const bool token_gate = a.gate && a.gate_rows == 1;
    float w1[NV][V], b1[NV][V], w2[NV][V], gt[NV][V];
    float s_w1[NV][V], s_b1[NV][V], s_w2[NV][V], s_b2[NV][V], s_g[NV][V];
    bool in[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int c = (n * TPR + lane) * V;
        in[n] = c < C;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            w1[n][j] = !TAIL || c + j < C ? 1.f : 0.f; b1[n][j] = 0.f; w2[n][j] = 1.f; gt[n][j] = a.bs;
            s_w1[n][j] = s_b1[n][j] = s_w2[n][j] = s_b2[n][j] = s_g[n][j] = 0.f;
        }
        if (!in[n]) continue;
        if (post) row_load_f<float, TAIL>(a.w1, c, C, w1[n]);
        if (LAYER && post && a.b1) row_load_f<float, TAIL>(a.b1, c, C, b1[n]);
        if (pre) row_load_f<float, TAIL>(a.w2, c, C, w2[n]);
    }
    auto load_gate = [&](long long grow) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * TPR + lane) * V;
            if (!in[n]) continue;
            if (a.gate_f32) row_load_f<float, TAIL>((const float*)a.gate + grow * C, c, C, gt[n]);
            else row_load_f<TY, TAIL>((const TY*)a.gate + grow * C, c, C, gt[n]);
#pragma unroll
            for (int j = 0; j < V; ++j) gt[n][j] *= a.bs;
        }
    };
    // blockIdx.y = gate row (its tokens' sums stay apart), blockIdx.x = workgroup among its tokens
    const long long group_rows = a.gate && !token_gate ? a.gate_rows : a.T;
    const long long first = (long long)blockIdx.y * group_rows + (long long)blockIdx.x * a.rows_per_wg;
    const long long end = (long long)(blockIdx.y + 1) * group_rows;
    if (a.gate && !token_gate) load_gate(blockIdx.y);
    // the next DEPTH rows' loads are in flight while this one's sums wait at their barriers
    constexpr int DEPTH = NV == 1 ? 2 : 1;
    constexpr bool AHEAD = NV == 1 || !LAYER;               // (16 channels a thread of LayerNorm leave no registers: 8192 x 6000
                                                            // bf16 forward and backward 486 us reading ahead, 280 us without.  Some of these widest
                                                            // forms still spill: LayerNorm 7 registers, with an fp32 x 14, with odd channels or one
                                                            // incoming gradient up to 66; RMS with an fp32 x 6 to 32)
    struct Raw {
        typename RawVec<TX, V>::type x[NV], dx[NV];
        typename RawVec<TY, V>::type y[NV], dh[NV];
        float4 st;
    } raw[DEPTH];
    const long long last = min(first + a.rows_per_wg, end) - 1;
    auto fetch = [&](int k, Raw& r) {
        const long long row = first + k + g;
        if constexpr (FULL) {
            const long long at = min(row, last);
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const long long e = at * C + min((n * TPR + lane) * V, C - V);
                r.x[n] = load_raw<TX, V>((const TX*)a.x + e);
                r.y[n] = load_raw<TY, V>((const TY*)a.y + e);
                r.dx[n] = load_raw<TX, V>((const TX*)a.dxo + e);
                r.dh[n] = load_raw<TY, V>((const TY*)a.dh + e);
            }
            r.st = *reinterpret_cast<const float4*>(a.stats + at * 4);
            return;
        }
        const bool live = k + g < a.rows_per_wg && row < end;
        const long long base = row * C;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * TPR + lane) * V;
            r.x[n] = (typename RawVec<TX, V>::type)(TX)0.f;
            r.dx[n] = r.x[n];
            r.y[n] = (typename RawVec<TY, V>::type)(TY)0.f;
            r.dh[n] = r.y[n];
            if (live && in[n]) {
                if (pre) r.x[n] = row_load<TX, TAIL>((const TX*)a.x + base, c, C);
                if (has_y) r.y[n] = row_load<TY, TAIL>((const TY*)a.y + base, c, C);
                if (a.dxo) r.dx[n] = row_load<TX, TAIL>((const TX*)a.dxo + base, c, C);
                if (pre) r.dh[n] = row_load<TY, TAIL>((const TY*)a.dh + base, c, C);
            }
        }
        r.st = make_float4(0.f, 1.f, 0.f, 1.f);
        if (live) r.st = *reinterpret_cast<const float4*>(a.stats + row * 4);
    };
    auto step = [&](int k, Raw& r) {
        const long long row = first + k + g;
        const bool live = k + g < a.rows_per_wg && row < end;
        const long long base = row * C;
        float x[NV][V], y[NV][V], dX[NV][V], dh[NV][V];
        if (!AHEAD) fetch(k, r);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            raw_to_float<TX, V>(r.x[n], x[n]);
            raw_to_float<TY, V>(r.y[n], y[n]);
            raw_to_float<TX, V>(r.dx[n], dX[n]);
            raw_to_float<TY, V>(r.dh[n], dh[n]);
            if (FULL && !live)
#pragma unroll
                for (int j = 0; j < V; ++j) dh[n][j] = 0.f;
        }
        const float4 st = r.st;
        if (AHEAD && (FULL || k + DEPTH * R < a.rows_per_wg)) fetch(k + DEPTH * R, r);
        if (token_gate && live) load_gate(row);
        const float m1 = st.x, r1 = st.y, m2 = st.z, r2 = st.w;
        // y <- yhat, x <- xhat of x'.  (An absent post norm is one of weight 1 on rows of mean 0 and deviation 1, an absent y is zero.)
#pragma unroll
        for (int n = 0; n < NV; ++n)
            if (in[n])
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    y[n][j] = (LAYER ? y[n][j] - m1 : y[n][j]) * r1;
                    const float t = LAYER ? fmaf(y[n][j], w1[n][j], b1[n][j]) : y[n][j] * w1[n][j];
                    const float x1 = fmaf(gt[n][j], t, a.rs * x[n][j]);
                    x[n][j] = (LAYER ? x1 - m2 : x1) * r2;
                }
        constexpr int K = LAYER ? 2 : 1;
        if (pre) {
            float s[K] = {};
#pragma unroll
            for (int n = 0; n < NV; ++n)
                if (in[n])
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        // (rows past the end hold zeros: they add nothing)
                        s_w2[n][j] = fmaf(dh[n][j], x[n][j], s_w2[n][j]);
                        if (LAYER) s_b2[n][j] += dh[n][j];
                        dh[n][j] *= w2[n][j];
                        s[0] = fmaf(dh[n][j], x[n][j], s[0]);
                        if (LAYER) s[K - 1] += dh[n][j];
                    }
            group_sum<TPR, R, K>(s, lds, slot);
            const float p = s[0] * inv * r2, q = LAYER ? s[K - 1] * inv : 0.f;
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    dX[n][j] = fmaf(r2, LAYER ? dh[n][j] - q : dh[n][j], fmaf(-p, x[n][j], dX[n][j]));
        }
        if (live)
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int c = (n * TPR + lane) * V;
                if (!in[n]) continue;
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = a.rs * dX[n][j];
                row_store<TX, TAIL>((TX*)a.dx + base, c, C, o);
            }
        if (!has_y) return;
        float s[K] = {};
        float dg[NV][V];
#pragma unroll
        for (int n = 0; n < NV; ++n)
            if (in[n])
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float t = LAYER ? fmaf(y[n][j], w1[n][j], b1[n][j]) : y[n][j] * w1[n][j];
                    dg[n][j] = t * dX[n][j];
                    const float dn = live ? gt[n][j] * dX[n][j] : 0.f;
                    s_g[n][j] += live ? dg[n][j] : 0.f;
                    s_w1[n][j] = fmaf(dn, y[n][j], s_w1[n][j]);
                    if (LAYER) s_b1[n][j] += dn;
                    dX[n][j] = dn * w1[n][j];
                    s[0] = fmaf(dX[n][j], y[n][j], s[0]);
                    if (LAYER) s[K - 1] += dX[n][j];
                }
        float p = 0.f, q = 0.f;
        if (post) {
            group_sum<TPR, R, K>(s, lds, slot);
            p = s[0] * inv * r1;
            q = LAYER ? s[K - 1] * inv : 0.f;
        }
        if (!live) return;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * TPR + lane) * V;
            if (!in[n]) continue;
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = fmaf(r1, LAYER ? dX[n][j] - q : dX[n][j], -p * y[n][j]);
            row_store<TY, TAIL>((TY*)a.dy + base, c, C, o);
            if (token_gate && a.dgate) {
#pragma unroll
                for (int j = 0; j < V; ++j) dg[n][j] *= a.bs;
                if (a.gate_f32) row_store<float, TAIL>((float*)a.dgate + base, c, C, dg[n]);
                else row_store<TY, TAIL>((TY*)a.dgate + base, c, C, dg[n]);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
        if (AHEAD && (FULL || i * R < a.rows_per_wg)) fetch(i * R, raw[i]);
    for (int k = 0; k < a.rows_per_wg; k += DEPTH * R) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i)
            if (k + i * R < a.rows_per_wg) step(k + i * R, raw[i]);
    }
    float* part = a.part + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * SUMS * C;
    auto flush = [&](int q, float (&t)[NV][V]) {
        if (!(a.want >> q & 1)) return;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * TPR + lane) * V;
            if constexpr (R > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < V; ++j) cols[threadIdx.x * V + j] = t[n][j];
                __syncthreads();
                if (g == 0)
                    for (int i = 1; i < R; ++i)
#pragma unroll
                        for (int j = 0; j < V; ++j) t[n][j] += cols[(i * TPR + lane) * V + j];
            }
            if (g == 0 && in[n]) row_store<float, TAIL>(part + (long long)q * C, c, C, t[n]);
        }
    };
    flush(SUM_W1, s_w1);
    flush(SUM_W2, s_w2);
    if constexpr (LAYER) {
        flush(SUM_B1, s_b1);
        flush(SUM_B2, s_b2);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int j = 0; j < V; ++j) s_g[n][j] *= a.bs;
    flush(SUM_G, s_g);
}

// out[q] = sum of the partial rows: 64 channels x 16 slices of the rows a workgroup; blockIdx.y = which output
struct NormSums { float* out[SUMS - 1]; void* dgate; int gate_f32, gate_type; int parts, groups, C, nq; int q[SUMS]; };
__global__ __launch_bounds__(1024) void block_norm_sums_kernel(const float* part, NormSums s) {
    __shared__ float red[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
    const bool is_gate = (int)blockIdx.y >= s.nq;            // rows nq.. of the grid: one gate row each
    const int q = is_gate ? (int)SUM_G : s.q[blockIdx.y];
    const int lo = is_gate ? ((int)blockIdx.y - s.nq) * s.parts : 0, hi = is_gate ? lo + s.parts : s.parts * s.groups;
    float t = 0.f;
    if (c < s.C)
#pragma unroll 8
        for (int i = lo + slice; i < hi; i += 16) t += part[((long long)i * SUMS + q) * s.C + c];
    red[slice][threadIdx.x & 63] = t;
    __syncthreads();
    if (slice || c >= s.C) return;
    t = 0.f;
    for (int i = 0; i < 16; ++i) t += red[i][threadIdx.x];
    if (!is_gate) { s.out[q][c] = t; return; }
    const long long at = (long long)((int)blockIdx.y - s.nq) * s.C + c;
    if (s.gate_f32) ((float*)s.dgate)[at] = t;
    else if (s.gate_type == TCVOM_TYPE_BF16) ((__bf16*)s.dgate)[at] = (__bf16)t;
    else if (s.gate_type == TCVOM_TYPE_F16) ((_Float16*)s.dgate)[at] = (_Float16)t;
    else ((float*)s.dgate)[at] = t;
}

static int bwd_groups(int C) { return C <= 128 ? 16 : C <= 512 ? 4 : C <= 1024 ? 2 : 1; }       // row groups of a workgroup (BWD_TABLE's R)
// workgroups a gate row (or in all): as many as fit the chip at once -- two of 256 threads a CU, one of 512 -- no more than there are rows for
static int bwd_wgs(int64_t T, int64_t groups, int C) {
    const int64_t n = ((C > 2048 ? 256 : 512) + groups - 1) / groups, most = (T / groups + bwd_groups(C) - 1) / bwd_groups(C);
    return (int)(n > most ? most : n);
}
// threads by channels: 8 channels a thread while the sums of 5 columns each leave room for them
#define BWD_TABLE(TX, TY, LAUNCH)                      \
    do {                                               \
        if (C <= 128) LAUNCH(TX, TY, 16, 16, 1);       \
        else if (C <= 512) LAUNCH(TX, TY, 64, 4, 1);   \
        else if (C <= 1024) LAUNCH(TX, TY, 128, 2, 1); \
        else if (C <= 2048) LAUNCH(TX, TY, 256, 1, 1); \
        else if (C <= 4096) LAUNCH(TX, TY, 512, 1, 1); \
        else LAUNCH(TX, TY, 512, 1, 2);                \
    } while (0)

extern "C" int64_t tcvom_block_norm_bwd_work(int64_t T, int32_t C, int64_t gate_groups) {
    if (T <= 0 || C <= 0 || gate_groups <= 0) return 0;
    return (int64_t)bwd_wgs(T, gate_groups, C) * gate_groups * SUMS * C;
}

extern "C" int tcvom_block_norm_bwd(const void* x, const void* y, const float* post_weight, const float* post_bias, const void* gate,
                                    int32_t gate_f32, int64_t gate_rows, const float* pre_weight, float branch_scale, float residual_scale,
                                    int32_t layer, const float* stats, const void* dx_out, const void* dh, void* dx, void* dy,
                                    float* dpost_weight, float* dpost_bias, void* dgate, float* dpre_weight, float* dpre_bias, float* work,
                                    int64_t work_floats, int64_t T, int32_t C, int32_t x_type, int32_t y_type, void* stream) {
    TCVOM_CHECK_ARG(x && dx && stats && T >= 0 && C > 0 && C <= TCVOM_MAX_NORM_CHANNELS, "block_norm_bwd: T=%lld C=%d (1..%d)", (long long)T,
                    C, TCVOM_MAX_NORM_CHANNELS);
    TCVOM_CHECK_ARG(norm_types_ok(x_type, y_type), "block_norm_bwd: types %d, %d", x_type, y_type);
    TCVOM_CHECK_ARG(y ? dy != nullptr : !post_weight && !gate, "block_norm_bwd: outputs / weights do not match y");
    TCVOM_CHECK_ARG(!gate || (gate_rows > 0 && T % gate_rows == 0), "block_norm_bwd: %lld tokens a gate row", (long long)gate_rows);
    TCVOM_CHECK_ARG((!dpost_weight && !dpost_bias) || post_weight, "block_norm_bwd: gradient of an absent post norm");
    TCVOM_CHECK_ARG((!dpre_weight && !dpre_bias) || (pre_weight && dh), "block_norm_bwd: gradient of an absent pre norm");
    TCVOM_CHECK_ARG(layer || (!post_bias && !dpost_bias && !dpre_bias), "block_norm_bwd: a bias belongs to LayerNorm");
    TCVOM_CHECK_ARG(!dgate || gate, "block_norm_bwd: gradient of an absent gate");
    TCVOM_CHECK_ARG(T < (1LL << 31), "block_norm_bwd: %lld tokens", (long long)T);
    if (T == 0) return 0;
    const bool token_gate = gate && gate_rows == 1 && T > 1;
    const int64_t groups = gate && !token_gate ? T / gate_rows : 1;
    TCVOM_CHECK_ARG(groups <= 32768, "block_norm_bwd: %lld gate rows of several tokens (at most 32768)", (long long)groups);
    TCVOM_CHECK_ARG(work && work_floats >= tcvom_block_norm_bwd_work(T, C, groups), "block_norm_bwd: %lld floats of workspace",
                    (long long)work_floats);
    NormArgs a = {};
    a.x = x; a.y = y; a.w1 = post_weight; a.b1 = post_bias; a.w2 = pre_weight;
    a.gate = gate; a.gate_f32 = gate_f32; a.gate_rows = gate ? (token_gate ? 1 : gate_rows) : 1;
    a.bs = y ? branch_scale : 0.f; a.rs = y ? residual_scale : 1.f; a.T = T; a.C = C;
    a.stats = (float*)stats; a.dxo = dx_out; a.dh = dh; a.dx = dx; a.dy = dy; a.part = work;
    a.dgate = token_gate ? dgate : nullptr;
    a.want = (dpost_weight ? 1 << SUM_W1 : 0) | (dpost_bias ? 1 << SUM_B1 : 0) | (dpre_weight ? 1 << SUM_W2 : 0) |
             (dpre_bias ? 1 << SUM_B2 : 0) | (dgate && !token_gate ? 1 << SUM_G : 0);
    const int R0 = bwd_groups(C), wgs = bwd_wgs(T, groups, C);
    const int64_t rows = T / groups;
    const hipStream_t st = (hipStream_t)stream;
    const int per = cdiv(cdiv(rows, wgs), R0) * R0;
    const int used = cdiv(rows, per);                        // <= wgs: rounding up to whole row groups can leave some without rows
    a.rows_per_wg = per;
    const dim3 grid(used, (unsigned)groups);
#define BWD_LAUNCH(TX, TY, TPR, R, NV, TAIL, FULL)                                                                                  \
    do {                                                                                                                           \
        if (layer) hipLaunchKernelGGL((block_norm_bwd_kernel<TX, TY, TPR, R, NV, TAIL, true, FULL>), grid, dim3(TPR * R), 0, st, a); \
        else hipLaunchKernelGGL((block_norm_bwd_kernel<TX, TY, TPR, R, NV, TAIL, false, FULL>), grid, dim3(TPR * R), 0, st, a);      \
    } while (0)
#define BWD(TX, TY, TPR, R, NV)                                      \
    do {                                                             \
        if (C % V) BWD_LAUNCH(TX, TY, TPR, R, NV, true, false);      \
        else if (full) BWD_LAUNCH(TX, TY, TPR, R, NV, false, true);  \
        else BWD_LAUNCH(TX, TY, TPR, R, NV, false, false);           \
    } while (0)
    const bool full = y && dx_out && dh && pre_weight;
    NORM_TYPES(BWD_TABLE, BWD);
#undef BWD
#undef BWD_LAUNCH
    TCVOM_LAUNCH_CHECK("block_norm_bwd");
    if (!a.want) return 0;
    NormSums s = {};
    float* outs[SUMS - 1] = {dpost_weight, dpost_bias, dpre_weight, dpre_bias};
    for (int q = 0; q < SUMS - 1; ++q) {
        s.out[q] = outs[q];
        if (outs[q]) s.q[s.nq++] = q;
    }
    s.dgate = dgate; s.gate_f32 = gate_f32; s.gate_type = y_type; s.parts = used; s.groups = (int)groups; s.C = C;
    const int gate_blocks = a.want >> SUM_G & 1 ? (int)groups : 0;
    hipLaunchKernelGGL(block_norm_sums_kernel, dim3(cdiv(C, 64), s.nq + gate_blocks), dim3(1024), 0, st, work, s);
    TCVOM_LAUNCH_CHECK("block_norm_sums");
    return 0;
}
