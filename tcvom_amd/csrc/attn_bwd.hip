// Backward of the attention with a relative position bias (attn.h), reached through tcvom_attn_bwd.
//   p  = exp(x - lse)             dv_j = sum_i p_ij do_i            dp_ij = <do_i, v_j>
//   ds = p (dp - delta_i),        delta_i = <do_i, out_i>           dbias[h][j - i - q_start] = sum ds
//   dq_i = scale sum_j ds_ij k_j                                    dk_j = scale sum_i ds_ij q_i
// Two kernels, each adding in registers what it owns: the queries' one (dq, delta, bucket sums) walks the keys, the keys' one (dk, dv
// over all heads that share them) walks the queries.  Scores are formed in both: 7 products instead of the 5 of a single pass, which
// would have to add dq (or dk, dv) into memory in an order that changes from run to run.
//
// Rounding to 16 bits: p and ds as operands of the matrix products, as the forward rounds p (fp16: p times 2^15, ds times a running power of
// two, ds_fit).  The bucket sums take ds in 32 bits.
#include "attn.h"

// ---- dq, delta, bucket sums: a wave owns 32 queries of one head (S^T and dP^T as in the forward), the workgroup walks tiles of 64 keys.
// Bucket sums: a tile past an end of the line adds to one register a lane.  A 32 x 32 block that crosses it is written to LDS skewed, key
// row n, query column c at [n][n - c + 31], where each of the 63 diagonals is a column that one lane adds up (the rest of the 64
// columns was zeroed once and never written), then onto the wave's own line of sums.  Every sum is made in program order: equal calls
// give equal bits.  (Adding the elements with LDS atomics took 53 cycles an instruction, one lane after the other: 16 of them a block
// were as long as its matrix products.)
//
// Bound as the forward by matrix plus vector time: 3 products and 5 vector instructions a score.  4 x 1024 tokens, 8 heads of 64, fp16: 43 us (one
// wave a SIMD, waiting 41 % of its time); 2 x 4080 causal, 16 heads of 128 on 4, bf16: 261 us = 785 TFLOP/s.  With the table's gradient five lines
// and the skewed blocks share a CU's LDS: beyond a reach of 280 (bidirectional; 560 one-sided) a CU holds one workgroup instead of two, 8 x 2048, 16
// heads of 64, bf16: 303 us at max_distance 256, 509 at 512, 585 at 1024.
template <class T, int DP, bool TABLE>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(AttnArgs a) {
    typedef typename Mma<T>::v8 v8;
    constexpr int KT = DP == 128 ? 32 : 64;                 // keys a tile: two waves a SIMD fit the registers
    constexpr int KS = DP / 16, DB = DP / 32, BM = 128, TILE = KT * DP;
    __shared__ __align__(16) T lk[2 * TILE];
    __shared__ __align__(16) T lv[2 * TILE];
    extern __shared__ float line_[];
    float* line = line_ + MARGIN;

    int bh, tile;
    work_item(a, blockIdx.x, a.B * a.H, bh, tile);
    if (a.causal) tile = a.tiles - 1 - tile;
    const int b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hkv);
    const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5, col = lane & 31;
    const int i0 = tile * BM, start = seq_start(a, b), len = seq_keys(a, b);
    const int i_last = min(i0 + BM, a.Nq) - 1;
    const int kend = a.causal ? max(0, min(len, i_last + start + 1)) : len;
    const int ntiles = (kend + KT - 1) / KT;
    const int reach = line_reach(a.bk), right = line_right(a.bk), last = reach + right;
    // [4][last + 1 + 2 MARGIN]: a line of sums for each wave, with margins as the bias has
    const int pitch = last + 1 + 2 * MARGIN;
    float* sums = line_ + pitch;
    __shared__ float skew[TABLE ? 4 * 32 * 64 : 1];
    if (TABLE) {
        for (int t = threadIdx.x; t < 4 * pitch; t += 256) sums[t] = 0.f;
        for (int t = threadIdx.x; t < 4 * 32 * 64; t += 256) skew[t] = 0.f;
    }
    float* mine = sums + wave * pitch + MARGIN;
    float* put = skew + (TABLE ? wave * (32 * 64) + 4 * half * 65 - col + 31 : 0);
    const float* get = skew + (TABLE ? wave * (32 * 64) + lane : 0);

    const T* Q = (const T*)a.q + b * a.qs[0] + h * a.qs[2];
    const T* K = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
    const T* V = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
    const T* dO = (const T*)a.dout + b * a.dos[0] + h * a.dos[2];
    const unsigned char* mask = a.key_mask ? a.key_mask + (long long)b * a.Nk : nullptr;

    const int w0 = i0 + wave * 32, qi = w0 + col;
    const long long stat = ((long long)b * a.H + h) * a.Nq + qi, orow = (((long long)b * a.Nq + qi) * a.H + h) * a.D;
    const float raw = qi < a.Nq ? a.lse[stat] : -INFINITY;
    v8 qf[KS], gf[KS];
    f32x4_t of[2 * KS];
    float delta = 0.f;
    // (every load is issued before one is waited for)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int d = s * 16 + half * 8;
        const bool ok = qi < a.Nq && d < a.D;
        qf[s] = load_or_zero<v8>(ok, Q + (long long)qi * a.qs[1] + d);
        gf[s] = load_or_zero<v8>(ok, dO + (long long)qi * a.dos[1] + d);
        if (TABLE) {
            of[2 * s] = load_or_zero<f32x4_t>(ok, a.out32 + orow + d);
            of[2 * s + 1] = load_or_zero<f32x4_t>(ok, a.out32 + orow + d + 4);
        } else {
            of[s] = __builtin_bit_cast(f32x4_t, load_or_zero<v8>(ok, (const T*)a.out + orow + d));
        }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const v8 o = __builtin_bit_cast(v8, of[s]);
#pragma unroll
        for (int j = 0; j < 8; ++j) delta = fmaf((float)gf[s][j], TABLE ? of[2 * s + j / 4][j % 4] : (float)o[j], delta);
    }
    // a row without a key has no gradient, whatever its dout holds
    const bool live = raw != -INFINITY;
    const float lse = live ? raw : 0.f;
    if (!live) {
        delta = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) gf[s] = qf[s] = v8{};
    }
    delta = half_sum(delta);
    if (half == 0 && qi < a.Nq) a.delta[stat] = delta;

    Mover<T, DP, KT> mk, mv;
    auto fetch = [&](int t) {
        const int k0 = t * KT;
        auto ok = [&](int r) { return mask[k0 + r] != 0; };
        mk.load(K + k0 * a.ks[1], a.ks[1], kend - k0, a.D, !mask, ok);
        mv.load(V + k0 * a.vs[1], a.vs[1], kend - k0, a.D, !mask, ok);
    };
    f32x16_t acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = zero16();
    float far_lo = 0.f, far_hi = 0.f, up = DS_UP<T>;
    const float c = a.scale * LOG2E;
    const unsigned rows_at = Tile<T, DP>::rows_at(lane), cols_at = Tile<T, DP>::cols_at(lane);
    if (ntiles > 0) fetch(0);
    fill_line(line, a, h, 256);
    if (ntiles > 0) {
        mk.store(lk);
        mv.store(lv);
    }
    arrived(qf);
    arrived(gf);
    __syncthreads();
    for (int t = 0; t < ntiles; ++t) {
        const int k0 = t * KT, buf = (t & 1) * TILE;
        const unsigned ra = keep(rows_at) + buf * 2, ca = keep(cols_at) + buf * 2;
        if (t + 1 < ntiles) fetch(t + 1);
        const bool holes = mask || i0 + BM > a.Nq || k0 + KT > min(len, a.causal ? w0 + start + 1 : len);
        unsigned long long see = 0;
        if (holes) {
            unsigned long long bits = ~0ull;
            if (mask) bits = __ballot(k0 + lane < a.Nk && mask[min(k0 + lane, a.Nk - 1)]);
            const int lim = live ? min(len, a.causal ? qi + start + 1 : len) - k0 : 0;
            see = lim >= 64 ? bits : lim <= 0 ? 0 : bits & ((1ull << lim) - 1);
        }
        const int rel_hi = k0 + KT - 1 - w0 - start, rel_lo = k0 - (w0 + 31) - start;
        const bool left = rel_hi <= -reach, near = !left && rel_lo < right;
        const float mul = near ? 1.f : c, add = (near ? 0.f : left ? line[0] : line[last]) - lse;
        float total = 0.f;
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb) {
            f32x16_t x = zero16(), g = zero16();
#pragma unroll
            for (int s = 0; s < KS; ++s) x = Mma<T>::mma(Tile<T, DP>::rows(lk, ra, kb * 32, s), qf[s], x);
#pragma unroll
            for (int s = 0; s < KS; ++s) g = Mma<T>::mma(Tile<T, DP>::rows(lv, ra, kb * 32, s), gf[s], g);
            if (near) {
                const float* at = line + (k0 + kb * 32 + 4 * half - qi - start + reach);
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], c, at[8 * (r / 4) + r % 4]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = exp2_hw(fmaf(x[r], mul, add)) * (g[r] - delta);
            if (holes) {
                const unsigned w = (unsigned)(see >> (32 * kb)) >> (4 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = pick(w, r, x[r], 0.f);
            }
            if (TABLE) {
                float s[4] = {0.f, 0.f, 0.f, 0.f};
                if (near) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) put[(8 * (r / 4) + r % 4) * 65] = x[r];
#pragma unroll
                    for (int n = 0; n < 32; ++n) s[n & 3] += get[n * 64];
                    // diagonal key - query = lane - 31 of the block (lane 63: none, zero)
                    mine[k0 + kb * 32 - w0 - start + reach + lane - 31] += (s[0] + s[1]) + (s[2] + s[3]);
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r & 3] += x[r];
                    total += (s[0] + s[1]) + (s[2] + s[3]);
                }
            }
            ds_fit<T>(x, up, acc);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const v8 p = pack_ds<T>(x, up, s);
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = Mma<T>::mma(Tile<T, DP>::cols(lk, ca, kb * 32 + s * 16, d), p, acc[d]);
            }
        }
        far_lo += left ? total : 0.f;
        far_hi += left ? 0.f : total;
        if (t + 1 < ntiles) {
            mk.store(lk + (TILE - buf));
            mv.store(lv + (TILE - buf));
        }
        __syncthreads();
    }
    if (qi < a.Nq) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = d * 32 + g * 8 + half * 4;
                if (at >= a.D) continue;
                typename Mma<T>::v4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (T)ds_down<T>(acc[d][4 * g + j] * a.scale, up);
                *reinterpret_cast<typename Mma<T>::v4*>((T*)a.dq + orow + at) = w;
            }
    }
    if (!TABLE) return;
    // the waves' lines become one, entry by entry in order (in place of the bias); what lies past its ends -- whole tiles and the
    // margins -- belongs to the end entries
    __shared__ float ends[2][4];
    const float lo = wave_sum(far_lo), hi = wave_sum(far_hi);
    if (lane == 0) {
        ends[0][wave] = lo;
        ends[1][wave] = hi;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < pitch; t += 256) {
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n) s += sums[n * pitch + t];
        line_[t] = s;
    }
    __syncthreads();
    for (int n = threadIdx.x; n < a.bk.num_buckets; n += 256) {
        int t0, t1;
        bucket_entries(a.bk, n, t0, t1);
        float s = 0.f;
        if (t0 < t1) {
            if (t0 == 0) {
                s = (ends[0][0] + ends[0][1]) + (ends[0][2] + ends[0][3]);
                t0 = -MARGIN;
            }
            if (t1 == last + 1) {
                s += (ends[1][0] + ends[1][1]) + (ends[1][2] + ends[1][3]);
                t1 = last + 1 + MARGIN;
            }
        }
        for (int t = t0; t < t1; ++t) s += line[t];
        a.part[(((long long)h * a.B + b) * a.tiles + tile) * a.bk.num_buckets + n] = s;
    }
}

// dtable[n][h] = sum over the workgroups of head h of attn_dq_kernel, in 64 bits, by a workgroup a head: 256 threads = buckets x slices of
// those workgroups.  The first workgroups of the dk / dv launch, which runs after that kernel.
__device__ __forceinline__ void sum_table(const AttnArgs& a, int h, double* red) {
    const int buckets = a.bk.num_buckets, slices = 256 / buckets, n = threadIdx.x % buckets, s = threadIdx.x / buckets;
    const long long parts = (long long)a.B * ((a.Nq + 127) / 128);
    double t = 0.;
    if (s < slices)
#pragma unroll 4
        for (long long i = s; i < parts; i += slices) t += (double)a.part[(h * parts + i) * buckets + n];
    red[threadIdx.x] = t;
    __syncthreads();
    if ((int)threadIdx.x >= buckets) return;
    t = 0.;
    for (int i = 0; i < slices; ++i) t += red[i * buckets + threadIdx.x];
    a.dtable[threadIdx.x * a.H + h] = (float)t;
}

// ---- dk, dv: a wave owns 32 keys of one key head, the workgroup (128 keys) walks the queries of every head that shares them, 32 at a
// time.  Scores here are S = Q K^T (rows = queries, columns = keys): p and ds are again the register operand of dV^T = dO^T P and
// dK^T = Q^T dS.
//
// Causal key tiles have very different numbers of queries, and a group of heads that share keys multiplies a workgroup's work: with
// few workgroups (attn_apart says how few) each head of a group gets workgroups of its own, which write fp32 partial sums [2][B][Nk][H][D] that
// attn_heads_kernel adds in order.  The tiles with most queries come first.
//
// Bound as above, 4 products a score.  4 x 1024 tokens, 8 heads of 64, fp16: 45 us (one wave a SIMD, waiting 40 % of its time); 2 x 4080
// causal, 16 heads of 128 on 4, bf16: 336 us = 812 TFLOP/s, attn_heads_kernel 23 us (150 MB, part of them still in the last cache).
template <class T, int DP>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(AttnArgs a) {
    typedef typename Mma<T>::v8 v8;
    constexpr int KS = DP / 16, DB = DP / 32, CH = DP / 8, QT = 32, BN = 128, TILE = QT * DP;
    __shared__ __align__(16) T lq[2 * TILE];
    __shared__ __align__(16) T lg[2 * TILE];
    constexpr bool VREG = DP < 128;                         // values, operand B of dP = dO V^T, in registers; width 128 has none left
    __shared__ __align__(16) T lv[VREG ? 8 : BN * DP];
    __shared__ __align__(16) float ls[4][QT], ld[4][QT];    // log-sums and deltas of the tiles: written two tiles ahead
    __shared__ int odds[4];                                 // a wave each: `odd` of its share of the line
    extern __shared__ float line_[];
    float* line = line_ + MARGIN;
    const int extra = a.dtable ? a.H : 0;
    if ((int)blockIdx.x < extra) {
        sum_table(a, blockIdx.x, reinterpret_cast<double*>(lq));
        return;
    }

    const int heads = a.apart ? a.H : a.Hkv, G = a.apart ? 1 : a.H / a.Hkv;      // of the grid, and of a workgroup
    int bh, tile;
    work_item(a, blockIdx.x - extra, a.B * heads, bh, tile);
    const int b = bh / heads, h0 = bh % heads * G, hk = h0 / (a.H / a.Hkv);
    const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5, col = lane & 31;
    const int start = seq_start(a, b), len = seq_keys(a, b);
    const int j0 = tile * BN, w0 = j0 + wave * 32, key = w0 + col;
    const int reach = line_reach(a.bk), right = line_right(a.bk), last = reach + right;
    const unsigned char* mask = a.key_mask ? a.key_mask + (long long)b * a.Nk : nullptr;
    const bool seen = key < len && (!mask || mask[key]);
    const T* K = (const T*)a.k + b * a.ks[0] + hk * a.ks[2] + (long long)key * a.ks[1];
    const T* V = (const T*)a.v + b * a.vs[0] + hk * a.vs[2] + (long long)key * a.vs[1];
    v8 kf[KS], vf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int d = s * 16 + half * 8;
        kf[s] = load_or_zero<v8>(seen && d < a.D, K + d);
        vf[s] = load_or_zero<v8>(seen && d < a.D, V + d);
        if constexpr (!VREG) *reinterpret_cast<v8*>(&lv[chunk_at<DP>(wave * 32 + col, s * 2 + half) * 8]) = vf[s];
    }
    f32x16_t dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        dk[d] = zero16();
        dv[d] = zero16();
    }
    float up = DS_UP<T>;
    const float c = a.scale * LOG2E;
    const unsigned rows_at = Tile<T, DP>::rows_at(lane), cols_at = Tile<T, DP>::cols_at(lane);
    constexpr float small = Mma<T>::shift > 0.f ? 1.f / 32768.f : 1.f;       // 2^-shift
    // queries that see a key of this workgroup: from i >= j0 - start on if causal, none if the keys do not exist
    const int i_first = a.causal ? max(0, j0 - start) / QT * QT : 0;
    const int nt = j0 < len && i_first < a.Nq ? (a.Nq - i_first + QT - 1) / QT : 0;
    Mover<T, DP, QT> mq, mg;
    constexpr int PER = Mover<T, DP, QT>::PER, STEP = Mover<T, DP, QT>::STEP;
    // head and first query of the tile that is fetched next: from the last queries back to the first, so that the workgroups of a causal
    // head, which end at different ones, start together
    const int i_last = i_first + (nt - 1) * QT;
    struct Place { int h, i; } at_q = {h0, i_last}, at_s = {h0, i_last};
    auto advance = [&](Place& p) {
        p.i -= QT;
        if (p.i < i_first) {
            p.i = i_last;
            ++p.h;
        }
    };
    float rs = 0.f, rd = 0.f;
    auto fetch_stats = [&]() {
        if (threadIdx.x < QT) {
            const long long stat = ((long long)b * a.H + at_s.h) * a.Nq + at_s.i + threadIdx.x;
            const bool ok = at_s.i + (int)threadIdx.x < a.Nq;
            rs = ok ? a.lse[stat] : -INFINITY;
            rd = ok ? a.delta[stat] : 0.f;
        }
        advance(at_s);
    };
    auto store_stats = [&](int t) {
        const unsigned n = DP == 128 ? keep(threadIdx.x) : threadIdx.x;
        if (n < QT) {
            ls[t & 3][n] = rs == -INFINITY ? INFINITY : rs - Mma<T>::shift;       // p = 0 in rows that are empty or past the end
            ld[t & 3][n] = rd * small;
        }
    };
    auto all = [](int) { return true; };
    auto fetch_q = [&]() {
        mq.load((const T*)a.q + b * a.qs[0] + at_q.h * a.qs[2] + at_q.i * a.qs[1], a.qs[1], a.Nq - at_q.i, a.D, true, all);
    };
    auto fetch_g = [&]() {
        mg.load((const T*)a.dout + b * a.dos[0] + at_q.h * a.dos[2] + at_q.i * a.dos[1], a.dos[1], a.Nq - at_q.i, a.D, true, all);
        advance(at_q);
    };
    // a row without a key has no gradient, whatever its q and dout hold: 0 x inf would not vanish in the products
    auto store = [&](Mover<T, DP, QT>& m, T* tiles, int t) {
#pragma unroll
        for (int n = 0; n < PER; ++n)
            if (ls[t & 3][(threadIdx.x / CH + n * STEP) % QT] == INFINITY) m.reg[n] = (u32x4_t){0, 0, 0, 0};
        m.store(tiles + (t & 1) * TILE);
    };
    const int total = nt * G;
    if (total > 0) {
        fetch_q();
        fetch_g();
        fetch_stats();
        store_stats(0);
        if (total > 1) {
            fetch_stats();
            store_stats(1);
        }
        __syncthreads();
        store(mq, lq, 0);
        store(mg, lg, 0);
    }
    arrived(kf);
    if constexpr (VREG) arrived(vf);
    int i0 = i_first, h = h0 - 1;
    int odd = 0;                                             // whether the head's bias has a NaN or +inf somewhere
    for (int t = 0; t < total; ++t) {
        const int buf = t & 1;
        i0 -= QT;
        const unsigned va = keep(rows_at), ra = va + buf * (QT * DP * 2), ca = keep(cols_at) + buf * (QT * DP * 2);
        if (i0 < i_first) {                                  // another head's bias
            i0 = i_last;
            __syncthreads();
            const int any = __any(fill_line(line, a, ++h, 256));
            if (lane == 0) odds[wave] = any;
            __syncthreads();
            odd = __builtin_amdgcn_readfirstlane(odds[0] | odds[1] | odds[2] | odds[3]);
        }
        // the next tile: at width 128 its dO is fetched once its Q has left the registers
        if (t + 2 < total) fetch_stats();
        if (t + 1 < total) {
            fetch_q();
            if (DP < 128) fetch_g();
        }
        f32x16_t x = zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) x = Mma<T>::mma(Tile<T, DP>::rows(lq, ra, 0, s), kf[s], x);
        const int rel_hi = w0 + 31 - i0 - start, rel_lo = w0 - (i0 + QT - 1) - start;
        const bool far = rel_hi <= -reach || rel_lo >= right;
        float sub[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 s4 = *reinterpret_cast<const float4*>(&ls[t & 3][8 * q + 4 * half]);
            sub[4 * q] = s4.x; sub[4 * q + 1] = s4.y; sub[4 * q + 2] = s4.z; sub[4 * q + 3] = s4.w;
        }
        if (far) {
            const float add = rel_hi <= -reach ? line[0] : line[last];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = exp2_hw(fmaf(x[r], c, add - sub[r]));
        } else {
            const float* at = line + (key - i0 - 4 * half - start + reach);
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = exp2_hw(fmaf(x[r], c, at[-8 * (r / 4) - r % 4] - sub[r]));
        }
        const int first = a.causal ? key - start - i0 - 4 * half : -1 << 30;     // the first row of the tile that sees the key, less 4 half
        if (odd) {                                           // rows that are empty or past the end: exp2(bias - inf) is not always 0 then
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 s4 = *reinterpret_cast<const float4*>(&ls[t & 3][8 * q + 4 * half]);
                x[4 * q] = s4.x == INFINITY ? 0.f : x[4 * q];
                x[4 * q + 1] = s4.y == INFINITY ? 0.f : x[4 * q + 1];
                x[4 * q + 2] = s4.z == INFINITY ? 0.f : x[4 * q + 2];
                x[4 * q + 3] = s4.w == INFINITY ? 0.f : x[4 * q + 3];
            }
        }
        if (!seen || first > -4) {
            const int from = seen ? first : 1 << 30;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (8 * (r / 4) + r % 4 < from) x[r] = 0.f;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const v8 p = pack_step<T>(x, s);
#pragma unroll
            for (int d = 0; d < DB; ++d) dv[d] = Mma<T>::mma(Tile<T, DP>::cols(lg, ca, s * 16, d), p, dv[d]);
        }
        if constexpr (DP == 128) {
            __builtin_amdgcn_sched_barrier(0);               // (the next product's operands would not fit beside this one's)
            if (t + 1 < total) {
                store(mq, lq, t + 1);
                fetch_g();
            }
        }
        f32x16_t g = zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) g = Mma<T>::mma(Tile<T, DP>::rows(lg, ra, 0, s), VREG ? vf[s] : Tile<T, DP>::rows(lv + wave * 32 * DP, va, 0, s), g);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 d4 = *reinterpret_cast<const float4*>(&ld[t & 3][8 * q + 4 * half]);
            x[4 * q] *= fmaf(g[4 * q], small, -d4.x);
            x[4 * q + 1] *= fmaf(g[4 * q + 1], small, -d4.y);
            x[4 * q + 2] *= fmaf(g[4 * q + 2], small, -d4.z);
            x[4 * q + 3] *= fmaf(g[4 * q + 3], small, -d4.w);
        }
        ds_fit<T>(x, up, dk);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const v8 p = pack_ds<T>(x, up, s);
#pragma unroll
            for (int d = 0; d < DB; ++d) dk[d] = Mma<T>::mma(Tile<T, DP>::cols(lq, ca, s * 16, d), p, dk[d]);
        }
        if (t + 1 < total) {
            if (DP < 128) store(mq, lq, t + 1);
            store(mg, lg, t + 1);
        }
        if (t + 2 < total) store_stats(t + 2);
        __syncthreads();
    }
    if (key >= a.Nk) return;
    if (a.apart) {
        float* dst = a.partial + (((long long)b * a.Nk + key) * a.H + h0) * a.D;
        const long long next = (long long)a.B * a.Nk * a.H * a.D;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int at = d * 32 + q * 8 + half * 4;
                if (at >= a.D) continue;
                *reinterpret_cast<float4*>(dst + at) = make_float4(ds_down<T>(dk[d][4 * q], up), ds_down<T>(dk[d][4 * q + 1], up),
                                                                   ds_down<T>(dk[d][4 * q + 2], up), ds_down<T>(dk[d][4 * q + 3], up));
                *reinterpret_cast<float4*>(dst + next + at) = make_float4(dv[d][4 * q], dv[d][4 * q + 1], dv[d][4 * q + 2], dv[d][4 * q + 3]);
            }
        return;
    }
    const long long row = (((long long)b * a.Nk + key) * a.Hkv + hk) * a.D;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = d * 32 + q * 8 + half * 4;
            if (at >= a.D) continue;
            typename Mma<T>::v4 w, u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = (T)ds_down<T>(dk[d][4 * q + j] * a.scale, up);
                u[j] = (T)(dv[d][4 * q + j] * small);
            }
            *reinterpret_cast<typename Mma<T>::v4*>((T*)a.dk + row + at) = w;
            *reinterpret_cast<typename Mma<T>::v4*>((T*)a.dv + row + at) = u;
        }
}

// dk, dv of a key head = the sums of its query heads' (attn_dkv_kernel, `apart`): 4 channels a thread
template <class T>
__global__ __launch_bounds__(256) void attn_heads_kernel(AttnArgs a) {
    const int G = a.H / a.Hkv, quads = a.D / 4;
    const long long n = (long long)a.B * a.Nk * a.Hkv * quads, at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= n) return;
    const long long row = at / quads;                       // (b, key, key head)
    const int c = (int)(at % quads) * 4;
    const float* src = a.partial + (row / a.Hkv * a.H + row % a.Hkv * G) * a.D + c + blockIdx.y * ((long long)a.B * a.Nk * a.H * a.D);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = 0; g < G; ++g) {
        const float4 f = *reinterpret_cast<const float4*>(src + (long long)g * a.D);
        s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w;
    }
    const float w = blockIdx.y ? (Mma<T>::shift > 0.f ? 1.f / 32768.f : 1.f) : a.scale;
    const typename Mma<T>::v4 v = {(T)(s.x * w), (T)(s.y * w), (T)(s.z * w), (T)(s.w * w)};
    *reinterpret_cast<typename Mma<T>::v4*>((T*)(blockIdx.y ? a.dv : a.dk) + row * a.D + c) = v;
}

// Heads apart: more workgroups, of equal lengths, for 8 bytes of workspace a channel of every head's keys and a pass over them.  The chip holds 512
// workgroups.  dk / dv apart against together, 16 heads on 4, bf16, us:
//     not causal, 2048 tokens, width 64: 384 workgroups (together) 333 / 363, 448: 363 / 350, 512: 438 / 408, 1024: 786 / 713; width 128, 448: 652 / 619
//     causal, key heads a multiple of 8 (longest tiles first, work_item): 512: 249 / 290, 640: 303 / 287, 1024: 500 / 427; width 128, 512: 452 / 560,
//     640: 569 / 538, 1024: 941 / 749
//     causal, others (tiles of a head one after the other, the last ones alone): 576: 264 / 348, 832: 392 / 504, 1152: 1010 / 1253, 1920: 1615 / 1889
static bool attn_apart(const tcvom_attn_desc* d) {
    const long long tiles = cdiv(d->Nk, 128), heads = (long long)d->B * d->Hkv;
    const int limit = !d->causal ? 447 : heads % 8 == 0 ? 512 : 2047;
    return d->H > d->Hkv && tiles * heads <= limit && tiles * d->B * d->H + d->H <= TCVOM_MAX_ATTN_WORKGROUPS;
}

template <class T, int DP>
static void launch_bwd(AttnArgs a, float* dtable, hipStream_t st) {
    a.tiles = cdiv(a.Nq, 128);
    const dim3 grid((unsigned)((long long)a.B * a.H * a.tiles));
    if (dtable) hipLaunchKernelGGL((attn_dq_kernel<T, DP, true>), grid, dim3(256), 5 * line_bytes(a), st, a);
    else hipLaunchKernelGGL((attn_dq_kernel<T, DP, false>), grid, dim3(256), line_bytes(a), st, a);
    a.tiles = cdiv(a.Nk, 128);
    a.dtable = dtable;
    const long long wgs = (long long)a.B * (a.apart ? a.H : a.Hkv) * a.tiles + (dtable ? a.H : 0);
    hipLaunchKernelGGL((attn_dkv_kernel<T, DP>), dim3((unsigned)wgs), dim3(256), line_bytes(a), st, a);
    if (a.apart)
        hipLaunchKernelGGL(attn_heads_kernel<T>, dim3(cdiv((long long)a.B * a.Nk * a.Hkv * (a.D / 4), 256), 2), dim3(256), 0, st, a);
}

extern "C" int64_t tcvom_attn_bwd_work(const tcvom_attn_desc* d) {
    if (!d || d->B <= 0 || d->H <= 0 || d->Hkv <= 0 || d->Nq < 0 || d->Nk < 0) return 0;
    const int64_t rows = (int64_t)d->B * d->H * d->Nq + (int64_t)d->B * d->H * cdiv(d->Nq, 128) * d->buckets.num_buckets;
    return (rows + 3) / 4 * 4 + (attn_apart(d) ? 2 * (int64_t)d->B * d->Nk * d->H * d->D : 0);
}

extern "C" int tcvom_attn_bwd(const tcvom_attn_desc* d, const void* q, const void* k, const void* v, const float* table, const void* out,
                              const float* out32, const float* lse, const void* dout, const int64_t* dout_stride, void* dq, void* dk,
                              void* dv, float* dtable, float* work, int64_t work_floats, void* stream) {
    AttnArgs a;
    if (const int rc = attn_check("attn_bwd", d, &a)) return rc;
    TCVOM_CHECK_ARG(d->B > 0 && d->Nq > 0 && d->Nk > 0, "attn_bwd: B=%d Nq=%d Nk=%d", d->B, d->Nq, d->Nk);
    TCVOM_CHECK_ARG(q && k && v && table && out && lse && dout && dout_stride && dq && dk && dv && work, "attn_bwd: null tensor");
    TCVOM_CHECK_ARG(!dtable || out32, "attn_bwd: the table's gradient needs the output in 32 bits");
    TCVOM_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(out32) && aligned16(dout) &&
                        aligned16(dq) && aligned16(dk) && aligned16(dv), "attn_bwd: tensors start at multiples of 16 bytes");
    TCVOM_CHECK_ARG((long long)d->B * d->H * cdiv(d->Nq, 128) <= TCVOM_MAX_ATTN_WORKGROUPS &&
                        (long long)d->B * d->Hkv * cdiv(d->Nk, 128) + d->H <= TCVOM_MAX_ATTN_WORKGROUPS,
                    "attn_bwd: %d sequences x %d heads x %d queries, %d keys", d->B, d->H, d->Nq, d->Nk);
    TCVOM_CHECK_ARG(work_floats >= tcvom_attn_bwd_work(d) && aligned16(work), "attn_bwd: %lld floats of workspace", (long long)work_floats);
    for (int n = 0; n < 3; ++n) {
        TCVOM_CHECK_ARG(dout_stride[n] % 8 == 0 && dout_stride[n] >= 0 && dout_stride[1] < (1 << 24), "attn_bwd: stride %lld of dout",
                        (long long)dout_stride[n]);
        a.dos[n] = dout_stride[n];
    }
    a.q = q; a.k = k; a.v = v; a.table = table; a.out = (void*)out; a.out32 = (float*)out32; a.lse = (float*)lse; a.dout = dout;
    a.dq = dq; a.dk = dk; a.dv = dv;
    a.delta = work;
    a.part = work + (int64_t)d->B * d->H * d->Nq;
    a.apart = attn_apart(d);
    if (a.apart) a.partial = work + tcvom_attn_bwd_work(d) - 2 * (int64_t)d->B * d->Nk * d->H * d->D;
    const hipStream_t st = (hipStream_t)stream;
    const int DP = attn_width(d->D);
    if (d->type == TCVOM_TYPE_BF16) {
        if (DP == 32) launch_bwd<__bf16, 32>(a, dtable, st);
        else if (DP == 64) launch_bwd<__bf16, 64>(a, dtable, st);
        else launch_bwd<__bf16, 128>(a, dtable, st);
    } else {
        if (DP == 32) launch_bwd<_Float16, 32>(a, dtable, st);
        else if (DP == 64) launch_bwd<_Float16, 64>(a, dtable, st);
        else launch_bwd<_Float16, 128>(a, dtable, st);
    }
    TCVOM_LAUNCH_CHECK("attn_bwd");
    return 0;
}
