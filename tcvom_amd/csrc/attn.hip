// Forward of the attention with a relative position bias (attn.h), reached through tcvom_attn_fwd.
#include "attn.h"

// a row without a key is zero; a sum that is NaN makes the row NaN
__device__ __forceinline__ float empty_or(float sum, float v) { return sum == 0.f ? 0.f : v; }

// ---- many queries: a workgroup of 4 waves takes 128 queries of one head, a wave 32 of them, all through the same tiles of 64 keys.
// K and V tiles go to LDS through registers (the next tile's loads are in flight during this tile's products), two buffers, one
// barrier a tile.  LO (training with a gradient of the table): a second product with what rounding dropped from the probabilities.
//
// Bound: the vector unit and the matrix unit in turns.  At width 64 a block of 32 x 32 scores takes 96 vector instructions, 16 of them
// exponentials of four times the length, and 8 products; with the two waves a SIMD that one frame of 8 heads gives, the counters see vector
// instructions in 66 % and products in 33 % of the cycles: hardly any of the one beside the other, and a wave waits for data or a barrier
// 22 % of its time.  Steady times (the clock of a fresh process takes some 150 calls to settle, 15 to 20 % slower until then): 8160 x 8160
// tokens, 8 heads of 64, bf16: 182 us = 749 TFLOP/s, four such frames 647 us = 843 TFLOP/s (a large library product: 1340).  4 x 1024, 8 heads
// of 64, fp16, LO: 28 us, one wave a SIMD; 2 x 4080 causal, 16 heads of 128 on 4, bf16, LO: 226 us = 905 TFLOP/s of its three products.  Slower or no faster: 64 queries a wave (5 % faster at width 64 only, no registers at 128),
// scores formed a tile ahead, row sums by a product with ones, products of the two key blocks in turn, a higher wave priority for them.
template <class T, int DP, bool LO>
__global__ __launch_bounds__(256, 2) void attn_fwd_kernel(AttnArgs a) {
    typedef typename Mma<T>::v8 v8;
    constexpr int KS = DP / 16, DB = DP / 32, BM = 128, TILE = KT * DP;
    // the running maximum may lag by 2^SLACK: probabilities then reach 2^(SLACK + SHIFT), the largest power of two of fp16
    constexpr float SLACK = 4.f, SHIFT = Mma<T>::shift > 0.f ? Mma<T>::shift - SLACK : 0.f;
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
    // keys any query of the workgroup sees
    const int i_last = min(i0 + BM, a.Nq) - 1;
    const int kend = a.causal ? max(0, min(len, i_last + start + 1)) : len;
    const int ntiles = (kend + KT - 1) / KT;
    const int reach = line_reach(a.bk), right = line_right(a.bk), last = reach + right;

    const T* Q = (const T*)a.q + b * a.qs[0] + h * a.qs[2];
    const T* K = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
    const T* V = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
    const unsigned char* mask = a.key_mask ? a.key_mask + (long long)b * a.Nk : nullptr;

    const int w0 = i0 + wave * 32, qi = w0 + col;          // the wave's first query, the lane's
    const int first_limit = min(len, a.causal ? w0 + start + 1 : len), my_limit = min(len, a.causal ? qi + start + 1 : len);
    v8 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int d = s * 16 + half * 8;
        qf[s] = load_or_zero<v8>(qi < a.Nq && d < a.D, Q + (long long)qi * a.qs[1] + d);
    }
    Mover<T, DP, KT> mk, mv;
    auto fetch = [&](int t) {
        const int k0 = t * KT;
        mk.load(K + k0 * a.ks[1], a.ks[1], kend - k0, a.D, true, [](int) { return true; });
        // values of masked keys count as zero: 0 x inf would not
        mv.load(V + k0 * a.vs[1], a.vs[1], kend - k0, a.D, !mask, [&](int r) { return mask[k0 + r] != 0; });
    };

    f32x16_t o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.f;
    const float c = a.scale * LOG2E;
    const unsigned rows_at = Tile<T, DP>::rows_at(lane), cols_at = Tile<T, DP>::cols_at(lane);
    if (ntiles > 0) fetch(0);
    fill_line(line, a, h, 256);                            // (the first tile's loads are in flight)
    if (ntiles > 0) {
        mk.store(lk);
        mv.store(lv);
    }
    arrived(qf);
    __syncthreads();
    for (int t = 0; t < ntiles; ++t) {
        const int k0 = t * KT, buf = (t & 1) * TILE;
        const unsigned ra = keep(rows_at) + buf * 2, ca = keep(cols_at) + buf * 2;
        if (t + 1 < ntiles) fetch(t + 1);
        f32x16_t x[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            x[kb] = zero16();
#pragma unroll
            for (int s = 0; s < KS; ++s) x[kb] = Mma<T>::mma(Tile<T, DP>::rows(lk, ra, kb * 32, s), qf[s], x[kb]);
        }
        // base-2 logits are mul x + add: one bias for a tile past an end of the line, else x takes its bias in place.  (One body for both:
        // two would cost a copy of the accumulators where they meet.)
        const int rel_hi = k0 + KT - 1 - w0 - start, rel_lo = k0 - (w0 + 31) - start;
        float mul = c, add = rel_hi <= -reach ? line[0] : line[last];
        if (rel_hi > -reach && rel_lo < right) {
            mul = 1.f;
            add = 0.f;
            const float* at = line + (k0 + 4 * half - qi - start + reach);          // entry of the lane's first key
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[kb][r] = fmaf(x[kb][r], c, at[kb * 32 + 8 * (r / 4) + r % 4]);
        }
        // keys the lane's query sees: bit n of `see` = key k0 + n
        if (mask || k0 + KT > first_limit) {
            unsigned long long bits = ~0ull;
            if (mask) bits = __ballot(k0 + lane < a.Nk && mask[min(k0 + lane, a.Nk - 1)]);
            const int lim = my_limit - k0;
            const unsigned long long see = lim >= 64 ? bits : lim <= 0 ? 0 : bits & ((1ull << lim) - 1);
            const unsigned s0 = (unsigned)see >> (4 * half), s1 = (unsigned)(see >> 32) >> (4 * half);
            if (!(add < INFINITY)) {                         // (a bias of NaN or +inf, added to -inf below, would reach rows that see none of these keys)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[kb][r] = fmaf(x[kb][r], c, add);
                mul = 1.f;
                add = 0.f;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x[0][r] = pick(s0, r, x[0][r], -INFINITY);
                x[1][r] = pick(s1, r, x[1][r], -INFINITY);
            }
        }
        const float mn = max2(m, fmaf(half_max(max2(max16(x[0]), max16(x[1]))), mul, add));
        if (__any(mn > m + SLACK)) {                         // (any new maximum: half of the tiles of 8160 keys instead of a few)
            const float alpha = exp2_hw(m - (mn == -INFINITY ? 0.f : mn));
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
            m = mn;
        }
        const float sub = SHIFT - (m == -INFINITY ? 0.f : m) + add;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x[kb][r] = exp2_hw(fmaf(x[kb][r], mul, sub));
                sum[r & 3] += x[kb][r];
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const v8 p = pack_step<T>(x[kb], s);
                v8 rest;
                if constexpr (LO) rest = pack_rest<T>(x[kb], p, s);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const v8 vf = Tile<T, DP>::cols(lv, ca, kb * 32 + s * 16, d);
                    o[d] = Mma<T>::mma(vf, p, o[d]);
                    if constexpr (LO) o[d] = Mma<T>::mma(vf, rest, o[d]);
                }
            }
        if (t + 1 < ntiles) {
            mk.store(lk + (TILE - buf));
            mv.store(lv + (TILE - buf));
        }
        __syncthreads();
    }
    const float sum = half_sum(l);
    const float inv = 1.f / sum;
    if (qi >= a.Nq) return;
    const long long row = ((long long)b * a.Nq + qi) * a.H + h;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = d * 32 + g * 8 + half * 4;
            if (at >= a.D) continue;
            typename Mma<T>::v4 w;
            f32x4_t f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[j] = empty_or(sum, o[d][4 * g + j] * inv);
                w[j] = (T)f[j];
            }
            *reinterpret_cast<typename Mma<T>::v4*>((T*)a.out + row * a.D + at) = w;
            if (LO) *reinterpret_cast<f32x4_t*>(a.out32 + row * a.D + at) = f;
        }
    if (a.lse && half == 0) a.lse[((long long)b * a.H + h) * a.Nq + qi] = sum == 0.f ? -INFINITY : m + log2f(sum) - SHIFT;
}

// ---- few queries (single tokens): bound by reading K and V once.  The G = H / Hkv heads that share keys times the queries are the 32
// columns of one score tile, so that shared keys are read once; the keys are cut into `splits` ranges for workgroups to fill the
// chip, and a range is dealt 32 keys at a time to 4 waves that keep their own maximum, sum and output and join at the end.
// K fragments go from memory to registers (a lane reads the 16 bytes it needs), V through a wave's own LDS rows to be transposed:
// no barrier inside the loop, the next 32 keys in flight.  8 caches of 32768 slots, 2 x 128 wide, bf16, lengths drawn between half
// and all (233 MB by the counters): 42 us = 5.5 TB/s (a plain read: 6.4), the join 4.7 us.
template <class T, int DP>
__global__ __launch_bounds__(256, 2) void attn_few_kernel(AttnArgs a) {
    typedef typename Mma<T>::v8 v8;
    constexpr int KS = DP / 16, DB = DP / 32, CH = DP / 8, PER = 32 * CH / 64;
    __shared__ __align__(16) T lv[4][32 * DP];                         // after the loop: 32 x DP floats of two waves at a time
    __shared__ float lm[4][32], ll[4][32];
    extern __shared__ float tab[];                                     // [buckets][G] in base 2, then the bucket of each line entry
    const int G = a.H / a.Hkv, rows = G * a.Nq;
    const int reach = line_reach(a.bk), right = line_right(a.bk), last = reach + right;
    unsigned char* bucket = (unsigned char*)(tab + a.bk.num_buckets * G);
    const int split = blockIdx.x % a.splits, rt = blockIdx.x / a.splits % a.tiles, bh = blockIdx.x / (a.splits * a.tiles);
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5, col = lane & 31;
    const int start = seq_start(a, b), len = seq_keys(a, b);
    const int kend = a.causal ? max(0, min(len, a.Nq + start)) : len;
    // this split's keys: an equal share of the existing ones, in whole rounds of 128
    const int share = (kend + a.splits * 128 - 1) / (a.splits * 128) * 128;
    const int ka = min(kend, split * share), kz = min(kend, ka + share);
    const int row = rt * 32 + col, g = min(row, rows - 1) / a.Nq, i = min(row, rows - 1) % a.Nq, h = hk * G + g;
    const bool live = row < rows;
    const T* Q = (const T*)a.q + b * a.qs[0] + h * a.qs[2] + (long long)i * a.qs[1];
    const T* K = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
    const T* V = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
    const unsigned char* mask = a.key_mask ? a.key_mask + (long long)b * a.Nk : nullptr;
    v8 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int d = s * 16 + half * 8;
        v8 z = {};
        qf[s] = z;
        if (live && d < a.D) qf[s] = *reinterpret_cast<const v8*>(Q + d);
    }
    v8 kf[KS];
    u32x4_t rv[PER];
    auto fetch = [&](int k0) {
        const int key = k0 + col;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 16 + half * 8;
            v8 z = {};
            kf[s] = z;
            if (key < kz && d < a.D) kf[s] = *reinterpret_cast<const v8*>(K + (long long)key * a.ks[1] + d);
        }
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int idx = n * 64 + lane, r = idx / CH, ch = idx % CH;
            u32x4_t z = {0, 0, 0, 0};
            rv[n] = z;
            if (k0 + r < kz && ch * 8 < a.D && (!mask || mask[k0 + r]))
                rv[n] = *reinterpret_cast<const u32x4_t*>(V + (long long)(k0 + r) * a.vs[1] + ch * 8);
        }
    };
    f32x16_t o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float c = a.scale * LOG2E;
    const unsigned cols_at = Tile<T, DP>::cols_at(lane);
    int k0 = ka + wave * 32;
    if (k0 < kz) fetch(k0);
    // (the first keys' loads are in flight)
    for (int t = threadIdx.x; t < a.bk.num_buckets * G; t += 256)
        tab[t] = base2_bias(a.table[(long long)(t / G) * a.H + hk * G + t % G]);
    for (int t = threadIdx.x; t <= last; t += 256) bucket[t] = (unsigned char)rel_bucket(a.bk, t - reach);
    __syncthreads();
    const float bias_lo = tab[bucket[0] * G + g], bias_hi = tab[bucket[last] * G + g];
    for (; k0 < kz; k0 += 128) {
        f32x16_t x;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) x = Mma<T>::mma(kf[s], qf[s], x);
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int idx = n * 64 + lane, r = idx / CH, ch = idx % CH;
            *reinterpret_cast<u32x4_t*>(&lv[wave][chunk_at<DP>(r, ch) * 8]) = rv[n];
        }
        unsigned bits = ~0u;
        if (mask) bits = (unsigned)__ballot(mask[min(k0 + col, a.Nk - 1)]);
        if (k0 + 128 < kz) fetch(k0 + 128);
        // one bias for the tile, or one for each element
        if (k0 + 31 - start <= -reach || k0 - (a.Nq - 1) - start >= right) {
            const float add = k0 + 31 - start <= -reach ? bias_lo : bias_hi;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], c, add);
        } else {
            const int at = k0 + 4 * half - i - start + reach;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int e = at + 8 * (r / 4) + r % 4;
                x[r] = fmaf(x[r], c, tab[bucket[min(max(e, 0), last)] * G + g]);
            }
        }
        const int lim = min(kz, a.causal ? i + start + 1 : kz) - k0;
        if (mask || k0 + 32 > kz || (a.causal && k0 + 32 > start + 1)) {
            const unsigned see = (lim >= 32 ? bits : lim <= 0 ? 0 : bits & ((1u << lim) - 1)) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = pick(see, r, x[r], -INFINITY);
        }
        const float mn = max2(m, half_max(max16(x)));
        const float base = mn == -INFINITY ? 0.f : mn;
        if (__any(mn > m)) {
            const float alpha = exp2_hw(m - base);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
            m = mn;
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[r] = exp2_hw(x[r] + (Mma<T>::shift - base));
            sum[r & 1] += x[r];
        }
        l += sum[0] + sum[1];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const v8 p = pack_step<T>(x, s);
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = Mma<T>::mma(Tile<T, DP>::cols(lv[wave], cols_at, s * 16, d), p, o[d]);
        }
    }
    // join the 4 waves: common maximum, then the outputs are added two waves at a time in LDS
    l = half_sum(l);
    if (half == 0) {
        lm[wave][col] = m;
        ll[wave][col] = l;
    }
    __syncthreads();
    float M = fmaxf(fmaxf(lm[0][col], lm[1][col]), fmaxf(lm[2][col], lm[3][col]));
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += ll[w][col] * exp2_hw(lm[w][col] - base);
    const float mine = exp2_hw(m - base);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= mine;
    // element (d, r) of a wave at [(d 16 + r) 64 + lane]: DP / 2 x 64 floats = 32 DP a wave, the size of two waves' V rows
    float* red = reinterpret_cast<float*>(&lv[0][0]);
    constexpr int WORDS = 32 * DP;
    for (int step = 2; step > 0; step >>= 1) {
        __syncthreads();
        if (wave >= step && wave < 2 * step)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) red[(wave - step) * WORDS + (d * 16 + r) * 64 + lane] = o[d][r];
        __syncthreads();
        if (wave < step)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] += red[wave * WORDS + (d * 16 + r) * 64 + lane];
    }
    if (wave != 0 || !live) return;
    const long long out_row = ((long long)b * a.Nq + i) * a.H + h;
    if (a.splits == 1) {
        const float inv = 1.f / L;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int at = d * 32 + q * 8 + half * 4;
                if (at >= a.D) continue;
                typename Mma<T>::v4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (T)empty_or(L, o[d][4 * q + j] * inv);
                *reinterpret_cast<typename Mma<T>::v4*>((T*)a.out + out_row * a.D + at) = w;
            }
        if (a.lse && half == 0) a.lse[((long long)b * a.H + h) * a.Nq + i] = L == 0.f ? -INFINITY : M + log2f(L) - Mma<T>::shift;
        return;
    }
    // partial [split][out_row][D + 2]: output, maximum, sum
    float* part = a.partial + ((long long)split * a.B * a.Nq * a.H + out_row) * (a.D + 4);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = d * 32 + q * 8 + half * 4;
            if (at < a.D) *reinterpret_cast<float4*>(part + at) = make_float4(o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]);
        }
    if (half == 0) {
        part[a.D] = M;
        part[a.D + 1] = L;
    }
}

// joins the splits of a row: a workgroup a row, a wave every fourth split, a lane 2 channels (D <= 128); all of a wave's loads are in
// flight at once, the waves meet in LDS.  128 rows of 16 splits, width 128: 4.8 us, a launch
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    __shared__ float red[4][64 * 2 + 1];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const long long rows = (long long)a.B * a.Nq * a.H, row = blockIdx.x;
    const int ld = a.D + 4, d = lane * 2;
    const float* p = a.partial + row * ld;
    const long long step = rows * ld;
    float M = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) M = max2(M, p[s * step + a.D]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = max2(M, __shfl_xor(M, o, 64));
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 8
    for (int s = wave; s < a.splits; s += 4) {
        const float w = exp2_hw(p[s * step + a.D] - base);
        float2 f = make_float2(0.f, 0.f);
        if (d < a.D) f = *reinterpret_cast<const float2*>(p + s * step + d);
        L += w * p[s * step + a.D + 1];
        o0 += w * f.x;
        o1 += w * f.y;
    }
    red[wave][d] = o0;
    red[wave][d + 1] = o1;
    if (lane == 0) red[wave][128] = L;
    __syncthreads();
    if (wave) return;
    L = (red[0][128] + red[1][128]) + (red[2][128] + red[3][128]);
    o0 = (red[0][d] + red[1][d]) + (red[2][d] + red[3][d]);
    o1 = (red[0][d + 1] + red[1][d + 1]) + (red[2][d + 1] + red[3][d + 1]);
    const float inv = 1.f / L;
    if (d < a.D) {
        typename Mma<T>::v2 w = {(T)empty_or(L, o0 * inv), (T)empty_or(L, o1 * inv)};
        *reinterpret_cast<typename Mma<T>::v2*>((T*)a.out + row * a.D + d) = w;
    }
    if (a.lse && lane == 0) {
        const long long b = row / ((long long)a.Nq * a.H), i = row / a.H % a.Nq, h = row % a.H;
        a.lse[(b * a.H + h) * a.Nq + i] = L == 0.f ? -INFINITY : M + log2f(L) - Mma<T>::shift;
    }
}

// ---------------------------------------------------------------------------------------------- host side
static_assert(sizeof(tcvom_attn_desc) == 664, "tcvom_amd/_lib.py: AttnDesc");
int attn_check(const char* who, const tcvom_attn_desc* d, AttnArgs* a) {
    if (!d) return tcvom_fail(TCVOM_ERR_ARG, "%s: null description", who);
    TCVOM_CHECK_ARG(d->type == TCVOM_TYPE_BF16 || d->type == TCVOM_TYPE_F16, "%s: type %d", who, d->type);
    TCVOM_CHECK_ARG(d->B >= 0 && d->H > 0 && d->Hkv > 0 && d->H % d->Hkv == 0, "%s: B=%d H=%d Hkv=%d", who, d->B, d->H, d->Hkv);
    TCVOM_CHECK_ARG(d->D >= 8 && d->D <= 128 && d->D % 8 == 0, "%s: head width %d (8..128, a multiple of 8)", who, d->D);
    TCVOM_CHECK_ARG(d->Nq >= 0 && d->Nk >= 0 && d->Nq <= (1 << 28) && d->Nk <= (1 << 28), "%s: Nq=%d Nk=%d", who, d->Nq, d->Nk);
    TCVOM_CHECK_ARG(d->q_start >= -(1 << 29) && d->q_start <= (1 << 29), "%s: q_start=%d", who, d->q_start);
    TCVOM_CHECK_ARG(d->scale > 0.f && d->scale < INFINITY, "%s: scale %g", who, d->scale);
    for (int n = 0; n < 3; ++n)
        TCVOM_CHECK_ARG(d->q_stride[n] % 8 == 0 && d->k_stride[n] % 8 == 0 && d->v_stride[n] % 8 == 0 && d->q_stride[n] >= 0 &&
                            d->k_stride[n] >= 0 && d->v_stride[n] >= 0, "%s: strides are multiples of 8 elements", who);
    TCVOM_CHECK_ARG(d->q_stride[1] < (1 << 24) && d->k_stride[1] < (1 << 24) && d->v_stride[1] < (1 << 24), "%s: tokens 2^24 elements apart", who);
    if (const int rc = check_buckets(who, &d->buckets)) return rc;
    *a = AttnArgs();
    a->B = d->B; a->Nq = d->Nq; a->Nk = d->Nk; a->H = d->H; a->Hkv = d->Hkv; a->D = d->D;
    a->causal = d->causal; a->q_start = d->q_start; a->scale = d->scale;
    a->k_lens = d->k_lens; a->q_starts = d->q_starts; a->key_mask = d->key_mask; a->bk = pad_buckets(d->buckets);
    for (int n = 0; n < 3; ++n) { a->qs[n] = d->q_stride[n]; a->ks[n] = d->k_stride[n]; a->vs[n] = d->v_stride[n]; }
    return 0;
}

// few queries: attn_few_kernel, whose LDS holds the biases of up to 64 heads that share keys
static bool attn_few(const tcvom_attn_desc* d) { return d->Nq <= 32 && d->H / d->Hkv <= 64; }
static void few_shape(const tcvom_attn_desc* d, int* tiles, int* splits) {
    *tiles = cdiv((long long)d->H / d->Hkv * d->Nq, 32);
    const long long wgs = (long long)d->B * d->Hkv * *tiles;
    // a workgroup a CU (two: 1 to 10 % slower), and at least 256 keys a workgroup (the join is a launch of 4 us)
    long long s = wgs ? 256 / wgs : 1;
    const long long most = d->Nk / 256;
    if (s > most) s = most;
    *splits = (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

extern "C" int64_t tcvom_attn_fwd_work(const tcvom_attn_desc* d) {
    if (!d || d->B <= 0 || d->Nq <= 0 || d->Hkv <= 0 || !attn_few(d)) return 0;
    int tiles, splits;
    few_shape(d, &tiles, &splits);
    return splits > 1 ? (int64_t)splits * d->B * d->Nq * d->H * (d->D + 4) : 0;
}

template <class T, int DP>
static void launch_fwd(AttnArgs a, const tcvom_attn_desc* d, hipStream_t st) {
    if (attn_few(d) && !a.out32) {
        const int last = line_reach(a.bk) + line_right(a.bk);
        few_shape(d, &a.tiles, &a.splits);
        const size_t lds = sizeof(float) * a.bk.num_buckets * (a.H / a.Hkv) + last + 1;
        const dim3 grid((unsigned)((long long)a.B * a.Hkv * a.tiles * a.splits));
        hipLaunchKernelGGL((attn_few_kernel<T, DP>), grid, dim3(256), lds, st, a);
        if (a.splits > 1)
            hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)((long long)a.B * a.Nq * a.H)), dim3(256), 0, st, a);
        return;
    }
    a.tiles = cdiv(a.Nq, 128);
    const dim3 grid((unsigned)((long long)a.B * a.H * a.tiles));
    const size_t lds = line_bytes(a);
    if (a.out32) hipLaunchKernelGGL((attn_fwd_kernel<T, DP, true>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((attn_fwd_kernel<T, DP, false>), grid, dim3(256), lds, st, a);
}

extern "C" int tcvom_attn_fwd(const tcvom_attn_desc* d, const void* q, const void* k, const void* v, const float* table, void* out,
                              float* out32, float* lse, float* work, int64_t work_floats, void* stream) {
    AttnArgs a;
    if (const int rc = attn_check("attn_fwd", d, &a)) return rc;
    if (d->B == 0 || d->Nq == 0) return 0;
    TCVOM_CHECK_ARG(q && table && out && (d->Nk == 0 || (k && v)), "attn_fwd: null tensor");
    TCVOM_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(out32), "attn_fwd: tensors start at multiples of 16 bytes");
    TCVOM_CHECK_ARG((long long)d->B * d->H * cdiv(d->Nq, 128) <= TCVOM_MAX_ATTN_WORKGROUPS, "attn_fwd: %d sequences x %d heads x %d queries", d->B, d->H, d->Nq);
    TCVOM_CHECK_ARG(work_floats >= tcvom_attn_fwd_work(d) && (work || tcvom_attn_fwd_work(d) == 0), "attn_fwd: %lld floats of workspace",
                    (long long)work_floats);
    a.q = q; a.k = k; a.v = v; a.table = table; a.out = out; a.out32 = out32; a.lse = lse; a.partial = work;
    const hipStream_t st = (hipStream_t)stream;
    const int DP = attn_width(d->D);
    if (d->type == TCVOM_TYPE_BF16) {
        if (DP == 32) launch_fwd<__bf16, 32>(a, d, st);
        else if (DP == 64) launch_fwd<__bf16, 64>(a, d, st);
        else launch_fwd<__bf16, 128>(a, d, st);
    } else {
        if (DP == 32) launch_fwd<_Float16, 32>(a, d, st);
        else if (DP == 64) launch_fwd<_Float16, 64>(a, d, st);
        else launch_fwd<_Float16, 128>(a, d, st);
    }
    TCVOM_LAUNCH_CHECK("attn_fwd");
    return 0;
}
