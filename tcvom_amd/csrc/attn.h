// Attention with a bucketed relative position bias, shared by attn.hip (forward) and attn_bwd.hip.
//     x[i][j] = scale <q_i, k_j> + bias[h][j - i - q_start],   p = softmax over the keys row i sees,   out_i = sum_j p[i][j] v_j
//
// Products on v_mfma_f32_32x32x16.  Scores are formed TRANSPOSED, S^T = K Q^T (rows = keys, columns = queries): a lane then holds one
// query (column lane & 31) and 16 keys of each 32-key block, key 8 (r / 4) + 4 (lane >> 5) + r % 4 in register r, so that a row's maximum
// and sum are sums inside the lane plus one exchange with lane ^ 32, and the exponentials, rounded to 16 bits, ARE the second
// operand of O^T = V^T P^T: the contraction index is permuted the same way on both sides (the transposing LDS read of V takes its 4-key
// rows in that order).  Everything is in base 2: scale and bias are multiplied by log2(e) once.
//
// A head's bias is a "line" of values over the clamped relative position (token_common.h) in LDS.  A tile of keys whose relative
// positions all lie past one end of the line adds a constant; the others read the line, 4 consecutive entries for 4 keys.
#pragma once
#include "token_common.h"

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2_t;

template <class T> struct Mma;
template <> struct Mma<__bf16> {
    typedef __attribute__((ext_vector_type(8))) __bf16 v8;
    typedef __attribute__((ext_vector_type(4))) __bf16 v4;
    typedef __attribute__((ext_vector_type(2))) __bf16 v2;
    static __device__ __forceinline__ f32x16_t mma(v8 a, v8 b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ v4 tr(const __bf16* p) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) v4*)p);
    }
    static constexpr float shift = 0.f;
};
template <> struct Mma<_Float16> {
    typedef __attribute__((ext_vector_type(8))) _Float16 v8;
    typedef __attribute__((ext_vector_type(4))) _Float16 v4;
    typedef __attribute__((ext_vector_type(2))) _Float16 v2;
    static __device__ __forceinline__ f32x16_t mma(v8 a, v8 b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ v4 tr(const _Float16* p) {
        typedef __attribute__((ext_vector_type(4))) __fp16 h4;
        return __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4*)p));
    }
    // probabilities are held as 2^shift p: most of a long row lies below fp16's smallest normal number, 2^-14
    static constexpr float shift = 15.f;
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KT = 64;                       // keys a tile

struct AttnArgs {
    const void *q, *k, *v;
    const float* table;                      // [buckets][H]
    void* out;                               // [B][Nq][H][D]
    float* out32;                            // ... before it is rounded, for the backward, or null
    float* lse;                              // [B][H][Nq], base 2, -inf for a row without a key
    const void* dout;
    void *dq, *dk, *dv;
    float *delta, *part, *dtable;            // backward: <dout, out> of every row; bucket sums of every workgroup; their result or null
    float* partial;                          // forward: the splits' outputs; backward: each head's dk and dv where a group is taken apart
    const int *k_lens, *q_starts;            // [B] or null
    const unsigned char* key_mask;           // [B][Nk] or null
    long long qs[3], ks[3], vs[3], dos[3];   // strides of batch, token, head in elements
    int B, Nq, Nk, H, Hkv, D, causal, q_start, splits, tiles, apart;
    float scale;                             // softmax scale, natural
    tcvom_rel_buckets bk;
};

// keys of sequence b that exist, and the position of its first query
__device__ __forceinline__ int seq_keys(const AttnArgs& a, int b) {
    if (!a.k_lens) return a.Nk;
    const int n = a.k_lens[b];
    return n < 0 ? 0 : n > a.Nk ? a.Nk : n;
}
__device__ __forceinline__ int seq_start(const AttnArgs& a, int b) {
    if (!a.q_starts) return a.q_start;
    const int s = a.q_starts[b];
    return s < -(1 << 29) ? -(1 << 29) : s > (1 << 29) ? (1 << 29) : s;
}

// workgroup -> (sequence and head, tile).  The hardware deals workgroups round-robin over the 8 XCDs, each with its own L2: the tiles of a
// head, which share keys and values (or queries), stay on one.  Tiles of causal heads differ in work: all heads' longest ones go
// first, so that none starts late (2 x 4080 tokens, 16 heads of 128: see attn_dkv_kernel); otherwise head by head, the fewest heads in an L2.
__device__ __forceinline__ void work_item(const AttnArgs& a, int id, int heads, int& bh, int& tile) {
    const int total = heads * a.tiles;
    if (a.causal && heads % 8 == 0) {
        tile = id / heads;
        bh = id % heads;
        return;
    }
    const int per = total / 8, whole = per * 8, item = id < whole ? (id & 7) * per + (id >> 3) : id;
    bh = item / a.tiles;
    tile = item % a.tiles;
}

// LDS position of 16-byte chunk c of row r, rows of DP elements.  The XOR spreads over the 64 banks (256 bytes) both (a) fragment reads, 16
// consecutive rows at one chunk, and (b) transposing reads, 4 consecutive rows at 4 consecutive chunks.
template <int DP> __device__ __forceinline__ int chunk_at(int r, int c) {
    if constexpr (DP == 128) return r * 16 + (c ^ (((r & 3) << 2) | ((r >> 2) & 3)));
    else if constexpr (DP == 64) return r * 8 + (c ^ (((r & 2) << 1) | ((r >> 2) & 3)));
    else return r * 4 + (c ^ ((r >> 2) & 3));
}

// NaN stays NaN; v_maximum3_f32
__device__ __forceinline__ float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max3(float a, float b, float c) { return max2(max2(a, b), c); }
__device__ __forceinline__ float half_max(float v) {       // maximum over lanes l and l ^ 32
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

template <class T>
__device__ __forceinline__ typename Mma<T>::v8 join(typename Mma<T>::v4 lo, typename Mma<T>::v4 hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// registers 8 s .. 8 s + 7 of a 32 x 32 block as the 16-bit operand of k-step s
template <class T>
__device__ __forceinline__ typename Mma<T>::v8 pack_step(const f32x16_t& p, int s) {
    typename Mma<T>::v8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)p[8 * s + i];
    return r;
}
// ... and what that rounding dropped, rounded again
template <class T>
__device__ __forceinline__ typename Mma<T>::v8 pack_rest(const f32x16_t& p, typename Mma<T>::v8 hi, int s) {
    typename Mma<T>::v8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)(p[8 * s + i] - (float)hi[i]);
    return r;
}

// Score gradients ds = p (dp - delta) as 16-bit operands.  They are as large as dout times p: in fp16 those of a long row, or of a small dout, lie
// below 2^-14, its smallest normal number, and those of a large dout times large values beyond its largest.  fp16 therefore holds
// 2^e ds, with an e (here up = 2^e) for each column of the product, a query of dq and a key of dk, that falls whenever a block of the column
// would pass 2^15: the block's largest then becomes 2^11 .. 2^12, the sums so far follow (times a power of two: no rounding), and 2^-e
// comes off in 32 bits at the store.  What is 2^26 times smaller than a column's largest still is a normal number.  bf16 has the exponents of
// fp32 and needs none of it.  4 x 1024 tokens, 8 heads of 64, fp16: dq
// 41.6 -> 43.0 us, dk / dv 39.8 -> 45.3 us; 2 x 4080 causal, 16 heads of 128 on 4: 268 -> 284 and 351 -> 363 us.
template <class T> constexpr float DS_UP = Mma<T>::shift > 0.f ? 0x1p100f : 1.f;
template <class T, int DB>
__device__ __forceinline__ void ds_fit(const f32x16_t& x, float& up, f32x16_t (&sums)[DB]) {
    if constexpr (Mma<T>::shift > 0.f) {
        float t[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) t[n] = max3(fabsf(x[4 * n]), fabsf(x[4 * n + 1]), fabsf(x[4 * n + 2]));
        const float top = half_max(max3(max3(t[0], fabsf(x[3]), t[1]), max3(fabsf(x[7]), t[2], fabsf(x[11])), max2(t[3], fabsf(x[15]))));
        if (__any(top * up > 32768.f)) {
            const int e = __builtin_amdgcn_frexp_expf(up) - 1, now = top * up > 32768.f ? min(e, 12 - __builtin_amdgcn_frexp_expf(top)) : e;
            const float f = ldexpf(1.f, now - e);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) sums[d][r] *= f;
            up = ldexpf(1.f, now);
        }
    }
}
template <class T>
__device__ __forceinline__ typename Mma<T>::v8 pack_ds(const f32x16_t& x, float up, int s) {
    if constexpr (!(Mma<T>::shift > 0.f)) return pack_step<T>(x, s);
    typename Mma<T>::v8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)(x[8 * s + i] * up);
    return r;
}
template <class T>
__device__ __forceinline__ float ds_down(float sum, float up) {
    return Mma<T>::shift > 0.f ? ldexpf(sum, 1 - __builtin_amdgcn_frexp_expf(up)) : sum;
}

// v, computed here: not hoisted out of a loop into a register of its own
__device__ __forceinline__ unsigned keep(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}
// v has arrived from memory from here on.  Without it the compiler, which cannot tell a loop's first turn from the others, waits for such a
// load inside the loop -- and with it for the next tile's, issued just before.
template <class V8, int N> __device__ __forceinline__ void arrived(V8 (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}
// Operands from an LDS tile of rows of DP elements (layout: chunk_at).  A lane's byte offset differs between steps by an XOR of a few low
// bits and a constant, so that one register and one instruction a step address them all.
template <class T, int DP> struct Tile {
    typedef typename Mma<T>::v8 v8;
    static constexpr int ROW = DP * 2;
    // rows r0 + (lane & 31), columns 16 s + 8 (lane >> 5) ..: operand of a product over the columns
    static __device__ __forceinline__ unsigned rows_at(int lane) { return chunk_at<DP>(lane & 31, lane >> 5) * 16; }
    static __device__ __forceinline__ v8 rows(const T* tile, unsigned off, int r0, int s) {
        return *reinterpret_cast<const v8*>(reinterpret_cast<const char*>(tile) + (off ^ (s << 5)) + r0 * ROW);
    }
    // column 32 d + (lane & 31), 16 rows from r0 (a multiple of 16) in the order of the score registers: operand of a product that
    // contracts the rows
    static __device__ __forceinline__ unsigned cols_at(int lane) {
        return chunk_at<DP>(4 * (lane >> 5) + ((lane & 15) >> 2), ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;
    }
    static __device__ __forceinline__ v8 cols(const T* tile, unsigned off, int r0, int d) {
        const char* p = reinterpret_cast<const char*>(tile) + r0 * ROW;
        return join<T>(Mma<T>::tr(reinterpret_cast<const T*>(p + (off ^ (d << 6)))),
                       Mma<T>::tr(reinterpret_cast<const T*>(p + (off ^ (d << 6) ^ 32) + 8 * ROW)));
    }
};
// 16 bytes of a row, zeros where `ok` is false
template <class V8, class T>
__device__ __forceinline__ V8 load_or_zero(bool ok, const T* p) {
    V8 z = {};
    if (ok) z = *reinterpret_cast<const V8*>(p);
    return z;
}
// One thread's share of moving a tile of ROWS rows from memory to registers and on to LDS (256 threads): rows threadIdx.x / CH + n 256 / CH,
// 16-byte chunk threadIdx.x % CH.
template <class T, int DP, int ROWS> struct Mover {
    static constexpr int CH = DP / 8, STEP = 256 / CH, PER = (ROWS * CH + 255) / 256;
    u32x4_t reg[PER];
    // rows `first` .. of the tile whose row 0 is at `base`; `left` of them exist, `ok(row)` says which count; the others are zeros
    template <class F>
    __device__ __forceinline__ void load(const T* base, long long stride, int left, int D, bool all, F ok) {
        const unsigned tid = DP == 128 ? keep(threadIdx.x) : threadIdx.x;        // (the widest kernels have no registers to hold offsets in)
        const int r0 = tid / CH, c = tid % CH;
        const unsigned off = (unsigned)(r0 * (int)stride + c * 8) * 2u;         // strides below 2^24 (attn_check)
        if (left >= ROWS && D == DP && all && (ROWS * CH) % 256 == 0) {
#pragma unroll
            for (int n = 0; n < PER; ++n)
                reg[n] = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const char*>(base + n * STEP * stride) + off);
            asm volatile("; whole tile");           // (else the last load is shared with the other form, behind its zeroes and their wait)
            return;
        }
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int r = r0 + n * STEP;
            u32x4_t z = {0, 0, 0, 0};
            if (r < ROWS && r < left && c * 8 < D && (all || ok(r)))
                z = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const char*>(base + n * STEP * stride) + off);
            reg[n] = z;
        }
    }
    __device__ __forceinline__ void store(T* tile) const {
        const unsigned tid = DP == 128 ? keep(threadIdx.x) : threadIdx.x;
        const int r0 = tid / CH, c = tid % CH;
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int r = r0 + n * STEP;
            if ((ROWS * CH) % 256 == 0 || r < ROWS) *reinterpret_cast<u32x4_t*>(&tile[chunk_at<DP>(r, c) * 8]) = reg[n];
        }
    }
};
__device__ __forceinline__ float max16(const f32x16_t& x) {
    return max3(max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[8])),
                max3(max3(x[9], x[10], x[11]), x[12], x[13]), max2(x[14], x[15]));
}
// x where the bit of `see` is set, else `other`; register r of a block stands for bit 8 (r / 4) + r % 4
__device__ __forceinline__ float pick(unsigned see, int r, float x, float other) {
    const unsigned m = (unsigned)__builtin_amdgcn_sbfe((int)see, 8 * (r / 4) + r % 4, 1);
    return __uint_as_float((__float_as_uint(x) & m) | (__float_as_uint(other) & ~m));
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }      // (a scalar: branches on it are uniform)
__device__ __forceinline__ f32x16_t zero16() {
    f32x16_t z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
// A bias in base 2.  Finite ones end at +-2^17: a larger one would swallow the score it is added to, and the rounding of maximum + bias
// (half of 2^-6 there, 64 at 1e9) becomes a factor on the row's probabilities.  Infinite ones stay: -inf takes a distance out.
__device__ __forceinline__ float base2_bias(float v) {
    const float x = v * LOG2E;
    return fabsf(x) > 131072.f && fabsf(v) != INFINITY ? copysignf(131072.f, x) : x;
}
// the line of head h, in base 2, in line[0 .. last]; its two ends are repeated MARGIN entries outwards, so that a tile of 64 x 64 that
// crosses the line reads it without clamping
constexpr int MARGIN = 128;
// ... returns whether this thread wrote a NaN or +inf
__device__ __forceinline__ bool fill_line(float* line, const AttnArgs& a, int h, int threads) {
    const int reach = line_reach(a.bk), last = reach + line_right(a.bk);
    bool odd = false;
    for (int t = (int)threadIdx.x - MARGIN; t <= last + MARGIN; t += threads) {
        const float v = base2_bias(a.table[rel_bucket(a.bk, min(max(t, 0), last) - reach) * a.H + h]);
        line[t] = v;
        odd |= !(v < INFINITY);
    }
    return odd;
}
static inline size_t line_bytes(const AttnArgs& a) { return sizeof(float) * (line_reach(a.bk) + line_right(a.bk) + 1 + 2 * MARGIN); }

// host side
static_assert(TCVOM_MAX_ATTN_WORKGROUPS < (1LL << 32) / 256, "a grid has fewer than 2^32 threads");
int attn_check(const char* who, const tcvom_attn_desc* d, AttnArgs* a);
static inline int attn_width(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
