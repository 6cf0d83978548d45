// Shared by the token operators (relbias.hip, attn*.hip, blocknorm*.hip): element types, 16-byte vectors, bucket arithmetic.
//
// Unlike the convolution kernels, which store the ONE 16-bit type of their build, these kernels are compiled for bf16, IEEE fp16 and
// (where it makes sense) fp32 elements in both builds and take the type as an argument (TCVOM_TYPE_F32 / TCVOM_TYPE_BF16 / TCVOM_TYPE_F16).  Their
// 16-bit stores round to nearest even and keep inf and NaN (no saturation): an overflow stays visible, as in torch.
#pragma once
#include "common.h"

template <class T> struct Elem;
template <> struct Elem<float> { static constexpr int kind = TCVOM_TYPE_F32; };
template <> struct Elem<__bf16> { static constexpr int kind = TCVOM_TYPE_BF16; };
template <> struct Elem<_Float16> { static constexpr int kind = TCVOM_TYPE_F16; };

// V consecutive elements at p as floats / from floats.  The types carry the alignment of one element: rows of an odd length start anywhere,
// and global memory takes 16-byte accesses at any address.
template <class T, int V> struct RawVec {
    typedef T type __attribute__((ext_vector_type(V)));
    typedef type any __attribute__((aligned(sizeof(T))));
};
template <class T, int V>
__device__ __forceinline__ typename RawVec<T, V>::type load_raw(const T* p) {
    return *reinterpret_cast<const typename RawVec<T, V>::any*>(p);
}
template <class T, int V>
__device__ __forceinline__ void raw_to_float(const typename RawVec<T, V>::type& q, float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = (float)q[j];
}
template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[V]) { raw_to_float<T, V>(load_raw<T, V>(p), f); }
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
    typename RawVec<T, V>::type q;
#pragma unroll
    for (int j = 0; j < V; ++j) q[j] = (T)f[j];
    *reinterpret_cast<typename RawVec<T, V>::any*>(p) = q;
}
// the first n of them (n <= V), the others zero / left alone
template <class T, int V>
__device__ __forceinline__ typename RawVec<T, V>::type load_first(const T* p, int n) {
    typename RawVec<T, V>::type q = (typename RawVec<T, V>::type)(T)0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) q[j] = p[j];
    return q;
}
template <class T, int V>
__device__ __forceinline__ void store_first(T* p, const float (&f)[V], int n) {
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) p[j] = (T)f[j];
}

// ---- buckets of relative positions (tcvom_rel_buckets, include/tcvom_hip.h)
// A bias depends on the clamped distance rel = key - query only, and every rel <= -reach shares one bucket, every rel >= right another:
// the kernels work on the "line" of values at rel = -reach .. right (reach = starts[n_starts - 1], right = reach if bidirectional else 0).
__host__ __device__ __forceinline__ int line_reach(const tcvom_rel_buckets& b) { return b.starts[b.n_starts - 1]; }
__host__ __device__ __forceinline__ int line_right(const tcvom_rel_buckets& b) { return b.bidirectional ? line_reach(b) : 0; }
// bucket of rel: a uniform loop over the borders, 16 at a time (one scalar load of the kernel arguments; pad_buckets fills the last 16)
__device__ __forceinline__ int rel_bucket(const tcvom_rel_buckets& b, int rel) {
    const int d = rel < 0 ? -rel : (b.bidirectional ? rel : 0);
    int n = d;
    if (d >= b.exact) n = b.exact - 1;
    for (int k = 0; k < b.n_starts; k += 16) {
        int more = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) more += d >= b.starts[k + i];
        n += more;                                            // (a distance below `exact` is below every border)
    }
    return n + (b.bidirectional && rel > 0 ? b.num_buckets / 2 : 0);
}
static_assert(TCVOM_MAX_BUCKET_STARTS % 16 == 0, "rel_bucket reads the borders 16 at a time");
static inline tcvom_rel_buckets pad_buckets(const tcvom_rel_buckets& b) {
    tcvom_rel_buckets p = b;
    for (int k = b.n_starts; k < TCVOM_MAX_BUCKET_STARTS; ++k) p.starts[k] = 1 << 30;
    return p;
}
// the line entries of bucket b: t0 <= t < t1 (possibly none)
__device__ __forceinline__ void bucket_entries(const tcvom_rel_buckets& bk, int b, int& t0, int& t1) {
    const int side = bk.bidirectional ? bk.num_buckets / 2 : bk.num_buckets, reach = line_reach(bk);
    const bool right = b >= side;
    const int n = right ? b - side : b;
    int d0 = n < bk.exact ? n : bk.starts[n - bk.exact];
    int d1 = n + 1 < bk.exact ? n + 1 : n + 1 < side ? bk.starts[n + 1 - bk.exact] : reach + 1;      // (the last bucket: distance reach)
    if (d1 > reach + 1) d1 = reach + 1;
    if (right) {
        if (d0 < 1) d0 = 1;
        t0 = reach + d0;
        t1 = reach + d1;
    } else {
        t0 = reach - d1 + 1;
        t1 = reach - d0 + 1;
    }
}

// host-side check of a bucket description; 0 or an error code with the message set
static inline int check_buckets(const char* who, const tcvom_rel_buckets* b) {
    if (!b) return tcvom_fail(TCVOM_ERR_ARG, "%s: null bucket description", who);
    const int side = b->bidirectional ? b->num_buckets / 2 : b->num_buckets;
    if (b->num_buckets < 2 || b->num_buckets > TCVOM_MAX_BUCKETS || (b->bidirectional && (b->num_buckets & 1)))
        return tcvom_fail(TCVOM_ERR_ARG, "%s: %d buckets (2..%d, even if bidirectional)", who, b->num_buckets, TCVOM_MAX_BUCKETS);
    if (b->exact < 1 || b->n_starts != side - b->exact || b->n_starts < 1 || b->n_starts > TCVOM_MAX_BUCKET_STARTS)
        return tcvom_fail(TCVOM_ERR_ARG, "%s: %d exact + %d shared buckets do not make %d a side", who, b->exact, b->n_starts, side);
    if (b->starts[0] != b->exact) return tcvom_fail(TCVOM_ERR_ARG, "%s: shared buckets start at %d, not %d", who, b->starts[0], b->exact);
    for (int k = 1; k < b->n_starts; ++k)
        if (b->starts[k] < b->starts[k - 1]) return tcvom_fail(TCVOM_ERR_ARG, "%s: bucket borders decrease", who);
    if (line_reach(*b) > TCVOM_MAX_BUCKET_REACH)
        return tcvom_fail(TCVOM_ERR_ARG, "%s: the last bucket starts at distance %d (at most %d)", who, line_reach(*b), TCVOM_MAX_BUCKET_REACH);
    return 0;
}

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
