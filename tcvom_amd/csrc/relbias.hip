// The relative position bias by buckets as a matrix, and the gradient of its table (tcvom_relbias_fwd / tcvom_relbias_bwd).
//     bias[h][i][j] = table[bucket(j - i - q_start)][h]          dtable[b][h] = sum over i, j with that bucket of dbias[h][i][j]
// Bound: HBM bytes of the matrix, written once (read once).  See token_common.h for the "line" of distinct values of a head.
#include "token_common.h"

// ---- forward: a wave a row.  The head's line is formed once a workgroup in LDS; a 16-byte vector whose distances all lie past one end
// of the line is a constant, the others look each element up.  8 x 2040 x 8160 bf16: 42 us = 6.3 TB/s (a fill reaches 6.9); 12 x 2041 x 2041
// fp32: 33 us = 6.1 TB/s; 8 x 1024 x 1024 bf16: 8.1 us.
template <class T>
__global__ __launch_bounds__(256) void relbias_fwd_kernel(const float* table, T* out, tcvom_rel_buckets bk, int heads, long long Nq,
                                                          long long Nk, long long q_start, int rows_per_wg) {
    extern __shared__ float line[];
    constexpr int V = 16 / sizeof(T);
    const int h = blockIdx.y, reach = line_reach(bk), right = line_right(bk), last = reach + right;
    for (int t = threadIdx.x; t <= last; t += 256) line[t] = table[rel_bucket(bk, t - reach) * heads + h];
    __syncthreads();
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float lo = line[0], hi = line[last];
    const long long i1 = min(Nq, ((long long)blockIdx.x + 1) * rows_per_wg);
    for (long long i = (long long)blockIdx.x * rows_per_wg + wave; i < i1; i += 4) {
        T* row = out + ((long long)h * Nq + i) * Nk;
        const long long shift = reach - i - q_start;              // line index of key j is j + shift, clamped
        auto at = [&](long long j) {
            const long long t = j + shift;
            return line[t < 0 ? 0 : t > last ? last : t];
        };
        // elements in front of the first 16-byte boundary, then whole vectors, then the tail
        long long head = ((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T);
        if (head > Nk) head = Nk;
        if (lane < head) row[lane] = (T)at(lane);
        const long long nv = (Nk - head) / V;
        for (long long n = lane; n < nv; n += 64) {
            const long long j = head + n * V;
            float f[V];
            if (j + V - 1 + shift <= 0 || j + shift >= last) {
                const float c = j + shift >= last ? hi : lo;
#pragma unroll
                for (int u = 0; u < V; ++u) f[u] = c;
            } else {
#pragma unroll
                for (int u = 0; u < V; ++u) f[u] = at(j + u);
            }
            store_vec<T, V>(row + j, f);
        }
        const long long j = head + nv * V + lane;
        if (j < Nk) row[j] = (T)at(j);
    }
}

extern "C" int tcvom_relbias_fwd(const float* table, void* out, const tcvom_rel_buckets* buckets, int32_t heads, int64_t q_len,
                                 int64_t k_len, int64_t q_start, int32_t type, void* stream) {
    TCVOM_CHECK_ARG(table && (out || q_len == 0 || k_len == 0) && heads > 0 && heads <= 65535 && q_len >= 0 && k_len >= 0, "relbias_fwd: heads=%d q_len=%lld k_len=%lld",
                    heads, (long long)q_len, (long long)k_len);
    TCVOM_CHECK_ARG(type >= TCVOM_TYPE_F32 && type <= TCVOM_TYPE_F16, "relbias_fwd: type %d", type);
    TCVOM_CHECK_ARG(q_len < (1LL << 31) && k_len < (1LL << 31) && q_start < (1LL << 40) && q_start > -(1LL << 40), "relbias_fwd: lengths");
    if (const int rc = check_buckets("relbias_fwd", buckets)) return rc;
    const tcvom_rel_buckets bk = pad_buckets(*buckets);
    if (q_len == 0 || k_len == 0) return 0;
    // 64 KB of output and more a workgroup, but at least 8 workgroups a CU while there are rows for it
    int64_t rows = cdiv(65536, k_len * (type == TCVOM_TYPE_F32 ? 4 : 2));
    const int64_t few = cdiv(q_len * heads, 2048);
    rows = ((rows < few ? rows : few) + 3) / 4 * 4;
    const int64_t fill = cdiv(q_len, 1 << 20) * 4;
    if (rows < fill) rows = fill;
    const dim3 grid(cdiv(q_len, rows), heads);
    const size_t lds = sizeof(float) * (line_reach(*buckets) + line_right(*buckets) + 1);
    const hipStream_t st = (hipStream_t)stream;
    if (type == TCVOM_TYPE_F32)
        hipLaunchKernelGGL(relbias_fwd_kernel<float>, grid, dim3(256), lds, st, table, (float*)out, bk, heads, q_len, k_len, q_start, (int)rows);
    else if (type == TCVOM_TYPE_BF16)
        hipLaunchKernelGGL(relbias_fwd_kernel<__bf16>, grid, dim3(256), lds, st, table, (__bf16*)out, bk, heads, q_len, k_len, q_start, (int)rows);
    else
        hipLaunchKernelGGL(relbias_fwd_kernel<_Float16>, grid, dim3(256), lds, st, table, (_Float16*)out, bk, heads, q_len, k_len, q_start, (int)rows);
    TCVOM_LAUNCH_CHECK("relbias_fwd");
    return 0;
}

// ---- backward: sums of dbias along the clamped diagonals of each chunk of rows, then the line entries of each bucket.
// Two kinds of workgroup in one launch (blockIdx.x): the BAND ones own 256 inner line entries each, a thread an entry: it walks the
// rows of the chunk, its key moving one step a row, so that a wave reads consecutive elements; the FAR one (the last) sums what lies
// past the two ends of the line, which is most of a long matrix, with 16-byte loads.  Each sum is made by one thread, or by a tree of
// fixed shape, and written once: no atomics, equal calls give equal bits.  12 x 2041 x 2041 fp32: 62 us = 3.2 TB/s, half of what a
// plain read of as much reaches (30 us): the waves wait 61 % of their time, a row's far sums one after the other; 8 x 1024 x 1024 bf16: 6.9 us.  Chunks of 8, 32 or 64 rows: no faster.
constexpr int BIAS_ROWS = 16;
// chunks of rows are blocks of the grid's second dimension, and a bucket's entries of all chunks are counted in 32 bits
static_assert(TCVOM_MAX_RELBIAS_BWD_QUERIES <= 65535 * BIAS_ROWS && TCVOM_MAX_RELBIAS_BWD_QUERIES / BIAS_ROWS * (TCVOM_MAX_BUCKET_REACH + 1LL) < (1LL << 31), "");
template <class T, int LANES>
__global__ __launch_bounds__(256) void relbias_bwd_kernel(const T* dout, float* part, tcvom_rel_buckets bk, long long Nq, long long Nk,
                                                          long long q_start) {
    __shared__ float red[2][4];
    constexpr int V = 16 / sizeof(T);
    const int h = blockIdx.z, reach = line_reach(bk), last = reach + line_right(bk);
    const long long i0 = (long long)blockIdx.y * BIAS_ROWS, i1 = min(Nq, i0 + BIAS_ROWS);
    const T* plane = dout + (long long)h * Nq * Nk;
    float* out = part + ((long long)h * gridDim.y + blockIdx.y) * (last + 1);
    if (blockIdx.x + 1 < gridDim.x) {
        const int t = 1 + (int)blockIdx.x * 256 + threadIdx.x;             // inner entry: rel = t - reach
        if (t >= last) return;
        const long long off = t - reach + q_start;                         // its key in row i is i + off
        const long long a = -off > i0 ? -off : i0, b = Nk - off < i1 ? Nk - off : i1;     // rows whose key exists
        const T* p = plane + i0 * Nk + i0 + off;
        float s[BIAS_ROWS];
#pragma unroll
        for (int u = 0; u < BIAS_ROWS; ++u) s[u] = i0 + u >= a && i0 + u < b ? (float)p[u * (Nk + 1)] : 0.f;
#pragma unroll
        for (int o = BIAS_ROWS / 2; o > 0; o >>= 1)
#pragma unroll
            for (int u = 0; u < o; ++u) s[u] += s[u + o];
        out[t] = s[0];
        return;
    }
    // a row to LANES lanes: 16 rows at once while they are short
    const int lane = threadIdx.x % LANES;
    float side[2] = {0.f, 0.f};
    for (long long i = i0 + threadIdx.x / LANES; i < i1; i += 256 / LANES) {
        const T* row = plane + i * Nk;
        // keys with line index <= 0 are j < jl, with index >= last j >= jr (last > 0)
        const long long jl = min(max(i + q_start - reach + 1, 0LL), Nk), jr = min(max(i + q_start - reach + last, 0LL), Nk);
        // of each side: up to V - 1 elements to a 16-byte boundary, vectors, up to V - 1 more; both sides and four vectors each at once
        const T* vec[2];
        int nv[2];
        T edge[2][2];
        bool in[2][2];
        float s[2][V];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const long long ja = w ? jr : 0, jb = w ? Nk : jl;
            const long long head = min((long long)(((16 - ((uintptr_t)(row + ja) & 15)) & 15) / sizeof(T)), jb - ja);
            nv[w] = (int)((jb - ja - head) / V);
            vec[w] = row + ja + head;
            const long long j = ja + head + (long long)nv[w] * V + lane;
            in[w][0] = lane < head;
            in[w][1] = j < jb;
            edge[w][0] = row[in[w][0] ? ja + lane : 0];
            edge[w][1] = row[in[w][1] ? j : 0];
#pragma unroll
            for (int u = 0; u < V; ++u) s[w][u] = 0.f;
        }
        for (int n = lane; n < max(nv[0], nv[1]); n += 4 * LANES) {
            typename RawVec<T, V>::type f[2][4];
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    f[w][k] = (typename RawVec<T, V>::type)(T)0.f;
                    if (n + LANES * k < nv[w]) f[w][k] = load_raw<T, V>(vec[w] + (long long)(n + LANES * k) * V);
                }
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int u = 0; u < V; ++u) s[w][u] += (float)f[w][k][u];
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            s[w][0] += in[w][0] ? (float)edge[w][0] : 0.f;
            s[w][1] += in[w][1] ? (float)edge[w][1] : 0.f;
#pragma unroll
            for (int o = V / 2; o > 0; o >>= 1)
#pragma unroll
                for (int u = 0; u < o; ++u) s[w][u] += s[w][u + o];
            side[w] += s[w][0];
        }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const float t = wave_sum(side[w]);
        if ((threadIdx.x & 63) == 0) red[w][threadIdx.x >> 6] = t;
    }
    __syncthreads();
    if (threadIdx.x < 2) out[threadIdx.x ? last : 0] = (red[threadIdx.x][0] + red[threadIdx.x][1]) + (red[threadIdx.x][2] + red[threadIdx.x][3]);
}

// dtable[b][h]: a workgroup a bucket and head adds the bucket's line entries of every chunk, in 64 bits
__global__ __launch_bounds__(256) void relbias_table_kernel(const float* part, float* dtable, tcvom_rel_buckets bk, int heads, int chunks) {
    __shared__ double red[4];
    const int b = blockIdx.x, h = blockIdx.y, last = line_reach(bk) + line_right(bk);
    int t0, t1;
    bucket_entries(bk, b, t0, t1);
    const int n = t1 - t0;
    const float* p = part + (long long)h * chunks * (last + 1) + t0;
    double s = 0.;
    if (n > 0)
#pragma unroll 4
        for (int e = threadIdx.x; e < n * chunks; e += 256) s += (double)p[(long long)(e / n) * (last + 1) + e % n];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) dtable[b * heads + h] = (float)((red[0] + red[1]) + (red[2] + red[3]));
}

extern "C" int64_t tcvom_relbias_bwd_work(const tcvom_rel_buckets* buckets, int32_t heads, int64_t q_len) {
    if (!buckets || buckets->n_starts < 1 || buckets->n_starts > TCVOM_MAX_BUCKET_STARTS || heads <= 0 || q_len <= 0) return 0;
    return (int64_t)heads * cdiv(q_len, BIAS_ROWS) * (line_reach(*buckets) + line_right(*buckets) + 1);
}

extern "C" int tcvom_relbias_bwd(const void* dout, float* dtable, float* work, int64_t work_floats, const tcvom_rel_buckets* buckets,
                                 int32_t heads, int64_t q_len, int64_t k_len, int64_t q_start, int32_t type, void* stream) {
    TCVOM_CHECK_ARG(dout && dtable && work && heads > 0 && heads <= 65535 && q_len > 0 && k_len > 0,
                    "relbias_bwd: heads=%d q_len=%lld k_len=%lld", heads, (long long)q_len, (long long)k_len);
    TCVOM_CHECK_ARG(type >= TCVOM_TYPE_F32 && type <= TCVOM_TYPE_F16, "relbias_bwd: type %d", type);
    TCVOM_CHECK_ARG(q_len <= TCVOM_MAX_RELBIAS_BWD_QUERIES && k_len < (1LL << 31) && q_start < (1LL << 40) && q_start > -(1LL << 40),
                    "relbias_bwd: lengths");
    if (const int rc = check_buckets("relbias_bwd", buckets)) return rc;
    const tcvom_rel_buckets bk = pad_buckets(*buckets);
    TCVOM_CHECK_ARG(work_floats >= tcvom_relbias_bwd_work(buckets, heads, q_len), "relbias_bwd: %lld floats of workspace", (long long)work_floats);
    const int last = line_reach(*buckets) + line_right(*buckets), chunks = cdiv(q_len, BIAS_ROWS);
    const dim3 grid(cdiv(last - 1, 256) + 1, chunks, heads);
    const hipStream_t st = (hipStream_t)stream;
#define RELBIAS_BWD(T, LANES) \
    hipLaunchKernelGGL((relbias_bwd_kernel<T, LANES>), grid, dim3(256), 0, st, (const T*)dout, work, bk, q_len, k_len, q_start)
    // 8 x 1024 x 1024 bf16: 7.0 us with 16 lanes a row, 11.5 us with a wave; 16 x 4000 x 64: 20 and 58; rows of 6 KB and more: the same
    if (k_len * (type == TCVOM_TYPE_F32 ? 4 : 2) <= 4096) {
        if (type == TCVOM_TYPE_F32) RELBIAS_BWD(float, 16);
        else if (type == TCVOM_TYPE_BF16) RELBIAS_BWD(__bf16, 16);
        else RELBIAS_BWD(_Float16, 16);
    } else {
        if (type == TCVOM_TYPE_F32) RELBIAS_BWD(float, 64);
        else if (type == TCVOM_TYPE_BF16) RELBIAS_BWD(__bf16, 64);
        else RELBIAS_BWD(_Float16, 64);
    }
#undef RELBIAS_BWD
    TCVOM_LAUNCH_CHECK("relbias_bwd");
    hipLaunchKernelGGL(relbias_table_kernel, dim3(buckets->num_buckets, heads), dim3(256), 0, st, work, dtable, bk, heads, chunks);
    TCVOM_LAUNCH_CHECK("relbias_table");
    return 0;
}
