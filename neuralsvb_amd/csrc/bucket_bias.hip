// bucket_bias.hip -- the learned relative-position bias by buckets as a [H][Tq][Tk] tensor, and its table's gradient.
//
//   bias[h][i][j] = table[bucket(j - i - start)][h],      dtable[k][h] = sum of dbias[h][i][j] over bucket(j - i - start) == k
//
// Both are HBM-bound: the forward writes, the backward reads H Tq Tk elements once (8 x 2048 x 2051 fp32, 134 MB: 24 us, 5.6 TB/s, and
// 45 us, 3.0 TB/s, and 8 us for the sums; 4 x 562 x 562: 7, 9 and 3 us, the time of a launch).  The bias of a pair depends on its diagonal
// alone.  Forward: a workgroup expands its head's table to one value per offset (constant beyond the last bucket border) in LDS and
// writes rows from it.  Backward: a thread owns offsets, not columns -- it walks down the rows along its diagonals, lanes side by
// side, so that the loads are contiguous and the sums stay in its registers without a scatter; then the diagonals of a bucket are
// added in LDS, in a fixed order.
#include "rel_bucket.h"

#define SVB_BB_ROWS 16            /* rows per workgroup, forward */
#define SVB_BB_BROWS 16           /* rows per workgroup, backward */
#define SVB_BB_OFFS 1024          /* offsets per workgroup, backward: 4 per thread */

typedef float svbb_f4 __attribute__((ext_vector_type(4)));
typedef unsigned short svbb_s4 __attribute__((ext_vector_type(4)));
typedef float svbb_f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short svbb_s4u __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ unsigned short svbb_bf16(float x) {
    const __bf16 h = (__bf16)x;
    unsigned short u;
    __builtin_memcpy(&u, &h, 2);
    return u;
}
template <typename T> struct SvbBb;
template <> struct SvbBb<float> {
    typedef svbb_f4 V;
    static __device__ __forceinline__ float ld(const float* p) { return *p; }
    static __device__ __forceinline__ void ld4(const float* p, float (&o)[4]) {
        const svbb_f4u t = *reinterpret_cast<const svbb_f4u*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = t[e];
    }
    static __device__ __forceinline__ float st(float x) { return x; }
};
template <> struct SvbBb<unsigned short> {
    typedef svbb_s4 V;
    static __device__ __forceinline__ float ld(const unsigned short* p) { return svb_bf16_f32(*p); }
    static __device__ __forceinline__ void ld4(const unsigned short* p, float (&o)[4]) {
        const svbb_s4u t = *reinterpret_cast<const svbb_s4u*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = svb_bf16_f32(t[e]);
    }
    static __device__ __forceinline__ unsigned short st(float x) { return svbb_bf16(x); }
};

template <typename T>
__global__ __launch_bounds__(256) void svb_bucket_bias_fwd_kernel(const T* table, T* bias, SvbRelBuckets bk, int H, int Tq, int Tk, int start,
                                                                  int chunks) {
    __shared__ T diag[2 * SVB_REL_MAX_REACH + 1];
    const int R = svb_bucket_reach(bk);
    const int h = blockIdx.x / chunks, i0 = (blockIdx.x - h * chunks) * SVB_BB_ROWS;
    for (int o = threadIdx.x; o <= 2 * R; o += 256) diag[o] = table[(size_t)svb_bucket_of(bk, o - R) * H + h];
    __syncthreads();
    const int i1 = min(i0 + SVB_BB_ROWS, Tq);
    for (int i = i0; i < i1; ++i) {
        T* out = bias + ((size_t)h * Tq + i) * Tk;
        const int q = start + i;                                        // offset of column j: j - q
        // whole 4-element groups of memory (rows start anywhere), then what is left at both ends
        const int head = min((int)((4 - (((size_t)out / sizeof(T)) & 3)) & 3), Tk);
        const int groups = (Tk - head) / 4;
        for (int g = threadIdx.x; g < groups; g += 256) {
            const int j = head + 4 * g;
            typename SvbBb<T>::V v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = diag[max(-R, min(R, j + e - q)) + R];
            *reinterpret_cast<typename SvbBb<T>::V*>(out + j) = v;
        }
        const int rest = Tk - 4 * groups;                               // < 7
        if ((int)threadIdx.x < rest) {
            const int j = (int)threadIdx.x < head ? (int)threadIdx.x : 4 * groups + (int)threadIdx.x;
            out[j] = diag[max(-R, min(R, j - q)) + R];
        }
    }
}

// grid: (row chunks * offset tiles, H).  Offsets are counted without `start` here (column = row + offset); those that a chunk's rows
// meet run from -(last row) on: tile0 .. tile0 + SVB_BB_OFFS - 1.  part [H][row chunks * offset tiles][n_buckets].
template <typename T>
__global__ __launch_bounds__(256) void svb_bucket_bias_bwd_kernel(const T* dbias, float* part, SvbRelBuckets bk, int Tq, int Tk, int start,
                                                                  int otiles) {
    __shared__ float sums[SVB_BB_OFFS];
    const int h = blockIdx.y, chunk = svb_uniform(blockIdx.x / otiles), i0 = chunk * SVB_BB_BROWS, i1 = min(i0 + SVB_BB_BROWS, Tq);
    const int tile0 = -(i0 + SVB_BB_BROWS - 1) + ((int)blockIdx.x - chunk * otiles) * SVB_BB_OFFS;
    const int o = tile0 + (int)threadIdx.x * 4;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const T* base = dbias + (size_t)h * Tq * Tk;
    // rows where all four columns i + o .. i + o + 3 exist, and those where some do
    const int any0 = max(i0, -o - 3), any1 = min(i1, Tk - o), all0 = max(i0, -o), all1 = min(i1, Tk - o - 3);
    if (all0 < all1) {
        const T* p = base + (size_t)all0 * Tk + (all0 + o);
        int i = all0;
        for (; i + 4 <= all1; i += 4) {                                 // four rows' loads in flight
            float t[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) SvbBb<T>::ld4(p + (size_t)u * (Tk + 1), t[u]);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += (t[0][e] + t[1][e]) + (t[2][e] + t[3][e]);
            p += 4 * ((size_t)Tk + 1);
        }
        for (; i < all1; ++i, p += (size_t)Tk + 1) {
            float t[4];
            SvbBb<T>::ld4(p, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += t[e];
        }
    }
    for (int i = any0; i < any1; ++i) {
        if (all0 < all1 && i == all0) i = all1;                         // (past the rows already added)
        if (i >= any1) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = i + o + e;
            if (j >= 0 && j < Tk) s[e] += SvbBb<T>::ld(base + (size_t)i * Tk + j);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[threadIdx.x * 4 + e] = s[e];
    __syncthreads();
    // a bucket's offsets are one run: find its ends in this tile, one wave per bucket in turn
    const int lane = threadIdx.x & 63;
    float* row = part + ((size_t)h * gridDim.x + blockIdx.x) * bk.n_buckets;
    for (int k = threadIdx.x >> 6; k < bk.n_buckets; k += 4) {
        int a, b;
        svb_bucket_range(bk, k, a, b);
        a = max(a + start - tile0, 0);
        b = min(b + start - tile0, SVB_BB_OFFS);
        float t = 0.f;
        for (int e = a + lane; e < b; e += 64) t += sums[e];
        t = svb_wave_sum(t);
        if (lane == 0) row[k] = t;
    }
}

// One workgroup per head: 16 row groups x 64 buckets, four rows of each in flight.
template <typename T>
__global__ __launch_bounds__(1024) void svb_bucket_table_kernel(const float* part, T* dtable, int rows, int nb, int H) {
    __shared__ float red[16][64];
    const int h = blockIdx.x, k = threadIdx.x & 63, g = threadIdx.x >> 6;
    const float* p = part + (size_t)h * rows * nb;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (k < nb)
        for (int r = g; r < rows; r += 64)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (r + 16 * u < rows) s[u] += p[(size_t)(r + 16 * u) * nb + k];
    red[g][k] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (g == 0 && k < nb) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < 16; ++q) t += red[q][k];
        dtable[(size_t)k * H + h] = SvbBb<T>::st(t);
    }
}

// (also the last step of the attention's backward: part [H][rows][nb])
int svb_bucket_table_reduce(const float* part, void* dtable, int rows, int nb, int H, int dtype, hipStream_t st) {
    if (dtype == SVB_DT_BF16) hipLaunchKernelGGL((svb_bucket_table_kernel<unsigned short>), dim3(H), dim3(1024), 0, st, part, (unsigned short*)dtable, rows, nb, H);
    else hipLaunchKernelGGL((svb_bucket_table_kernel<float>), dim3(H), dim3(1024), 0, st, part, (float*)dtable, rows, nb, H);
    SVB_CHECK_LAUNCH();
    return SVB_OK;
}

// offsets j - i and start + i stay far inside 32 bits
static bool svbb_sizes(int H, int Tq, int Tk, int start) {
    return H > 0 && Tq > 0 && Tk > 0 && Tq <= (1 << 27) && Tk <= (1 << 27) && start >= -(1 << 28) && start <= (1 << 28);
}

extern "C" int svb_bucket_bias_fwd(const void* table, void* bias, const SvbRelBuckets* buckets, int H, int Tq, int Tk, int q_start, int dtype,
                                   void* stream) {
    if (!table || !bias || !svb_bucket_valid(buckets) || !svbb_sizes(H, Tq, Tk, q_start)) return SVB_ERR_ARG;
    const int chunks = (Tq + SVB_BB_ROWS - 1) / SVB_BB_ROWS;
    if ((dtype != SVB_DT_F32 && dtype != SVB_DT_BF16) || (long)H * chunks >= (1 << 24)) return SVB_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(H * chunks));
    SvbRelBuckets bk = *buckets;
    svb_bucket_fill(&bk);
    if (dtype == SVB_DT_BF16)
        hipLaunchKernelGGL((svb_bucket_bias_fwd_kernel<unsigned short>), grid, dim3(256), 0, (hipStream_t)stream, (const unsigned short*)table,
                           (unsigned short*)bias, bk, H, Tq, Tk, q_start, chunks);
    else
        hipLaunchKernelGGL((svb_bucket_bias_fwd_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, (const float*)table, (float*)bias,
                           bk, H, Tq, Tk, q_start, chunks);
    SVB_CHECK_LAUNCH();
    return SVB_OK;
}

static void svbb_bwd_grid(int Tq, int Tk, long* x, long* y) {
    *x = ((long)Tk + SVB_BB_BROWS - 1 + SVB_BB_OFFS - 1) / SVB_BB_OFFS;
    *y = ((long)Tq + SVB_BB_BROWS - 1) / SVB_BB_BROWS;
}

extern "C" size_t svb_bucket_bias_bwd_workspace_floats(int H, int Tq, int Tk, int n_buckets) {
    if (H <= 0 || Tq <= 0 || Tk <= 0 || n_buckets <= 0) return 0;
    long x, y;
    svbb_bwd_grid(Tq, Tk, &x, &y);
    return (size_t)H * x * y * n_buckets;
}

extern "C" int svb_bucket_bias_bwd(const void* dbias, void* dtable, const SvbRelBuckets* buckets, float* ws, int H, int Tq, int Tk, int q_start,
                                   int dtype, void* stream) {
    if (!dbias || !dtable || !ws || !svb_bucket_valid(buckets) || !svbb_sizes(H, Tq, Tk, q_start)) return SVB_ERR_ARG;
    long x, y;
    svbb_bwd_grid(Tq, Tk, &x, &y);
    if ((dtype != SVB_DT_F32 && dtype != SVB_DT_BF16) || H > 65535 || H * x * y >= (1 << 24)) return SVB_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(x * y), (unsigned)H);
    if (dtype == SVB_DT_BF16)
        hipLaunchKernelGGL((svb_bucket_bias_bwd_kernel<unsigned short>), grid, dim3(256), 0, (hipStream_t)stream, (const unsigned short*)dbias, ws,
                           *buckets, Tq, Tk, q_start, (int)x);
    else
        hipLaunchKernelGGL((svb_bucket_bias_bwd_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, (const float*)dbias, ws, *buckets, Tq, Tk,
                           q_start, (int)x);
    SVB_CHECK_LAUNCH();
    return svb_bucket_table_reduce(ws, dtable, (int)(x * y), buckets->n_buckets, H, dtype, (hipStream_t)stream);
}
