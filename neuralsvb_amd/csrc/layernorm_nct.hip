// layernorm_nct.hip -- LayerNorm over the channels of an NCT tensor with its gradient, fp32 and bf16.
//
//   y = (x - mu) rs gamma + beta,   mu, var over the C channels of a position, rs = 1 / sqrt(var + eps)
//   g = dy gamma,  xh = (x - mu) rs:   dx = rs (g - mean_c(g) - xh mean_c(g xh)),   dgamma = sum dy xh,   dbeta = sum dy
// Positions past the end of a row: the last lanes of a row step back so that their VEC positions end with it (T >= VEC).  They repeat
// positions of their neighbours, bit for bit -- same loads, same order of sums, same stores --, and count `skip` of them out of the
// affine sums.  No access needs a tail.
//
// HBM-bound: forward reads and writes x once, backward reads x and dy and writes dx (32 x 1024 x 2048 bf16: forward 66 us, 4.1 TB/s;
// backward 145 us, 2.8 TB/s, and 5 us for the sums; 32 x 512 x 700 fp32: 23 us, and 31 + 4 us).  A workgroup owns whole columns, so it has to
// hold C values of each: LPR lanes side by side along time take VEC values (16 bytes) each, NT / LPR rows of them cover that many
// channels at once, and P such passes stay in registers -- all loads of a tile are in flight together and nothing is read twice.
// Sums over channels: in-lane over the passes, lanes of a wave by shuffles, waves through LDS; variance from centred values.
// The affine gradients are sums over positions: a thread keeps those of its own P channels in registers over all the tiles that its
// workgroup walks, then one partial row per workgroup goes to memory and a second launch adds the rows in order (the same order in
// every run).  One workgroup writes the result itself.
#include "rel_bucket.h"
#include <svb_opaque.h>

/* workgroups of the backward that walk tiles: one per CU.  With two of them dx waits for a second round of loads on each CU and the affine
   sums have twice the rows: both launches of 32 x 512 x 700 fp32 46 us instead of 38, of 32 x 1024 x 2048 bf16 159 instead of 150 */
#define SVB_LN_MAX_WG 256

typedef float svbl_f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned svbl_u4 __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ unsigned short svbl_bf16(float x) {
    const __bf16 h = (__bf16)x;
    unsigned short u;
    __builtin_memcpy(&u, &h, 2);
    return u;
}

// P rows of VEC values as loaded (bf16 stays packed).  Rows start at any element (odd T), so the 16-byte accesses claim the alignment
// of one.  fresh(): the compiler forgets what it computed from them, so that a tile costs its raw registers and not its floats as well.
template <typename T, int VEC, int P> struct SvbLnTile {
    static constexpr int DW = VEC == 1 ? 1 : 4;
    unsigned r[P * DW];
    __device__ __forceinline__ void fresh() {
#pragma unroll
        for (int i = 0; i < P * DW; ++i) svb_opaque(r[i]);
    }
    __device__ __forceinline__ void zero(int p) {
#pragma unroll
        for (int e = 0; e < DW; ++e) r[p * DW + e] = 0u;
    }
    __device__ __forceinline__ void load(int p, const float* s) {
        if (VEC == 1) { r[p * DW] = __float_as_uint(s[0]); return; }
        const svbl_f4 t = *reinterpret_cast<const svbl_f4*>(s);
#pragma unroll
        for (int e = 0; e < DW; ++e) r[p * DW + e] = __float_as_uint(t[e]);
    }
    __device__ __forceinline__ void load(int p, const unsigned short* s) {
        if (VEC == 1) { r[p * DW] = (unsigned)s[0] << 16; return; }
        const svbl_u4 t = *reinterpret_cast<const svbl_u4*>(s);
#pragma unroll
        for (int e = 0; e < DW; ++e) r[p * DW + e] = t[e];
    }
    __device__ __forceinline__ float get(int p, int e) const {
        if (VEC != 8) return __uint_as_float(r[p * DW + e]);
        const unsigned u = r[p * DW + ((e >> 1) & (DW - 1))];
        return __uint_as_float(e & 1 ? u & 0xffff0000u : u << 16);
    }
};
template <int VEC>
__device__ __forceinline__ void svbl_store(float* p, const float (&o)[VEC]) {
    if (VEC == 4) {
        svbl_f4 t;
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] = o[e];
        *reinterpret_cast<svbl_f4*>(p) = t;
    } else p[0] = o[0];
}
template <int VEC>
__device__ __forceinline__ void svbl_store(unsigned short* p, const float (&o)[VEC]) {
    if (VEC == 8) {
        svbl_u4 t;
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) t[e] = (unsigned)svbl_bf16(o[2 * e]) | ((unsigned)svbl_bf16(o[2 * e + 1]) << 16);
        *reinterpret_cast<svbl_u4*>(p) = t;
    } else p[0] = svbl_bf16(o[0]);
}
__device__ __forceinline__ float svbl_ld(const float* p, int n) { return n > 0 ? p[0] : 0.f; }
__device__ __forceinline__ float svbl_ld(const unsigned short* p, int n) { return n > 0 ? svb_bf16_f32(p[0]) : 0.f; }

// sum of s[] over the workgroup's rows (threads of one lane column): shuffles inside a wave, then one LDS row per wave
template <int VEC, int LPR, int NT>
__device__ __forceinline__ void svbl_rows_sum(float (&s)[VEC], float* red, int col) {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) s[e] += __shfl_xor(s[e], o, 64);
    __syncthreads();                                                    // (the previous reduction's reads are done)
    if ((threadIdx.x & 63) < LPR) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) red[(threadIdx.x >> 6) * (LPR * VEC) + col * VEC + e] = s[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) t += red[w * (LPR * VEC) + col * VEC + e];
        s[e] = t;
    }
}

struct SvbLnArgs {
    const void *x, *gamma, *beta, *dy;
    void *y, *dx, *dgamma, *dbeta;
    float *mean, *rstd, *part;
    int B, C, T, tiles, affine_bf16;      // tiles: along time, per batch entry
    float eps;
};

// One tile per workgroup, C <= P NT / LPR channels in registers.
template <typename T, int VEC, int LPR, int NT, int P>
__global__ __launch_bounds__(NT) void svb_ln_nct_fwd_kernel(SvbLnArgs a) {
    constexpr int ROWS = NT / LPR;
    __shared__ float red[NT / 64 * LPR * VEC];
    __shared__ float2 affine[P * ROWS];
    const int col = threadIdx.x & (LPR - 1), row = threadIdx.x / LPR;
    for (int c = threadIdx.x; c < a.C; c += NT)                         // (read behind the barriers of the reductions)
        affine[c] = make_float2(a.gamma ? svb_ld_table(a.gamma, c, a.affine_bf16) : 1.f, a.beta ? svb_ld_table(a.beta, c, a.affine_bf16) : 0.f);
    const int item = svb_xcd_item(blockIdx.x, gridDim.x);
    const int b = svb_uniform(item / a.tiles), t0 = min((item - b * a.tiles) * (LPR * VEC) + col * VEC, a.T - VEC);
    // uniform bases and 32-bit byte offsets inside one batch entry: the scalar-base form of the loads, one register per address
    const char* x = (const char*)((const T*)a.x + (size_t)b * a.C * a.T);
    char* y = (char*)((T*)a.y + (size_t)b * a.C * a.T);
    const unsigned step = (unsigned)(ROWS * sizeof(T)) * (unsigned)a.T, off = (unsigned)sizeof(T) * ((unsigned)row * (unsigned)a.T + t0);
    SvbLnTile<T, VEC, P> v;
    float s[VEC], mu[VEC], rs[VEC];
    const float inv_c = 1.f / (float)a.C;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        v.zero(p);
        if (p * ROWS + row < a.C) v.load(p, (const T*)(x + (off + p * step)));
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        s[e] = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) s[e] += v.get(p, e);
    }
    svbl_rows_sum<VEC, LPR, NT>(s, red, col);
    v.fresh();
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        mu[e] = s[e] * inv_c;
        s[e] = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const float d = p * ROWS + row < a.C ? v.get(p, e) - mu[e] : 0.f;
            s[e] = fmaf(d, d, s[e]);
        }
    }
    svbl_rows_sum<VEC, LPR, NT>(s, red, col);
    v.fresh();
#pragma unroll
    for (int e = 0; e < VEC; ++e) rs[e] = 1.f / sqrtf(s[e] * inv_c + a.eps);
    if (a.mean && row == 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) { a.mean[(size_t)b * a.T + t0 + e] = mu[e]; a.rstd[(size_t)b * a.T + t0 + e] = rs[e]; }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = p * ROWS + row;
        if (c < a.C) {
            const float2 gb = affine[c];
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = fmaf((v.get(p, e) - mu[e]) * rs[e], gb.x, gb.y);
            svbl_store<VEC>((T*)(y + (off + p * step)), o);
        }
    }
}

__device__ __forceinline__ void svbl_st_affine(void* p, int c, float v, int is_bf16) {
    if (is_bf16) ((unsigned short*)p)[c] = svbl_bf16(v);
    else ((float*)p)[c] = v;
}

// Walks the tiles blockIdx.x, + gridDim.x, ...; part [gridDim.x][2][C].
template <typename T, int VEC, int LPR, int NT, int P>
__global__ __launch_bounds__(NT) void svb_ln_nct_bwd_kernel(SvbLnArgs a) {
    constexpr int ROWS = NT / LPR;
    __shared__ float red[NT / 64 * LPR * VEC];
    const int col = threadIdx.x & (LPR - 1), row = threadIdx.x / LPR;
    __shared__ float gam[P * ROWS];
    const float inv_c = 1.f / (float)a.C;
    float dg[P], db[P];
    for (int c = threadIdx.x; c < P * ROWS; c += NT) gam[c] = a.gamma && c < a.C ? svb_ld_table(a.gamma, c, a.affine_bf16) : 1.f;
#pragma unroll
    for (int p = 0; p < P; ++p) dg[p] = db[p] = 0.f;
    __syncthreads();
    const int all = a.B * a.tiles;
    for (int tile = svb_xcd_item(blockIdx.x, gridDim.x); tile < all; tile += gridDim.x) {
        const int b = svb_uniform(tile / a.tiles), want = (tile - b * a.tiles) * (LPR * VEC) + col * VEC;
        const int t0 = min(want, a.T - VEC), skip = want - t0;          // (skip >= VEC: nothing of its own)
        const size_t base = (size_t)b * a.C * a.T;
        const char *x = (const char*)((const T*)a.x + base), *dy = (const char*)((const T*)a.dy + base);
        char* dx = (char*)((T*)a.dx + base);
        const unsigned step = (unsigned)(ROWS * sizeof(T)) * (unsigned)a.T, off0 = (unsigned)sizeof(T) * (unsigned)t0;
        const unsigned off = off0 + (unsigned)sizeof(T) * (unsigned)row * (unsigned)a.T;
        SvbLnTile<T, VEC, P> vx, vd;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const unsigned at = p * ROWS + row < a.C ? off + p * step : off0;      // (a row that does not exist: any address that does)
            vx.load(p, (const T*)(x + at));
            vd.load(p, (const T*)(dy + at));
        }
        float mu[VEC], rs[VEC], s1[VEC], s2[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            mu[e] = a.mean[(size_t)b * a.T + t0 + e];
            rs[e] = a.rstd[(size_t)b * a.T + t0 + e];
            s1[e] = s2[e] = 0.f;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const bool has = p * ROWS + row < a.C;
            const float gp = gam[p * ROWS + row];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = has ? vd.get(p, e) : 0.f, xh = has ? (vx.get(p, e) - mu[e]) * rs[e] : 0.f, g = d * gp;
                s1[e] += g;
                s2[e] = fmaf(g, xh, s2[e]);
                const float own = e >= skip ? d : 0.f;
                dg[p] = fmaf(own, e >= skip ? xh : 0.f, dg[p]);
                db[p] += own;
            }
            svb_opaque(dg[p]);                                          // (summed here: moved down behind the reductions the sums would keep
            svb_opaque(db[p]);                                          //  every pass's floats alive, 140 registers)
        }
        if (a.dx) {                                                     // (workgroup-uniform)
            svbl_rows_sum<VEC, LPR, NT>(s1, red, col);
            svbl_rows_sum<VEC, LPR, NT>(s2, red, col);
            vx.fresh();
            vd.fresh();
#pragma unroll
            for (int p = 0; p < P; ++p) {
                if (p * ROWS + row < a.C) {
                    const float gp = gam[p * ROWS + row];
                    float o[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float xh = (vx.get(p, e) - mu[e]) * rs[e];
                        o[e] = rs[e] * (vd.get(p, e) * gp - s1[e] * inv_c - xh * (s2[e] * inv_c));
                    }
                    svbl_store<VEC>((T*)(dx + (off + p * step)), o);
                }
            }
        }
    }
    if (!a.dgamma && !a.dbeta) return;
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) { dg[p] += __shfl_xor(dg[p], o, 64); db[p] += __shfl_xor(db[p], o, 64); }
        const int c = p * ROWS + row;
        if (col == 0 && c < a.C) {
            if (gridDim.x == 1) {
                if (a.dgamma) svbl_st_affine(a.dgamma, c, dg[p], a.affine_bf16);
                if (a.dbeta) svbl_st_affine(a.dbeta, c, db[p], a.affine_bf16);
            } else {
                a.part[(size_t)blockIdx.x * 2 * a.C + c] = dg[p];
                a.part[(size_t)blockIdx.x * 2 * a.C + a.C + c] = db[p];
            }
        }
    }
}

// More channels (or longer rows) than the register form takes: 32 positions x G channel groups, values read again for each use (they come
// from L2).  The forward is a chain of C / G loads in each of its three passes: 32 groups where there are channels for them
// (4 x 1500 x 700 fp32 66 us, 207 with 8 groups).
template <typename T, int G>
__global__ __launch_bounds__(32 * G) void svb_ln_nct_fwd_wide_kernel(SvbLnArgs a) {
    __shared__ float red[2][G][32];
    const int tl = threadIdx.x & 31, cg = threadIdx.x >> 5;
    const int b = blockIdx.x / a.tiles, t = (blockIdx.x - b * a.tiles) * 32 + tl;
    const int n = a.T - t;
    const size_t base = (size_t)b * a.C * a.T + (n > 0 ? t : 0);
    const T* x = (const T*)a.x + base;
    float s = 0.f;
    for (int c = cg; c < a.C; c += G) s += svbl_ld(x + (size_t)c * a.T, n);
    red[0][cg][tl] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int q = 0; q < G; ++q) s += red[0][q][tl];
    const float mu = s / (float)a.C;
    s = 0.f;
    for (int c = cg; c < a.C; c += G) { const float d = svbl_ld(x + (size_t)c * a.T, n) - mu; s = fmaf(d, d, s); }
    red[1][cg][tl] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int q = 0; q < G; ++q) s += red[1][q][tl];
    const float rs = 1.f / sqrtf(s / (float)a.C + a.eps);
    if (a.mean && cg == 0 && n > 0) { a.mean[(size_t)b * a.T + t] = mu; a.rstd[(size_t)b * a.T + t] = rs; }
    for (int c = cg; c < a.C; c += G) {
        const float g = a.gamma ? svb_ld_table(a.gamma, c, a.affine_bf16) : 1.f;
        const float bt = a.beta ? svb_ld_table(a.beta, c, a.affine_bf16) : 0.f;
        const float o[1] = {fmaf((svbl_ld(x + (size_t)c * a.T, n) - mu) * rs, g, bt)};
        if (n > 0) svbl_store<1>((T*)a.y + base + (size_t)c * a.T, o);
    }
}

// (a workgroup adds its tiles' affine sums to its own row of `part`, which it sets in its first tile)
template <typename T>
__global__ __launch_bounds__(256) void svb_ln_nct_bwd_wide_kernel(SvbLnArgs a) {
    __shared__ float red[2][8][32];
    const int tl = threadIdx.x & 31, cg = threadIdx.x >> 5;
    const int all = a.B * a.tiles;
    float* pg = a.part + (size_t)blockIdx.x * 2 * a.C;
    for (int tile = blockIdx.x; tile < all; tile += gridDim.x) {
        const int b = tile / a.tiles, t = (tile - b * a.tiles) * 32 + tl;
        const int n = a.T - t;
        const size_t base = (size_t)b * a.C * a.T + (n > 0 ? t : 0);
        const float mu = n > 0 ? a.mean[(size_t)b * a.T + t] : 0.f, rs = n > 0 ? a.rstd[(size_t)b * a.T + t] : 0.f;
        float s1 = 0.f, s2 = 0.f;
        for (int c = cg; c < a.C; c += 8) {
            const float d = svbl_ld((const T*)a.dy + base + (size_t)c * a.T, n);
            const float xh = (svbl_ld((const T*)a.x + base + (size_t)c * a.T, n) - mu) * rs, g = d * (a.gamma ? svb_ld_table(a.gamma, c, a.affine_bf16) : 1.f);
            s1 += g;
            s2 = fmaf(g, xh, s2);
            if (a.dgamma || a.dbeta) {
                float sg = d * xh, sb = d;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { sg += __shfl_xor(sg, o, 64); sb += __shfl_xor(sb, o, 64); }
                if (tl == 0) {
                    const bool first = tile == (int)blockIdx.x;
                    pg[c] = first ? sg : pg[c] + sg;
                    pg[a.C + c] = first ? sb : pg[a.C + c] + sb;
                }
            }
        }
        if (!a.dx) continue;
        __syncthreads();
        red[0][cg][tl] = s1;
        red[1][cg][tl] = s2;
        __syncthreads();
        s1 = s2 = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) { s1 += red[0][q][tl]; s2 += red[1][q][tl]; }
        s1 /= (float)a.C;
        s2 /= (float)a.C;
        for (int c = cg; c < a.C; c += 8) {
            const float xh = (svbl_ld((const T*)a.x + base + (size_t)c * a.T, n) - mu) * rs;
            const float g = svbl_ld((const T*)a.dy + base + (size_t)c * a.T, n) * (a.gamma ? svb_ld_table(a.gamma, c, a.affine_bf16) : 1.f);
            const float o[1] = {rs * (g - s1 - xh * s2)};
            if (n > 0) svbl_store<1>((T*)a.dx + base + (size_t)c * a.T, o);
        }
    }
}

// dgamma | dbeta = sums of the rows of part [rows][2 C]: 32 columns x 32 row groups per workgroup, four rows of each in flight
__global__ __launch_bounds__(1024) void svb_ln_nct_affine_kernel(const float* part, int rows, int C, void* dgamma, void* dbeta, int is_bf16) {
    __shared__ float red[32][33];
    const int cl = threadIdx.x & 31, rg = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < 2 * C)
        for (int r = rg; r < rows; r += 128)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (r + 32 * u < rows) s[u] += part[(size_t)(r + 32 * u) * 2 * C + c];
    red[rg][cl] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    float t = red[cl][rg];                                              // column rg's 32 groups, one per lane
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) t += __shfl_xor(t, o, 64);
    const int c2 = blockIdx.x * 32 + rg;
    if (cl == 0 && c2 < 2 * C) {
        if (c2 < C) { if (dgamma) svbl_st_affine(dgamma, c2, t, is_bf16); }
        else if (dbeta) svbl_st_affine(dbeta, c2 - C, t, is_bf16);
    }
}

// ---- host: the tile of a call -------------------------------------------------------------------------------------------
// 8 lanes of 16 bytes (a 128-byte line) along time, unless T is so short that most of them would have no position: then 4 lanes of
// one element.  Threads by C so that 8 passes hold it (4-lane form: 16 passes of 64 rows).
struct SvbLnPlan { int positions, rows; };                               // rows: channels in registers; 0: the wide form
static SvbLnPlan svbl_plan(int C, int T, int dtype) {
    if (C > 1024 || 1024L * T > 0x3fffffffL) return {32, 0};
    if (T <= 8) return {4, 1024};
    return {(dtype == SVB_DT_BF16 ? 64 : 32) / (C <= 512 ? 1 : 2), C <= 256 ? 256 : C <= 512 ? 512 : 1024};
}

template <typename T, int VEC>
static void svbl_launch(bool fwd, const SvbLnArgs& a, const SvbLnPlan& p, unsigned grid, hipStream_t st) {
#define SVBL_GO(V, L, N, P)                                                                                         \
    do {                                                                                                             \
        if (fwd) hipLaunchKernelGGL((svb_ln_nct_fwd_kernel<T, V, L, N, P>), dim3(grid), dim3(N), 0, st, a);          \
        else hipLaunchKernelGGL((svb_ln_nct_bwd_kernel<T, V, L, N, P>), dim3(grid), dim3(N), 0, st, a);              \
    } while (0)
    if (p.rows == 0) {
        if (fwd && a.C > 256) hipLaunchKernelGGL((svb_ln_nct_fwd_wide_kernel<T, 32>), dim3(grid), dim3(1024), 0, st, a);
        else if (fwd) hipLaunchKernelGGL((svb_ln_nct_fwd_wide_kernel<T, 8>), dim3(grid), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((svb_ln_nct_bwd_wide_kernel<T>), dim3(grid), dim3(256), 0, st, a);
    } else if (p.positions == 4) SVBL_GO(1, 4, 256, 16);
    else if (p.rows == 256) SVBL_GO(VEC, 8, 256, 8);
    else if (p.rows == 512) SVBL_GO(VEC, 8, 512, 8);
    else SVBL_GO(VEC, 4, 512, 8);
#undef SVBL_GO
}

static int svbl_threads(const SvbLnPlan& p, int C) { return p.rows == 0 ? (C > 256 ? 1024 : 256) : p.rows > 256 && p.positions != 4 ? 512 : 256; }
static bool svbl_fits(int B, int C, int T, int dtype, SvbLnPlan* p, int* tiles) {
    *p = svbl_plan(C, T, dtype);
    *tiles = (T + p->positions - 1) / p->positions;
    // (a launch has less than 2^32 threads; the tiles of all entries are counted in 31 bits)
    return *tiles <= 0xffffffffL / svbl_threads(*p, C) && (long)B * *tiles <= 0x7fffffffL - SVB_LN_MAX_WG;
}
static bool svbl_dtypes(int dtype, int affine_dtype) {
    return (dtype == SVB_DT_F32 && affine_dtype == SVB_DT_F32) || (dtype == SVB_DT_BF16 && (affine_dtype == SVB_DT_F32 || affine_dtype == SVB_DT_BF16));
}

extern "C" int svb_ln_nct_fwd(const void* x, const void* gamma, const void* beta, void* y, float* mean, float* rstd, int B, int C, int T,
                              float eps, int dtype, int affine_dtype, void* stream) {
    if (!x || !y || B <= 0 || C <= 0 || T <= 0 || (!mean != !rstd)) return SVB_ERR_ARG;
    SvbLnArgs a = {};
    SvbLnPlan p;
    if (!svbl_dtypes(dtype, affine_dtype) || !svbl_fits(B, C, T, dtype, &p, &a.tiles)) return SVB_ERR_UNSUPPORTED;
    a.gamma = gamma; a.beta = beta;
    a.C = C; a.T = T; a.eps = eps; a.affine_bf16 = affine_dtype == SVB_DT_BF16;
    const size_t entry = (size_t)C * T * (dtype == SVB_DT_BF16 ? 2 : 4);
    const int most = (int)(0xffffffffL / svbl_threads(p, C) / a.tiles);      // batch entries of a launch
    for (int b = 0; b < B; b += a.B) {
        a.B = B - b < most ? B - b : most;
        a.x = (const char*)x + b * entry;
        a.y = (char*)y + b * entry;
        a.mean = mean ? mean + (size_t)b * T : nullptr;
        a.rstd = mean ? rstd + (size_t)b * T : nullptr;
        if (dtype == SVB_DT_BF16) svbl_launch<unsigned short, 8>(true, a, p, (unsigned)(a.B * a.tiles), (hipStream_t)stream);
        else svbl_launch<float, 4>(true, a, p, (unsigned)(a.B * a.tiles), (hipStream_t)stream);
        SVB_CHECK_LAUNCH();
    }
    return SVB_OK;
}

// workgroups of the backward: one per tile up to SVB_LN_MAX_WG, then an even number of tiles for each
static int svbl_bwd_grid(long all) {
    const long per = (all + SVB_LN_MAX_WG - 1) / SVB_LN_MAX_WG;
    return (int)((all + per - 1) / per);
}

extern "C" size_t svb_ln_nct_bwd_workspace_floats(int B, int C, int T, int dtype) {
    if (B <= 0 || C <= 0 || T <= 0) return 0;
    const SvbLnPlan p = svbl_plan(C, T, dtype);
    return (size_t)svbl_bwd_grid((long)B * ((T + p.positions - 1) / p.positions)) * 2 * (size_t)C;
}

extern "C" int svb_ln_nct_bwd(const void* x, const void* gamma, const void* dy, const float* mean, const float* rstd, void* dx, void* dgamma,
                              void* dbeta, float* ws, int B, int C, int T, int dtype, int affine_dtype, void* stream) {
    if (!x || !dy || !mean || !rstd || B <= 0 || C <= 0 || T <= 0 || ((dgamma || dbeta) && !ws)) return SVB_ERR_ARG;
    if (!dx && !dgamma && !dbeta) return SVB_OK;
    SvbLnArgs a = {};
    SvbLnPlan p;
    if (!svbl_dtypes(dtype, affine_dtype) || !svbl_fits(B, C, T, dtype, &p, &a.tiles)) return SVB_ERR_UNSUPPORTED;
    a.x = x; a.gamma = gamma; a.dy = dy; a.mean = (float*)mean; a.rstd = (float*)rstd; a.dx = dx; a.dgamma = dgamma; a.dbeta = dbeta;
    a.part = ws; a.B = B; a.C = C; a.T = T; a.affine_bf16 = affine_dtype == SVB_DT_BF16;
    const int grid = svbl_bwd_grid((long)B * a.tiles);
    if (dtype == SVB_DT_BF16) svbl_launch<unsigned short, 8>(false, a, p, (unsigned)grid, (hipStream_t)stream);
    else svbl_launch<float, 4>(false, a, p, (unsigned)grid, (hipStream_t)stream);
    SVB_CHECK_LAUNCH();
    if ((dgamma || dbeta) && (grid > 1 || p.rows == 0)) {
        hipLaunchKernelGGL(svb_ln_nct_affine_kernel, dim3((unsigned)((2 * C + 31) / 32)), dim3(1024), 0, (hipStream_t)stream, (const float*)ws,
                           grid, C, dgamma, dbeta, (int)a.affine_bf16);
        SVB_CHECK_LAUNCH();
    }
    return SVB_OK;
}
