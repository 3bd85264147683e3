// bucket_attn_bwd.hip -- gradients of the attention with a learned relative-position bias by buckets.
//
//   t_ij = log2(e) (scale q_i . k_j + bias),  P_ij = 2^(t_ij - m_i) / l_i  (recomputed),  dP_ij = dout_i . v_j,  delta_i = dout_i . out_i
//   dS_ij = P_ij (dP_ij - delta_i):   dv_j = sum_i P_ij dout_i,  dk_j = scale sum_i dS_ij q_i,  dq_i = scale sum_j dS_ij k_j,
//   dtable[k][h] = sum of dS_ij over the pairs of bucket k
//
// Two kernels, each of which owns what it sums, so that every sum has one order and nothing is added atomically between workgroups:
// the first owns 32 queries per wave and walks the keys (dq, dtable, delta), the second owns 32 keys per wave and walks the queries of
// all heads that share them (dk, dv).  That is seven products instead of five; the scores are computed in the orientation in which
// their registers are the next product's operand (attn_tiles.h), so dS never moves between lanes.
//
// delta needs what rounding the output to bf16 destroys -- the sums over a bucket cancel, and the table's gradient is fp32 --, so the
// forward keeps the output in fp32 for bf16 tensors.  P and dS are rounded to bf16 as operands for bf16 tensors (relative 2^-8 each at most,
// averaged over the sum), and cut into three parts for fp32 tensors; dtable sums dS in fp32 before any rounding.
// Bound, as the forward, by what a wave does between its products, and in the second kernel by one wave per SIMD above dk 64 (its two sums
// take 128 registers of each lane at dk 128): B2 H16/4 dk128 T2048 causal bf16 154 to 160 us (dq: three products, 330 TFLOP/s) and 169 us (dk,
// dv: four, 407 TFLOP/s); B32 H4 dk64 T562 fp32 164 and 241 us (569 and 516 TFLOP/s of bf16 products).
// P comes from the forward's maximum and sum as the forward had it: of a row with nearly all its weight on one key, dS of that key is what
// the others' small weights leave.  Where 32 bits hold nothing of them (l == 1: P == 1) its dS is 0, dP - delta being rounding noise alone.
//
// dtable: dS of pairs further than the last bucket border is summed in registers.  Nearer pairs are summed along the diagonals of each
// 32 x 32 sub-tile: the tile goes to LDS skewed, row (key - query) mod 32, which puts the diagonals d and d - 32 side by side into one row of
// 32, and comes back one row half per lane.  That is 16 writes and 4 wide reads per lane; adding each value to its offset's sum with an LDS
// atomic instead (87 cycles each, measured) took 37 of the 61 us of this kernel at B24 H4 dk48 T211.  The sums per offset stay in LDS, an
// array per wave, and are added in order at the end, then over the offsets of each bucket.
#include "attn_tiles.h"

int svb_bucket_attn_check(const SvbBucketAttn* a);
int svb_bucket_table_reduce(const float* part, void* dtable, int rows, int nb, int H, int dtype, hipStream_t st);

struct SvbBattnBwd {
    const void* dout;
    void *dq, *dk, *dv;
    float *delta, *part;           // [B][H][Tq]; [H][B * query tiles][n_buckets] or NULL
    float* kv_part;                // [2][splits][B][Hkv dk][Tk] sums of dS q and P dout, or NULL: one split, dk and dv are written
    int splits;
};

__device__ __forceinline__ float svbt_ds(float p, float dp, float delta) {
    return (p == 1.f ? 0.f : p) * (dp - delta);                         // (p == 1: its row's sum is exactly 1; NaN and infinities stay)
}

// Adds a sub-tile's diagonal sums to diag[key - query], one wave.  s: register r is key svbt_row(r, kb) of query l31; skew: [32][36] floats
// (rows of 36: the writes of 32 lanes, 35 words apart, and the 16-byte reads fall on different banks).
#define SVBT_SKEW_P 36
__device__ __forceinline__ void svbt_diag_add(float* skew, float* diag, const f32x16& s, int l31, int kb) {
    const int t = svbt_fresh(4 * kb - l31);
    __builtin_amdgcn_wave_barrier();                                    // (the last sub-tile's reads are done)
#pragma unroll
    for (int r = 0; r < 16; ++r) skew[((svbt_reg(r) + t) & 31) * SVBT_SKEW_P + l31] = s[r];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // row l31, queries 16 kb .. 16 kb + 15: those up to 31 - l31 are of diagonal l31, the others of l31 - 32
    const int last = 31 - l31 - 16 * kb;
    float here = 0.f, there = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const float4 v = *reinterpret_cast<const float4*>(skew + l31 * SVBT_SKEW_P + 16 * kb + 4 * m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            here += 4 * m + e <= last ? v[e] : 0.f;                     // (a choice each: a difference would carry a NaN over)
            there += 4 * m + e <= last ? 0.f : v[e];
        }
    }
    here += __shfl_xor(here, 32, 64);
    there += __shfl_xor(there, 32, 64);
    diag[kb ? l31 - 32 : l31] += kb ? there : here;                     // (64 different offsets)
}

// One sub-tile's scores -> dS in place; rows are keys, this lane's query has maximum m, 1 / sum inv and delta.  NEAR: the bias varies; bias0: at row 0.
template <bool NEAR>
__device__ __forceinline__ void svbt_weights_q(f32x16& s, const f32x16& dp, float c, const float* bias0, float flat, float m, float inv, float delta) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = svbt_ds(__builtin_amdgcn_exp2f(fmaf(s[r], c, NEAR ? bias0[svbt_reg(r)] : flat) - m) * inv, dp[r], delta);
}

// ---- dq, dtable, delta: 4 waves x 32 queries, keys staged ----------------------------------------------------------------------------
template <typename T, int DKP, int KT, bool DOUBLE, bool TINY>
__global__ __launch_bounds__(256, SvbtParts<T>::NS == 1 || DKP <= 64 ? 2 : 1) void svb_bucket_attn_dq_kernel(SvbBucketAttn a, SvbBattnBwd g, int qtiles) {
    // (FRESH, both ways in one build: B2 H16/4 dk128 T2048 causal bf16 171 -> 158 us, B32 H4 dk64 T562 fp32 169 -> 156; elsewhere it costs
    // 1 to 3 %)
    typedef SvbtTile<T, DKP, KT, 256, TINY, DKP == 128 || (SvbtParts<T>::NS == 3 && DKP == 64)> Tile;
    constexpr int NS = Tile::NS, NK = DKP / 16, NDB = DKP / 32, NSUB = KT / 32;
    constexpr int BUF = NS * (2 * Tile::ROWS_BYTES + Tile::COLS_BYTES);
    constexpr bool PACED = NS == 3 || DKP <= 64;                        // (wide bf16 heads: no registers to read ahead into, 194 us instead of 164)
    HIP_DYNAMIC_SHARED(char, smem)
    const int lane = threadIdx.x & 63, wave = svb_uniform(threadIdx.x >> 6), l31 = lane & 31, kb = lane >> 5;
    int bh, qt;
    svbt_item(blockIdx.x, a.B * a.H, qtiles, a.causal, bh, qt);
    if (a.causal) qt = qtiles - 1 - qt;
    const int b = svb_uniform(bh / a.H), h = bh - b * a.H, hk = svb_uniform(h / (a.H / a.Hkv));
    const int i0 = qt * 128, i = i0 + wave * 32 + l31;
    const bool has = i < a.Tq;
    const int start = svbt_start(a, b), R = svb_bucket_reach(a.buckets), nb = a.buckets.n_buckets;

    const T* k = (const T*)a.k + b * a.k_sb + (long long)hk * a.dk * a.k_sc;
    const T* v = (const T*)a.v + b * a.v_sb + (long long)hk * a.dk * a.v_sc;
    const float* keep = a.keep ? a.keep + (size_t)b * a.Tk : nullptr;
    Tile tk(false), tv(true);
    float kept = 1.f;
    auto fetch = [&](int t) {
        tk.load(k, a.k_sc, t * KT, a.Tk, a.dk);
        tv.load(v, a.v_sc, t * KT, a.Tk, a.dk);
        if (keep) kept = keep[min(t * KT + lane, a.Tk - 1)];
    };
    // own operands, and delta on the way
    const T* q = (const T*)a.q + b * a.q_sb + (long long)h * a.dk * a.q_sc;
    const size_t head = ((size_t)b * a.H + h) * a.dk * a.Tq;
    const int ic = has ? i : 0;
    const size_t row = ((size_t)b * a.H + h) * a.Tq + ic;
    // a query that sees no key has no part in anything, whatever q and dout hold there
    const float m = has ? a.stats[row] : SVBT_INF, inv = has ? a.stats[(size_t)a.B * a.H * a.Tq + row] : 0.f;
    svbt_bf16x8 qf[NK][NS], of[NK][NS];
    float delta = 0.f;
    {
        SvbtOwn<T, NK> own_q, own_do;
        SvbtOwn<float, NK> own_o;
        own_do.load((const T*)g.dout + head, a.Tq, ic, kb, a.dk);
        own_o.load((NS == 3 ? (const float*)a.out : a.out_f32) + head, a.Tq, ic, kb, a.dk);
        own_q.load(q, a.q_sc, ic, kb, a.dk);
        if (g.dq || g.part) fetch(0);                                   // (uniform)
        const bool sees = m != SVBT_INF;
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            float v8[8], o8[8];
            own_do.get(s, kb, a.dk, sees, v8);
            own_o.get(s, kb, a.dk, sees, o8);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                delta = fmaf(v8[e], o8[e], delta);
                if (s & 1) v8[e] = -v8[e];                              // (see dp_neg below)
            }
            svbt_frag8<NS>(v8, of[s]);
        }
        own_q.frags(kb, a.dk, sees, qf);
    }
    delta += __shfl_xor(delta, 32, 64);
    if (has && kb == 0) g.delta[row] = delta;
    if (!g.dq && !g.part) return;                                       // (only delta is wanted; uniform)

    const int span = (2 * (R + SVBT_PAD) + 1 + 3) & ~3;
    unsigned* s_bad = (unsigned*)(smem + (DOUBLE ? 2 : 1) * BUF);        // [SVBT_BAD_WORDS]
    float* s_bias = (float*)(s_bad + SVBT_BAD_WORDS);
    float* s_skew = s_bias + span;                                      // [4][32][SVBT_SKEW_P]
    float* s_diag = s_skew + 4 * 32 * SVBT_SKEW_P;                       // [4][span], by offset + R + PAD; then [2][4] far sums
    svbt_fill_bias(s_bias, a, h, R, 256);
    if (threadIdx.x < SVBT_BAD_WORDS) s_bad[threadIdx.x] = 0u;
    if (g.part)
        for (int e = threadIdx.x; e < 4 * span; e += 256) s_diag[e] = 0.f;
    float *my_skew = s_skew + wave * 32 * SVBT_SKEW_P, *my_diag = s_diag + wave * span + R + SVBT_PAD;

    int end = keep ? svbt_keep_end(keep, a.Tk, lane) : a.Tk;
    if (a.causal) end = max(0, min(end, start + min(i0 + 128, a.Tq)));
    const int p0 = start + i0 + wave * 32, p1 = p0 + 31, p = start + i;
    const int tiles = (end + KT - 1) / KT;
    const int part = a.causal ? start + i0 + 1 : 0x7fffffff;            // from here on a key is hidden from some of the queries here
    const float c = a.scale * SVBT_LOG2E;

    f32x16 acc[NDB];
#pragma unroll
    for (int d = 0; d < NDB; ++d) svbt_zero(acc[d]);
    float sum_past = 0.f, sum_ahead = 0.f;

    unsigned long long seen = ~0ull;                                    // of the tile in LDS: the keys that exist and are kept
    constexpr unsigned long long ALL = KT == 64 ? ~0ull : 0xffffffffull;
    auto bits = [&](int t) { return ALL & __ballot(t * KT + lane < end && kept != 0.f); };
    auto put = [&](int t) {
        const unsigned long long m = seen == ALL ? ~0ull : seen;
        tk.settle(t * KT, a.Tk, m);
        tv.settle(t * KT, a.Tk, m);
        char* buf = smem + (DOUBLE ? (t & 1) * BUF : 0);
        tv.template store<true, false>(buf + NS * Tile::ROWS_BYTES, nullptr);
        // (rows as they are: a score that is not finite stays with its pair)
        const bool some = t * KT + KT > part;                           // (uniform)
        if (NS == 1 || some) {
            tk.template store<true, false>(buf, nullptr);
            if (some) tk.clear_bad(t * KT, part, s_bad);
            tk.template store<false, true>(nullptr, buf + 2 * NS * Tile::ROWS_BYTES);
        } else tk.template store<true, true>(buf, buf + 2 * NS * Tile::ROWS_BYTES);   // (cuts each value once)
    };
    if (KT > part) __syncthreads();                                     // (uniform; s_bad is zero, for later tiles behind their barriers)
    if (tiles > 0) {
        seen = bits(0);
        put(0);
    }
    __syncthreads();
    const float past = s_bias[0], ahead = s_bias[2 * (R + SVBT_PAD)];
    for (int t = 0; t < tiles; ++t) {
        const unsigned long long now = seen;
        const int j0 = t * KT;
        if (t + 1 < tiles) fetch(t + 1);
        const char* krows = smem + (DOUBLE ? (t & 1) * BUF : 0);
        const char* vrows = krows + NS * Tile::ROWS_BYTES;
        const char* kcols = vrows + NS * Tile::ROWS_BYTES;
        if (now != 0ull && !(a.causal && j0 > p1)) {
            const bool edge = now != ALL || (a.causal && j0 + KT - 1 > p0) || i0 + wave * 32 + 32 > a.Tq;
            const bool behind = j0 + KT - 1 - p0 <= -R, before = j0 - p1 >= R;
            const float flat = behind ? past : ahead;
#pragma unroll 1
            for (int u = 0; u < NSUB; ++u) {
                // The matrix cores round the accumulator towards -inf.  In dP that is the same small offset for every pair, and a
                // bucket's sum over millions of pairs shows it (1e-5 of the table's gradient): the odd steps go into an accumulator of
                // their own with the other sign, and the offsets cancel in the difference.
                f32x16 s, dp, dp_neg;
                svbt_zero(s);
                svbt_zero(dp);
                svbt_zero(dp_neg);
#pragma unroll
                for (int x = 0; x < NK; ++x) {
                    svbt_bf16x8 f[NS];
                    Tile::row_frag(krows, u, x, l31, kb, f);
                    svbt_mma<NS, false>(s, f, qf[x]);
                    Tile::row_frag(vrows, u, x, l31, kb, f);
                    svbt_mma<NS, false>(x & 1 ? dp_neg : dp, f, of[x]);
                }
                if (PACED) svbt_pace<NS, 2 * NK * NS>();
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] -= dp_neg[r];
                const unsigned su = has ? (unsigned)(now >> (32 * u)) >> (4 * kb) : 0u;
                const int o0 = svbt_fresh(j0 + 32 * u + 4 * kb - p);     // offset of register row 0
                const bool far = behind || before;
                if (far) svbt_weights_q<false>(s, dp, c, nullptr, flat, m, inv, delta);
                else svbt_weights_q<true>(s, dp, c, s_bias + (o0 + R + SVBT_PAD), flat, m, inv, delta);
                if (edge) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = (su >> svbt_reg(r) & 1u) && !(a.causal && o0 + svbt_reg(r) > 0) ? s[r] : 0.f;
                }
                if (far) {
                    float sum = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += s[r];
                    if (behind) sum_past += sum;
                    else sum_ahead += sum;
                } else if (g.part) svbt_diag_add(my_skew, my_diag + (j0 + 32 * u - p0), s, l31, kb);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = s[8 * x + e];
                    svbt_bf16x8 sf[NS];
                    svbt_frag8<NS>(w, sf);
#pragma unroll
                    for (int d = 0; d < NDB; ++d) {
                        svbt_bf16x8 f[NS];
                        Tile::col_frag(kcols, d, u, x, l31, kb, f);
                        svbt_mma<NS, false>(acc[d], f, sf);
                    }
                }
                if (PACED) svbt_pace<NS, 2 * NDB * NS>();
            }
        }
        if (t + 1 < tiles) {
            if (!DOUBLE) __syncthreads();
            seen = bits(t + 1);
            put(t + 1);
        }
        __syncthreads();
    }
    if (g.part) {
        float* far = s_diag + 4 * span;
        sum_past = svb_wave_sum(sum_past);
        sum_ahead = svb_wave_sum(sum_ahead);
        if (lane == 0) { far[wave] = sum_past; far[4 + wave] = sum_ahead; }
        __syncthreads();
        for (int e = threadIdx.x; e < span; e += 256) {
            s_diag[e] = (s_diag[e] + s_diag[span + e]) + (s_diag[2 * span + e] + s_diag[3 * span + e]);
        }
        __syncthreads();
        float* part = g.part + (((size_t)h * a.B + b) * qtiles + qt) * nb;
        for (int e = wave; e < nb; e += 4) {
            int o_a, o_b;
            svb_bucket_range(a.buckets, e, o_a, o_b);
            float t = 0.f;
            for (int o = max(o_a + R + SVBT_PAD, 0) + lane; o < min(o_b + R + SVBT_PAD, 2 * (R + SVBT_PAD) + 1); o += 64) t += s_diag[o];
            t = svb_wave_sum(t);
            if (o_a <= -R - SVBT_PAD && o_b > -R - SVBT_PAD) t += (far[0] + far[1]) + (far[2] + far[3]);
            if (o_a <= R + SVBT_PAD && o_b > R + SVBT_PAD) t += (far[4] + far[5]) + (far[6] + far[7]);
            if (lane == 0) part[e] = t;
        }
    }
    if (!g.dq) return;
    const uint4 bad = *reinterpret_cast<const uint4*>(s_bad);
    if ((bad.x | bad.y | bad.z | bad.w) != 0u) svbt_add_bad<T, NDB>(acc, s_bad, SVBT_BAD_WORDS, k, a.k_sc, a.dk, part, p, kb);
    if (!has) return;
    T* dq = (T*)g.dq + head + i;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int ch = 32 * d + svbt_row(r, kb);
            if (ch < a.dk) svbt_store(dq + (size_t)ch * a.Tq, acc[d][r] * a.scale);
        }
}

// One sub-tile's scores -> P and dP -> dS, in place; rows are queries.  NEAR: the bias varies; bias0: at row 0.  st: the sub-tile's
// rows' maxima from 4 kb on, KT further their 1 / sum, 2 KT further their delta.
template <bool NEAR, int KT>
__device__ __forceinline__ void svbt_weights_kv(f32x16& s, f32x16& dp, float c, const float* bias0, float flat, const float* st) {
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
        const float4 m = *reinterpret_cast<const float4*>(st + 8 * r4), inv = *reinterpret_cast<const float4*>(st + KT + 8 * r4),
                     d = *reinterpret_cast<const float4*>(st + 2 * KT + 8 * r4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 4 * r4 + e;
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, NEAR ? bias0[-svbt_reg(r)] : flat) - m[e]) * inv[e];
            dp[r] = svbt_ds(s[r], dp[r], d[e]);
        }
    }
}

// ---- dk, dv: 4 waves x 32 keys, queries of the heads that share them staged -----------------------------------------------------------
// The (head, query tile) steps of a key tile can be split over workgroups: each then leaves its sums in memory, to be added in order.
template <typename T, int DKP, int KT, bool DOUBLE, bool TINY>
__global__ __launch_bounds__(256, DKP <= (SvbtParts<T>::NS == 1 ? 64 : 32) ? 2 : 1) void svb_bucket_attn_dkv_kernel(SvbBucketAttn a, SvbBattnBwd g, int ktiles) {
    // (FRESH: B16 H4 dk32 T700 bf16 62 -> 48 us, B8 H4 dk128 T562 fp32 206 -> 202; elsewhere it costs 0 to 3 %)
    typedef SvbtTile<T, DKP, KT, 256, TINY, SvbtParts<T>::NS == 1 ? DKP == 32 : DKP == 128> Tile;
    constexpr int NS = Tile::NS, NK = DKP / 16, NDB = DKP / 32, NSUB = KT / 32;
    constexpr int TILE = NS * 2 * (Tile::ROWS_BYTES + Tile::COLS_BYTES), BUF = TILE + 3 * KT * 4;
    HIP_DYNAMIC_SHARED(char, smem)
    const int lane = threadIdx.x & 63, wave = svb_uniform(threadIdx.x >> 6), l31 = lane & 31, kb = lane >> 5;
    int bk, ks;
    svbt_item(blockIdx.x, a.B * a.Hkv, ktiles * g.splits, a.causal, bk, ks);
    const int kt = svb_uniform(ks / g.splits), split = ks - kt * g.splits;
    const int b = svb_uniform(bk / a.Hkv), hk = bk - b * a.Hkv, G = svb_uniform(a.H / a.Hkv);
    const int jt = kt * 128, jw = jt + wave * 32, j = jw + l31;
    const int start = svbt_start(a, b), R = svb_bucket_reach(a.buckets);
    const bool has = j < a.Tk;                                          // kept: some query sees the key (rows of a tile beyond the last query do not count)
    const bool kept = has && (!a.keep || a.keep[(size_t)b * a.Tk + j] != 0.f) && !(a.causal && j >= start + a.Tq);
    float* s_bias = (float*)(smem + (DOUBLE ? 2 : 1) * BUF);

    const T* k = (const T*)a.k + b * a.k_sb + (long long)hk * a.dk * a.k_sc;
    const T* v = (const T*)a.v + b * a.v_sb + (long long)hk * a.dk * a.v_sc;
    SvbtOwn<T, NK> own_k, own_v;
    own_k.load(k, a.k_sc, has ? j : 0, kb, a.dk);
    own_v.load(v, a.v_sc, has ? j : 0, kb, a.dk);
    const bool all_kept = __ballot(!kept) == 0ull, none_kept = __ballot(kept) == 0ull;
    f32x16 dk[NDB], dv[NDB];
#pragma unroll
    for (int d = 0; d < NDB; ++d) { svbt_zero(dk[d]); svbt_zero(dv[d]); }

    // queries that see a key of this workgroup: i >= first
    const int first = a.causal ? max(0, min(jt - start, a.Tq)) / KT : 0;
    const int tiles = max(0, (a.Tq + KT - 1) / KT - first);
    const float c = a.scale * SVBT_LOG2E;
    Tile tq(false), td(true);
    float stat = 0.f, row_max = 0.f;                                    // thread n KT + i: maximum, 1 / sum or delta of row i; the lane's row's maximum
    const int n0 = svb_uniform((int)((long long)G * tiles * split / g.splits)), n1 = svb_uniform((int)((long long)G * tiles * (split + 1) / g.splits));
    auto fetch = [&](int n) {
        const int hh = hk * G + svb_uniform(n / tiles), i0 = (first + n % tiles) * KT;
        const size_t hd = (size_t)b * a.H + hh;
        tq.load((const T*)a.q + b * a.q_sb + (long long)hh * a.dk * a.q_sc, a.q_sc, i0, a.Tq, a.dk);
        td.load((const T*)g.dout + hd * a.dk * a.Tq, a.Tq, i0, a.Tq, a.dk);
        if (threadIdx.x < 3 * KT) {
            const int i = i0 + (threadIdx.x & (KT - 1));
            const float none = threadIdx.x < KT ? SVBT_INF : 0.f;       // (a query that does not exist has P = 0)
            const float* of = threadIdx.x < KT ? a.stats : threadIdx.x < 2 * KT ? a.stats + (size_t)a.B * a.H * a.Tq : g.delta;
            stat = i < a.Tq ? of[hd * a.Tq + i] : none;
        }
        row_max = a.stats[hd * a.Tq + min(i0 + lane, a.Tq - 1)];
    };
    auto put = [&](int n) {
        const int i0 = (first + n % tiles) * KT;
        // a query that sees no key has no part in dk and dv, whatever q and dout hold there
        constexpr unsigned long long OTHERS = KT == 64 ? 0ull : ~0xffffffffull;
        const unsigned long long seen = OTHERS | __ballot(row_max != SVBT_INF);
        tq.settle(i0, a.Tq, seen);
        td.settle(i0, a.Tq, seen);
        char* buf = smem + (DOUBLE ? (n & 1) * BUF : 0);
        tq.template store<true, true>(buf, buf + 2 * NS * Tile::ROWS_BYTES);
        td.template store<true, true>(buf + NS * Tile::ROWS_BYTES, buf + NS * (2 * Tile::ROWS_BYTES + Tile::COLS_BYTES));
        if (threadIdx.x < 3 * KT) ((float*)(buf + TILE))[threadIdx.x] = stat;
    };
    float past = 0.f, ahead = 0.f;
    if (n0 < n1) fetch(n0);
    svbt_bf16x8 kf[NK][NS], vf[NK][NS];
    own_k.frags(kb, a.dk, kept, kf);
    own_v.frags(kb, a.dk, kept, vf);
    if (n0 < n1) put(n0);
    for (int n = n0; n < n1; ++n) {
        if (n == n0 || n % tiles == 0) {                                           // a new head's bias (every thread is behind the last tile's barrier)
            svbt_fill_bias(s_bias, a, hk * G + n / tiles, R, 256);
            __syncthreads();
            past = s_bias[0];
            ahead = s_bias[2 * (R + SVBT_PAD)];
        }
        if (n + 1 < n1) fetch(n + 1);
        const char* qrows = smem + (DOUBLE ? (n & 1) * BUF : 0);
        const char* drows = qrows + NS * Tile::ROWS_BYTES;
        const char* qcols = drows + NS * Tile::ROWS_BYTES;
        const char* dcols = qcols + NS * Tile::COLS_BYTES;
        const float* stats = (const float*)(qrows + TILE);
        const int pt = start + (first + n % tiles) * KT;                // position of the tile's first query
        if (!none_kept && !(a.causal && jw > pt + KT - 1)) {              // (wave-uniform)
            const bool edge = !all_kept || (a.causal && jw + 31 > pt);
            const bool behind = jw + 31 - pt <= -R, before = jw - (pt + KT - 1) >= R;
            const float flat = behind ? past : ahead;
#pragma unroll 1
            for (int u = 0; u < NSUB; ++u) {
                f32x16 s, dp;
                svbt_zero(s);
                svbt_zero(dp);
#pragma unroll
                for (int x = 0; x < NK; ++x) {
                    svbt_bf16x8 f[NS];
                    Tile::row_frag(qrows, u, x, l31, kb, f);
                    svbt_mma<NS, true>(s, f, kf[x]);
                    Tile::row_frag(drows, u, x, l31, kb, f);
                    svbt_mma<NS, true>(dp, f, vf[x]);
                }
                svbt_pace<NS, 2 * NK * NS>();
                const int o0 = svbt_fresh(j - (pt + 32 * u + 4 * kb));   // offset of register row 0
                const float* st = stats + 32 * u + 4 * kb;
                if (behind || before) svbt_weights_kv<false, KT>(s, dp, c, nullptr, flat, st);
                else svbt_weights_kv<true, KT>(s, dp, c, s_bias + (o0 + R + SVBT_PAD), flat, st);
                if (edge) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const bool sees = kept && !(a.causal && o0 - svbt_reg(r) > 0);
                        s[r] = sees ? s[r] : 0.f;
                        dp[r] = sees ? dp[r] : 0.f;
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float w[8], z[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) { w[e] = s[8 * x + e]; z[e] = dp[8 * x + e]; }
                    svbt_bf16x8 pf[NS], sf[NS];
                    svbt_frag8<NS>(w, pf);
                    svbt_frag8<NS>(z, sf);
#pragma unroll
                    for (int d = 0; d < NDB; ++d) {
                        svbt_bf16x8 f[NS];
                        Tile::col_frag(dcols, d, u, x, l31, kb, f);
                        svbt_mma<NS, false>(dv[d], f, pf);
                        Tile::col_frag(qcols, d, u, x, l31, kb, f);
                        svbt_mma<NS, false>(dk[d], f, sf);
                    }
                }
                svbt_pace<NS, 4 * NDB * NS>();
            }
        }
        if (n + 1 < n1) {
            if (!DOUBLE) __syncthreads();
            put(n + 1);
        }
        __syncthreads();
    }
    if (!has) return;
    const size_t head = ((size_t)b * a.Hkv + hk) * a.dk * a.Tk + j, all = (size_t)a.B * a.Hkv * a.dk * a.Tk;
    float* pk = g.kv_part + split * all + head;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int ch = 32 * d + svbt_row(r, kb);
            if (ch >= a.dk) continue;
            const float sk = kept ? dk[d][r] : 0.f, sv = kept ? dv[d][r] : 0.f;        // (0 times a NaN of q or dout is one)
            if (g.splits > 1) {
                pk[(size_t)ch * a.Tk] = sk;
                pk[g.splits * all + (size_t)ch * a.Tk] = sv;
            } else {
                svbt_store((T*)g.dk + head + (size_t)ch * a.Tk, sk * a.scale);
                svbt_store((T*)g.dv + head + (size_t)ch * a.Tk, sv);
            }
        }
}

// dk (blockIdx.y 0, times scale) and dv (1) from their splits
template <typename T>
__global__ __launch_bounds__(256) void svb_bucket_attn_kv_sum_kernel(SvbBattnBwd g, size_t all, float scale) {
    const float* part = g.kv_part + blockIdx.y * g.splits * all;
    T* out = (T*)(blockIdx.y ? g.dv : g.dk);
    const float f = blockIdx.y ? 1.f : scale;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        float t = 0.f;
        for (int s = 0; s < g.splits; ++s) t += part[s * all + i];
        svbt_store(out + i, t * f);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
// Splits of a key tile's steps: workgroups for two per CU (B2 H16/4 dk128 T2048 causal has 128 key tiles: 859 us with one split), of at
// least four steps each.  (With splits the same case took 191 us and 15 us for the sums.)
static int kv_splits(const SvbBucketAttn* a) {
    const long tiles = (long)a->B * a->Hkv * ((a->Tk + 127) / 128), steps = (long)(a->H / a->Hkv) * ((a->Tq + 63) / 64);
    const long want = (512 + tiles - 1) / tiles, most = steps / 4 < 8 ? steps / 4 : 8;
    return (int)(want < most ? want : most > 1 ? most : 1);
}

template <typename K>
static int bwd_lds(K* kern, int lds) {
    return lds > 65536 && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess;
}

template <typename T, int DKP, int KT, bool DOUBLE, bool TINY = false>
static int dq_launch(const SvbBucketAttn* a, const SvbBattnBwd& g, hipStream_t st) {
    typedef SvbtTile<T, DKP, KT, 256, TINY, false> Tile;
    const int span = svbt_span(a->buckets), qtiles = (a->Tq + 127) / 128;
    const int lds = (DOUBLE ? 2 : 1) * Tile::NS * (2 * Tile::ROWS_BYTES + Tile::COLS_BYTES) + (SVBT_BAD_WORDS + (g.part ? 5 * span + 4 * 32 * SVBT_SKEW_P + 8 : span)) * 4;
    auto* kern = svb_bucket_attn_dq_kernel<T, DKP, KT, DOUBLE, TINY>;
    if (bwd_lds(kern, lds)) return SVB_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a->B * a->H * qtiles)), dim3(256), lds, st, *a, g, qtiles);
    SVB_CHECK_LAUNCH();
    return SVB_OK;
}

template <typename T, int DKP, int KT, bool DOUBLE, bool TINY = false>
static int dkv_launch(const SvbBucketAttn* a, const SvbBattnBwd& g, hipStream_t st) {
    typedef SvbtTile<T, DKP, KT, 256, TINY, false> Tile;
    const int span = svbt_span(a->buckets), ktiles = (a->Tk + 127) / 128;
    const int lds = (DOUBLE ? 2 : 1) * (2 * Tile::NS * (Tile::ROWS_BYTES + Tile::COLS_BYTES) + 3 * KT * 4) + span * 4;
    auto* kern = svb_bucket_attn_dkv_kernel<T, DKP, KT, DOUBLE, TINY>;
    if (bwd_lds(kern, lds)) return SVB_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a->B * a->Hkv * ktiles * g.splits)), dim3(256), lds, st, *a, g, ktiles);
    SVB_CHECK_LAUNCH();
    if (g.splits > 1) {
        const size_t all = (size_t)a->B * a->Hkv * a->dk * a->Tk;
        const unsigned grid = (unsigned)((all + 255) / 256 < 2048 ? (all + 255) / 256 : 2048);
        hipLaunchKernelGGL((svb_bucket_attn_kv_sum_kernel<T>), dim3(grid, 2), dim3(256), 0, st, g, all, a->scale);
        SVB_CHECK_LAUNCH();
    }
    return SVB_OK;
}

static size_t delta_floats(const SvbBucketAttn* a) { return ((size_t)a->B * a->H * a->Tq + 3) & ~(size_t)3; }
static size_t table_floats(const SvbBucketAttn* a) {
    return ((size_t)a->H * a->B * ((a->Tq + 127) / 128) * a->buckets.n_buckets + 3) & ~(size_t)3;
}

extern "C" size_t svb_bucket_attn_bwd_workspace_floats(const SvbBucketAttn* a) {
    if (svb_bucket_attn_check(a) != SVB_OK) return 0;
    const int splits = kv_splits(a);
    return delta_floats(a) + table_floats(a) + (splits > 1 ? 2 * (size_t)splits * a->B * a->Hkv * a->dk * a->Tk : 0);
}

extern "C" int svb_bucket_attn_bwd(const SvbBucketAttn* call, const SvbBucketAttnGrad* g, void* stream) {
    int rc = svb_bucket_attn_check(call);
    if (rc != SVB_OK) return rc;
    SvbBucketAttn filled = *call;
    svb_bucket_fill(&filled.buckets);
    const SvbBucketAttn* a = &filled;
    if (!g || !g->dout || !g->ws || !a->stats || (a->dtype == SVB_DT_BF16 && !a->out_f32) || (!g->d_k != !g->d_v)) return SVB_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    SvbBattnBwd w = {g->dout, g->d_q, g->d_k, g->d_v, g->ws, g->d_table ? g->ws + delta_floats(a) : nullptr, nullptr, kv_splits(a)};
    if (w.splits > 1) w.kv_part = g->ws + delta_floats(a) + table_floats(a);
    // (double buffers where two workgroups of them fit a CU)
    if (a->dtype == SVB_DT_BF16) {
        typedef unsigned short T;
        rc = a->Tk < 4 ? dq_launch<T, 128, 32, false, true>(a, w, st) : a->dk <= 32 ? dq_launch<T, 32, 64, true>(a, w, st)
             : a->dk <= 64 ? dq_launch<T, 64, 64, true>(a, w, st) : a->dk <= 96 ? dq_launch<T, 96, 32, false>(a, w, st)
             : dq_launch<T, 128, 32, false>(a, w, st);
        if (rc == SVB_OK && w.dk)
            rc = a->Tq < 4 ? dkv_launch<T, 128, 64, false, true>(a, w, st) : a->dk <= 32 ? dkv_launch<T, 32, 64, true>(a, w, st)
                 : a->dk <= 64 ? dkv_launch<T, 64, 64, true>(a, w, st) : a->dk <= 96 ? dkv_launch<T, 96, 64, false>(a, w, st)
                 : dkv_launch<T, 128, 64, false>(a, w, st);
    } else {
        typedef float T;
        rc = a->Tk < 4 ? dq_launch<T, 128, 32, false, true>(a, w, st) : a->dk <= 32 ? dq_launch<T, 32, 32, true>(a, w, st)
             : a->dk <= 64 ? dq_launch<T, 64, 32, false>(a, w, st) : a->dk <= 96 ? dq_launch<T, 96, 32, false>(a, w, st)
             : dq_launch<T, 128, 32, false>(a, w, st);
        if (rc == SVB_OK && w.dk)
            rc = a->Tq < 4 ? dkv_launch<T, 128, 32, false, true>(a, w, st) : a->dk <= 32 ? dkv_launch<T, 32, 32, true>(a, w, st)
                 : a->dk <= 64 ? dkv_launch<T, 64, 64, false>(a, w, st) : a->dk <= 96 ? dkv_launch<T, 96, 32, false>(a, w, st)
                 : dkv_launch<T, 128, 32, false>(a, w, st);
    }
    if (rc != SVB_OK || !g->d_table) return rc;
    return svb_bucket_table_reduce(w.part, g->d_table, a->B * ((a->Tq + 127) / 128), a->buckets.n_buckets, a->H, a->table_dtype, st);
}
