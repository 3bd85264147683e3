// bucket_attn_fwd.hip -- attention with a learned relative-position bias by buckets, forward.
//
//   t_ij = log2(e) (scale q_i . k_j + table[bucket(j - p_i)][h]),   P_ij = 2^(t_ij - m_i) / l_i,   out_i = sum_j P_ij v_j
// over the keys that query i sees, one pass over the keys with the running maximum m and sum l; nothing of size Tq x Tk exists.
// Scores are computed transposed, S^T = K Q^T, one query per lane column: a query's maximum and sum are 16 registers and one exchange
// with the other half of the wave, and S^T turns into the B operand of  O^T = V^T P^T  without moving (attn_tiles.h).
// P is rounded to bf16 for bf16 tensors (relative 2^-9 per weight, averaged over the keys; l sums what was not rounded) and cut into
// three parts for fp32 tensors.  A training forward of bf16 tensors takes P in three parts too: the backward gets delta_i = dout_i . out_i
// from this output, and the sums of dS over a bucket cancel down to delta's error (B2 H16/4 dk128 T2048: the table's gradient is 5e-4
// off with one part, 1e-6 with two, 2e-7 with three, as with 32-bit arithmetic throughout).
//
// The bias of a pair is that of its diagonal: a head's table is expanded to one value per offset in LDS.  A tile of keys that lies
// further than the last bucket border from all queries of a wave has one bias for all its pairs and reads none.
#include "attn_tiles.h"

// softmax state and output of 32 queries in one wave
template <int NDB> struct SvbtState {
    f32x16 o[NDB];
    float m, l;                    // l: of this lane's half of the keys
};

// One 32-key sub-tile's scores -> t (log2 units) in place.  NEAR: the bias varies.  EDGE: some pair is hidden.
// qo: offset of this lane's query against the first key of the sub-tile, p_i - j0 (keys j0 + row have offset row - qo).
template <bool NEAR, bool EDGE>
__device__ __forceinline__ void svbt_scores(f32x16& s, float c, const float* s_bias, int R, float flat, int qo, bool causal, unsigned seen, int kb) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int row = svbt_row(r, kb);
        float bias = flat;
        if (NEAR) bias = s_bias[max(-R, min(R, row - qo)) + R];
        s[r] = fmaf(s[r], c, bias);
        if (EDGE) s[r] = (seen >> row & 1u) && !(causal && row > qo) ? s[r] : -SVBT_INF;
    }
}

// KT keys: scores in s[NSUB] -> weights in place, state updated.  (m stays -inf while a query has seen nothing; its weights are 0)
template <int NSUB, int NDB>
__device__ __forceinline__ void svbt_softmax(f32x16 (&s)[NSUB], SvbtState<NDB>& st) {
    float mb = s[0][0];
#pragma unroll
    for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) mb = fmaxf(mb, s[u][r]);
    mb = fmaxf(mb, __shfl_xor(mb, 32, 64));
    const float m_new = fmaxf(st.m, mb);
    if (__ballot(m_new > st.m) != 0ull) {                               // (wave-uniform) some query has a new maximum
        const float alpha = m_new == -SVBT_INF ? 1.f : __builtin_amdgcn_exp2f(st.m - m_new);
        st.l *= alpha;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[d][r] *= alpha;
        st.m = m_new;
    }
    const float m_use = m_new == -SVBT_INF ? 0.f : m_new;
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - m_use);
            sum += s[u][r];
        }
    st.l += sum;
}

// ---- query tiles: 4 waves x 32 queries, keys staged through LDS, the next tile's loads in flight during this one's products ------------
// PP: parts of P
template <typename T, int DKP, int KT, bool DOUBLE, int PP>
__global__ __launch_bounds__(256, 1) void svb_bucket_attn_fwd_kernel(SvbBucketAttn a, int qtiles) {
    typedef SvbtTile<T, DKP, KT, 256> Tile;
    constexpr int NS = Tile::NS, NK = DKP / 16, NDB = DKP / 32, NSUB = KT / 32;
    constexpr int BUF = NS * (Tile::ROWS_BYTES + Tile::COLS_BYTES);
    HIP_DYNAMIC_SHARED(char, smem)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, kb = lane >> 5;
    const int item = svbt_item(blockIdx.x, gridDim.x);
    const int bh = item / qtiles, b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hkv);
    const int qt = a.causal ? qtiles - 1 - (item - bh * qtiles) : item - bh * qtiles;      // (causal: the longest rows first)
    const int i0 = qt * 128, i = i0 + wave * 32 + l31;
    const bool has = i < a.Tq;
    const int start = svbt_start(a, b);
    const int R = svb_bucket_reach(a.buckets);
    float* s_bias = (float*)(smem + (DOUBLE ? 2 : 1) * BUF);
    svbt_fill_bias(s_bias, a, h, R, 256);

    const T* q = (const T*)a.q + b * a.q_sb + (long long)h * a.dk * a.q_sc;
    const T* k = (const T*)a.k + b * a.k_sb + (long long)hk * a.dk * a.k_sc;
    const T* v = (const T*)a.v + b * a.v_sb + (long long)hk * a.dk * a.v_sc;
    const float* keep = a.keep ? a.keep + (size_t)b * a.Tk : nullptr;
    svbt_bf16x8 qf[NK][NS];
#pragma unroll
    for (int s = 0; s < NK; ++s) svbt_own_frag<T, NS>(q, a.q_sc, i, s, kb, a.dk, has, qf[s]);

    // keys that anyone here sees end at `end`; this wave's queries are at positions p0 .. p1
    int end = keep ? svbt_keep_end(keep, a.Tk, lane) : a.Tk;
    if (a.causal) end = max(0, min(end, start + min(i0 + 128, a.Tq)));
    const int p0 = start + i0 + wave * 32, p1 = p0 + 31, p = start + i;
    const int tiles = (end + KT - 1) / KT;

    SvbtState<NDB> st;
#pragma unroll
    for (int d = 0; d < NDB; ++d) svbt_zero(st.o[d]);
    st.m = -SVBT_INF;
    st.l = 0.f;
    const float c = a.scale * SVBT_LOG2E;

    Tile tk, tv;
    unsigned long long seen = ~0ull;
    auto fetch = [&](int t) {                                            // loads of tile t
        tk.load(k, a.k_sc, t * KT, end, a.dk);
        tv.load(v, a.v_sc, t * KT, end, a.dk);
    };
    constexpr unsigned long long ALL = KT == 64 ? ~0ull : 0xffffffffull;
    auto bits = [&](int t) {
        return ALL & (keep ? svbt_keep_bits(keep[min(t * KT + lane, a.Tk - 1)], t * KT, end, lane) : __ballot(t * KT + lane < end));
    };
    auto put = [&](int t) {                                              // registers -> LDS
        if (keep) { tk.hide(seen); tv.hide(seen); }
        char* buf = smem + (DOUBLE ? (t & 1) * BUF : 0);
        tk.template store<true, false>(buf, nullptr);
        tv.template store<false, true>(nullptr, buf + NS * Tile::ROWS_BYTES);
    };
    if (tiles > 0) {
        fetch(0);
        seen = bits(0);
        put(0);
    }
    __syncthreads();
    const float past = s_bias[0], ahead = s_bias[2 * R];
    for (int t = 0; t < tiles; ++t) {
        const unsigned long long now = seen;
        const int j0 = t * KT;
        if (t + 1 < tiles) fetch(t + 1);
        const char* rows = smem + (DOUBLE ? (t & 1) * BUF : 0);
        const char* cols = rows + NS * Tile::ROWS_BYTES;
        if (now != 0ull && !(a.causal && j0 > p1)) {                    // (wave-uniform; the matrix instructions need whole waves)
            f32x16 s[NSUB];
#pragma unroll
            for (int u = 0; u < NSUB; ++u) {
                svbt_zero(s[u]);
#pragma unroll
                for (int x = 0; x < NK; ++x) {
                    svbt_bf16x8 f[NS];
                    Tile::row_frag(rows, u, x, l31, kb, f);
                    svbt_mma<NS, false>(s[u], f, qf[x]);
                }
            }
            const bool edge = now != ALL || (a.causal && j0 + KT - 1 > p0);
            const bool behind = j0 + KT - 1 - p0 <= -R, before = j0 - p1 >= R;
            const float flat = behind ? past : ahead;
#pragma unroll
            for (int u = 0; u < NSUB; ++u) {
                const unsigned su = (unsigned)(now >> (32 * u));
                const int qo = p - (j0 + 32 * u);
                if (behind || before) {
                    if (edge) svbt_scores<false, true>(s[u], c, s_bias, R, flat, qo, a.causal, su, kb);
                    else svbt_scores<false, false>(s[u], c, s_bias, R, flat, qo, a.causal, su, kb);
                } else {
                    if (edge) svbt_scores<true, true>(s[u], c, s_bias, R, flat, qo, a.causal, su, kb);
                    else svbt_scores<true, false>(s[u], c, s_bias, R, flat, qo, a.causal, su, kb);
                }
            }
            svbt_softmax<NSUB, NDB>(s, st);
#pragma unroll
            for (int u = 0; u < NSUB; ++u)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = s[u][8 * x + e];
                    svbt_bf16x8 pf[PP];
                    svbt_frag8<PP>(w, pf);
#pragma unroll
                    for (int d = 0; d < NDB; ++d) {
                        svbt_bf16x8 f[NS];
                        Tile::col_frag(cols, d, u, x, l31, kb, f);
                        if constexpr (PP == NS) svbt_mma<NS, false>(st.o[d], f, pf);
                        else {
#pragma unroll
                            for (int n = PP - 1; n >= 0; --n) st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[0], pf[n], st.o[d], 0, 0, 0);
                        }
                    }
                }
        }
        if (t + 1 < tiles) {
            if (!DOUBLE) __syncthreads();                               // (this tile's fragments are read)
            seen = bits(t + 1);
            put(t + 1);
        }
        __syncthreads();
    }

    const float l = st.l + __shfl_xor(st.l, 32, 64);
    const float inv = l > 0.f ? 1.f / l : 0.f;                          // (no key: zeros)
    if (!has) return;
    const size_t head = ((size_t)b * a.H + h) * a.dk;
    T* out = (T*)a.out + head * a.Tq + i;
    float* out_f32 = a.out_f32 ? a.out_f32 + head * a.Tq + i : nullptr;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int ch = 32 * d + svbt_row(r, kb);
            if (ch < a.dk) {
                const float o = st.o[d][r] * inv;
                svbt_store(out + (size_t)ch * a.Tq, o);
                if (out_f32) out_f32[(size_t)ch * a.Tq] = o;
            }
        }
    if (a.lse && kb == 0) a.lse[((size_t)b * a.H + h) * a.Tq + i] = l > 0.f ? st.m + __log2f(l) : SVBT_INF;
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
int svb_bucket_attn_check(const SvbBucketAttn* a) {
    if (!a || !a->q || !a->k || !a->v || !a->table || !a->out) return SVB_ERR_ARG;
    if (a->B <= 0 || a->H <= 0 || a->Hkv <= 0 || a->dk <= 0 || a->Tq <= 0 || a->Tk <= 0 || a->H % a->Hkv) return SVB_ERR_ARG;
    if (!svb_bucket_valid(&a->buckets)) return SVB_ERR_ARG;
    if ((a->dtype != SVB_DT_F32 && a->dtype != SVB_DT_BF16) || (a->table_dtype != SVB_DT_F32 && a->table_dtype != SVB_DT_BF16)) return SVB_ERR_UNSUPPORTED;
    if (a->dk > 128 || a->Tq > (1 << 28) || a->Tk > (1 << 28) || a->q_start < -(1 << 28) || a->q_start > (1 << 28)) return SVB_ERR_UNSUPPORTED;
    if ((long)a->B * a->H * ((a->Tq + 31) / 32) > 0x7fffffffL || (long)a->B * a->Hkv * ((a->Tk + 31) / 32) > 0x7fffffffL) return SVB_ERR_UNSUPPORTED;
    return SVB_OK;
}

template <typename T, int DKP, int KT, bool DOUBLE, int PP>
static int fwd_launch(const SvbBucketAttn* a, hipStream_t st) {
    typedef SvbtTile<T, DKP, KT, 256> Tile;
    const int lds = (DOUBLE ? 2 : 1) * Tile::NS * (Tile::ROWS_BYTES + Tile::COLS_BYTES) + (2 * svb_bucket_reach(a->buckets) + 1) * 4;
    auto* kern = svb_bucket_attn_fwd_kernel<T, DKP, KT, DOUBLE, PP>;
    if (lds > 65536 && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) return SVB_ERR_LAUNCH;
    const int qtiles = (a->Tq + 127) / 128;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a->B * a->H * qtiles)), dim3(256), lds, st, *a, qtiles);
    SVB_CHECK_LAUNCH();
    return SVB_OK;
}

extern "C" size_t svb_bucket_attn_fwd_workspace_floats(const SvbBucketAttn* a) {
    (void)a;
    return 0;
}

extern "C" int svb_bucket_attn_fwd(const SvbBucketAttn* a, float* ws, void* stream) {
    (void)ws;
    const int rc = svb_bucket_attn_check(a);
    if (rc != SVB_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
#define SVB_FWD_GO(T, KT, PP)                                                                                     \
    return a->dk <= 32 ? fwd_launch<T, 32, KT, true, PP>(a, st) : a->dk <= 64 ? fwd_launch<T, 64, KT, true, PP>(a, st) \
         : a->dk <= 96 ? fwd_launch<T, 96, KT, true, PP>(a, st) : fwd_launch<T, 128, KT, true, PP>(a, st)
    if (a->dtype == SVB_DT_F32) SVB_FWD_GO(float, 32, 3);
    if (a->lse) SVB_FWD_GO(unsigned short, 64, 3);
    SVB_FWD_GO(unsigned short, 64, 1);
#undef SVB_FWD_GO
}
