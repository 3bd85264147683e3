// bucket_attn_fwd.hip -- attention with a learned relative-position bias by buckets, forward.
//
//   t_ij = log2(e) (scale q_i . k_j + table[bucket(j - p_i)][h]),   P_ij = 2^(t_ij - m_i) / l_i,   out_i = sum_j P_ij v_j
// over the keys that query i sees, one pass over the keys with the running maximum m and sum l; nothing of size Tq x Tk exists.
// Scores are computed transposed, S^T = K Q^T, one query per lane column: a query's maximum and sum are 16 registers and one exchange
// with the other half of the wave, and S^T turns into the B operand of  O^T = V^T P^T  without moving (attn_tiles.h).
// P is rounded to bf16 for bf16 tensors (relative 2^-8 per weight at most, averaged over the keys; l sums what was not rounded) and cut into
// three parts for fp32 tensors.  A training forward of bf16 tensors takes P in three parts too: the backward gets delta_i = dout_i . out_i
// from this output, and the sums of dS over a bucket cancel down to delta's error (B2 H16/4 dk128 T2048: the table's gradient is 5e-4
// off with one part, 1e-6 with two, 2e-7 with three, as with 32-bit arithmetic throughout).
//
// The bias of a pair is that of its diagonal: a head's table is expanded to one value per offset in LDS.  A tile of keys that lies
// further than the last bucket border from all queries of a wave has one bias for all its pairs and reads none.
//
// Bound by what a wave does between its products (kernel times; B2 H16/4 dk128 T2048 causal bf16: 89 us, 386 TFLOP/s; in training 118 us,
// with P V in three parts 582 TFLOP/s issued; B2 H8 dk64 T2000 causal: 38 us, 213 TFLOP/s, 512 workgroups at once, the longest with a chain of
// 16 tiles of 128 keys; B32 H4 dk64 T562 fp32: 104 us, 597 TFLOP/s of bf16 products): a 32 x 32 sub-tile is 512 ticks of the matrix core at dk 128 and about as many of
// exponentials, sums and roundings, one after the other, and two workgroups share a CU.
#include "attn_tiles.h"
#include <type_traits>

// softmax state and output of 32 queries in one wave
template <int NDB> struct SvbtState {
    f32x16 o[NDB];
    float m, l;                    // l: of this lane's half of the keys
};

// One 32-key sub-tile's scores -> t (log2 units) in place.  NEAR: the bias varies.  EDGE: some pair is hidden.
// o0: offset of register row 0 of this lane, j0 + 4 kb - p_i; bias0: the bias at o0; seen: the sub-tile's key bits from 4 kb on.
template <bool NEAR, bool EDGE>
__device__ __forceinline__ void svbt_scores(f32x16& s, float c, const float* bias0, float flat, int o0, bool causal, unsigned seen) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        s[r] = fmaf(s[r], c, NEAR ? bias0[svbt_reg(r)] : flat);
        if (EDGE) s[r] = (seen >> svbt_reg(r) & 1u) && !(causal && o0 + svbt_reg(r) > 0) ? s[r] : -SVBT_INF;
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

// ---- query tiles: 4 waves, keys staged through LDS, the next tile's loads in flight during this one's products --------------------------
// PP: parts of P.  KG: the waves are 4 / KG groups of 32 queries, each tile's keys are split over KG waves, which join at the end.
template <typename T, int DKP, int KT, bool DOUBLE, int PP, int KG, bool TINY>
__global__ __launch_bounds__(256, SvbtParts<T>::NS == 3 && DKP == 128 ? 1 : 2) void svb_bucket_attn_fwd_kernel(SvbBucketAttn a, int qtiles) {
    // (FRESH, both ways in one build: B2 H16/4 dk128 T2048 causal bf16 104 -> 84 us, training 134 -> 112; to dk 64 it costs 3 %)
    typedef SvbtTile<T, DKP, KT, 256, TINY, DKP == 128> Tile;
    constexpr int NS = Tile::NS, NK = DKP / 16, NDB = DKP / 32, NSUB = KT / 32 / KG, QW = 4 / KG;
    constexpr int BUF = NS * (Tile::ROWS_BYTES + Tile::COLS_BYTES);
    HIP_DYNAMIC_SHARED(char, smem)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, kb = lane >> 5;
    int bh, qt;
    svbt_item(blockIdx.x, a.B * a.H, qtiles, a.causal, bh, qt);
    if (a.causal) qt = qtiles - 1 - qt;                                 // (the longest rows first)
    const int b = svb_uniform(bh / a.H), h = bh - b * a.H, hk = svb_uniform(h / (a.H / a.Hkv));
    const int qw = wave % QW, k0 = wave / QW * (NSUB * 32);             // this wave's queries, and its keys of a tile
    const int i0 = qt * (32 * QW), i = i0 + qw * 32 + l31;
    const bool has = i < a.Tq;
    const T* q = (const T*)a.q + b * a.q_sb + (long long)h * a.dk * a.q_sc;
    const T* k = (const T*)a.k + b * a.k_sb + (long long)hk * a.dk * a.k_sc;
    const T* v = (const T*)a.v + b * a.v_sb + (long long)hk * a.dk * a.v_sc;
    const float* keep = a.keep ? a.keep + (size_t)b * a.Tk : nullptr;
    Tile tk(false), tv(true);
    constexpr int NB64 = (KT + 63) / 64;
    float kept[NB64];
#pragma unroll
    for (int w = 0; w < NB64; ++w) kept[w] = 1.f;
    auto fetch = [&](int t) {                                            // loads of tile t
        tk.load(k, a.k_sc, t * KT, a.Tk, a.dk);
        tv.load(v, a.v_sc, t * KT, a.Tk, a.dk);
        if (keep) {
#pragma unroll
            for (int w = 0; w < NB64; ++w) kept[w] = keep[min(t * KT + 64 * w + lane, a.Tk - 1)];
        }
    };
    fetch(0);
    SvbtOwn<T, NK> own;
    own.load(q, a.q_sc, has ? i : 0, kb, a.dk);
    const int start = svbt_start(a, b);
    const int R = svb_bucket_reach(a.buckets);
    unsigned* s_bad = (unsigned*)(smem + (DOUBLE ? 2 : 1) * BUF);        // [SVBT_BAD_WORDS]
    float* s_bias = (float*)(s_bad + SVBT_BAD_WORDS);
    svbt_fill_bias(s_bias, a, h, R, 256);
    if (threadIdx.x < SVBT_BAD_WORDS) s_bad[threadIdx.x] = 0u;

    // keys that anyone here sees end at `end`; this wave's queries are at positions p0 .. p1
    int end = keep ? svbt_keep_end(keep, a.Tk, lane) : a.Tk;
    if (a.causal) end = max(0, min(end, start + min(i0 + 32 * QW, a.Tq)));
    const int p0 = start + i0 + qw * 32, p1 = p0 + 31, p = start + i;
    const int tiles = (end + KT - 1) / KT;
    const int part = a.causal ? start + i0 + 1 : 0x7fffffff;            // from here on a key is hidden from some of the queries here
    svbt_bf16x8 qf[NK][NS];
    own.frags(kb, a.dk, has, qf);

    SvbtState<NDB> st;
#pragma unroll
    for (int d = 0; d < NDB; ++d) svbt_zero(st.o[d]);
    st.m = -SVBT_INF;
    st.l = 0.f;
    const float c = a.scale * SVBT_LOG2E;

    unsigned long long seen[NB64];                                      // of the tile in LDS: the keys that exist and are kept
    constexpr unsigned long long ALL = KT == 32 ? 0xffffffffull : ~0ull;
    auto put = [&](int t) {                                              // registers -> LDS
#pragma unroll
        for (int w = 0; w < NB64; ++w) seen[w] = ALL & __ballot(t * KT + 64 * w + lane < end && kept[w] != 0.f);
        const unsigned long long m = seen[0] == ALL ? ~0ull : seen[0];
        tk.settle(t * KT, a.Tk, m, seen[NB64 - 1] | ~ALL);
        tv.settle(t * KT, a.Tk, m, seen[NB64 - 1] | ~ALL);
        if (t * KT + KT > part) tv.clear_bad(t * KT, part, s_bad);       // (uniform)
        char* buf = smem + (DOUBLE ? (t & 1) * BUF : 0);
        tk.template store<true, false>(buf, nullptr);
        tv.template store<false, true>(nullptr, buf + NS * Tile::ROWS_BYTES);
    };
    if (KT > part) __syncthreads();                                     // (uniform; s_bad is zero, for later tiles behind their barriers)
    if (tiles > 0) put(0);
    __syncthreads();
    const float past = s_bias[0], ahead = s_bias[2 * (R + SVBT_PAD)];
    for (int t = 0; t < tiles; ++t) {
        constexpr unsigned long long MINE = NSUB == 2 ? ~0ull : 0xffffffffull;
        const unsigned long long now = (NB64 == 2 ? seen[wave / QW] : seen[0] >> k0) & MINE;
        const int j0 = t * KT + k0;
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
                    Tile::row_frag(rows, k0 / 32 + u, x, l31, kb, f);
                    svbt_mma<NS, false>(s[u], f, qf[x]);
                }
            }
            svbt_pace<NS, NSUB * NK * NS>();
            const bool edge = now != MINE || (a.causal && j0 + 32 * NSUB - 1 > p0);
            const bool behind = j0 + 32 * NSUB - 1 - p0 <= -R, before = j0 - p1 >= R;
            const float flat = behind ? past : ahead;
#pragma unroll
            for (int u = 0; u < NSUB; ++u) {
                const unsigned su = (unsigned)(now >> (32 * u)) >> (4 * kb);
                const int o0 = svbt_fresh(j0 + 32 * u + 4 * kb - p);
                if (behind || before) {
                    if (edge) svbt_scores<false, true>(s[u], c, nullptr, flat, o0, a.causal, su);
                    else svbt_scores<false, false>(s[u], c, nullptr, flat, o0, a.causal, su);
                } else {
                    const float* bias0 = s_bias + (o0 + R + SVBT_PAD);
                    if (edge) svbt_scores<true, true>(s[u], c, bias0, flat, o0, a.causal, su);
                    else svbt_scores<true, false>(s[u], c, bias0, flat, o0, a.causal, su);
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
                        Tile::col_frag(cols, d, k0 / 32 + u, x, l31, kb, f);
                        if constexpr (PP == NS) svbt_mma<NS, false>(st.o[d], f, pf);
                        else {
#pragma unroll
                            for (int n = PP - 1; n >= 0; --n) st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[0], pf[n], st.o[d], 0, 0, 0);
                        }
                    }
                }
            if (PP == NS) svbt_pace<NS, NSUB * 2 * NDB * NS>();
        }
        if (t + 1 < tiles) {
            if (!DOUBLE) __syncthreads();                               // (this tile's fragments are read)
            put(t + 1);
        }
        __syncthreads();
    }

    if constexpr (KG == 2) {                                            // (the last tile is read)
        constexpr int N = 16 * NDB + 2;                                 // a lane's state, lanes innermost
        static_assert(QW * N * 256 <= BUF, "the tile's LDS holds the states");
        float* s_st = (float*)smem + qw * N * 64 + lane;
        if (wave >= QW) {
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) s_st[(16 * d + r) * 64] = st.o[d][r];
            s_st[(N - 2) * 64] = st.m;
            s_st[(N - 1) * 64] = st.l;
        }
        __syncthreads();
        if (wave >= QW) return;
        const float m1 = s_st[(N - 2) * 64], m = fmaxf(st.m, m1), m_use = m == -SVBT_INF ? 0.f : m;
        const float f0 = __builtin_amdgcn_exp2f(st.m - m_use), f1 = __builtin_amdgcn_exp2f(m1 - m_use);
        st.m = m;
        st.l = st.l * f0 + s_st[(N - 1) * 64] * f1;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[d][r] = st.o[d][r] * f0 + s_st[(16 * d + r) * 64] * f1;
    }
    const float l = st.l + __shfl_xor(st.l, 32, 64);
    const float inv = l == 0.f ? 0.f : 1.f / l;                         // (no key: zeros; NaN stays)
    const uint4 bad = *reinterpret_cast<const uint4*>(s_bad);
    if ((bad.x | bad.y | bad.z | bad.w) != 0u) svbt_add_bad<T, NDB>(st.o, s_bad, SVBT_BAD_WORDS, v, a.v_sc, a.dk, part, p, kb);
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
    // (apart: added up, the logarithm of a sum near 1 is lost behind a large maximum, and with it the weight of the other keys)
    if (a.stats && kb == 0) {
        float* stats = a.stats + ((size_t)b * a.H + h) * a.Tq + i;
        stats[0] = l > 0.f ? st.m : l == 0.f ? SVBT_INF : l;            // (NaN: the row has keys, and NaN gradients)
        stats[(size_t)a.B * a.H * a.Tq] = inv;
    }
}

// ---- few query rows: the cache's keys split over waves and workgroups ------------------------------------------------------------------
// A new token per request reads each cached key and value once and computes little: HBM-bound, and one workgroup per head would leave
// the chip empty.  The rows of a wave are the (query head, query) pairs that share a key / value head (at most 32, so a shared head is read
// once); every wave takes its own run of keys in tiles of 64, straight from memory to operands:
//   K: a lane loads the key pair 2 l31, 2 l31 + 1 of a channel (consecutive lanes, whole lines); a permutation makes the even and the odd
//      keys' operands, two 32-key score tiles.  Register r of tile p is then key 2 row(r) + p, and the registers 4 g .. 4 g + 3 of both tiles,
//      interleaved, are the eight consecutive keys 16 g + 8 kb + 0..7
//   V: 16 bytes of consecutive keys of a channel per lane, in just that order.
// Waves join in LDS, workgroups in a second launch from [split][row] parts (m, l, sum of P v) in memory, in order.
// 16 requests, H16/4 dk64, caches of 8192 filled to three quarters on average (101 MB): 26 to 29 us, 3.5 TB/s, and 6 us for the join.
struct SvbFewParts {
    float *o, *ml;                 // [item][split][rows][dk], [item][split][rows][2]; NULL: one split, out is written
    int splits;
};

// A tile whose 64 keys do not all count (the last one, one with hidden keys) reads 64 keys all the same: it steps back from the end of
// the rows (Tk >= 64) and counts only what is its own.  Channels that do not exist read one that does: their q is 0, their outputs are
// not written.
// Addresses: a uniform row pointer and a 32-bit lane offset (8 channel pitches of at most 2^25 elements).
template <typename T>
struct SvbFewRows {
    const char* row;                   // of channel d
    long long step, dk, d;
    unsigned off0, off1;               // this lane's byte offset without and with its 8 kb channels
    // (opaque, and walked: the loop over tiles would otherwise keep pointers and conditions per row in more scalar registers than there are)
    __device__ __forceinline__ SvbFewRows(const T* k, long long sc, int j, int kb, int dk_) : row((const char*)k), step(sc * (long long)sizeof(T)), dk(dk_), d(0) {
        svb_opaque_uniform(step);
        svb_opaque_uniform(dk);
        off0 = (unsigned)sizeof(T) * (unsigned)j;
        off1 = off0 + (unsigned)(8 * kb) * (unsigned)step;
    }
    __device__ __forceinline__ const char* next(bool skip8) {             // channel d + 8 kb; then the next (skip8: the next 16's first)
        const char* p = row + (d + 8 < dk ? off1 : off0);
        const int n = skip8 ? 9 : 1;
#pragma unroll
        for (int i = 0; i < n; ++i, ++d) row += d + 1 < dk ? step : 0;
        return p;
    }
};
template <typename T, int NK> struct SvbFewKeys;
template <int NK> struct SvbFewKeys<unsigned short, NK> {
    unsigned r[NK][8];                                                  // (even | odd << 16) of channel 16 s + 8 kb + e
    __device__ __forceinline__ void load(SvbFewRows<unsigned short> rows) {
#pragma unroll
        for (int s = 0; s < NK; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) __builtin_memcpy(&r[s][e], rows.next(e == 7), 4);
    }
    __device__ __forceinline__ void frag(int s, int p, svbt_bf16x8 (&f)[1]) const {
        unsigned u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned a = r[s][2 * e], b = r[s][2 * e + 1];
            u[e] = p ? a >> 16 | (b & 0xffff0000u) : (a & 0xffffu) | b << 16;
        }
        __builtin_memcpy(&f[0], u, 16);
    }
};
template <int NK> struct SvbFewKeys<float, NK> {
    float r[NK][8][2];
    __device__ __forceinline__ void load(SvbFewRows<float> rows) {
#pragma unroll
        for (int s = 0; s < NK; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) __builtin_memcpy(r[s][e], rows.next(e == 7), 8);
    }
    __device__ __forceinline__ void frag(int s, int p, svbt_bf16x8 (&f)[3]) const {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = r[s][e][p];
        svbt_frag8<3>(v, f);
    }
};
// eight consecutive keys of one channel as loaded, and as operand; `seen`: the bits of those that count (the others become zero)
template <typename T> struct SvbFewValues;
template <> struct SvbFewValues<unsigned short> {
    unsigned r[4];
    __device__ __forceinline__ void load(const unsigned short* p) { __builtin_memcpy(r, p, 16); }
    __device__ __forceinline__ unsigned bad() const {                   // the bits of those that are not finite
        unsigned found = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned m = e & 1 ? 0x7f800000u : 0x7f80u;
            found |= (r[e >> 1] & m) == m ? 1u << e : 0u;
        }
        return found;
    }
    template <bool FULL>
    __device__ __forceinline__ void frag(unsigned seen, svbt_bf16x8 (&f)[1]) const {
        unsigned u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            u[e] = FULL ? r[e] : r[e] & ((seen >> (2 * e) & 1 ? 0xffffu : 0u) | (seen >> (2 * e + 1) & 1 ? 0xffff0000u : 0u));
        __builtin_memcpy(&f[0], u, 16);
    }
};
template <> struct SvbFewValues<float> {
    float r[8];
    __device__ __forceinline__ void load(const float* p) { __builtin_memcpy(r, p, 32); }
    __device__ __forceinline__ unsigned bad() const {
        unsigned found = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) found |= svbt_bad(r[e]) ? 1u << e : 0u;
        return found;
    }
    template <bool FULL>
    __device__ __forceinline__ void frag(unsigned seen, svbt_bf16x8 (&f)[3]) const {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = FULL || (seen >> e & 1) ? r[e] : 0.f;
        svbt_frag8<3>(v, f);
    }
};

template <typename T, int DKP>
__global__ __launch_bounds__(256, DKP * SvbtParts<T>::NS > 192 || DKP == 128 ? 1 : 2) void svb_bucket_attn_few_kernel(SvbBucketAttn a, SvbFewParts parts) {
    constexpr int NS = SvbtParts<T>::NS, NK = DKP / 16, NDB = DKP / 32;
    HIP_DYNAMIC_SHARED(char, smem)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, kb = lane >> 5;
    const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
    const int G = svb_uniform(a.H / a.Hkv), rows = G * a.Tq, nb = a.buckets.n_buckets, R = svb_bucket_reach(a.buckets);
    const bool has = l31 < rows;
    const int hl = has ? l31 / a.Tq : 0, i = has ? l31 - hl * a.Tq : 0, h = hk * G + hl;
    const T* q = (const T*)a.q + b * a.q_sb + (long long)h * a.dk * a.q_sc;
    const T* k = (const T*)a.k + b * a.k_sb + (long long)hk * a.dk * a.k_sc;
    const T* v = (const T*)a.v + b * a.v_sb + (long long)hk * a.dk * a.v_sc;
    const float* keep = a.keep ? a.keep + (size_t)b * a.Tk : nullptr;
    const int start = svbt_start(a, b), p = start + i;
    const int end = a.causal ? max(0, min(a.Tk, start + a.Tq)) : a.Tk;
    // this wave's run of keys: whole tiles of 64, even over all waves of all splits
    const int tiles = (end + 63) / 64, runs = parts.splits * 4, run = split * 4 + wave;
    const int per = (tiles + runs - 1) / runs, t0 = min(run * per, tiles), t1 = min(t0 + per, tiles);
    // A tile's K registers are free once its scores are made, its V registers at its end: the next tile's loads go there and then.
    SvbFewKeys<T, NK> kt;
    SvbFewValues<T> vt[4][NDB];
    float kept = 1.f;
    long long vrow[NDB];                                                // this lane's channel (one that exists) of V, from key 8 kb on
#pragma unroll
    for (int d = 0; d < NDB; ++d) vrow[d] = min(32 * d + l31, a.dk - 1) * a.v_sc + 8 * kb;
    auto load_k = [&](int t) {                                          // (any t: the tile that ends with the rows is the last one)
        const int j0 = min(64 * t, a.Tk - 64);
        kt.load(SvbFewRows<T>(k, a.k_sc, j0 + 2 * l31, kb, a.dk));
        if (keep) kept = keep[j0 + lane];
    };
    auto load_v = [&](int t) {
        const int j0 = min(64 * t, a.Tk - 64);
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int d = 0; d < NDB; ++d) vt[g][d].load(v + vrow[d] + (j0 + 16 * g));
    };
    SvbtOwn<T, NK> own;
    own.load(q, a.q_sc, i, kb, a.dk);
    if (NS == 1) { load_k(t0); load_v(t0); }                             // (fp32: two tiles' values spill, a tile loads its own)

    float* s_tab = (float*)smem;                                        // [G][nb]
    unsigned char* s_idx = (unsigned char*)(s_tab + G * nb);             // [2 R + 1]
    for (int e = threadIdx.x; e < G * nb; e += 256)
        s_tab[e] = svb_ld_table(a.table, (size_t)(e % nb) * a.H + hk * G + e / nb, a.table_dtype == SVB_DT_BF16) * SVBT_LOG2E;
    for (int o = threadIdx.x; o <= 2 * R; o += 256) s_idx[o] = (unsigned char)svb_bucket_of(a.buckets, o - R);
    svbt_bf16x8 qf[NK][NS];
    own.frags(kb, a.dk, has, qf);
    const float c = a.scale * SVBT_LOG2E;
    SvbtState<NDB> st;
#pragma unroll
    for (int d = 0; d < NDB; ++d) svbt_zero(st.o[d]);
    st.m = -SVBT_INF;
    st.l = 0.f;
    __syncthreads();
    const float* tab = s_tab + hl * nb;
    const float past = tab[s_idx[0]], ahead = tab[s_idx[2 * R]];

    unsigned bad = 0u;                                                  // of keys start + 1 ..: those that svbt_add_bad adds below

    auto tile = [&](int t, auto full_c) {
        constexpr bool FULL = decltype(full_c)::value;                   // 64 keys, all of them seen by every row
        const int j0 = FULL ? 64 * t : min(64 * t, a.Tk - 64);
        if (NS != 1) { load_k(t); load_v(t); }
        unsigned long long seen = ~0ull;
        if (!FULL) seen = __ballot(j0 + lane >= 64 * t && j0 + lane < end && kept != 0.f);
        f32x16 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            svbt_zero(s[u]);
#pragma unroll
            for (int x = 0; x < NK; ++x) {
                svbt_bf16x8 f[NS];
                kt.frag(x, u, f);
                svbt_mma<NS, false>(s[u], f, qf[x]);
            }
        }
        if (NS == 1 && t + 1 < t1) load_k(t + 1);
        const bool flat = j0 + 63 - start <= -R || j0 - (start + a.Tq - 1) >= R;
        const float fb = j0 + 63 - start <= -R ? past : ahead;
        // key of register r of tile u: 2 svbt_reg(r) + u + 8 kb
        const int o0 = svbt_fresh(j0 + 8 * kb - p);
        const unsigned w0 = (unsigned)seen >> (8 * kb), w1 = (unsigned)(seen >> 32) >> (8 * kb);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = 2 * svbt_reg(r) + u, o = o0 + key;
                float bias = fb;
                if (!flat) bias = tab[s_idx[max(-R, min(R, o)) + R]];
                s[u][r] = fmaf(s[u][r], c, bias);
                if (!FULL) s[u][r] = ((r < 8 ? w0 : w1) >> (key & 31) & 1u) && !(a.causal && o > 0) ? s[u][r] : -SVBT_INF;
            }
        svbt_softmax<2, NDB>(s, st);
        // keys that only some of the rows see: as SvbtTile::clear_bad
        unsigned long long some = 0ull;
        if (!FULL && a.causal && a.Tq > 1 && j0 + 63 > start) some = start + 1 <= j0 ? seen : seen & ~0ull << (start + 1 - j0);      // (uniform)
        unsigned found[2] = {0u, 0u};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = s[e & 1][4 * g + (e >> 1)];
            svbt_bf16x8 pf[NS];
            svbt_frag8<NS>(w, pf);
#pragma unroll
            for (int d = 0; d < NDB; ++d) {
                unsigned sees = (unsigned)(seen >> (16 * g + 8 * kb)) & 0xffu;
                if (!FULL && some != 0ull) {
                    const unsigned n = vt[g][d].bad() & (unsigned)(some >> (16 * g + 8 * kb));
                    found[g >> 1] |= (n & 0xffu) << (16 * (g & 1) + 8 * kb);
                    sees &= ~n;
                }
                svbt_bf16x8 f[NS];
                vt[g][d].template frag<FULL>(sees, f);
                svbt_mma<NS, false>(st.o[d], f, pf);
            }
        }
        if (!FULL && some != 0ull) {
            const unsigned long long m = (unsigned long long)found[1] << 32 | found[0];
            bad |= (unsigned)(start + 1 <= j0 ? m << (j0 - start - 1) : m >> (start + 1 - j0));       // (keys up to start + 31)
        }
        if (NS == 1 && t + 1 < t1) load_v(t + 1);
    };
    // Whole tiles first, the others behind them: two loops, since one with both bodies keeps both bodies' registers alive.  bf16: without the
    // masks 28 us instead of 33 (16 requests, 8192 cached keys); fp32 is bound by its six products, and one body is the shorter code.
    const int whole = NS != 1 || keep ? t0 : max(t0, min(t1, (a.causal ? min(end, start + 1) : end) / 64));
    if constexpr (NS == 1)
        for (int t = t0; t < whole; ++t) tile(t, std::true_type{});
    for (int t = whole; t < t1; ++t) tile(t, std::false_type{});
    st.l += __shfl_xor(st.l, 32, 64);
    if (a.causal && a.Tq > 1) {                                         // (uniform)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) bad |= __shfl_xor(bad, o, 64);
        svbt_add_bad<T, NDB>(st.o, &bad, 1, v, a.v_sc, a.dk, start + 1, p, kb);
    }

    // join of the four waves
    __syncthreads();                                                    // (the tables are read)
    float* s_ml = (float*)smem;                                         // [4][32][2]
    float* s_o = s_ml + 256;                                            // [4][DKP][32]
    if (kb == 0) { s_ml[(wave * 32 + l31) * 2] = st.m; s_ml[(wave * 32 + l31) * 2 + 1] = st.l; }
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) s_o[(wave * DKP + 32 * d + svbt_row(r, kb)) * 32 + l31] = st.o[d][r];
    __syncthreads();
    const size_t item = ((size_t)b * a.Hkv + hk) * parts.splits + split;
    for (int e = threadIdx.x; e < rows * a.dk; e += 256) {
        const int ch = e / rows, r = e - ch * rows;                     // (rows innermost: LDS in order)
        float m = -SVBT_INF, l = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, s_ml[(w * 32 + r) * 2]);
        const float m_use = m == -SVBT_INF ? 0.f : m;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_ml[(w * 32 + r) * 2] - m_use);
            l = fmaf(s_ml[(w * 32 + r) * 2 + 1], f, l);
            o = fmaf(s_o[(w * DKP + ch) * 32 + r], f, o);
        }
        const int g = r / a.Tq, i2 = r - g * a.Tq;
        if (!parts.o) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            svbt_store((T*)a.out + (((size_t)b * a.H + hk * G + g) * a.dk + ch) * a.Tq + i2, o * inv);
        } else {
            parts.o[(item * rows + r) * a.dk + ch] = o;
            if (ch == 0) { parts.ml[(item * rows + r) * 2] = m; parts.ml[(item * rows + r) * 2 + 1] = l; }
        }
    }
}

// out of one (batch entry, key / value head, row) from its splits: one wave, lanes along the channels
template <typename T>
__global__ __launch_bounds__(256) void svb_bucket_attn_join_kernel(SvbBucketAttn a, SvbFewParts parts, int total) {
    const int id = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (id >= total) return;
    const int G = a.H / a.Hkv, rows = G * a.Tq, r = id % rows, bh = id / rows, b = bh / a.Hkv, hk = bh - b * a.Hkv;
    const float* ml = parts.ml + ((size_t)bh * parts.splits * rows + r) * 2;
    float m = -SVBT_INF;
    for (int s = lane; s < parts.splits; s += 64) m = fmaxf(m, ml[(size_t)s * rows * 2]);
    m = svb_wave_max(m);
    const float m_use = m == -SVBT_INF ? 0.f : m;
    float l = 0.f, o[2] = {0.f, 0.f};
    const float* po = parts.o + ((size_t)bh * parts.splits * rows + r) * a.dk;
    for (int s = 0; s < parts.splits; ++s) {
        const float f = __builtin_amdgcn_exp2f(ml[(size_t)s * rows * 2] - m_use);
        l = fmaf(ml[(size_t)s * rows * 2 + 1], f, l);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (lane + 64 * u < a.dk) o[u] = fmaf(po[(size_t)s * rows * a.dk + lane + 64 * u], f, o[u]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int g = r / a.Tq, i = r - g * a.Tq;
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < a.dk) svbt_store((T*)a.out + (((size_t)b * a.H + hk * G + g) * a.dk + lane + 64 * u) * a.Tq + i, o[u] * inv);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
int svb_bucket_attn_check(const SvbBucketAttn* a) {
    if (!a || !a->q || !a->k || !a->v || !a->table || !a->out) return SVB_ERR_ARG;
    if (a->B <= 0 || a->H <= 0 || a->Hkv <= 0 || a->dk <= 0 || a->Tq <= 0 || a->Tk <= 0 || a->H % a->Hkv) return SVB_ERR_ARG;
    if (!svb_bucket_valid(&a->buckets)) return SVB_ERR_ARG;
    if ((a->dtype != SVB_DT_F32 && a->dtype != SVB_DT_BF16) || (a->table_dtype != SVB_DT_F32 && a->table_dtype != SVB_DT_BF16)) return SVB_ERR_UNSUPPORTED;
    // (channel pitches: a lane's offset over 16 channels stays in 32 bits)
    if (a->q_sc < 0 || a->q_sc > (1 << 25) || a->k_sc < 0 || a->k_sc > (1 << 25) || a->v_sc < 0 || a->v_sc > (1 << 25)) return SVB_ERR_UNSUPPORTED;
    if (a->dk > 128 || a->Tq > (1 << 25) || a->Tk > (1 << 25) || a->q_start < -(1 << 28) || a->q_start > (1 << 28)) return SVB_ERR_UNSUPPORTED;
    // (a launch has less than 2^32 threads; dk and dv take up to 8 workgroups per 128 keys)
    if (a->B > (1 << 24) || a->H > (1 << 24) || (long)a->B * a->H * ((a->Tq + 63) / 64) >= (1 << 24) || (long)a->B * a->Hkv * ((a->Tk + 127) / 128) >= (1 << 24))
        return SVB_ERR_UNSUPPORTED;
    return SVB_OK;
}

template <typename T, int DKP, int KT, bool DOUBLE, int PP, int KG, bool TINY = false>
static int fwd_launch(const SvbBucketAttn* a, hipStream_t st) {
    typedef SvbtTile<T, DKP, KT, 256, TINY, DKP == 128> Tile;
    const int lds = (DOUBLE ? 2 : 1) * Tile::NS * (Tile::ROWS_BYTES + Tile::COLS_BYTES) + (SVBT_BAD_WORDS + svbt_span(a->buckets)) * 4;
    auto* kern = svb_bucket_attn_fwd_kernel<T, DKP, KT, DOUBLE, PP, KG, TINY>;
    if (lds > 65536 && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) return SVB_ERR_LAUNCH;
    constexpr int ROWS = 128 / KG;
    const int qtiles = (a->Tq + ROWS - 1) / ROWS;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a->B * a->H * qtiles)), dim3(256), lds, st, *a, qtiles);
    SVB_CHECK_LAUNCH();
    return SVB_OK;
}

// Few rows: what a wave holds in its 32 columns, a tile of keys at least, and nothing kept for a backward.  Splits: enough workgroups for two per CU, at least
// 256 keys (a tile for each wave) in each; 0: not this form.
static int few_splits(const SvbBucketAttn* a) {
    if (a->stats || (long)(a->H / a->Hkv) * a->Tq > 32 || a->Tk < 64 || a->B > 65535 || a->Hkv > 65535) return 0;
    const int most = (a->Tk + 255) / 256, want = 512 / max(1, min(512, a->B * a->Hkv));
    return max(1, min(most, want));
}

extern "C" size_t svb_bucket_attn_fwd_workspace_floats(const SvbBucketAttn* a) {
    if (svb_bucket_attn_check(a) != SVB_OK) return 0;                    // (sizes whose products below fit their types)
    const int n = few_splits(a);
    return n > 1 ? (size_t)a->B * a->H * a->Tq * n * (a->dk + 2) : 0;
}

template <typename T, int DKP>
static int few_launch(const SvbBucketAttn* a, float* ws, int splits, hipStream_t st) {
    const int G = a->H / a->Hkv, rows = G * a->Tq;
    SvbFewParts parts = {nullptr, nullptr, splits};
    if (splits > 1) {
        parts.o = ws;
        parts.ml = ws + (size_t)a->B * a->H * a->Tq * splits * a->dk;
    }
    const int tables = G * a->buckets.n_buckets * 4 + 2 * svb_bucket_reach(a->buckets) + 1, join = (256 + 4 * DKP * 32) * 4;
    const int lds = tables > join ? tables : join;
    auto* kern = svb_bucket_attn_few_kernel<T, DKP>;
    if (lds > 65536 && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) return SVB_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)splits, (unsigned)a->Hkv, (unsigned)a->B), dim3(256), lds, st, *a, parts);
    SVB_CHECK_LAUNCH();
    if (splits > 1) {
        const int total = a->B * a->Hkv * rows;
        hipLaunchKernelGGL((svb_bucket_attn_join_kernel<T>), dim3((unsigned)((total + 3) / 4)), dim3(256), 0, st, *a, parts, total);
        SVB_CHECK_LAUNCH();
    }
    return SVB_OK;
}

extern "C" int svb_bucket_attn_fwd(const SvbBucketAttn* call, float* ws, void* stream) {
    const int rc = svb_bucket_attn_check(call);
    if (rc != SVB_OK) return rc;
    SvbBucketAttn filled = *call;
    svb_bucket_fill(&filled.buckets);
    const SvbBucketAttn* a = &filled;
    hipStream_t st = (hipStream_t)stream;
    const int splits = few_splits(a);
    if (splits > 1 && !ws) return SVB_ERR_ARG;
#define SVB_FEW_GO(T)                                                                                              \
    return a->dk <= 32 ? few_launch<T, 32>(a, ws, splits, st) : a->dk <= 64 ? few_launch<T, 64>(a, ws, splits, st) \
         : a->dk <= 96 ? few_launch<T, 96>(a, ws, splits, st) : few_launch<T, 128>(a, ws, splits, st)
    if (splits && a->dtype == SVB_DT_F32) SVB_FEW_GO(float);
    if (splits) SVB_FEW_GO(unsigned short);
#undef SVB_FEW_GO
    // (double buffers where two workgroups of them fit a CU)
#define SVB_FWD_GO(T, K64, KT, PP, D96, KG)                                                                                \
    return a->Tk < 4 ? fwd_launch<T, 128, KT, true, PP, 1, true>(a, st)                                                        \
         : a->dk <= 32 ? fwd_launch<T, 32, K64, true, PP, KG>(a, st) : a->dk <= 64 ? fwd_launch<T, 64, K64, true, PP, KG>(a, st) \
         : a->dk <= 96 ? fwd_launch<T, 96, KT, D96, PP, KG>(a, st) : fwd_launch<T, 128, KT, true, PP, KG>(a, st)
    if (a->dtype == SVB_DT_F32) SVB_FWD_GO(float, 32, 32, 3, false, 1);
    // At most one workgroup of 128 queries per CU and several tiles of keys: workgroups of 64 queries, twice as many, the keys of a tile over
    // two waves, tiles of 128 keys up to dk 64.  Both ways in one build: B2 H8 dk64 T2000 causal (256 workgroups become 512) 52 -> 41 us,
    // training 72 -> 48 (38 and 47 with the steps since); B4 H8 dk96 T1000 causal: 38 -> 34; B24 H4 dk48 T211, where a join and a bigger tile save nothing: 14.5 -> 16.5.  Between one and two workgroups per CU
    // (B7 H8 dk64 T1100 causal) the forward takes 39 us this way instead of 36.  fp32 tensors have six products per tile to wait behind.
    const bool thin = a->Tk > 256 && (long)a->B * a->H * ((a->Tq + 127) / 128) <= 256;
    if (a->stats && thin) SVB_FWD_GO(unsigned short, 128, 64, 3, true, 2);
    if (a->stats) SVB_FWD_GO(unsigned short, 64, 64, 3, true, 1);
    if (thin) SVB_FWD_GO(unsigned short, 128, 64, 1, true, 2);
    SVB_FWD_GO(unsigned short, 64, 64, 1, true, 1);
#undef SVB_FWD_GO
}
