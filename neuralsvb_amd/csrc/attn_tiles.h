// attn_tiles.h -- tiles, fragments and products shared by bucket_attn_fwd.hip and bucket_attn_bwd.hip.
//
// Tensors are in the conv layout: a head's channels are rows, time is contiguous.  The matrix instruction (32x32x16, bf16, fp32
// accumulate) takes from lane l = (l31 = l & 31, kb = l >> 5) eight consecutive k of row / column l31: k = 8 kb + 0..7.  A product over
// the channels (scores) therefore needs a tile with the channels innermost, a product over time (values, gradients) one with time
// innermost.  Tiles go global -> registers -> LDS in 4 x 4 blocks (4 channels x 4 positions, one 8- or 16-byte load per channel), and
// each block is written in the orientation that its product reads:
//   rows  [position][channel]   pitch 2 DKP + 16 bytes
//   cols  [channel][position]   pitch 2 KT + 16 bytes, positions of each 16 reordered as 0-3, 8-11, 4-7, 12-15
// Both pitches are odd multiples of 16 bytes: the 16-byte fragment reads of consecutive lanes fall on different banks.  The reordering
// follows from the result layout: register r of lane (l31, kb) holds row 8 (r >> 2) + 4 kb + (r & 3) of column l31.  Registers 8 s .. 8 s + 7
// are thus the eight k of the next product's B operand for the positions 16 s + {4 kb + 0..3, 8 + 4 kb + 0..3} -- nothing moves
// between lanes from one product to the next.
//
// fp32 tensors: every operand is cut into three bf16 parts (24 bits of mantissa), six products, smallest first.  The parts of a tile
// are separate planes in LDS, cut once per workgroup.
#pragma once
#include "rel_bucket.h"
#include <svb_opaque.h>

typedef __bf16 svbt_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 svbt_bf16x2 __attribute__((ext_vector_type(2)));
typedef float svbt_f2 __attribute__((ext_vector_type(2)));
typedef float svbt_f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned svbt_u2u __attribute__((ext_vector_type(2), aligned(2)));

#define SVBT_LOG2E 1.4426950408889634f
#define SVBT_INF __builtin_inff()
#define SVBT_BAD_WORDS 4               /* bits of the keys that a workgroup's 128 queries see in part */

// T: float or unsigned short (bf16)
template <typename T> struct SvbtParts;
template <> struct SvbtParts<float> { static constexpr int NS = 3; };
template <> struct SvbtParts<unsigned short> { static constexpr int NS = 1; };

__device__ __forceinline__ unsigned svbt_pack2(float a, float b) {
    const svbt_f2 v = {a, b};
    const svbt_bf16x2 h = __builtin_convertvector(v, svbt_bf16x2);
    unsigned u;
    __builtin_memcpy(&u, &h, 4);
    return u;
}
__device__ __forceinline__ float svbt_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float svbt_hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

// two floats -> NS packed bf16 pairs that add up to them (to 2^-8, 2^-16, 2^-24 of each)
template <int NS>
__device__ __forceinline__ void svbt_parts2(float a, float b, unsigned (&p)[NS]) {
    p[0] = svbt_pack2(a, b);
    if constexpr (NS >= 2) {
        const float ra = a - svbt_lo(p[0]), rb = b - svbt_hi(p[0]);
        p[1] = svbt_pack2(ra, rb);
        if constexpr (NS == 3) p[2] = svbt_pack2(ra - svbt_lo(p[1]), rb - svbt_hi(p[1]));
    }
}
// eight floats -> NS operand fragments
template <int NS>
__device__ __forceinline__ void svbt_frag8(const float* v, svbt_bf16x8 (&f)[NS]) {
    unsigned u[NS][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned p[NS];
        svbt_parts2<NS>(v[2 * e], v[2 * e + 1], p);
#pragma unroll
        for (int n = 0; n < NS; ++n) u[n][e] = p[n];
    }
#pragma unroll
    for (int n = 0; n < NS; ++n) __builtin_memcpy(&f[n], u[n], 16);
}
// acc += A B.  `FLIP` issues the two mixed orders of three-part operands the other way round, so that A B and (B^T A^T)^T are equal
// bit for bit: the backward recomputes the scores in both orientations and compares them with the forward's maximum.
template <int NS, bool FLIP>
__device__ __forceinline__ void svbt_mma(f32x16& acc, const svbt_bf16x8 (&a)[NS], const svbt_bf16x8 (&b)[NS]) {
    if constexpr (NS == 3) {
        constexpr int X = FLIP ? 0 : 1, Y = FLIP ? 1 : 0;
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2 * X], b[2 * Y], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2 * Y], b[2 * X], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[X], b[Y], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[Y], b[X], acc, 0, 0, 0);
    }
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], acc, 0, 0, 0);
}
// Order of a block of READS fragment reads (one part each) and their products: a few reads run ahead of the products.  Left alone, the
// compiler saves registers instead: it reads into the ones that the last product has just used, and every product waits for its own read
// (backward kernels, B8 H4 dk96 T562 fp32: dq 95 -> 90 us, dk and dv 138 -> 131; B1 H8 dk64 T4000 causal bf16: dk and dv 129 -> 119).
template <int NS, int READS>
__device__ __forceinline__ void svbt_pace() {
    constexpr int AHEAD = READS < 4 ? READS : NS == 3 ? 6 : 4, PER = NS == 3 ? 2 : 1;        // (products per read)
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < READS - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, PER * AHEAD, 0);
}
__device__ __forceinline__ void svbt_zero(f32x16& a) {
#pragma unroll
    for (int r = 0; r < 16; ++r) a[r] = 0.f;
}
// row of a 32 x 32 result that register r of this lane holds: svbt_reg(r) + 4 kb
__device__ __forceinline__ constexpr int svbt_reg(int r) { return 8 * (r >> 2) + (r & 3); }
__device__ __forceinline__ int svbt_row(int r, int kb) { return svbt_reg(r) + 4 * kb; }
// a value of this tile that the compiler may not take apart: sums of it and 16 or 32 constants would otherwise be split into what changes
// per tile and what does not, and the latter kept in as many registers through the whole loop
__device__ __forceinline__ int svbt_fresh(int x) {
    unsigned u = (unsigned)x;
    svb_opaque(u);
    return (int)u;
}

// not finite, or (fp32) beyond what three bf16 parts can hold: the first part would round to infinity
__device__ __forceinline__ bool svbt_bad(float x) { return (__float_as_uint(x) & 0x7fffffffu) > 0x7f7f7fffu; }

__device__ __forceinline__ float svbt_load(const float* p) { return *p; }
__device__ __forceinline__ float svbt_load(const unsigned short* p) { return svb_bf16_f32(*p); }
__device__ __forceinline__ void svbt_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void svbt_store(unsigned short* p, float v) { *p = (unsigned short)svbt_pack2(v, v); }

// Operands of this lane's own column t (position), channels 16 s + 8 kb + 0..7: read once per workgroup, 32 lanes along time.  Loaded
// without a branch (t has to exist, a channel that does not exist reads the last one) -- a load under a condition is waited for before the
// next one -- and taken apart later: a workgroup begins by issuing these, its first tile and its tables together, one memory latency in all.
template <typename T, int NK>
struct SvbtOwn {
    T r[NK][8];
    __device__ __forceinline__ void load(const T* base, long long sc, int t, int kb, int dk) {
#pragma unroll
        for (int s = 0; s < NK; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) r[s][e] = base[min(16 * s + 8 * kb + e, dk - 1) * sc + t];
    }
    // the values of step s; `has` false or a channel beyond dk: zeros, whatever memory holds there
    __device__ __forceinline__ void get(int s, int kb, int dk, bool has, float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = has && 16 * s + 8 * kb + e < dk ? svbt_load(&r[s][e]) : 0.f;
    }
    template <int NS>
    __device__ __forceinline__ void frags(int kb, int dk, bool has, svbt_bf16x8 (&f)[NK][NS]) const {
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            float v[8];
            get(s, kb, dk, has, v);
            svbt_frag8<NS>(v, f[s]);
        }
    }
};

// ---- staged tiles ----------------------------------------------------------------------------------------------------------
// One 4 channel x 4 position block as loaded.  row(c): the c-th channel's four elements, any element-aligned address.
template <typename T> struct SvbtBlock;
template <> struct SvbtBlock<unsigned short> {
    unsigned r[4][2];
    __device__ __forceinline__ void row(int c, const unsigned short* p) {
        const svbt_u2u t = *reinterpret_cast<const svbt_u2u*>(p);
        r[c][0] = t.x;
        r[c][1] = t.y;
    }
    __device__ __forceinline__ void row_n(int c, const unsigned short* p, int n) {                       // n < 4 elements
        r[c][0] = (n > 0 ? (unsigned)p[0] : 0u) | (n > 1 ? (unsigned)p[1] << 16 : 0u);
        r[c][1] = n > 2 ? (unsigned)p[2] : 0u;
    }
    // the block was loaded `by` elements too early (4 or more: nothing of it exists)
    __device__ __forceinline__ void shift(int by) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const unsigned long long v = by < 4 ? ((unsigned long long)r[c][1] << 32 | r[c][0]) >> (16 * by) : 0ull;
            r[c][0] = (unsigned)v;
            r[c][1] = (unsigned)(v >> 32);
        }
    }
    // positions whose bit is not set become zero
    __device__ __forceinline__ void hide(unsigned seen) {
        const unsigned m0 = (seen & 1 ? 0xffffu : 0u) | (seen & 2 ? 0xffff0000u : 0u), m1 = (seen & 4 ? 0xffffu : 0u) | (seen & 8 ? 0xffff0000u : 0u);
#pragma unroll
        for (int c = 0; c < 4; ++c) { r[c][0] &= m0; r[c][1] &= m1; }
    }
    // elements that are not finite become zero, at the positions of `which`; -> the positions where there were some
    __device__ __forceinline__ unsigned clear_bad(unsigned which) {
        unsigned any = 0u, found = 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) any |= (r[c][h] & 0x7f807f80u) + 0x00800080u;                  // (an exponent of ones carries)
        if ((any & 0x80008000u) == 0u) return 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned m = e & 1 ? 0x7f800000u : 0x7f80u;
                if ((which >> e & 1u) && (r[c][e >> 1] & m) == m) {
                    r[c][e >> 1] &= e & 1 ? 0xffffu : 0xffff0000u;
                    found |= 1u << e;
                }
            }
        return found;
    }
    __device__ __forceinline__ void parts(unsigned (&o)[1][4][2]) const {
#pragma unroll
        for (int c = 0; c < 4; ++c) { o[0][c][0] = r[c][0]; o[0][c][1] = r[c][1]; }
    }
};
template <> struct SvbtBlock<float> {
    float r[4][4];
    __device__ __forceinline__ void row(int c, const float* p) {
        const svbt_f4u t = *reinterpret_cast<const svbt_f4u*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[c][e] = t[e];
    }
    __device__ __forceinline__ void row_n(int c, const float* p, int n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[c][e] = e < n ? p[e] : 0.f;
    }
    __device__ __forceinline__ void shift(int by) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (by & 2) { r[c][0] = r[c][2]; r[c][1] = r[c][3]; r[c][2] = r[c][3] = 0.f; }
            if (by & 1) { r[c][0] = r[c][1]; r[c][1] = r[c][2]; r[c][2] = r[c][3]; r[c][3] = 0.f; }
#pragma unroll
            for (int e = 0; e < 4; ++e) r[c][e] = by < 4 ? r[c][e] : 0.f;
        }
    }
    __device__ __forceinline__ void hide(unsigned seen) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) r[c][e] = seen >> e & 1 ? r[c][e] : 0.f;
    }
    __device__ __forceinline__ unsigned clear_bad(unsigned which) {
        unsigned most = 0u, found = 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = max(most, __float_as_uint(r[c][e]) & 0x7fffffffu);
        if (!svbt_bad(__uint_as_float(most))) return 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((which >> e & 1u) && svbt_bad(r[c][e])) {
                    r[c][e] = 0.f;
                    found |= 1u << e;
                }
        return found;
    }
    __device__ __forceinline__ void parts(unsigned (&o)[3][4][2]) const {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                unsigned p[3];
                svbt_parts2<3>(r[c][2 * h], r[c][2 * h + 1], p);
#pragma unroll
                for (int n = 0; n < 3; ++n) o[n][c][h] = p[n];
            }
    }
};

// KT positions x DKP channels of one tensor: NB blocks per thread of NT threads.
// A block that reaches over the end of the rows is loaded earlier, so that it ends with them, and moved into place before it is stored:
// the loads have no branches and stay in flight together.  A channel >= dk reads channel dk - 1: own operands are 0 there, and result
// rows of such channels are not written.
// TINY: rows of less than 4 elements, read one by one (a form of its own: with both in one loop the loads are waited for where they join).
// FRESH: addresses are computed anew for each tile, not kept in registers over the loop -- for the kernels that run out of registers (a spilled
// address comes back through memory, behind the tile's first loads) or get room for another workgroup.
template <typename T, int DKP, int KT, int NT, bool TINY, bool FRESH>
struct SvbtTile {
    static constexpr int NS = SvbtParts<T>::NS, JB = KT / 4, BLOCKS = JB * (DKP / 4), NB = (BLOCKS + NT - 1) / NT;
    static constexpr int ROWP = 2 * DKP + 16, COLP = 2 * KT + 16;                       // pitches, bytes
    static constexpr int ROWS_BYTES = KT * ROWP, COLS_BYTES = DKP * COLP;              // one part's plane
    // Block `id`: 32 consecutive threads take 4 blocks along time and 8 along the channels -- their 8-byte writes of rows then fall on
    // all 64 banks once (rows of positions 4 apart are 16 banks apart), where 16 blocks along time share 16 banks' width.  The loads' shorter
    // runs (32 or 64 bytes) cost less: B1 H8 dk64 T4000 causal bf16 forward 72 -> 62 us, dq 152 -> 135, dk and dv 120 -> 109.
    static __device__ __forceinline__ int pos(int id) { return 4 * ((id & 3) + 4 * ((id >> 5) % (JB / 4))); }
    static __device__ __forceinline__ int chan(int id) { return 4 * ((id >> 2 & 7) + 8 * ((id >> 5) / (JB / 4))); }
    SvbtBlock<T> b[NB];
    int tid;                           // this thread's first block
    // second: of two tiles staged together, the one that begins where the first ends (small tiles leave threads without a block)
    __device__ __forceinline__ explicit SvbtTile(bool second) : tid(second && 2 * BLOCKS <= NT ? (threadIdx.x + NT - BLOCKS) % NT : threadIdx.x) {}

    // positions j0 .. j0 + KT - 1 of rows of L elements at `base`, channel pitch sc (<= 2^25)
    __device__ __forceinline__ void load(const T* base, long long sc, int j0, int L, int dk) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = tid + i * NT, j = j0 + pos(id);
            if (BLOCKS % NT != 0 && id >= BLOCKS) continue;
            const int d = FRESH ? svbt_fresh(min(chan(id), dk - 1)) : min(chan(id), dk - 1), more = dk - 1 - d;
            long long off = (long long)d * sc + max(0, min(j, L - 4));
            svb_opaque(off);                                            // (one offset per block through the loop, not one per row)
            const T* p = base + off;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const T* pc = p + (size_t)(unsigned)min(c, more) * (unsigned)sc;
                if (TINY) b[i].row_n(c, pc, L - j);
                else b[i].row(c, pc);
            }
        }
    }
    // after the loads: blocks over the end into place, and positions whose bit is not set to zero (`seen` == ~0: all count; seen2: from 64 on)
    __device__ __forceinline__ void settle(int j0, int L, unsigned long long seen, unsigned long long seen2 = ~0ull) {
        if (!TINY && j0 + KT > L) {                                     // (uniform, as the next)
#pragma unroll
            for (int i = 0; i < NB; ++i) b[i].shift(max(0, j0 + pos(tid + i * NT) - (L - 4)));
        }
        if ((seen & seen2) != ~0ull) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int at = pos(tid + i * NT);
                b[i].hide((unsigned)((at < 64 ? seen : seen2) >> (at & 63)) & 15u);
            }
        }
    }
    // Causal tiles on the diagonal hold keys that only some of the workgroup's queries see.  Their weight is 0 for the others, but 0 times
    // an infinity or NaN is NaN: such elements of positions >= from become zero, and their positions' bits, counted from `from`, are set in
    // bad[] (LDS).  svbt_add_bad then gives them to the queries that see them.
    __device__ __forceinline__ void clear_bad(int j0, int from, unsigned* bad) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = tid + i * NT, j = j0 + pos(id);
            if (BLOCKS % NT != 0 && id >= BLOCKS) continue;
            unsigned found = b[i].clear_bad(from <= j ? 15u : from < j + 4 ? 15u << (from - j) & 15u : 0u);
            while (found) {
                const int n = j + __builtin_ctz(found) - from;
                found &= found - 1;
                atomicOr(bad + (n >> 5), 1u << (n & 31));
            }
        }
    }
    template <bool ROWS, bool COLS>
    __device__ __forceinline__ void store(char* rows, char* cols) const {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = tid + i * NT, d = chan(id), j = pos(id);
            if (BLOCKS % NT == 0 || id < BLOCKS) {
                unsigned o[NS][4][2];
                b[i].parts(o);
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    if (COLS) {
                        const int at = (j & ~15) + ((j & 4) << 1) + ((j & 8) >> 1);                    // 0, 4, 8, 12 -> 0, 8, 4, 12
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *reinterpret_cast<uint2*>(cols + n * COLS_BYTES + (d + c) * COLP + 2 * at) = make_uint2(o[n][c][0], o[n][c][1]);
                    }
                    if (ROWS) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const unsigned a0 = o[n][0][e >> 1], a1 = o[n][1][e >> 1], a2 = o[n][2][e >> 1], a3 = o[n][3][e >> 1];
                            const uint2 w = e & 1 ? make_uint2(a0 >> 16 | (a1 & 0xffff0000u), a2 >> 16 | (a3 & 0xffff0000u))
                                                  : make_uint2((a0 & 0xffffu) | a1 << 16, (a2 & 0xffffu) | a3 << 16);
                            *reinterpret_cast<uint2*>(rows + n * ROWS_BYTES + (j + e) * ROWP + 2 * d) = w;
                        }
                    }
                }
            }
        }
    }
    // A operand, rows = positions 32 sub + l31, k = channels 16 s + 8 kb + 0..7
    static __device__ __forceinline__ void row_frag(const char* rows, int sub, int s, int l31, int kb, svbt_bf16x8 (&f)[NS]) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const uint4 t = *reinterpret_cast<const uint4*>(rows + n * ROWS_BYTES + (32 * sub + l31) * ROWP + 32 * s + 16 * kb);
            __builtin_memcpy(&f[n], &t, 16);
        }
    }
    // A operand, rows = channels 32 db + l31, k = the positions of registers 8 s .. 8 s + 7 of sub-tile sub
    static __device__ __forceinline__ void col_frag(const char* cols, int db, int sub, int s, int l31, int kb, svbt_bf16x8 (&f)[NS]) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const uint4 t = *reinterpret_cast<const uint4*>(cols + n * COLS_BYTES + (32 * db + l31) * COLP + 64 * sub + 32 * s + 16 * kb);
            __builtin_memcpy(&f[n], &t, 16);
        }
    }
};

// What clear_bad took out of a tile's columns, added to the sums o[] of the query at position p where it sees them.  base, sc: the rows that
// were staged; from: the key of bit 0 of bad[].  (twice: beyond the largest bf16 that is infinite too)  Rare, and then a memory latency a key.
template <typename T, int NDB>
__device__ __forceinline__ void svbt_add_bad(f32x16 (&o)[NDB], const unsigned* bad, int words, const T* base, long long sc, int dk, int from, int p, int kb) {
#pragma unroll 1
    for (int w = 0; w < words; ++w)
#pragma unroll 1
        for (unsigned bits = bad[w]; bits; bits &= bits - 1) {
            const int j = from + 32 * w + __builtin_ctz(bits);
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float x = svbt_load(base + (min(32 * d + svbt_row(r, kb), dk - 1) * sc + j));
                    o[d][r] += j <= p && svbt_bad(x) ? x + x : 0.f;
                }
        }
}

// ---- positions and masks -----------------------------------------------------------------------------------------------------
// position of query 0 of batch entry b; far beyond any key it makes no difference how far
__device__ __forceinline__ int svbt_start(const SvbBucketAttn& a, int b) {
    int s = a.q_start;
    if (a.q_start_b) s = a.q_start_b[b];                                // (a branch: a choice between the two addresses is a flat load)
    return max(-(1 << 29), min(1 << 29, s));
}
// Per-offset tables in LDS reach SVBT_PAD beyond the last bucket border R: a tile of up to 64 x 32 pairs that has any pair nearer than R
// has none further than R + 94, so its pairs index them without a clamp -- one address per sub-tile, the rest in the instructions.
#define SVBT_PAD 96
// bias of this head per offset o in [-R - PAD, R + PAD], times log2(e) (every thread of the workgroup; the caller synchronises)
__device__ __forceinline__ void svbt_fill_bias(float* s_bias, const SvbBucketAttn& a, int h, int R, int nt) {
    for (int o = threadIdx.x; o <= 2 * (R + SVBT_PAD); o += nt)
        s_bias[o] = svb_ld_table(a.table, (size_t)svb_bucket_of(a.buckets, o - R - SVBT_PAD) * a.H + h, a.table_dtype == SVB_DT_BF16) * SVBT_LOG2E;
}
static inline int svbt_span(const SvbRelBuckets& b) { return (2 * (svb_bucket_reach(b) + SVBT_PAD) + 1 + 3) & ~3; }
// last kept key + 1 of a batch entry (0: none), by one wave; 512 keys' loads in flight, from the end
__device__ __forceinline__ int svbt_keep_end(const float* keep, int n, int lane) {
    for (int j0 = (n - 1) / 512 * 512; j0 >= 0; j0 -= 512) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = keep[min(j0 + 64 * u + lane, n - 1)];
        int last = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const unsigned long long m = __ballot(j0 + 64 * u + lane < n && v[u] != 0.f);
            if (m) last = j0 + 64 * u + 64 - __builtin_clzll(m);
        }
        if (last) return last;
    }
    return 0;
}
// (group, tile) of workgroup `id` of groups x tiles.  A group's workgroups read the same keys or queries, so they belong on one XCD
// (workgroups go round the 8 in turn).  LONG_FIRST: tile 0 of every group is the longest, the last is short; a group's tiles one after the
// other would leave the long ones of the last groups to the end (B2 H16 dk128 T2048 causal, dk and dv as they were then: 364 us that way, 250
// this way; 169 with the steps since).
__device__ __forceinline__ void svbt_item(int id, int groups, int tiles, bool long_first, int& group, int& tile) {
    if (long_first) {
        if ((groups & 7) == 0) {                                         // the groups of this XCD, tile by tile
            const int n = groups >> 3, r = id >> 3;
            tile = svb_uniform(r / n);
            group = (id & 7) * n + r - tile * n;
        } else {
            tile = svb_uniform(id / groups);
            group = id - tile * groups;
        }
    } else {
        const int item = svb_xcd_item(id, groups * tiles);
        group = svb_uniform(item / tiles);
        tile = item - group * tiles;
    }
}
