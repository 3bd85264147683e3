// rel_bucket.h -- the bucket of a relative position, shared by bucket_bias.hip and bucket_attn_{fwd,bwd}.hip.
//
// A key at offset  o = key - query  falls into one of n_buckets: with `both`, half of the buckets serve o > 0 and half o <= 0 and
// the distance is m = |o|; without it only the past counts, m = max(-o, 0).  Of a side's w buckets the first half hold one
// distance each (m < near), the others grow geometrically up to max_distance:  bucket = near + #{t : edge[t] <= m}.
// edge[t] is the least m with  near (max_distance / near)^((t+1) / (w - near)) <= m,  found by the caller in whole numbers, so
// that a distance on a border has one answer; beyond the last edge nothing changes any more.
#pragma once
#include "svb_common.h"
#include "../../include/svb_hip.h"

// A value that is the same in every lane but was computed by vector instructions (an integer division is), as a scalar: pointers built
// from it are scalar then, and a load takes a scalar base and a 32-bit offset instead of a register pair per address.
__device__ __forceinline__ int svb_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Work item of workgroup `id` of `total`: workgroups go round the 8 XCDs in turn, each with an L2 of its own; consecutive items on one
// XCD share what they read there (the keys of one head, the two halves of a line).
__device__ __forceinline__ int svb_xcd_item(int id, int total) {
    const int x = id & 7, q = total >> 3, r = total & 7;
    return x * q + min(x, r) + (id >> 3);
}

// least distance from which a side's bucket stays the same
static __host__ __device__ __forceinline__ int svb_bucket_reach(const SvbRelBuckets& b) {
    return b.n_edge > 0 ? b.edge[b.n_edge - 1] : b.near;
}

__device__ __forceinline__ int svb_bucket_of(const SvbRelBuckets& b, int off) {
    int base = 0, m = off < 0 ? -off : 0;
    if (b.both && off > 0) { base = b.n_buckets / 2; m = off; }
    if (m < b.near) return base + m;
    // all of the edges, unused ones never reached (svb_bucket_fill): a loop up to n_edge waits for a scalar load in each round
    int k = base + b.near;
#pragma unroll
    for (int t = 0; t < SVB_REL_MAX_EDGES; ++t) k += b.edge[t] <= m ? 1 : 0;
    return k;
}
// host: the edges beyond n_edge, for svb_bucket_of
static inline void svb_bucket_fill(SvbRelBuckets* b) {
    for (int t = b->n_edge; t < SVB_REL_MAX_EDGES; ++t) b->edge[t] = 0x7fffffff;
}

// the offsets a <= o < b that bucket k holds (one run; empty where k is not used)
#define SVB_REL_FAR 0x3fffffff
__device__ __forceinline__ void svb_bucket_range(const SvbRelBuckets& bk, int k, int& a, int& b) {
    const int side = bk.both ? bk.n_buckets / 2 : bk.n_buckets, m = bk.both && k >= side ? k - side : k;
    // distances lo <= d < hi of the side's bucket m
    const int lo = m <= bk.near ? m : (m - bk.near <= bk.n_edge ? bk.edge[m - bk.near - 1] : SVB_REL_FAR);
    const int hi = m < bk.near ? m + 1 : (m - bk.near < bk.n_edge ? bk.edge[m - bk.near] : SVB_REL_FAR);
    if (bk.both && k >= side) { a = max(lo, 1); b = hi; }
    else { a = 1 - hi; b = !bk.both && m == 0 ? SVB_REL_FAR : 1 - lo; }
}

// host: is this a partition that the kernels can index with?
static inline bool svb_bucket_valid(const SvbRelBuckets* b) {
    if (!b || b->n_buckets < 2 || b->n_buckets > SVB_REL_MAX_BUCKETS || (b->both && (b->n_buckets & 1))) return false;
    const int side = b->both ? b->n_buckets / 2 : b->n_buckets;
    if (b->near < 1 || b->n_edge < 0 || b->n_edge > SVB_REL_MAX_EDGES || b->near + b->n_edge + 1 > side) return false;
    int last = b->near;
    for (int t = 0; t < b->n_edge; ++t) {
        if (b->edge[t] < last || b->edge[t] > SVB_REL_MAX_REACH) return false;
        last = b->edge[t];
    }
    return b->near <= SVB_REL_MAX_REACH;
}

__device__ __forceinline__ float svb_bf16_f32(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ float svb_ld_table(const void* t, size_t i, int is_bf16) {
    return is_bf16 ? svb_bf16_f32(((const unsigned short*)t)[i]) : ((const float*)t)[i];
}
