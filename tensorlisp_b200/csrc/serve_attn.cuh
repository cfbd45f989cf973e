// What the kernels of k_serve_attn.cu and k_serve_attn_tc.cu share: a sequence's extent, its keys' addresses, a draft's ancestors.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"

namespace tlb {

// Query rows [q0, q0 + nq) and keys [k0, k0 + nk) of a sequence, as the caller gave them or, where they reach outside the rows or tables
// (ok false), none: a packed one is skipped, a paged one's rows are zero. nk - nq keys lie in front of the first query's own.
struct ServeSeq {
    int64_t q0, k0, nk;
    int nq;
    bool ok;
};
__device__ __forceinline__ ServeSeq serve_seq(const ServeAttn &a, int s) {
    ServeSeq r;
    if (a.paged) {
        const int64_t ctx = a.context[s];
        const int n = a.counts[s];
        r.ok = ctx >= 0 && n >= 0 && n <= a.drafts && ctx + n <= (int64_t)a.max_blocks * a.block_size;
        r.q0 = (int64_t)s * a.drafts;
        r.k0 = 0;
        r.nq = r.ok ? n : 0;
        r.nk = r.ok ? ctx + n : 0;
        return r;
    }
    const int64_t q0 = a.q_off[s], q1 = a.q_off[s + 1], k0 = a.kv_off[s], k1 = a.kv_off[s + 1];
    r.ok = q0 >= 0 && q1 >= q0 && q1 <= a.q_rows && k0 >= 0 && k1 >= k0 && k1 <= a.kv_rows;
    r.q0 = r.ok ? q0 : 0;
    r.k0 = r.ok ? k0 : 0;
    r.nq = r.ok ? (int)(q1 - q0) : 0;
    r.nk = r.ok ? k1 - k0 : 0;
    return r;
}

struct ServeRow {
    const char *k, *v;   // null: the block id lies outside the pools (reported)
};
template <bool PAGED>
__device__ __forceinline__ ServeRow serve_kv_row(const ServeAttn &a, int s, const ServeSeq &q, int kvh, int64_t key) {
    if (!PAGED) {
        const int64_t row = q.k0 + key;
        return {(const char *)a.k + row * a.k_stride + (int64_t)kvh * a.hs * 2, (const char *)a.v + row * a.v_stride + (int64_t)kvh * a.hs * 2};
    }
    const int32_t blk = a.tables[(int64_t)s * a.max_blocks + key / a.block_size];
    if (blk < 0 || blk >= a.pool_blocks) {
        if (a.err) report_error(a.err, TLB_ERR_INDEX);
        return {nullptr, nullptr};
    }
    const int64_t at = ((((int64_t)blk * a.kv_heads + kvh) * a.block_size + key % a.block_size) * a.hs) * 2;
    return {(const char *)a.k + at, (const char *)a.v + at};
}

// Bit d: draft d is draft i itself or one of its ancestors. A parent has to come before its child (-1: the context); another one is
// reported and ends the walk.
__device__ __forceinline__ uint64_t serve_ancestors(const ServeAttn &a, int s, int i) {
    const int32_t *parents = a.parents + (int64_t)s * a.drafts;
    uint64_t bits = 0;
    while (i >= 0) {
        bits |= 1ull << i;
        const int up = parents[i];
        if (up < -1 || up >= i) {
            if (a.err) report_error(a.err, TLB_ERR_INDEX);
            break;
        }
        i = up;
    }
    return bits;
}

template <typename T>
__device__ __forceinline__ void serve_unpack(const uint4 &raw, float (&f)[8]);
template <>
__device__ __forceinline__ void serve_unpack<__half>(const uint4 &raw, float (&f)[8]) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float2 x = __half22float2(h[e]);
        f[2 * e] = x.x;
        f[2 * e + 1] = x.y;
    }
}
template <>
__device__ __forceinline__ void serve_unpack<__nv_bfloat16>(const uint4 &raw, float (&f)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        f[2 * e] = __uint_as_float(w[e] << 16);
        f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
}
template <typename T>
__device__ __forceinline__ T serve_round(float x);
template <>
__device__ __forceinline__ __half serve_round<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 serve_round<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace tlb
