// Attention of a serving batch without a mask tensor: causal over packed sequences of different lengths, and of a tree of drafted
// tokens over the paged cache. Here: the kernel for any head size (a multiple of 8 up to 512), and the moves of accepted drafts.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,   w_ij = exp(scale q_i . k_j)  over the keys j that query i sees
//
// packed: sequence s has the query rows [q_off[s], q_off[s+1]) and the key rows [kv_off[s], kv_off[s+1]); its last query sees all of
// its keys, the one before it one less, and so on. paged: draft i of a sequence sees the cached context, itself and its ancestors.
// A query that sees nothing gives zeros.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "kernels.h"
#include "pdl.cuh"
#include "serve_attn.cuh"

namespace tlb {

// One CTA per (query, head): a warp per key in turn, a lane per 16 bytes of the row (C of them where rows are longer than a warp's
// 512 bytes), f32 products, running maximum and sums per warp, the warps merged through shared memory. Only visible keys are read. A
// head reads its keys from L2 after the first of its group has. Bound by a warp's chain of load, product, shuffles and exponential per key: one prompt of 333
// tokens, 32 + 8 heads, takes 185 us at head size 256 and 283 at 512, 1000 tokens of 256 1533 us (10 at the tensor cores' rate); 32 sequences x 16 drafts behind 2048
// tokens 5.9 ms at 256 and 9.3 ms at 512, as keys and values are read again for every draft and query head. Two streams of such rows do not fit the
// tensor memory beside their scores, so they are not on the tensor-core kernel as it is; one stream with two tiles of 64 scores would fit up to 256.
template <typename T, bool PAGED, int C>
__global__ void __launch_bounds__(128) k_serve_attn_any(const ServeAttn a) {
    griddep_launch();
    griddep_wait();
    constexpr int WARPS = 4;
    __shared__ float ml[WARPS][2];
    __shared__ float accs[WARPS][C * 256];
    __shared__ int seq_s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = (int)blockIdx.x, head = blockIdx.y, kvh = head / (a.heads / a.kv_heads);
    if (threadIdx.x == 0) seq_s = a.seqs;
    __syncthreads();
    if (blockIdx.x == 0 && head == 0 && a.err) {
        bool bad = false;
        for (int s = threadIdx.x; s < a.seqs; s += 128) bad |= !serve_seq(a, s).ok;
        if (bad) report_error(a.err, TLB_ERR_INDEX);
    }
    if (PAGED) {
        if (threadIdx.x == 0) seq_s = row / a.drafts;
    } else {
        for (int s = threadIdx.x; s < a.seqs; s += 128) {
            const ServeSeq q = serve_seq(a, s);
            if (q.ok && row >= q.q0 && row < q.q0 + q.nq) atomicMin(&seq_s, s);
        }
    }
    __syncthreads();
    const int seq = seq_s;
    if (seq >= a.seqs) return;   // a row behind the last sequence
    const ServeSeq sq = serve_seq(a, seq);
    const int i = row - (int)sq.q0;
    uint64_t bits = 0;
    if (PAGED && i < sq.nq) bits = serve_ancestors(a, seq, i);
    const int64_t keys = i < sq.nq ? max((int64_t)0, sq.nk - sq.nq + i + 1) : 0;
    const int64_t ctx = sq.nk - sq.nq;   // paged: keys in front of the drafts
    const int chunks = a.hs >> 3;
    float qf[C][8], acc[C][8];
    const char *q0 = (const char *)a.q + (int64_t)row * a.q_stride + (int64_t)head * a.hs * 2;
#pragma unroll
    for (int c = 0; c < C; c++) {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (lane + 32 * c < chunks) raw = *reinterpret_cast<const uint4 *>(q0 + (lane + 32 * c) * 16);
        serve_unpack<T>(raw, qf[c]);
#pragma unroll
        for (int e = 0; e < 8; e++) acc[c][e] = 0.f;
    }
    float m_run = -CUDART_INF_F, l_run = -0.f;   // -0 until there is a key: -0 + 0 is +0 (a flag of its own takes up to 4 % of the time)
    const float scale_log2 = a.scale * 1.4426950408889634f;
    for (int64_t key = warp; key < keys; key += WARPS) {
        if (PAGED && key >= ctx && !((bits >> (key - ctx)) & 1)) continue;
        const ServeRow at = serve_kv_row<PAGED>(a, seq, sq, kvh, key);
        if (!at.k) continue;
        uint4 vraw[C];
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            uint4 kraw = make_uint4(0, 0, 0, 0);
            vraw[c] = make_uint4(0, 0, 0, 0);
            if (lane + 32 * c < chunks) {
                kraw = *reinterpret_cast<const uint4 *>(at.k + (lane + 32 * c) * 16);
                vraw[c] = *reinterpret_cast<const uint4 *>(at.v + (lane + 32 * c) * 16);
            }
            float kf[8];
            serve_unpack<T>(kraw, kf);
#pragma unroll
            for (int e = 0; e < 8; e++) dot = fmaf(qf[c][e], kf[e], dot);
        }
#pragma unroll
        for (int sh = 16; sh > 0; sh >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, sh);
        const float sc = dot * scale_log2;
        const float m_new = fmaxf(m_run, sc);
        const float m_use = m_new == -CUDART_INF_F ? 0.f : m_new;
        const float corr = exp2f(m_run - m_use), pw = exp2f(sc - m_use);
        m_run = m_new;
        l_run = l_run * corr + pw;
#pragma unroll
        for (int c = 0; c < C; c++) {
            float vf[8];
            serve_unpack<T>(vraw[c], vf);
#pragma unroll
            for (int e = 0; e < 8; e++) acc[c][e] = fmaf(pw, vf[e], acc[c][e] * corr);
        }
    }
    if (lane == 0) {
        ml[warp][0] = m_run;
        ml[warp][1] = l_run;
    }
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) accs[warp][(lane + 32 * c) * 8 + e] = acc[c][e];
    __syncthreads();
    float m = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < WARPS; w++) m = fmaxf(m, ml[w][0]);
    const float mu = m == -CUDART_INF_F ? 0.f : m;
    T *dst = reinterpret_cast<T *>((char *)a.out + (int64_t)row * a.out_stride) + (int64_t)head * a.hs;
    for (int d = threadIdx.x; d < a.hs; d += 128) {
        float l = 0.f, o = 0.f;
        bool sees = false;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            sees |= __float_as_uint(ml[w][1]) != 0x80000000u;
            const float f = exp2f(ml[w][0] - mu);   // 0 for a warp without a key
            l += ml[w][1] * f;
            o += accs[w][d] * f;
        }
        dst[d] = serve_round<T>(sees ? o / l : 0.f);   // of nothing but scores of -inf: 0 / 0
    }
}

const char *serve_attn_refusal(const ServeAttn &a) {
    if (a.hs < 8 || a.hs > 512 || a.hs % 8) return "the head size must be a multiple of 8 up to 512";
    if (a.kv_heads < 1 || a.heads < 1 || a.heads % a.kv_heads || a.heads > 65535) return "the query heads must be a multiple of the kv heads";
    if (a.seqs < 0 || a.seqs > 0x7fffff00 || a.q_rows < 0 || a.q_rows > 0x7fffff00 || a.kv_rows < 0 || a.kv_rows > 0x7fffff00) return "more than 2^31 - 256 rows";
    if (!(a.scale > 0.f) || a.scale > 1e38f) return "the scale must be positive and finite";
    if (a.paged) {
        if (a.bf16) return "the cache holds f16";
        if (a.drafts < 1 || a.drafts > TREE_MAX_DRAFTS) return "1 to 64 drafted tokens per sequence";
        if (a.block_size < 1 || (a.block_size & (a.block_size - 1)) || a.max_blocks < 1) return "the block size must be a power of two";
        if ((int64_t)a.max_blocks * a.block_size > 0x7fffff00) return "block tables of more than 2^31 - 256 tokens";
        if (a.pool_blocks < 0 || a.pool_blocks > 0x7fffffff) return "pools of more than 2^31 - 1 pages";
    }
    return nullptr;
}

template <typename T, bool PAGED>
static cudaError_t launch_any(const ServeAttn &a, cudaStream_t st) {
    const dim3 grid((unsigned)a.q_rows, (unsigned)a.heads);
    return a.hs <= 256 ? launch_pdl(k_serve_attn_any<T, PAGED, 1>, grid, dim3(128), 0, st, a) : launch_pdl(k_serve_attn_any<T, PAGED, 2>, grid, dim3(128), 0, st, a);
}
uint64_t serve_attn_scratch_bytes(const ServeAttn &a, int sm_count) {
    return a.q_rows && a.seqs && serve_attn_tc_supported(a) ? serve_attn_tc_scratch_bytes(a, sm_count) : 0;
}
cudaError_t launch_serve_attn(const ServeAttn &a, void *scratch, int sm_count, cudaStream_t st) {
    if (a.q_rows == 0 || a.seqs == 0) return cudaSuccess;
    if (serve_attn_tc_supported(a)) return launch_serve_attn_tc(a, scratch, sm_count, st);
    if (a.paged) return launch_any<__half, true>(a, st);
    return a.bf16 ? launch_any<__nv_bfloat16, false>(a, st) : launch_any<__half, false>(a, st);
}

// ---------------------------------------------------------------- accepted drafts
// CTA (sequence, layer, K or V): a thread owns 16 bytes of every token's row and moves them in the path's order, eight reads in flight. The
// path rises, so its j-th place is j or later: what a batch of eight writes is never read by a later one. Latency bound (a chain of three
// loads in front of the move): 32 sequences x 32 layers with up to 16 drafts, 8 heads of 128, 14.4 us behind one another in a graph (67 MB, 4.7 TB/s), one sequence with
// 8 drafts 2.8 us.
__global__ void __launch_bounds__(128) k_cache_keep(const CacheKeep a) {
    griddep_launch();
    griddep_wait();
    __shared__ int64_t from[TREE_MAX_DRAFTS], to[TREE_MAX_DRAFTS];
    const int seq = blockIdx.x, tid = threadIdx.x;
    const int count = a.counts[seq], ctx = a.context[seq];
    const int64_t cap = (int64_t)a.max_blocks * a.block_size;
    bool bad = count < 0 || count > a.drafts || ctx < 0 || ctx > cap;
    if (!bad && tid < count) {
        const int32_t *path = a.path + (int64_t)seq * a.drafts;
        const int32_t *table = a.tables + (int64_t)seq * a.max_blocks;
        const int at = path[tid];
        bad = at < (tid ? path[tid - 1] + 1 : 0) || at >= a.drafts || (int64_t)ctx + at >= cap;
        if (!bad) {
            // rows of [kv head][slot][16 bytes]: the first of the token, its heads lie block_size rows apart
            const int64_t p0 = (int64_t)ctx + at, p1 = (int64_t)ctx + tid;
            const int32_t b0 = table[p0 / a.block_size], b1 = table[p1 / a.block_size];
            bad = b0 < 0 || b0 >= a.pool_blocks || b1 < 0 || b1 >= a.pool_blocks;
            from[tid] = (int64_t)b0 * a.kv_heads * a.block_size + p0 % a.block_size;
            to[tid] = (int64_t)b1 * a.kv_heads * a.block_size + p1 % a.block_size;
        }
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0 && a.err) report_error(a.err, TLB_ERR_INDEX);
        return;
    }
    uint4 *pool = reinterpret_cast<uint4 *>(blockIdx.z ? (char *)a.vpool + a.v_layer * (int64_t)blockIdx.y : (char *)a.kpool + a.k_layer * (int64_t)blockIdx.y);
    const int cpr = a.hs / 8;
    for (int x = tid; x < a.kv_heads * cpr; x += 128) {
        const int64_t head = (int64_t)(x / cpr) * a.block_size, c = x % cpr;
        for (int j0 = 0; j0 < count; j0 += 8) {
            uint4 v[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j0 + j < count) v[j] = pool[(from[j0 + j] + head) * cpr + c];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j0 + j < count && to[j0 + j] != from[j0 + j]) pool[(to[j0 + j] + head) * cpr + c] = v[j];
        }
    }
}
cudaError_t launch_cache_keep(const CacheKeep &a, cudaStream_t st) {
    if (a.seqs == 0 || a.layers == 0) return cudaSuccess;
    return launch_pdl(k_cache_keep, dim3((unsigned)a.seqs, (unsigned)a.layers, 2), dim3(128), 0, st, a);
}

}  // namespace tlb
