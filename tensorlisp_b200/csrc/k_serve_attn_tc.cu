// The attention of k_serve_attn.cu on the 5th-generation tensor cores: head sizes up to 128, f16 or bf16.
//
// A tile of 128 rows holds `tpt` tokens x the query heads of one KV head (token by token, so a short sequence or a few drafts fill it as
// well as they can), a key tile 64 or 128 keys. Keys and values come by TMA from where they lie (rows of any stride, or pages), 128-byte
// swizzled; V is read as the MN-major operand, so nothing is packed or transposed first. Columns past the head size and rows past the
// tensors are filled with zeros by the copy.
//
//   S = Q K^T (f32, tensor memory),  P = 2^(scale S - m) in the inputs' type, written over S,  O += P V (f32, tensor memory)
//
// Two streams of S and O per CTA keep the tensor core busy while the exponentials of the other one are taken:
//   SHARE  a pair of row tiles against every key tile (prompts)
//   else   one row tile, key tiles in turn; the two O are joined at the end (drafts, chunks of few tokens)
// Each has four warps, a thread per row. The maximum m that a row's exponents refer to moves when a tile's maximum has outgrown it by 2^8
// (the factor cancels; P stays far inside f16), so O is rescaled rarely. The row sums add P as it was rounded, so a dominant key's rounding
// cancels.
//
// Work is shared out evenly: the units are (row tile, KV head, key tile), in one line over all sequences, and every CTA takes an equal
// stretch of it (one persistent CTA per SM). Row tiles that are cut leave (m, l, O) in the workspace and k_serve_join adds them up. Lengths
// are read on the device, so the same launch serves any batch.
//
// Tiles at the diagonal, at the end of a sequence or in the tree are `special`: scores are masked by index, and because 0 x NaN is not 0,
// a warp looks through their values first: rows behind the sequence's end become zero, and so do values that are not finite, which the rows that see
// them get added afterwards (add_odd_values).
//
// What bounds it. Prompts: a 128 x 128 x 16 MMA takes 60 to 75 cycles to issue and execute, which was 62 % of the time of 1 x 8192 tokens (32 + 8 heads of 128) at 480 us
// (now 488 to 500 us in a graph, 1.10 to 1.13 PFLOP/s while the clock holds, 570 us and 965 TFLOP/s under the power cap); the rest is the chain of a stream (read S 250 cycles,
// maximum 400, exponentials 1400, P V and the next Q K 1024) where the other one does not cover it. Drafts: 48 sequences x 32 drafts over up to 8192 tokens 167 to 172 us
// = 4.9 to 5.1 TB/s, 204 us = 4.2 TB/s at 1520 MHz under the power cap. The same with pages of 16, 32, 64 and 128 tokens, and longer as the clock falls: not the pages' bytes but the
// streams' work per key tile (64 additions more per row and tile within the exponentials: 160 -> 185 us). Short calls: the plan (5000 cycles from the kernel's start to the first copy), an epilogue of 3000 and the joining launch (3 us).
// Polynomials for some of the exponentials (25, 38, 50 %: 500 us -> 527, 555, 622), P handed over in halves (489 -> 500) and P beside S for heads of 64 (74 -> 82)
// lost.
//
// Every wait is bounded (tc_common.cuh); one that gives up sets the status word to 2.
#include <algorithm>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "kernels.h"
#include "mm_terms.cuh"
#include "pdl.cuh"
#include "serve_attn.cuh"
#include "tc_common.cuh"

namespace tlb {

cudaError_t tc_encode_sw128(CUtensorMap *map, const void *base, int rank, const uint64_t *dims, const uint64_t *strides, const uint32_t *box, bool bf16);

namespace sat {
constexpr int T = 128;
constexpr int THREADS = 384;            // warp 0 shares out the work and copies queries and keys, 3 values, 1 issues MMAs, 2 looks through special tiles, 4-7 and 8-11 are the streams
constexpr float RESCALE_STEP = 8.f;     // in the base-2 domain
constexpr uint32_t O_COL = 256;         // S / P of stream x at column 128 x, O at 256 + 128 x
constexpr int ODD_RING = 16;
constexpr int REGS_ROLES = 88, REGS_STREAMS = 200;   // registers of a thread (setmaxnreg): the streams hold a row of 128 scores

// Keys of a tile. 64 without SHARE: a tile of values is held for a shorter time and more of them are on their way in the same room. With SHARE an MMA
// takes 60 to 75 cycles whether it has 64 keys or 128, so head size 128 takes 128
__host__ __device__ constexpr int key_tile(int hsp, bool share) { return share && hsp == 128 ? 128 : 64; }
// Tiles of S (and the P written over it) that a stream has in tensor memory. Two of them keep a stream's exponentials going while the tile in front is
// multiplied: 24 prompts of up to 1000 tokens, 16 heads of 64, 62 us against 74 with one tile of 128 keys. Heads of 128 have room for two only of 64 keys: 1 x 8192
// 531 us against 483
__host__ __device__ constexpr int buffers(int hsp, bool share) { return share && hsp == 64 ? 2 : 1; }
// What a row tile costs beside its key tiles, in key tiles. us with 1, 2, 4, 6: 1 x 8192 546, 506, 500, 511; tree 48 x 32 over
// up to 8192 182, 180, 174, 172. With 2, 3, 5, 8: 24 x 1000 of head size 64 63, 60, 62, 66
constexpr int overhead(bool share) { return share ? 3 : 5; }
// A CTA's least share, in key tiles. us with 3, 4, 6 of 64: tree 1 x 8 behind 500 12.6, 13.4, 14.6; behind 2000 14.9, 15.5, 15.5; prompt of 37 behind 500 14.1, 14.3, 15.1
constexpr int least_share(bool share) { return share ? 4 : 3; }
__host__ __device__ constexpr int stages(int hsp, bool share) { return hsp == 128 ? (share ? 2 : 6) : 8; }
__host__ __device__ constexpr int smem_bytes(int hsp, bool share) { return ((share ? 2 : 1) * T + 2 * stages(hsp, share) * key_tile(hsp, share)) * hsp * 2; }

struct Place {
    int seq, kvh, r;
    int64_t off;    // units of this row tile in front of the place
};
// The row tile that a CTA's stretch ends in, if it begins there and others go on with it
struct Cut {
    int parts;      // 0: none
    int kvh, token0;
    int q0, nq, ctx;   // the sequence's queries, keys in front of the first one's own
    int pad[2];
};
struct Params {
    CUtensorMap q, k, v;
    ServeAttn a;
    float scale_log2;
    int pool_rows;            // paged: rows of a pool
    int group, tpt, tt;       // heads per KV head; tokens of a row tile; of the row tiles that a unit covers
    int ctas, overhead, min_units;   // of a row tile; a CTA's least share
    Cut *cuts;                // [CTA], for k_serve_join
    float *partial;           // [CTA][2]: (m, l) of the rows, then O as [hsp / 4][rows][4], which the writers' lanes (rows) fill side by side
};

// ---- the line of work
// sum of floor((a i + b) / m) for 0 <= i < n; a n + b below 2^32. The points under a line, counted as in Euclid's algorithm: whole multiples of m first, what is left with
// the axes exchanged
__device__ __forceinline__ int64_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    int64_t s = 0;
    while (n > 0) {
        const uint32_t qa = a / m, qb = b / m;
        s += (int64_t)n * (n - 1) / 2 * qa + (int64_t)n * qb;
        a -= qa * m;
        b -= qb * m;
        const uint32_t y = a * n + b;   // what is left of it, turned on its side
        if (y < m) break;
        n = y / m;
        b = y - n * m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return s;
}
template <bool PAGED>
__device__ __forceinline__ int row_tiles(const Params &p, const ServeSeq &s) { return ((PAGED ? p.a.drafts : s.nq) + p.tt - 1) / p.tt; }
// key tiles of row tile r
template <bool PAGED, int KT>
__device__ __forceinline__ int key_tiles(const Params &p, const ServeSeq &s, int r) {
    if (PAGED) return r * p.tt < s.nq ? (int)((s.nk + KT - 1) / KT) : 0;
    const int64_t last = min((int64_t)s.nq, (int64_t)(r + 1) * p.tt) - 1 + s.nk - s.nq;   // the last key that its last token sees
    return last < 0 ? 0 : (int)(last / KT) + 1;
}
// units of row tiles [0, r)
template <bool PAGED, int KT>
__device__ __forceinline__ int64_t units_before(const Params &p, const ServeSeq &s, int r) {
    int64_t u = (int64_t)r * p.overhead;
    if (PAGED) return u + (int64_t)min(r, (s.nq + p.tt - 1) / p.tt) * ((s.nk + KT - 1) / KT);
    const int R = row_tiles<false>(p, s);
    const int full = min(r, R - 1);
    const int64_t off = s.nk - s.nq;
    const int first = off < 0 ? (int)min((int64_t)full, -off / p.tt) : 0;   // row tiles that see nothing
    if (full > first) {   // floor((off + (i + 1) tt - 1) / KT) + 1 of the tiles in between; whole key tiles of off go in front
        const int64_t b = off + (int64_t)(first + 1) * p.tt - 1 + KT;
        u += (int64_t)(full - first) * (b / KT) + floor_sum((uint32_t)(full - first), KT, (uint32_t)p.tt, (uint32_t)(b % KT));
    }
    if (r == R && R > 0) u += key_tiles<false, KT>(p, s, R - 1);
    return u;
}
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {   // of numbers that are not negative; 64-bit division takes ten times as long
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
// By one warp: the number of all units, and the place of one
struct LaneSeq {
    ServeSeq q;
    int64_t units;
};
template <bool PAGED, int KT>
__device__ __forceinline__ LaneSeq lane_seq(const Params &p, int s) {
    LaneSeq r;
    r.units = 0;
    if (s < p.a.seqs) {
        r.q = serve_seq(p.a, s);
        r.units = units_before<PAGED, KT>(p, r.q, row_tiles<PAGED>(p, r.q)) * p.a.kv_heads;
    }
    return r;
}
// first: sequence `lane`, with which find_unit begins
template <bool PAGED, int KT>
__device__ __forceinline__ int64_t total_units(const Params &p, LaneSeq &first) {
    const int lane = threadIdx.x & 31;
    first = lane_seq<PAGED, KT>(p, lane);
    int64_t u = first.units;
    for (int s = lane + 32; s < p.a.seqs; s += 32) u += lane_seq<PAGED, KT>(p, s).units;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
    return u;
}
template <bool PAGED, int KT>
__device__ __forceinline__ Place find_unit(const Params &p, int64_t at, const LaneSeq &first, ServeSeq &q) {
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < p.a.seqs; s0 += 32) {
        const LaneSeq mine = s0 ? lane_seq<PAGED, KT>(p, s0 + lane) : first;
        int64_t upto = mine.units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned in = __ballot_sync(0xffffffffu, at < upto);
        if (in) {
            const int l = __ffs(in) - 1;
            Place w;
            w.seq = s0 + l;
            at -= __shfl_sync(0xffffffffu, upto - mine.units, l);
            const int64_t head = divide(__shfl_sync(0xffffffffu, mine.units, l), p.a.kv_heads);
            w.kvh = (int)divide(at, head);
            at -= w.kvh * head;
            q.q0 = __shfl_sync(0xffffffffu, mine.q.q0, l);
            q.k0 = __shfl_sync(0xffffffffu, mine.q.k0, l);
            q.nk = __shfl_sync(0xffffffffu, mine.q.nk, l);
            q.nq = __shfl_sync(0xffffffffu, mine.q.nq, l);
            q.ok = true;
            // the last row tile that starts at or before `at`: 32 places at a time
            int lo = 0, n = row_tiles<PAGED>(p, q);
            int64_t before = 0;
            while (n > 1) {
                const int step = (n + 31) / 32, r = lo + lane * step;
                const int64_t x = lane * step < n ? units_before<PAGED, KT>(p, q, r) : INT64_MAX;
                const int k = __popc(__ballot_sync(0xffffffffu, x <= at)) - 1;
                before = __shfl_sync(0xffffffffu, x, k);
                lo += k * step;
                n = min(step, n - k * step);
            }
            w.r = lo;
            w.off = at - before;
            return w;
        }
        at -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return {p.a.seqs, 0, 0, 0};
}
__device__ __forceinline__ int64_t share_of(const Params &p, int64_t total) { return max((int64_t)p.min_units, divide(total + p.ctas - 1, p.ctas)); }

// A stretch of the key tiles of one row tile, as the copying warp tells it to the others
struct Segment {
    int seq, kvh, token0;         // the row tile's first token within the sequence
    int q0, k0, nq, nk;           // the sequence
    int n, t0, t1;                // key tiles [t0, t1) of n; t0 = -1: no more
    int special;                  // tiles from here on are
    __device__ __forceinline__ int ctx() const { return nk - nq; }   // keys in front of the sequence's first query
};
constexpr int SEG_RING = 4;
template <bool PAGED, int KT>
struct Walk {
    Place at;
    int64_t left;
    int loaded = -1, tiles = 0;   // the sequence at hand and its row tiles
    ServeSeq sq;
    __device__ __forceinline__ bool next(const Params &p, Segment &g) {
        while (left > 0 && at.seq < p.a.seqs) {
            if (loaded != at.seq) {
                sq = serve_seq(p.a, at.seq);
                tiles = row_tiles<PAGED>(p, sq);
                loaded = at.seq;
            }
            if (at.r >= tiles) {
                at.r = 0;
                if (tiles == 0 || ++at.kvh == p.a.kv_heads) {
                    at.kvh = 0;
                    at.seq++;
                }
                continue;
            }
            const int n = key_tiles<PAGED, KT>(p, sq, at.r);
            const int64_t take = min(left, n + p.overhead - at.off), off = at.off;
            g.seq = at.seq;
            g.kvh = at.kvh;
            g.token0 = at.r * p.tt;
            g.q0 = (int)sq.q0;
            g.k0 = (int)sq.k0;
            g.nq = sq.nq;
            g.nk = (int)sq.nk;
            g.n = n;
            g.t0 = (int)min(off, (int64_t)n);
            g.t1 = (int)min(off + take, (int64_t)n);
            // keys that every row of the unit sees: the context, or what its first token sees
            g.special = (PAGED ? g.ctx() : max(0, g.token0 + g.ctx() + 1)) / KT;
            left -= take;
            at.off += take;
            if (at.off == n + p.overhead) {
                at.off = 0;
                at.r++;
            }
            if (g.t1 > g.t0 || (n == 0 && off == 0)) return true;
        }
        return false;
    }
};

// What a row sees: keys up to `lim` (-1: none), or (PAGED, where lim is not -1) the context and the drafts of `bits`
struct RowView {
    int lim;
    uint64_t bits;
};
template <bool PAGED>
__device__ __forceinline__ bool sees(const RowView &v, int ctx, int key) {
    if (!PAGED) return key <= v.lim;
    return key < ctx ? v.lim >= 0 : key - ctx < 64 && ((v.bits >> (key - ctx)) & 1);
}
// bit i: the row sees key key0 + i
template <bool PAGED>
__device__ __forceinline__ uint32_t seen32(const RowView &v, int ctx, int key0) {
    if (!PAGED) {
        const int n = v.lim - key0 + 1;
        return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
    }
    if (v.lim < 0) return 0u;
    const int d = key0 - ctx;   // draft of bit 0
    if (d <= -32) return 0xffffffffu;
    if (d < 0) return ((1u << -d) - 1u) | (uint32_t)(v.bits << -d);
    return d < 64 ? (uint32_t)(v.bits >> d) : 0u;
}
// Parents of drafts lane and lane + 32 of a sequence, and from them the ancestors of draft i (serve_ancestors of all 64 by doubling:
// a step joins the ancestors of where the walk stands and doubles its stride)
__device__ __forceinline__ int2 load_parents(const ServeAttn &a, int seq, int count) {
    const int32_t *parents = a.parents + (int64_t)seq * a.drafts;
    const int lane = threadIdx.x & 31;
    return make_int2(lane < count ? parents[lane] : -1, lane + 32 < count ? parents[lane + 32] : -1);
}
__device__ __forceinline__ uint64_t ancestors_of(int2 up, int i, int *err) {
    const int lane = threadIdx.x & 31;
    if ((up.x < -1 || up.x >= lane || up.y < -1 || up.y >= lane + 32) && err) report_error(err, TLB_ERR_INDEX);
    if (up.x < -1 || up.x >= lane) up.x = -1;
    if (up.y < -1 || up.y >= lane + 32) up.y = -1;
    uint32_t x0 = 1u << lane, y0 = 0, y1 = 1u << lane;   // masks of drafts lane (only drafts below 32) and lane + 32
    auto at = [&](uint32_t lo, uint32_t hi, int j) {     // the value of draft j, by its lane
        const uint32_t a = __shfl_sync(0xffffffffu, lo, j & 31), b = __shfl_sync(0xffffffffu, hi, j & 31);
        return j < 32 ? a : b;
    };
#pragma unroll
    for (int step = 0; step < 6; step++) {
        const uint32_t a0 = at(x0, y0, up.x), b0 = at(x0, y0, up.y), b1 = at(0u, y1, up.y);
        const int ux = (int)at((uint32_t)up.x, (uint32_t)up.y, up.x), uy = (int)at((uint32_t)up.x, (uint32_t)up.y, up.y);
        if (up.x >= 0) {
            x0 |= a0;
            up.x = ux;
        }
        if (up.y >= 0) {
            y0 |= b0;
            y1 |= b1;
            up.y = uy;
        }
    }
    return (uint64_t)at(x0, y0, i) | (uint64_t)at(0u, y1, i) << 32;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void fma2(float &x, float &y, uint64_t s, uint64_t c) {
    uint64_t r = pack2(x, y);
    asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(r) : "l"(s), "l"(c));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
template <bool BF16>
__device__ __forceinline__ uint32_t round2(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// a += low half of w, b += the high one
template <bool BF16>
__device__ __forceinline__ void add_halves(uint32_t w, float &a, float &b) {
    if (BF16) asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.bf16 %0, l, %0;\n\tadd.rn.f32.bf16 %1, h, %1;\n\t}" : "+f"(a), "+f"(b) : "r"(w));
    else asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.f16 %0, l, %0;\n\tadd.rn.f32.f16 %1, h, %1;\n\t}" : "+f"(a), "+f"(b) : "r"(w));
}
__device__ __forceinline__ void ld32(uint32_t taddr, float *x) {
    uint32_t *r = reinterpret_cast<uint32_t *>(x);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tma_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(tc::su32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(tc::su32(bar))
                 : "memory");
}
// MN-major, 128-byte swizzle: rows of 64 elements, eight of them to a group of 1 KB; the second 64 columns lie HALF bytes further on
template <int HALF>
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(HALF >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// A row's pieces of 16 bytes (32 columns: four of them) turned around among four lanes: piece i is then row (lane & ~3) + i's, its part lane & 3,
// so that four lanes write 64 bytes of a row side by side instead of 32 lanes to 32 rows
__device__ __forceinline__ void turn4(uint4 (&w)[4]) {
    const int lane = threadIdx.x & 31;
    auto swap = [&](uint4 &a, uint4 &b, int mask) {   // the lane with the bit gives a and takes into it, the other one b
        const bool up = lane & mask;
        uint4 x = up ? a : b;
        x.x = __shfl_xor_sync(0xffffffffu, x.x, mask);
        x.y = __shfl_xor_sync(0xffffffffu, x.y, mask);
        x.z = __shfl_xor_sync(0xffffffffu, x.z, mask);
        x.w = __shfl_xor_sync(0xffffffffu, x.w, mask);
        if (up) a = x;
        else b = x;
    };
    swap(w[0], w[1], 1);
    swap(w[2], w[3], 1);
    swap(w[0], w[2], 2);
    swap(w[1], w[3], 2);
}

// ---- values of special tiles that are not finite, added to the results of a row that sees them (they were zero in the product)
// part: null where the segment is a whole row tile and its results lie in `out` already divided (inv), else its sums (rows of them); m: what the
// exponents refer to
template <typename E, bool PAGED, int KT>
__device__ __noinline__ void add_odd_values(const Params &p, const Segment &g, RowView v, int token, int head, float m, float inv, float *part, int rows, int prow) {
    ServeSeq sq;
    sq.q0 = g.q0;
    sq.k0 = g.k0;
    sq.nq = g.nq;
    sq.nk = g.nk;
    sq.ok = true;
    const char *q = (const char *)p.a.q + (int64_t)(g.q0 + token) * p.a.q_stride + (int64_t)head * p.a.hs * 2;
    E *dst = reinterpret_cast<E *>((char *)p.a.out + (int64_t)(g.q0 + token) * p.a.out_stride) + (int64_t)head * p.a.hs;
    const int ctx = g.ctx(), k1 = (int)min((int64_t)g.nk, (int64_t)g.t1 * KT);
    for (int key = max(g.t0, g.special) * KT; key < k1; key++) {
        if (!sees<PAGED>(v, ctx, key)) continue;
        const ServeRow at = serve_kv_row<PAGED>(p.a, g.seq, sq, g.kvh, key);
        if (!at.v) continue;
        float weight = -1.f;   // worked out at the first value of the key
        for (int c = 0; c < p.a.hs; c++) {
            const float y = (float)reinterpret_cast<const E *>(at.v)[c];
            if (fabsf(y) < CUDART_INF_F) continue;
            if (weight == -1.f) {
                float s = 0.f;
                for (int d = 0; d < p.a.hs; d++) s = fmaf((float)reinterpret_cast<const E *>(q)[d], (float)reinterpret_cast<const E *>(at.k)[d], s);
                weight = ex2(s * p.scale_log2 - m) * inv;
            }
            if (part) {
                float *o = part + rows * 2 + ((size_t)(c / 4) * rows + prow) * 4 + c % 4;
                *o = fmaf(weight, y, *o);
            } else {
                dst[c] = serve_round<E>(fmaf(weight, y, (float)dst[c]));
            }
        }
    }
}
}  // namespace sat

template <int HSP, bool BF16, bool PAGED, bool SHARE>
__global__ void __launch_bounds__(sat::THREADS, 1) k_serve_attn_tc(const __grid_constant__ sat::Params p) {
    using namespace tc;
    using namespace sat;
    using E = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    constexpr int BUFS = buffers(HSP, SHARE), KT = key_tile(HSP, SHARE), NS = stages(HSP, SHARE), HALVES = HSP / 64, NQ = SHARE ? 2 : 1;
    constexpr int QTILE = T * HSP * 2, QHALF = T * 128, TILE = KT * HSP * 2, KHALF = KT * 128;   // bytes; halves: 64 columns
    constexpr uint32_t FMT = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(T >> 4) << 24);
    constexpr uint32_t IDESC_QK = FMT | ((uint32_t)(KT >> 3) << 17), IDESC_PV = FMT | (1u << 16) | ((uint32_t)(HSP >> 3) << 17);
    extern __shared__ __align__(1024) uint8_t smem[];   // behind up to 3 KB of the arrays below: with six stages of 64 keys of 128 values the 227 KB are full
    uint8_t *qs = smem, *ks = qs + NQ * QTILE, *vs = ks + NS * TILE;
    __shared__ uint64_t bar_q, bar_qfree, bar_k[NS], bar_kfree[NS], bar_v[NS], bar_vfree[NS], bar_fix[NS], bar_s[2][BUFS], bar_p[2][BUFS], bar_o[2][BUFS], bar_od, bar_pair;
    __shared__ uint32_t tmem_base_s;
    __shared__ int s_fail;
    __shared__ volatile int odd_ring[ODD_RING];   // segment + 1 of those whose special tiles hold values that are not finite
    __shared__ Segment segs[SEG_RING];
    __shared__ uint64_t bar_seg[SEG_RING], bar_segfree[SEG_RING];
    __shared__ float pair_ml[2][T][2];
    volatile int *fail = &s_fail;

    // warp: known to be the same in all lanes, so that roles are branched to as one (with tid >> 5 alone: trees of 32 x 16 64 -> 71 us, 24 x 1000 63 -> 67)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        mbar_init(&bar_q, 1);
        mbar_init(&bar_qfree, 1);
        for (int i = 0; i < NS; i++) {
            mbar_init(&bar_k[i], 1);
            mbar_init(&bar_kfree[i], 1);
            mbar_init(&bar_v[i], 1);
            mbar_init(&bar_vfree[i], 1);
            mbar_init(&bar_fix[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            for (int b = 0; b < BUFS; b++) {
                mbar_init(&bar_s[i][b], 1);
                mbar_init(&bar_p[i][b], 4);
                mbar_init(&bar_o[i][b], 1);
            }
        }
        mbar_init(&bar_od, 8);
        mbar_init(&bar_pair, 8);
        for (int i = 0; i < SEG_RING; i++) {
            mbar_init(&bar_seg[i], 1);
            mbar_init(&bar_segfree[i], 11);   // every warp but the one that writes
        }
        s_fail = 0;
        for (int i = 0; i < ODD_RING; i++) odd_ring[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(&tmem_base_s, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Kernels behind may start only now: one that took this SM's tensor memory first would hold it until this CTA, which would wait for it, is over
    griddep_launch();
    griddep_wait();
    if (warp == 2 && blockIdx.x == 0 && p.a.err) {
        for (int s = lane; s < p.a.seqs; s += 32)
            if (!serve_seq(p.a, s).ok) report_error(p.a.err, TLB_ERR_INDEX);
        __syncwarp();
    }
    const uint32_t tmem = tmem_base_s;
    Segment g;
    int g_at = 0;   // segments seen
    auto next = [&]() {
        const int r = g_at % SEG_RING;
        mbar_wait_nap(&bar_seg[r], (uint32_t)(g_at / SEG_RING) & 1u, fail, 0);
        g = segs[r];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_segfree[r]);
        g_at++;
        // A warp goes on or leaves as one, also where a wait gave up and what it read is half written. (Either form for both: trees 32 x 16 72 and 48 x 32 177 us
        // against 66 and 160, 24 x 1000 68 and 1 x 8192 511 against 65 and 489)
        if (PAGED) {
            if (__any_sync(0xffffffffu, *fail)) g.t0 = -1;
            return g.t0 >= 0;
        }
        g.t0 = __shfl_sync(0xffffffffu, g.t0, 0);
        return g.t0 >= 0 && !__any_sync(0xffffffffu, *fail);
    };

    // The tiles of a segment on their way to a ring of stages (warp 0: keys, warp 3: values)
    auto copy_tiles = [&](uint8_t *ring, const CUtensorMap *map, uint64_t *full, uint64_t *free, int &tile, auto &&before, auto &&behind) {
        // paged: a box per page and 64 columns, a lane each. The page ids are loaded a tile ahead; pages that are not needed and bad ids lie past the
        // pool: zeros
        const int bs = p.a.block_size, shift = 31 - __clz(bs), rows = min(bs, KT), pages = KT / rows;   // 1 to 16 of a tile
        const int pg = lane % pages, h = lane / pages;
        auto page_id = [&](int j) {
            const int key = j * KT + pg * rows;
            return PAGED && h < HALVES && j < g.t1 && key < g.nk ? p.a.tables[(int64_t)g.seq * p.a.max_blocks + (key >> shift)] : -1;
        };
        int id = page_id(g.t0);
        for (int j = g.t0; j < g.t1; j++, tile++) {
            before(j);
            const int s = tile % NS;
            int row = p.pool_rows;
            if (PAGED) {
                const int key = j * KT + pg * rows;
                if (id >= 0 && id < p.a.pool_blocks) row = (id * p.a.kv_heads + g.kvh) * bs + (key & (bs - 1));
                else if (h < HALVES && key < g.nk && p.a.err) report_error(p.a.err, TLB_ERR_INDEX);
                id = page_id(j + 1);
            }
            mbar_wait_nap(&free[s], (uint32_t)(tile / NS + 1) & 1u, fail, 32);
            if (__any_sync(0xffffffffu, *fail)) return;
            if (lane == 0) mbar_expect_tx(&full[s], TILE);
            __syncwarp();
            if (PAGED) {
                if (h < HALVES) tma_2d(ring + s * TILE + h * KHALF + pg * rows * 128, map, h * 64, row, &full[s]);
            } else if (lane < HALVES) {
                tma_3d(ring + s * TILE + lane * KHALF, map, lane * 64, g.kvh, g.k0 + j * KT, &full[s]);
            }
            behind(j);
        }
    };
    if (warp < 4) {   // one instruction for the whole warpgroup, in front of its roles
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ROLES));
        if (warp == 0) {
            // ---- copies. The keys of a segment's first tiles are on their way before its queries, whose room the segment in front still uses.
            Walk<PAGED, KT> walk;
            int64_t share, stretch;
            {
                LaneSeq seq0;
                const int64_t total = total_units<PAGED, KT>(p, seq0);
                share = share_of(p, total);
                const int64_t first = share * blockIdx.x;
                walk.left = stretch = min(share, total - first);
                walk.at = {p.a.seqs, 0, 0, 0};
                if (walk.left > 0) {
                    walk.at = find_unit<PAGED, KT>(p, first, seq0, walk.sq);
                    walk.tiles = row_tiles<PAGED>(p, walk.sq);
                    walk.loaded = walk.at.seq;
                }
            }
            auto tell = [&](const Segment &x) {
                const int r = g_at % SEG_RING;
                mbar_wait_nap(&bar_segfree[r], (uint32_t)(g_at / SEG_RING + 1) & 1u, fail, 32);
                if (lane == 0) {
                    segs[r] = x;
                    mbar_arrive(&bar_seg[r]);
                }
                g_at++;
            };
            int tile = 0, seg = 0;
            Segment ahead;
            auto look_ahead = [&]() {
                if (!walk.next(p, ahead)) ahead.t0 = -1;
                tell(ahead);
            };
            look_ahead();
            while (ahead.t0 >= 0 && !__any_sync(0xffffffffu, *fail)) {
                g = ahead;
                if (g.t1 == g.t0) {   // a row tile that sees nothing has no part in the pipeline's counts
                    look_ahead();
                    continue;
                }
                bool have_q = false;
                auto load_q = [&]() {
                    if (lane == 0) {
                        mbar_wait_nap(&bar_qfree, (uint32_t)(seg + 1) & 1u, fail, 32);
                        mbar_expect_tx(&bar_q, (uint32_t)(NQ * HALVES * 128 * p.group * p.tpt));
                        for (int x = 0; x < NQ; x++)
                            for (int h = 0; h < HALVES; h++)
                                tma_3d(qs + x * QTILE + h * QHALF, &p.q, h * 64, g.kvh * p.group, g.q0 + g.token0 + x * p.tpt, &bar_q);
                    }
                    have_q = true;
                };
                const int look_at = min(g.t0 + 1, g.t1 - 1);
                copy_tiles(ks, &p.k, bar_k, bar_kfree, tile, [&](int j) {
                    if (!have_q && (j - g.t0 >= NS || __any_sync(0xffffffffu, mbar_test(su32(&bar_qfree), (uint32_t)(seg + 1) & 1u)))) load_q();
                }, [&](int j) {
                    if (j == look_at) look_ahead();   // the next segment, while this one's tiles are on their way
                });
                if (__any_sync(0xffffffffu, *fail)) break;
                if (!have_q) load_q();
                __syncwarp();
                seg++;
            }
            if (lane == 0) {
                Cut cut{};
                const int64_t off = walk.at.off;
                if (walk.left == 0 && off > 0 && off <= stretch) {   // further than the stretch is long: it begins in one in front
                    const int n = key_tiles<PAGED, KT>(p, walk.sq, walk.at.r);
                    if (off < n) cut = {1 + (int)divide(n - off + share - 1, share), walk.at.kvh, walk.at.r * p.tt, (int)walk.sq.q0, walk.sq.nq, (int)(walk.sq.nk - walk.sq.nq), {}};
                }
                p.cuts[blockIdx.x] = cut;
            }
        } else if (warp == 1) {
            // ---- MMA issue: S of a tile follows O of the tile that had its columns, which has read the P that it overwrites. With SHARE streams are constants of the
            // code: with them taken from a step's number, 1 x 8192 takes 500 us against 483 and 24 x 1000 of head size 64 73 against 64.
            const bool leader = elect_one();
            int tile = 0, seg = 0;
            uint32_t n_p[2] = {0, 0};
            while (next()) {
                const int n = g.t1 - g.t0;
                if (n == 0) continue;
                auto buffer = [&](int i) { return BUFS == 2 ? (tile + i) & 1 : 0; };
                auto column = [&](int x, int i) { return (uint32_t)(x * T + buffer(i) * KT); };   // of S and P
                auto issue_s = [&](int x, int i) {
                    const int s = (tile + i) % NS;
                    tc_fence_after();
                    if (leader) {
    #pragma unroll
                        for (int h = 0; h < HALVES; h++) {
                            const uint64_t qd = plain::desc_sw128(su32(qs + (SHARE ? x * QTILE : 0) + h * QHALF)), kd = plain::desc_sw128(su32(ks + s * TILE + h * KHALF));
    #pragma unroll
                            for (int e = 0; e < 4; e++) umma_f16(tmem + column(x, i), qd + 2 * e, kd + 2 * e, IDESC_QK, (h | e) ? 1u : 0u);
                        }
                        umma_commit(&bar_s[x][buffer(i)]);
                        if (!SHARE || x == 1) {
                            umma_commit(&bar_kfree[s]);
                            if (i == n - 1) umma_commit(&bar_qfree);
                        }
                    }
                    __syncwarp();
                };
                auto issue_o = [&](int x, int i) {
                    const int s = (tile + i) % NS;
                    mbar_wait_nap(&bar_p[x][buffer(i)], (BUFS == 2 ? (uint32_t)(tile + i) >> 1 : n_p[x]) & 1u, fail, 0);
                    if (i == 0 && x == 0 && seg > 0) mbar_wait_nap(&bar_od, (uint32_t)(seg - 1) & 1u, fail, 0);
                    tc_fence_after();
                    if (leader) {
                        const uint64_t vd = desc_mn<KHALF>(su32(vs + s * TILE));
    #pragma unroll
                        for (int e = 0; e < KT / 16; e++)
                            umma_f16_ta(tmem + O_COL + (uint32_t)(x * T), tmem + column(x, i) + (uint32_t)(e * 8), vd + (uint64_t)(e * 128), IDESC_PV, (i > (SHARE ? 0 : 1) || e) ? 1u : 0u);
                        umma_commit(&bar_o[x][buffer(i)]);
                        if (!SHARE || x == 1) umma_commit(&bar_vfree[s]);
                    }
                    __syncwarp();
                    n_p[x]++;
                };
                auto wait_for = [&](uint64_t *bar, int i) { mbar_wait_nap(&bar[(tile + i) % NS], (uint32_t)((tile + i) / NS) & 1u, fail, 0); };
                mbar_wait_nap(&bar_q, (uint32_t)seg & 1u, fail, 0);
                // (taking a P that is ready before keys that are not, so that a tile of values is free sooner: 185 us against 177 at 48 x 4096)
                constexpr int AHEAD = SHARE ? BUFS : 2;
                for (int i = 0; i < min(AHEAD, n); i++) {
                    wait_for(bar_k, i);
                    issue_s(SHARE ? 0 : i, i);
                    if (SHARE) issue_s(1, i);
                }
                for (int i = 0; i < n; i++) {
                    const bool more = i + AHEAD < n;
                    wait_for(bar_fix, i);
                    issue_o(SHARE ? 0 : i & 1, i);
                    if (more) {
                        wait_for(bar_k, i + AHEAD);
                        issue_s(SHARE ? 0 : i & 1, i + AHEAD);
                    }
                    if (SHARE) {
                        issue_o(1, i);
                        if (more) issue_s(1, i + AHEAD);
                    }
                }
                tile += n;
                seg++;
            }
        } else if (warp == 2) {
            // ---- every tile of values passes here, in order, on its way to the MMAs. Special ones: rows behind the end become zero, the others are
            // looked through
            int tile = 0, seg = 0;
            while (next()) {
                if (g.t1 == g.t0) continue;
                for (int j = g.t0; j < g.t1; j++, tile++) {
                    const int s = tile % NS;
                    mbar_wait_nap(&bar_v[s], (uint32_t)(tile / NS) & 1u, fail, 0);
                    if (j >= g.special) {
                        const int live = min(KT, g.nk - j * KT);
                        uint4 *v = reinterpret_cast<uint4 *>(vs + s * TILE);
                        constexpr uint32_t EXP = BF16 ? 0x7f807f80u : 0x7c007c00u, ONE = BF16 ? 0x00800080u : 0x04000400u;   // one more than all ones carries into the sign
                        uint32_t odd = 0;
    #pragma unroll 8
                        for (int i = lane; i < TILE / 16; i += 32) {
                            if (((i >> 3) & (KT - 1)) >= live) {
                                v[i] = make_uint4(0, 0, 0, 0);
                            } else {
                                const uint4 w = v[i];
                                odd |= ((w.x & EXP) + ONE) | ((w.y & EXP) + ONE) | ((w.z & EXP) + ONE) | ((w.w & EXP) + ONE);
                            }
                        }
                        if (__any_sync(0xffffffffu, odd & 0x80008000u)) {
                            odd_ring[seg % ODD_RING] = seg + 1;
                            uint32_t *e = reinterpret_cast<uint32_t *>(v);
                            for (int i = lane; i < TILE / 4; i += 32) e[i] &= ~((((e[i] & EXP) + ONE) >> 15 & 0x00010001u) * 0xffffu);
                        }
                    }
                    if (j >= g.special) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar_fix[s]);
                }
                seg++;
            }
        } else if (warp == 3) {
            int tile = 0;
            while (next()) copy_tiles(vs, &p.v, bar_v, bar_vfree, tile, [](int) {}, [](int) {});
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_STREAMS));
        // ---- the streams
        const int x = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const uint32_t s_at = lanes + (uint32_t)(x * T), o_at = lanes + O_COL + (uint32_t)(x * T);
        int seg = 0, n_pair = 0;
        uint32_t done[2] = {0, 0};   // tiles of either stream so far
        // The eight warps of both streams wait for one another, as bounded as every other wait: a warp that has left after a wait gave up arrives no more
        auto pair_sync = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_pair);
            mbar_wait_nap(&bar_pair, (uint32_t)n_pair++ & 1u, fail, 20);
        };
        while (next()) {
            const int ctx = g.ctx();
            const int token = g.token0 + (SHARE ? x * p.tpt : 0) + row / p.group, head = g.kvh * p.group + row % p.group;
            const bool live_row = row < p.tpt * p.group && token < (PAGED ? p.a.drafts : g.nq);
            RowView view;
            view.bits = 0;
            view.lim = live_row && token < g.nq ? ctx + token : -1;
            int2 parents;
            if (PAGED) parents = load_parents(p.a, g.seq, g.nq);   // on their way while the tiles of the context are looked at
            bool have_bits = false;
            const int n = g.t1 - g.t0;
            const int mine = SHARE ? n : (n + 1 - x) / 2, other = SHARE ? n : (n + x) / 2;
            float m_ref = 0.f, l = 0.f;
            bool have_ref = false;
            for (int i = 0; i < mine; i++) {
                const int j = g.t0 + (SHARE ? i : 2 * i + x);
                const uint32_t t = done[x] + i, b = BUFS == 2 ? t & 1u : 0u;   // the stream's tile; its buffer, for the (t / BUFS)th time
                mbar_wait_nap(&bar_s[x][b], t / BUFS & 1u, fail, 0);
                tc_fence_after();
                float y[KT];
#pragma unroll
                for (int c = 0; c < KT / 32; c++) ld32(s_at + b * KT + 32 * c, y + 32 * c);
                tmem_ld_wait();
                if (j >= g.special) {
                    if (PAGED && !have_bits) {
                        view.bits = ancestors_of(parents, token & 63, p.a.err);
                        have_bits = true;
                    }
#pragma unroll
                    for (int c = 0; c < KT / 32; c++) {
                        const uint32_t seen = seen32<PAGED>(view, ctx, j * KT + 32 * c);
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (!((seen >> e) & 1u)) y[32 * c + e] = -CUDART_INF_F;
                    }
                }
                float mxs[4] = {y[0], y[1], y[2], y[3]};   // four chains
#pragma unroll
                for (int e = 4; e + 8 <= KT; e += 8)
#pragma unroll
                    for (int c = 0; c < 4; c++) mxs[c] = max3(mxs[c], y[e + c], y[e + 4 + c]);
#pragma unroll
                for (int c = 0; c < 4; c++) mxs[c] = fmaxf(mxs[c], y[KT - 4 + c]);
                const float mx = fmaxf(max3(mxs[0], mxs[1], mxs[2]), mxs[3]) * p.scale_log2;
                float alpha = 1.f;
                if (!have_ref) {
                    if (mx != -CUDART_INF_F) {
                        m_ref = mx;
                        have_ref = true;   // nothing has been added up for this row yet
                    }
                } else if (mx > m_ref + RESCALE_STEP) {
                    alpha = ex2(m_ref - mx);
                    m_ref = mx;
                }
                if (__any_sync(0xffffffffu, alpha != 1.f)) {   // never on a segment's first tile
                    mbar_wait_nap(&bar_o[x][(t - 1) % BUFS], (t - 1) / BUFS & 1u, fail, 0);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HSP / 32; c++) {
                        float o[32];
                        ld32(o_at + 32 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] *= alpha;
                        st32(o_at + 32 * c, reinterpret_cast<const uint32_t *>(o));
                    }
                    l *= alpha;
                }
                const uint64_t sc = pack2(p.scale_log2, p.scale_log2), ref = pack2(-m_ref, -m_ref);
#pragma unroll
                for (int c = 0; c < KT / 64; c++) {
                    uint32_t w[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        float a = y[64 * c + 2 * e], b = y[64 * c + 2 * e + 1];
                        fma2(a, b, sc, ref);
                        a = ex2(a);
                        b = ex2(b);
                        w[e] = round2<BF16>(a, b);
                    }
                    st32(s_at + b * KT + 32 * c, w);
#pragma unroll
                    for (int e = 0; e < 32; e++) y[32 * c + e] = __uint_as_float(w[e]);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_p[x][b]);
                // The sums of P as it was rounded, while it is multiplied: O has the same roundings, so the weights add up to 1 however far the reference lags.
                // Sums of the unrounded values: 24 x 1000 62 us against 65, chunks 72 against 74, 1 x 8192 472 against 488; with the reference lagging by up to 2^8 a dominant
                // key's weight was off by up to 2^-8 in bf16. Within the loop of the exponentials: trees 74 and 185 us against 66 and 160
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < KT / 2; e++) add_halves<BF16>(__float_as_uint(y[e]), sum[2 * (e & 1)], sum[2 * (e & 1) + 1]);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
            done[x] += mine;
            done[x ^ 1] += other;
            // ---- the segment's result: O / l, or (m, l, O) where the row tile was cut
            const uint32_t last = done[x] - 1;
            if (mine > 0) mbar_wait_nap(&bar_o[x][last % BUFS], last / BUFS & 1u, fail, 0);
            if (!SHARE && other > 0) mbar_wait_nap(&bar_o[x ^ 1][0], (done[x ^ 1] - 1) & 1u, fail, 0);
            tc_fence_after();
            const bool odd = n > 0 && odd_ring[seg % ODD_RING] == seg + 1;
            const bool whole = g.t0 == 0 && g.t1 == g.n;
            float *part = whole ? nullptr : p.partial + ((size_t)blockIdx.x * 2 + (g.t0 > 0 ? 0 : 1)) * (NQ * T) * (2 + HSP);
            const int prow = (SHARE ? x * T : 0) + row;
            {
                float f_mine = 1.f, f_other = 0.f;
                if (!SHARE && n > 0) {
                    // nobody is still reading what the segment in front left here: its O has come, and P V of a segment follows bar_od of the one in front
                    pair_ml[x][row][0] = have_ref ? m_ref : -CUDART_INF_F;
                    pair_ml[x][row][1] = l;
                    pair_sync();
                    const float m2 = pair_ml[x ^ 1][row][0], l2 = pair_ml[x ^ 1][row][1], m1 = have_ref ? m_ref : -CUDART_INF_F;
                    m_ref = fmaxf(m1, m2);
                    if (m_ref == -CUDART_INF_F) m_ref = 0.f;
                    f_mine = ex2(m1 - m_ref);
                    f_other = ex2(m2 - m_ref);
                    l = l * f_mine + l2 * f_other;
                }
                if (view.lim < 0) l = 0.f;   // a row that sees nothing, or no token's
                const float inv = view.lim < 0 ? 0.f : 1.f / l;   // l = 0 of one that does: nothing but scores of -inf, 0 / 0
                if (whole) {
                    f_mine *= inv;
                    f_other *= inv;
                } else if (SHARE || x == 0) {
                    *reinterpret_cast<float2 *>(part + prow * 2) = make_float2(m_ref, l);
                }
                // where the rows of this lane's four go (turn4)
                const int64_t at = (int64_t)(g.q0 + token) * p.a.out_stride + (int64_t)head * p.a.hs * 2;
                char *dst[4];
                bool ok[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    dst[i] = (char *)p.a.out + __shfl_sync(0xffffffffu, at, (lane & ~3) + i) + (lane & 3) * 16;
                    ok[i] = __shfl_sync(0xffffffffu, (int)live_row, (lane & ~3) + i);
                }
                // SHARE: a stream writes its rows; else half of the columns each
                constexpr int COLS = SHARE ? HSP : HSP / 2;
                const int c_first = SHARE ? 0 : x * COLS;
#pragma unroll 1
                for (int c0 = c_first; c0 < c_first + COLS; c0 += 32) {
                    __syncwarp();
                    float o[32];
                    ld32(o_at + c0, o);
                    tmem_ld_wait();
                    // a stream without a tile has left nothing there; a row that sees nothing has sums of zero, but a row of padding may hold anything
                    if (mine > 0) {
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] *= f_mine;
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = 0.f;
                    }
                    if (!SHARE && other > 0) {
                        float o2[32];
                        ld32(lanes + O_COL + (uint32_t)((x ^ 1) * T) + c0, o2);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = fmaf(o2[e], f_other, o[e]);
                    }
                    if (PAGED && view.lim < 0) {
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = 0.f;
                    }
                    if (whole) {
                        uint4 w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            w[i] = make_uint4(round2<BF16>(o[8 * i], o[8 * i + 1]), round2<BF16>(o[8 * i + 2], o[8 * i + 3]), round2<BF16>(o[8 * i + 4], o[8 * i + 5]),
                                              round2<BF16>(o[8 * i + 6], o[8 * i + 7]));
                        turn4(w);
                        if (c0 + (lane & 3) * 8 < p.a.hs) {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (ok[i]) *reinterpret_cast<uint4 *>(dst[i] + c0 * 2) = w[i];
                        }
                    } else if (live_row) {
                        float4 *to = reinterpret_cast<float4 *>(part + NQ * T * 2) + (size_t)(c0 / 4) * (NQ * T) + prow;
#pragma unroll
                        for (int e = 0; e < 8; e++) to[e * NQ * T] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                }
                if (odd) {
                    // the rows' results, some of them written by other lanes or (halves of the columns) the other stream's warps, are all there
                    if (SHARE) __syncwarp();
                    else pair_sync();
                    if (PAGED && !have_bits) view.bits = ancestors_of(parents, token & 63, p.a.err);
                    if (view.lim >= 0 && (SHARE || x == 0)) add_odd_values<E, PAGED, KT>(p, g, view, token, head, m_ref, whole ? inv : 1.f, part, NQ * T, prow);
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (n == 0) continue;
            if (lane == 0) mbar_arrive(&bar_od);
            seg++;
        }
    }
    // only after a wait has given up: this CTA's copies are over before its shared memory is
    if (*fail && tid == 0) {
        mbar_wait_limit(&bar_q, 0, 1u << 12);
        for (int i = 0; i < 2 * NS; i++) {
            mbar_wait_limit(&bar_k[i >> 1], i & 1, 1u << 10);
            mbar_wait_limit(&bar_v[i >> 1], i & 1, 1u << 10);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
    if (tid == 0 && s_fail && p.a.err) report_error(p.a.err, 2);
}

// Row tiles that were cut: CTA (c, rows) adds up the parts of the one that begins in stretch c of the line and reaches over its end. Bound by two trips to L2, what
// is cut and then all of (m, l, O) of up to four parts at once, and by the launch.
template <int HSP, bool BF16, bool PAGED, bool SHARE>
__global__ void __launch_bounds__(256) k_serve_join(const __grid_constant__ sat::Params p) {
    using namespace sat;
    constexpr int NQ = SHARE ? 2 : 1, ROWS = NQ * T, SLOT = ROWS * (2 + HSP), W = HSP / 32;   // float4s of a thread
    griddep_launch();
    griddep_wait();
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Cut cut = p.cuts[c];
    // 32 rows: a lane's row is its own, a warp's columns an eighth of them
    const int row = blockIdx.y * 32 + lane, x = row / T, rr = row % T;
    const int token = cut.token0 + x * p.tpt + rr / p.group, head = cut.kvh * p.group + rr % p.group;
    if (cut.parts == 0 || rr >= p.tpt * p.group || token >= (PAGED ? p.a.drafts : cut.nq)) return;
    auto slot = [&](int i) { return p.partial + ((size_t)(c + i) * 2 + (i ? 0 : 1)) * SLOT; };
    float m = -CUDART_INF_F, l = 0.f;
    float4 o[W];
#pragma unroll
    for (int e = 0; e < W; e++) o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < cut.parts; i0 += 4) {
        float2 ml[4];
        float4 y[4][W];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            ml[u] = make_float2(0.f, 0.f);
            if (i0 + u >= cut.parts) continue;
            ml[u] = *reinterpret_cast<const float2 *>(slot(i0 + u) + row * 2);
            const float4 *s = reinterpret_cast<const float4 *>(slot(i0 + u) + ROWS * 2) + (size_t)(warp * W) * ROWS + row;
#pragma unroll
            for (int e = 0; e < W; e++) y[u][e] = s[(size_t)e * ROWS];
        }
        float top = m;
        bool some = false;
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (ml[u].y != 0.f) {   // l = 0: the row sees nothing in this part
                top = fmaxf(top, ml[u].x);   // a NaN is passed over and comes in with the part's l
                some = true;
            }
        if (!some) continue;
        const float keep = ex2(m - top);
        m = top;
        l *= keep;
#pragma unroll
        for (int e = 0; e < W; e++) o[e] = make_float4(o[e].x * keep, o[e].y * keep, o[e].z * keep, o[e].w * keep);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (ml[u].y == 0.f) continue;
            const float f = ex2(ml[u].x - m);
            l = fmaf(ml[u].y, f, l);
#pragma unroll
            for (int e = 0; e < W; e++) o[e] = make_float4(fmaf(y[u][e].x, f, o[e].x), fmaf(y[u][e].y, f, o[e].y), fmaf(y[u][e].z, f, o[e].z), fmaf(y[u][e].w, f, o[e].w));
        }
    }
    const float inv = (PAGED ? token >= cut.nq : cut.ctx + token < 0) ? 0.f : 1.f / l;   // a row that sees nothing; l = 0 of one that does: 0 / 0
    char *dst = (char *)p.a.out + (int64_t)(cut.q0 + token) * p.a.out_stride + (int64_t)head * p.a.hs * 2;
#pragma unroll
    for (int e = 0; e < W; e += 2) {
        const int col = warp * (HSP / 8) + e * 4;
        if (col < p.a.hs)
            *reinterpret_cast<uint4 *>(dst + col * 2) = make_uint4(round2<BF16>(o[e].x * inv, o[e].y * inv), round2<BF16>(o[e].z * inv, o[e].w * inv),
                                                                   round2<BF16>(o[e + 1].x * inv, o[e + 1].y * inv), round2<BF16>(o[e + 1].z * inv, o[e + 1].w * inv));
    }
}

// ---------------------------------------------------------------- host side
// The register shares must not exceed what a CTA is launched with, or the streams would wait for theirs for good, and shared memory of both kinds has to fit
// (serve_attn_tc_configure).
static bool g_sat_fits = true;
bool serve_attn_tc_supported(const ServeAttn &a) {
    if (!g_sat_fits || !tc_available() || a.hs > 128 || a.heads / a.kv_heads > sat::T) return false;
    if (a.paged) return a.block_size >= 8 && a.pool_blocks > 0 && a.pool_blocks * a.kv_heads * a.block_size < 0x7fffffff;
    return a.kv_rows > 0;
}
// A pair of row tiles per unit where sequences fill more than one on average. While a pair takes a whole sequence, only if the pairs' key tiles are more than the
// SMs. us with pairs and without, 32 + 8 heads of 128: 1 x 37 tokens 10.0, 8.8; 8 x 40 12.9, 10.9; 64 x 60 31.6, 34.6; 8 x 40 behind 4000 39, 44; 1 x 100 (two pairs
// a head) 11.4, 13.7; 64 x 100 53, 70
static bool sat_share(const ServeAttn &a, int sm_count) {
    const int64_t rows = a.q_rows * (a.heads / a.kv_heads), tile = (int64_t)a.seqs * sat::T;
    return !a.paged && rows > tile && (rows > 2 * tile || (a.kv_rows + tile - 1) / tile * a.seqs * a.kv_heads > sm_count);
}
static int sat_padded(const ServeAttn &a) { return a.hs <= 64 ? 64 : 128; }
static int64_t most_key_tiles(const ServeAttn &a, int kt) { return ((a.paged ? (int64_t)a.max_blocks * a.block_size : a.kv_rows) + kt - 1) / kt; }
static int sat_ctas(const ServeAttn &a, int sm_count) {
    const bool share = sat_share(a, sm_count);
    const int64_t tt = (int64_t)(sat::T / (a.heads / a.kv_heads)) * (share ? 2 : 1);
    const int64_t tiles = a.paged ? (a.drafts + tt - 1) / tt * a.seqs : a.q_rows / tt + a.seqs;
    const int64_t kt = sat::key_tile(sat_padded(a), share), keys = most_key_tiles(a, (int)kt);
    const double units = (double)tiles * a.kv_heads * (double)(keys + sat::overhead(share)), least = sat::least_share(share);
    return units / least < sm_count ? std::max(1, (int)(units / least + 1)) : sm_count;
}
static uint64_t sat_cuts_bytes(int ctas) { return ((uint64_t)ctas * sizeof(sat::Cut) + 255) / 256 * 256; }
uint64_t serve_attn_tc_scratch_bytes(const ServeAttn &a, int sm_count) {
    const uint64_t ctas = (uint64_t)sat_ctas(a, sm_count);
    return sat_cuts_bytes((int)ctas) + ctas * 2 * (sat_share(a, sm_count) ? 2 : 1) * sat::T * (2 + sat_padded(a)) * 4;
}
template <int HSP, bool BF16, bool PAGED, bool SHARE>
static cudaError_t sat_launch(const sat::Params &p, int ctas, cudaStream_t st) {
    cudaError_t e = launch_pdl(k_serve_attn_tc<HSP, BF16, PAGED, SHARE>, dim3((unsigned)ctas), dim3(sat::THREADS), sat::smem_bytes(HSP, SHARE), st, p);
    if (e == cudaSuccess && ctas > 1 && most_key_tiles(p.a, sat::key_tile(HSP, SHARE)) > 1)   // a single key tile is never cut
        e = launch_pdl(k_serve_join<HSP, BF16, PAGED, SHARE>, dim3((unsigned)ctas - 1, (SHARE ? 2 : 1) * sat::T / 32), dim3(256), 0, st, p);
    return e;
}
template <int HSP, bool BF16, bool PAGED, bool SHARE>
static void sat_configure() {
    cudaFuncAttributes at;
    int device, room;
    const int tiles = sat::smem_bytes(HSP, SHARE);
    if (cudaFuncGetAttributes(&at, k_serve_attn_tc<HSP, BF16, PAGED, SHARE>) != cudaSuccess || cudaGetDevice(&device) != cudaSuccess ||
        cudaDeviceGetAttribute(&room, cudaDevAttrMaxSharedMemoryPerBlockOptin, device) != cudaSuccess || at.numRegs * sat::THREADS < 128 * sat::REGS_ROLES + 256 * sat::REGS_STREAMS ||
        ((int)at.sharedSizeBytes + 1023) / 1024 * 1024 + tiles > room ||
        cudaFuncSetAttribute(k_serve_attn_tc<HSP, BF16, PAGED, SHARE>, cudaFuncAttributeMaxDynamicSharedMemorySize, tiles) != cudaSuccess) {
        cudaGetLastError();
        g_sat_fits = false;
    }
}
void serve_attn_tc_configure() {
    sat_configure<64, false, false, false>();
    sat_configure<64, false, false, true>();
    sat_configure<64, true, false, false>();
    sat_configure<64, true, false, true>();
    sat_configure<128, false, false, false>();
    sat_configure<128, false, false, true>();
    sat_configure<128, true, false, false>();
    sat_configure<128, true, false, true>();
    sat_configure<64, false, true, false>();
    sat_configure<128, false, true, false>();
}
cudaError_t launch_serve_attn_tc(const ServeAttn &a, void *scratch, int sm_count, cudaStream_t st) {
    using namespace sat;
    Params p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.group = a.heads / a.kv_heads;
    p.tpt = T / p.group;
    const bool share = sat_share(a, sm_count);
    p.tt = p.tpt * (share ? 2 : 1);
    const int kt = key_tile(sat_padded(a), share);
    p.overhead = overhead(share);
    p.min_units = least_share(share);
    const uint64_t hs = (uint64_t)a.hs;
    cudaError_t e;
    {
        const uint64_t dims[3] = {hs, (uint64_t)a.heads, (uint64_t)a.q_rows}, strides[2] = {hs * 2, (uint64_t)a.q_stride};
        const uint32_t box[3] = {64, (uint32_t)p.group, (uint32_t)p.tpt};
        e = tc_encode_sw128(&p.q, a.q, 3, dims, strides, box, a.bf16);
    }
    for (int i = 0; i < 2 && e == cudaSuccess; i++) {
        if (a.paged) {
            p.pool_rows = (int)(a.pool_blocks * a.kv_heads * a.block_size);
            const uint64_t dims[2] = {hs, (uint64_t)p.pool_rows}, strides[1] = {hs * 2};
            const uint32_t box[2] = {64, (uint32_t)std::min(a.block_size, kt)};
            e = tc_encode_sw128(i ? &p.v : &p.k, i ? a.v : a.k, 2, dims, strides, box, false);
            continue;
        }
        const uint64_t dims[3] = {hs, (uint64_t)a.kv_heads, (uint64_t)a.kv_rows}, strides[2] = {hs * 2, (uint64_t)(i ? a.v_stride : a.k_stride)};
        const uint32_t box[3] = {64, 1, (uint32_t)kt};
        e = tc_encode_sw128(i ? &p.v : &p.k, i ? a.v : a.k, 3, dims, strides, box, a.bf16);
    }
    if (e != cudaSuccess) return e;
    const int ctas = p.ctas = sat_ctas(a, sm_count);
    p.cuts = (Cut *)scratch;
    p.partial = (float *)((char *)scratch + sat_cuts_bytes(ctas));
    if (a.paged) return a.hs <= 64 ? sat_launch<64, false, true, false>(p, ctas, st) : sat_launch<128, false, true, false>(p, ctas, st);
    if (a.hs <= 64) {
        if (a.bf16) return share ? sat_launch<64, true, false, true>(p, ctas, st) : sat_launch<64, true, false, false>(p, ctas, st);
        return share ? sat_launch<64, false, false, true>(p, ctas, st) : sat_launch<64, false, false, false>(p, ctas, st);
    }
    if (a.bf16) return share ? sat_launch<128, true, false, true>(p, ctas, st) : sat_launch<128, true, false, false>(p, ctas, st);
    return share ? sat_launch<128, false, false, true>(p, ctas, st) : sat_launch<128, false, false, false>(p, ctas, st);
}

}  // namespace tlb
