// Log probabilities of given tokens, entropy and the most likely tokens of rows of logits, in one pass over them.
//
//   lse = m + log s,  s = sum exp(x - m),  t = sum exp(x - m) (x - m),  m = max x
//   log p(token) = x_token - lse,   entropy = -sum p log p = log s - t / s
//
// Two launches. k_logprobs_scan cuts every row into stretches, so that a single row fills the GPU too; a stretch leaves (m, s, t), held
// per thread in f32 and rescaled when a thread's maximum moves, and the maximum of every segment (what a warp loads at once: 32 x 16
// bytes). k_logprobs_finish joins the stretches of a row. The most likely tokens lie in the segments whose maxima are the largest
// (among equal ones the first), so it picks those segments first and reads only them again.
//
// 512 rows of 128256 f32: the scan 45 us = 5.8 TB/s (the logits' bytes, 48 % of the issue slots), the finish 10 behind it (chains of a row's selection, 0.3 of
// the issue slots). One row: 8.8 us for both, latency. The finish reads the picked segments as 16-byte pieces that stay in registers: value by value and twice,
// 333 rows of 32000 bf16 took 18.5 us for both, 14.1 now.
//
// A row that holds a NaN or +inf has no distribution: its floats are NaN, its ids -1. Tokens at -inf are never listed: where fewer than
// asked for are left, the remaining ids are -1 at -inf; a row of nothing else has entropy 0 and log probabilities of -inf.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <type_traits>

#include "kernels.h"
#include "pdl.cuh"

namespace tlb {

namespace lp {
constexpr int THREADS = 256, WARPS = THREADS / 32, UNROLL = 4;
constexpr float LOG2E = 1.4426950408889634f;

template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T), SEG = 32 * N;
};
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__half x) { return __half2float(x); }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }
// order of floats as integers; -0 and 0 are one value
__device__ __forceinline__ int order(float x) {
    const int b = __float_as_int(x + 0.f);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unorder(int o) { return __int_as_float(o ^ ((o >> 31) & 0x7fffffff)); }

struct Sums {
    float m, s, t;
};
__device__ __forceinline__ float warp_max(float x) {   // NaNs have no part in it
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
// d = x - m is at least -1e4 in products with exp(d), which is 0 there: no 0 x inf
__device__ __forceinline__ void move_to(Sums &v, float m) {   // the sums with another maximum
    const float d = fmaxf(v.m - (m == -CUDART_INF_F ? 0.f : m), -1e4f), f = ex2(d * LOG2E);
    v.t = f * fmaf(d, v.s, v.t);
    v.s *= f;
    v.m = m;
}
__device__ __forceinline__ Sums join_warp(Sums v) {   // in every lane
    move_to(v, warp_max(v.m));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.s += __shfl_xor_sync(0xffffffffu, v.s, o);
        v.t += __shfl_xor_sync(0xffffffffu, v.t, o);
    }
    return v;
}
// A row's 16-byte pieces start `shift` elements in front of it; only whole pieces inside the row are read as such. Outside it: -inf.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T *row, int vocab, int first) {
    constexpr int N = Vec<T>::N;
    if (first >= 0 && first + N <= vocab) return __ldg(reinterpret_cast<const uint4 *>(row + first));
    uint32_t w[4];
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = first + i >= 0 && first + i < vocab ? reinterpret_cast<const uint32_t *>(row)[first + i] : 0xff800000u;
    } else {
        const uint32_t none = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int j = first + 2 * i;
            const uint32_t lo = j >= 0 && j < vocab ? reinterpret_cast<const uint16_t *>(row)[j] : none;
            const uint32_t hi = j + 1 >= 0 && j + 1 < vocab ? reinterpret_cast<const uint16_t *>(row)[j + 1] : none;
            w[i] = lo | hi << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <typename T>
__device__ __forceinline__ int shift_of(const T *row) { return (int)(((uintptr_t)row & 15) / sizeof(T)); }

struct Scan {
    Logprobs a;
    Sums *part;        // [rows][splits]
    float *seg_max;    // [rows][turns][UNROLL], null: no alternatives asked for
    int splits, turns, turns_per_split;
};
}  // namespace lp

template <typename T>
__global__ void __launch_bounds__(lp::THREADS) k_logprobs_scan(const __grid_constant__ lp::Scan p) {
    using namespace lp;
    constexpr int N = Vec<T>::N, SEG = Vec<T>::SEG;
    griddep_launch();
    griddep_wait();
    __shared__ Sums sh[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row_i = blockIdx.y + (int64_t)blockIdx.z * 65535;
    if (row_i >= p.a.rows) return;
    const T *row = reinterpret_cast<const T *>((const char *)p.a.logits + row_i * p.a.stride);
    const int shift = shift_of(row), vocab = (int)p.a.vocab;
    const int q0 = (int)blockIdx.x * p.turns_per_split, q1 = min(p.turns, q0 + p.turns_per_split);
    // a turn: UNROLL segments in a row; the next one's pieces are on their way while these are added up
    uint4 raw[UNROLL];
    auto fetch = [&](int q) {
        const int first = q * UNROLL * SEG - shift;
        if (first >= 0 && first + UNROLL * SEG <= vocab) {
            const uint4 *at = reinterpret_cast<const uint4 *>(row + first) + lane;
#pragma unroll
            for (int u = 0; u < UNROLL; u++) raw[u] = __ldg(at + 32 * u);
        } else {
#pragma unroll
            for (int u = 0; u < UNROLL; u++) raw[u] = load_piece<T>(row, vocab, first + u * SEG + lane * N);
        }
    };
    float m = -CUDART_INF_F;
    uint64_t sums = 0, prods = 0;   // pairs: s and t of even and odd elements
    if (q0 + warp < q1) fetch(q0 + warp);
    for (int q = q0 + warp; q < q1; q += WARPS) {
        float x[UNROLL][N];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const T *e = reinterpret_cast<const T *>(&raw[u]);
#pragma unroll
            for (int i = 0; i < N; i++) x[u][i] = value(e[i]);
        }
        if (q + WARPS < q1) fetch(q + WARPS);
        float mx = m, mu[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            mu[u] = x[u][0];
#pragma unroll
            for (int i = 1; i < N; i++) mu[u] = fmaxf(mu[u], x[u][i]);
            mx = fmaxf(mx, mu[u]);
        }
        if (p.seg_max) {
#pragma unroll
            for (int u = 0; u < UNROLL; u++) mu[u] = warp_max(mu[u]);
            if (lane == 0) *reinterpret_cast<float4 *>(p.seg_max + (row_i * p.turns + q) * UNROLL) = make_float4(mu[0], mu[1], mu[2], mu[3]);
        }
        if (mx > m) {
            const float d = fmaxf(m - mx, -1e4f), f = ex2(d * LOG2E);
            prods = mul2(pack2(f, f), fma2(pack2(d, d), sums, prods));   // as move_to
            sums = mul2(pack2(f, f), sums);
            m = mx;
        }
        const float ref = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float2 d = unpack2(add2(pack2(x[u][i], x[u][i + 1]), pack2(-ref, -ref)));
                const uint64_t at = pack2(max_nan(d.x, -1e4f), max_nan(d.y, -1e4f));
                const float2 a = unpack2(mul2(at, pack2(LOG2E, LOG2E)));
                const uint64_t e = pack2(ex2(a.x), ex2(a.y));
                sums = add2(sums, e);
                prods = fma2(e, at, prods);
            }
    }
    const float2 s2 = unpack2(sums), t2 = unpack2(prods);
    Sums v = {m, s2.x + s2.y, t2.x + t2.y};
    v = join_warp(v);
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    if (warp > 0) return;
    v = join_warp(lane < WARPS ? sh[lane] : Sums{-CUDART_INF_F, 0.f, 0.f});
    if (lane == 0) p.part[row_i * p.splits + blockIdx.x] = v;
}

namespace lp {
// A candidate as one number: the larger value first, of equal ones the lower id; 0: none. -inf is no candidate.
using Key = uint64_t;
__device__ __forceinline__ Key key_of(float x, uint32_t id) { return x > -CUDART_INF_F ? (uint64_t)((uint32_t)order(x) ^ 0x80000000u) << 32 | (0xffffffffu - id) : 0; }
__device__ __forceinline__ uint32_t id_of(Key k) { return 0xffffffffu - (uint32_t)k; }
__device__ __forceinline__ float value_of(Key k) { return unorder((int)((uint32_t)(k >> 32) ^ 0x80000000u)); }

// The k largest of the threads' candidates, each(f) calls f for a thread's, to out[0..k) (0 where they run out). The k-th best of what groups of four
// threads have is a bound: what is at least as good lies in k groups, which look through their shares again and put it on a list, whose entries then
// count who is in front of them.
// (Rounds of one maximum each took 24 us for 20 of 1000 segments and 20 of 2560 values; ranks of all 256 threads' bests 18.) The list holds LIST
// entries: up to LIST / (4 k) of a thread; more candidates are picked in rounds.
constexpr int GROUP = 4, GROUPS = THREADS / GROUP, LIST = 4096;
static_assert(GROUPS >= LOGPROBS_MAX_TOP, "the bound is one group's");
struct Select {
    Key best[GROUPS], list[LIST], bound;
    int n;
};
__device__ __forceinline__ bool select_takes(int64_t n, int k) { return (n + THREADS - 1) / THREADS * GROUP * k <= LIST; }
template <typename F>
__device__ __forceinline__ void select(int k, const F &each, Key *out, Select &sh) {
    Key mine = 0;
    each([&](Key c) { mine = max(mine, c); });
    Key group = max(mine, (Key)__shfl_xor_sync(0xffffffffu, mine, 1));
    group = max(group, (Key)__shfl_xor_sync(0xffffffffu, group, 2));
    if (threadIdx.x % GROUP == 0) sh.best[threadIdx.x / GROUP] = group;
    if (threadIdx.x == 0) {
        sh.bound = 1;   // fewer than k groups have any: all candidates
        sh.n = 0;
    }
    if (threadIdx.x < k) out[threadIdx.x] = 0;
    __syncthreads();
    if (threadIdx.x < GROUPS) {
        const Key b = sh.best[threadIdx.x];
        int ahead = 0;
#pragma unroll 16
        for (int i = 0; i < GROUPS; i++) ahead += sh.best[i] > b;
        if (ahead == k - 1 && b) sh.bound = b;
    }
    __syncthreads();
    const Key bound = sh.bound;
    if (mine >= bound)
        each([&](Key c) {
            if (c >= bound) sh.list[atomicAdd(&sh.n, 1)] = c;
        });
    __syncthreads();
    const int listed = sh.n;
    for (int i = threadIdx.x; i < listed; i += THREADS) {
        const Key c = sh.list[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < listed; j++) rank += sh.list[j] > c;
        if (rank < k) out[rank] = c;
    }
    __syncthreads();
}
// The same in rounds, for any number of candidates: every thread keeps the best of its share behind the last one picked.
template <typename F>
__device__ __forceinline__ void pick(int n, int k, const F &at, Key *out, Key (*sh)[WARPS]) {
    Key last = ~0ull;
    auto next = [&]() {
        Key b = 0;
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const Key c = at(i);
            if (c < last) b = max(b, c);
        }
        return b;
    };
    Key mine = next();
    for (int r = 0; r < k; r++) {
        Key w = mine;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w = max(w, (Key)__shfl_xor_sync(0xffffffffu, w, o));
        if ((threadIdx.x & 31) == 0) sh[r & 1][threadIdx.x >> 5] = w;
        __syncthreads();
        w = sh[r & 1][0];
#pragma unroll
        for (int i = 1; i < WARPS; i++) w = max(w, sh[r & 1][i]);
        if (threadIdx.x == 0) out[r] = w;
        if (w && mine == w) {
            last = w;
            mine = next();
        }
    }
    __syncthreads();
}
}  // namespace lp

template <typename T>
__global__ void __launch_bounds__(lp::THREADS) k_logprobs_finish(const __grid_constant__ lp::Scan p) {
    using namespace lp;
    constexpr int SEG = Vec<T>::SEG;
    griddep_launch();
    griddep_wait();
    __shared__ Sums row_s;
    __shared__ float log_s_s;
    __shared__ Key rounds[2][WARPS], segs[LOGPROBS_MAX_TOP], best[LOGPROBS_MAX_TOP];
    __shared__ Select sel;
    const int64_t row_i = blockIdx.x;
    const Logprobs &a = p.a;
    const T *row = reinterpret_cast<const T *>((const char *)a.logits + row_i * a.stride);
    if (threadIdx.x < 32) {   // the other warps begin to look for the alternatives
        const int32_t tok = a.logprob && a.tokens ? a.tokens[row_i] : -1;
        const float logit = tok >= 0 && tok < a.vocab ? value(row[tok]) : 0.f;
        Sums v = {-CUDART_INF_F, 0.f, 0.f};
        for (int i = threadIdx.x; i < p.splits; i += 32) {
            Sums w = p.part[row_i * p.splits + i];
            const float m = fmaxf(v.m, w.m);
            move_to(v, m);
            move_to(w, m);
            v.s += w.s;
            v.t += w.t;
        }
        v = join_warp(v);
        const bool undefined = !(v.s == v.s), empty = v.s == 0.f;   // a NaN or +inf among the logits; nothing but -inf
        const float log_s = logf(v.s);
        if (threadIdx.x == 0) {
            row_s = v;
            log_s_s = log_s;
            if (a.logprob) {
                float y = 0.f;
                if (tok >= 0 && tok < a.vocab) {
                    y = undefined ? CUDART_NAN_F : (empty ? -CUDART_INF_F : (logit - v.m) - log_s);
                } else if (tok != -1) {
                    y = CUDART_NAN_F;
                    if (a.err) report_error(a.err, TLB_ERR_INDEX);
                }
                a.logprob[row_i * a.out_step] = y;
            }
            if (a.entropy) a.entropy[row_i * a.out_step] = undefined ? CUDART_NAN_F : (empty ? 0.f : log_s - v.t / v.s);
        }
    }
    if (a.top == 0) return;
    const float *seg_max = p.seg_max + row_i * p.turns * UNROLL;
    const int shift = shift_of(row), n = p.turns * UNROLL;
    const auto segment = [&](int i) { return key_of(seg_max[i], (uint32_t)i); };
    if (select_takes(n, a.top)) {
        Key near[4];   // one trip for the first of a thread's
#pragma unroll
        for (int u = 0; u < 4; u++) near[u] = threadIdx.x + u * THREADS < n ? segment(threadIdx.x + u * THREADS) : 0;
        select(a.top, [&](const auto &f) {
#pragma unroll
            for (int u = 0; u < 4; u++) f(near[u]);
#pragma unroll 4
            for (int i = threadIdx.x + 4 * THREADS; i < n; i += THREADS) f(segment(i));
        }, segs, sel);
    } else {
        pick(n, a.top, segment, segs, rounds);
    }
    // A warp's segments, in 16-byte pieces that stay in registers
    constexpr int N = Vec<T>::N, MOST = LOGPROBS_MAX_TOP / WARPS;
    static_assert(MOST * N * GROUP * LOGPROBS_MAX_TOP <= LIST, "the values of the segments always fit the list");
    uint4 raw[MOST];
    int first[MOST];
#pragma unroll
    for (int u = 0; u < MOST; u++) {
        const int i = (threadIdx.x >> 5) + u * WARPS;
        const Key seg = i < a.top ? segs[i] : 0;
        first[u] = seg ? (int)id_of(seg) * SEG - shift + (threadIdx.x & 31) * N : (int)a.vocab;
        if (seg) raw[u] = load_piece<T>(row, (int)a.vocab, first[u]);
    }
    select(a.top, [&](const auto &f) {
#pragma unroll
        for (int u = 0; u < MOST; u++) {
            if (first[u] >= (int)a.vocab) continue;
            const T *e = reinterpret_cast<const T *>(&raw[u]);
#pragma unroll
            for (int i = 0; i < N; i++) f(key_of(value(e[i]), (uint32_t)(first[u] + i)));   // past the ends: -inf
        }
    }, best, sel);
    if (threadIdx.x < a.top) {
        const Sums v = row_s;
        const bool undefined = !(v.s == v.s);
        const float log_s = log_s_s;
        const Key b = undefined ? 0 : best[threadIdx.x];
        const int64_t at = row_i * a.top_step + threadIdx.x;
        if (a.ids_f32) ((float *)a.top_ids)[at] = b ? (float)id_of(b) : -1.f;
        else ((int32_t *)a.top_ids)[at] = b ? (int32_t)id_of(b) : -1;
        a.top_logprobs[at] = undefined ? CUDART_NAN_F : (b ? (value_of(b) - v.m) - log_s : -CUDART_INF_F);
    }
}

// ---------------------------------------------------------------- host side
template <typename T>
static lp::Scan lp_plan(const Logprobs &a, int sm_count, uint64_t *bytes) {
    lp::Scan p{};
    p.a = a;
    constexpr int64_t TURN = (int64_t)lp::Vec<T>::SEG * lp::UNROLL;
    static_assert(LOGPROBS_MAX_VOCAB + TURN + lp::Vec<T>::N <= 0x7fffffff, "a turn that begins in front of the row's end ends below 2^31");
    p.turns = (int)((a.vocab + lp::Vec<T>::N - 1 + TURN - 1) / TURN);   // wherever in 16 bytes a row starts
    // Eight turns of every warp where there are rows enough for 24 CTAs per SM, down to one; with few rows, CTAs of fewer warps' turns
    int64_t per = 8 * lp::WARPS;
    const auto ctas = [&](int64_t n) { return a.rows * ((p.turns + n - 1) / n); };
    while (per > lp::WARPS && ctas(per) < (int64_t)sm_count * 24) per /= 2;
    while (per > 2 && ctas(per) < sm_count) per /= 2;
    p.turns_per_split = (int)std::max<int64_t>(per, (p.turns + 255) / 256);
    p.splits = (p.turns + p.turns_per_split - 1) / p.turns_per_split;
    *bytes = ((uint64_t)a.rows * p.splits * sizeof(lp::Sums) + 15) / 16 * 16 + (a.top ? (uint64_t)a.rows * p.turns * lp::UNROLL * 4 : 0);
    return p;
}
template <typename T>
static cudaError_t lp_launch(const Logprobs &a, void *scratch, int sm_count, cudaStream_t st) {
    uint64_t bytes;
    lp::Scan p = lp_plan<T>(a, sm_count, &bytes);
    p.part = (lp::Sums *)scratch;
    p.seg_max = a.top ? (float *)((char *)scratch + ((uint64_t)a.rows * p.splits * sizeof(lp::Sums) + 15) / 16 * 16) : nullptr;
    const dim3 grid((unsigned)p.splits, (unsigned)std::min<int64_t>(a.rows, 65535), (unsigned)((a.rows + 65534) / 65535));
    const cudaError_t e = launch_pdl(k_logprobs_scan<T>, grid, dim3(lp::THREADS), 0, st, p);
    return e != cudaSuccess ? e : launch_pdl(k_logprobs_finish<T>, dim3((unsigned)a.rows), dim3(lp::THREADS), 0, st, p);
}
uint64_t logprobs_scratch_bytes(const Logprobs &a, int sm_count) {
    uint64_t bytes = 0;
    if (a.type == TLB_TYPE_F32) lp_plan<float>(a, sm_count, &bytes);
    else lp_plan<__half>(a, sm_count, &bytes);
    return bytes;
}
cudaError_t launch_logprobs(const Logprobs &a, void *scratch, int sm_count, cudaStream_t st) {
    if (a.rows == 0) return cudaSuccess;
    if (a.type == TLB_TYPE_F32) return lp_launch<float>(a, scratch, sm_count, st);
    return a.type == TLB_TYPE_F16 ? lp_launch<__half>(a, scratch, sm_count, st) : lp_launch<__nv_bfloat16>(a, scratch, sm_count, st);
}

}  // namespace tlb
