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
// A row that holds a NaN or +inf has no distribution: its floats are NaN, its ids -1. Tokens at -inf are never listed: where fewer than
// asked for are left, the remaining ids are -1 at -inf; a row of nothing else has entropy 0 and log probabilities of -inf.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

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
// d = x - m is at least -1e4 in products with exp(d), which is 0 there: no 0 x inf
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    const float m = fmaxf(a.m, b.m), mu = m == -CUDART_INF_F ? 0.f : m;
    const float da = fmaxf(a.m - mu, -1e4f), db = fmaxf(b.m - mu, -1e4f);
    const float fa = ex2(da * LOG2E), fb = ex2(db * LOG2E);
    return {m, a.s * fa + b.s * fb, fa * (a.t + da * a.s) + fb * (b.t + db * b.s)};
}
__device__ __forceinline__ Sums join_block(Sums v, Sums *sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums w;
        w.m = __shfl_xor_sync(0xffffffffu, v.m, o);
        w.s = __shfl_xor_sync(0xffffffffu, v.s, o);
        w.t = __shfl_xor_sync(0xffffffffu, v.t, o);
        v = join(v, w);
    }
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < WARPS; w++) v = join(v, sh[w]);
    return v;
}
// A row's 16-byte pieces start `shift` elements in front of it; only whole pieces inside the row are read as such.
template <typename T>
__device__ __forceinline__ void load_piece(const T *row, int64_t vocab, int64_t first, float (&x)[Vec<T>::N]) {
    constexpr int N = Vec<T>::N;
    if (first >= 0 && first + N <= vocab) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(row + first));
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = value(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = first + i >= 0 && first + i < vocab ? value(row[first + i]) : -CUDART_INF_F;
    }
}
template <typename T>
__device__ __forceinline__ int shift_of(const T *row) { return (int)(((uintptr_t)row & 15) / sizeof(T)); }

struct Scan {
    Logprobs a;
    Sums *part;        // [rows][splits]
    float *seg_max;    // [rows][segs], null: no alternatives asked for
    int splits, segs, segs_per_split;
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
    const int shift = shift_of(row);
    const int s0 = (int)blockIdx.x * p.segs_per_split, s1 = min(p.segs, s0 + p.segs_per_split);
    Sums v = {-CUDART_INF_F, 0.f, 0.f};
    for (int seg = s0 + warp; seg < s1; seg += WARPS * UNROLL) {
        float x[UNROLL][N];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const int g = seg + u * WARPS;
            if (g < s1) {
                load_piece<T>(row, p.a.vocab, (int64_t)g * SEG + lane * N - shift, x[u]);
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) x[u][i] = -CUDART_INF_F;
            }
        }
        float mx = -CUDART_INF_F;
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            float mu = x[u][0];
#pragma unroll
            for (int i = 1; i < N; i++) mu = fmaxf(mu, x[u][i]);
            if (p.seg_max) {
                const int best = __reduce_max_sync(0xffffffffu, order(mu));
                const int g = seg + u * WARPS;
                if (lane == 0 && g < s1) p.seg_max[row_i * p.segs + g] = unorder(best);
            }
            mx = fmaxf(mx, mu);
        }
        if (mx > v.m) {
            const float d = fmaxf(v.m - mx, -1e4f), f = ex2(d * LOG2E);
            v.t = f * (v.t + d * v.s);
            v.s *= f;
            v.m = mx;
        }
        const float m = v.m == -CUDART_INF_F ? 0.f : v.m;
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float d = x[u][i] - m, e = ex2(d * LOG2E);
                v.s += e;
                v.t = fmaf(e, fmaxf(d, -1e4f), v.t);
            }
    }
    v = join_block(v, sh);
    if (threadIdx.x == 0) p.part[row_i * p.splits + blockIdx.x] = v;
}

namespace lp {
struct Best {
    int o;         // order() of the value
    uint32_t id;   // 0xffffffff: none
};
constexpr int NONE = INT32_MIN;
__device__ __forceinline__ bool after(int o, uint32_t id, const Best &last) { return o < last.o || (o == last.o && id > last.id); }

// The k largest of n candidates at(i) -> Best, equal values by rising id, to out[0..k) (id 0xffffffff where they run out). Every thread keeps
// the best of its share; the winner's thread looks for its next one, which comes after it in the order.
template <typename F>
__device__ __forceinline__ void pick(int n, int k, const F &at, Best *out, Best (*sh)[WARPS]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Best last = {INT32_MAX, 0};
    auto next = [&]() {
        Best b = {NONE, 0xffffffffu};
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const Best c = at(i);
            if (c.o > NONE && after(c.o, c.id, last) && (c.o > b.o || (c.o == b.o && c.id < b.id))) b = c;
        }
        return b;
    };
    Best mine = next();
    for (int r = 0; r < k; r++) {
        const int o = __reduce_max_sync(0xffffffffu, mine.o);
        const uint32_t id = __reduce_min_sync(0xffffffffu, mine.o == o ? mine.id : 0xffffffffu);
        if (lane == 0) sh[r & 1][warp] = {o, id};
        __syncthreads();
        Best w = sh[r & 1][0];
#pragma unroll
        for (int i = 1; i < WARPS; i++) {
            const Best c = sh[r & 1][i];
            if (c.o > w.o || (c.o == w.o && c.id < w.id)) w = c;
        }
        if (threadIdx.x == 0) out[r] = w;
        if (w.id == 0xffffffffu) {
            for (int j = r + 1 + (int)threadIdx.x; j < k; j += THREADS) out[j] = w;
            break;
        }
        if (mine.id == w.id) {
            last = mine;
            mine = next();
        }
    }
    __syncthreads();
}
// -inf and what the order puts below it are no candidates
__device__ __forceinline__ int candidate(float x) { return x > -CUDART_INF_F ? order(x) : NONE; }
}  // namespace lp

template <typename T>
__global__ void __launch_bounds__(lp::THREADS) k_logprobs_finish(const __grid_constant__ lp::Scan p) {
    using namespace lp;
    constexpr int SEG = Vec<T>::SEG;
    griddep_launch();
    griddep_wait();
    __shared__ Sums sh[WARPS];
    __shared__ Best bsh[2][WARPS], segs[LOGPROBS_MAX_TOP], best[LOGPROBS_MAX_TOP];
    const int64_t row_i = blockIdx.x;
    const Logprobs &a = p.a;
    const T *row = reinterpret_cast<const T *>((const char *)a.logits + row_i * a.stride);
    Sums v = {-CUDART_INF_F, 0.f, 0.f};
    for (int i = threadIdx.x; i < p.splits; i += THREADS) v = join(v, p.part[row_i * p.splits + i]);
    v = join_block(v, sh);
    const bool undefined = !(v.s == v.s), empty = v.s == 0.f;   // a NaN or +inf among the logits; nothing but -inf
    const float log_s = logf(v.s);
    if (threadIdx.x == 0) {
        if (a.logprob) {
            const int32_t tok = a.tokens ? a.tokens[row_i] : -1;
            float y = 0.f;
            if (tok >= 0 && tok < a.vocab) {
                y = undefined ? CUDART_NAN_F : (empty ? -CUDART_INF_F : (value(row[tok]) - v.m) - log_s);
            } else if (tok != -1) {
                y = CUDART_NAN_F;
                if (a.err) report_error(a.err, TLB_ERR_INDEX);
            }
            a.logprob[row_i * a.out_step] = y;
        }
        if (a.entropy) a.entropy[row_i * a.out_step] = undefined ? CUDART_NAN_F : (empty ? 0.f : log_s - v.t / v.s);
    }
    if (a.top == 0) return;
    if (!undefined && !empty) {
        const float *seg_max = p.seg_max + row_i * p.segs;
        const int shift = shift_of(row);
        pick(p.segs, a.top, [&](int i) { return Best{candidate(seg_max[i]), (uint32_t)i}; }, segs, bsh);
        pick(a.top * SEG, a.top, [&](int i) {
            const uint32_t seg = segs[i / SEG].id;
            const int64_t id = (int64_t)seg * SEG + i % SEG - shift;
            if (seg == 0xffffffffu || id < 0 || id >= a.vocab) return Best{NONE, 0xffffffffu};
            return Best{candidate(value(row[id])), (uint32_t)id};
        }, best, bsh);
    } else {
        if (threadIdx.x < a.top) best[threadIdx.x] = {NONE, 0xffffffffu};
        __syncthreads();
    }
    if (threadIdx.x < a.top) {
        const Best b = best[threadIdx.x];
        const bool none = b.id == 0xffffffffu;
        const int64_t at = row_i * a.top_step + threadIdx.x;
        if (a.ids_f32) ((float *)a.top_ids)[at] = none ? -1.f : (float)b.id;
        else ((int32_t *)a.top_ids)[at] = none ? -1 : (int32_t)b.id;
        a.top_logprobs[at] = undefined ? CUDART_NAN_F : (none ? -CUDART_INF_F : (unorder(b.o) - v.m) - log_s);
    }
}

// ---------------------------------------------------------------- host side
template <typename T>
static lp::Scan lp_plan(const Logprobs &a, int sm_count, uint64_t *bytes) {
    lp::Scan p{};
    p.a = a;
    p.segs = (int)((a.vocab + lp::Vec<T>::N - 1 + lp::Vec<T>::SEG - 1) / lp::Vec<T>::SEG);   // wherever in 16 bytes a row starts
    const int64_t most = std::min<int64_t>(256, (p.segs + lp::WARPS - 1) / lp::WARPS);
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(most, (sm_count * 32 + a.rows - 1) / std::max<int64_t>(a.rows, 1)));
    p.segs_per_split = (p.segs + p.splits - 1) / p.splits;
    p.splits = std::max(1, (p.segs + p.segs_per_split - 1) / p.segs_per_split);
    *bytes = ((uint64_t)a.rows * p.splits * sizeof(lp::Sums) + 15) / 16 * 16 + (a.top ? (uint64_t)a.rows * p.segs * 4 : 0);
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
