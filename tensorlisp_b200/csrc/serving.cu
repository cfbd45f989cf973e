// C entry points of the serving operators on device arrays (include/tlb200.h): argument checks, the caller's stream, no allocation.
#include <algorithm>

#include "kernels.h"
#include "tlb_internal.h"

using namespace tlb;

namespace {

// The caller's current device is what it was when the call returns.
struct OnDevice {
    int before = -1;
    bool ok;
    explicit OnDevice(int ordinal) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        ok = before == ordinal || cudaSetDevice(ordinal) == cudaSuccess;
        if (before == ordinal) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

bool aligned(const void *p, uint64_t n) { return (uintptr_t)p % n == 0; }
// [p, p + n) and [q, q + m) share a byte
bool overlap(const void *p, uint64_t n, const void *q, uint64_t m) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return p && q && n && m && a < b + m && b < a + n;
}
// rows of `n` bytes, `stride` bytes apart; a dense array is one row
struct Range {
    const void *p;
    uint64_t n;
    uint64_t rows = 1, stride = 0;
    uint64_t span() const { return rows ? (rows - 1) * stride + n : 0; }
};
// Rows with one step, and a row beside others, share a byte unless each lies in the other's gaps: columns of one wide buffer do not. Different steps:
// judged by where the arrays begin and end.
bool share(const Range &a, const Range &b) {
    if (!overlap(a.p, a.span(), b.p, b.span())) return false;
    if (a.rows > 1 && b.rows > 1 && a.stride != b.stride) return true;
    const uint64_t step = a.rows > 1 ? a.stride : b.stride;
    if ((a.rows == 1 && b.rows == 1) || step == 0 || a.n > step || b.n > step) return true;
    const uint64_t x = (uintptr_t)a.p % step, y = (uintptr_t)b.p % step, d = y >= x ? y - x : y + step - x;   // from a row of a to the next of b
    return d < a.n || step - d < b.n;
}
// what a call writes shares no byte with anything else of it
bool clash(std::initializer_list<Range> writes, std::initializer_list<Range> reads) {
    for (const Range *w = writes.begin(); w != writes.end(); w++) {
        for (const Range *x = w + 1; x != writes.end(); x++)
            if (share(*w, *x)) return true;
        for (const Range &r : reads)
            if (share(*w, r)) return true;
    }
    return false;
}
bool numbers(std::initializer_list<const void *> arrays) {
    for (const void *p : arrays)
        if (!aligned(p, 4)) return false;
    return true;
}
const char *const NUMBERS = "numbers must lie on 4-byte boundaries", *const CLASH = "a result or the workspace overlaps another array";
bool product_fits(std::initializer_list<uint64_t> f) {
    unsigned __int128 n = 1;
    for (uint64_t x : f) {
        n *= x;
        if (n >> 62) return false;
    }
    return true;
}
tlb_status enqueued(const char *what, cudaError_t e) {
    if (e == cudaSuccess) return TLB_OK;
    cudaGetLastError();
    return fail(TLB_EXECUTION, std::string(what) + ": " + cuda_msg(e));
}
cudaStream_t stream_of(tlb_device *dev, void *stream) { return stream ? (cudaStream_t)stream : dev->stream; }

ServeAttn serve_args(const tlb_packed_attention_args &p) {
    ServeAttn a{};
    a.bf16 = p.type == TLB_TYPE_BF16;
    a.seqs = (int)std::min<uint32_t>(p.seqs, 0x7fffffff);
    a.heads = (int)std::min<uint32_t>(p.heads, 0x7fffffff);
    a.kv_heads = (int)std::min<uint32_t>(p.kv_heads, 0x7fffffff);
    a.hs = (int)std::min<uint32_t>(p.head_size, 0x7fffffff);
    a.scale = p.scale;
    a.q = p.q;
    a.out = p.out;
    a.q_stride = (int64_t)p.q_stride;
    a.out_stride = (int64_t)p.out_stride;
    a.q_rows = (int64_t)std::min<uint64_t>(p.q_rows, 1ull << 62);
    a.k = p.k;
    a.v = p.v;
    a.k_stride = (int64_t)p.k_stride;
    a.v_stride = (int64_t)p.v_stride;
    a.kv_rows = (int64_t)std::min<uint64_t>(p.kv_rows, 1ull << 62);
    a.q_off = p.q_offsets;
    a.kv_off = p.kv_offsets ? p.kv_offsets : p.q_offsets;
    a.err = p.status;
    return a;
}
ServeAttn serve_args(const tlb_tree_attention_args &p) {
    ServeAttn a{};
    const auto i = [](uint32_t x) { return (int)std::min<uint32_t>(x, 0x7fffffff); };
    a.paged = true;
    a.seqs = i(p.seqs);
    a.heads = i(p.heads);
    a.kv_heads = i(p.kv_heads);
    a.hs = i(p.head_size);
    a.scale = p.scale;
    a.q = p.q;
    a.out = p.out;
    a.q_stride = a.out_stride = (int64_t)a.heads * a.hs * 2;
    a.q_rows = (int64_t)a.seqs * p.drafts;
    a.k = p.k_pool;
    a.v = p.v_pool;
    a.tables = p.tables;
    a.context = p.context;
    a.counts = p.counts;
    a.parents = p.parents;
    a.drafts = i(p.drafts);
    a.block_size = i(p.block_size);
    a.max_blocks = i(p.max_blocks);
    a.pool_blocks = (int64_t)std::min<uint64_t>(p.pool_blocks, 1ull << 62);
    a.err = p.status;
    return a;
}
Logprobs logprob_args(const tlb_token_logprobs_args &p) {
    Logprobs a{};
    a.type = p.type;
    a.rows = (int64_t)std::min<uint64_t>(p.rows, 1ull << 62);
    a.vocab = (int64_t)std::min<uint64_t>(p.vocab, 1ull << 62);
    a.stride = (int64_t)p.stride;
    a.top = (int)std::min<uint32_t>(p.top, 0x7fffffff);
    a.logits = p.logits;
    a.tokens = p.tokens;
    a.logprob = p.logprob;
    a.entropy = p.entropy;
    a.top_ids = p.top_ids;
    a.top_logprobs = p.top_logprobs;
    a.out_step = 1;
    a.top_step = a.top;
    a.err = p.status;
    return a;
}
const char *logprobs_refusal(const Logprobs &a) {
    if (a.type != TLB_TYPE_F32 && a.type != TLB_TYPE_F16 && a.type != TLB_TYPE_BF16) return "logits must be f32, f16 or bf16";
    if (a.top > LOGPROBS_MAX_TOP) return "at most 32 alternatives";
    if (a.rows > 0x7fffffff || a.vocab < 1 || a.vocab > LOGPROBS_MAX_VOCAB) return "1 to 2^31 - 2048 tokens, up to 2^31 - 1 rows";
    return nullptr;
}

}  // namespace

extern "C" {

uint64_t tlb_packed_attention_workspace(tlb_device *dev, const tlb_packed_attention_args *args) {
    if (!dev || !args) return 0;
    const ServeAttn a = serve_args(*args);
    return serve_attn_refusal(a) ? 0 : serve_attn_scratch_bytes(a, dev->prop.multiProcessorCount);
}
tlb_status tlb_packed_attention(tlb_device *dev, const tlb_packed_attention_args *args, void *stream) {
    const std::string me = "tlb_packed_attention: ";
    if (!dev || !args) return fail(TLB_INVALID, me + "null argument");
    if (args->type != TLB_TYPE_F16 && args->type != TLB_TYPE_BF16) return fail(TLB_UNSUPPORTED, me + "queries, keys, values and result must be f16 or bf16");
    const ServeAttn a = serve_args(*args);
    if (const char *why = serve_attn_refusal(a)) return fail(TLB_UNSUPPORTED, me + why);
    if (a.seqs == 0 || a.q_rows == 0) return TLB_OK;
    if (!a.q || !a.out || !a.q_off || (a.kv_rows && (!a.k || !a.v))) return fail(TLB_INVALID, me + "null argument");
    const uint64_t q_row = (uint64_t)a.heads * a.hs * 2, kv_row = (uint64_t)a.kv_heads * a.hs * 2;
    for (uint64_t s : {args->q_stride, args->k_stride, args->v_stride, args->out_stride})
        if (s % 16 || s >> 40) return fail(TLB_INVALID, me + "rows must lie a multiple of 16 bytes apart (below 2^40)");
    if (args->q_stride < q_row || args->out_stride < q_row || args->k_stride < kv_row || args->v_stride < kv_row)
        return fail(TLB_INVALID, me + "a row is longer than its stride");
    if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16)) return fail(TLB_INVALID, me + "rows must start on 16-byte boundaries");
    if (!numbers({a.q_off, a.kv_off, a.err})) return fail(TLB_INVALID, me + NUMBERS);
    for (uint64_t rows : {(uint64_t)a.q_rows, (uint64_t)a.kv_rows})
        if (!product_fits({rows, std::max({args->q_stride, args->k_stride, args->v_stride, args->out_stride})})) return fail(TLB_INVALID, me + "sizes overflow");
    const uint64_t need = serve_attn_scratch_bytes(a, dev->prop.multiProcessorCount), off = ((uint64_t)a.seqs + 1) * 4;
    const uint64_t q_rows = (uint64_t)a.q_rows, kv_rows = (uint64_t)a.kv_rows;
    if (clash({{a.out, q_row, q_rows, args->out_stride}, {args->workspace, need}, {a.err, 4}},
              {{a.q, q_row, q_rows, args->q_stride}, {a.k, kv_row, kv_rows, args->k_stride}, {a.v, kv_row, kv_rows, args->v_stride}, {a.q_off, off}, {a.kv_off, off}}))
        return fail(TLB_INVALID, me + CLASH);
    if (need && (!args->workspace || args->workspace_bytes < need || !aligned(args->workspace, 16)))
        return fail(TLB_INVALID, me + "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed, got " + std::to_string(args->workspace ? args->workspace_bytes : 0));
    OnDevice on(dev->ordinal);
    if (!on.ok) return fail(TLB_NO_DEVICE, me + "cannot make the device current");
    return enqueued("tlb_packed_attention", launch_serve_attn(a, args->workspace, dev->prop.multiProcessorCount, stream_of(dev, stream)));
}

uint64_t tlb_tree_attention_workspace(tlb_device *dev, const tlb_tree_attention_args *args) {
    if (!dev || !args) return 0;
    const ServeAttn a = serve_args(*args);
    return serve_attn_refusal(a) ? 0 : serve_attn_scratch_bytes(a, dev->prop.multiProcessorCount);
}
tlb_status tlb_tree_attention(tlb_device *dev, const tlb_tree_attention_args *args, void *stream) {
    const std::string me = "tlb_tree_attention: ";
    if (!dev || !args) return fail(TLB_INVALID, me + "null argument");
    const ServeAttn a = serve_args(*args);
    if (const char *why = serve_attn_refusal(a)) return fail(TLB_UNSUPPORTED, me + why);
    if (a.seqs == 0) return TLB_OK;
    if (!a.q || !a.out || !a.tables || !a.context || !a.counts || !a.parents || (a.pool_blocks && (!a.k || !a.v))) return fail(TLB_INVALID, me + "null argument");
    if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16)) return fail(TLB_INVALID, me + "q, out and the pools must start on 16-byte boundaries");
    const uint64_t row = (uint64_t)a.heads * a.hs * 2, page = (uint64_t)a.kv_heads * a.block_size * a.hs * 2;
    if (!product_fits({(uint64_t)a.pool_blocks, page}) || !product_fits({(uint64_t)a.q_rows, row})) return fail(TLB_INVALID, me + "sizes overflow");
    if (!numbers({a.tables, a.context, a.counts, a.parents, a.err})) return fail(TLB_INVALID, me + NUMBERS);
    const uint64_t need = serve_attn_scratch_bytes(a, dev->prop.multiProcessorCount), pool = (uint64_t)a.pool_blocks * page, rows = (uint64_t)a.q_rows * row, n = (uint64_t)a.seqs * 4;
    if (clash({{a.out, rows}, {args->workspace, need}, {a.err, 4}},
              {{a.q, rows}, {a.k, pool}, {a.v, pool}, {a.tables, n * (uint64_t)a.max_blocks}, {a.context, n}, {a.counts, n}, {a.parents, n * (uint64_t)a.drafts}}))
        return fail(TLB_INVALID, me + CLASH);
    if (need && (!args->workspace || args->workspace_bytes < need || !aligned(args->workspace, 16)))
        return fail(TLB_INVALID, me + "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed, got " + std::to_string(args->workspace ? args->workspace_bytes : 0));
    OnDevice on(dev->ordinal);
    if (!on.ok) return fail(TLB_NO_DEVICE, me + "cannot make the device current");
    return enqueued("tlb_tree_attention", launch_serve_attn(a, args->workspace, dev->prop.multiProcessorCount, stream_of(dev, stream)));
}

tlb_status tlb_cache_keep(tlb_device *dev, const tlb_cache_keep_args *args, void *stream) {
    const std::string me = "tlb_cache_keep: ";
    if (!dev || !args) return fail(TLB_INVALID, me + "null argument");
    const tlb_cache_keep_args &p = *args;
    if (p.head_size < 8 || p.head_size > 512 || p.head_size % 8) return fail(TLB_UNSUPPORTED, me + "the head size must be a multiple of 8 up to 512");
    if (p.drafts < 1 || p.drafts > (uint32_t)TREE_MAX_DRAFTS) return fail(TLB_UNSUPPORTED, me + "1 to 64 drafted tokens per sequence");
    if (p.kv_heads < 1 || p.kv_heads > 65535 || p.layers > 65535 || p.seqs > 0x7fffffff || p.block_size < 1 || p.block_size > 0x7fffffff || p.max_blocks < 1 || p.max_blocks > 0x7fffffff ||
        p.pool_blocks > 0x7fffffff)
        return fail(TLB_UNSUPPORTED, me + "at most 65535 layers and kv heads, 2^31 - 1 pages, and pages of at least one token");
    const uint64_t page = (uint64_t)p.kv_heads * p.block_size * p.head_size * 2;
    if (!product_fits({p.pool_blocks, page})) return fail(TLB_INVALID, me + "sizes overflow");
    if (p.seqs == 0 || p.layers == 0 || p.pool_blocks == 0) return TLB_OK;
    if (!p.k_pools || !p.v_pools || !p.tables || !p.context || !p.counts || !p.path) return fail(TLB_INVALID, me + "null argument");
    const uint64_t pool = p.pool_blocks * page;
    if (!aligned(p.k_pools, 16) || !aligned(p.v_pools, 16) || p.k_layer_stride % 16 || p.v_layer_stride % 16 || p.k_layer_stride >> 46 || p.v_layer_stride >> 46)
        return fail(TLB_INVALID, me + "pools must start on 16-byte boundaries");
    const Range keys{p.k_pools, pool, p.layers, p.k_layer_stride}, values{p.v_pools, pool, p.layers, p.v_layer_stride};
    const bool both = (p.layers > 1 && (p.k_layer_stride < pool || p.v_layer_stride < pool)) || share(keys, values);
    if (both) return fail(TLB_INVALID, me + "two pools overlap");
    if (!numbers({p.tables, p.context, p.counts, p.path, p.status})) return fail(TLB_INVALID, me + NUMBERS);
    const uint64_t n = (uint64_t)p.seqs * 4;
    if (clash({keys, values, {p.status, 4}}, {{p.tables, n * p.max_blocks}, {p.context, n}, {p.counts, n}, {p.path, n * p.drafts}})) return fail(TLB_INVALID, me + CLASH);
    CacheKeep a{};
    a.kpool = p.k_pools;
    a.vpool = p.v_pools;
    a.k_layer = (int64_t)p.k_layer_stride;
    a.v_layer = (int64_t)p.v_layer_stride;
    a.layers = (int)p.layers;
    a.kv_heads = (int)p.kv_heads;
    a.hs = (int)p.head_size;
    a.block_size = (int)p.block_size;
    a.seqs = (int)p.seqs;
    a.max_blocks = (int)p.max_blocks;
    a.drafts = (int)p.drafts;
    a.pool_blocks = (int64_t)p.pool_blocks;
    a.tables = p.tables;
    a.context = p.context;
    a.path = p.path;
    a.counts = p.counts;
    a.err = p.status;
    OnDevice on(dev->ordinal);
    if (!on.ok) return fail(TLB_NO_DEVICE, me + "cannot make the device current");
    return enqueued("tlb_cache_keep", launch_cache_keep(a, stream_of(dev, stream)));
}

uint64_t tlb_token_logprobs_workspace(tlb_device *dev, const tlb_token_logprobs_args *args) {
    if (!dev || !args) return 0;
    const Logprobs a = logprob_args(*args);
    return logprobs_refusal(a) ? 0 : logprobs_scratch_bytes(a, dev->prop.multiProcessorCount);
}
tlb_status tlb_token_logprobs(tlb_device *dev, const tlb_token_logprobs_args *args, void *stream) {
    const std::string me = "tlb_token_logprobs: ";
    if (!dev || !args) return fail(TLB_INVALID, me + "null argument");
    const Logprobs a = logprob_args(*args);
    if (const char *why = logprobs_refusal(a)) return fail(TLB_UNSUPPORTED, me + why);
    if (a.rows == 0) return TLB_OK;
    const uint64_t elem = a.type == TLB_TYPE_F32 ? 4 : 2, row = (uint64_t)a.vocab * elem;
    if (!a.logits || (a.top && (!a.top_ids || !a.top_logprobs)) || (a.tokens && !a.logprob)) return fail(TLB_INVALID, me + "null argument");
    if (args->stride % elem || !aligned(a.logits, elem) || args->stride < row || args->stride >> 40) return fail(TLB_INVALID, me + "rows overlap or are not aligned to their values");
    if (!numbers({a.tokens, a.logprob, a.entropy, a.top_ids, a.top_logprobs, a.err})) return fail(TLB_INVALID, me + NUMBERS);
    if (!product_fits({(uint64_t)a.rows, args->stride})) return fail(TLB_INVALID, me + "sizes overflow");
    const uint64_t need = logprobs_scratch_bytes(a, dev->prop.multiProcessorCount), n = (uint64_t)a.rows * 4, nk = n * a.top;
    if (clash({{a.logprob, n}, {a.entropy, n}, {a.top_ids, nk}, {a.top_logprobs, nk}, {args->workspace, need}, {a.err, 4}}, {{a.logits, row, (uint64_t)a.rows, args->stride}, {a.tokens, n}}))
        return fail(TLB_INVALID, me + CLASH);
    if (!args->workspace || args->workspace_bytes < need || !aligned(args->workspace, 16))
        return fail(TLB_INVALID, me + "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed, got " + std::to_string(args->workspace ? args->workspace_bytes : 0));
    OnDevice on(dev->ordinal);
    if (!on.ok) return fail(TLB_NO_DEVICE, me + "cannot make the device current");
    return enqueued("tlb_token_logprobs", launch_logprobs(a, args->workspace, dev->prop.multiProcessorCount, stream_of(dev, stream)));
}

}  // extern "C"
