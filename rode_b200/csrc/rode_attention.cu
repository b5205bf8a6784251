// C entry points of the attention operators: argument checks, workspaces, which kernels a call runs on.
#include <algorithm>

#include "rode_attention.cuh"

namespace rode {
namespace {

constexpr int kMaxRows = 1 << 30;
constexpr int kMaxHeads = 65535;  // gridDim.y

int check_shape(const char *what, int dtype, int heads, int kv_heads, int dim, float scale) {
    if (dtype != RODE_F32 && dtype != RODE_F16 && dtype != RODE_BF16)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", what, dtype);
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads > kMaxHeads)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: heads = %d must be a positive multiple of kv_heads = %d, at most %d", what,
                    heads, kv_heads, kMaxHeads);
    if (dim <= 0 || dim % 4 != 0 || dim > 256)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: dim = %d must be a multiple of 4, at most 256", what, dim);
    if (!(scale > -INFINITY && scale < INFINITY)) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: scale must be finite", what);
    return RODE_OK;
}

int check_window(const char *what, int window, int sinks) {
    if (window <= 0 || sinks < 0)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: window = %d must be positive, sinks = %d must not be negative", what, window,
                    sinks);
    return RODE_OK;
}

// No operand has more rows than this, so that larger windows (INT_MAX for "no window") and more sinks say the same; and a position (at most 2^30 on either
// side of 0) plus or minus a window stays within 32 bits, as the kernels need it.
Window window_of(int window, int sinks, int heads, int kv_heads, int dim, float scale) {
    return {std::min(window, kMaxRows), std::min(sinks, kMaxRows), heads, kv_heads, dim, scale};
}

size_t element_bytes(int dtype) { return dtype == RODE_F32 ? 4 : 2; }

// Elements (of a power of two) that the base and all strides are multiples of, at most `most`.
bool aligned_heads(const rode_heads_t &x, int dtype, long long elements) {
    return aligned_to(x.data, elements * element_bytes(dtype)) && x.batch % elements == 0 && x.row % elements == 0 &&
           x.head % elements == 0;
}

int check_operand(const char *what, const char *name, const rode_heads_t *x, int dtype, bool read) {
    if (!read) return RODE_OK;
    if (x == nullptr || x->data == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: null pointer %s", what, name);
    if (x->batch < 0 || x->row < 0 || x->head < 0)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: %s has a negative stride", what, name);
    if (!aligned_heads(*x, dtype, 4))
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: base and strides of %s must be aligned to 4 elements", what, name);
    return RODE_OK;
}

int check_result(const char *what, const char *name, const void *x, bool written) {
    if (written && x == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: null pointer %s", what, name);
    if (written && !aligned_to(x, 16)) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: %s must be 16-byte aligned", what, name);
    return RODE_OK;
}

int check_workspace(const char *what, const void *ws, size_t have, size_t need) {
    if (need == 0) return RODE_OK;
    if (ws == nullptr || have < need)
        return fail(RODE_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", what, need, ws == nullptr ? 0 : have);
    if (!aligned_to(ws, 16)) return fail(RODE_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", what);
    return RODE_OK;
}

int check_packed(const char *what, int n_seq, const int *q_offsets, const int *k_offsets, int q_rows, int k_rows) {
    if (q_rows < 0 || k_rows < 0 || q_rows > kMaxRows || k_rows > kMaxRows)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: q_rows = %d and k_rows = %d must be 0 to 2^30", what, q_rows, k_rows);
    if ((q_offsets == nullptr) != (k_offsets == nullptr))
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: offsets of queries and keys, or neither", what);
    if (q_offsets == nullptr ? n_seq != 1 : (n_seq < 0 || n_seq > kMaxRows))
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: bad number of sequences %d", what, n_seq);
    return RODE_OK;
}

#define RODE_TRY(expr)                            \
    do {                                          \
        if (const int rode_e_ = (expr)) return rode_e_; \
    } while (0)

size_t delta_bytes(int q_rows, int heads) { return (static_cast<size_t>(q_rows) * heads * sizeof(float) + 255) / 256 * 256; }

// How a call on caches is cut up (Cached), and the floats of its workspace.
struct Parts {
    int chunk, ctas, prefix;
    bool whole;
    size_t prefix_rows, own_rows, piece_rows, bytes;
};

// Own keys: as many CTAs as are resident at a time, two per SM, with equal shares of all blocks (step_batch 207 us with whole segments, 188 so); segments of
// at most 256 keys stay whole and save the joining, and so do they behind a prefix where there are enough of them, for there CTAs must be free to go
// to the SMs that the prefix leaves.
// Prefix, 16-bit operands: CTAs of 256 rows of queries, one per SM, which the tensor cores bound, while the own keys' are bound by memory and take
// whatever SMs are left; so the prefix gets the SMs in proportion to its time (own keys at 5.4 TB/s with caches half full; blocks of 128 keys at
// 1.75 us, as measured at head dimension 128 with two tiles of requests in a CTA: smaller heads and CTAs with one tile are faster, and the prefix is then done
// before the own keys are).  fp32: CTAs of 64 rows, parts down to 64 keys.
Parts plan_parts(int dtype, int batch, int prefix, long long seen, int heads, int kv_heads, int dim) {
    Parts p = {};
    p.whole = true;
    if (batch == 0) return p;
    const int group = heads / kv_heads, sms = sm_count();
    const bool half = dtype != RODE_F32;
    p.chunk = half ? kTensorCoreChunk : kSimpleChunk;
    const long long segments = static_cast<long long>(batch) * kv_heads * ((group + p.chunk - 1) / p.chunk);
    const long long least = half ? 256 : 64;  // keys
    p.whole = seen <= least || (prefix > 0 && segments >= 2 * sms);
    p.ctas = static_cast<int>(p.whole ? segments : std::min((prefix > 0 ? 8ll : 2ll) * sms, segments * ((seen + least - 1) / least)));
    if (prefix > 0) {
        const int per_cta = half ? 2 * std::max(128 / group, 1) : std::max(64 / group, 1);
        const long long ctas = (static_cast<long long>(batch) + per_cta - 1) / per_cta * kv_heads;
        long long share = 2 * sms;
        if (half) {
            const double own_us = 0.5 * 4.0 * batch * kv_heads * static_cast<double>(seen) * dim / 5.4e6;
            const double prefix_us = ctas * ((prefix + 127) / 128) * 1.75 / sms;
            share = static_cast<long long>(sms * prefix_us / (prefix_us + own_us));
        }
        p.prefix = static_cast<int>(std::min(std::max((share + ctas / 2) / ctas, 1ll), (prefix + least - 1) / least));
    }
    const size_t rows = static_cast<size_t>(batch) * heads;
    p.prefix_rows = p.prefix * rows;
    p.own_rows = p.prefix > 0 ? rows : 0;
    p.piece_rows = p.whole ? 0 : 2ull * p.ctas * p.chunk;
    p.bytes = (p.prefix_rows + p.own_rows + p.piece_rows) * (dim + 1) * sizeof(float);
    return p;
}

int run_cached(const char *what, int dtype, Cached c, const Parts &parts, void *workspace, size_t workspace_bytes,
               cudaStream_t stream) {
    RODE_TRY(check_workspace(what, workspace, workspace_bytes, parts.bytes));
    c.chunk = parts.chunk;
    c.whole = parts.whole;
    c.ctas = parts.ctas;
    c.prefix_parts = parts.prefix;
    const size_t dim = c.win.dim;
    c.prefix_out = static_cast<float *>(workspace);
    c.own_out = c.prefix_out + parts.prefix_rows * dim;
    c.piece_out = c.own_out + parts.own_rows * dim;
    c.prefix_lse = c.piece_out + parts.piece_rows * dim;
    c.own_lse = c.prefix_lse + parts.prefix_rows;
    c.piece_lse = c.own_lse + parts.own_rows;
    const bool tensor_cores = step_takes(dtype, c);
    if (!tensor_cores && c.chunk != kSimpleChunk) {  // 16-bit operands that are not whole 16-byte units
        c.chunk = kSimpleChunk;
        if (c.whole) c.ctas = c.batch * c.win.kv_heads * ((c.win.heads / c.win.kv_heads + kSimpleChunk - 1) / kSimpleChunk);
    }
    if (parts.prefix > 0) RODE_TRY(tiles_take_shared(dtype, c) ? tiles_shared(dtype, c, stream) : simple_shared(dtype, c, stream));
    RODE_TRY(tensor_cores ? step_on_tensor_cores(dtype, c, stream) : simple_step(dtype, c, stream));
    if (parts.prefix > 0 || !parts.whole) RODE_TRY(join_parts(dtype, c, stream));
    return RODE_OK;
}

}  // namespace
}  // namespace rode

using namespace rode;

extern "C" {

int rode_window_attention(int dtype, int n_seq, const int *q_offsets, const int *k_offsets, int q_rows, int k_rows,
                          int heads, int kv_heads, int dim, int window, int sinks, float scale, int clear,
                          const rode_heads_t *q, const rode_heads_t *k, const rode_heads_t *v, void *out, void *out_rest,
                          float *lse, rode_stream_t stream) {
    const char *what = "rode_window_attention";
    RODE_TRY(check_shape(what, dtype, heads, kv_heads, dim, scale));
    RODE_TRY(check_window(what, window, sinks));
    RODE_TRY(check_packed(what, n_seq, q_offsets, k_offsets, q_rows, k_rows));
    RODE_TRY(check_operand(what, "q", q, dtype, q_rows > 0));
    RODE_TRY(check_operand(what, "k", k, dtype, q_rows > 0 && k_rows > 0));
    RODE_TRY(check_operand(what, "v", v, dtype, q_rows > 0 && k_rows > 0));
    RODE_TRY(check_result(what, "out", out, q_rows > 0));
    RODE_TRY(check_result(what, "out_rest", out_rest, out_rest != nullptr));
    if (q_rows == 0) return RODE_OK;
    Prompt p = {};
    p.seqs = {q_offsets, k_offsets, n_seq, q_rows, k_rows};
    p.win = window_of(window, sinks, heads, kv_heads, dim, scale);
    p.q = *q;
    if (k_rows > 0) {
        p.k = *k;
        p.v = *v;
    }
    p.out = out;
    p.rest = dtype == RODE_F32 ? nullptr : out_rest;
    p.lse = lse;
    p.clear = clear != 0;
    return tiles_take_prompt(dtype, p) ? tiles_prompt(dtype, p, stream) : simple_prompt(dtype, p, stream);
}

int rode_window_attention_backward_workspace_bytes(int dtype, int n_seq, int q_rows, int k_rows, int heads, int kv_heads, int dim,
                                                   int window, int sinks, size_t *bytes) {
    const char *what = "rode_window_attention_backward_workspace_bytes";
    if (bytes == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: null pointer bytes", what);
    RODE_TRY(check_shape(what, dtype, heads, kv_heads, dim, 1.f));
    RODE_TRY(check_window(what, window, sinks));
    if (q_rows < 0 || q_rows > kMaxRows || k_rows < 0 || k_rows > kMaxRows || n_seq < 0 || n_seq > kMaxRows)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: q_rows = %d, k_rows = %d and n_seq = %d must be 0 to 2^30", what, q_rows, k_rows,
                    n_seq);
    const FarPlan far = plan_far(n_seq, true, q_rows, kv_heads, dim, window, sinks);
    // (fp32 never runs on the kernels that cut far queries off, nor 16-bit types on those that want the heads apart)
    *bytes = delta_bytes(q_rows, heads) + (dtype == RODE_F32 ? simple_backward_bytes(dtype, n_seq, k_rows, heads, kv_heads, dim)
                                                            : far.near_bytes + far.far_bytes);
    return RODE_OK;
}

int rode_window_attention_backward(int dtype, int n_seq, const int *q_offsets, const int *k_offsets, int q_rows,
                                   int k_rows, int heads, int kv_heads, int dim, int window, int sinks, float scale,
                                   int clear, const rode_heads_t *q, const rode_heads_t *k, const rode_heads_t *v,
                                   const void *out, const void *out_rest, const float *lse, const rode_heads_t *dout,
                                   void *dq, void *dk, void *dv, void *workspace, size_t workspace_bytes,
                                   rode_stream_t stream) {
    const char *what = "rode_window_attention_backward";
    RODE_TRY(check_shape(what, dtype, heads, kv_heads, dim, scale));
    RODE_TRY(check_window(what, window, sinks));
    RODE_TRY(check_packed(what, n_seq, q_offsets, k_offsets, q_rows, k_rows));
    const bool both = q_rows > 0 && k_rows > 0, keys = dk != nullptr || dv != nullptr;
    RODE_TRY(check_operand(what, "q", q, dtype, q_rows > 0));
    RODE_TRY(check_operand(what, "k", k, dtype, both || (keys && k_rows > 0)));
    RODE_TRY(check_operand(what, "v", v, dtype, both || (keys && k_rows > 0)));
    RODE_TRY(check_operand(what, "dout", dout, dtype, q_rows > 0));
    RODE_TRY(check_result(what, "out", out, q_rows > 0));
    RODE_TRY(check_result(what, "out_rest", out_rest, out_rest != nullptr));
    RODE_TRY(check_result(what, "dq", dq, q_rows > 0));
    RODE_TRY(check_result(what, "dk", dk, keys && k_rows > 0));
    RODE_TRY(check_result(what, "dv", dv, keys && k_rows > 0));
    if (q_rows > 0 && lse == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: null pointer lse", what);
    size_t need = 0;
    RODE_TRY(rode_window_attention_backward_workspace_bytes(dtype, n_seq, q_rows, k_rows, heads, kv_heads, dim, window, sinks, &need));
    RODE_TRY(check_workspace(what, workspace, workspace_bytes, need));
    if (q_rows == 0 && (k_rows == 0 || !keys)) return RODE_OK;
    Prompt p = {};
    p.seqs = {q_offsets, k_offsets, n_seq, q_rows, k_rows};
    p.win = window_of(window, sinks, heads, kv_heads, dim, scale);
    if (q_rows > 0) {
        p.q = *q;
        p.dout = *dout;
    }
    if (k_rows > 0 && k != nullptr && v != nullptr) {
        p.k = *k;
        p.v = *v;
    }
    p.out = const_cast<void *>(out);
    p.rest = dtype == RODE_F32 ? nullptr : const_cast<void *>(out_rest);
    p.lse = const_cast<float *>(lse);
    p.dq = dq;
    p.dk = dk;
    p.dv = dv;
    p.delta = static_cast<float *>(workspace);
    p.clear = clear != 0;
    if (!tiles_take_backward(dtype, p)) {
        if (simple_backward_bytes(dtype, n_seq, k_rows, heads, kv_heads, dim) > 0 && keys)
            p.head_part = p.delta + delta_bytes(q_rows, heads) / sizeof(float);
        return simple_prompt_backward(dtype, p, stream);
    }
    const FarPlan far = plan_far(n_seq, q_offsets != nullptr, q_rows, kv_heads, dim, window, sinks);
    if (keys) {
        p.far_chunk = far.chunk;
        p.far_slots = far.slots;
        p.near_part = p.delta + delta_bytes(q_rows, heads) / sizeof(float);
        p.far_part = p.near_part + far.near_bytes / sizeof(float);
    }
    return tiles_backward(dtype, p, stream);
}

static int check_cached_sizes(const char *what, int batch, int heads, int prefix, int capacity) {
    if (batch < 0 || batch > kMaxRows || prefix < 0 || prefix > kMaxRows || capacity < 0 || capacity > kMaxRows)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: batch = %d, prefix = %d and capacity = %d must be 0 to 2^30", what, batch, prefix,
                    capacity);
    if (static_cast<long long>(batch) * heads > 2147483647ll)
        return fail(RODE_ERR_INVALID_ARGUMENT, "%s: batch * heads = %lld must be less than 2^31", what, static_cast<long long>(batch) * heads);
    return RODE_OK;
}

static long long seen_at_most(int capacity, int window, int sinks) {
    const long long seen = static_cast<long long>(window) + sinks;
    return seen < capacity ? seen : capacity;
}

int rode_window_attention_step_workspace_bytes(int dtype, int batch, int capacity, int heads, int kv_heads, int dim, int window,
                                               int sinks, size_t *bytes) {
    const char *what = "rode_window_attention_step_workspace_bytes";
    if (bytes == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: null pointer bytes", what);
    RODE_TRY(check_shape(what, dtype, heads, kv_heads, dim, 1.f));
    RODE_TRY(check_window(what, window, sinks));
    RODE_TRY(check_cached_sizes(what, batch, heads, 0, capacity));
    *bytes = plan_parts(dtype, batch, 0, seen_at_most(capacity, window, sinks), heads, kv_heads, dim).bytes;
    return RODE_OK;
}

int rode_window_attention_step(int dtype, int batch, int capacity, int heads, int kv_heads, int dim, int window,
                               int sinks, float scale, const rode_heads_t *q, const rode_heads_t *k_cache,
                               const rode_heads_t *v_cache, const int *lengths, void *out, void *workspace,
                               size_t workspace_bytes, rode_stream_t stream) {
    const char *what = "rode_window_attention_step";
    RODE_TRY(check_shape(what, dtype, heads, kv_heads, dim, scale));
    RODE_TRY(check_window(what, window, sinks));
    RODE_TRY(check_cached_sizes(what, batch, heads, 0, capacity));
    RODE_TRY(check_operand(what, "q", q, dtype, batch > 0));
    RODE_TRY(check_operand(what, "k_cache", k_cache, dtype, batch > 0 && capacity > 0));
    RODE_TRY(check_operand(what, "v_cache", v_cache, dtype, batch > 0 && capacity > 0));
    RODE_TRY(check_result(what, "out", out, batch > 0));
    if (batch > 0 && lengths == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: null pointer lengths", what);
    if (batch == 0) return RODE_OK;
    Cached c = {};
    c.batch = batch;
    c.capacity = capacity;
    c.win = window_of(window, sinks, heads, kv_heads, dim, scale);
    c.q = *q;
    if (capacity > 0) {
        c.k = *k_cache;
        c.v = *v_cache;
    }
    c.lengths = lengths;
    c.out = out;
    return run_cached(what, dtype, c, plan_parts(dtype, batch, 0, seen_at_most(capacity, window, sinks), heads, kv_heads, dim), workspace,
                      workspace_bytes, stream);
}

int rode_shared_prefix_attention_workspace_bytes(int dtype, int batch, int prefix, int capacity, int heads, int kv_heads, int dim,
                                                 size_t *bytes) {
    const char *what = "rode_shared_prefix_attention_workspace_bytes";
    if (bytes == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: null pointer bytes", what);
    RODE_TRY(check_shape(what, dtype, heads, kv_heads, dim, 1.f));
    RODE_TRY(check_cached_sizes(what, batch, heads, prefix, capacity));
    *bytes = plan_parts(dtype, batch, prefix, capacity, heads, kv_heads, dim).bytes;
    return RODE_OK;
}

int rode_shared_prefix_attention(int dtype, int batch, int prefix, int capacity, int heads, int kv_heads, int dim,
                                 float scale, const rode_heads_t *q, const rode_heads_t *prefix_k,
                                 const rode_heads_t *prefix_v, const rode_heads_t *k_cache, const rode_heads_t *v_cache,
                                 const int *lengths, void *out, void *workspace, size_t workspace_bytes,
                                 rode_stream_t stream) {
    const char *what = "rode_shared_prefix_attention";
    RODE_TRY(check_shape(what, dtype, heads, kv_heads, dim, scale));
    RODE_TRY(check_cached_sizes(what, batch, heads, prefix, capacity));
    RODE_TRY(check_operand(what, "q", q, dtype, batch > 0));
    RODE_TRY(check_operand(what, "prefix_k", prefix_k, dtype, batch > 0 && prefix > 0));
    RODE_TRY(check_operand(what, "prefix_v", prefix_v, dtype, batch > 0 && prefix > 0));
    RODE_TRY(check_operand(what, "k_cache", k_cache, dtype, batch > 0 && capacity > 0));
    RODE_TRY(check_operand(what, "v_cache", v_cache, dtype, batch > 0 && capacity > 0));
    RODE_TRY(check_result(what, "out", out, batch > 0));
    if (batch > 0 && lengths == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "%s: null pointer lengths", what);
    if (batch == 0) return RODE_OK;
    Cached c = {};
    c.batch = batch;
    c.capacity = capacity;
    c.prefix = prefix;
    // every row of the own cache up to the length
    c.win = window_of(kMaxRows, 0, heads, kv_heads, dim, scale);
    c.q = *q;
    if (prefix > 0) {
        c.pk = *prefix_k;
        c.pv = *prefix_v;
    }
    if (capacity > 0) {
        c.k = *k_cache;
        c.v = *v_cache;
    }
    c.lengths = lengths;
    c.out = out;
    return run_cached(what, dtype, c, plan_parts(dtype, batch, prefix, capacity, heads, kv_heads, dim), workspace, workspace_bytes, stream);
}

int rode_attention_waits_failed(int *failed) {
    if (failed == nullptr) return fail(RODE_ERR_INVALID_ARGUMENT, "rode_attention_waits_failed: null pointer failed");
    return tiles_waits_failed(failed);
}

}  // extern "C"
