// Torch binding of the attention operators, part of the module rode_sddmm_cuda: checks of tensors, outputs and workspaces from the
// caching allocator, launches on torch's current stream of the operands' device.  No kernels.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <tuple>

#include "rode_b200.h"

namespace {

using torch::Tensor;
using OptionalTensor = c10::optional<Tensor>;

Tensor empty_on(at::IntArrayRef sizes, at::ScalarType dtype, const c10::Device &device) {
    return at::detail::empty_cuda(sizes, dtype, device, c10::nullopt);
}

void check_status(int status) {
    if (status == RODE_OK) return;
    TORCH_CHECK_VALUE(status != RODE_ERR_INVALID_ARGUMENT, "rode_b200: ", rode_last_error());
    TORCH_CHECK(false, "rode_b200: ", rode_last_error());
}

int dtype_of(const Tensor &q) {
    const auto t = q.scalar_type();
    TORCH_CHECK_TYPE(t == torch::kFloat32 || t == torch::kFloat16 || t == torch::kBFloat16,
                     "q must be float32, float16 or bfloat16, got ", t);
    return t == torch::kFloat32 ? RODE_F32 : t == torch::kFloat16 ? RODE_F16 : RODE_BF16;
}

int to_int(int64_t x, const char *name) {
    TORCH_CHECK_VALUE(x >= 0 && x <= (1 << 30), name, " must be 0 to 2^30, got ", x);
    return static_cast<int>(x);
}

// A window larger than any sequence is no window.
int window_of(int64_t window) {
    TORCH_CHECK_VALUE(window >= 1, "window must be at least 1, got ", window);
    return static_cast<int>(std::min<int64_t>(window, 1 << 30));
}
int sinks_of(int64_t sinks) {
    TORCH_CHECK_VALUE(sinks >= 0, "sinks must not be negative, got ", sinks);
    return static_cast<int>(std::min<int64_t>(sinks, 1 << 30));
}

void check_like(const Tensor &x, const char *name, const Tensor &q, int64_t dim) {
    TORCH_CHECK_VALUE(x.dim() == dim, name, " must have ", dim, " dimensions, got ", x.dim());
    TORCH_CHECK_TYPE(x.scalar_type() == q.scalar_type(), name, " must be ", q.scalar_type(), " like q, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.device() == q.device(), name, " must be on ", q.device(), " like q, got ", x.device());
}

void check_ints(const Tensor &x, const char *name, const Tensor &q) {
    TORCH_CHECK_TYPE(x.scalar_type() == torch::kInt32, name, " must be int32, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() == 1 && x.is_contiguous(), name, " must be contiguous and have one dimension");
    TORCH_CHECK_VALUE(x.device() == q.device(), name, " must be on ", q.device(), " like q, got ", x.device());
}

// Base and strides as the kernels want them: of `elements` each, no dimension repeated by a stride of 0 or walked backwards.
bool fits(const Tensor &x, int64_t elements) {
    const int64_t last = x.dim() - 1;
    if (x.size(last) > 1 && x.stride(last) != 1) return false;
    if (reinterpret_cast<uintptr_t>(x.data_ptr()) % (elements * x.element_size()) != 0) return false;
    for (int64_t i = 0; i < last; ++i)
        if (x.size(i) > 1 && (x.stride(i) <= 0 || x.stride(i) % elements != 0)) return false;
    return true;
}
// The tensor itself where the tensor cores can take it as it lies (16-byte units; smaller ones where its rows have no more), else
// a contiguous copy.
Tensor fitting(const Tensor &x) {
    int64_t elements = 16 / x.element_size();
    if (x.size(x.dim() - 1) % elements != 0) elements = 4;
    if (x.numel() == 0 || fits(x, elements)) return x;
    const Tensor copy = x.clone(at::MemoryFormat::Contiguous);
    return copy;
}

// Strides of dimensions of one element say nothing: 0, which any kernel can take.
long long stride_of(const Tensor &x, int64_t i) { return x.size(i) > 1 ? x.stride(i) : 0; }

rode_heads_t rows_heads(const Tensor &x) { return {x.data_ptr(), 0, stride_of(x, 0), stride_of(x, 1)}; }
rode_heads_t batch_heads(const Tensor &x) { return {x.data_ptr(), stride_of(x, 0), 0, stride_of(x, 1)}; }
rode_heads_t batch_rows_heads(const Tensor &x) {
    return {x.data_ptr(), stride_of(x, 0), stride_of(x, 1), stride_of(x, 2)};
}

struct Sequences {
    int n = 1;
    const int *q = nullptr, *k = nullptr;
};

Sequences sequences(const Tensor &q, const Tensor &k, const OptionalTensor &q_offsets, const OptionalTensor &k_offsets) {
    Sequences s;
    if (!q_offsets.has_value()) {
        TORCH_CHECK_VALUE(!k_offsets.has_value(), "k_offsets without q_offsets");
        return s;
    }
    check_ints(*q_offsets, "q_offsets", q);
    TORCH_CHECK_VALUE(q_offsets->numel() >= 1, "q_offsets must have one entry more than there are sequences");
    s.n = to_int(q_offsets->numel() - 1, "sequences");
    s.q = s.k = q_offsets->data_ptr<int>();
    if (k_offsets.has_value()) {
        check_ints(*k_offsets, "k_offsets", q);
        TORCH_CHECK_VALUE(k_offsets->numel() == q_offsets->numel(), "k_offsets must have as many entries as q_offsets, got ",
                          k_offsets->numel(), " and ", q_offsets->numel());
        s.k = k_offsets->data_ptr<int>();
    } else {
        TORCH_CHECK_VALUE(k.size(0) == q.size(0), "without k_offsets, k must have as many rows as q, got ", k.size(0), " and ",
                          q.size(0));
    }
    return s;
}

void check_prompt(const Tensor &q, const Tensor &k, const Tensor &v) {
    TORCH_CHECK_VALUE(q.is_cuda(), "q must be on a CUDA device; rode_b200 has no CPU path");
    check_like(q, "q", q, 3);
    check_like(k, "k", q, 3);
    check_like(v, "v", q, 3);
    TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "k and v must have one shape, got ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK_VALUE(k.size(2) == q.size(2), "k must have the head dimension of q, got ", k.size(2), " and ", q.size(2));
}

// With want_lse (for the backward call): the result, what rounding took from it (16-bit types), the logarithms of the sums.
std::tuple<Tensor, Tensor, Tensor> window_forward(const Tensor &q_in, const Tensor &k_in, const Tensor &v_in, int64_t window,
                                                      int64_t sinks, const OptionalTensor &q_offsets,
                                                      const OptionalTensor &k_offsets, double scale, bool want_lse) {
    check_prompt(q_in, k_in, v_in);
    const int dtype = dtype_of(q_in);
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Sequences s = sequences(q_in, k_in, q_offsets, k_offsets);
    const Tensor q = fitting(q_in), k = fitting(k_in), v = fitting(v_in);
    const int rows = to_int(q.size(0), "rows of q"), heads = to_int(q.size(1), "heads"), dim = to_int(q.size(2), "dim");
    Tensor out = empty_on(q.sizes(), q.scalar_type(), q.device());
    Tensor lse, rest;
    if (want_lse && dtype != RODE_F32) rest = empty_on(q.sizes(), q.scalar_type(), q.device());
    if (want_lse) lse = empty_on({heads, rows}, torch::kFloat32, q.device());
    const rode_heads_t qh = rows_heads(q), kh = rows_heads(k), vh = rows_heads(v);
    check_status(rode_window_attention(dtype, s.n, s.q, s.k, rows, to_int(k.size(0), "rows of k"), heads,
                                       to_int(k.size(1), "key heads"), dim, window_of(window), sinks_of(sinks),
                                       static_cast<float>(scale), 1, &qh, &kh, &vh, out.data_ptr(),
                                       rest.defined() ? rest.data_ptr() : nullptr, want_lse ? lse.data_ptr<float>() : nullptr,
                                       at::cuda::getCurrentCUDAStream(q.device().index()).stream()));
    return {out, rest, lse};
}

// out, rest and lse are window_forward's.
std::tuple<Tensor, Tensor, Tensor> window_backward(const Tensor &q_in, const Tensor &k_in, const Tensor &v_in, const Tensor &out,
                                                    const Tensor &rest, const Tensor &lse, const Tensor &dout_in, int64_t window, int64_t sinks,
                                                    const OptionalTensor &q_offsets, const OptionalTensor &k_offsets, double scale,
                                                    bool want_keys) {
    const int dtype = dtype_of(q_in);
    check_like(dout_in, "the gradient of the result", q_in, 3);
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Sequences s = sequences(q_in, k_in, q_offsets, k_offsets);
    const Tensor q = fitting(q_in), k = fitting(k_in), v = fitting(v_in), dout = fitting(dout_in);
    const int rows = to_int(q.size(0), "rows of q"), heads = to_int(q.size(1), "heads"), dim = to_int(q.size(2), "dim");
    Tensor dq = empty_on(q.sizes(), q.scalar_type(), q.device());
    Tensor dk, dv;
    if (want_keys) {
        dk = empty_on(k.sizes(), q.scalar_type(), q.device());
        dv = empty_on(k.sizes(), q.scalar_type(), q.device());
    }
    size_t bytes = 0;
    check_status(rode_window_attention_backward_workspace_bytes(dtype, s.n, rows, to_int(k.size(0), "rows of k"), heads,
                                                                to_int(k.size(1), "key heads"), dim, window_of(window), sinks_of(sinks),
                                                                &bytes));
    Tensor ws = empty_on({static_cast<int64_t>(bytes)}, torch::kUInt8, q.device());
    const rode_heads_t qh = rows_heads(q), kh = rows_heads(k), vh = rows_heads(v), gh = rows_heads(dout);
    check_status(rode_window_attention_backward(
        dtype, s.n, s.q, s.k, rows, to_int(k.size(0), "rows of k"), heads, to_int(k.size(1), "key heads"), dim, window_of(window),
        sinks_of(sinks), static_cast<float>(scale), 1, &qh, &kh, &vh, out.data_ptr(), rest.defined() ? rest.data_ptr() : nullptr,
        lse.data_ptr<float>(), &gh, dq.data_ptr(),
        want_keys ? dk.data_ptr() : nullptr, want_keys ? dv.data_ptr() : nullptr, ws.data_ptr(), bytes,
        at::cuda::getCurrentCUDAStream(q.device().index()).stream()));
    return {dq, dk, dv};
}

OptionalTensor given(const Tensor &x) { return x.defined() ? OptionalTensor(x) : OptionalTensor(); }

// (In C++: a training step of a few thousand tokens is bound by the host, and the same in Python took 100 us of it.)
struct WindowAttention : torch::autograd::Function<WindowAttention> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, int64_t window,
                          int64_t sinks, const OptionalTensor &q_offsets, const OptionalTensor &k_offsets, double scale) {
        auto [out, rest, lse] = window_forward(q, k, v, window, sinks, q_offsets, k_offsets, scale, true);
        ctx->save_for_backward({q, k, v, out, rest, lse, q_offsets.value_or(Tensor()), k_offsets.value_or(Tensor())});
        ctx->saved_data["window"] = window;
        ctx->saved_data["sinks"] = sinks;
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list dout) {
        const auto saved = ctx->get_saved_variables();
        torch::autograd::variable_list grads(8);
        const bool twice = torch::GradMode::is_enabled();
        {
            const torch::NoGradGuard guard;
            std::tie(grads[0], grads[1], grads[2]) =
                window_backward(saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], dout[0], ctx->saved_data["window"].toInt(),
                                ctx->saved_data["sinks"].toInt(), given(saved[6]), given(saved[7]), ctx->saved_data["scale"].toDouble(),
                                ctx->needs_input_grad(1) || ctx->needs_input_grad(2));
        }
        if (twice) {  // the gradients themselves have none: an error when somebody asks for it
            torch::autograd::variable_list some;
            for (int i = 0; i < 3; ++i)
                if (grads[i].defined()) some.push_back(grads[i].detach().set_requires_grad(true));
            auto error = std::make_shared<torch::autograd::DelayedError>("rode_window_attention can be differentiated once only",
                                                                         static_cast<int64_t>(some.size()));
            some = (*error)(std::move(some));
            for (size_t i = 0, n = 0; i < 3; ++i)
                if (grads[i].defined()) grads[i] = some[n++];
        }
        return grads;
    }
};

// Derivatives that an operator does not have are refused: a result that silently has none would train on nothing.
void refuse_tangents(const char *what, std::initializer_list<const Tensor *> operands) {
    for (const Tensor *x : operands)
        TORCH_CHECK_NOT_IMPLEMENTED(!x->_fw_grad(/*level=*/0).defined(), what, " has no derivative in forward mode");
}
void refuse_gradients(const char *what, std::initializer_list<const Tensor *> operands) {
    refuse_tangents(what, operands);
    if (!torch::GradMode::is_enabled()) return;
    for (const Tensor *x : operands)
        TORCH_CHECK_NOT_IMPLEMENTED(!x->requires_grad(), what, " is not differentiable and an operand requires gradients; call it under torch.no_grad()");
}

Tensor py_window_attention(const Tensor &q, const Tensor &k, const Tensor &v, int64_t window, int64_t sinks,
                           const OptionalTensor &q_offsets, const OptionalTensor &k_offsets, double scale) {
    refuse_tangents("rode_window_attention", {&q, &k, &v});
    if (torch::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
        return WindowAttention::apply(q, k, v, window, sinks, q_offsets, k_offsets, scale);
    return std::get<0>(window_forward(q, k, v, window, sinks, q_offsets, k_offsets, scale, false));
}

// Caches are read where they lie: a copy would cost more than the call.
void check_cache(const Tensor &x, const char *name, const Tensor &q, int64_t dim) {
    check_like(x, name, q, dim);
    TORCH_CHECK_VALUE(x.size(dim - 1) == q.size(2), name, " must have the head dimension of q, got ", x.size(dim - 1), " and ",
                      q.size(2));
    TORCH_CHECK_VALUE(x.numel() == 0 || fits(x, 4), name,
                      " must lie with its last dimension contiguous, and its base and other strides multiples of 4 elements");
}

struct Caches {
    rode_heads_t q, k, v;
    int dtype, batch, capacity, heads, kv_heads, dim;
};

Caches check_caches(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &lengths) {
    TORCH_CHECK_VALUE(q.is_cuda(), "q must be on a CUDA device; rode_b200 has no CPU path");
    check_like(q, "q", q, 3);
    Caches c;
    c.dtype = dtype_of(q);
    check_cache(k_cache, "k_cache", q, 4);
    check_cache(v_cache, "v_cache", q, 4);
    check_ints(lengths, "lengths", q);
    TORCH_CHECK_VALUE(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have one shape, got ", k_cache.sizes(), " and ",
                      v_cache.sizes());
    TORCH_CHECK_VALUE(k_cache.size(0) == q.size(0) && lengths.size(0) == q.size(0),
                      "q, the caches and lengths must have one batch size, got ", q.size(0), ", ", k_cache.size(0), " and ",
                      lengths.size(0));
    c.batch = to_int(q.size(0), "batch");
    c.capacity = to_int(k_cache.size(1), "capacity");
    c.heads = to_int(q.size(1), "heads");
    c.kv_heads = to_int(k_cache.size(2), "key heads");
    c.dim = to_int(q.size(2), "dim");
    c.k = batch_rows_heads(k_cache);
    c.v = batch_rows_heads(v_cache);
    return c;
}

Tensor py_window_step(const Tensor &q_in, const Tensor &k_cache, const Tensor &v_cache, const Tensor &lengths, int64_t window,
                      int64_t sinks, double scale) {
    refuse_gradients("rode_window_attention_step", {&q_in, &k_cache, &v_cache});
    const Caches c = check_caches(q_in, k_cache, v_cache, lengths);
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Tensor q = fitting(q_in);
    Tensor out = empty_on(q.sizes(), q.scalar_type(), q.device());
    size_t bytes = 0;
    check_status(rode_window_attention_step_workspace_bytes(c.dtype, c.batch, c.capacity, c.heads, c.kv_heads, c.dim, window_of(window),
                                                            sinks_of(sinks), &bytes));
    Tensor ws;
    if (bytes > 0) ws = empty_on({static_cast<int64_t>(bytes)}, torch::kUInt8, q.device());
    const rode_heads_t qh = batch_heads(q);
    check_status(rode_window_attention_step(c.dtype, c.batch, c.capacity, c.heads, c.kv_heads, c.dim, window_of(window),
                                            sinks_of(sinks), static_cast<float>(scale), &qh, &c.k, &c.v, lengths.data_ptr<int>(),
                                            out.data_ptr(), bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                                            at::cuda::getCurrentCUDAStream(q.device().index()).stream()));
    return out;
}

Tensor py_shared_prefix(const Tensor &q_in, const Tensor &prefix_k, const Tensor &prefix_v, const Tensor &k_cache,
                        const Tensor &v_cache, const Tensor &lengths, double scale) {
    refuse_gradients("rode_shared_prefix_attention", {&q_in, &prefix_k, &prefix_v, &k_cache, &v_cache});
    const Caches c = check_caches(q_in, k_cache, v_cache, lengths);
    check_cache(prefix_k, "prefix_k", q_in, 3);
    check_cache(prefix_v, "prefix_v", q_in, 3);
    TORCH_CHECK_VALUE(prefix_k.sizes() == prefix_v.sizes(), "prefix_k and prefix_v must have one shape, got ", prefix_k.sizes(),
                      " and ", prefix_v.sizes());
    TORCH_CHECK_VALUE(prefix_k.size(1) == c.kv_heads, "the prefix must have the caches' heads, got ", prefix_k.size(1), " and ",
                      c.kv_heads);
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Tensor q = fitting(q_in);
    const int prefix = to_int(prefix_k.size(0), "prefix");
    Tensor out = empty_on(q.sizes(), q.scalar_type(), q.device());
    size_t bytes = 0;
    check_status(rode_shared_prefix_attention_workspace_bytes(c.dtype, c.batch, prefix, c.capacity, c.heads, c.kv_heads, c.dim, &bytes));
    Tensor ws;
    if (bytes > 0) ws = empty_on({static_cast<int64_t>(bytes)}, torch::kUInt8, q.device());
    const rode_heads_t qh = batch_heads(q), pk = rows_heads(prefix_k), pv = rows_heads(prefix_v);
    check_status(rode_shared_prefix_attention(c.dtype, c.batch, prefix, c.capacity, c.heads, c.kv_heads, c.dim,
                                              static_cast<float>(scale), &qh, &pk, &pv, &c.k, &c.v, lengths.data_ptr<int>(),
                                              out.data_ptr(), bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                                              at::cuda::getCurrentCUDAStream(q.device().index()).stream()));
    return out;
}

bool py_waits_failed(int64_t device) {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    int failed = 0;
    check_status(rode_attention_waits_failed(&failed));
    return failed != 0;
}

}  // namespace

void bind_attention(pybind11::module_ &m) {
    namespace py = pybind11;
    m.def("window_attention", &py_window_attention, "Window-and-sinks attention over packed sequences, differentiable (CUDA)",
          py::arg("q"), py::arg("k"), py::arg("v"), py::arg("window"), py::arg("sinks"), py::arg("q_offsets"), py::arg("k_offsets"),
          py::arg("scale"));
    m.def("window_attention_step", &py_window_step, "Window-and-sinks attention of one token per sequence (CUDA)", py::arg("q"),
          py::arg("k_cache"), py::arg("v_cache"), py::arg("lengths"), py::arg("window"), py::arg("sinks"), py::arg("scale"));
    m.def("shared_prefix_attention", &py_shared_prefix, "Attention of one token per request behind a shared prefix (CUDA)",
          py::arg("q"), py::arg("prefix_k"), py::arg("prefix_v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("lengths"),
          py::arg("scale"));
    m.def("attention_waits_failed", &py_waits_failed, "Whether a kernel on the device gave up a wait (synchronises)", py::arg("device"),
          py::call_guard<py::gil_scoped_release>());
}
