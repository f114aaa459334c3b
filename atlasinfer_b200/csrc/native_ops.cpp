// Host path of the operators around a decoder step's linears: the norm with the residual sum, linears with an epilogue, log
// probabilities.  As in native_kv.cpp; the Python functions (decoder_ops.py) say what the arguments are.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "atlas_b200.h"

namespace py = pybind11;

void check_status_code(int status, const char *what);   // native.cpp

namespace {

using Tensor = at::Tensor;
using Maybe = std::optional<at::Tensor>;

std::string shape_of(const Tensor &t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}
void *stream_of(const Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
bool is_16(const Tensor &t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
int dtype_code(const Tensor &t) { return t.scalar_type() == at::kHalf ? ATLAS_DTYPE_F16 : t.scalar_type() == at::kBFloat16 ? ATLAS_DTYPE_BF16 : ATLAS_DTYPE_F32; }
const void *ptr_or_null(const Tensor &t) { return t.numel() ? t.data_ptr() : nullptr; }

// [..., n] as rows of n neighbouring numbers (copied if they are not)
Tensor rows_of(const Tensor &t, int64_t n) {
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, n});
    return r.size(1) > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}
int64_t row_stride(const Tensor &rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

void same_place(const Tensor &t, const Tensor &like, const char *name) {
    if (t.device() != like.device()) throw py::value_error(std::string(name) + " must be on the device of the other tensors");
}
// `t` in the type of x or in fp32; says which
bool wide(const Tensor &t, const Tensor &x, const char *name) {
    if (t.scalar_type() != at::kFloat && t.scalar_type() != x.scalar_type())
        throw py::type_error(std::string(name) + " must be fp32 or have the dtype of x, got " + c10::toString(t.scalar_type()));
    same_place(t, x, name);
    return t.scalar_type() == at::kFloat;
}

std::pair<Tensor, Tensor> residual_norm(const Tensor &x_in, const Maybe &residual_in, const Maybe &weight_in, const Maybe &bias_in, const Maybe &post_in,
                                        const Maybe &gate_in, double scale, double eps, double weight_offset, bool centered) {
    if (!is_16(x_in)) throw py::type_error(std::string("x must be fp16 or bf16, got ") + c10::toString(x_in.scalar_type()));
    if (x_in.dim() < 1 || x_in.size(-1) < 1) throw py::value_error("x must be [..., hidden], got " + shape_of(x_in));
    if (!x_in.is_cuda()) throw py::value_error("x must be on a CUDA device");
    const int64_t hidden = x_in.size(-1);
    AtlasResidualNorm a = {};
    Tensor residual, gate, weight, bias, post;
    const c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = x_in.numel() ? rows_of(x_in, hidden) : x_in.reshape({0, hidden});
    if (residual_in) {
        if (wide(*residual_in, x_in, "residual")) a.wide |= ATLAS_WIDE_STREAM;
        if (residual_in->sizes() != x_in.sizes()) throw py::value_error("residual must be " + shape_of(x_in) + ", got " + shape_of(*residual_in));
        if (x_in.numel()) residual = rows_of(*residual_in, hidden);
    }
    if (gate_in) {
        if (wide(*gate_in, x_in, "gate")) a.wide |= ATLAS_WIDE_GATE;
        const bool one = gate_in->dim() == 1 && gate_in->size(0) == hidden;
        if (!one && gate_in->sizes() != x_in.sizes()) throw py::value_error("gate must be [hidden] or " + shape_of(x_in) + ", got " + shape_of(*gate_in));
        if (x_in.numel()) {
            gate = one ? gate_in->contiguous() : rows_of(*gate_in, hidden);
            a.gate_stride = one ? 0 : row_stride(gate);
        }
    }
    auto vector = [&](const Maybe &t, const char *name, int bit) {
        if (!t) return Tensor();
        if (wide(*t, x_in, name)) a.wide |= bit;
        if (t->dim() != 1 || t->size(0) != hidden) throw py::value_error(std::string(name) + " must be [hidden], got " + shape_of(*t));
        return t->contiguous();
    };
    weight = vector(weight_in, "weight", ATLAS_WIDE_WEIGHT);
    bias = vector(bias_in, "bias", ATLAS_WIDE_BIAS);
    post = vector(post_in, "post_weight", ATLAS_WIDE_POST_WEIGHT);
    const bool as_it_is = !residual_in && !gate_in && !post_in && scale == 1.0;   // the stream is x
    Tensor normed = at::empty(x_in.sizes(), x_in.options());
    Tensor stream = as_it_is ? x_in : at::empty(x_in.sizes(), residual_in ? residual_in->options() : x_in.options());
    if (x_in.numel() == 0) return {normed, stream};
    a.dtype = dtype_code(x);
    a.centered = centered;
    a.scale = (float)scale, a.eps = (float)eps, a.weight_offset = (float)weight_offset;
    a.tokens = x.size(0), a.hidden = hidden;
    a.x = x.data_ptr(), a.x_stride = row_stride(x);
    if (residual.defined()) a.residual = residual.data_ptr(), a.residual_stride = row_stride(residual);
    if (gate.defined()) a.gate = gate.data_ptr();
    if (weight.defined()) a.weight = weight.data_ptr();
    if (bias.defined()) a.bias = bias.data_ptr();
    if (post.defined()) a.post_weight = post.data_ptr();
    a.normed = normed.data_ptr(), a.stream_out = as_it_is ? nullptr : stream.data_ptr();
    check_status_code(atlas_residual_norm(&a, stream_of(x)), "atlas_residual_norm");
    return {normed, stream};
}

// Linears launched plainly, where `on` (native.cpp).
class Plainly {
   public:
    explicit Plainly(bool on) : on_(on) { if (on_) was_ = atlas_qlinear_plain_launch(1); }
    ~Plainly() { if (on_) atlas_qlinear_plain_launch(was_); }
    Plainly(const Plainly &) = delete;

   private:
    bool on_;
    int was_ = 0;
};

// `weight`, `up`: tiles, scales, chunk pointers, entries, values of a kernel layout (`up` may be empty)
Tensor fused_linear(const Tensor &x_in, const std::vector<Tensor> &weight, const Maybe &bias, const std::vector<Tensor> &up, const Maybe &up_bias, int64_t n,
                    int64_t k, int64_t bs, const Maybe &residual_in, int64_t activation, double scale, const Tensor &status, bool pending) {
    if (!is_16(x_in)) throw py::type_error(std::string("x must be fp16 or bf16, got ") + c10::toString(x_in.scalar_type()));
    if (x_in.dim() < 1 || x_in.size(-1) != k)
        throw py::value_error("x is " + shape_of(x_in) + ", the weight expects " + std::to_string(k) + " features");
    std::vector<int64_t> shape(x_in.sizes().begin(), x_in.sizes().end());
    shape.back() = n;
    const c10::cuda::CUDAGuard guard(x_in.device());
    AtlasFusedLinear a = {};
    Tensor residual;
    if (residual_in) {
        if (residual_in->scalar_type() != x_in.scalar_type()) throw py::type_error(std::string("residual must have the dtype of x, got ") + c10::toString(residual_in->scalar_type()));
        same_place(*residual_in, x_in, "residual");
        if (residual_in->sizes() != at::IntArrayRef(shape)) throw py::value_error("residual must have the shape of the result, got " + shape_of(*residual_in));
    }
    Tensor y = at::empty(shape, x_in.options());
    if (y.numel() == 0) return y;
    Tensor x = rows_of(x_in, k);
    if (x.size(0) > 1 && x.stride(0) < k) x = x.contiguous();
    if (residual_in) {
        residual = rows_of(*residual_in, n);
        if (residual.size(0) > 1 && residual.stride(0) < n) residual = residual.contiguous();
        a.residual = residual.data_ptr(), a.ldr = row_stride(residual);
    }
    bool converted = false;
    std::vector<Tensor> held;
    auto put = [&](AtlasWeight &w, const std::vector<Tensor> &buffers, const Maybe &b) {
        w.tiles = (const uint8_t *)buffers[0].data_ptr(), w.scales_tiled = buffers[1].data_ptr(), w.outlier_chunk_ptr = (const int32_t *)buffers[2].data_ptr();
        w.outlier_entries = (const uint32_t *)ptr_or_null(buffers[3]), w.outlier_vals_sorted = ptr_or_null(buffers[4]);
        if (!b) return;
        held.push_back(b->to(at::kHalf).contiguous());
        converted |= !held.back().is_same(*b);
        w.bias = held.back().data_ptr();
    };
    put(a.weight, weight, bias);
    if (!up.empty()) put(a.up, up, up_bias);
    a.dtype = dtype_code(x), a.activation = (int32_t)activation;
    a.x = x.data_ptr(), a.m = x.size(0), a.ldx = row_stride(x), a.n_rows = n, a.n_cols = k, a.block_size = (int32_t)bs;
    a.scale = (float)scale;
    a.y = y.data_ptr(), a.ldy = n;
    a.workspace_bytes = atlas_fused_linear_workspace_bytes(&a);
    const Tensor workspace = at::empty({(int64_t)a.workspace_bytes}, x.options().dtype(at::kByte));
    a.workspace = workspace.numel() ? workspace.data_ptr() : nullptr;
    a.status = (int32_t *)status.data_ptr();
    const Plainly plain(pending || converted);   // (a bias converted just now is written by the kernel in front)
    check_status_code(atlas_fused_linear(&a, stream_of(x)), "atlas_fused_linear");
    return y;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor &logits_in, const Tensor &tokens_in, int64_t top, double temperature) {
    if (!is_16(logits_in) && logits_in.scalar_type() != at::kFloat)
        throw py::type_error(std::string("logits must be fp16, bf16 or fp32, got ") + c10::toString(logits_in.scalar_type()));
    if (logits_in.dim() < 1 || logits_in.size(-1) < 1) throw py::value_error("logits must be [..., vocabulary], got " + shape_of(logits_in));
    if (!logits_in.is_cuda()) throw py::value_error("logits must be on a CUDA device");
    if (tokens_in.scalar_type() != at::kInt && tokens_in.scalar_type() != at::kLong) throw py::type_error("tokens must be int32 or int64");
    const int64_t vocab = logits_in.size(-1);
    if (tokens_in.sizes() != logits_in.sizes().slice(0, logits_in.dim() - 1))
        throw py::value_error("tokens must have the shape of the logits' rows, got " + shape_of(tokens_in) + " for " + shape_of(logits_in));
    same_place(tokens_in, logits_in, "tokens");
    if (top < 0 || top > vocab) throw py::value_error("top " + std::to_string(top) + " of " + std::to_string(vocab));
    const c10::cuda::CUDAGuard guard(logits_in.device());
    const auto wide_options = logits_in.options().dtype(at::kFloat);
    std::vector<int64_t> shape(tokens_in.sizes().begin(), tokens_in.sizes().end());
    Tensor logprobs = at::empty(shape, wide_options), entropy = at::empty(shape, wide_options);
    shape.push_back(top);
    Tensor top_tokens = at::empty(shape, wide_options.dtype(at::kLong)), top_logprobs = at::empty(shape, wide_options);
    AtlasTokenLogprobs a = {};
    a.temperature = (float)temperature;
    a.dtype = dtype_code(logits_in), a.top = (int32_t)std::min<int64_t>(top, INT32_MAX), a.token_bytes = (int32_t)tokens_in.element_size();
    a.rows = tokens_in.numel(), a.vocab = vocab;
    Tensor logits, tokens;
    if (a.rows) {
        logits = rows_of(logits_in, vocab), tokens = tokens_in.contiguous();
        a.logits_stride = row_stride(logits), a.logits = logits.data_ptr(), a.tokens = tokens.data_ptr();
        a.logprobs = logprobs.data_ptr<float>(), a.entropy = entropy.data_ptr<float>();
        if (top) a.top_tokens = top_tokens.data_ptr<int64_t>(), a.top_logprobs = top_logprobs.data_ptr<float>();
    }
    check_status_code(atlas_token_logprobs(&a, stream_of(logits_in)), "atlas_token_logprobs");
    return {logprobs, entropy, top_tokens, top_logprobs};
}

}  // namespace

void bind_ops(py::module_ &m) {
    m.def("residual_norm", &residual_norm, py::call_guard<py::gil_scoped_release>());
    m.def("fused_linear", &fused_linear, py::call_guard<py::gil_scoped_release>());
    m.def("token_logprobs", &token_logprobs, py::call_guard<py::gil_scoped_release>());
}
