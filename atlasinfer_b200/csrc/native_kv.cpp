// Host path of the operators between a decoder layer's linears: queries and keys, the 4-bit cache, attention over it.
//
// As in native.cpp: argument checks, allocations and the launch in one native call; the Python functions (kv_cache.py) say
// what the arguments are.  Wrong types raise TypeError, wrong shapes ValueError, shapes without a kernel NotImplementedError.
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

// fp16 or bf16 [tokens, heads, head_dim] on a GPU, in a layout that the kernels read (copied if it is not)
Tensor heads_tensor(const Tensor &t, const char *name, const Tensor *like = nullptr) {
    if (t.scalar_type() != at::kHalf && t.scalar_type() != at::kBFloat16)
        throw py::type_error(std::string(name) + " must be fp16 or bf16, got " + c10::toString(t.scalar_type()));
    if (t.dim() != 3) throw py::value_error(std::string(name) + " must be [tokens, heads, head_dim], got " + shape_of(t));
    if (!t.is_cuda()) throw py::value_error(std::string(name) + " must be on a CUDA device");
    if (like) {
        if (t.scalar_type() != like->scalar_type()) throw py::type_error(std::string(name) + " must have the dtype of the other tensors");
        if (t.device() != like->device()) throw py::value_error(std::string(name) + " must be on the device of the other tensors");
        if (t.size(0) != like->size(0) || t.size(2) != like->size(2))
            throw py::value_error(std::string(name) + " is " + shape_of(t) + ", which does not go with " + shape_of(*like));
    }
    const bool fits = (t.size(2) == 1 || t.stride(2) == 1) && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15);
    if (fits || t.numel() == 0) return t;
    return t.clone(at::MemoryFormat::Contiguous);   // (a contiguous view at an odd address is copied too)
}

Tensor index_tensor(const Tensor &t, const char *name, int64_t n, const c10::Device &device, bool only_int32 = false) {
    if (t.scalar_type() != at::kInt && (only_int32 || t.scalar_type() != at::kLong))
        throw py::type_error(std::string(name) + (only_int32 ? " must be int32" : " must be int32 or int64"));
    if (t.dim() != 1 || t.size(0) != n) throw py::value_error(std::string(name) + " must be [" + std::to_string(n) + "], got " + shape_of(t));
    if (t.device() != device) throw py::value_error(std::string(name) + " must be on the device of the other tensors");
    return t.contiguous();
}

Tensor weight_tensor(const Tensor &t, const char *name, const Tensor &x, bool &wide) {
    if (t.scalar_type() != at::kFloat && t.scalar_type() != x.scalar_type())
        throw py::type_error(std::string(name) + " must be fp32 or have the dtype of the queries and keys");
    if (t.dim() != 1 || t.size(0) != x.size(2)) throw py::value_error(std::string(name) + " must be [head_dim], got " + shape_of(t));
    if (t.device() != x.device()) throw py::value_error(std::string(name) + " must be on the device of the queries and keys");
    wide = t.scalar_type() == at::kFloat;
    return reinterpret_cast<uintptr_t>(t.data_ptr()) & 15 ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
}

void check_cache(const Tensor &data, const Tensor &like, int64_t kv_heads, int64_t head_dim, int64_t cache_dim) {
    if (data.device() != like.device()) throw py::value_error("the cache must be on the device of the other tensors");
    if (data.size(1) != kv_heads) throw py::value_error("the cache holds " + std::to_string(data.size(1)) + " heads, got " + std::to_string(kv_heads));
    if (head_dim != cache_dim) throw py::value_error("the cache holds heads of " + std::to_string(cache_dim) + ", got " + std::to_string(head_dim));
}

int dtype_code(const Tensor &t) { return t.scalar_type() == at::kHalf ? ATLAS_DTYPE_F16 : ATLAS_DTYPE_BF16; }
void *stream_of(const Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// (q', k'): norms and rotation; with a cache (data, its head_dim and page size, slots) keys and values go there and k' is absent.
std::pair<Maybe, Maybe> norm_rotate(const Maybe &q_in, const Tensor &k_in, const Maybe &v_in, const Maybe &table_in, const Maybe &positions_in,
                                    const Maybe &q_weight_in, const Maybe &k_weight_in, double eps, double weight_offset, bool interleaved,
                                    const Maybe &data, int64_t cache_dim, int64_t page_size, const Maybe &slots_in) {
    const Tensor k = heads_tensor(k_in, "k");
    const Tensor q = q_in ? heads_tensor(*q_in, "q", &k) : Tensor(), v = v_in ? heads_tensor(*v_in, "v", &k) : Tensor();
    const int64_t tokens = k.size(0);
    AtlasTokens a = {};
    a.dtype = dtype_code(k);
    a.kv_heads = (int32_t)k.size(1), a.head_dim = (int32_t)k.size(2), a.q_heads = q_in ? (int32_t)q.size(1) : 0;
    a.tokens = tokens;
    Tensor table, positions, qw, kw, slots;
    if (table_in) {
        if (!positions_in) throw py::value_error("a table needs positions");
        if (table_in->scalar_type() != at::kFloat) throw py::type_error("table must be fp32");
        if (table_in->dim() != 2 || table_in->size(0) < 1) throw py::value_error("table must be [positions, rotary_dim], got " + shape_of(*table_in));
        if (table_in->device() != k.device()) throw py::value_error("table must be on the device of the other tensors");
        table = reinterpret_cast<uintptr_t>(table_in->data_ptr()) & 15 ? table_in->clone(at::MemoryFormat::Contiguous) : table_in->contiguous();
        positions = index_tensor(*positions_in, "positions", tokens, k.device());
        a.table = table.const_data_ptr<float>(), a.table_rows = table.size(0);
        a.rotary_dim = (int32_t)std::min<int64_t>(table.size(1), INT32_MAX);
        a.positions = positions.numel() ? positions.data_ptr() : nullptr, a.position_bytes = (int32_t)positions.element_size();
    }
    bool q_wide = false, k_wide = false;
    if (q_weight_in && q_in) qw = weight_tensor(*q_weight_in, "q_weight", k, q_wide);
    if (k_weight_in) kw = weight_tensor(*k_weight_in, "k_weight", k, k_wide);
    if (qw.defined() && kw.defined() && q_wide != k_wide) throw py::type_error("q_weight and k_weight must have one dtype");
    a.weights_f32 = q_wide || k_wide;
    a.q_weight = qw.defined() ? qw.data_ptr() : nullptr, a.k_weight = kw.defined() ? kw.data_ptr() : nullptr;
    a.eps = (float)eps, a.weight_offset = (float)weight_offset, a.interleaved = interleaved;
    const c10::cuda::CUDAGuard guard(k.device());
    if (data) {
        if (v.size(1) != k.size(1)) throw py::value_error("v must have the heads of k, got " + shape_of(v));
        check_cache(*data, k, k.size(1), k.size(2), cache_dim);
        if (data->numel() == 0) throw py::value_error("the cache has no pages");
        slots = index_tensor(*slots_in, "slots", tokens, k.device());
        a.cache = data->data_ptr(), a.num_pages = data->size(0), a.page_size = (int32_t)page_size;
        a.slots = slots.numel() ? slots.data_ptr() : nullptr, a.slot_bytes = (int32_t)slots.element_size();
        a.v = v.data_ptr(), a.v_token_stride = v.stride(0), a.v_head_stride = v.stride(1);
    }
    Maybe q_out, k_out;
    if (q_in) {
        q_out = at::empty({tokens, q.size(1), q.size(2)}, q.options());
        a.q = q.data_ptr(), a.q_out = q_out->data_ptr(), a.q_token_stride = q.stride(0), a.q_head_stride = q.stride(1);
    }
    if (!data) {
        k_out = at::empty({tokens, k.size(1), k.size(2)}, k.options());
        a.k_out = k_out->data_ptr();
    }
    a.k = k.data_ptr(), a.k_token_stride = k.stride(0), a.k_head_stride = k.stride(1);
    if (tokens == 0) return {q_out, k_out};
    check_status_code(atlas_norm_rotate(&a, stream_of(k)), "atlas_norm_rotate");
    return {q_out, k_out};
}

std::pair<Tensor, Tensor> kv_load(const Tensor &data, int64_t head_dim, int64_t page_size, const Tensor &slots_in, bool bf16) {
    if (slots_in.dim() != 1) throw py::value_error("slots must be one-dimensional, got " + shape_of(slots_in));
    const Tensor slots = index_tensor(slots_in, "slots", slots_in.size(0), data.device());
    const c10::cuda::CUDAGuard guard(data.device());
    const auto options = data.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
    Tensor k = at::empty({slots.size(0), data.size(1), head_dim}, options), v = at::empty_like(k);
    check_status_code(atlas_kv_load(data.numel() ? data.data_ptr() : nullptr, data.size(0), (int)data.size(1), (int)head_dim, (int)page_size,
                                    slots.numel() ? slots.data_ptr() : nullptr, (int)slots.element_size(), slots.size(0),
                                    bf16 ? ATLAS_DTYPE_BF16 : ATLAS_DTYPE_F16, k.data_ptr(), v.data_ptr(), stream_of(data)), "atlas_kv_load");
    return {k, v};
}

Tensor kv_attention(const Tensor &q_in, const Tensor &data, int64_t head_dim, int64_t page_size, const Tensor &table_in, const Tensor &lengths_in,
                    const Maybe &starts_in, int64_t max_queries, int64_t window, int64_t sinks, double scale, const Tensor &status) {
    const Tensor q = heads_tensor(q_in, "q");
    check_cache(data, q, data.size(1), q.size(2), head_dim);
    if (q.size(1) == 0 || q.size(1) % data.size(1)) throw py::value_error("q has " + std::to_string(q.size(1)) + " heads, which is no multiple of the cache's " + std::to_string(data.size(1)));
    if (table_in.scalar_type() != at::kInt) throw py::type_error("page_table must be int32");
    if (table_in.dim() != 2) throw py::value_error("page_table must be [sequences, pages], got " + shape_of(table_in));
    if (table_in.device() != q.device()) throw py::value_error("page_table must be on the device of q");
    const int64_t batch = table_in.size(0), total = q.size(0);
    const Tensor table = table_in.size(1) <= 1 || table_in.stride(1) == 1 ? table_in : table_in.contiguous();
    const Tensor lengths = index_tensor(lengths_in, "lengths", batch, q.device(), true);
    Tensor starts;
    if (starts_in) {
        starts = index_tensor(*starts_in, "query_starts", batch + 1, q.device(), true);
        if (max_queries < 0) max_queries = total;
    } else {
        if (batch ? total % batch : total) throw py::value_error(std::to_string(total) + " queries of " + std::to_string(batch) + " sequences need query_starts");
        max_queries = batch ? total / batch : 0;
    }
    if (window < 0 || sinks < 0) throw py::value_error("window and sinks must not be negative");
    const c10::cuda::CUDAGuard guard(q.device());
    Tensor out = at::empty({total, q.size(1), q.size(2)}, q.options());
    if (out.numel() == 0) return out;
    AtlasKvAttention a = {};
    a.dtype = dtype_code(q);
    a.q_heads = (int32_t)q.size(1), a.kv_heads = (int32_t)data.size(1), a.head_dim = (int32_t)q.size(2);
    a.q = q.data_ptr(), a.q_token_stride = q.stride(0), a.q_head_stride = q.stride(1);
    a.out = out.data_ptr();
    a.total_queries = total, a.batch = batch, a.max_queries = std::min(max_queries, total);
    a.cache = data.numel() ? data.data_ptr() : nullptr, a.num_pages = data.size(0);
    a.page_size = (int32_t)page_size, a.window = (int32_t)std::min<int64_t>(window, INT32_MAX), a.sinks = (int32_t)std::min<int64_t>(sinks, INT32_MAX);
    a.scale = (float)scale;
    a.page_table = table.numel() ? table.const_data_ptr<int32_t>() : nullptr, a.table_stride = table.stride(0), a.max_pages = table.size(1);
    a.lengths = lengths.const_data_ptr<int32_t>(), a.query_starts = starts.defined() ? starts.const_data_ptr<int32_t>() : nullptr;
    a.workspace_bytes = atlas_kv_attention_workspace_bytes(&a);
    Tensor workspace = at::empty({(int64_t)a.workspace_bytes}, q.options().dtype(at::kByte));
    a.workspace = workspace.numel() ? workspace.data_ptr() : nullptr;
    a.status = (int32_t *)status.data_ptr();
    check_status_code(atlas_kv_attention(&a, stream_of(q)), "atlas_kv_attention");
    return out;
}

}  // namespace

void bind_kv(py::module_ &m) {
    m.def("norm_rotate", &norm_rotate, py::call_guard<py::gil_scoped_release>());
    m.def("kv_load", &kv_load, py::call_guard<py::gil_scoped_release>());
    m.def("kv_attention", &kv_attention, py::call_guard<py::gil_scoped_release>());
}
