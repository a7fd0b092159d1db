// torch_calls.cpp -- the attention side's entry points for torch tensors.
//
// A decoding step makes these calls for every layer, with two or three
// microseconds of GPU work in each; through ctypes the call itself took ten.
// The functions here check what the C ABI cannot see of a tensor (its shape, its
// device), allocate the outputs on the current stream, and call the C entries,
// whose addresses the Python package hands over (bind), so that there is one
// library and one set of kernels.  Refusals are raised as the package's FmError.
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>

#include "freemoe_b200.h"

namespace py = pybind11;
using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

namespace {

struct Entries {
    decltype(&fmcuda_last_error) last_error;
    decltype(&fmcuda_add_rms_norm) norm;
    decltype(&fmcuda_rope_append) rope;
    decltype(&fmcuda_paged_attention_workspace_bytes) attention_bytes;
    decltype(&fmcuda_paged_attention) attention;
} entries{};
PyObject *error_class = nullptr; // FmError(code, message)

[[noreturn]] void refuse(int code, const std::string &message) {
    py::object error = py::reinterpret_borrow<py::object>(error_class)(code, message);
    PyErr_SetObject(error_class, error.ptr());
    throw py::error_already_set();
}

void check(int rc) {
    if (rc) refuse(rc, entries.last_error());
}

void need(bool ok, const char *message, int code = FM_STATUS_SHAPE_MISMATCH) {
    if (!ok) refuse(code, message);
}

int32_t dtype_of(const Tensor &t) {
    switch (t.scalar_type()) {
    case at::kFloat: return FM_X_F32;
    case at::kBFloat16: return FM_X_BF16;
    case at::kHalf: return FM_X_F16;
    default: return -1; // refused by the C entry
    }
}

// The device of the call: the current one, where every tensor has to be.
struct Here {
    c10::DeviceIndex device;
    explicit Here(const Tensor &first) {
        need(first.is_cuda(), "a tensor is not on a CUDA device", FM_STATUS_INVALID_ARGUMENT);
        device = c10::cuda::current_device();
        (*this)(first);
    }
    void operator()(const Tensor &t) const {
        if (!t.is_cuda() || t.device().index() != device)
            refuse(FM_STATUS_INVALID_ARGUMENT, "a tensor is not on the current device, cuda:" + std::to_string(device));
    }
    void operator()(const MaybeTensor &t) const {
        if (t) (*this)(*t);
    }
    void *stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
};

void *at_of(const MaybeTensor &t) { return t ? t->data_ptr() : nullptr; }

bool dense(const Tensor &t) { return t.size(-1) == 1 || t.stride(-1) == 1; }

Tensor run_norm(const Tensor &x, const Tensor &weight, const MaybeTensor &residual, double epsilon, const Tensor &y,
                int32_t y_dtype, float *scales, const Here &here) {
    here(weight), here(residual);
    need(weight.dim() == 1 && weight.size(0) == x.size(1) && (!residual || residual->sizes() == x.sizes()),
         "norm takes [tokens, d_model], a weight of d_model and a residual like x");
    need(dense(x) && dense(weight) && (!residual || dense(*residual)), "norm inputs must be contiguous in their rows");
    Tensor h;
    fmcuda_rms_norm_args a{};
    if (residual) {
        // like the residual in memory too: the C entry takes one stride for both
        h = at::empty_strided(residual->sizes(), residual->strides(), residual->options());
        a.residual = residual->data_ptr();
        a.residual_out = h.data_ptr();
        a.residual_stride = residual->stride(0);
        a.residual_dtype = dtype_of(*residual);
    }
    a.x = x.data_ptr();
    a.weight = weight.data_ptr();
    a.y = y.data_ptr();
    a.scales = scales;
    a.x_stride = x.stride(0);
    a.y_stride = y.stride(0);
    a.x_dtype = dtype_of(x);
    a.weight_dtype = dtype_of(weight);
    a.y_dtype = y_dtype;
    a.tokens = static_cast<uint32_t>(x.size(0));
    a.d_model = static_cast<uint32_t>(x.size(1));
    a.epsilon = static_cast<float>(epsilon);
    check(entries.norm(&a, here.stream()));
    return h;
}

void need_rows(const Tensor &x) {
    need(x.dim() == 2 && x.size(0) <= UINT32_MAX && x.size(1) <= UINT32_MAX, "norm takes [tokens, d_model]");
}

std::tuple<Tensor, MaybeTensor> add_rms_norm(const Tensor &x, const Tensor &weight, const MaybeTensor &residual,
                                             double epsilon, std::optional<at::ScalarType> out_dtype) {
    need_rows(x);
    const Here here(x);
    const Tensor y = at::empty(x.sizes(), x.options().dtype(out_dtype.value_or(x.scalar_type())));
    const Tensor h = run_norm(x, weight, residual, epsilon, y, dtype_of(y), nullptr, here);
    return {y, residual ? MaybeTensor(h) : std::nullopt};
}

std::tuple<Tensor, Tensor, MaybeTensor> add_rms_norm_fp8(const Tensor &x, const Tensor &weight,
                                                         const MaybeTensor &residual, double epsilon) {
    need_rows(x);
    const Here here(x);
    const Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    const Tensor scales = at::empty({x.size(0), (x.size(1) + 127) / 128}, x.options().dtype(at::kFloat));
    const Tensor h =
        run_norm(x, weight, residual, epsilon, codes, FM_X_E4M3, static_cast<float *>(scales.data_ptr()), here);
    return {codes, scales, residual ? MaybeTensor(h) : std::nullopt};
}

Tensor rope_append(const Tensor &q, const MaybeTensor &k, const MaybeTensor &v, const Tensor &positions,
                   const Tensor &inv_freq, const MaybeTensor &k_cache, const MaybeTensor &v_cache,
                   const MaybeTensor &slots, bool interleaved, double attention_factor,
                   std::optional<at::ScalarType> out_dtype) {
    need(q.dim() == 3, "q is [tokens, heads, head_dim]");
    const Here here(q);
    here(k), here(v), here(positions), here(inv_freq), here(k_cache), here(v_cache), here(slots);
    const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
    need(tokens <= INT32_MAX && heads <= INT32_MAX && dim <= INT32_MAX, "too many tokens in a call");
    need(positions.dim() == 1 && positions.size(0) == tokens && positions.scalar_type() == at::kInt &&
             positions.is_contiguous() && inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kFloat &&
             inv_freq.is_contiguous() && inv_freq.size(0) <= INT32_MAX / 2,
         "positions are int32 [tokens], inv_freq is float32 [rot_dim / 2]");
    need(dense(q), "q, k, v and caches must be contiguous in their heads");
    fmcuda_rope_append_args a{};
    at::ScalarType kind = out_dtype.value_or(q.scalar_type());
    if (k || v || k_cache || v_cache || slots) {
        need(k && v && k_cache && v_cache && slots, "k, v, their caches and slots come together",
             FM_STATUS_INVALID_ARGUMENT);
        need(k->dim() == 3 && k->size(0) == tokens && k->size(2) == dim && v->sizes() == k->sizes(),
             "k and v are [tokens, kv_heads, head_dim]");
        need(k_cache->dim() == 4 && v_cache->sizes() == k_cache->sizes() && v_cache->strides() == k_cache->strides() &&
                 k_cache->size(1) == k->size(1) && k_cache->size(3) == dim && k_cache->size(0) <= INT32_MAX &&
                 k_cache->size(2) <= INT32_MAX,
             "caches are [pages, kv_heads, page_size, head_dim], of one layout");
        need(slots->dim() == 1 && slots->size(0) == tokens && slots->scalar_type() == at::kLong &&
                 slots->is_contiguous(),
             "slots are int64 [tokens]");
        kind = k_cache->scalar_type();
        need(k->scalar_type() == q.scalar_type() && v->scalar_type() == q.scalar_type() &&
                 v_cache->scalar_type() == kind && out_dtype.value_or(kind) == kind,
             "q, k and v have one type, the output and the caches have one", FM_STATUS_INVALID_ARGUMENT);
        need(dense(*k) && dense(*v) && dense(*k_cache), "q, k, v and caches must be contiguous in their heads");
        a.k = k->data_ptr();
        a.v = v->data_ptr();
        a.k_cache = k_cache->data_ptr();
        a.v_cache = v_cache->data_ptr();
        a.slots = static_cast<const int64_t *>(slots->data_ptr());
        a.k_token_stride = k->stride(0);
        a.k_head_stride = k->stride(1);
        a.v_token_stride = v->stride(0);
        a.v_head_stride = v->stride(1);
        a.cache_page_stride = k_cache->stride(0);
        a.cache_head_stride = k_cache->stride(1);
        a.cache_row_stride = k_cache->stride(2);
        a.kv_heads = static_cast<uint32_t>(k->size(1));
        a.n_pages = static_cast<uint32_t>(k_cache->size(0));
        a.page_size = static_cast<uint32_t>(k_cache->size(2));
    }
    const Tensor out = at::empty(q.sizes(), q.options().dtype(kind));
    a.q = q.data_ptr();
    a.q_out = out.data_ptr();
    a.positions = static_cast<const int32_t *>(positions.data_ptr());
    a.inv_freq = static_cast<const float *>(inv_freq.data_ptr());
    a.q_token_stride = q.stride(0);
    a.q_head_stride = q.stride(1);
    a.q_out_token_stride = heads * dim;
    a.q_out_head_stride = dim;
    a.in_dtype = dtype_of(q);
    a.out_dtype = dtype_of(out);
    a.tokens = static_cast<uint32_t>(tokens);
    a.heads = static_cast<uint32_t>(heads);
    a.head_dim = static_cast<uint32_t>(dim);
    a.rot_dim = static_cast<uint32_t>(2 * inv_freq.size(0));
    a.interleaved = interleaved;
    a.attention_factor = static_cast<float>(attention_factor);
    check(entries.rope(&a, here.stream()));
    return out;
}

std::tuple<Tensor, MaybeTensor> paged_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache,
                                                const Tensor &page_table, const Tensor &q_start, const Tensor &kv_len,
                                                int64_t max_q_len, int64_t max_kv_len, std::optional<double> scale,
                                                bool causal, int64_t window, bool return_lse,
                                                const MaybeTensor &workspace) {
    need(q.dim() == 3 && k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes() &&
             v_cache.strides() == k_cache.strides() && k_cache.size(3) == q.size(2) && q.size(2) > 0,
         "q is [tokens, heads, head_dim], caches are [pages, kv_heads, page_size, head_dim], of one layout");
    const Here here(q);
    here(k_cache), here(v_cache), here(page_table), here(q_start), here(kv_len), here(workspace);
    need(k_cache.scalar_type() == q.scalar_type() && v_cache.scalar_type() == q.scalar_type(),
         "q and the caches have one type", FM_STATUS_INVALID_ARGUMENT);
    const int64_t seqs = kv_len.dim() == 1 ? kv_len.size(0) : -1;
    need(page_table.dim() == 2 && page_table.size(0) == seqs && q_start.dim() == 1 && q_start.size(0) == seqs + 1,
         "page_table is [seqs, pages], q_start [seqs + 1], kv_len [seqs]");
    need(page_table.scalar_type() == at::kInt && q_start.scalar_type() == at::kInt &&
             kv_len.scalar_type() == at::kInt && q_start.is_contiguous() && kv_len.is_contiguous(),
         "page_table, q_start and kv_len are int32", FM_STATUS_INVALID_ARGUMENT);
    need(max_q_len >= 0 && max_kv_len >= 0 && window >= 0, "lengths must not be negative", FM_STATUS_INVALID_ARGUMENT);
    need(max_kv_len <= INT32_MAX && window <= UINT32_MAX && q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX &&
             seqs < INT32_MAX && k_cache.size(0) <= INT32_MAX && k_cache.size(1) <= INT32_MAX &&
             k_cache.size(2) <= INT32_MAX && q.size(2) <= INT32_MAX,
         "attention lengths out of range");
    need(page_table.size(1) * k_cache.size(2) >= max_kv_len, "page table is shorter than max_kv_len");
    need(q.stride(2) == 1 && k_cache.stride(3) == 1 && (page_table.size(1) <= 1 || page_table.stride(1) == 1),
         "q, caches and page_table must be contiguous in their last dimension");
    const Tensor out = at::empty(q.sizes(), q.options());
    Tensor lse;
    fmcuda_paged_attention_args a{};
    if (return_lse) {
        lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
        a.lse = static_cast<float *>(lse.data_ptr());
    }
    a.q = q.data_ptr();
    a.k_cache = k_cache.data_ptr();
    a.v_cache = v_cache.data_ptr();
    a.out = out.data_ptr();
    a.page_table = static_cast<const int32_t *>(page_table.data_ptr());
    a.q_start = static_cast<const int32_t *>(q_start.data_ptr());
    a.kv_len = static_cast<const int32_t *>(kv_len.data_ptr());
    a.q_token_stride = q.stride(0);
    a.q_head_stride = q.stride(1);
    a.out_token_stride = q.size(1) * q.size(2);
    a.out_head_stride = q.size(2);
    a.cache_page_stride = k_cache.stride(0);
    a.cache_head_stride = k_cache.stride(1);
    a.cache_row_stride = k_cache.stride(2);
    a.page_table_stride = page_table.stride(0);
    a.dtype = dtype_of(q);
    a.seqs = static_cast<uint32_t>(seqs);
    a.tokens = static_cast<uint32_t>(q.size(0));
    a.heads = static_cast<uint32_t>(q.size(1));
    a.kv_heads = static_cast<uint32_t>(k_cache.size(1));
    a.head_dim = static_cast<uint32_t>(q.size(2));
    a.n_pages = static_cast<uint32_t>(k_cache.size(0));
    a.page_size = static_cast<uint32_t>(k_cache.size(2));
    a.max_q_len = static_cast<uint32_t>(max_q_len < q.size(0) ? max_q_len : q.size(0));
    a.max_kv_len = static_cast<uint32_t>(max_kv_len);
    a.causal = causal;
    a.window = static_cast<uint32_t>(window);
    a.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2))));
    Tensor own;
    void *at = at_of(workspace);
    uint64_t bytes = workspace ? workspace->nbytes() : 0;
    if (!workspace) {
        check(entries.attention_bytes(&a, &bytes));
        if (bytes) {
            own = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
            at = own.data_ptr();
        }
    }
    check(entries.attention(&a, at, bytes, here.stream()));
    return {out, return_lse ? MaybeTensor(lse) : std::nullopt};
}

void bind(py::object error, uint64_t last_error, uint64_t norm, uint64_t rope, uint64_t attention_bytes,
          uint64_t attention) {
    error_class = error.release().ptr(); // kept for the life of the process
    entries.last_error = reinterpret_cast<decltype(entries.last_error)>(last_error);
    entries.norm = reinterpret_cast<decltype(entries.norm)>(norm);
    entries.rope = reinterpret_cast<decltype(entries.rope)>(rope);
    entries.attention_bytes = reinterpret_cast<decltype(entries.attention_bytes)>(attention_bytes);
    entries.attention = reinterpret_cast<decltype(entries.attention)>(attention);
}

} // namespace

PYBIND11_MODULE(_torch_calls, m) {
    m.def("bind", &bind);
    m.def("add_rms_norm", &add_rms_norm);
    m.def("add_rms_norm_fp8", &add_rms_norm_fp8);
    m.def("rope_append", &rope_append);
    m.def("paged_attention", &paged_attention);
}
