// Paged key / value cache of the `paras` device: its writer, its reader and the attention of new tokens over it, each
// through the C ABI (include/paras_b200.h, "paged key / value cache").  No counterpart in the reference, whose
// attention (csrc/ops/attention_ops.cpp:71-136) takes dense tensors of one length.
//
//   paras::paged_kv_write(k, v, k_cache, v_cache, page_table, kv_lens, cu_q, k_exp?, v_exp?)     caches in place
//   paras::paged_kv_read(k_cache, v_cache, page_table, cu_kv, total, dtype?, k_exp?, v_exp?) -> (k, v)
//   paras::paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_q, max_q, ...) -> (out, lse)
//
// Caches are [pages, kv heads, page, D] of any strides with contiguous rows, in the tokens' dtype or float8_e4m3fn
// with exponent bytes k_exp / v_exp [pages, kv heads, page].  Lengths and page numbers stay on the device.
//
// The functions take tensors of the `paras` device, and, for torch_paras.abi, torch.cuda ones with the stream to launch
// on (the arguments are checked and packed in C++: in Python that costs more than the smallest kernels run).
#include "ops/paged_ops.h"

#include <torch/library.h>

#include "core/device_runtime.h"

namespace paras {

Place place_of(const at::Tensor& t, int64_t stream) {
    if (t.device().type() == kDevice) return {Runtime::get().gpu_of(t), nullptr};
    TORCH_CHECK(t.is_cuda(), "paras: expected a paras or CUDA tensor, got one on ", t.device());
    return {int(t.get_device()), reinterpret_cast<void*>(stream)};
}

namespace {

using at::Tensor;

void fill_cache(paras_paged_cache& c, const Tensor& k, const Tensor& v, const Tensor& table, const OptTensor& ke,
                const OptTensor& ve, const Tensor& rows, const char* what) {
    TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(),
                "paras ", what, ": caches must be two [pages, kv heads, page, D] tensors of one type");
    TORCH_CHECK(k.size(3) <= 1 || (k.stride(3) == 1 && v.stride(3) == 1), "paras ", what, ": cache rows must be contiguous");
    TORCH_CHECK(table.dim() == 2 && table.scalar_type() == c10::kInt && (table.size(1) <= 1 || table.stride(1) == 1),
                "paras ", what, ": page_table must be int32 [sequences, pages] with contiguous rows");
    for (const Tensor* t : {&k, &v, &table})
        TORCH_CHECK(t->device() == rows.device(), "paras ", what, ": tensors are on different devices");
    for (int64_t n : {k.size(0), k.size(1), k.size(2), k.size(3), table.size(0), table.size(1)})
        TORCH_CHECK(n <= INT32_MAX, "paras ", what, ": a size exceeds 2^31 - 1");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    for (int i = 0; i < 3; ++i) {
        c.k_strides[i] = k.stride(i);
        c.v_strides[i] = v.stride(i);
    }
    const bool has_exp = (ke && ke->defined()) || (ve && ve->defined());
    if (k.scalar_type() == c10::kFloat8_e4m3fn) {
        c.cache_dtype = PARAS_E4M3;
        for (const OptTensor* e : {&ke, &ve})
            TORCH_CHECK(*e && (*e)->defined() && (*e)->sizes() == k.sizes().slice(0, 3) && (*e)->element_size() == 1 &&
                            (*e)->device() == rows.device(),
                        "paras ", what, ": an 8-bit cache needs k_exp and v_exp, bytes of shape [pages, kv heads, page]");
        c.k_exp = static_cast<uint8_t*>(ke->data_ptr());
        c.v_exp = static_cast<uint8_t*>(ve->data_ptr());
        for (int i = 0; i < 3; ++i) {
            c.k_exp_strides[i] = ke->stride(i);
            c.v_exp_strides[i] = ve->stride(i);
        }
    } else {
        TORCH_CHECK(!has_exp, "paras ", what, ": k_exp and v_exp belong to an 8-bit cache");
        c.cache_dtype = dtype_code(k.scalar_type());
        TORCH_CHECK(c.cache_dtype >= 0, "paras ", what, ": unsupported cache dtype ", k.scalar_type());
    }
    c.pages = int32_t(k.size(0));
    c.Hkv = int32_t(k.size(1));
    c.page = int32_t(k.size(2));
    c.D = int32_t(k.size(3));
    c.page_table = static_cast<const int32_t*>(table.data_ptr());
    c.table_stride = table.stride(0);
    c.B = int32_t(table.size(0));
    c.max_pages = int32_t(table.size(1));
}

const int32_t* index_array(const Tensor& t, int64_t n, const Tensor& rows, const char* what, const char* name) {
    TORCH_CHECK(t.dim() == 1 && t.scalar_type() == c10::kInt && t.size(0) == n && t.is_contiguous() && t.device() == rows.device(),
                "paras ", what, ": ", name, " must be a contiguous int32 vector of ", n, " entries on the tensors' device");
    return static_cast<const int32_t*>(t.data_ptr());
}

// Token rows whose last dim is contiguous, as the kernels read them.
Tensor rows_of(const Tensor& t, int64_t heads, int64_t D, const char* what, const char* name) {
    TORCH_CHECK(t.dim() == 3 && (heads < 0 || t.size(1) == heads) && t.size(2) == D,
                "paras ", what, ": ", name, " must be [tokens, heads, D] and fit the cache");
    TORCH_CHECK(dtype_code(t.scalar_type()) >= 0, "paras ", what, ": unsupported dtype ", t.scalar_type());
    TORCH_CHECK(t.size(0) <= INT32_MAX, "paras ", what, ": more than 2^31 - 1 tokens");
    return (D <= 1 || t.stride(2) == 1) ? t : t.contiguous();
}

}  // namespace

void paged_kv_write(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache, const Tensor& page_table,
                    const Tensor& kv_lens, const Tensor& cu_q, const OptTensor& k_exp, const OptTensor& v_exp, int64_t stream) {
    PARAS_TRACE_OP("paras::paged_kv_write");
    const char* what = "paged_kv_write";
    const Place at = place_of(k, stream);
    c10::DeviceGuard guard(k.device());
    paras_paged_kv_args a{};
    fill_cache(a.cache, k_cache, v_cache, page_table, k_exp, v_exp, k, what);
    TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.device() == k.device(),
                "paras paged_kv_write: k and v must have one type, shape and device");
    Tensor kr = rows_of(k, a.cache.Hkv, a.cache.D, what, "k"), vr = rows_of(v, a.cache.Hkv, a.cache.D, what, "v");
    a.k = kr.data_ptr();
    a.v = vr.data_ptr();
    for (int i = 0; i < 2; ++i) {
        a.k_strides[i] = kr.stride(i);
        a.v_strides[i] = vr.stride(i);
    }
    a.kv_lens = index_array(kv_lens, a.cache.B, k, what, "kv_lens");
    a.cu = index_array(cu_q, int64_t(a.cache.B) + 1, k, what, "cu_q");
    a.T = int32_t(k.size(0));
    a.dtype = dtype_code(k.scalar_type());
    a.gpu = at.gpu;
    a.stream = at.stream;
    PARAS_ABI(paras_b200_paged_kv_write(&a));
}

std::tuple<Tensor, Tensor> paged_kv_read(const Tensor& k_cache, const Tensor& v_cache, const Tensor& page_table,
                                         const Tensor& cu_kv, int64_t total, std::optional<c10::ScalarType> dtype,
                                         const OptTensor& k_exp, const OptTensor& v_exp, const OptTensor& out_k,
                                         const OptTensor& out_v, int64_t stream) {
    PARAS_TRACE_OP("paras::paged_kv_read");
    const char* what = "paged_kv_read";
    const Place at = place_of(k_cache, stream);
    c10::DeviceGuard guard(k_cache.device());
    TORCH_CHECK(total >= 0 && total <= INT32_MAX, "paras paged_kv_read: total must be within 0 .. 2^31 - 1");
    TORCH_CHECK(k_cache.dim() == 4, "paras paged_kv_read: caches must be [pages, kv heads, page, D]");
    const auto to = dtype.value_or(k_cache.scalar_type() == c10::kFloat8_e4m3fn ? c10::kBFloat16 : k_cache.scalar_type());
    TORCH_CHECK(dtype_code(to) >= 0, "paras paged_kv_read: unsupported dtype ", to);
    Tensor k, v;
    TORCH_CHECK(out_k.has_value() == out_v.has_value(), "paras paged_kv_read: the outputs are given both or not at all");
    if (out_k && out_v) {
        k = *out_k;
        v = *out_v;
        TORCH_CHECK(rows_of(k, k_cache.size(1), k_cache.size(3), what, "k").is_same(k) &&
                        rows_of(v, k_cache.size(1), k_cache.size(3), what, "v").is_same(v) && k.size(0) == total && v.size(0) == total &&
                        v.scalar_type() == k.scalar_type() && k.device() == k_cache.device() && v.device() == k.device(),
                    "paras paged_kv_read: the two outputs must have one type, the cache's device, contiguous rows and `total` of them");
        TORCH_CHECK(!dtype || *dtype == k.scalar_type(), "paras paged_kv_read: the outputs have type ", k.scalar_type(), ", not the dtype asked for");
    } else {
        k = at::empty({total, k_cache.size(1), k_cache.size(3)}, k_cache.options().dtype(to));
        v = at::empty_like(k);
    }
    paras_paged_kv_args a{};
    fill_cache(a.cache, k_cache, v_cache, page_table, k_exp, v_exp, k, what);
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    for (int i = 0; i < 2; ++i) {
        a.k_strides[i] = k.stride(i);
        a.v_strides[i] = v.stride(i);
    }
    a.cu = index_array(cu_kv, int64_t(a.cache.B) + 1, k, what, "cu_kv");
    a.T = int32_t(total);
    a.dtype = dtype_code(k.scalar_type());
    a.gpu = at.gpu;
    a.stream = at.stream;
    PARAS_ABI(paras_b200_paged_kv_read(&a));
    return {k, v};
}

std::tuple<Tensor, Tensor> paged_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                                           const Tensor& page_table, const Tensor& kv_lens, const Tensor& cu_q, int64_t max_q,
                                           bool is_causal, std::optional<double> scale, const OptTensor& k_exp,
                                           const OptTensor& v_exp, const OptTensor& out_given, bool want_lse,
                                           const OptTensor& workspace, int64_t stream, size_t* workspace_bytes) {
    PARAS_TRACE_OP("paras::paged_attention");
    const char* what = "paged_attention";
    const Place at = place_of(q, stream);
    c10::DeviceGuard guard(q.device());
    paras_paged_attn_args a{};
    fill_cache(a.cache, k_cache, v_cache, page_table, k_exp, v_exp, q, what);
    Tensor qr = rows_of(q, -1, a.cache.D, what, "q"), out, lse;
    TORCH_CHECK(max_q >= 0, "paras paged_attention: max_q is negative");
    if (out_given && out_given->defined()) {
        out = *out_given;
        TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == q.device() &&
                        (a.cache.D <= 1 || out.stride(2) == 1),
                    "paras paged_attention: out must have q's shape, type and device and contiguous rows");
    } else {
        out = workspace_bytes ? Tensor() : at::empty(q.sizes(), q.options());
    }
    if (want_lse) lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(c10::kFloat));
    a.q = qr.data_ptr();
    a.out = out.defined() ? out.data_ptr() : nullptr;
    a.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
    for (int i = 0; i < 2; ++i) {
        a.q_strides[i] = qr.stride(i);
        // (a workspace is measured for contiguous rows: other ones never need more)
        a.o_strides[i] = out.defined() ? out.stride(i) : (i == 0 ? q.size(1) : 1) * q.size(2);
    }
    a.kv_lens = index_array(kv_lens, a.cache.B, q, what, "kv_lens");
    a.cu = index_array(cu_q, int64_t(a.cache.B) + 1, q, what, "cu_q");
    a.T = int32_t(q.size(0));
    a.Hq = int32_t(q.size(1));
    a.max_q = int32_t(std::min<int64_t>(max_q, q.size(0)));
    a.dtype = dtype_code(q.scalar_type());
    a.causal = is_causal;
    a.gpu = at.gpu;
    a.stream = at.stream;
    a.scale = scale ? *scale : 1.0 / std::sqrt(double(a.cache.D));
    if (workspace && workspace->defined()) {
        TORCH_CHECK(workspace->device() == q.device() && workspace->is_contiguous(),
                    "paras paged_attention: workspace must be contiguous and on q's device");
        a.workspace = workspace->data_ptr();
        a.workspace_bytes = workspace->nbytes();
    }
    if (workspace_bytes) {
        PARAS_ABI(paras_b200_paged_attn_workspace_bytes(&a, workspace_bytes));
    } else {
        PARAS_ABI(paras_b200_paged_attn(&a));
    }
    return {out, lse};
}

}  // namespace paras

TORCH_LIBRARY_FRAGMENT(paras, m) {
    m.def("paged_kv_write(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, Tensor kv_lens, "
          "Tensor cu_q, Tensor(c!)? k_exp=None, Tensor(d!)? v_exp=None) -> ()");
    m.def("paged_kv_read(Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor cu_kv, int total, ScalarType? dtype=None, "
          "Tensor? k_exp=None, Tensor? v_exp=None) -> (Tensor, Tensor)");
    m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor kv_lens, Tensor cu_q, int max_q, "
          "bool is_causal=True, float? scale=None, Tensor? k_exp=None, Tensor? v_exp=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(paras, PrivateUse1, m) {
    using paras::OptTensor;
    m.impl("paged_kv_write", [](const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                const at::Tensor& page_table, const at::Tensor& kv_lens, const at::Tensor& cu_q, const OptTensor& k_exp,
                                const OptTensor& v_exp) {
        paras::paged_kv_write(k, v, k_cache, v_cache, page_table, kv_lens, cu_q, k_exp, v_exp, 0);
    });
    m.impl("paged_kv_read", [](const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& page_table, const at::Tensor& cu_kv,
                               int64_t total, std::optional<c10::ScalarType> dtype, const OptTensor& k_exp, const OptTensor& v_exp) {
        return paras::paged_kv_read(k_cache, v_cache, page_table, cu_kv, total, dtype, k_exp, v_exp, {}, {}, 0);
    });
    m.impl("paged_attention", [](const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& page_table,
                                 const at::Tensor& kv_lens, const at::Tensor& cu_q, int64_t max_q, bool is_causal, std::optional<double> scale,
                                 const OptTensor& k_exp, const OptTensor& v_exp) {
        return paras::paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_q, max_q, is_causal, scale, k_exp, v_exp, {}, true, {},
                                      0, nullptr);
    });
}
