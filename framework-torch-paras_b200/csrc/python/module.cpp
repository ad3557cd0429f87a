// Python extension module `torch_paras._C`: thin bindings over the device runtime, with the
// same names the reference exports (csrc/python/module.cpp:30-78) so its Python package API
// (device_count, synchronize, manual_seed, empty_cache, memory statistics, is_bad_fork)
// carries over unchanged.  Loading this module also runs the static registrations of the
// allocator, device guard, hooks and operators.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/utils/pybind.h>

#include "core/device_runtime.h"
#include "ops/paged_ops.h"

namespace py = pybind11;

PYBIND11_MODULE(_C, m) {
    m.doc() = "B200-native hot path behind the paras PrivateUse1 device";

    m.def("device_count", [] { return paras::Runtime::get().device_count(); });
    m.def("gpu_count", [] { return paras::Runtime::get().gpu_count(); });
    m.def("backend_name", [] { return std::string(paras_b200_backend_name()); });
    m.def("abi_version", [] { return paras_b200_abi_version(); });
    m.def("device_name", [](int index) { return paras::Runtime::get().device_name(index); });
    m.def("is_gpu_device", [](int index) {
        paras::Runtime::get().check_index(index);
        return paras::Runtime::get().is_gpu(index);
    });
    m.def("synchronize", [](int index) {
        py::gil_scoped_release no_gil;
        paras::Runtime::get().synchronize(index);
    });
    m.def("synchronize_all", [] {
        py::gil_scoped_release no_gil;
        paras::Runtime::get().synchronize_all();
    });
    m.def("manual_seed", [](int index, uint64_t seed) { paras::Runtime::get().set_seed(index, seed); });
    m.def("manual_seed_all", [](uint64_t seed) { paras::Runtime::get().set_seed_all(seed); });
    m.def("empty_cache", [] {
        py::gil_scoped_release no_gil;
        paras::Runtime::get().empty_cache_all();
    });
    m.def("allocated_bytes", [](int index) { return paras::Runtime::get().allocated_bytes(index); });
    m.def("cached_bytes", [](int index) { return paras::Runtime::get().cached_bytes(index); });
    m.def("is_bad_fork", [] { return paras::Runtime::bad_fork(); });
    m.def("sdpa_last_kernel", [] { return std::string(paras_b200_sdpa_last_kernel()); });
    // The calls of torch_paras.abi on torch.cuda tensors (`stream`: raw handle) that are short enough for Python's checks to show.
    using T = at::Tensor;
    using O = paras::OptTensor;
    m.def("paged_attn_last_kernel", [] { return std::string(paras_b200_paged_attn_last_kernel()); });
    m.def("paged_kv_write", &paras::paged_kv_write);
    m.def("paged_kv_read", [](const T& k_cache, const T& v_cache, const T& page_table, const T& cu_kv, int64_t total, const py::object& dtype,
                              const O& k_exp, const O& v_exp, const O& out_k, const O& out_v, int64_t stream) {
        std::optional<c10::ScalarType> to;
        if (!dtype.is_none()) {
            if (!THPDtype_Check(dtype.ptr())) throw py::type_error("paras paged_kv_read: dtype must be a torch.dtype");
            to = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
        }
        return paras::paged_kv_read(k_cache, v_cache, page_table, cu_kv, total, to, k_exp, v_exp, out_k, out_v, stream);
    });
    m.def("paged_attention", [](const T& q, const T& k_cache, const T& v_cache, const T& page_table, const T& kv_lens, const T& cu_q,
                                int64_t max_q, bool causal, std::optional<double> scale, const O& k_exp, const O& v_exp, const O& out,
                                bool want_lse, const O& workspace, int64_t stream) {
        return paras::paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_q, max_q, causal, scale, k_exp, v_exp, out, want_lse,
                                      workspace, stream, nullptr);
    });
    m.def("paged_attn_workspace_bytes", [](const T& q, const T& k_cache, const T& v_cache, const T& page_table, const T& kv_lens,
                                           const T& cu_q, int64_t max_q, bool causal, const O& k_exp, const O& v_exp) {
        size_t n = 0;
        paras::paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_q, max_q, causal, {}, k_exp, v_exp, {}, false, {}, 0, &n);
        return n;
    });
    m.def("add_rms_norm", &paras::add_rms_norm);
    m.def("add_rms_norm_quant", &paras::add_rms_norm_quant);
    m.def("add_rms_norm_backward", &paras::add_rms_norm_backward);
    // Raw stream handle of a paras GPU device, for interop (e.g. wrapping in torch.cuda.ExternalStream).
    m.def("raw_stream", [](int index) {
        void* s = nullptr;
        PARAS_ABI(paras_b200_stream(paras::Runtime::get().gpu_of(index), &s));
        return reinterpret_cast<uintptr_t>(s);
    });
}
