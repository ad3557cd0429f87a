// The paged cache's and the residual norm's calls as C++ functions on tensors of the `paras` device or torch.cuda ones
// (with the stream to launch on; ignored for `paras` tensors, whose library stream orders them).
#pragma once

#include <ATen/ATen.h>

#include <optional>
#include <tuple>

namespace paras {

using OptTensor = std::optional<at::Tensor>;

struct Place {
    int gpu;         // CUDA ordinal
    void* stream;
};
Place place_of(const at::Tensor& t, int64_t stream);

void paged_kv_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
                    const at::Tensor& page_table, const at::Tensor& kv_lens, const at::Tensor& cu_q, const OptTensor& k_exp,
                    const OptTensor& v_exp, int64_t stream);
std::tuple<at::Tensor, at::Tensor> paged_kv_read(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& page_table,
                                                 const at::Tensor& cu_kv, int64_t total, std::optional<c10::ScalarType> dtype,
                                                 const OptTensor& k_exp, const OptTensor& v_exp, const OptTensor& out_k,
                                                 const OptTensor& out_v, int64_t stream);
// (out, lse or an undefined tensor); with `workspace_bytes` only that is asked for, and nothing runs.
std::tuple<at::Tensor, at::Tensor> paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                                   const at::Tensor& page_table, const at::Tensor& kv_lens, const at::Tensor& cu_q,
                                                   int64_t max_q, bool is_causal, std::optional<double> scale, const OptTensor& k_exp,
                                                   const OptTensor& v_exp, const OptTensor& out, bool want_lse,
                                                   const OptTensor& workspace, int64_t stream, size_t* workspace_bytes);

// (y, h, rstd or undefined); h is x where there is no residual
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm(const at::Tensor& x, const OptTensor& residual, const OptTensor& weight,
                                                            double eps, bool want_rstd, int64_t stream);
// (q, scales, h)
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_quant(const at::Tensor& x, const OptTensor& residual, const OptTensor& weight,
                                                                  double eps, int64_t group, int64_t stream);
// (grad_x, grad_weight or undefined)
std::tuple<at::Tensor, at::Tensor> add_rms_norm_backward(const at::Tensor& grad_y, const OptTensor& grad_h, const at::Tensor& h,
                                                         const OptTensor& weight, const at::Tensor& rstd, int64_t stream);

}  // namespace paras
