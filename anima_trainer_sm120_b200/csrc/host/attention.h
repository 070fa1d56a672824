// Attention and the joint q / k RMSNorm + rotary embedding as native autograd nodes.
#pragma once

#include "common.h"

namespace anima_host {

// q (B, Lq, H, D), k and v (B, Lk, Hk, D) bf16, any strides; lengths int32 [B]: keys of each sample. Returns (out, lse); lse is
// undefined unless it is wanted or a gradient is.
std::tuple<Tensor, OptTensor> attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths, bool causal,
                                        double scale, bool want_lse);
// q (B, Lq, H, D), k (B, Lk, Hk, D) bf16, any strides; weights [D]; tables fp32 [L, D] or [B, L, D]
std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                        const OptTensor& cos, const OptTensor& sin, double eps);

}  // namespace anima_host
