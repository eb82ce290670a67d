// Host launch interface of the model operators (experts.cu, grad_clip.cu).
#pragma once

#include "collective/kernels.hpp"
#include "ugdr/experts.h"

#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

namespace ugdr::coll {

uint64_t expert_wait_ns();  // bound of the waits in the experts' kernels
int launch_count_check(const ugdr_x_experts &m, cudaStream_t s);  // for calls without rows
int launch_expert_ffn(const ugdr_x_experts &m, const void *x, void *y, void *h, float *gu, cudaStream_t s);
int launch_expert_ffn_backward(const ugdr_x_experts &m, const void *dy, const void *x, const void *h, const float *gu,
                               void *dgu, void *dx, void *dw_in, void *dw_out, cudaStream_t s);

// A plan in memory: n tensors, then n + 1 first-chunk indices.
constexpr uint32_t kGradChunk = 4096;  // elements; a tensor's last chunk may be shorter
int launch_grad_sum_squares(const void *plan, int n, uint64_t chunks, double *partials, double *sum_squares,
                            cudaStream_t s);
int launch_grad_clip(const void *plan, int n, uint64_t chunks, double *partials, const double *sum_squares,
                     float max_norm, float *norm_out, cudaStream_t s);

// The operators' kernels, for resource reports.
int expert_kernels(const KernelRef **out);
int grad_kernels(const KernelRef **out);

}  // namespace ugdr::coll
