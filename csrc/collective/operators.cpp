// C ABI of the model operators: argument checks, then the launches of experts.cu and grad_clip.cu.
#include "collective/operators.hpp"

#include <atomic>
#include <cstring>

namespace {

constexpr uint64_t kDefaultWaitNs = 5ull * 1000 * 1000 * 1000;
std::atomic<uint64_t> g_wait_ns{kDefaultWaitNs};

bool aligned16(const void *p) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned32(const void *p) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % 32 == 0; }

bool valid(const ugdr_x_experts *m) {
    return m != nullptr && m->counts != nullptr && m->status != nullptr && aligned16(m->w_in) && aligned16(m->w_out) &&
           m->rows <= UGDR_X_EXPERTS_MAX_ROWS && m->nexp >= 1 && m->nexp <= UGDR_X_EXPERTS_MAX && m->hidden >= 8 &&
           m->hidden <= UGDR_X_EXPERTS_MAX_SIZE && m->hidden % 8 == 0 && m->inner >= 8 &&
           m->inner <= UGDR_X_EXPERTS_MAX_SIZE && m->inner % 8 == 0 &&
           (m->type == UGDR_X_TYPE_BF16 || m->type == UGDR_X_TYPE_FP16) &&
           (m->act == UGDR_X_ACT_SILU || m->act == UGDR_X_ACT_GELU);
}

size_t element_bytes(int type) { return type == UGDR_X_TYPE_FP32 ? 4 : 2; }

}  // namespace

uint64_t ugdr::coll::expert_wait_ns() { return g_wait_ns.load(std::memory_order_relaxed); }

extern "C" {

uint64_t ugdr_x_set_expert_wait_ns(uint64_t ns) { return g_wait_ns.exchange(ns == 0 ? kDefaultWaitNs : ns); }

int ugdr_x_expert_ffn(const ugdr_x_experts *m, const void *x, void *y, void *h, float *gu, void *stream) {
    if (!valid(m)) return int(cudaErrorInvalidValue);
    if (m->rows == 0) return ugdr::coll::launch_count_check(*m, static_cast<cudaStream_t>(stream));
    if (!aligned16(x) || !aligned16(y) || !aligned16(h) || (gu != nullptr && !aligned32(gu)))
        return int(cudaErrorInvalidValue);
    return ugdr::coll::launch_expert_ffn(*m, x, y, h, gu, static_cast<cudaStream_t>(stream));
}

int ugdr_x_expert_ffn_backward(const ugdr_x_experts *m, const void *dy, const void *x, const void *h, const float *gu,
                               void *dgu, void *dx, void *dw_in, void *dw_out, void *stream) {
    if (!valid(m) || !aligned16(dw_in) || !aligned16(dw_out)) return int(cudaErrorInvalidValue);
    const auto s = static_cast<cudaStream_t>(stream);
    if (m->rows == 0) {
        const size_t block = size_t(m->nexp) * size_t(m->inner) * size_t(m->hidden) * 2;
        if (const cudaError_t e = cudaMemsetAsync(dw_in, 0, 2 * block, s); e != cudaSuccess) return int(e);
        if (const cudaError_t e = cudaMemsetAsync(dw_out, 0, block, s); e != cudaSuccess) return int(e);
        return ugdr::coll::launch_count_check(*m, s);
    }
    if (!aligned16(dy) || !aligned16(x) || !aligned16(h) || !aligned32(gu) || !aligned16(dgu) || !aligned16(dx))
        return int(cudaErrorInvalidValue);
    return ugdr::coll::launch_expert_ffn_backward(*m, dy, x, h, gu, dgu, dx, dw_in, dw_out, s);
}

size_t ugdr_x_grad_plan_bytes(int n) {
    if (n < 0) return 0;
    return size_t(n) * sizeof(ugdr_x_grad) + (size_t(n) + 1) * sizeof(uint32_t);
}

int ugdr_x_grad_plan(const ugdr_x_grad *grads, int n, void *plan, uint64_t *chunks) {
    if (n < 0 || (n > 0 && grads == nullptr) || plan == nullptr || chunks == nullptr) return int(cudaErrorInvalidValue);
    uint64_t at = 0;
    auto *first = static_cast<uint8_t *>(plan) + size_t(n) * sizeof(ugdr_x_grad);
    for (int i = 0; i <= n; ++i) {
        const uint32_t at32 = uint32_t(at);
        std::memcpy(first + size_t(i) * sizeof(at32), &at32, sizeof(at32));
        if (i == n) break;
        const ugdr_x_grad &g = grads[i];
        if (g.grad_type < UGDR_X_TYPE_BF16 || g.grad_type > UGDR_X_TYPE_FP32 ||
            (g.out_type != g.grad_type && g.out_type != UGDR_X_TYPE_FP32))
            return int(cudaErrorInvalidValue);
        if (g.count > 0 && (g.grad == nullptr || reinterpret_cast<uintptr_t>(g.grad) % element_bytes(g.grad_type) ||
                            g.out == nullptr || reinterpret_cast<uintptr_t>(g.out) % element_bytes(g.out_type)))
            return int(cudaErrorInvalidValue);
        if (g.count > (uint64_t(1) << 44)) return int(cudaErrorInvalidValue);
        // In place works element by element; elements of another size would land on ones yet to be read.
        const auto in = reinterpret_cast<uintptr_t>(g.grad), out = reinterpret_cast<uintptr_t>(g.out);
        if (g.count > 0 && (in != out || g.out_type != g.grad_type) && out < in + g.count * element_bytes(g.grad_type) &&
            in < out + g.count * element_bytes(g.out_type))
            return int(cudaErrorInvalidValue);
        // A tensor's first chunk begins before its first element, on a boundary of 8 elements.
        const size_t width = element_bytes(g.grad_type);
        const uint64_t lead = in % (8 * width) / width;
        if (g.count > 0) at += (g.count + lead + ugdr::coll::kGradChunk - 1) / ugdr::coll::kGradChunk;
        if (at > UINT32_MAX) return int(cudaErrorInvalidValue);
    }
    if (n > 0) std::memcpy(plan, grads, size_t(n) * sizeof(ugdr_x_grad));
    *chunks = at;
    return int(cudaSuccess);
}

int ugdr_x_grad_sum_squares(const void *plan, int n, uint64_t chunks, double *partials, double *sum_squares,
                            void *stream) {
    if (n < 0 || !aligned16(plan) || partials == nullptr || sum_squares == nullptr || chunks > UINT32_MAX)
        return int(cudaErrorInvalidValue);
    return ugdr::coll::launch_grad_sum_squares(plan, n, chunks, partials, sum_squares,
                                               static_cast<cudaStream_t>(stream));
}

int ugdr_x_grad_clip(const void *plan, int n, uint64_t chunks, double *partials, const double *sum_squares,
                     float max_norm, float *norm_out, void *stream) {
    if (n < 0 || !aligned16(plan) || (partials == nullptr && sum_squares == nullptr) || norm_out == nullptr ||
        chunks > UINT32_MAX || !(max_norm >= 0.f))
        return int(cudaErrorInvalidValue);
    return ugdr::coll::launch_grad_clip(plan, n, chunks, partials, sum_squares, max_norm, norm_out,
                                        static_cast<cudaStream_t>(stream));
}

}  // extern "C"
