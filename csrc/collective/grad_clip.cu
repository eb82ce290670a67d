// Global gradient norm over many tensors, and clipping.
//
//   s = sum_i sum_j g_ij^2,  norm = sqrt(s),  out_ij = g_ij * min(1, max_norm / (norm + 1e-6))
//
// Both passes are bound by memory: the norm reads every gradient once, the scaling reads it again
// and writes it.  The tensors are cut into chunks of 4096 elements, counted through all tensors, and
// every block takes an equal, contiguous run of chunks, so a list of hundreds of small tensors and
// one of a few huge ones load the GPU alike, in one launch.  The sums depend on nothing but the
// plan and the grid: no atomics.
//
// Measured on a B200: 200 tensors of 1 M bf16 elements are read in 63 us (6.4 TB/s) and scaled into
// fp32 in 207 us (0.40 GB read, 0.8 GB written: writing alone goes at 3.9 TB/s here, in torch's fill
// too); 1.4e9 elements take 1.89 ms for both.
//
// Squares of 8 neighbours are summed in fp32 (an error of a few 2^-24) and those sums in fp64, so
// the length of the list costs no precision.  A group whose fp32 sum leaves the range in which that
// holds (overflow, or squares near fp32's smallest numbers) is summed again in fp64.
#include "collective/operators.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace ugdr::coll {
namespace {

constexpr int kThreads = 512;
constexpr int kGroup = 8;    // elements a thread takes at once: 16 or 32 bytes
constexpr int kInFlight = 8;  // 8 / element size groups in flight per thread: 64 bytes
constexpr int kNormBlocks = 3, kScaleBlocks = 2;  // per SM: some find their next tensor while the others read
static_assert(kThreads * kGroup == kGradChunk, "one group per thread and chunk");

template <int TYPE> struct Element;
template <> struct Element<UGDR_X_TYPE_BF16> {
    using type = __nv_bfloat16;
};
template <> struct Element<UGDR_X_TYPE_FP16> {
    using type = __half;
};
template <> struct Element<UGDR_X_TYPE_FP32> {
    using type = float;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float &d, float v) { d = v; }
__device__ __forceinline__ void from_float(__half &d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_float(__nv_bfloat16 &d, float v) { d = __float2bfloat16_rn(v); }

template <typename T> struct alignas(sizeof(T) * kGroup) Group {
    T v[kGroup];
};

template <typename T> __device__ __forceinline__ Group<T> load_group(const T *p) {
    Group<T> g;
    if constexpr (sizeof(T) == 4) {
        uint32_t *w = reinterpret_cast<uint32_t *>(g.v);
        asm volatile("ld.global.v8.u32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(p)
                     : "memory");
    } else {
        uint32_t *w = reinterpret_cast<uint32_t *>(g.v);
        asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "l"(p)
                     : "memory");
    }
    return g;
}
template <typename T> __device__ __forceinline__ void store_group(T *p, const Group<T> &g) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(g.v);
    if constexpr (sizeof(T) == 4)
        asm volatile("st.global.v8.u32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                     "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    else
        asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                     : "memory");
}

template <typename O, typename T> __device__ __forceinline__ Group<O> scaled(const Group<T> &g, float coef) {
    Group<O> o;
#pragma unroll
    for (int j = 0; j < kGroup; ++j) from_float(o.v[j], to_float(g.v[j]) * coef);
    return o;
}

// The tensor list of a plan: the tensors and the chunk that each begins with.
struct Plan {
    const ugdr_x_grad *grads;
    const uint32_t *first;
    int n;
};

// The tensor that holds `chunk`: every thread looks at some of them, one finds it.
__device__ int tensor_of(const Plan &p, uint32_t chunk) {
    __shared__ int found;
    for (int i = threadIdx.x; i < p.n; i += kThreads)
        if (p.first[i] <= chunk && chunk < p.first[i + 1]) found = i;
    __syncthreads();
    const int i = found;
    __syncthreads();
    return i;
}

__device__ double block_sum(double v) {
    __shared__ double warp_sums[kThreads / 32];
    for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threadIdx.x % 32 == 0) warp_sums[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kThreads / 32; ++w) v += warp_sums[w];
    return v;
}

template <typename T> __device__ __forceinline__ float squares(const Group<T> &g) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kGroup; ++j) s = fmaf(to_float(g.v[j]), to_float(g.v[j]), s);
    return s;
}
template <typename T> __device__ __forceinline__ bool all_zero(const Group<T> &g) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(g.v);
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < int(sizeof(g) / 4); ++j) any |= w[j];
    return (any & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) == 0;
}
// Whether a group's fp32 sum of squares `s` says less than it should: numbers whose squares fp32 cannot
// hold.  A sum of 0 that comes from zeros is right, and they are not read a second time: 600 M bf16
// elements, half of their groups zeros (an embedding's rows that no token used), take 186 us like any
// others, and took 267 us when zeros counted as unsafe.
template <typename T> __device__ __forceinline__ bool unsafe(float s, const Group<T> &g) {
    return !(s < 3e38f && s > 1e-30f) && !all_zero(g);
}
__device__ __forceinline__ double squares_wide(float a, double sum) { return fma(double(a), double(a), sum); }

// The squares of `n` groups of one thread, a chunk apart.
template <typename T> __device__ __noinline__ double squares_wide(const T *p, int n) {
    double sum = 0;
#pragma unroll 1
    for (int u = 0; u < n; ++u, p += kGradChunk) {
        const Group<T> g = load_group(p);
#pragma unroll
        for (int j = 0; j < kGroup; ++j) sum = squares_wide(to_float(g.v[j]), sum);
    }
    return sum;
}

// Elements before the tensor's first that make its base a multiple of a group's bytes: chunk c
// holds the elements [4096 c - lead, 4096 (c + 1) - lead) that exist, so that every whole group is
// one aligned load whatever the tensor's own alignment.
template <typename T> __device__ __forceinline__ uint32_t lead_of(const T *p) {
    return uint32_t(reinterpret_cast<uintptr_t>(p) % (sizeof(T) * kGroup) / sizeof(T));
}

// The chunks of [c0, c1) in which this thread's group lies in the tensor as a whole: [a, b).
struct Mine {
    uint32_t a, b;
};
__device__ __forceinline__ Mine my_chunks(uint32_t c0, uint32_t c1, uint32_t lead, int64_t n) {
    const uint32_t a = c0 + (c0 == 0 && lead != 0 && threadIdx.x == 0);
    const int64_t last = n + lead - kGroup * int64_t(threadIdx.x + 1);  // begins no further than here
    const uint32_t b = last < 0 ? a : uint32_t(min(int64_t(c1), last / kGradChunk + 1));
    return {a, max(a, b)};
}

// The elements outside whole groups, before the first and behind the last: f(index), from the thread
// and the chunk that they belong to.
template <typename F> __device__ __forceinline__ void partial_groups(uint32_t c0, uint32_t c1, uint32_t lead, int64_t n, F f) {
    if (c0 == 0 && lead != 0 && threadIdx.x == 0)
        for (int64_t i = 0; i < min(int64_t(kGroup - lead), n); ++i) f(i);
    const int64_t groups = (n + lead) / kGroup, chunk = groups / kThreads;
    if (chunk >= c0 && chunk < c1 && threadIdx.x == uint32_t(groups % kThreads) && groups * kGroup >= lead)
        for (int64_t i = groups * kGroup - lead; i < n; ++i) f(i);
}

// The squares of the chunks [c0, c1) of one tensor.
template <int TYPE> __device__ double span_squares(const ugdr_x_grad &t, uint32_t c0, uint32_t c1) {
    using T = typename Element<TYPE>::type;
    constexpr int kUnroll = kInFlight / sizeof(T);
    const T *g = static_cast<const T *>(t.grad);
    const uint32_t lead = lead_of(g);
    const int64_t n = int64_t(t.count);
    const Mine w = my_chunks(c0, c1, lead, n);
    const T *p = g + (int64_t(w.a) * kGradChunk + threadIdx.x * kGroup - int64_t(lead));
    double acc = 0;
    int left = int(w.b - w.a);
    for (; left >= kUnroll; left -= kUnroll, p += kUnroll * kGradChunk) {
        Group<T> v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = load_group(p + u * kGradChunk);
        double sum = 0;
        bool wide = false;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const float q = squares(v[u]);
            wide |= unsafe(q, v[u]);
            sum += double(q);
        }
        acc += wide ? squares_wide(p, kUnroll) : sum;
    }
    if (left > 0) {  // at once too: the last of them stands in for those missing
        Group<T> v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = load_group(p + min(u, left - 1) * kGradChunk);
        double sum = 0;
        bool wide = false;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const float q = squares(v[u]);
            wide |= unsafe(q, v[u]);
            sum += u < left ? double(q) : 0.0;
        }
        acc += wide ? squares_wide(p, left) : sum;
    }
    partial_groups(c0, c1, lead, n, [&](int64_t i) { acc = squares_wide(to_float(g[i]), acc); });
    return acc;
}

__device__ __forceinline__ uint32_t share(uint32_t chunks, uint32_t block) {
    return uint32_t(uint64_t(chunks) * block / gridDim.x);
}

__global__ void __launch_bounds__(kThreads, kNormBlocks) grad_norm_kernel(Plan p, uint32_t chunks, double *partials) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t c1 = share(chunks, blockIdx.x + 1);
    uint32_t c = share(chunks, blockIdx.x);
    double acc = 0;
    if (c < c1) {
        for (int i = tensor_of(p, c); c < c1; ++i) {
            const ugdr_x_grad t = p.grads[i];
            const uint32_t first = p.first[i], end = min(p.first[i + 1], c1);
            if (c >= end) continue;  // a tensor without elements
            if (t.grad_type == UGDR_X_TYPE_BF16)
                acc += span_squares<UGDR_X_TYPE_BF16>(t, c - first, end - first);
            else if (t.grad_type == UGDR_X_TYPE_FP16)
                acc += span_squares<UGDR_X_TYPE_FP16>(t, c - first, end - first);
            else
                acc += span_squares<UGDR_X_TYPE_FP32>(t, c - first, end - first);
            c = end;
        }
    }
    acc = block_sum(acc);
    if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

__device__ double partial_sum(const double *partials, int n) {
    double v = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) v += partials[i];
    return block_sum(v);
}

__global__ void __launch_bounds__(kThreads) grad_sum_kernel(const double *partials, int n, double *sum_squares) {
    const double s = partial_sum(partials, n);
    if (threadIdx.x == 0) *sum_squares = s;
}

// The chunks [c0, c1) of one tensor scaled into an output whose whole groups are not aligned: neighbours to
// neighbouring threads.  Out of line, since the other path's registers spilled beside it.
template <typename T, typename O>
__device__ __noinline__ void span_scale_apart(const T *g, O *out, int64_t n, uint32_t lead, uint32_t c0, uint32_t c1,
                                              float coef) {
    for (uint32_t c = c0; c < c1; ++c) {
        const int64_t at = int64_t(c) * kGradChunk - int64_t(lead) + threadIdx.x;
#pragma unroll
        for (int j = 0; j < kGroup; ++j)
            if (at + j * kThreads >= 0 && at + j * kThreads < n)
                from_float(out[at + j * kThreads], to_float(g[at + j * kThreads]) * coef);
    }
}

// The chunks [c0, c1) of one tensor scaled, the last ones first.
template <int IN, int OUT> __device__ void span_scale(const ugdr_x_grad &t, uint32_t c0, uint32_t c1, float coef) {
    using T = typename Element<IN>::type;
    using O = typename Element<OUT>::type;
    constexpr int kUnroll = 4;
    const T *g = static_cast<const T *>(t.grad);
    O *out = static_cast<O *>(t.out);
    const uint32_t lead = lead_of(g);
    const int64_t n = int64_t(t.count);
    const auto one = [&](int64_t i) { from_float(out[i], to_float(g[i]) * coef); };
    if (lead_of(out) != lead) return span_scale_apart(g, out, n, lead, c0, c1, coef);
    const Mine w = my_chunks(c0, c1, lead, n);
    const int64_t begin = int64_t(w.b) * kGradChunk + threadIdx.x * kGroup - int64_t(lead);
    const T *p = g + begin;
    O *o = out + begin;
    int left = int(w.b - w.a);
    for (; left >= kUnroll; left -= kUnroll) {
        Group<T> v[kUnroll];
        p -= kUnroll * kGradChunk;
        o -= kUnroll * kGradChunk;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = load_group(p + u * kGradChunk);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) store_group(o + u * kGradChunk, scaled<O>(v[u], coef));
    }
    if (left > 0) {
        Group<T> v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = load_group(p - min(u + 1, left) * kGradChunk);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (u < left) store_group(o - (u + 1) * kGradChunk, scaled<O>(v[u], coef));
    }
    partial_groups(c0, c1, lead, n, one);
}

// Every block sums the partial sums itself, in one order, so no block waits for another; then it
// scales its run of chunks backwards: what the norm pass read last is what the L2 still holds.
__global__ void __launch_bounds__(kThreads, kScaleBlocks) grad_scale_kernel(Plan p, uint32_t chunks, const double *partials,
                                                                 int npartials, float max_norm, float *norm_out) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the norm kernel's sums are there
    const double norm = sqrt(partial_sum(partials, npartials));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = float(norm);
    const double ratio = double(max_norm) / (norm + 1e-6);
    const float coef = ratio > 1.0 ? 1.f : float(ratio);  // a NaN stays one
    const uint32_t c0 = share(chunks, blockIdx.x);
    uint32_t c = share(chunks, blockIdx.x + 1);
    if (c0 >= c) return;
    for (int i = tensor_of(p, c - 1); c > c0; --i) {
        const ugdr_x_grad t = p.grads[i];
        const uint32_t first = p.first[i], from = max(first, c0);
        if (from >= c) continue;
        const uint32_t a = from - first, b = c - first;
        c = from;
        if (coef == 1.f && t.out == t.grad && t.out_type == t.grad_type) continue;
        if (t.grad_type == UGDR_X_TYPE_BF16) {
            if (t.out_type == UGDR_X_TYPE_BF16)
                span_scale<UGDR_X_TYPE_BF16, UGDR_X_TYPE_BF16>(t, a, b, coef);
            else
                span_scale<UGDR_X_TYPE_BF16, UGDR_X_TYPE_FP32>(t, a, b, coef);
        } else if (t.grad_type == UGDR_X_TYPE_FP16) {
            if (t.out_type == UGDR_X_TYPE_FP16)
                span_scale<UGDR_X_TYPE_FP16, UGDR_X_TYPE_FP16>(t, a, b, coef);
            else
                span_scale<UGDR_X_TYPE_FP16, UGDR_X_TYPE_FP32>(t, a, b, coef);
        } else {
            span_scale<UGDR_X_TYPE_FP32, UGDR_X_TYPE_FP32>(t, a, b, coef);
        }
    }
}

Plan as_plan(const void *plan, int n) {
    const auto *grads = static_cast<const ugdr_x_grad *>(plan);
    return {grads, reinterpret_cast<const uint32_t *>(grads + n), n};
}

// As many blocks as the SMs hold, fewer when there are fewer chunks; at least one, which writes the sum
// or the norm.
int blocks_for(uint64_t chunks, int per_sm) {
    int device = 0, sms = 148;
    cudaGetDevice(&device);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    const uint64_t most = uint64_t(sms) * per_sm < UGDR_X_GRAD_PARTIALS ? uint64_t(sms) * per_sm : UGDR_X_GRAD_PARTIALS;
    return int(chunks < 1 ? 1 : chunks < most ? chunks : most);
}

}  // namespace

int grad_kernels(const KernelRef **out) {
    static const KernelRef refs[] = {
        {"grad_norm_kernel", reinterpret_cast<const void *>(&grad_norm_kernel), kThreads},
        {"grad_sum_kernel", reinterpret_cast<const void *>(&grad_sum_kernel), kThreads},
        {"grad_scale_kernel", reinterpret_cast<const void *>(&grad_scale_kernel), kThreads},
    };
    *out = refs;
    return int(sizeof(refs) / sizeof(refs[0]));
}

int launch_grad_sum_squares(const void *plan, int n, uint64_t chunks, double *partials, double *sum_squares,
                            cudaStream_t s) {
    const int blocks = blocks_for(chunks, kNormBlocks);
    grad_norm_kernel<<<blocks, kThreads, 0, s>>>(as_plan(plan, n), uint32_t(chunks), partials);
    grad_sum_kernel<<<1, kThreads, 0, s>>>(partials, blocks, sum_squares);
    return int(cudaGetLastError());
}

int launch_grad_clip(const void *plan, int n, uint64_t chunks, double *partials, const double *sum_squares,
                     float max_norm, float *norm_out, cudaStream_t s) {
    const int blocks = blocks_for(chunks, kNormBlocks);
    if (sum_squares == nullptr)
        grad_norm_kernel<<<blocks, kThreads, 0, s>>>(as_plan(plan, n), uint32_t(chunks), partials);
    // Launched while the norm kernel runs: its blocks start as those of the norm kernel end.
    cudaLaunchAttribute programmatic{};
    programmatic.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    programmatic.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(blocks_for(chunks, kScaleBlocks)));
    config.blockDim = dim3(kThreads);
    config.stream = s;
    config.attrs = &programmatic;
    config.numAttrs = sum_squares == nullptr ? 1 : 0;
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return int(e);
    return int(cudaLaunchKernelEx(&config, grad_scale_kernel, as_plan(plan, n), uint32_t(chunks),
                                  static_cast<const double *>(sum_squares == nullptr ? partials : sum_squares),
                                  sum_squares == nullptr ? blocks : 1, max_norm, norm_out));
}

}  // namespace ugdr::coll
