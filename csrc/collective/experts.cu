// The experts' gated feed-forward block on rows grouped by expert, forward and backward.
//
//   g = x Wg^T, u = x Wu^T, h = a(g) * u, y = h Wo^T                      (rows of one expert)
//   dh = dy Wo, dg = dh * u * a'(g), du = dh * a(g), dx = dg Wg + du Wu
//   dWg = dg^T x, dWu = du^T x, dWo = dy^T h
//
// Plain tiled kernels: one 64 x 64 tile of a product per block, fp32 accumulation.
#include "collective/operators.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace ugdr::coll {
namespace {

constexpr int kTile = 64, kDepth = 16, kBlock = 256;

__device__ __forceinline__ float load(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// The activation and its derivative.
__device__ __forceinline__ float act(float g, int kind) {
    if (kind == UGDR_X_ACT_SILU) return g / (1.f + expf(-g));
    return 0.5f * g * (1.f + erff(g * 0.70710678f));
}
__device__ __forceinline__ float act_grad(float g, int kind) {
    if (kind == UGDR_X_ACT_SILU) {
        const float s = 1.f / (1.f + expf(-g));
        return s * (1.f + g * (1.f - s));
    }
    return 0.5f * (1.f + erff(g * 0.70710678f)) + g * 0.39894228f * expf(-0.5f * g * g);
}

struct Shape {
    const int32_t *counts;
    unsigned int *status;
    int64_t rows;
    int nexp, hidden, inner, act;
};

struct Rows {
    int expert;
    int64_t first, end;  // rows [first, end), of one expert
};

// Row range of expert e.
__device__ Rows rows_of(const Shape &m, int e) {
    int64_t at = 0;
    for (int i = 0; i < e; ++i) at += max(m.counts[i], 0);
    at = min(at, m.rows);
    return {e, at, min(at + max(m.counts[e], 0), m.rows)};
}

// The `tile`-th piece of at most kTile rows of one expert (expert -1: there are fewer).
__device__ Rows row_tile(const Shape &m, int tile) {
    int64_t at = 0;
    bool bad = false;
    Rows r{-1, 0, 0};
    for (int e = 0; e < m.nexp; ++e) {
        const int64_t n = m.counts[e];
        bad |= n < 0;
        const int64_t end = min(at + max(n, int64_t(0)), m.rows);
        bad |= at + n > m.rows;
        const int tiles = int((end - at + kTile - 1) / kTile);
        if (r.expert < 0 && tile < tiles) {
            r = {e, at + int64_t(tile) * kTile, 0};
            r.end = min(r.first + kTile, end);
        }
        tile -= tiles;
        at = end;
    }
    if (bad) atomicExch(m.status, 2u);
    return r;
}

enum Product { kUp, kDown, kBack, kInput };

// One tile of a product whose rows are the experts' rows.
//   kUp     out = h = a(x Wg^T) * (x Wu^T)  (and gu)     a_rows = x
//   kDown   out = y = h Wo^T                             a_rows = h
//   kBack   out = dgu from dh = dy Wo and gu             a_rows = dy
//   kInput  out = dx = dgu (Wg; Wu)                      a_rows = dgu
template <typename T, Product P>
__global__ void __launch_bounds__(kBlock) rows_kernel(Shape m, const T *a_rows, const T *w, T *out, T *gu) {
    constexpr int kB = P == kUp ? 2 : 1;
    __shared__ float sa[kDepth][kTile + 1], sb[kB][kDepth][kTile + 1];
    __shared__ Rows tile;
    if (threadIdx.x == 0) tile = row_tile(m, blockIdx.y);
    __syncthreads();
    const Rows r = tile;
    if (r.expert < 0) return;
    const int H = m.hidden, F = m.inner;
    const int features = P == kUp || P == kBack ? F : H;
    const int depth = P == kUp || P == kBack ? H : P == kDown ? F : 2 * F;
    const T *we = w + int64_t(r.expert) * H * F * (P == kUp || P == kInput ? 2 : 1);
    const int f0 = blockIdx.x * kTile, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[kB][4][4] = {};
    for (int k0 = 0; k0 < depth; k0 += kDepth) {
        for (int i = threadIdx.x; i < kTile * kDepth; i += kBlock) {
            const int k = k0 + i % kDepth, row = i / kDepth;
            sa[i % kDepth][row] =
                k < depth && r.first + row < r.end ? load(a_rows + (r.first + row) * int64_t(depth) + k) : 0.f;
        }
        for (int b = 0; b < kB; ++b) {
            for (int i = threadIdx.x; i < kTile * kDepth; i += kBlock) {
                // Weights with the depth innermost (kUp, kDown), or the feature.
                const bool inner_depth = P == kUp || P == kDown;
                const int kk = inner_depth ? i % kDepth : i / kTile, ff = inner_depth ? i / kDepth : i % kTile;
                const int k = k0 + kk, f = f0 + ff;
                float v = 0.f;
                if (k < depth && f < features)
                    v = load(we + (inner_depth ? (int64_t(b) * features + f) * depth + k : int64_t(k) * features + f));
                sb[b][kk][ff] = v;
            }
        }
        __syncthreads();
        for (int k = 0; k < kDepth; ++k)
            for (int b = 0; b < kB; ++b)
                for (int i = 0; i < 4; ++i)
                    for (int j = 0; j < 4; ++j) acc[b][i][j] += sa[k][ty * 4 + i] * sb[b][k][tx + 16 * j];
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
        const int64_t row = r.first + ty * 4 + i;
        if (row >= r.end) continue;
        for (int j = 0; j < 4; ++j) {
            const int f = f0 + tx + 16 * j;
            if (f >= features) continue;
            if constexpr (P == kUp) {
                if (gu != nullptr) {
                    store(gu + row * 2 * F + f, acc[0][i][j]);
                    store(gu + row * 2 * F + F + f, acc[kB - 1][i][j]);
                }
                store(out + row * F + f, act(acc[0][i][j], m.act) * acc[kB - 1][i][j]);
            } else if constexpr (P == kBack) {
                const float g = load(gu + row * 2 * F + f), u = load(gu + row * 2 * F + F + f);
                store(out + row * 2 * F + f, acc[0][i][j] * u * act_grad(g, m.act));
                store(out + row * 2 * F + F + f, acc[0][i][j] * act(g, m.act));
            } else {
                store(out + row * features + f, acc[0][i][j]);
            }
        }
    }
}

// One tile of an expert's weight gradient: out[m][n] = sum over its rows of a[row][m] * b[row][n].
template <typename T>
__global__ void __launch_bounds__(kBlock) weights_kernel(Shape m, const T *a, int am, const T *b, int bn, T *out) {
    __shared__ float sa[kDepth][kTile], sb[kDepth][kTile];
    __shared__ Rows range;
    if (threadIdx.x == 0) range = rows_of(m, blockIdx.z);
    __syncthreads();
    const Rows r = range;
    const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int64_t r0 = r.first; r0 < r.end; r0 += kDepth) {
        for (int i = threadIdx.x; i < kTile * kDepth; i += kBlock) {
            const int64_t row = r0 + i / kTile;
            const int c = i % kTile;
            sa[i / kTile][c] = row < r.end && m0 + c < am ? load(a + row * am + m0 + c) : 0.f;
            sb[i / kTile][c] = row < r.end && n0 + c < bn ? load(b + row * bn + n0 + c) : 0.f;
        }
        __syncthreads();
        for (int k = 0; k < kDepth; ++k)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] += sa[k][ty * 4 + i] * sb[k][tx + 16 * j];
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int mm = m0 + ty * 4 + i, nn = n0 + tx + 16 * j;
            if (mm < am && nn < bn) store(out + (int64_t(r.expert) * am + mm) * bn + nn, acc[i][j]);
        }
}

Shape shape_of(const ugdr_x_experts &m) {
    return {m.counts, m.status, int64_t(m.rows), m.nexp, m.hidden, m.inner, m.act};
}

unsigned tiles(int64_t n) { return unsigned((n + kTile - 1) / kTile); }

template <typename T>
int forward(const ugdr_x_experts &m, const void *x, void *y, void *h, void *gu, cudaStream_t s) {
    const Shape sh = shape_of(m);
    const unsigned row_tiles = tiles(int64_t(m.rows)) + unsigned(m.nexp);
    rows_kernel<T, kUp><<<dim3(tiles(m.inner), row_tiles), kBlock, 0, s>>>(
        sh, static_cast<const T *>(x), static_cast<const T *>(m.w_in), static_cast<T *>(h), static_cast<T *>(gu));
    rows_kernel<T, kDown><<<dim3(tiles(m.hidden), row_tiles), kBlock, 0, s>>>(
        sh, static_cast<const T *>(h), static_cast<const T *>(m.w_out), static_cast<T *>(y), nullptr);
    return int(cudaGetLastError());
}

template <typename T>
int backward(const ugdr_x_experts &m, const void *dy, const void *x, const void *h, const void *gu, void *dgu,
             void *dx, void *dw_in, void *dw_out, cudaStream_t s) {
    const Shape sh = shape_of(m);
    const unsigned row_tiles = tiles(int64_t(m.rows)) + unsigned(m.nexp), e = unsigned(m.nexp);
    rows_kernel<T, kBack><<<dim3(tiles(m.inner), row_tiles), kBlock, 0, s>>>(
        sh, static_cast<const T *>(dy), static_cast<const T *>(m.w_out), static_cast<T *>(dgu),
        const_cast<T *>(static_cast<const T *>(gu)));
    weights_kernel<T><<<dim3(tiles(m.inner), tiles(m.hidden), e), kBlock, 0, s>>>(
        sh, static_cast<const T *>(dy), m.hidden, static_cast<const T *>(h), m.inner, static_cast<T *>(dw_out));
    weights_kernel<T><<<dim3(tiles(m.hidden), tiles(2 * int64_t(m.inner)), e), kBlock, 0, s>>>(
        sh, static_cast<const T *>(dgu), 2 * m.inner, static_cast<const T *>(x), m.hidden, static_cast<T *>(dw_in));
    // Last, so that dx may be dy or x itself.
    rows_kernel<T, kInput><<<dim3(tiles(m.hidden), row_tiles), kBlock, 0, s>>>(
        sh, static_cast<const T *>(dgu), static_cast<const T *>(m.w_in), static_cast<T *>(dx), nullptr);
    return int(cudaGetLastError());
}

}  // namespace

int launch_expert_ffn(const ugdr_x_experts &m, const void *x, void *y, void *h, void *gu, cudaStream_t s) {
    return m.type == UGDR_X_TYPE_BF16 ? forward<__nv_bfloat16>(m, x, y, h, gu, s) : forward<__half>(m, x, y, h, gu, s);
}

int launch_expert_ffn_backward(const ugdr_x_experts &m, const void *dy, const void *x, const void *h, const void *gu,
                               void *dgu, void *dx, void *dw_in, void *dw_out, cudaStream_t s) {
    return m.type == UGDR_X_TYPE_BF16 ? backward<__nv_bfloat16>(m, dy, x, h, gu, dgu, dx, dw_in, dw_out, s)
                                      : backward<__half>(m, dy, x, h, gu, dgu, dx, dw_in, dw_out, s);
}

}  // namespace ugdr::coll
