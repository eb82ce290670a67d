// The experts' gated feed-forward block on rows grouped by expert, forward and backward.
//
//   g = x Wg^T, u = x Wu^T, h = a(g) * u, y = h Wo^T                      (rows of one expert)
//   dh = dy Wo, dg = dh * u * a'(g), du = dh * a(g), dx = dg Wg + du Wu
//   dWg = dg^T x, dWu = du^T x, dWo = dy^T h
//
// Six grouped matrix products, one persistent kernel template: with some hundred rows per expert
// they are bound by the tensor cores, with a few rows by reading the weights.
//
// * A pair of CTAs (a cluster of 2 on one TPC) works on one tile with tcgen05.mma.cta_group::2.
//   The 256 rows of the tile's M are weight rows ("features": 128 per CTA), and its N, 32 to 256 in
//   steps of 32, are rows of one expert.  So the ragged dimension is the one that the instruction
//   takes in small steps: a group of 20 rows costs an N of 32, not a tile of 128 or 256, and the
//   same kernel serves single tokens.  Each CTA loads its 128 features and half of the N rows:
//   32 KB per 64-deep step at N = 256, which the L2 can deliver (64 B/clk per SM) while the
//   pair's tensor cores take 512 clocks for it.
// * The weight gradients sum over an expert's rows instead: M and N are the two weight dimensions.
//   Rows that follow the group in the last 64-deep step must not count, whatever they hold: a
//   warp overwrites them with zeros in shared memory, up to the 16 that one instruction takes.
// * Warp 0 issues the TMA loads into a ring of stages, warp 1 of the leading CTA the matrix
//   instructions, warp 2 clears tails, warps 4 to 11 move finished accumulators out of TMEM, where
//   two tiles' accumulators fit, so that they overlap the next tile's products.
// * Every pair walks the tile list by itself (tile t, t + pairs, ...): the row counts are read on
//   the device, and no CTA waits for another outside its pair.
//
// Roundings to the 16-bit type: h, dg and du, once each, because they are operands of the next
// product.  The projections g and u that the backward pass reads are kept in fp32: in 16 bits they
// made dx and dw_in 1.8 times as far off as one rounding of the result does, against 1.4 times now.
//
// Measured on a B200, 8 experts of 2,048 rows, 7168 x 2048, bf16: the six products take 638, 305
// (y), 324, 317 (dw_out), 633 (dw_in) and 618 us (dx), 1.49 to 1.58 PFLOP/s at the 1.37 to 1.45 GHz
// that the power limit leaves, with the tensor pipes 87 to 93 % busy over the whole of the kernels.  One
// row for each of 32 experts reads their 2.8 GB at 6.8 TB/s.  In between, a step takes the ring's
// latency, 0.26 us with few rows and 0.29 us with 256.
//
// Every wait is bounded (ugdr_x_set_expert_wait_ns): one that runs out sets *status and ends the kernel.
#include "collective/operators.hpp"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

namespace ugdr::coll {
namespace {

constexpr int kThreads = 384;       // 12 warps: 4 that feed the tensor cores, 8 for the epilogue
constexpr int kCheckThreads = 256;
constexpr int kHalf = 128;          // features of a tile per CTA: the lanes of TMEM
constexpr int kPairFeatures = 256;
constexpr int kMaxN = 256;
constexpr int kStepN = 32;
constexpr int kDepth = 64;          // elements per stage along the summed dimension: 128 bytes
constexpr int kBoxes = 4;           // TMA boxes of 128, 64, 32 and 16 rows
constexpr int kMaxStages = 10;
constexpr int kChunk = 16;          // rows (or columns of a gradient) that an epilogue group moves at once
constexpr int kMaxOrdered = 512;
constexpr int kBand = 8;            // row tiles that run through all features before the next
constexpr uint32_t kOperandBytes = kHalf * kDepth * 2;  // one CTA's half of A, or of B for the largest N
constexpr uint32_t kRingBytes = 6 * 2 * kOperandBytes;  // 6 stages for the largest N, 10 for the smallest
constexpr int kStagingRow = kHalf + 4;                  // floats; the 4 keep 16-byte reads apart
constexpr uint32_t kStagingBytes = kChunk * kStagingRow * 4;

enum Product { kUp, kDown, kBack, kInput, kGradOut, kGradIn };
template <Product P> constexpr bool kWeightGrad = P == kGradOut || P == kGradIn;
// Whether A's features lie next to each other in memory (else its summed dimension does).
template <Product P> constexpr bool kFeaturesInner = P != kUp && P != kDown;

struct Shape {
    const int32_t *counts;
    unsigned int *status;
    uint64_t wait_ns;  // bound of every wait
    int rows, nexp, hidden, inner, act;
    int stages;            // of the ring, and the bytes of one: B's part is what the rows can need
    uint32_t stage_bytes;
};

struct Shared {
    alignas(8) uint64_t full[kMaxStages], empty[kMaxStages], tail[kMaxStages], tmem_full[2], tmem_empty[2];
    uint32_t tmem;
    int aborted;
    long long scan[kThreads / 32];
    uint16_t order[kMaxOrdered];  // weight gradients: the experts, those with the most rows first
};
constexpr size_t shared_bytes(int nexp) {
    return 1024 + kRingBytes + 2 * kStagingBytes + sizeof(Shared) + (size_t(nexp) + 1) * 4;
}
static_assert(shared_bytes(UGDR_X_EXPERTS_MAX) <= 232448, "227 KB of shared memory per CTA");

// ---- PTX ---------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint64_t gtime() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ void store_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
// The same shared address in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_cluster(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\n"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
                 "selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}
// Waits until the barrier's phase of `parity` is over.  False: the wait, or another of this CTA,
// ran out, and the caller gives up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, Shared &sh, const Shape &m) {
    uint64_t since = 0;
    for (uint32_t spins = 1; !mbar_try(bar, parity); ++spins) {
        if (spins % 64 != 0) continue;
        if (*reinterpret_cast<volatile int *>(&sh.aborted)) return false;
        const uint64_t now = gtime();
        if (since == 0) since = now;
        if (now - since > m.wait_ns) {
            *reinterpret_cast<volatile int *>(&sh.aborted) = 1;
            atomicExch(m.status, 1u);
            return false;
        }
    }
    return true;
}

// TMA loads into this CTA; the bytes are counted by `bar`, here or in the pair's other CTA.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2,
                                         int c3) {
    asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
}

// Operand descriptors for 128-byte swizzled tiles (rows of 128 bytes, atoms of 8 rows).  With the
// summed dimension inner, 8 features to an atom and 1024 bytes to the next 8.  With the features
// inner, 64 of them to an atom of 8 summed positions, 1024 bytes to the next 8 positions and one
// tile of 64 x 128 bytes to the next 64 features.  The lower half begins with the address in units of
// 16 bytes, to which offsets can be added.  (Above its 18 bits a shared address names the CTA.)
template <bool FEATURES_INNER> __device__ __forceinline__ uint32_t operand(uint32_t addr) {
    constexpr uint32_t kLeading = FEATURES_INNER ? kDepth * 128 / 16 : 1;
    return (addr >> 4 & 0x3fff) | kLeading << 16;
}
constexpr uint32_t kOperandUpper = 1024 / 16 | 1u << 14 | 2u << 29;  // stride, version, swizzle
// From one instruction's 16 summed positions to the next's.
template <bool FEATURES_INNER> constexpr uint32_t kOperandStep = FEATURES_INNER ? 16 * 128 / 16 : 16 * 2 / 16;

__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.u32 p, %4, 0;\n"
                 "mov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\n"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n}" ::"r"(d),
                 "r"(a), "r"(b), "r"(idesc), "r"(uint32_t(add)), "r"(kOperandUpper)
                 : "memory");
}
// Arrives on `bar` of both CTAs of the pair, `mask` in the cluster, once the instructions issued
// before are done.
__device__ __forceinline__ void mma_commit(uint32_t bar, uint16_t mask) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     bar),
                 "h"(mask)
                 : "memory");
}
// Programmatic launches: the next kernel of the stream may begin its set-up, and this one waits here
// until the kernels before it are over and their writes visible.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 16 columns of this warp's 32 TMEM lanes: v[j] is column j of lane threadIdx.x % 32, once
// tmem_wait() is over.
__device__ __forceinline__ void tmem_request(uint32_t addr, uint32_t (&r)[kChunk]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15])
                 : "r"(addr)
                 : "memory");
}
// The registers pass through, so that no use of them can move before the wait.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[kChunk]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[8]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr)
                 : "memory");
}
// The four warps of an epilogue group, 0 or 1, meet.
__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
// Whether all of them say so: one that gives up takes the others along.
__device__ __forceinline__ bool group_all(int group, bool ok) {
    uint32_t all;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\n"
                 "bar.red.and.pred q, %2, 128, p;\nselp.u32 %0, 1, 0, q;\n}"
                 : "=r"(all)
                 : "r"(uint32_t(ok)), "r"(1 + group)
                 : "memory");
    return all != 0;
}

// ---- tiles -------------------------------------------------------------------------------------

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

struct Tile {
    int expert;
    int feature;  // first of the pair's features
    int part;     // kGradIn: 0 the gate's, 1 the up projection's weights
    int first;    // rows products: the tile's first row.  Weight gradients: the group's
    int rows;     // likewise, of the tile or the group
    int column;   // weight gradients: first of the N
};

// Features of a tile of the pair: with kUp 128 of the gate and the same 128 of the up projection.
template <Product P> constexpr int kTileFeatures = P == kUp ? kPairFeatures / 2 : kPairFeatures;

template <Product P> __device__ __forceinline__ int steps_of(const Shape &m, int rows) {
    if (kWeightGrad<P>) return ceil_div(rows, kDepth);
    if (P == kInput) return 2 * ceil_div(m.inner, kDepth);
    return ceil_div(P == kDown ? m.inner : m.hidden, kDepth);
}

// Walks a worker's share of the tile list: one tile of every round.
//
// An expert's rows are cut into as few tiles as kMaxN allows, of about the same size, all but the last a
// multiple of kStepN.  Shared memory, 128 bytes per clock, sets the price of a tile of N rows: a step
// writes 128 + N / 2 clocks' worth and its four instructions read 4 (32 + N / 8), together 256 + N,
// beside 2 N for the products.  So N = 256 is in balance, and 32 experts of 288 rows, as 160 + 128, take
// 1.44 times as long as of 256 (832 and 577 us, 7168 x 2048).  (Tiles of up to 512 rows, whose features
// are loaded once and read by two instructions, gained 4 % from 264 to 320 rows and cost 3 to 6 %
// elsewhere, for accumulators that cannot take turns as a whole.)
//
// A weight gradient's tiles take as long as their expert has rows, so the experts with the most rows
// come first, and the pairs take turns forwards and backwards: over 28,813 rows of 17 uneven experts,
// 1968 x 680, dw_out and dw_in took 161 and 193 us in the experts' order, and 144 and 178 this way.
// (An expert with most of the rows still bounds them by one of its tiles.)
template <Product P> struct Tiles {
    const int *first;  // first row of each expert's group, and the end of the last
    const uint16_t *order;
    int nexp, mtiles, mparts, ntiles, worker, workers;
    int turn = 0, at = -1, expert = 0, base = 0, size = 0, n = 0, columns = 0, per = 0;

    // `worker` of those that share the list.
    __device__ Tiles(const Shape &m, const int *first_, const uint16_t *order_, int worker_, int workers_)
        : first(first_), order(order_), nexp(m.nexp), worker(worker_), workers(workers_) {
        const int features = P == kUp || P == kBack || P == kGradIn ? m.inner : m.hidden;
        mparts = ceil_div(features, kTileFeatures<P>);
        mtiles = P == kGradIn ? 2 * mparts : mparts;
        ntiles = P == kGradOut ? ceil_div(m.inner, kMaxN) : P == kGradIn ? ceil_div(m.hidden, kMaxN) : 0;
    }
    __device__ __forceinline__ bool next(Tile &out) {
        const int t = turn * workers + (kWeightGrad<P> && (turn & 1) ? workers - 1 - worker : worker);
        ++turn;
        while (t >= base + size) {
            if (++at >= nexp) return false;
            expert = kWeightGrad<P> && nexp <= kMaxOrdered ? order[at] : at;
            base += size;
            n = first[expert + 1] - first[expert];
            columns = kWeightGrad<P> ? ntiles : ceil_div(n, kMaxN);
            if (columns > 0) per = ceil_div(ceil_div(n, columns), kStepN) * kStepN;
            size = mtiles * columns;
        }
        // Bands of kBand N tiles; inside, all N tiles of one feature tile before the next, so that
        // pairs that run together share weights and rows in the L2.
        int mtile = t - base, ntile = 0;
        if (columns > 1) {
            const int band = columns <= kBand ? 0 : mtile / (kBand * mtiles), width = min(kBand, columns - band * kBand);
            const int in_band = mtile - band * kBand * mtiles;
            mtile = in_band / width;
            ntile = band * kBand + in_band - mtile * width;
        }
        out.expert = expert;
        out.part = P == kGradIn ? mtile >= mparts : 0;
        out.feature = (mtile - out.part * mparts) * kTileFeatures<P>;
        if (kWeightGrad<P>) {
            out.first = first[expert];
            out.rows = n;
            out.column = ntile * kMaxN;
        } else {
            out.first = first[expert] + ntile * per;
            out.rows = min(per, n - ntile * per);
            out.column = 0;
        }
        return true;
    }
};

// The first kernel of a call (kUp, kBack) waits for the kernels before the call.  The others may start
// while their predecessor in the call runs, and load early what that one does not write.
template <Product P> constexpr bool kFirstOfCall = P == kUp || P == kBack;
template <Product P> constexpr bool kEarlyA = P == kDown || P == kInput || P == kGradOut;
template <Product P> constexpr bool kEarlyB = P == kGradIn || P == kGradOut;

// First rows of the groups into first[0 .. nexp]: a scan over the block's threads.
__device__ void scan_counts(const Shape &m, Shared &sh, int *first) {
    const int per = ceil_div(m.nexp, kThreads), lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int e0 = min(m.nexp, int(threadIdx.x) * per), e1 = min(m.nexp, e0 + per);
    long long own = 0;
    bool bad = false;
    for (int e = e0; e < e1; ++e) {
        const int c = m.counts[e];
        bad |= c < 0;
        own += first[e] = max(c, 0);
    }
    long long upto = own;
    for (int o = 1; o < 32; o *= 2) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += sh.scan[w];
    long long at = upto - own;
    for (int e = e0; e < e1; ++e) {
        const int c = first[e];
        first[e] = int(min(at, (long long)m.rows));
        at += c;
    }
    if (threadIdx.x == kThreads - 1) {
        first[m.nexp] = int(min(upto, (long long)m.rows));
        bad |= upto > m.rows;
    }
    if (bad && blockIdx.x == 0) atomicExch(m.status, 2u);
}

// The experts by their rows, the most first, equal ones in their order.
__device__ void order_experts(const Shape &m, const int *first, uint16_t *order) {
    for (int e = threadIdx.x; e < m.nexp; e += kThreads) {
        const int n = first[e + 1] - first[e];
        int before = 0;
        for (int o = 0; o < m.nexp; ++o) {
            const int other = first[o + 1] - first[o];
            before += other > n || (other == n && o < e);
        }
        order[before] = uint16_t(e);
    }
}

// ---- elements ----------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float *v) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
}
// A whole 32-byte sector of global memory at once: halves of one, stored one after the other, are two
// writes for the L2.
__device__ __forceinline__ void store8(float *p, const float *v) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                 "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}
template <typename T> __device__ __forceinline__ void store16(T *p, const float *v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(pack2(v[0], v[1], T())),
                 "r"(pack2(v[2], v[3], T())), "r"(pack2(v[4], v[5], T())), "r"(pack2(v[6], v[7], T())),
                 "r"(pack2(v[8], v[9], T())), "r"(pack2(v[10], v[11], T())), "r"(pack2(v[12], v[13], T())),
                 "r"(pack2(v[14], v[15], T()))
                 : "memory");
}
__device__ __forceinline__ void load8_global(const float *p, float *v) {
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void load8(const float *p, float *v) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

__device__ __forceinline__ void add8(const float *p, float (&v)[8]) {
    float w[8];
    load8(p, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += w[j];
}

// a(g) and a'(g).  silu's exponential and quotient are the approximate ones: together off by less
// than (|g| + 8) 2^-23 of the value, which goes under in the rounding to 16 bits (2^-12 of it at best).
// 1 + exp(-g) is between 1 and infinity.  From 2^126 on, at g < -87.3, the quotient is 0: it is below
// 2^-126 there, and a(g) and a'(g) below 2^-119.
struct Act {
    float a, da;
};
__device__ __forceinline__ Act silu(float g) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    return {g * s, s * (1.f + g * (1.f - s))};
}
// gelu: g Phi(g), with Phi(-|g|) = exp(-g^2 / 2) t q(t), t = 1 / (1 + 0.3 |g|), so that the lower tail keeps
// its relative precision, which 1 + erf does not (off by 4 % at g = -5, and 0 from -5.5 on).  q is a least
// squares fit, reweighted towards the smallest largest relative error (1.5e-7), to
// exp(g^2 / 2) Phi(-|g|) / t at 2000 Chebyshev nodes over |g| <= 14.  With the approximate exponential,
// which the derivative needs too, and quotient, Phi is off by less than (g^2 + 12) 2^-23 of its value, down
// to g = -13, where it leaves fp32's normal numbers.
__device__ __forceinline__ Act gelu(float g) {
    const float t = __fdividef(1.f, 1.f + 0.3f * fabsf(g)), e = __expf(-0.5f * g * g);
    float q = 0.0356748775f;
    q = fmaf(q, t, -0.157203496f);
    q = fmaf(q, t, 0.206354201f);
    q = fmaf(q, t, -0.0536842458f);
    q = fmaf(q, t, 0.128561929f);
    q = fmaf(q, t, 0.0999134108f);
    q = fmaf(q, t, 0.120753966f);
    q = fmaf(q, t, 0.119629301f);
    q *= t * e;
    const float p = g > 0.f ? 1.f - q : q;
    return {g * p, p + g * 0.39894228f * e};
}

// ---- the kernel --------------------------------------------------------------------------------

// B's boxes: half of the N rows, rounded up to 32, is a sum of at most two of 128, 64 and 32, and
// the smallest half has one of 16.  With boxes of 16 rows only, 224 rows per expert took longer than
// 256; with 32 at least, single rows per expert read their weights at 5.6 TB/s instead of 6.3.
struct Maps {
    CUtensorMap a, b[kBoxes];
};

// A place in the ring of stages: its shared addresses, kept rather than computed, because the two
// threads that walk the ring are what short steps wait for.
struct Ring {
    uint32_t stage, bar;  // the stage, and an offset into each array of barriers
    uint32_t parity;
    __device__ __forceinline__ void next(const Shape &m, uint32_t stage0) {
        stage += m.stage_bytes;
        bar += 8;
        if (bar == uint32_t(m.stages) * 8) stage = stage0, bar = 0, parity ^= 1;
    }
};

// The thread that issues a CTA's loads.  Its loop is what a stage of few rows takes longest for, so
// it is kept short: a loop of its own for every set of boxes, whose maps are then known.  (Picking
// the map by an index made single rows per expert take 1.3 times as long.)  And what is not a loop
// over the steps is there once only: instructions that a kernel meets first are read from memory.
template <Product P> struct Loader {
    const Maps &maps;
    const Shape &m;
    Shared &sh;
    const uint32_t stage0, empty, full, tail, rank;  // barriers: `full` in the leading CTA
    const int part_steps;                            // kInput: steps through the gate's half of the depth
    Ring at;
    bool started = false;

    __device__ __forceinline__ bool wait() { return mbar_wait(empty + at.bar, at.parity, sh, m); }

    // Steps [k0, k1) of a tile.
    __device__ __forceinline__ bool load_tile(const Tile &t, int k0, int k1) {
        const int half = kWeightGrad<P> ? kHalf : ceil_div(t.rows, kStepN) * kStepN / 2;
        const int load = half == 16 ? 16 : ceil_div(half, 32) * 32;  // rows of B from this CTA's half on
        if (!started) {
            k0 = load_first(t, half, load, k0, k1);
            started = true;
        }
        if (kWeightGrad<P> || load == 128) return load_steps<128>(t, half, k0, k1);
        return load == 96   ? load_steps<96>(t, half, k0, k1)
               : load == 64 ? load_steps<64>(t, half, k0, k1)
               : load == 32 ? load_steps<32>(t, half, k0, k1)
                            : load_steps<16>(t, half, k0, k1);
    }

    // The kernel's first steps, as many as there are stages: what does not come from the kernel before,
    // then, once that is over, the rest.  Returns the first step that is left.
    __device__ __forceinline__ int load_first(const Tile &t, int half, int load, int k0, int k1) {
        const int filled = min(k1, k0 + m.stages);
        const Ring begin = at;
        for (int k = k0; k < filled; ++k, at.next(m, stage0)) {
            const uint32_t bar = barrier(t, k);
            mbar_expect_cluster(bar, kOperandBytes + uint32_t(load) * kDepth * 2);
            if (kEarlyA<P>) load_a(t, k, bar);
            if (kEarlyB<P>) load_b(load, t, half, k, bar);
        }
        if (!kEarlyA<P> || !kEarlyB<P>) {
            wait_previous();
            at = begin;
            for (int k = k0; k < filled; ++k, at.next(m, stage0)) {
                const uint32_t bar = barrier(t, k);
                if (!kEarlyA<P>) load_a(t, k, bar);
                if (!kEarlyB<P>) load_b(load, t, half, k, bar);
            }
        }
        return filled;
    }

    template <int LOAD> __device__ __forceinline__ bool load_steps(const Tile &t, int half, int k0, int k1) {
        for (int k = k0; k < k1; ++k, at.next(m, stage0)) {
            if (!wait()) return false;
            const uint32_t bar = barrier(t, k);
            mbar_expect_cluster(bar, kOperandBytes + uint32_t(LOAD) * kDepth * 2);
            load_a(t, k, bar);
            load_b(LOAD, t, half, k, bar);
        }
        return true;
    }

    // Where a step's bytes are counted.  A last step that reaches past the group goes to the warp that
    // clears its tail.
    __device__ __forceinline__ uint32_t barrier(const Tile &t, int k) const {
        return (kWeightGrad<P> && (k + 1) * kDepth > t.rows ? tail : full) + at.bar;
    }

    __device__ __forceinline__ void load_a(const Tile &t, int k, uint32_t bar) const {
        const int feature = t.feature + int(rank) * (kTileFeatures<P> / 2), depth = k * kDepth;
        if constexpr (P == kUp) {
            tma_load(at.stage, &maps.a, bar, depth, feature, 0, t.expert);
        } else if constexpr (P == kDown) {
            tma_load(at.stage, &maps.a, bar, depth, feature, t.expert);
        } else {
            const int part = P == kInput ? k >= part_steps : 0;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t dst = at.stage + uint32_t(c) * kOperandBytes / 2;
                const int f = feature + c * 64;
                if constexpr (P == kBack)
                    tma_load(dst, &maps.a, bar, f, depth, t.expert);
                else if constexpr (P == kInput)
                    tma_load(dst, &maps.a, bar, f, depth - part * part_steps * kDepth, part, t.expert);
                else if constexpr (P == kGradOut)
                    tma_load(dst, &maps.a, bar, f, t.first + depth);
                else
                    tma_load(dst, &maps.a, bar, f, t.part, t.first + depth);
            }
        }
    }

    __device__ __forceinline__ void load_b(int load, const Tile &t, int half, int k, uint32_t bar) const {
        const uint32_t b = at.stage + kOperandBytes;
        const int depth = k * kDepth;
        if constexpr (kWeightGrad<P>) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
                tma_load(b + uint32_t(c) * kOperandBytes / 2, &maps.b[0], bar, t.column + int(rank) * kHalf + c * 64,
                         t.first + depth);
        } else {
            const int row = t.first + int(rank) * half, part = P == kInput ? k >= part_steps : 0;
            int r = 0;
#pragma unroll
            for (int i = 0; i < kBoxes; ++i) {
                constexpr int kFirst = kHalf;
                if ((load & kFirst >> i) == 0) continue;
                if constexpr (P == kInput)
                    tma_load(b + uint32_t(r) * kDepth * 2, &maps.b[i], bar, depth - part * part_steps * kDepth, part,
                             row + r);
                else
                    tma_load(b + uint32_t(r) * kDepth * 2, &maps.b[i], bar, depth, row + r);
                r += kFirst >> i;
            }
        }
    }
};

// The thread that issues a pair's matrix instructions.
template <typename T, Product P> struct Issuer {
    static constexpr bool kInnerA = kFeaturesInner<P>, kInnerB = kWeightGrad<P>;
    const Shape &m;
    Shared &sh;
    const uint32_t stage0, full, empty;
    const uint16_t mask;
    Ring at;

    __device__ __forceinline__ bool wait() {
        if (!mbar_wait(full + at.bar, at.parity, sh, m)) return false;
        fence_after();
        return true;
    }
    // The products of the current stage, `parts` times 16 deep.
    __device__ __forceinline__ void multiply(uint32_t d, uint32_t idesc, int parts, bool add) const {
        const uint32_t a = operand<kInnerA>(at.stage), b = operand<kInnerB>(at.stage + kOperandBytes);
#pragma unroll
        for (int i = 0; i < kDepth / 16; ++i)
            if (i < parts) mma(d, a + i * kOperandStep<kInnerA>, b + i * kOperandStep<kInnerB>, idesc, add || i > 0);
    }
    // The instruction: its types, layouts and N.
    static __device__ __forceinline__ uint32_t instruction(int rows) {
        constexpr uint32_t kType = std::is_same_v<T, __nv_bfloat16> ? 1 : 0;
        return 1u << 4 | kType << 7 | kType << 10 | uint32_t(kInnerA) << 15 | uint32_t(kInnerB) << 16 |
               uint32_t(kPairFeatures / 16) << 24 | uint32_t(ceil_div(rows, kStepN) * (kStepN / 8)) << 17;
    }

    // Steps [k0, k1) of a tile into the accumulator at d.
    __device__ __forceinline__ bool run(const Tile &t, uint32_t d, int k0, int k1) {
        const uint32_t idesc = instruction(kWeightGrad<P> ? kMaxN : t.rows);
        for (int k = k0; k < k1; ++k, at.next(m, stage0)) {
            if (!wait()) return false;
            int parts = kDepth / 16;
            if (kWeightGrad<P>) parts = min(parts, ceil_div(t.rows - k * kDepth, 16));
            multiply(d, idesc, parts, k > k0);
            mma_commit(empty + at.bar, mask);
        }
        return true;
    }
};

// What a row product does with 8 of a row's features: `a` are their sums (kUp: the gate's, and `b`
// the up projection's), `g` and `u` with kBack the projections that the forward pass kept.
template <typename T, Product P>
__device__ __forceinline__ void finish(const Shape &m, T *out, float *gu, int64_t row, int f, const float (&a)[8],
                                       const float (&b)[8], const float (&g)[8], const float (&u)[8]) {
    if constexpr (P == kUp) {
        if (gu != nullptr) {
            store8(gu + row * 2 * m.inner + f, a);
            store8(gu + row * 2 * m.inner + m.inner + f, b);
        }
        float h[8];
        if (m.act == UGDR_X_ACT_SILU) {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = silu(a[j]).a * b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = gelu(a[j]).a * b[j];
        }
        store8(out + row * m.inner + f, h);
    } else if constexpr (P == kBack) {
        float dg[8], du[8];
        if (m.act == UGDR_X_ACT_SILU) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const Act s = silu(g[j]);
                dg[j] = a[j] * u[j] * s.da;
                du[j] = a[j] * s.a;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const Act s = gelu(g[j]);
                dg[j] = a[j] * u[j] * s.da;
                du[j] = a[j] * s.a;
            }
        }
        store8(out + row * 2 * m.inner + f, dg);
        store8(out + row * 2 * m.inner + m.inner + f, du);
    } else {
        store8(out + row * m.hidden + f, a);
    }
}

// A kernel's shared memory, barriers, TMEM and row counts, set up by all threads of a cluster.
struct Setup {
    uint8_t *ring;
    float *staging;
    Shared *sh;
    int *first;
    uint32_t stage0, rank, leader;  // rank: 0 or 1 in the pair, whose first CTA is `leader` of the cluster
};

template <Product P> __device__ __forceinline__ Setup set_up(const Maps &maps, const Shape &m) {
    extern __shared__ uint8_t raw[];
    Setup k;
    k.ring = raw + (0u - smem_addr(raw)) % 1024;  // an offset, not a rounded pointer: accesses stay known to be shared
    k.staging = reinterpret_cast<float *>(k.ring + kRingBytes);
    k.sh = reinterpret_cast<Shared *>(reinterpret_cast<uint8_t *>(k.staging) + 2 * kStagingBytes);
    k.first = reinterpret_cast<int *>(k.sh + 1);
    k.stage0 = smem_addr(k.ring);
    k.rank = cta_rank() & 1;
    k.leader = cta_rank() - k.rank;
    Shared &sh = *k.sh;
    if (threadIdx.x < kMaxStages) {
        mbar_init(smem_addr(&sh.full[threadIdx.x]), 2);  // both CTAs' loads, counted in the leading CTA
        mbar_init(smem_addr(&sh.empty[threadIdx.x]), 1);
        mbar_init(smem_addr(&sh.tail[threadIdx.x]), 1);
        if (threadIdx.x < 2) {
            mbar_init(smem_addr(&sh.tmem_full[threadIdx.x]), 1);
            mbar_init(smem_addr(&sh.tmem_empty[threadIdx.x]), 16);  // 8 epilogue warps of each CTA
        }
        if (threadIdx.x == 0) sh.aborted = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x / 32 == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sh.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
    fence_before();
    cluster_sync();
    fence_after();
    if (kFirstOfCall<P>) wait_previous();
    launch_next();  // only now, so that the next kernel of the call finds the call's inputs complete
    scan_counts(m, sh, k.first);
    __syncthreads();
    if (kWeightGrad<P> && m.nexp <= kMaxOrdered) {
        order_experts(m, k.first, sh.order);
        __syncthreads();
    }
    return k;
}

// The end of a kernel, for all threads of a cluster.
__device__ __forceinline__ void tear_down(const Setup &k) {
    __syncthreads();
    if (k.sh->aborted) {  // loads and instructions that are still under way end within this time
        for (const uint64_t since = gtime(); gtime() - since < 2'000'000;) __nanosleep(1000);
        __syncwarp();
    }
    fence_before();
    cluster_sync();
    if (threadIdx.x / 32 == 2) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(k.sh->tmem) : "memory");
    }
}

template <Product P> __device__ __forceinline__ Loader<P> loader_of(const Maps &maps, const Shape &m, const Setup &k) {
    Shared &sh = *k.sh;
    return {maps,
            m,
            sh,
            k.stage0,
            smem_addr(sh.empty),
            map_to(smem_addr(sh.full), k.leader),
            map_to(smem_addr(sh.tail), k.leader + k.rank),
            k.rank,
            ceil_div(m.inner, kDepth),
            {k.stage0, 0, 1}};  // parity 1: every stage is free
}
template <typename T, Product P> __device__ __forceinline__ Issuer<T, P> issuer_of(const Shape &m, const Setup &k) {
    return {m, *k.sh, k.stage0, smem_addr(k.sh->full), smem_addr(k.sh->empty), uint16_t(3u << k.leader),
            {k.stage0, 0, 0}};
}

// The warp that clears tails: rows behind a group in its last step, up to the next 16, become zeros.
struct TailClearer {
    const Shape &m;
    Shared &sh;
    const Setup &k;
    uint32_t it = 0, phases = 0;  // steps so far, and the phase of each stage's barrier for tails

    // After steps [k0, k1) of a tile of a group of `rows`.
    __device__ __forceinline__ bool clear(int rows, int k0, int k1) {
        const int last = rows % kDepth;
        it += uint32_t(k1 - k0);
        if (k1 == k0 || last == 0 || k1 * kDepth < rows) return true;
        const uint32_t s = (it - 1) % uint32_t(m.stages);
        if (!mbar_wait(smem_addr(&sh.tail[s]), phases >> s & 1, sh, m)) return false;
        phases ^= 1u << s;
        uint8_t *stage = k.ring + s * m.stage_bytes;
        const int count = ceil_div(last, 16) * 16 - last;  // rows of 128 bytes, in each of 4 tiles
        for (int i = threadIdx.x % 32; i < count * 4 * 8; i += 32) {
            const int tile = i / (count * 8), piece = i % (count * 8);
            reinterpret_cast<uint4 *>(stage + tile * (kDepth * 128) + last * 128)[piece] = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (threadIdx.x % 32 == 0) mbar_arrive_cluster(map_to(smem_addr(&sh.full[s]), k.leader));
        __syncwarp();
        return true;
    }
};

// One product, a pair of CTAs per tile.
template <typename T, Product P>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    expert_kernel(const __grid_constant__ Maps maps, const Shape m, T *out, float *gu) {
    const Setup k = set_up<P>(maps, m);
    Shared &sh = *k.sh;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    Tiles<P> tiles(m, k.first, sh.order, pair, pairs);
    Tile t;
    uint32_t acc = 0;  // accumulators used so far: they take turns

    if (warp == 0 && lane == 0) {
        Loader<P> loader = loader_of<P>(maps, m, k);
        while (tiles.next(t))
            if (!loader.load_tile(t, 0, steps_of<P>(m, t.rows))) break;
        wait_previous();  // in any case: a kernel is over only when those before it are
    } else if (warp == 1 && lane == 0 && k.rank == 0) {
        Issuer<T, P> issuer = issuer_of<T, P>(m, k);
        while (tiles.next(t)) {
            const int steps = steps_of<P>(m, t.rows);
            if (steps == 0) continue;
            if (!mbar_wait(smem_addr(&sh.tmem_empty[acc & 1]), (acc / 2 + 1) & 1, sh, m)) break;
            fence_after();
            if (!issuer.run(t, sh.tmem + (acc & 1) * kMaxN, 0, steps)) break;
            mma_commit(smem_addr(&sh.tmem_full[acc & 1]), issuer.mask);
            ++acc;
        }
    } else if (warp == 2 && kWeightGrad<P>) {
        TailClearer clearer{m, sh, k};
        while (tiles.next(t))
            if (!clearer.clear(t.rows, 0, steps_of<P>(m, t.rows))) break;
    } else if (warp >= 4) {
        // Finished accumulators.  This warp's TMEM lanes are features 32 (warp % 4) ... + 31; its
        // group of four warps takes every other chunk of columns.
        const int quarter = warp % 4, group = warp / 4 - 1;
        const uint32_t lanes = sh.tmem + (uint32_t(quarter * 32) << 16), empty = map_to(smem_addr(sh.tmem_empty), k.leader);
        while (tiles.next(t)) {
            const bool none = steps_of<P>(m, t.rows) == 0;
            const int feature = t.feature + int(k.rank) * (kTileFeatures<P> / 2);
            if (!none) {
                if (!group_all(group, mbar_wait(smem_addr(&sh.tmem_full[acc & 1]), (acc / 2) & 1, sh, m)))
                    break;
                fence_after();
            }
            const uint32_t columns = lanes + (acc & 1) * kMaxN;
            if constexpr (kWeightGrad<P>) {
                // A thread has one row of the gradient and writes its columns.
                const int width = P == kGradOut ? m.inner : m.hidden, height = P == kGradOut ? m.hidden : m.inner;
                const int f = feature + quarter * 32 + lane;
                T *row = out + ((int64_t(t.expert) * (P == kGradIn ? 2 : 1) + t.part) * height + f) * width + t.column;
                const bool sectors = width % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0;
                uint32_t r[kChunk];
#pragma unroll
                for (int j = 0; j < kChunk; ++j) r[j] = 0;
                if (!none) tmem_request(columns + group * kChunk, r);
                for (int c = group * kChunk; c < kMaxN; c += 2 * kChunk) {
                    float v[kChunk];
                    if (!none) tmem_wait(r);
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) v[j] = __uint_as_float(r[j]);
                    if (!none && c + 2 * kChunk < kMaxN) tmem_request(columns + c + 2 * kChunk, r);
                    if (f >= height || t.column + c >= width) continue;
                    if (sectors) {
                        store16(row + c, v);
                    } else {
                        store8(row + c, v);
                        if (t.column + c + 8 < width) store8(row + c + 8, v + 8);
                    }
                }
            } else {
                // A chunk of rows at a time, turned around in shared memory: then 8 lanes hold 64
                // of a row's features, 8 next to each other per lane.
                const int r = quarter * 4 + lane / 8;
                float *buffer = k.staging + group * (kStagingBytes / 4);
                uint32_t v[kChunk];
                [[maybe_unused]] float g[2][8], u[2][8];  // kBack: the projections of the next chunk's rows
                const auto request = [&](int c) {
                    if (c >= t.rows) return;
                    tmem_request(columns + c, v);
                    if constexpr (P == kBack) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int f = feature + i * 64 + lane % 8 * 8;
                            const int64_t row = t.first + c + r;
                            if (c + r < t.rows && f < m.inner) {
                                load8_global(gu + row * 2 * m.inner + f, g[i]);
                                load8_global(gu + row * 2 * m.inner + m.inner + f, u[i]);
                            }
                        }
                    }
                };
                request(group * kChunk);
                for (int c = group * kChunk; c < t.rows; c += 2 * kChunk) {
                    const int64_t row = t.first + c + r;
                    tmem_wait(v);
#pragma unroll
                    for (int j = 0; j < kChunk; ++j)
                        buffer[j * kStagingRow + quarter * 32 + lane] = __uint_as_float(v[j]);
                    [[maybe_unused]] float gc[2][8], uc[2][8];
                    if constexpr (P == kBack) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) gc[j / 8][j % 8] = g[j / 8][j % 8], uc[j / 8][j % 8] = u[j / 8][j % 8];
                    }
                    request(c + 2 * kChunk);
                    group_sync(group);
                    const float *sums = buffer + r * kStagingRow + lane % 8 * 8;
#pragma unroll
                    for (int i = 0; i < (P == kUp ? 1 : 2); ++i) {
                        const int f = feature + i * 64 + lane % 8 * 8;
                        if (c + r >= t.rows || f >= (P == kUp || P == kBack ? m.inner : m.hidden)) continue;
                        float a[8], b[8];
                        load8(sums + i * 64, a);
                        if (P == kUp) load8(sums + 64, b);
                        finish<T, P>(m, out, gu, row, f, a, b, gc[i], uc[i]);
                    }
                    group_sync(group);  // the buffer is free again
                }
            }
            if (!none) {
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(empty + (acc & 1) * 8);
                ++acc;
            }
        }
    }
    tear_down(k);
}

// One product of few tiles: the pairs of a cluster share a tile, each with a part of the steps, and
// add their sums up through distributed shared memory, in the pairs' order.  A tile's K loop runs at
// the latency of its ring, so one pair reads weights at a few hundred GB/s however idle the GPU is:
// a [1, 5632] x [5632, 2048] product has 8 tiles, and took 27.9 us with a pair each, 13.1 with four.
// Likewise dw_out of 25,409 rows of one expert, 144 x 2440, with 10 tiles: 131 and 50 us.  There are as
// many clusters as tiles at least (split_of), so a cluster has one tile or none.
template <typename T, Product P>
__global__ void __launch_bounds__(kThreads, 1)
    expert_split_kernel(const __grid_constant__ Maps maps, const Shape m, T *out, float *gu) {
    const Setup k = set_up<P>(maps, m);
    Shared &sh = *k.sh;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int split = int(cluster_size()) / 2, part = int(k.leader) / 2;
    const int cluster = int(blockIdx.x) / (2 * split), clusters = int(gridDim.x) / (2 * split);
    Tiles<P> tiles(m, k.first, sh.order, cluster, clusters);
    Tile t;
    if (tiles.next(t)) {
        const int steps = steps_of<P>(m, t.rows), k0 = steps * part / split, k1 = steps * (part + 1) / split;
        const int n = kWeightGrad<P> ? kMaxN : ceil_div(t.rows, kStepN) * kStepN, columns = n / split;  // each pair's
        const int feature = t.feature + int(k.rank) * (kTileFeatures<P> / 2);
        if (warp == 0 && lane == 0) {
            loader_of<P>(maps, m, k).load_tile(t, k0, k1);
        } else if (warp == 1 && lane == 0 && k.rank == 0) {
            Issuer<T, P> issuer = issuer_of<T, P>(m, k);
            if (k1 > k0 && issuer.run(t, sh.tmem, k0, k1)) mma_commit(smem_addr(&sh.tmem_full[0]), issuer.mask);
        } else if (warp == 2 && kWeightGrad<P>) {
            TailClearer{m, sh, k}.clear(t.rows, k0, k1);
        } else if (warp >= 4 && k1 > k0) {
            mbar_wait(smem_addr(&sh.tmem_full[0]), 0, sh, m);
        }
        __syncthreads();
        const bool fine = !sh.aborted;  // else the waits ran out: nothing is stored
        // The sums, [part][column][feature], go where the epilogue's staging is, or, if that is too
        // small, into the ring, once every pair's products are over and no load is under way.
        const bool apart = n * kStagingRow * 4 <= int(2 * kStagingBytes);
        float *sums = apart ? k.staging : reinterpret_cast<float *>(k.ring);
        if (!apart) cluster_sync();
        fence_after();
        if (fine && warp >= 4 && k1 > k0) {
            const int quarter = warp % 4, group = warp / 4 - 1;
            for (int c = group * 8; c < n; c += 16) {
                float v[8];
                tmem_load(sh.tmem + (uint32_t(quarter * 32) << 16) + c, v);
                const uint32_t to = map_to(smem_addr(sums), uint32_t(c / columns * 2) + k.rank) +
                                    ((part * columns + c % columns) * kStagingRow + quarter * 32 + lane) * 4;
#pragma unroll
                for (int j = 0; j < 8; ++j) store_cluster(to + j * kStagingRow * 4, v[j]);
            }
        }
        fence_before();
        cluster_sync();  // the sums are there
        if constexpr (kWeightGrad<P>) {
            // A thread adds up 8 columns of one row of the gradient.
            const int width = P == kGradOut ? m.inner : m.hidden, height = P == kGradOut ? m.hidden : m.inner;
            for (int i = threadIdx.x; fine && i < kHalf * (columns / 8); i += kThreads) {
                const int f = feature + i % kHalf, c = i / kHalf * 8, column = t.column + part * columns + c;
                if (f >= height || column >= width) continue;
                float a[8] = {};
                for (int p = 0; p < split; ++p) {
                    if (steps * p / split == steps * (p + 1) / split) continue;  // had no steps
                    const float *from = sums + (p * columns + c) * kStagingRow + i % kHalf;
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[j] += from[j * kStagingRow];
                }
                store8(out + ((int64_t(t.expert) * (P == kGradIn ? 2 : 1) + t.part) * height + f) * width + column, a);
            }
        } else {
            constexpr int kGroups = P == kUp ? 8 : 16;
            const int mine = min(columns, t.rows - part * columns);
            for (int i = threadIdx.x; fine && i < mine * kGroups; i += kThreads) {
                const int column = i / kGroups, f = feature + i % kGroups * 8;
                const int64_t row = t.first + part * columns + column;
                if (f >= (P == kUp || P == kBack ? m.inner : m.hidden)) continue;
                float a[8] = {}, b[8] = {}, g[8], u[8];
                if constexpr (P == kBack) {
                    load8_global(gu + row * 2 * m.inner + f, g);
                    load8_global(gu + row * 2 * m.inner + m.inner + f, u);
                }
                for (int p = 0; p < split; ++p) {
                    const float *from = sums + (p * columns + column) * kStagingRow + i % kGroups * 8;
                    add8(from, a);
                    if (P == kUp) add8(from + 64, b);
                }
                finish<T, P>(m, out, gu, row, f, a, b, g, u);
            }
        }
    }
    if (threadIdx.x == 0) wait_previous();
    tear_down(k);
}

// A call without rows has nothing to do but to look for counts that say otherwise.
__global__ void count_check_kernel(const int32_t *counts, int nexp, unsigned int *status) {
    int any = 0;
    for (int e = threadIdx.x; e < nexp; e += blockDim.x) any |= counts[e];
    if (__syncthreads_or(any) && threadIdx.x == 0) atomicExch(status, 2u);
}

// ---- launches ----------------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return EncodeFn(nullptr);
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// A dense tensor of 16-bit elements, the innermost dimension first; boxes of 64 elements (128
// swizzled bytes) by `box` in the other dimensions.  Reads past an end of a dimension give zeros.
struct Dense {
    const void *base;
    int rank;
    cuuint64_t dims[4];
    cuuint32_t box[4];
};

template <typename T> bool encode(CUtensorMap *map, const Dense &d) {
    cuuint64_t strides[3];
    cuuint32_t ones[4] = {1, 1, 1, 1};
    cuuint64_t bytes = 2;
    for (int i = 0; i + 1 < d.rank; ++i) strides[i] = bytes *= d.dims[i];
    const auto type = std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode_fn() != nullptr &&
           encode_fn()(map, type, cuuint32_t(d.rank), const_cast<void *>(d.base), d.dims, strides, d.box, ones,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a kernel can have on a device at once, asked for once: CTAs (one per SM), or clusters of 4 and
// 8 CTAs, of which fewer fit than the SMs' number says, since a cluster lies within one GPC.
struct Residency {
    int sms, clusters4, clusters8;
};
cudaError_t residency(const void *kernel, bool split, int device, int index, Residency *out) {
    constexpr int kDevices = 64, kKernels = 24;
    static std::atomic<uint64_t> known[kDevices][kKernels];  // sms, clusters8 and clusters4, 16 bits each
    const bool kept = device < kDevices;
    if (uint64_t v = kept ? known[device][index].load(std::memory_order_acquire) : 0; v != 0) {
        *out = {int(v & 0xffff), int(v >> 32 & 0xffff), int(v >> 16 & 0xffff)};
        return cudaSuccess;
    }
    *out = {};
    constexpr int kBytes = int(shared_bytes(UGDR_X_EXPERTS_MAX));
    if (cudaError_t e = cudaDeviceGetAttribute(&out->sms, cudaDevAttrMultiProcessorCount, device); e != cudaSuccess)
        return e;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        e != cudaSuccess)
        return e;
    for (unsigned size = 4; split && size <= 8; size *= 2) {
        cudaLaunchAttribute attribute{};
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim = {size, 1, 1};
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(size);
        config.blockDim = dim3(kThreads);
        config.dynamicSmemBytes = kBytes;
        config.attrs = &attribute;
        config.numAttrs = 1;
        if (cudaError_t e = cudaOccupancyMaxActiveClusters(size == 4 ? &out->clusters4 : &out->clusters8, kernel, &config);
            e != cudaSuccess)
            return e;
    }
    if (kept)
        known[device][index].store(uint64_t(out->clusters4) << 32 | uint64_t(out->clusters8) << 16 | uint64_t(out->sms),
                                   std::memory_order_release);
    return cudaSuccess;
}

// Pairs that share a tile: as many as let every tile have a cluster of the launch, where the steps
// are enough to gain by it.  What counts is known here from above only: a tile for each expert, or row
// if those are fewer, and one for every kMaxN rows; for the weight gradients, whose steps are an
// expert's rows, their mean.
template <Product P> int split_of(const ugdr_x_experts &m, const Residency &on) {
    const auto tiles_of = [](int64_t n, int64_t size) { return (n + size - 1) / size; };
    const int64_t features = P == kUp || P == kBack || P == kGradIn ? m.inner : m.hidden;
    int64_t tiles = tiles_of(features, kTileFeatures<P>), depth = 0;
    if (kWeightGrad<P>) {
        tiles *= m.nexp * (P == kGradIn ? 2 : 1) * tiles_of(P == kGradOut ? m.inner : m.hidden, kMaxN);
        depth = int64_t(m.rows / uint64_t(m.nexp));
    } else {
        tiles *= (m.rows < uint64_t(m.nexp) ? int64_t(m.rows) : m.nexp) + int64_t(m.rows / kMaxN);
        depth = P == kDown ? m.inner : P == kInput ? 2 * int64_t(m.inner) : m.hidden;
    }
    // Adding the parts up takes 2 to 3 us, a step 0.26 to 0.29 us: 15 of 20 saved, or 14 of 28, gain by it.
    if (tiles <= on.clusters8 && depth >= 20 * kDepth) return 4;
    return tiles <= on.clusters4 && depth >= 28 * kDepth ? 2 : 1;
}

// One product.  `a` and `b` are its operands: the weights and the rows, or the two row tensors of a
// weight gradient.
template <typename T, Product P>
cudaError_t launch(const ugdr_x_experts &m, const void *a, const void *b, void *out, float *gu, cudaStream_t s) {
    const cuuint64_t H = cuuint64_t(m.hidden), F = cuuint64_t(m.inner), R = m.rows, E = cuuint64_t(m.nexp);
    Dense da, db;
    if (P == kUp)
        da = {a, 4, {H, F, 2, E}, {64, 64, 2, 1}};
    else if (P == kInput)
        da = {a, 4, {H, F, 2, E}, {64, 64, 1, 1}};
    else if (P == kDown)
        da = {a, 3, {F, H, E}, {64, 128, 1}};
    else if (P == kBack)
        da = {a, 3, {F, H, E}, {64, 64, 1}};
    else if (P == kGradOut)
        da = {a, 2, {H, R}, {64, 64}};
    else
        da = {a, 3, {F, 2, R}, {64, 1, 64}};
    if (P == kInput)
        db = {b, 3, {F, 2, R}, {64, 1, 0}};
    else
        db = {b, 2, {P == kUp || P == kBack || P == kGradIn ? H : F, R}, {64, 0}};
    // The most rows of B that a CTA can have to load per step, in whole boxes.
    int load = kHalf;
    if (!kWeightGrad<P> && m.rows < kMaxN) {
        const int half = (int(m.rows) + kStepN - 1) / kStepN * kStepN / 2;
        load = half == 16 ? 16 : (half + 31) / 32 * 32;
    }
    const uint32_t stage_bytes = kOperandBytes + uint32_t(load) * kDepth * 2;
    const int stages = int(kRingBytes / stage_bytes) < kMaxStages ? int(kRingBytes / stage_bytes) : kMaxStages;
    Maps maps;
    if (!encode<T>(&maps.a, da)) return cudaErrorInvalidValue;
    for (int i = 0; i < (kWeightGrad<P> ? 1 : kBoxes); ++i) {
        if (kHalf >> i > load) continue;  // too large ever to be asked for
        db.box[db.rank - 1] = kWeightGrad<P> ? kDepth : kHalf >> i;
        if (!encode<T>(&maps.b[i], db)) return cudaErrorInvalidValue;
    }
    const Shape shape{m.counts, m.status, expert_wait_ns(), int(m.rows), m.nexp, m.hidden, m.inner, m.act, stages, stage_bytes};

    int device = 0;
    if (cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return e;
    constexpr int kIndex = int(P) * 2 + std::is_same_v<T, __half>;
    auto *kernel = expert_kernel<T, P>, *split_kernel = expert_split_kernel<T, P>;
    Residency plain, clusters;
    if (cudaError_t e = residency(reinterpret_cast<const void *>(kernel), false, device, kIndex, &plain); e != cudaSuccess)
        return e;
    if (cudaError_t e = residency(reinterpret_cast<const void *>(split_kernel), true, device, 12 + kIndex, &clusters);
        e != cudaSuccess)
        return e;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(plain.sms / 2 * 2));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = shared_bytes(m.nexp);
    config.stream = s;
    config.attrs = attributes;
    config.numAttrs = 1;
    if (const int split = split_of<P>(m, clusters); split > 1) {
        kernel = split_kernel;
        attributes[1].id = cudaLaunchAttributeClusterDimension;
        attributes[1].val.clusterDim = {unsigned(2 * split), 1, 1};
        config.gridDim = dim3(unsigned(split == 4 ? 8 * clusters.clusters8 : 4 * clusters.clusters4));
        config.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&config, kernel, maps, shape, static_cast<T *>(out), gu);
}

template <typename T>
int forward(const ugdr_x_experts &m, const void *x, void *y, void *h, float *gu, cudaStream_t s) {
    cudaError_t e = launch<T, kUp>(m, m.w_in, x, h, gu, s);
    if (e == cudaSuccess) e = launch<T, kDown>(m, m.w_out, h, y, nullptr, s);
    return int(e);
}

template <typename T>
int backward(const ugdr_x_experts &m, const void *dy, const void *x, const void *h, const float *gu, void *dgu,
             void *dx, void *dw_in, void *dw_out, cudaStream_t s) {
    cudaError_t e = launch<T, kBack>(m, m.w_out, dy, dgu, const_cast<float *>(gu), s);
    if (e == cudaSuccess) e = launch<T, kGradOut>(m, dy, h, dw_out, nullptr, s);
    if (e == cudaSuccess) e = launch<T, kGradIn>(m, dgu, x, dw_in, nullptr, s);
    // Last, so that dx may be dy or x itself.
    if (e == cudaSuccess) e = launch<T, kInput>(m, m.w_in, dgu, dx, nullptr, s);
    return int(e);
}

#define UGDR_EXPERT(KERNEL, T, NAME, P, LABEL) \
    {#KERNEL "<" NAME ", " LABEL ">", reinterpret_cast<const void *>(&KERNEL<T, P>), kThreads, int(shared_bytes(UGDR_X_EXPERTS_MAX))}
#define UGDR_EXPERT_ALL(KERNEL, T, NAME)                                                                    \
    UGDR_EXPERT(KERNEL, T, NAME, kUp, "up"), UGDR_EXPERT(KERNEL, T, NAME, kDown, "down"),                    \
        UGDR_EXPERT(KERNEL, T, NAME, kBack, "back"), UGDR_EXPERT(KERNEL, T, NAME, kInput, "input"),          \
        UGDR_EXPERT(KERNEL, T, NAME, kGradOut, "grad out"), UGDR_EXPERT(KERNEL, T, NAME, kGradIn, "grad in")

}  // namespace

int expert_kernels(const KernelRef **out) {
    static const KernelRef refs[] = {
        UGDR_EXPERT_ALL(expert_kernel, __nv_bfloat16, "bf16"), UGDR_EXPERT_ALL(expert_kernel, __half, "fp16"),
        UGDR_EXPERT_ALL(expert_split_kernel, __nv_bfloat16, "bf16"), UGDR_EXPERT_ALL(expert_split_kernel, __half, "fp16"),
        {"count_check_kernel", reinterpret_cast<const void *>(&count_check_kernel), kCheckThreads}};
    *out = refs;
    return int(sizeof(refs) / sizeof(refs[0]));
}

int launch_count_check(const ugdr_x_experts &m, cudaStream_t s) {
    count_check_kernel<<<1, kCheckThreads, 0, s>>>(m.counts, m.nexp, m.status);
    return int(cudaGetLastError());
}

int launch_expert_ffn(const ugdr_x_experts &m, const void *x, void *y, void *h, float *gu, cudaStream_t s) {
    return m.type == UGDR_X_TYPE_BF16 ? forward<__nv_bfloat16>(m, x, y, h, gu, s) : forward<__half>(m, x, y, h, gu, s);
}

int launch_expert_ffn_backward(const ugdr_x_experts &m, const void *dy, const void *x, const void *h, const float *gu,
                               void *dgu, void *dx, void *dw_in, void *dw_out, cudaStream_t s) {
    return m.type == UGDR_X_TYPE_BF16 ? backward<__nv_bfloat16>(m, dy, x, h, gu, dgu, dx, dw_in, dw_out, s)
                                      : backward<__half>(m, dy, x, h, gu, dgu, dx, dw_in, dw_out, s);
}

}  // namespace ugdr::coll
