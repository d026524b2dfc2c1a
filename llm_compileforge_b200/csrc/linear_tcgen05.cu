// Matrix product with bias, activation, gate and residual, dense or grouped by ragged row ranges, on the sm_100a tensor cores.
//
// out[r, n] = act(sum_k x[i, k] W_e[k, n] + b_e[n]) * (sum_k x[i, k] V_e[k, n] + c_e[n]) + residual[r, n], i = row_index[r]
//
// The product is computed transposed: a tile is 128 output columns ("features", the M side of the MMA) by up to kTok rows of
// out ("tokens", the N side).  A ragged last tile then costs what its rows cost (N is any multiple of 16) instead of a full
// 128-row panel, and one token against a large matrix - decode - reads the matrix once with 16 columns of MMA behind it.
// With a gate, a tile's 128 features are 64 columns of W and the same 64 of V, so gate and up value of an output meet in one
// thread block whatever the shape.
//
// Persistent thread blocks walk the tiles; accumulators are double-buffered in tensor memory (2 x kTok columns):
//   warp 8      weights' producer: per 64-wide K step two TMA boxes of 64 features
//   warp 10     rows' producer: boxes of box_rows token rows, or, with a row index, row gathers of four rows (about 60 clocks
//               each, whatever they bring: right for the few rows an expert has in decode; for many a pass before this kernel
//               lays the rows out in index order).  One warp for both was the bound of every shape: a wait that succeeds 80
//               clocks, a box 53, 600 a K step with the rest, against 512 for its MMAs.
//   warp 9      one thread issues tcgen05.mma kind::f16 (N = tokens, K 16, four per step); the weight operand is MN-major for
//               [K, N] storage and K-major for [N, K], straight from 128-byte-swizzled shared memory
//   warps 0-7   epilogue, two groups of four warps that take every other 16 or 32 tokens: through a transposing buffer in shared
//               memory, so that rows of out and residual move as 8 bytes a lane; bias, activation, gate, residual in fp32,
//               one rounding
// Many rows a group (kPair): a cluster of two thread blocks owns 256 features x 256 tokens with cta_group::2 MMAs (M 256): each
// block loads its 128 features and half of the tokens, the leader's MMAs read both, each block's tensor memory receives its
// own features.
// Few tiles (decode): a cluster of up to eight thread blocks owns one tile, each taking a part of K; every block lays its sums
// into its own operand buffers, by then free, and after a cluster barrier adds its share of the tokens over all blocks' shared
// memory in the order of the ranks - no workspace, no atomics, the same bits every time.
// Group offsets are read on the device; each thread block lays the groups' tiles out in shared memory before it starts.
// Every wait is bounded; one that runs out sets SFB_STATUS_WAIT_TIMEOUT and the block leaves through the common teardown.

#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "linear.cuh"

namespace sfb {
namespace {

constexpr int kFeat = 128, kStepK = 64;
constexpr int kWBytes = kFeat * kStepK * 2;      // a K step's weights: two boxes of 64 features
constexpr int kHalfBytes = kWBytes / 2;
constexpr int kEpilogueWarps = 8, kWeightWarp = 8, kMmaWarp = 9, kRowWarp = 10, kThreads = 352;
constexpr uint64_t kWaitNanoseconds = 2000000000;  // no wait of a kernel that takes milliseconds comes near it
constexpr int kMaxSplit = 8;

constexpr int kMaxStages = 9;
enum {
    B_FULL = 0,
    B_EMPTY = kMaxStages,
    B_ACC_FULL = 2 * kMaxStages,
    B_ACC_EMPTY = B_ACC_FULL + 2,
    B_COUNT = B_ACC_EMPTY + 2
};

// A kernel's shape: token columns of a tile, thread blocks an SM, whether a cluster of two shares each tile.  The number of
// pipeline stages follows from the shared memory that a launch gives a block.
template <int TOK, int BLOCKS, bool PAIR>
struct Shape {
    static constexpr int kTok = TOK, kBlocks = BLOCKS;
    static constexpr bool kPair = PAIR;
    static constexpr int kRows = PAIR ? TOK / 2 : TOK;  // token rows in one block's shared memory
    static constexpr int kRound = PAIR ? 32 : 16;       // what the MMA's N is a multiple of
    // The epilogue takes this many tokens at a time: 32 where the registers allow it; at 16 a 256-token tile took 860 clocks each
    static constexpr int kChunk = TOK >= 128 ? 32 : 16;
    static constexpr int kStaging = kChunk * kFeat * 4;  // fp32 [chunk][128 features]
    static constexpr int kBuffers = TOK == 64 ? 2 : 1;   // of an epilogue group
    static constexpr int kStage = kWBytes + kRows * 128;  // of one K step
    static constexpr int smem(int steps, int groups) { return 1024 + steps * kStage + 2 * kBuffers * kStaging + B_COUNT * 8 + 16 + 2 * (groups + 1) * 4; }
    static constexpr int stages(int budget, int groups, int sub) {  // of `sub` K steps each
        const int n = (budget - smem(0, groups)) / (sub * kStage);
        return n < kMaxStages ? n : kMaxStages;
    }
};
// Few tokens: the weights' way from HBM bounds.  With more tiles than SMs two blocks an SM share it evenly whatever the number
// of tiles, and one's start, last tile and epilogue run beside the other's loads.
using Shape32 = Shape<32, 2, false>;
using Shape64 = Shape<64, 2, false>;
using Shape128 = Shape<128, 1, false>;
using ShapePair = Shape<256, 1, true>;
constexpr int kSmemPerBlock = 232448, kSmemPerHalf = 233472 / 2 - 1024;  // of one block an SM, of each of two
template <typename S>
constexpr bool fits() {  // a pipeline at all, and room for a tile's sums in it
    const int one = S::stages(kSmemPerHalf, kMaxGroups, 1), two = S::stages(kSmemPerBlock, kMaxGroups, 2);
    return (S::kBlocks == 1 || (one >= 2 && S::kTok * kFeat * 4 <= one * S::kStage)) && two >= 2 && (S::kPair || S::kTok * kFeat * 4 <= two * 2 * S::kStage);
}
static_assert(fits<Shape32>() && fits<Shape64>() && fits<Shape128>() && fits<ShapePair>(), "shared memory");

struct TileArgs {
    const void *bias, *up_bias, *residual;
    void* out;
    const int32_t *offsets, *row_index;
    int* status;
    int64_t out_stride, res_stride, bias_stride, up_bias_stride;
    int rows, x_rows, N, n_k, groups;
    int feat_tiles;  // column tiles of out
    int box_rows;    // token rows of one TMA box
    int stages;      // of the operand pipeline
    int sub;         // 64-wide K steps of a stage, behind one pair of barriers
    int split;       // thread blocks that share a tile's K steps (= cluster size, without kPair); above 1 one tile a cluster
    int block;       // token tiles that run together through the feature tiles (L2 reuse of x and W)
    int act;
    bool gated, nk, out_f32, vec;
    bool ordered;    // the kernel before this one is order_rows_kernel, and only x comes from it
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint64_t nanoseconds() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// CLUSTER: for barriers on which other blocks of the cluster arrive; what they wrote before is visible after.
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    if constexpr (CLUSTER)
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    else
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// Waits kWaitNanoseconds at most.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    if (mbar_try<CLUSTER>(bar, parity)) return true;
    const uint64_t begun = nanoseconds();
    do {
        if (mbar_try<CLUSTER>(bar, parity)) return true;
    } while (nanoseconds() - begun < kWaitNanoseconds);
    return false;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t local, uint32_t rank) {  // the same shared-memory offset in block `rank`
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// W consecutive floats from this block's shared memory, or (PEER) that of any block of the cluster
template <int W, bool PEER>
__device__ __forceinline__ void ld_shared(float* v, uint32_t addr) {
    if constexpr (PEER) {
        if constexpr (W == 4) asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
        else if constexpr (W == 2) asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
        else asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[0]) : "r"(addr) : "memory");
    } else {
        if constexpr (W == 4) asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
        else if constexpr (W == 2) asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
        else asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[0]) : "r"(addr) : "memory");
    }
}
template <bool PAIR>  // PAIR: the bytes are reported to a barrier of the cluster's leader
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
// Four rows of a map whose box is one row high, side by side at dst.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int4 r) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(bar)
                 : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst, uint32_t cols) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t cols) {
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <bool PAIR>  // PAIR: arrives on this barrier in both thread blocks
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                       uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %2};\n mov.b64 db, {%3, %4};\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n}\n"
            ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %2};\n mov.b64 db, {%3, %4};\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n}\n"
            ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
            : "memory");
}
// N columns of this lane's row, waited for in the same statement: between a load and its wait nothing may touch the registers,
// and across two statements the compiler could.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[N]) {
    static_assert(N == 16 || N == 32, "columns");
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    if constexpr (N == 16)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr)
            : "memory");
    else
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(taddr)
            : "memory");
}
// Shared-memory matrix descriptor words (sm_100 format): start address and leading byte offset in 16-byte units; stride byte
// offset, version 1, 128-byte swizzle.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo_bytes) { return ((addr >> 4) & 0x3fff) | (((lbo_bytes >> 4) & 0x3fff) << 16); }
__device__ __forceinline__ uint32_t desc_hi(uint32_t sbo_bytes) { return ((sbo_bytes >> 4) & 0x3fff) | (1u << 14) | (2u << 29); }
// Instruction descriptor for kind::f16: fp32 accumulate, 16-bit A/B, A MN-major or K-major, B K-major.
__device__ __forceinline__ uint32_t instr_desc(bool bf16, bool a_mn_major, int m, int n) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn_major ? 1u : 0u) << 15) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
    if constexpr (BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
// Whether any of an epilogue group's four warps failed; all of them come here, so none waits for one that has left.
__device__ __forceinline__ bool group_any(int barrier, bool failed) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r)
                 : "r"((uint32_t)failed), "r"(barrier)
                 : "memory");
    return r != 0;
}
__device__ __forceinline__ void group_sync(int barrier) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(barrier) : "memory"); }

// Two fp32 operations an instruction, each rounded as by itself.
struct Two {
    uint64_t v;
    __device__ __forceinline__ Two(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
    __device__ __forceinline__ explicit Two(float both) : Two(both, both) {}
    __device__ __forceinline__ float2 get() const {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(a.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return a;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v));
    return a;
}
__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// h Phi(h), two at a time: Phi(-x) = 2^P(x), P the polynomial of degree 11 that fits log2 Phi(-x) on [0, 13.2] best where 2^P may
// be off by the smaller of 2^-12 of itself and 6e-8 (Lawson's iteration).  With the rounding of its terms and of ex2 h Phi(h) comes
// out within 3e-7 |h|, and for -12.9 <= h < 0 within 2^-11 of itself, a quarter of bf16's half step and less above -6; below, where
// Phi is no normal number, it is zero.  One exponential and thirteen multiply-adds: the tile's epilogue is bound by the FMA pipes.  A
// [1001, 2048] x [2048, 8192] product took 34.3 us with a fit of one exponential, one division and one value at a time, 32.2 with
// exp(-x^2 / 2) times a polynomial of degree 11; measured in turn, 32.1 with a polynomial of degree 8 (22 % off at h = -7) and 32.5
// with this; with erfcf the epilogue alone took four times the MMAs.
__device__ __forceinline__ void gelu_erf(float& a, float& b) {
    constexpr float c[12] = {-9.999998212e-01f, -1.151115060e+00f, -4.591248930e-01f, -5.274898559e-02f, 7.415628992e-03f, -3.830976493e-04f,
                             -1.012203720e-04f, 2.793559543e-05f, -3.357467222e-06f, 2.251555600e-07f, -8.138483665e-09f, 1.236985236e-10f};
    const Two x(fminf(fabsf(a), 13.2f), fminf(fabsf(b), 13.2f));
    Two p(c[11]);
#pragma unroll
    for (int i = 10; i >= 0; --i) p = fma2(p, x, Two(c[i]));
    const float2 e = p.get();
    const Two q(exp2_approx(e.x), exp2_approx(e.y));
    const float2 lo = q.get(), hi = fma2(q, Two(-1.f), Two(1.f)).get();
    const float2 y = mul2(Two(a, b), Two(a < 0.f ? lo.x : hi.x, b < 0.f ? lo.y : hi.y)).get();
    a = y.x;
    b = y.y;
}
template <int W>
__device__ __forceinline__ void activate_all(float (&h)[W], int act) {
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < W; ++i) h[i] = f(h[i]);
    };
    if (act == SFB_ACT_SILU) each([](float v) { return activate<SFB_ACT_SILU>(v); });
    else if (act == SFB_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < W; i += 2) gelu_erf(h[i], h[i + 1]);
    }
    else if (act == SFB_ACT_GELU_TANH) each([](float v) { return activate<SFB_ACT_GELU_TANH>(v); });
    else if (act == SFB_ACT_RELU) each([](float v) { return activate<SFB_ACT_RELU>(v); });
}

struct Tile {
    int group, row0, rows, feat;
};
// The groups of a call in shared memory: group e has rows off[e] .. off[e + 1], and tiles[e] token tiles lie before it.
struct Groups {
    const int *off, *tiles;
    int n;
    // Tile t: groups one after another; inside a group blocks of `block` token tiles, token tiles fastest, then features.  A
    // group's rows are spread evenly over its token tiles, in multiples of `round`.
    __device__ __forceinline__ Tile at(int t, int feat_tiles, int block, int round) const {
        int e = 0;
        for (int step = kMaxGroups / 2; step > 0; step >>= 1)
            if (e + step < n && tiles[e + step] * feat_tiles <= t) e += step;
        const int nt = tiles[e + 1] - tiles[e], count = off[e + 1] - off[e];
        int i = t - tiles[e] * feat_tiles;
        const int b = i / (block * feat_tiles);
        const int g = min(block, nt - b * block);
        i -= b * block * feat_tiles;
        const int f = i / g, m = b * block + i - f * g;
        const int per = ((count + nt - 1) / nt + round - 1) / round * round;
        return {e, off[e] + m * per, min(per, count - m * per), f};
    }
};

template <typename S, bool BF16>
__global__ void __launch_bounds__(kThreads, S::kBlocks)
linear_tcgen05_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap umap,
                      const TileArgs a) {
    extern __shared__ uint8_t smem_raw[];
    constexpr int kTok = S::kTok, kStage = S::kStage;
    const uint32_t stages = (uint32_t)a.stages, sub = (uint32_t)a.sub, stage_bytes = sub * kStage;
    constexpr bool PAIR = S::kPair;
    using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = PAIR ? 1 : a.split, cluster = PAIR ? 2 : split;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const int unit = (int)blockIdx.x / cluster, n_units = (int)gridDim.x / cluster;
    const bool gather = !PAIR && a.row_index != nullptr;  // kPair: rows of x in the order of out

    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    float* staging = reinterpret_cast<float*>(base_ptr + stages * stage_bytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base_ptr + stages * stage_bytes + 2 * S::kBuffers * S::kStaging);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + B_COUNT);
    int* g_off = reinterpret_cast<int*>(tmem_slot + 4);
    int* g_tiles = g_off + a.groups + 1;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
    auto leader_bar = [&](int i) { return PAIR ? peer_addr(bar(i), 0) : bar(i); };

    if (warp == kWeightWarp) {  // one barrier a lane
        if (lane < 3) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &wmap : lane == 1 ? &xmap : &umap) : "memory");
        for (int i = lane; i < B_COUNT; i += 32)
            mbar_init(bar(i), i < B_EMPTY ? 2 : i < B_ACC_EMPTY ? 1 : kEpilogueWarps * (PAIR ? 2 : 1));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kMmaWarp) tmem_alloc<PAIR>(smem_u32(tmem_slot), 2 * kTok);
    // The previous kernel is waited for as late as may be: here where offsets come from it, without groups once the block has set
    // itself up.  order_rows_kernel lets this one start when all before it has ended: only who reads its rows waits for it,
    // the pipeline fills with weights meanwhile.
    if (a.offsets && !a.ordered) wait_for_previous();
    if (warp == 0) {  // the groups' rows, and the running number of token tiles
        int before = 0, top = a.offsets ? group_offset(a.offsets[0], 0, a.rows) : 0;
        bool bad = a.offsets && top != a.offsets[0];
        if (lane == 0) g_off[0] = top;
        for (int e0 = 0; e0 < a.groups; e0 += 32) {
            const int e = e0 + lane;
            const int raw = a.offsets && e < a.groups ? a.offsets[e + 1] : a.rows;
            int hi = group_offset(raw, top, a.rows);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, hi, o);
                if (lane >= o) hi = max(hi, up);
            }
            int lo = __shfl_up_sync(0xffffffffu, hi, 1);
            if (lane == 0) lo = top;
            top = __shfl_sync(0xffffffffu, hi, 31);
            bad |= hi != raw;
            const int own = e < a.groups ? (hi - lo + kTok - 1) / kTok : 0;
            int sum = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            if (e < a.groups) { g_off[e + 1] = hi; g_tiles[e] = before + sum - own; }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) g_tiles[a.groups] = before;
        if (bad && a.status) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
    }
    tc_fence_before();
    __syncthreads();
    let_next_start();
    if constexpr (PAIR) cluster_sync();  // the other block's barriers exist before anything is sent to them
    tc_fence_after();
    if (!a.offsets || (a.ordered && warp == kRowWarp)) wait_for_previous();
    const uint32_t tmem = *tmem_slot;
    const Groups groups{g_off, g_tiles, a.groups};
    const int tiles_total = g_tiles[a.groups] * a.feat_tiles;
    const int k_first = PAIR ? 0 : (int)((int64_t)a.n_k * rank / split), k_end = PAIR ? a.n_k : (int)((int64_t)a.n_k * (rank + 1) / split);
    const int feats = a.gated ? kFeat / 2 : kFeat;  // columns of out that this thread block computes of a tile
    // first such column of a tile; and of a tile's tokens (PAIR: the MMA takes half of its N from each block) the ones whose
    // rows of x this block brings in
    auto column0 = [&](const Tile& t) { return (PAIR ? 2 * t.feat + rank : t.feat) * feats; };
    auto half_of = [&](const Tile& t) { return PAIR ? (t.rows + 31) / 32 * 16 : t.rows; };
    auto own_rows = [&](const Tile& t, int r) { return PAIR ? max(0, min(half_of(t), t.rows - r * half_of(t))) : t.rows; };
    bool timed_out = false;

    if (warp == kWeightWarp) {
        // ========================= weights' producer ==========================
        if (lane == 0) {
            const uint32_t bytes = (PAIR ? 2 : 1) * kWBytes;
            const CUtensorMap* const second = a.gated ? &umap : &wmap;
            const uint32_t full0 = leader_bar(B_FULL);
            uint32_t s = 0, ephase = 1;
            for (int t = unit; t < tiles_total && !timed_out; t += n_units) {
                const Tile tile = groups.at(t, a.feat_tiles, a.block, S::kRound);
                const int n0 = column0(tile), n1 = n0 + (a.gated ? 0 : 64);
                for (int k = k_first; k < k_end; k += sub) {
                    if (!mbar_wait<PAIR>(bar(B_EMPTY + s), ephase)) { timed_out = true; break; }
                    const int end = min(k + (int)sub, k_end);
                    if (!PAIR || rank == 0) mbar_expect_tx(bar(B_FULL + s), (end - k) * bytes);
                    const uint32_t full = full0 + 8 * s;
                    uint32_t dst = base + s * stage_bytes;
                    for (int k0 = k * kStepK; k0 < end * kStepK; k0 += kStepK, dst += kStage) {
                        tma_load_3d<PAIR>(dst, &wmap, full, a.nk ? k0 : n0, a.nk ? n0 : k0, tile.group);
                        tma_load_3d<PAIR>(dst + kHalfBytes, second, full, a.nk ? k0 : n1, a.nk ? n1 : k0, tile.group);
                    }
                    if (++s == stages) { s = 0; ephase ^= 1; }
                }
            }
            // the leader's commits arrive in both blocks: none may still be under way when this one leaves
            for (uint32_t i = 0; PAIR && i < stages && !timed_out; ++i) {
                timed_out = !mbar_wait<PAIR>(bar(B_EMPTY + s), ephase);
                if (++s == stages) { s = 0; ephase ^= 1; }
            }
        }
    } else if (warp == kRowWarp) {
        // =========================== rows' producer ===========================
        // Lane j loads the j-th box, with a row index the j-th four rows.
        const uint32_t full0 = leader_bar(B_FULL);
        uint32_t s = 0, ephase = 1;
        for (int t = unit; t < tiles_total && !timed_out; t += n_units) {
            const Tile tile = groups.at(t, a.feat_tiles, a.block, S::kRound);
            auto boxes_of = [&](int r) { return gather ? (tile.rows + 3) / 4 : (own_rows(tile, r) + a.box_rows - 1) / a.box_rows; };
            const int boxes = boxes_of(rank), all = PAIR ? boxes_of(0) + boxes_of(1) : boxes;
            const uint32_t bytes = all * (gather ? 4 : a.box_rows) * 128;
            const int row = tile.row0 + (PAIR ? rank * half_of(tile) : 0) + lane * a.box_rows;
            const uint32_t place = base + kWBytes + lane * (gather ? 512 : a.box_rows * 128);
            int4 quad = make_int4(0, 0, 0, 0);
            if (gather) {
                int r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int m = 4 * lane + i;
                    r[i] = m < tile.rows ? a.row_index[tile.row0 + m] : 0;
                    if (r[i] < 0 || r[i] >= a.x_rows) {
                        if (a.status) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
                        r[i] = 0;
                    }
                }
                quad = make_int4(r[0], r[1], r[2], r[3]);
            }
            for (int k = k_first; k < k_end; k += sub) {
                // (all lanes step together: one without a box that fell behind would miss a phase that it waits for)
                if (!__all_sync(0xffffffffu, mbar_wait<PAIR>(bar(B_EMPTY + s), ephase))) { timed_out = true; break; }
                const int end = min(k + (int)sub, k_end);
                if (lane == 0 && (!PAIR || rank == 0)) mbar_expect_tx(bar(B_FULL + s), (end - k) * bytes);
                uint32_t dst = place + s * stage_bytes;
                for (int k0 = k * kStepK; k0 < end * kStepK && lane < boxes; k0 += kStepK, dst += kStage) {
                    if (gather) tma_gather4(dst, &xmap, full0 + 8 * s, k0, quad);
                    else tma_load_2d<PAIR>(dst, &xmap, full0 + 8 * s, k0, row);
                }
                if (++s == stages) { s = 0; ephase ^= 1; }
            }
        }
    } else if (warp == kMmaWarp) {
        // ============================ MMA issuer ==============================
        if (lane == 0 && (!PAIR || rank == 0)) {
            // [K, N] weights: rows of k, blocks of 64 features 8 KB apart, 16 k further = 2 KB; [N, K]: rows of features, 16 k
            // further = 32 bytes inside the swizzled row
            const uint32_t w_lo0 = desc_lo(base, a.nk ? 16 : kHalfBytes), x_lo0 = desc_lo(base + kWBytes, 16), hi = desc_hi(1024);
            const uint32_t w_step = a.nk ? 2 : 128;
            bool ok = true;
            uint32_t s = 0, phase = 0, off = 0;
            int it = 0;
            for (int t = unit; t < tiles_total && ok; t += n_units, ++it) {
                const Tile tile = groups.at(t, a.feat_tiles, a.block, S::kRound);
                const uint32_t idesc = instr_desc(BF16, !a.nk, PAIR ? 2 * kFeat : kFeat, (tile.rows + S::kRound - 1) / S::kRound * S::kRound);
                const int buf = it & 1;
                ok = mbar_wait<PAIR>(bar(B_ACC_EMPTY + buf), ((it >> 1) & 1) ^ 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * kTok;
                for (int k = k_first; k < k_end; k += sub) {
                    ok = mbar_wait<PAIR>(bar(B_FULL + s), phase);
                    if (!ok) break;
                    tc_fence_after();
                    mma_ss<PAIR>(d, w_lo0 + off, hi, x_lo0 + off, hi, idesc, k > k_first);
                    mma_ss<PAIR>(d, w_lo0 + off + w_step, hi, x_lo0 + off + 2, hi, idesc, 1);
                    mma_ss<PAIR>(d, w_lo0 + off + 2 * w_step, hi, x_lo0 + off + 4, hi, idesc, 1);
                    mma_ss<PAIR>(d, w_lo0 + off + 3 * w_step, hi, x_lo0 + off + 6, hi, idesc, 1);
                    if (k + 1 < min(k + (int)sub, k_end)) {  // the stage's second K step
                        const uint32_t o = off + (kStage >> 4);
                        mma_ss<PAIR>(d, w_lo0 + o, hi, x_lo0 + o, hi, idesc, 1);
                        mma_ss<PAIR>(d, w_lo0 + o + w_step, hi, x_lo0 + o + 2, hi, idesc, 1);
                        mma_ss<PAIR>(d, w_lo0 + o + 2 * w_step, hi, x_lo0 + o + 4, hi, idesc, 1);
                        mma_ss<PAIR>(d, w_lo0 + o + 3 * w_step, hi, x_lo0 + o + 6, hi, idesc, 1);
                    }
                    tc_commit<PAIR>(bar(B_EMPTY + s));
                    ++s;
                    off += stage_bytes >> 4;
                    if (s == stages) { s = 0; off = 0; phase ^= 1; }
                }
                if (ok) tc_commit<PAIR>(bar(B_ACC_FULL + buf));
            }
            timed_out = !ok;
        }
    } else {
        // ============================== epilogue ==============================
        const int group = warp >> 2, w4 = warp & 3;  // this group takes chunks group, group + 2, ..
        const int sync_id = 1 + group;
        constexpr int kChunk = S::kChunk, kStaged = S::kStaging / 4;
        float* const stage0 = staging + S::kBuffers * group * kStaged;
        bool ok = true, gone = false;  // a warp whose wait ran out; its group then leaves together, at the next tile
        int it = 0, used = 0;          // chunks that this group has staged
        const int cols = a.gated ? 2 : 4;  // columns of out that a lane writes for a token
        // vec: lane l holds columns cols * l ..; else l, l + 32, ..
        const int col0 = a.vec ? cols * lane : lane, col_step = a.vec ? 1 : 32;
        float bias[4] = {}, up_bias[2] = {};
        Tile tile{};
        int buf = 0, n = 0, chunks = 0;
        uint32_t acc = 0;
        // Once per tile: what does not need the accumulator, then the wait for it
        auto release = [&] {  // the accumulator goes back: the next-but-one tile may overwrite it
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(leader_bar(B_ACC_EMPTY + buf));
                else mbar_arrive(bar(B_ACC_EMPTY + buf));
            }
        };
        auto wait_accumulator = [&] {
            if (ok) ok = mbar_wait<PAIR>(bar(B_ACC_FULL + buf), (it >> 1) & 1);
            gone = group_any(sync_id, !ok);
            if (gone) return ok = false;
            tc_fence_after();
            if (group >= chunks) release();
            return true;
        };
        // bias, activation and gate of COUNT tokens' sums
        auto finish = [&](auto& q, auto gated) {
            constexpr int COUNT = sizeof(q) / sizeof(q[0]);
            if constexpr (decltype(gated)::value) {
                float g[2 * COUNT];
#pragma unroll
                for (int j = 0; j < COUNT; ++j) { g[2 * j] = q[j][0] + bias[0]; g[2 * j + 1] = q[j][1] + bias[1]; }
                activate_all(g, a.act);
#pragma unroll
                for (int j = 0; j < COUNT; ++j) { q[j][0] = g[2 * j] * (q[j][2] + up_bias[0]); q[j][1] = g[2 * j + 1] * (q[j][3] + up_bias[1]); }
            } else {
                float h[4 * COUNT];
#pragma unroll
                for (int j = 0; j < 4 * COUNT; ++j) h[j] = q[j / 4][j % 4] + bias[j % 4];
                activate_all(h, a.act);
#pragma unroll
                for (int j = 0; j < 4 * COUNT; ++j) q[j / 4][j % 4] = h[j];
            }
        };

        // Before chunk c is staged: whoever still reads the buffer's last one must be done.  With two buffers that follows from the
        // barrier of the chunk between, with one chunk a tile from the next tile's.
        auto buffer_free = [&](int c) {
            if (S::kBuffers == 1 && kTok > 2 * kChunk && c != group) group_sync(sync_id);
        };
        // A tile of 16-bit rows in whole pieces, the usual case: no branch between the loads of a chunk, the residual on its way
        // to L2 while the MMAs run.  (With the choices made value by value 16 tokens took 1500 clocks, with a residual 5500.)
        auto whole_pieces = [&](auto gated, auto with_residual) {
            constexpr bool GATED = decltype(gated)::value, RES = decltype(with_residual)::value;
            constexpr int kEach = kChunk / 4;
            using Word = std::conditional_t<GATED, uint32_t, uint2>;
            const bool in = n < a.N;  // N is a multiple of cols
            const int64_t row0 = tile.row0 + group * kChunk + w4;
            T* out = static_cast<T*>(a.out) + row0 * a.out_stride + n;
            const T* res = RES ? static_cast<const T*>(a.residual) + row0 * a.res_stride + n : nullptr;
            if constexpr (RES) {
                // 16 lanes cover a row's 128 bytes of pieces: one of them asks for the line
                for (int m = 4 * group + w4; m < tile.rows; m += 8)
                    if (in && (lane & 15) == 0)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const T*>(a.residual) + (tile.row0 + m) * a.res_stride + n));
            }
            if (!wait_accumulator()) return;
            for (int c = group; c < chunks; c += 2, ++used) {
                float* stage = stage0 + (S::kBuffers == 2 ? (used & 1) * kStaged : 0);
                const int left = tile.rows - c * kChunk;
                Word r[RES ? kEach : 1];
                if constexpr (RES) {
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        r[i] = Word{};
                        if (in && w4 + 4 * i < left) r[i] = *reinterpret_cast<const Word*>(res + 4 * i * a.res_stride);
                    }
                    res += 2 * kChunk * a.res_stride;
                }
                {
                    float v[kChunk];
                    tmem_ld<kChunk>(acc + c * kChunk, v);
                    if (c + 2 >= chunks) release();
                    buffer_free(c);
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) stage[i * kFeat + w4 * 32 + lane] = v[i];
                }
                group_sync(sync_id);
                float q[kEach][4];
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const uint32_t row = smem_u32(stage + (w4 + 4 * i) * kFeat);
                    if constexpr (GATED) {
                        ld_shared<2, false>(q[i], row + 8u * (uint32_t)lane);
                        ld_shared<2, false>(q[i] + 2, row + 256u + 8u * (uint32_t)lane);
                    } else {
                        ld_shared<4, false>(q[i], row + 16u * (uint32_t)lane);
                    }
                }
                finish(q, gated);
                if constexpr (RES) {
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        if constexpr (GATED) {
                            const float2 f = unpack2<BF16>(r[i]);
                            q[i][0] += f.x; q[i][1] += f.y;
                        } else {
                            const float2 f = unpack2<BF16>(r[i].x), g = unpack2<BF16>(r[i].y);
                            q[i][0] += f.x; q[i][1] += f.y; q[i][2] += g.x; q[i][3] += g.y;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    if (in && w4 + 4 * i < left) {
                        if constexpr (GATED) *reinterpret_cast<uint32_t*>(out + 4 * i * a.out_stride) = pack2<BF16>(q[i][0], q[i][1]);
                        else *reinterpret_cast<uint2*>(out + 4 * i * a.out_stride) = make_uint2(pack2<BF16>(q[i][0], q[i][1]), pack2<BF16>(q[i][2], q[i][3]));
                    }
                out += 2 * kChunk * a.out_stride;
            }
        };

        // Every other form (fp32 out, rows that do not divide into pieces, K split over a cluster), one token at a time
        auto residual_of = [&](int64_t row, float (&r)[4]) {
            auto each = [&](auto* p) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < cols && n + i * col_step < a.N) r[i] = to_float(p[row * a.res_stride + n + i * col_step]);
            };
            if (!a.residual) return;
            if (a.out_f32) each(static_cast<const float*>(a.residual));
            else each(static_cast<const T*>(a.residual));
        };
        auto one_token = [&](float (&q)[1][4], const float (&r)[4], int64_t row) {
            if (a.gated) finish(q, std::true_type{});
            else finish(q, std::false_type{});
            auto each = [&](auto* p) {
                using O = std::remove_pointer_t<decltype(p)>;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < cols && n + i * col_step < a.N) p[row * a.out_stride + n + i * col_step] = from_float<O>(a.residual ? q[0][i] + r[i] : q[0][i]);
            };
            if (a.out_f32) each(static_cast<float*>(a.out));
            else each(static_cast<T*>(a.out));
        };
        // a token's staged sums for this lane, from the row at `addr` (of any block): its columns; with a gate those of the gate,
        // then those of the up projection
        auto staged = [&](uint32_t addr, auto peer, float (&q)[4]) {
            constexpr bool P = decltype(peer)::value;
            if (!a.vec) {
#pragma unroll
                for (int i = 0; i < 4; ++i) ld_shared<1, P>(q + i, addr + 4u * (uint32_t)(lane + 32 * i));
            } else if (a.gated) {
                ld_shared<2, P>(q, addr + 8u * (uint32_t)lane);
                ld_shared<2, P>(q + 2, addr + 256u + 8u * (uint32_t)lane);
            } else {
                ld_shared<4, P>(q, addr + 16u * (uint32_t)lane);
            }
        };
        auto any_form = [&] {
            if (!wait_accumulator()) return;
            for (int c = group; c < chunks; c += 2, ++used) {
                const int left = tile.rows - c * kChunk;
                float* stage = stage0 + (S::kBuffers == 2 ? (used & 1) * kStaged : 0);
                float v[kChunk];
                tmem_ld<kChunk>(acc + c * kChunk, v);
                if (c + 2 >= chunks) release();
                buffer_free(c);
#pragma unroll
                for (int i = 0; i < kChunk; ++i) stage[i * kFeat + w4 * 32 + lane] = v[i];
                group_sync(sync_id);
                for (int m = w4; m < min(left, kChunk); m += 4) {
                    float q[1][4], r[4] = {};
                    residual_of(tile.row0 + c * kChunk + m, r);
                    staged(smem_u32(stage + m * kFeat), std::false_type{}, q[0]);
                    one_token(q, r, tile.row0 + c * kChunk + m);
                }
            }
        };
        // K split: this block's sums into its own shared memory, then its share of the tokens over everyone's
        auto split_form = [&] {
            const bool there = wait_accumulator();
            float* sums = reinterpret_cast<float*>(base_ptr);  // all MMAs are done: the operands' room is free
            for (int c = group; there && c < chunks; c += 2) {
                float v[kChunk];
                tmem_ld<kChunk>(acc + c * kChunk, v);
#pragma unroll
                for (int i = 0; i < kChunk; ++i)
                    if (c * kChunk + i < tile.rows) sums[(c * kChunk + i) * kFeat + w4 * 32 + lane] = v[i];
            }
            int m = rank * kEpilogueWarps + warp;
            float r[4] = {};
            if (m < tile.rows) residual_of(tile.row0 + m, r);
            __syncwarp();
            cluster_sync();  // (1)
            for (; there && m < tile.rows; m += split * kEpilogueWarps) {
                float q[1][4] = {}, part[kMaxSplit][4];
#pragma unroll
                for (int p = 0; p < kMaxSplit; ++p)
                    if (p < split) staged(peer_addr(smem_u32(sums + m * kFeat), p), std::true_type{}, part[p]);
#pragma unroll
                for (int p = 0; p < kMaxSplit; ++p)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (p < split) q[0][i] += part[p][i];
                if (m >= split * kEpilogueWarps) residual_of(tile.row0 + m, r);
                one_token(q, r, tile.row0 + m);
            }
        };

        const bool whole = a.vec && !a.out_f32;
        for (int t = unit; t < tiles_total && !gone; t += n_units, ++it) {  // (split: at most once)
            tile = groups.at(t, a.feat_tiles, a.block, S::kRound);
            buf = it & 1;
            n = column0(tile) + col0;
            chunks = (tile.rows + kChunk - 1) / kChunk;
            acc = tmem + ((uint32_t)(w4 * 32) << 16) + buf * kTok;
            const T* bp = a.bias ? static_cast<const T*>(a.bias) + tile.group * a.bias_stride : nullptr;
            const T* cp = a.up_bias ? static_cast<const T*>(a.up_bias) + tile.group * a.up_bias_stride : nullptr;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = n + i * col_step;
                const bool in = i < cols && c < a.N;
                bias[i] = bp && in ? to_float(bp[c]) : 0.f;
                if (i < 2) up_bias[i] = cp && in ? to_float(cp[c]) : 0.f;
            }
            if (split > 1) split_form();
            else if (!whole) any_form();
            else if (a.gated && a.residual) whole_pieces(std::true_type{}, std::true_type{});
            else if (a.gated) whole_pieces(std::true_type{}, std::false_type{});
            else if (a.residual) whole_pieces(std::false_type{}, std::true_type{});
            else whole_pieces(std::false_type{}, std::false_type{});
        }
        timed_out = !ok;
    }
    if (timed_out) settle();
    if (timed_out && a.status && lane == 0) atomicOr(a.status, SFB_STATUS_WAIT_TIMEOUT);
    // ---- teardown: every warp arrives here; in a cluster no block leaves while another may still use its shared memory
    __syncwarp();
    if (split > 1 && (warp >= kEpilogueWarps || unit >= tiles_total)) cluster_sync();  // (1), where not passed above
    tc_fence_before();
    __syncthreads();
    if (cluster > 1) cluster_sync();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc<PAIR>(tmem, 2 * kTok);
    }
}

// Rows of x in the order of out: ordered[r, :] = x[row_index[r], :].  A warp keeps 2 KB of the rows and walks them, the index read
// one row ahead.  Only an index that is no row needs the groups: inside one it counts as row 0 and is flagged, outside it is what
// the router leaves behind the last row and nothing is written.  (Rows outside every group with an index that is a row are copied
// like the others; nobody reads them.)  16384 rows of 4096 take
// 23 us, 4096 of 1024 2.5 (a block a row, its 256 threads in step and without the index ahead: 26 and 4.7).
constexpr int kPieceValues = 1024;
__global__ void __launch_bounds__(256) order_rows_kernel(const uint16_t* __restrict__ x, int64_t x_stride, const int32_t* __restrict__ row_index,
                                                         const int32_t* __restrict__ offsets, int groups, int rows, int x_rows, int K, int pieces,
                                                         uint16_t* __restrict__ ordered, int64_t ordered_stride, int* status) {
    wait_for_previous();
    let_next_start();  // in this order: what the next kernel reads of others than this one is then there when it starts
    const int lane = threadIdx.x & 31;
    const int block = (int)blockIdx.x / pieces, p = (int)blockIdx.x - block * pieces, step = (int)gridDim.x / pieces * 8;
    int r = block * 8 + (int)(threadIdx.x >> 5);
    int next = r < rows ? row_index[r] : 0;
    int first = -1, end = -1;  // of the rows inside groups, once asked for
    for (; r < rows; r += step) {
        int i = next;
        if (r + step < rows) next = row_index[r + step];
        if (i < 0 || i >= x_rows) {
            if (first < 0) {
                first = group_offset(offsets[0], 0, rows);
                end = first;
                for (int e = lane; e < groups; e += 32) end = group_offset(offsets[e + 1], end, rows);
                end = __reduce_max_sync(0xffffffffu, end);
            }
            if (r < first || r >= end) continue;
            if (status && lane == 0) atomicOr(status, SFB_STATUS_BAD_ROW_INDEX);
            i = 0;
        }
        const uint16_t* src = x + (int64_t)i * x_stride;
        uint16_t* dst = ordered + (int64_t)r * ordered_stride;
        const int c = p * kPieceValues + lane * 8;
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j * 256 + 8 <= K) v[j] = *reinterpret_cast<const uint4*>(src + c + j * 256);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j * 256 + 8 <= K) *reinterpret_cast<uint4*>(dst + c + j * 256) = v[j];
        const int tail = K & ~7;
        if (p == pieces - 1 && lane < K - tail) dst[tail + lane] = src[tail + lane];
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static std::once_flag once;
    static EncodeTiledFn fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) == cudaSuccess &&
            res == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// A map over 16-bit values [d2, d1, d0] (rank 2: [d1, d0]) with a box of 64 x box1 (x 1), 128-byte swizzle.
bool encode(CUtensorMap* map, const void* base, int rank, int64_t d0, int64_t d1, int64_t d2, int64_t stride1, int64_t stride2, int box1) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)d0, (cuuint64_t)d1, (cuuint64_t)d2};
    const cuuint64_t strides[2] = {(cuuint64_t)stride1 * 2, (cuuint64_t)stride2 * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box1, 1};
    const cuuint32_t es[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What TMA can address: bases and row strides in multiples of 16 bytes, rows that do not overlap.
bool rows_for_tma(const void* base, int64_t inner, int64_t rows, int64_t stride, int64_t outer, int64_t outer_stride) {
    if (reinterpret_cast<uintptr_t>(base) % 16) return false;
    if (rows > 1 && (stride % 8 || stride < inner)) return false;
    return outer <= 1 || (outer_stride % 8 == 0 && outer_stride >= 8 && outer_stride < (1LL << 38));
}

// How many clusters of `size` blocks of a kernel, one block an SM, the device holds at once (0: none); asked once per kernel,
// device and size.
int resident_clusters(const void* kernel, int size, int dev, int sms) {
    struct Known { const void* kernel; int size, dev, clusters; };
    constexpr int kMost = 1024;  // kernels x sizes x devices of any machine; asked again beyond
    static std::mutex mu;
    static Known known[kMost];
    static int count = 0;
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < count; ++i)
        if (known[i].kernel == kernel && known[i].size == size && known[i].dev == dev) return known[i].clusters;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)size; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(sms / size * size)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = kSmemPerBlock;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) clusters = 0;
    cudaGetLastError();  // a refusal only means "not available"
    clusters = std::max(0, std::min(clusters, sms / size));
    if (count < kMost) known[count++] = {kernel, size, dev, clusters};
    return clusters;
}

template <typename S, bool BF16>
int launch_tiles(const CUtensorMap* maps, TileArgs a, int64_t units, bool shared_sm, int dev, int sms, cudaStream_t stream) {
    auto kernel = linear_tcgen05_kernel<S, BF16>;
    const void* k = reinterpret_cast<const void*>(kernel);
    const int rc = allow_shared_memory_once(k, kSmemPerBlock);
    if (rc != SFB_OK) return rc;
    a.sub = shared_sm ? 1 : 2;
    a.stages = S::stages(shared_sm ? kSmemPerHalf : kSmemPerBlock, a.groups, a.sub);
    const int cluster = S::kPair ? 2 : a.split, smem = S::smem(a.stages * a.sub, a.groups);
    int resident = sms * (shared_sm ? 2 : 1);
    if (cluster > 1 && (resident = resident_clusters(k, cluster, dev, sms)) == 0)
        return fail(SFB_ERR_CUDA, "linear: the device holds no cluster of %d thread blocks", cluster);
    const unsigned grid = (unsigned)((a.split > 1 ? units : std::min<int64_t>(units, resident)) * cluster);
    return launch_after(kernel, grid, kThreads, smem, (unsigned)cluster, stream, maps[0], maps[1], maps[2], a);
}

}  // namespace

// Every candidate shape is priced in clocks: a start and the last tile's epilogue, and between them the longer of the weights'
// way from HBM (3400 bytes a clock) and the rounds of tiles on the busiest SM x their K steps x a step.  A step takes the longest
// of its MMAs (2 clocks a token column, with what lies between them 2.3 for a
// pair), its operands' way into shared memory (72 bytes a clock an SM), the issuing thread's chain (380 clocks with two steps a stage, 600 with one) and the row gathers (62 clocks for four rows); two blocks an SM share
// the first two.  A split launches a cluster for every tile and exchanges sums at its end; how many clusters run at once goes
// by the smallest of the eight groups of SMs that a cluster must lie in.
static LinearPlan price_shapes(int64_t rows, int64_t K, int64_t N, int64_t groups, bool grouped, bool gated, bool indexed, bool ordered, int sms) {
    LinearPlan best{};
    int64_t best_cost = -1;
    const int64_t n_k = ceil_div(K, (int64_t)kStepK), mean = grouped ? ceil_div(rows, groups) : rows, used = grouped ? std::min(groups, rows) : 1;
    // only the mean of the groups is known here: a group is taken to have two standard deviations of an even draw more
    const int64_t likely = grouped ? mean + (int64_t)(2 * std::sqrt((double)mean)) : rows;
    const int64_t from_hbm = used * K * N * (gated ? 4 : 2) / 3400;
    auto consider = [&](int tokens, bool pair, int split, bool order) {
        const int64_t tiles_a_group = ceil_div(likely, (int64_t)tokens), width = ceil_div(ceil_div(mean, ceil_div(mean, (int64_t)tokens)), (int64_t)16) * 16;
        const int64_t feat_tiles = ceil_div(N, (int64_t)((gated ? kFeat / 2 : kFeat) * (pair ? 2 : 1)));
        const int64_t tiles = used * tiles_a_group * feat_tiles, blocks = tiles * (pair ? 2 : split);
        const int an_sm = tokens <= 64 && blocks > sms ? 2 : 1;
        const int64_t slots = std::max<int64_t>(1, pair ? sms / 2 : split == 1 ? sms * an_sm : 8 * (std::max(1, sms / 8 - 2) * an_sm / split));
        const int64_t rounds = ceil_div(tiles, slots), bytes = kWBytes + width * (pair ? 64 : 128);
        int64_t step = std::max<int64_t>(an_sm * std::max(pair ? 23 * width / 10 : 2 * width, bytes / 72), an_sm == 2 ? 600 : 380);
        if (indexed && !order) step = std::max(step, an_sm * std::min(width, mean) / 4 * 62);
        // an uneven last round costs bandwidth too, if less than its share
        const int64_t hbm = rounds > 1 ? (from_hbm + from_hbm * rounds * slots / tiles) / 2 : from_hbm, on_sm = rounds * ceil_div(n_k, (int64_t)split) * step;
        // the two overlap, but not wholly
        int64_t cost = 6000 + 25 * width + std::max(hbm, on_sm) + std::min(hbm, on_sm) / 4 + (an_sm - 1) * 1500;
        if (split > 1) cost += 3000 + 300 * split + 6000 * (rounds - 1);
        if (order) cost += 1500 + rows * K / 2000;  // the pass that orders the rows
        if (best_cost < 0 || cost < best_cost) { best_cost = cost; best = {tokens, pair ? 1 : 0, split, order ? 1 : 0, an_sm, feat_tiles}; }
    };
    for (int order = 0; order <= (indexed && ordered ? 1 : 0); ++order) {
        for (int tokens : {32, 64, 128})
            for (int split = 1; split <= kMaxSplit && split <= n_k; ++split) consider(tokens, false, split, order);
        if (!indexed || order) consider(256, true, 1, order);
    }
    return best;
}

// Pricing takes two microseconds of host time and a program calls with the same sizes again and again: each thread keeps the
// shapes of the last sizes it met.
LinearPlan plan_linear(int64_t rows, int64_t K, int64_t N, int64_t groups, bool grouped, bool gated, bool indexed, bool ordered, int sms) {
    struct Priced { int64_t rows, K, N, groups; int flags, sms; LinearPlan plan; };
    thread_local Priced known[64] = {};
    const int flags = 16 | grouped | gated << 1 | indexed << 2 | ordered << 3;
    Priced& p = known[(uint64_t)(rows * 31 + K * 17 + N * 7 + groups * 3 + flags) * 0x9e3779b97f4a7c15ULL >> 58];
    if (p.rows != rows || p.K != K || p.N != N || p.groups != groups || p.flags != flags || p.sms != sms)
        p = {rows, K, N, groups, flags, sms, price_shapes(rows, K, N, groups, grouped, gated, indexed, ordered, sms)};
    return p.plan;
}

int launch_linear_tcgen05(const LinearArgs& in, cudaStream_t stream) {
    if (in.dtype != SFB_BF16 && in.dtype != SFB_F16) return SFB_ERR_UNSUPPORTED;
    const bool nk = in.w_stride[1] == 1 && in.layout == SFB_WEIGHT_NK;
    const int64_t inner = nk ? in.K : in.N, outer = nk ? in.N : in.K;
    const int ri = nk ? 2 : 1;  // the stride between rows of the stored matrix
    if (!rows_for_tma(in.x, in.K, in.x_rows, in.x_stride, 1, 0) || !rows_for_tma(in.w, inner, outer, in.w_stride[ri], in.groups, in.w_stride[0]) ||
        (in.up && !rows_for_tma(in.up, inner, outer, in.up_stride[ri], in.groups, in.up_stride[0])))
        return SFB_ERR_UNSUPPORTED;
    int dev = 0, sms = 0;
    SFB_CUDA_CHECK(cudaGetDevice(&dev));
    SFB_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // rows by their index: the pass that puts them in order needs a workspace
    const int64_t ordered_stride = ceil_div(in.K, (int64_t)8) * 8, ordered_bytes = in.rows * ordered_stride * 2;
    const bool can_order = in.row_index && in.workspace && in.workspace_bytes >= ordered_bytes && reinterpret_cast<uintptr_t>(in.workspace) % 16 == 0;
    const LinearPlan plan = plan_linear(in.rows, in.K, in.N, in.groups, in.offsets != nullptr, in.up != nullptr, in.row_index != nullptr, can_order, sms);
    const int64_t token_tiles = ceil_div(in.rows, (int64_t)plan.tokens) + (in.offsets ? std::min(in.groups, in.rows) : 0);
    if (token_tiles * plan.feat_tiles > 0x7fffffffLL) return SFB_ERR_UNSUPPORTED;

    TileArgs a{};
    a.bias = in.bias; a.up_bias = in.up_bias; a.residual = in.residual; a.out = in.out;
    a.offsets = in.offsets; a.row_index = plan.order ? nullptr : in.row_index; a.status = in.status;
    a.out_stride = in.out_stride; a.res_stride = in.res_stride; a.bias_stride = in.bias_stride; a.up_bias_stride = in.up_bias_stride;
    a.rows = (int)in.rows; a.x_rows = (int)in.x_rows; a.N = (int)in.N; a.n_k = (int)ceil_div(in.K, (int64_t)kStepK); a.groups = (int)in.groups;
    a.feat_tiles = (int)plan.feat_tiles; a.split = plan.split; a.act = in.act;
    a.gated = in.up != nullptr; a.nk = nk; a.out_f32 = in.out_dtype == SFB_F32;
    a.ordered = plan.order;
    a.block = 8;
    // rows of a box: all where they fit one (in eights); else 32, or 64 of a pair's 128, the last one bringing in some too many
    a.box_rows = !in.offsets && in.rows <= 32 ? (int)(ceil_div(in.rows, (int64_t)8) * 8) : plan.pair ? 64 : 32;
    const bool order = plan.order;
    const void* x = order ? in.workspace : in.x;
    const int64_t x_rows = order ? in.rows : in.x_rows, x_row = order || x_rows == 1 ? ordered_stride : in.x_stride;
    if (order) {
        const int64_t pieces = ceil_div(in.K, (int64_t)kPieceValues), blocks = pieces * std::min(ceil_div(in.rows, (int64_t)8), std::max<int64_t>(1, 8 * sms / pieces));
        const int rc = launch_after(order_rows_kernel, (unsigned)blocks, 256, 0, 1, stream, static_cast<const uint16_t*>(in.x), in.x_stride, in.row_index,
                                    in.offsets, (int)in.groups, (int)in.rows, (int)in.x_rows, (int)in.K, (int)pieces,
                                    static_cast<uint16_t*>(in.workspace), ordered_stride, in.status);
        if (rc != SFB_OK) return rc;
    }
    // rows of out and residual in pieces of `cols` values where all of them start on one
    const int cols = a.gated ? 2 : 4, piece = cols * (a.out_f32 ? 4 : 2);
    auto pieces = [&](const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % piece == 0 && stride % cols == 0; };
    a.vec = in.N % cols == 0 && pieces(in.out, in.out_stride) && (!in.residual || pieces(in.residual, in.res_stride));

    CUtensorMap maps[3];
    auto weight = [&](CUtensorMap* m, const void* base, const int64_t* stride) {
        const int64_t row = outer > 1 ? stride[ri] : ceil_div(inner, (int64_t)8) * 8, group = in.groups > 1 ? stride[0] : 8;
        return encode(m, base, 3, inner, outer, in.groups, row, group, 64);
    };
    if (!encode(&maps[0], x, 2, in.K, x_rows, 1, x_row, 0, a.row_index ? 1 : a.box_rows) || !weight(&maps[1], in.w, in.w_stride)) return SFB_ERR_UNSUPPORTED;
    if (in.up) { if (!weight(&maps[2], in.up, in.up_stride)) return SFB_ERR_UNSUPPORTED; }
    else maps[2] = maps[1];

    const int64_t units = token_tiles * plan.feat_tiles;
    const bool bf16 = in.dtype == SFB_BF16;
    auto go = [&](auto shape) {
        using S = decltype(shape);
        return bf16 ? launch_tiles<S, true>(maps, a, units, plan.blocks_an_sm == 2, dev, sms, stream) : launch_tiles<S, false>(maps, a, units, plan.blocks_an_sm == 2, dev, sms, stream);
    };
    if (plan.pair) return go(ShapePair{});
    return plan.tokens == 32 ? go(Shape32{}) : plan.tokens == 64 ? go(Shape64{}) : go(Shape128{});
}

}  // namespace sfb
