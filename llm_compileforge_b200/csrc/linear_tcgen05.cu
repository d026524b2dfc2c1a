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
//   warp 4    TMA producer: per 64-wide K step two boxes of 64 features, and the token rows as boxes of box_rows rows or, with a
//             row index, four rows per gather load; one lane per box
//   warp 5    one thread issues tcgen05.mma kind::f16 (M 128, N = tokens, K 16, four per step); the weight operand is
//             MN-major for [K, N] storage and K-major for [N, K], straight from 128-byte-swizzled shared memory
//   warps 0-3 epilogue: 16 tokens at a time through a transposing buffer in shared memory, so that rows of out and
//             residual move as 8 bytes a lane; bias, activation, gate, residual in fp32, one rounding
// Few tiles (decode): a cluster of up to eight thread blocks shares a tile, each taking a part of K; the parts meet in the
// epilogue through distributed shared memory, summed in the order of the ranks - no workspace, no atomics, the same bits
// every time.
// Group offsets are read on the device; each thread block lays the groups' tiles out in shared memory before it starts.
// Every wait is bounded; one that runs out sets SFB_STATUS_WAIT_TIMEOUT and the block leaves through the common teardown.

#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "linear.cuh"

namespace sfb {
namespace {

constexpr int kFeat = 128, kStepK = 64, kChunk = 16;
constexpr int kWBytes = kFeat * kStepK * 2;      // a K step's weights: two boxes of 64 features
constexpr int kHalfBytes = kWBytes / 2;
constexpr int kStaging = kChunk * kFeat * 4;     // fp32 [16 tokens][128 features]
constexpr int kThreads = 192;
constexpr uint32_t kSpin = 1u << 21;
constexpr int kMaxSplit = 8;

constexpr int kMaxStages = 9;
enum {
    B_FULL = 0,
    B_EMPTY = kMaxStages,
    B_ACC_FULL = 2 * kMaxStages,
    B_ACC_EMPTY = B_ACC_FULL + 2,
    B_PART_FULL = B_ACC_EMPTY + 2,   // a chunk's partial sums lie in every block's staging buffer
    B_PART_EMPTY = B_PART_FULL + 2,  // every block has read the chunk
    B_COUNT = B_PART_EMPTY + 2
};

constexpr int stage_bytes(int tok) { return kWBytes + tok * 128; }
constexpr int smem_bytes(int tok, int stages, int groups) {
    return 1024 + stages * stage_bytes(tok) + 2 * kStaging + B_COUNT * 8 + 16 + (3 * groups + 1) * 4;
}

struct TileArgs {
    const void *bias, *up_bias, *residual;
    void* out;
    const int32_t *offsets, *row_index;
    int* status;
    int64_t out_stride, res_stride, bias_stride, up_bias_stride;
    int rows, x_rows, N, n_k, groups;
    int feat_tiles;  // column tiles of out
    int box_rows;    // token rows of one TMA box
    int split;       // thread blocks that share a tile's K steps (= cluster size)
    int block;       // token tiles that run together through the feature tiles (L2 reuse of x and W)
    int act;
    bool gated, nk, out_f32, vec;
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
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < kSpin; ++i) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}
// The same for barriers on which other blocks of the cluster arrive: what they wrote before is visible after.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < kSpin; ++i) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
    }
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
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
                 : "memory");
}
// Four rows of a map whose box is one row high, side by side at dst.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int4 r) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %2};\n mov.b64 db, {%3, %4};\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n}\n"
        ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
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
// Whether any of the four epilogue warps failed; all of them come here, so none waits for one that has left.
__device__ __forceinline__ bool epilogue_any(bool failed) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r)
                 : "r"((uint32_t)failed)
                 : "memory");
    return r != 0;
}
__device__ __forceinline__ void epilogue_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

template <int W>
__device__ __forceinline__ void activate_all(float (&h)[W], int act) {
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < W; ++i) h[i] = f(h[i]);
    };
    if (act == SFB_ACT_SILU) each([](float v) { return __fdividef(v, 1.f + __expf(-v)); });
    else if (act == SFB_ACT_GELU) each([](float v) { return activate<SFB_ACT_GELU>(v); });
    else if (act == SFB_ACT_GELU_TANH) each([](float v) { return __fdividef(v, 1.f + __expf(-1.5957691216057308f * (v + 0.044715f * v * v * v))); });
    else if (act == SFB_ACT_RELU) each([](float v) { return activate<SFB_ACT_RELU>(v); });
}

struct Tile {
    int group, row0, rows, feat;
};
// The groups of a call in shared memory: first row, number of rows, and token tiles before each group.
struct Groups {
    const int *lo, *count, *tiles;
    int n;
    // Tile t: groups one after another; inside a group blocks of `block` token tiles, token tiles fastest, then features.  A
    // group's rows are spread evenly over its token tiles, in sixteens.
    __device__ __forceinline__ Tile at(int t, int tok, int feat_tiles, int block) const {
        int e = 0;
        for (int step = 512; step > 0; step >>= 1)
            if (e + step < n && tiles[e + step] * feat_tiles <= t) e += step;
        const int nt = tiles[e + 1] - tiles[e];
        int i = t - tiles[e] * feat_tiles;
        const int b = i / (block * feat_tiles);
        const int g = min(block, nt - b * block);
        i -= b * block * feat_tiles;
        const int f = i / g, m = b * block + i - f * g;
        const int per = token_rows(count[e], nt);
        return {e, lo[e] + m * per, min(per, count[e] - m * per), f};
    }
    static __device__ __forceinline__ int token_rows(int count, int nt) { return (((count + nt - 1) / nt) + 15) & ~15; }
};

template <int kTok, int kStages, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
linear_tcgen05_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap umap,
                      const TileArgs a) {
    extern __shared__ uint8_t smem_raw[];
    static_assert(kStages <= kMaxStages, "barrier slots");
    constexpr int kStage = stage_bytes(kTok);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = a.split;
    const int rank = split > 1 ? (int)cluster_rank() : 0;
    const int unit = (int)blockIdx.x / split, n_units = (int)gridDim.x / split;

    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    float* staging = reinterpret_cast<float*>(base_ptr + kStages * kStage);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base_ptr + kStages * kStage + 2 * kStaging);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + B_COUNT);
    int* g_lo = reinterpret_cast<int*>(tmem_slot + 4);
    int* g_count = g_lo + a.groups;
    int* g_tiles = g_count + a.groups;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar(B_FULL + s), 1);
            mbar_init(bar(B_EMPTY + s), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(B_ACC_FULL + i), 1);
            mbar_init(bar(B_ACC_EMPTY + i), 4);
            mbar_init(bar(B_PART_FULL + i), 4 * split);
            mbar_init(bar(B_PART_EMPTY + i), 4 * split);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 5) tmem_alloc(smem_u32(tmem_slot), 2 * kTok);
    if (warp == 0) {  // the groups' rows, and the running number of token tiles
        int before = 0, top = a.offsets ? group_offset(a.offsets[0], 0, a.rows) : 0;
        bool bad = a.offsets && top != a.offsets[0];
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
            if (e < a.groups) { g_lo[e] = lo; g_count[e] = hi - lo; g_tiles[e] = before + sum - own; }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) g_tiles[a.groups] = before;
        if (bad && a.status) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
    }
    tc_fence_before();
    __syncthreads();
    if (split > 1) cluster_sync();  // the other blocks' barriers exist before anything is sent to them
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Groups groups{g_lo, g_count, g_tiles, a.groups};
    const int tiles_total = g_tiles[a.groups] * a.feat_tiles;
    const int k_first = (int)((int64_t)a.n_k * rank / split), k_end = (int)((int64_t)a.n_k * (rank + 1) / split);
    const int feats = a.gated ? kFeat / 2 : kFeat;  // columns of out in a tile
    bool timed_out = false;

    if (warp == 4) {
        // ============================ TMA producer ============================
        // Lanes 0 and 1 load the weights; without a row index lane 2 + j loads token box j, with one every lane the rows of
        // its quads of tokens.
        uint32_t s = 0, ephase = 1;
        for (int t = unit; t < tiles_total && !timed_out; t += n_units) {
            const Tile tile = groups.at(t, kTok, a.feat_tiles, a.block);
            const int n0 = tile.feat * feats + (a.gated ? 0 : lane * 64);  // lanes 0 and 1
            const CUtensorMap* my_w = a.gated && lane == 1 ? &umap : &wmap;
            const int boxes = a.row_index ? (tile.rows + 3) / 4 : (tile.rows + a.box_rows - 1) / a.box_rows;
            const uint32_t bytes = kWBytes + boxes * (a.row_index ? 4 : a.box_rows) * 128;
            int4 quad[kTok / 128 > 0 ? (kTok + 127) / 128 : 1];
            constexpr int kQuads = sizeof(quad) / sizeof(quad[0]);
            if (a.row_index) {
#pragma unroll
                for (int q = 0; q < kQuads; ++q) {
                    int r[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int m = 4 * (lane + 32 * q) + i;
                        r[i] = m < tile.rows ? a.row_index[tile.row0 + m] : 0;
                        if (r[i] < 0 || r[i] >= a.x_rows) {
                            if (a.status) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
                            r[i] = 0;
                        }
                    }
                    quad[q] = make_int4(r[0], r[1], r[2], r[3]);
                }
            }
            for (int k = k_first; k < k_end; ++k) {
                if (!mbar_wait(bar0 + 8u * (B_EMPTY + s), ephase)) { timed_out = true; break; }
                const uint32_t full = bar0 + 8u * (B_FULL + s), dst = base + s * kStage;
                if (lane == 0) mbar_expect_tx(full, bytes);
                __syncwarp();
                const int k0 = k * kStepK;
                if (lane < 2) tma_load_3d(dst + lane * kHalfBytes, my_w, full, a.nk ? k0 : n0, a.nk ? n0 : k0, tile.group);
                if (a.row_index) {
#pragma unroll
                    for (int q = 0; q < kQuads; ++q)
                        if (lane + 32 * q < boxes) tma_gather4(dst + kWBytes + (lane + 32 * q) * 512, &xmap, full, k0, quad[q]);
                } else if (lane >= 2 && lane - 2 < boxes) {
                    tma_load_2d(dst + kWBytes + (lane - 2) * a.box_rows * 128, &xmap, full, k0, tile.row0 + (lane - 2) * a.box_rows);
                }
                if (++s == kStages) { s = 0; ephase ^= 1; }
            }
        }
        timed_out = __any_sync(0xffffffffu, timed_out);
    } else if (warp == 5) {
        // ============================ MMA issuer ==============================
        if (lane == 0) {
            // [K, N] weights: rows of k, blocks of 64 features 8 KB apart, 16 k further = 2 KB; [N, K]: rows of features, 16 k
            // further = 32 bytes inside the swizzled row
            const uint32_t w_lo0 = desc_lo(base, a.nk ? 16 : kHalfBytes), x_lo0 = desc_lo(base + kWBytes, 16), hi = desc_hi(1024);
            const uint32_t w_step = a.nk ? 2 : 128;
            bool ok = true;
            uint32_t s = 0, phase = 0, off = 0;
            int it = 0;
            for (int t = unit; t < tiles_total && ok; t += n_units, ++it) {
                const Tile tile = groups.at(t, kTok, a.feat_tiles, a.block);
                const uint32_t idesc = instr_desc(BF16, !a.nk, kFeat, (tile.rows + 15) & ~15);
                const int buf = it & 1;
                ok = mbar_wait(bar(B_ACC_EMPTY + buf), ((it >> 1) & 1) ^ 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * kTok;
                for (int k = k_first; k < k_end; ++k) {
                    ok = mbar_wait(bar0 + 8u * (B_FULL + s), phase);
                    if (!ok) break;
                    tc_fence_after();
                    mma_ss(d, w_lo0 + off, hi, x_lo0 + off, hi, idesc, k > k_first);
                    mma_ss(d, w_lo0 + off + w_step, hi, x_lo0 + off + 2, hi, idesc, 1);
                    mma_ss(d, w_lo0 + off + 2 * w_step, hi, x_lo0 + off + 4, hi, idesc, 1);
                    mma_ss(d, w_lo0 + off + 3 * w_step, hi, x_lo0 + off + 6, hi, idesc, 1);
                    tc_commit(bar0 + 8u * (B_EMPTY + s));
                    ++s;
                    off += kStage >> 4;
                    if (s == kStages) { s = 0; off = 0; phase ^= 1; }
                }
                if (ok) tc_commit(bar(B_ACC_FULL + buf));
            }
            timed_out = !ok;
        }
    } else {
        // ============================== epilogue ==============================
        using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
        bool ok = true;
        int it = 0, chunk = 0;
        const int cols = a.gated ? 2 : 4;  // columns of out that a lane writes for a token
        for (int t = unit; t < tiles_total; t += n_units, ++it) {
            const Tile tile = groups.at(t, kTok, a.feat_tiles, a.block);
            const int buf = it & 1, n0 = tile.feat * feats;
            // vec: lane l holds columns cols * l ..; else l, l + 32, ..
            const int col0 = a.vec ? cols * lane : lane, col_step = a.vec ? 1 : 32;
            float bias[4] = {}, up_bias[4] = {};
            const T* bp = a.bias ? static_cast<const T*>(a.bias) + tile.group * a.bias_stride : nullptr;
            const T* cp = a.up_bias ? static_cast<const T*>(a.up_bias) + tile.group * a.up_bias_stride : nullptr;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = n0 + col0 + i * col_step;
                if (i < cols && n < a.N) {
                    if (bp) bias[i] = to_float(bp[n]);
                    if (cp) up_bias[i] = to_float(cp[n]);
                }
            }
            if (ok) ok = mbar_wait(bar(B_ACC_FULL + buf), (it >> 1) & 1);
            if (epilogue_any(!ok)) { ok = false; break; }
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + buf * kTok;
            const int chunks = (tile.rows + kChunk - 1) / kChunk;

            // one token's row out of `sums` (four staged values of this lane): bias, activation, gate, residual, store
            auto finish = [&](int m, float4 sums) {
                const int64_t row = tile.row0 + m;
                float h[4] = {sums.x, sums.y, sums.z, sums.w}, v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] += i < cols ? bias[i] : up_bias[i - 2];
                if (a.gated) {
                    float g[2] = {h[0], h[1]};
                    activate_all(g, a.act);
                    v[0] = g[0] * h[2]; v[1] = g[1] * h[3]; v[2] = v[3] = 0.f;
                } else {
                    activate_all(h, a.act);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = h[i];
                }
                const int n = n0 + col0;
                if (a.vec) {
                    if (n >= a.N) return;  // N is a multiple of cols
                    if (a.out_f32) {
                        float* o = static_cast<float*>(a.out) + row * a.out_stride + n;
                        const float* r = static_cast<const float*>(a.residual) + row * a.res_stride + n;
                        if (a.gated) {
                            float2 q = a.residual ? *reinterpret_cast<const float2*>(r) : make_float2(0.f, 0.f);
                            *reinterpret_cast<float2*>(o) = make_float2(v[0] + q.x, v[1] + q.y);
                        } else {
                            float4 q = a.residual ? *reinterpret_cast<const float4*>(r) : make_float4(0.f, 0.f, 0.f, 0.f);
                            *reinterpret_cast<float4*>(o) = make_float4(v[0] + q.x, v[1] + q.y, v[2] + q.z, v[3] + q.w);
                        }
                        return;
                    }
                    T* o = static_cast<T*>(a.out) + row * a.out_stride + n;
                    const T* r = static_cast<const T*>(a.residual) + row * a.res_stride + n;
                    if (a.gated) {
                        if (a.residual) {
                            const float2 q = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(r));
                            v[0] += q.x; v[1] += q.y;
                        }
                        *reinterpret_cast<uint32_t*>(o) = pack2<BF16>(v[0], v[1]);
                    } else {
                        if (a.residual) {
                            const uint2 u = *reinterpret_cast<const uint2*>(r);
                            const float2 q = unpack2<BF16>(u.x), p = unpack2<BF16>(u.y);
                            v[0] += q.x; v[1] += q.y; v[2] += p.x; v[3] += p.y;
                        }
                        *reinterpret_cast<uint2*>(o) = make_uint2(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]));
                    }
                    return;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = n + 32 * i;
                    if (i >= cols || c >= a.N) continue;
                    if (a.out_f32) {
                        const float q = a.residual ? static_cast<const float*>(a.residual)[row * a.res_stride + c] : 0.f;
                        static_cast<float*>(a.out)[row * a.out_stride + c] = v[i] + q;
                    } else {
                        const float q = a.residual ? to_float(static_cast<const T*>(a.residual)[row * a.res_stride + c]) : 0.f;
                        static_cast<T*>(a.out)[row * a.out_stride + c] = from_float<T>(v[i] + q);
                    }
                }
            };
            // a token's staged sums for this lane, from the row at `addr` (of any block): its columns; with a gate those of the
            // gate, then those of the up projection
            auto staged = [&](uint32_t addr, auto peer) {
                constexpr bool P = decltype(peer)::value;
                float q[4];
                if (!a.vec) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) ld_shared<1, P>(q + i, addr + 4u * (uint32_t)(lane + 32 * i));
                } else if (a.gated) {
                    ld_shared<2, P>(q, addr + 8u * (uint32_t)lane);
                    ld_shared<2, P>(q + 2, addr + 256u + 8u * (uint32_t)lane);
                } else {
                    ld_shared<4, P>(q, addr + 16u * (uint32_t)lane);
                }
                return make_float4(q[0], q[1], q[2], q[3]);
            };

            for (int c = 0; c < chunks; ++c, ++chunk) {
                float v[kChunk];
                tmem_ld16(acc + c * kChunk, v);
                if (c == chunks - 1) {  // the accumulator goes back: the next-but-one tile may overwrite it
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(B_ACC_EMPTY + buf));
                }
                const int b = chunk & 1, left = tile.rows - c * kChunk;
                float* stage = staging + b * (kStaging / 4);
                if (split == 1) {
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) stage[i * kFeat + warp * 32 + lane] = v[i];
                    epilogue_sync();  // one barrier a chunk: a buffer is written again two chunks on, after the next chunk's barrier
#pragma unroll
                    for (int i = 0; i < kChunk / 4; ++i) {
                        const int m = warp + 4 * i;
                        if (m < left) finish(c * kChunk + m, staged(smem_u32(stage + m * kFeat), std::false_type{}));
                    }
                } else {
                    ok = ok && mbar_wait_cluster(bar(B_PART_EMPTY + b), ((chunk >> 1) & 1) ^ 1);
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < kChunk; ++i)
                        if (i < left) stage[i * kFeat + warp * 32 + lane] = v[i];
                    __syncwarp();
                    if (lane < split) mbar_arrive_cluster(peer_addr(bar(B_PART_FULL + b), lane));
                    ok = mbar_wait_cluster(bar(B_PART_FULL + b), (chunk >> 1) & 1);
                    if (!ok) break;
                    for (int m = rank * 4 + warp; m < min(left, kChunk); m += 4 * split) {
                        const uint32_t row = smem_u32(stage + m * kFeat);
                        float4 sums = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int p = 0; p < split; ++p) {
                            const float4 q = staged(peer_addr(row, p), std::true_type{});
                            sums.x += q.x; sums.y += q.y; sums.z += q.z; sums.w += q.w;
                        }
                        finish(c * kChunk + m, sums);
                    }
                    __syncwarp();
                    if (lane < split) mbar_arrive_cluster(peer_addr(bar(B_PART_EMPTY + b), lane));
                }
            }
        }
        timed_out = !ok;
    }
    if (timed_out && a.status && lane == 0) atomicOr(a.status, SFB_STATUS_WAIT_TIMEOUT);
    // ---- teardown: every warp arrives here; with a cluster no block leaves while another may still read its sums
    tc_fence_before();
    __syncthreads();
    if (split > 1) cluster_sync();
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * kTok);
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

template <int kTok, int kStages, bool BF16>
int launch_tiles(const CUtensorMap* maps, const TileArgs& a, int64_t units, int sms, cudaStream_t stream) {
    auto kernel = linear_tcgen05_kernel<kTok, kStages, BF16>;
    const int rc = allow_shared_memory_once(reinterpret_cast<const void*>(kernel), smem_bytes(kTok, kStages, kMaxGroups));
    if (rc != SFB_OK) return rc;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)a.split; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(units, sms / a.split) * a.split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)smem_bytes(kTok, kStages, a.groups);
    cfg.stream = stream;
    cfg.attrs = &attr; cfg.numAttrs = a.split > 1 ? 1 : 0;
    SFB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], a));
    return SFB_OK;
}

}  // namespace

LinearPlan plan_linear(int64_t rows, int64_t K, int64_t N, int64_t groups, bool grouped, bool gated, int sms) {
    LinearPlan p{};
    // Token width: the rows of a group, twice the mean where only the mean is known, in the next power of two
    const int64_t want = grouped ? 2 * ceil_div(rows, groups) : rows;
    p.tokens = want <= 32 ? 32 : want <= 64 ? 64 : want <= 128 ? 128 : 256;
    p.feat_tiles = ceil_div(N, (int64_t)(gated ? kFeat / 2 : kFeat));
    const int64_t token_tiles = grouped ? std::max(std::min(groups, rows), ceil_div(rows, (int64_t)p.tokens)) : ceil_div(rows, (int64_t)p.tokens);
    const int64_t tiles = token_tiles * p.feat_tiles, n_k = ceil_div(K, (int64_t)kStepK);
    // Split of K: rounds of tiles x (K steps + what a tile costs besides them, in steps)
    p.split = 1;
    int64_t best = -1;
    for (int s = 1; s <= kMaxSplit && s <= n_k; ++s) {
        const int64_t cost = ceil_div(tiles, (int64_t)std::max(1, sms / s)) * (ceil_div(n_k, (int64_t)s) + (s > 1 ? 8 : 4));
        if (best < 0 || cost < best) { best = cost; p.split = s; }
    }
    return p;
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
    const LinearPlan plan = plan_linear(in.rows, in.K, in.N, in.groups, in.offsets != nullptr, in.up != nullptr, sms);
    const int64_t token_tiles = ceil_div(in.rows, (int64_t)plan.tokens) + (in.offsets ? std::min(in.groups, in.rows) : 0);
    if (token_tiles * plan.feat_tiles > 0x7fffffffLL) return SFB_ERR_UNSUPPORTED;

    TileArgs a{};
    a.bias = in.bias; a.up_bias = in.up_bias; a.residual = in.residual; a.out = in.out;
    a.offsets = in.offsets; a.row_index = in.row_index; a.status = in.status;
    a.out_stride = in.out_stride; a.res_stride = in.res_stride; a.bias_stride = in.bias_stride; a.up_bias_stride = in.up_bias_stride;
    a.rows = (int)in.rows; a.x_rows = (int)in.x_rows; a.N = (int)in.N; a.n_k = (int)ceil_div(in.K, (int64_t)kStepK); a.groups = (int)in.groups;
    a.feat_tiles = (int)plan.feat_tiles; a.split = plan.split; a.act = in.act;
    a.gated = in.up != nullptr; a.nk = nk; a.out_f32 = in.out_dtype == SFB_F32;
    a.block = 8;
    // one box where the rows fit one (in eights), boxes of 32 else: the last one of a group brings in at most 31 rows too many
    a.box_rows = !in.offsets && in.rows <= 32 ? (int)(ceil_div(in.rows, (int64_t)8) * 8) : 32;
    // rows of out and residual in pieces of `cols` values where all of them start on one
    const int cols = a.gated ? 2 : 4, piece = cols * (a.out_f32 ? 4 : 2);
    auto pieces = [&](const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % piece == 0 && stride % cols == 0; };
    a.vec = in.N % cols == 0 && pieces(in.out, in.out_stride) && (!in.residual || pieces(in.residual, in.res_stride));

    CUtensorMap maps[3];
    auto weight = [&](CUtensorMap* m, const void* base, const int64_t* stride) {
        const int64_t row = outer > 1 ? stride[ri] : ceil_div(inner, (int64_t)8) * 8, group = in.groups > 1 ? stride[0] : 8;
        return encode(m, base, 3, inner, outer, in.groups, row, group, 64);
    };
    const int64_t x_row = in.x_rows > 1 ? in.x_stride : ceil_div(in.K, (int64_t)8) * 8;
    if (!encode(&maps[0], in.x, 2, in.K, in.x_rows, 1, x_row, 0, in.row_index ? 1 : a.box_rows) || !weight(&maps[1], in.w, in.w_stride)) return SFB_ERR_UNSUPPORTED;
    if (in.up) { if (!weight(&maps[2], in.up, in.up_stride)) return SFB_ERR_UNSUPPORTED; }
    else maps[2] = maps[1];

    const int64_t units = token_tiles * plan.feat_tiles;
    const bool bf16 = in.dtype == SFB_BF16;
    auto go = [&](auto tok, auto stages) {
        constexpr int kTok = decltype(tok)::value, kStages = decltype(stages)::value;
        return bf16 ? launch_tiles<kTok, kStages, true>(maps, a, units, sms, stream) : launch_tiles<kTok, kStages, false>(maps, a, units, sms, stream);
    };
    using std::integral_constant;
    // about 190 KB of operands in flight whatever the width
    switch (plan.tokens) {
        case 32: return go(integral_constant<int, 32>{}, integral_constant<int, 9>{});
        case 64: return go(integral_constant<int, 64>{}, integral_constant<int, 8>{});
        case 128: return go(integral_constant<int, 128>{}, integral_constant<int, 6>{});
        default: return go(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    }
}

}  // namespace sfb
