// Dense and grouped matrix products with an epilogue, expert routing and combining: launch arguments and what the
// kernels share.
#pragma once

#include <utility>

#include "sfb_common.cuh"

namespace sfb {

// out[r, n] = act(sum_k x[i, k] w[e, k, n] + bias[e, n]) * (sum_k x[i, k] up[e, k, n] + up_bias[e, n]) + residual[r, n]
// for the rows r of group e, offsets[e] <= r < offsets[e + 1], with i = row_index[r] (or r).  Every part but the first
// product may be missing; without offsets all rows are group 0.
struct LinearArgs {
    const void *x, *w, *up, *bias, *up_bias, *residual;
    void* out;
    const int32_t* offsets;    // [groups + 1] or nullptr
    const int32_t* row_index;  // [rows] or nullptr
    int64_t x_stride, out_stride, res_stride;  // elements between rows
    int64_t w_stride[3], up_stride[3];         // group, k, n
    int64_t bias_stride, up_bias_stride;       // group
    int64_t rows, x_rows, K, N, groups;
    int layout, dtype, out_dtype, act;
    int* status;
    void* workspace;  // rows * ceil(K / 8) * 16 bytes, or nullptr: room for the rows of x in the order of out
    int64_t workspace_bytes;
};
int launch_linear_generic(const LinearArgs& a, cudaStream_t stream);
// Returns SFB_ERR_UNSUPPORTED (leaving the error text alone) for types and alignments outside what TMA and the tensor cores
// take; the caller then runs the generic kernel.
int launch_linear_tcgen05(const LinearArgs& a, cudaStream_t stream);
struct LinearPlan {
    int tokens;          // rows of out in a tile, at most
    int pair;            // 1: a cluster of two thread blocks on each tile (256 features)
    int split;           // thread blocks that share a tile's K steps
    int order;           // 1: rows of x are put in the order of out first
    int blocks_an_sm;    // 1 or 2 resident thread blocks
    int64_t feat_tiles;  // tiles across the columns of out
};
LinearPlan plan_linear(int64_t rows, int64_t K, int64_t N, int64_t groups, bool grouped, bool gated, bool indexed, bool ordered, int sms);
constexpr int kOrderedRows = 16;  // mean rows of a group from which a call with a row index asks for that workspace

constexpr int kMaxGroups = 1024;  // groups (experts) of one call
constexpr int kMaxTopK = 32;

struct RouteArgs {
    const void* logits;
    int64_t logits_stride;
    int32_t* ids;          // [T, k]
    float* weights;        // [T, k]
    int32_t* offsets;      // [E + 1]
    int32_t* token_rows;   // [T k]
    int32_t* positions;    // [T, k]
    int32_t* counts;       // [blocks, E] scratch
    int64_t tokens;
    int experts, top_k, renormalize, dtype;
};
constexpr int kRouteTokens = 128;  // tokens of one thread block
int launch_moe_route(const RouteArgs& a, cudaStream_t stream);

struct CombineArgs {
    const void *y, *residual;
    const int32_t* positions;
    const float* weights;
    void* out;
    int64_t y_stride, res_stride, out_stride, pos_stride, weight_stride;
    int64_t tokens, y_rows, hidden;
    int top_k, dtype;
    int* status;
};
int launch_moe_combine(const CombineArgs& a, cudaStream_t stream);

#ifdef __CUDACC__
// These kernels follow one another (router, product, product, sum), so each is launched before the one before it has ended
// (programmatic dependent launch): its blocks start where that one's have left, set themselves up and wait here.  Every thread
// that reads or writes global memory passes wait_for_previous first (but for the product behind order_rows_kernel, which has
// waited for it); let_next_start comes when a block holds all that it will
// ask the SM for, so a waiting successor cannot keep anything from it.  A kernel that does not take part ends before its
// successor starts.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), unsigned grid, unsigned block, int smem, unsigned cluster, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster; attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(block); cfg.dynamicSmemBytes = (size_t)smem; cfg.stream = stream;
    cfg.attrs = attrs; cfg.numAttrs = cluster > 1 ? 2 : 1;
    SFB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...));
    return SFB_OK;
}

// After a wait that ran out: copies may still be on their way into this block's shared memory, so the thread stays a while (20 ms,
// thousands of times what a copy takes) before the block may end.
__device__ __forceinline__ void settle() {
    uint64_t begun, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(begun));
    do {
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    } while (now - begun < 20000000);
}

// Group offsets come from the device and are not trusted: each is clamped to [0, rows], and one below an offset before it
// counts as that one.  Groups then never overlap or leave the rows, whatever the array holds.
__device__ __forceinline__ int group_offset(int raw, int before, int rows) { return max(before, min(raw, rows)); }

// 1 / (1 + 2^t) from t - 8.  The sum is formed 2^8 smaller than it is: its reciprocal then stays a normal number until t = 134, and
// h / (1 + 2^t), h itself some ten to ninety, until it is none itself (unscaled it became zero from t = 126 on).
__device__ __forceinline__ float logistic_exp2(float t_minus_8) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t_minus_8));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 0x1p-8f));
    return r * 0x1p-8f;
}
constexpr double kLog2E = 1.4426950408889634, kTanhGelu = 1.5957691216057308 * kLog2E;  // log2 e, 2 sqrt(2 / pi) log2 e

// The activations in fp32.  silu and the tanh form of gelu as h * logistic(.), the erf form as h/2 * erfc(-h / sqrt 2):
// none of them subtracts nearly equal numbers for large negative h.  (The erf form on the tensor cores: linear_tcgen05.cu.)
template <int ACT>
__device__ __forceinline__ float activate(float h) {
    if constexpr (ACT == SFB_ACT_SILU) return h * logistic_exp2(fmaf(h, (float)-kLog2E, -8.f));
    if constexpr (ACT == SFB_ACT_GELU) return 0.5f * h * erfcf(-0.70710678118654752f * h);
    if constexpr (ACT == SFB_ACT_GELU_TANH) return h * logistic_exp2(fmaf(h, fmaf(h * h, (float)(-kTanhGelu * 0.044715), (float)-kTanhGelu), -8.f));
    if constexpr (ACT == SFB_ACT_RELU) return h < 0.f ? 0.f : h;
    return h;
}
__device__ __forceinline__ float activate(float h, int act) {
    switch (act) {
        case SFB_ACT_SILU: return activate<SFB_ACT_SILU>(h);
        case SFB_ACT_GELU: return activate<SFB_ACT_GELU>(h);
        case SFB_ACT_GELU_TANH: return activate<SFB_ACT_GELU_TANH>(h);
        case SFB_ACT_RELU: return activate<SFB_ACT_RELU>(h);
        default: return h;
    }
}
#endif

}  // namespace sfb
