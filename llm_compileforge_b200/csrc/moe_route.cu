// Expert routing: every token's top_k experts, their softmax weights, and the assignments sorted by expert.
//
// A logit of -inf or NaN never chooses its expert.  The chosen experts of a token are the first top_k in the order
// (larger logit, lower index); their weights are exp(l - max) over the sum of the chosen ones (renormalize) or of all
// experts.  The sort is stable (expert, then token): row of (t, e) = offsets[e] + number of tokens before t that chose e.
//
// One warp selects for one token: a lane holds every 32nd logit as a key whose unsigned order is the float order, and
// top_k rounds of a warp-wide maximum take the winners.  A token chooses an expert at most once, so what a block of 128
// tokens chose is one 128-bit mask per expert: a token's rank is a population count of the mask below it, whatever order
// the bits were set in - the result does not depend on the order of the atomics.
// With at most 128 tokens one launch does everything; with more, the blocks' counts go through a scan over the blocks
// and a second launch places the rows.  Bound: launch latency for few tokens, the selection rounds for many.

#include <algorithm>

#include "linear.cuh"

namespace sfb {
namespace {

constexpr int kRouteThreads = 512, kWarps = kRouteThreads / 32, kWords = kRouteTokens / 32;

__device__ __forceinline__ uint32_t order_key(float v) {  // 0: not a candidate
    if (!(v > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 and +0 tie
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ float exp_below(float v, float top) { return top == INFINITY ? (v == INFINITY ? 1.f : 0.f) : expf(v - top); }

// Exclusive sum over s[0 .. n), n <= 2 * kRouteThreads, in place; s[n] receives the total.
__device__ void block_exclusive_sum(int* s, int n) {
    __shared__ int warp_total[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int a = 2 * tid < n ? s[2 * tid] : 0, b = 2 * tid + 1 < n ? s[2 * tid + 1] : 0;
    int sum = a + b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    if (lane == 31) warp_total[warp] = sum;
    __syncthreads();
    int before = sum - a - b;
    for (int w = 0; w < warp; ++w) before += warp_total[w];
    if (2 * tid < n) s[2 * tid] = before;
    if (2 * tid + 1 < n) s[2 * tid + 1] = before + a;
    if (2 * tid == n - 1) s[n] = before + a;
    if (2 * tid + 1 == n - 1) s[n] = before + a + b;
    __syncthreads();
}

__device__ __forceinline__ int mask_count(const uint32_t* m) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < kWords; ++w) c += __popc(m[w]);
    return c;
}

// Writes the rows of this block's assignments; start[e] is the row of the block's first token of expert e, total the
// number of assignments in all.
__device__ void place_rows(const RouteArgs& a, const uint32_t (*mask)[kWords], const int* start, const int16_t* ids, int64_t t0, int n_tokens,
                           int total) {
    for (int i = threadIdx.x; i < n_tokens * a.top_k; i += kRouteThreads) {
        const int e = ids[i], t = i / a.top_k;
        int row = -1;
        if (e >= 0) {
            row = start[e] + __popc(mask[e][t >> 5] & ((1u << (t & 31)) - 1u));
            for (int w = 0; w < (t >> 5); ++w) row += __popc(mask[e][w]);
            a.token_rows[row] = (int32_t)(t0 + t);
        }
        a.positions[t0 * a.top_k + i] = row;
    }
    const int64_t all = a.tokens * a.top_k;
    for (int64_t r = total + (int64_t)blockIdx.x * kRouteThreads + threadIdx.x; r < all; r += (int64_t)gridDim.x * kRouteThreads) a.token_rows[r] = -1;
}

template <typename T, int PER>
__global__ void __launch_bounds__(kRouteThreads) route_select_kernel(const RouteArgs a) {
    __shared__ uint32_t mask[32 * PER][kWords];
    __shared__ int16_t ids[kRouteTokens * kMaxTopK];
    __shared__ int start[32 * PER + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t0 = (int64_t)blockIdx.x * kRouteTokens;
    const int n_tokens = (int)min((int64_t)kRouteTokens, a.tokens - t0);
    for (int i = threadIdx.x; i < 32 * PER * kWords; i += kRouteThreads) (&mask[0][0])[i] = 0u;
    __syncthreads();

    for (int t = warp; t < n_tokens; t += kWarps) {
        const T* l = static_cast<const T*>(a.logits) + (t0 + t) * a.logits_stride;
        uint32_t key[PER], best = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = lane + 32 * i < a.experts ? order_key(to_float(l[lane + 32 * i])) : 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) best = max(best, key[i]);
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        const float top_value = key_value(top);
        float sum = 0.f;
        if (!a.renormalize && top) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (key[i]) sum += exp_below(key_value(key[i]), top_value);
            sum = warp_sum(sum);
        }
        int my_id = -1;
        float my_weight = 0.f;
        for (int j = 0; j < a.top_k; ++j) {
            best = 0;
            int at = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (key[i] > best) { best = key[i]; at = i; }  // ascending i: the lowest index of equal keys
            const uint32_t m = __reduce_max_sync(0xffffffffu, best);
            if (!m) break;
            const int e = (int)__reduce_min_sync(0xffffffffu, best == m ? (unsigned)(lane + 32 * at) : 0xffffffffu);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane + 32 * i == e) key[i] = 0u;
            if (lane == j) { my_id = e; my_weight = exp_below(key_value(m), top_value); }
        }
        if (a.renormalize) sum = warp_sum(my_weight);
        if (lane < a.top_k) {
            const int64_t o = (t0 + t) * a.top_k + lane;
            a.ids[o] = my_id;
            a.weights[o] = my_id >= 0 ? my_weight / sum : 0.f;
            ids[t * a.top_k + lane] = (int16_t)my_id;
            if (my_id >= 0) atomicOr(&mask[my_id][t >> 5], 1u << (t & 31));
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) {
        const int c = mask_count(mask[e]);
        start[e] = c;
        if (gridDim.x > 1) a.counts[(int64_t)blockIdx.x * a.experts + e] = c;
    }
    if (gridDim.x > 1) return;
    __syncthreads();
    block_exclusive_sum(start, a.experts);
    for (int e = threadIdx.x; e <= a.experts; e += kRouteThreads) a.offsets[e] = start[e];
    place_rows(a, mask, start, ids, t0, n_tokens, start[a.experts]);
}

// counts [blocks, E] -> for every expert the sum over the blocks before; row `blocks` receives the totals.
// 32 experts per thread block, 32 threads down the blocks for each.
__global__ void __launch_bounds__(1024) route_scan_kernel(int32_t* counts, int blocks, int experts) {
    __shared__ int part[32][33];
    const int c = threadIdx.x & 31, p = threadIdx.x >> 5, e = blockIdx.x * 32 + c;
    const int each = (blocks + 31) / 32, b0 = min(blocks, p * each), b1 = min(blocks, b0 + each);
    int sum = 0;
    if (e < experts)
        for (int b = b0; b < b1; ++b) sum += counts[(int64_t)b * experts + e];
    part[p][c] = sum;
    __syncthreads();
    int before = 0;
    for (int q = 0; q < p; ++q) before += part[q][c];
    if (e >= experts) return;
    for (int b = b0; b < b1; ++b) {
        const int v = counts[(int64_t)b * experts + e];
        counts[(int64_t)b * experts + e] = before;
        before += v;
    }
    if (p == 31) counts[(int64_t)blocks * experts + e] = before;
}

__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs a) {
    __shared__ uint32_t mask[kMaxGroups][kWords];
    __shared__ int16_t ids[kRouteTokens * kMaxTopK];
    __shared__ int start[kMaxGroups + 1];
    const int64_t t0 = (int64_t)blockIdx.x * kRouteTokens;
    const int n_tokens = (int)min((int64_t)kRouteTokens, a.tokens - t0);
    for (int i = threadIdx.x; i < a.experts * kWords; i += kRouteThreads) (&mask[0][0])[i] = 0u;
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) start[e] = a.counts[(int64_t)gridDim.x * a.experts + e];
    __syncthreads();
    for (int i = threadIdx.x; i < n_tokens * a.top_k; i += kRouteThreads) {
        const int e = a.ids[t0 * a.top_k + i], t = i / a.top_k;
        ids[i] = (int16_t)e;
        if (e >= 0) atomicOr(&mask[e][t >> 5], 1u << (t & 31));
    }
    block_exclusive_sum(start, a.experts);
    const int total = start[a.experts];
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= a.experts; e += kRouteThreads) a.offsets[e] = start[e];
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) start[e] += a.counts[(int64_t)blockIdx.x * a.experts + e];
    __syncthreads();
    place_rows(a, mask, start, ids, t0, n_tokens, total);
}

template <typename T>
void launch_select(const RouteArgs& a, unsigned blocks, cudaStream_t stream) {
    if (a.experts <= 64) route_select_kernel<T, 2><<<blocks, kRouteThreads, 0, stream>>>(a);
    else if (a.experts <= 128) route_select_kernel<T, 4><<<blocks, kRouteThreads, 0, stream>>>(a);
    else if (a.experts <= 256) route_select_kernel<T, 8><<<blocks, kRouteThreads, 0, stream>>>(a);
    else route_select_kernel<T, 32><<<blocks, kRouteThreads, 0, stream>>>(a);
}

}  // namespace

int launch_moe_route(const RouteArgs& a, cudaStream_t stream) {
    const unsigned blocks = (unsigned)ceil_div(a.tokens, (int64_t)kRouteTokens);
    if (a.dtype == SFB_F32) launch_select<float>(a, blocks, stream);
    else if (a.dtype == SFB_BF16) launch_select<__nv_bfloat16>(a, blocks, stream);
    else launch_select<__half>(a, blocks, stream);
    SFB_CUDA_CHECK(cudaGetLastError());
    if (blocks == 1) return SFB_OK;
    route_scan_kernel<<<(unsigned)ceil_div((int64_t)a.experts, (int64_t)32), 1024, 0, stream>>>(a.counts, (int)blocks, a.experts);
    SFB_CUDA_CHECK(cudaGetLastError());
    route_place_kernel<<<blocks, kRouteThreads, 0, stream>>>(a);
    SFB_CUDA_CHECK(cudaGetLastError());
    return SFB_OK;
}

}  // namespace sfb
