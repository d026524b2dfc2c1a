// Expert routing: every token's top_k experts, their softmax weights, and the assignments sorted by expert.
//
// A logit of -inf or NaN never chooses its expert.  The chosen experts of a token are the first top_k in the order
// (larger logit, lower index); their weights are exp(l - max) over the sum of the chosen ones (renormalize) or of all
// experts.  The sort is stable (expert, then token): row of (t, e) = offsets[e] + number of tokens before t that chose e.
//
// One warp selects for one token: a lane holds every 32nd logit as a key whose unsigned order is the float order, sorted;
// top_k rounds of a warp-wide maximum over the lanes' first keys take the winners.  16-bit logits carry their index in the
// key's lower half (complemented: the lower index wins), so a round is one reduction; fp32 needs a second for the index.
// A token chooses an expert at most once, so what a block of 128 tokens chose is one 128-bit mask per expert: a token's rank
// is a population count of the mask below it, whatever order the bits were set in - the result does not depend on the order
// of the atomics.
// With at most 128 tokens one launch does everything; with more, a second launch adds up the blocks' counts and places the
// rows (from 256 blocks up, where every block adding all counts would be quadratic, a scan comes in between).
// Bound: launch latency for few tokens, the selection rounds' instructions for many.

#include <algorithm>

#include "linear.cuh"

namespace sfb {
namespace {

constexpr int kRouteThreads = 1024, kWarps = kRouteThreads / 32, kWords = kRouteTokens / 32;
constexpr unsigned kSumBlocks = 256;  // up to here the placing blocks add the counts themselves

__device__ __forceinline__ uint32_t order_key(float v) {  // 0: not a candidate
    if (!(v > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 and +0 tie
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ float exp_below(float v, float top) { return top == INFINITY ? (v == INFINITY ? 1.f : 0.f) : expf(v - top); }

// Exclusive sum over s[0 .. n), n <= kRouteThreads, in place; s[n] receives the total.
__device__ void block_exclusive_sum(int* s, int n) {
    __shared__ int warp_total[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int own = tid < n ? s[tid] : 0;
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    if (lane == 31) warp_total[warp] = sum;
    __syncthreads();
    const int others = __reduce_add_sync(0xffffffffu, lane < warp ? warp_total[lane] : 0);
    if (tid < n) s[tid] = others + sum - own;
    if (tid == n - 1) s[n] = others + sum;
    __syncthreads();
}
static_assert(kMaxGroups <= kRouteThreads && kWarps <= 32, "one expert a thread");

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

// A lane's logits lane, lane + 32, ... with their rounds of selection.
template <typename T, int PER>
struct Lane {
    static constexpr bool kPacked = sizeof(T) == 2;  // key << 16 | ~index; a 16-bit float's key has 16 bits
    uint32_t key[PER];
    int index[kPacked ? 1 : PER];

    __device__ __forceinline__ void load(const T* l, int lane, int experts) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + 32 * i;
            const float v = e < experts ? to_float(l[e]) : -INFINITY;
            uint32_t k = order_key(v);
            if constexpr (kPacked) {
                if (k) k = pack(v, e);
            } else {
                index[i] = e;
            }
            key[i] = k;
        }
    }
    // The 16-bit key of a 16-bit float, never 0 for a candidate (only -inf and NaNs lie below the lowest)
    static __device__ __forceinline__ uint32_t pack(float v, int e) {
        const T t = from_float<T>(v + 0.f);
        uint32_t b = *reinterpret_cast<const uint16_t*>(&t);
        b = b & 0x8000u ? 0xffffu & ~b : b | 0x8000u;
        return b << 16 | (0xffffu - (uint32_t)e);
    }
    static __device__ __forceinline__ float value(uint32_t k) {
        if constexpr (kPacked) {
            const uint32_t b = k >> 16;
            const uint16_t h = (uint16_t)(b & 0x8000u ? b & 0x7fffu : ~b);
            return to_float(*reinterpret_cast<const T*>(&h));
        } else {
            return key_value(k);
        }
    }
    // Odd-even transposition with strict comparisons: equal keys keep their order, the lower index first
    __device__ __forceinline__ void sort() {
#pragma unroll
        for (int r = 0; r < PER; ++r)
#pragma unroll
            for (int i = r & 1; i + 1 < PER; i += 2) {
                if constexpr (kPacked) {
                    const uint32_t hi = max(key[i], key[i + 1]), lo = min(key[i], key[i + 1]);
                    key[i] = hi; key[i + 1] = lo;
                } else {
                    const bool swap = key[i] < key[i + 1];
                    const uint32_t k = key[i];
                    const int x = index[i];
                    key[i] = swap ? key[i + 1] : k; index[i] = swap ? index[i + 1] : x;
                    key[i + 1] = swap ? k : key[i + 1]; index[i + 1] = swap ? x : index[i + 1];
                }
            }
    }
    // The best key of the warp (0: none left) and its expert; it is taken out.
    __device__ __forceinline__ uint32_t take(int& expert) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, key[0]);
        bool won;
        if constexpr (kPacked) {
            expert = (int)(0xffffu - (m & 0xffffu));
            won = key[0] == m;
        } else {
            expert = (int)__reduce_min_sync(0xffffffffu, key[0] == m ? (unsigned)index[0] : 0xffffffffu);
            won = key[0] == m && index[0] == expert;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            key[i] = won ? (i + 1 < PER ? key[i + 1 < PER ? i + 1 : i] : 0u) : key[i];
            if constexpr (!kPacked)
                if (i + 1 < PER) index[i] = won ? index[i + 1 < PER ? i + 1 : i] : index[i];
        }
        return m;
    }
};

template <typename T, int PER>
__global__ void __launch_bounds__(kRouteThreads) route_select_kernel(const RouteArgs a) {
    __shared__ uint32_t mask[32 * PER][kWords];
    __shared__ int16_t ids[kRouteTokens * kMaxTopK];
    __shared__ int start[32 * PER + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t0 = (int64_t)blockIdx.x * kRouteTokens;
    const int n_tokens = (int)min((int64_t)kRouteTokens, a.tokens - t0);
    let_next_start();
    for (int i = threadIdx.x; i < 32 * PER * kWords; i += kRouteThreads) (&mask[0][0])[i] = 0u;
    wait_for_previous();
    __syncthreads();

    for (int t = warp; t < n_tokens; t += kWarps) {
        Lane<T, PER> l;
        l.load(static_cast<const T*>(a.logits) + (t0 + t) * a.logits_stride, lane, a.experts);
        l.sort();
        const uint32_t top = __reduce_max_sync(0xffffffffu, l.key[0]);
        const float top_value = Lane<T, PER>::value(top);
        float sum = 0.f;
        if (!a.renormalize && top) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (l.key[i]) sum += exp_below(Lane<T, PER>::value(l.key[i]), top_value);
            sum = warp_sum(sum);
        }
        int my_id = -1;
        uint32_t my_key = 0;
        for (int j = 0; j < a.top_k; ++j) {
            int e;
            const uint32_t m = l.take(e);
            if (!m) break;
            if (lane == j) { my_id = e; my_key = m; }
        }
        const float my_weight = my_id >= 0 ? exp_below(Lane<T, PER>::value(my_key), top_value) : 0.f;
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

// scanned: the counts have been through route_scan_kernel; else every block adds those it needs.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs a, bool scanned) {
    __shared__ uint32_t mask[kMaxGroups][kWords];
    __shared__ int16_t ids[kRouteTokens * kMaxTopK];
    __shared__ int start[kMaxGroups + 1], before[kMaxGroups];
    const int64_t t0 = (int64_t)blockIdx.x * kRouteTokens;
    const int n_tokens = (int)min((int64_t)kRouteTokens, a.tokens - t0), blocks = (int)gridDim.x;
    for (int i = threadIdx.x; i < a.experts * kWords; i += kRouteThreads) (&mask[0][0])[i] = 0u;
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) start[e] = before[e] = 0;
    let_next_start();
    __syncthreads();
    wait_for_previous();
    for (int i = threadIdx.x; i < n_tokens * a.top_k; i += kRouteThreads) {
        const int e = a.ids[t0 * a.top_k + i], t = i / a.top_k;
        ids[i] = (int16_t)e;
        if (e >= 0) atomicOr(&mask[e][t >> 5], 1u << (t & 31));
    }
    if (scanned) {
        for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) {
            start[e] = a.counts[(int64_t)blocks * a.experts + e];
            before[e] = a.counts[(int64_t)blockIdx.x * a.experts + e];
        }
    } else {
        // a thread adds every parts-th block's count of its expert
        const int parts = kRouteThreads / a.experts, part = threadIdx.x / a.experts, e = threadIdx.x - part * a.experts;
        if (part < parts) {
            int all = 0, below = 0;
#pragma unroll 8
            for (int b = part; b < blocks; b += parts) {
                const int c = a.counts[(int64_t)b * a.experts + e];
                all += c;
                below += b < (int)blockIdx.x ? c : 0;
            }
            atomicAdd(&start[e], all);
            atomicAdd(&before[e], below);
        }
    }
    __syncthreads();
    block_exclusive_sum(start, a.experts);
    const int total = start[a.experts];
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= a.experts; e += kRouteThreads) a.offsets[e] = start[e];
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) start[e] += before[e];
    __syncthreads();
    place_rows(a, mask, start, ids, t0, n_tokens, total);
}

template <typename T>
int launch_select(const RouteArgs& a, unsigned blocks, cudaStream_t stream) {
    auto go = [&](auto kernel) { return launch_after(kernel, blocks, kRouteThreads, 0, 1, stream, a); };
    if (a.experts <= 64) return go(route_select_kernel<T, 2>);
    if (a.experts <= 128) return go(route_select_kernel<T, 4>);
    if (a.experts <= 256) return go(route_select_kernel<T, 8>);
    return go(route_select_kernel<T, 32>);
}

}  // namespace

int launch_moe_route(const RouteArgs& a, cudaStream_t stream) {
    const unsigned blocks = (unsigned)ceil_div(a.tokens, (int64_t)kRouteTokens);
    const int rc = a.dtype == SFB_F32 ? launch_select<float>(a, blocks, stream)
                   : a.dtype == SFB_BF16 ? launch_select<__nv_bfloat16>(a, blocks, stream) : launch_select<__half>(a, blocks, stream);
    if (rc != SFB_OK || blocks == 1) return rc;
    const bool scanned = blocks > kSumBlocks;
    if (scanned) {
        route_scan_kernel<<<(unsigned)ceil_div((int64_t)a.experts, (int64_t)32), 1024, 0, stream>>>(a.counts, (int)blocks, a.experts);
        SFB_CUDA_CHECK(cudaGetLastError());
    }
    return launch_after(route_place_kernel, blocks, kRouteThreads, 0, 1, stream, a, scanned);
}

}  // namespace sfb
