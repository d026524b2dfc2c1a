// Expert routing: every token's top_k experts, their softmax weights, and the assignments sorted by expert.
//
// A logit of -inf or NaN never chooses its expert.  The chosen experts of a token are the first top_k in the order
// (larger logit, lower index); their weights are exp(l - max) over the sum of the chosen ones (renormalize) or of all
// experts.  The sort is stable (expert, then token): row of (t, e) = offsets[e] + number of tokens before t that chose e.
//
// One warp selects for one token: a lane holds consecutive logits as keys whose unsigned order is the float order, sorted;
// top_k rounds of a warp-wide maximum over the lanes' first keys take the winners.  16-bit logits carry their index in the
// key's lower half (complemented: the lower index wins), so a round is one reduction; fp32 needs a second for the index.
// A token chooses an expert at most once, so what a block of 128 tokens chose is one 128-bit mask per expert: a token's rank
// is a population count of the mask below it, whatever order the bits were set in - the result does not depend on the order
// of the atomics.
// With at most 128 tokens one launch does everything; with more, a second launch adds up the blocks' counts and places the
// rows (from 256 blocks up, where every block adding all counts would be quadratic, a scan comes in between).
// Bound: launch latency for few tokens.  Many take two dependent launches, of 16384 tokens of 128 experts 11.4 and 7.7 us (of 256 15.3
// and 9.7; each by itself, caches cold), where the bytes would take 1: a block per 128 tokens fills 128 of 148 SMs once, and the second
// launch reads the choices back and adds every block's counts.  The selection's instructions, about 200 a token and warp, are 3 to 4 us of it.

#include <algorithm>
#include <type_traits>

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

// A lane's PER consecutive logits with their rounds of selection.
template <typename T, int PER>
struct Lane {
    static constexpr bool kPacked = sizeof(T) == 2;  // key << 16 | ~index; a 16-bit float's key has 16 bits
    uint32_t key[PER];
    int index[kPacked ? 1 : PER];

    __device__ __forceinline__ void load(const T* l, int lane, int experts, bool vector) {
        T v[PER];
        if (vector && (lane + 1) * PER <= experts) {
            using Vec = std::conditional_t<sizeof(T) * PER == 4, uint32_t, std::conditional_t<sizeof(T) * PER == 8, uint2, uint4>>;
            constexpr int kVecs = sizeof(T) * PER <= 16 ? 1 : (int)(sizeof(T) * PER / 16);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) reinterpret_cast<Vec*>(v)[i] = reinterpret_cast<const Vec*>(l + lane * PER)[i];
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = lane * PER + i < experts ? l[lane * PER + i] : from_float<T>(-INFINITY);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane * PER + i;
            if constexpr (kPacked) {
                key[i] = half_key(*reinterpret_cast<const uint16_t*>(&v[i]), e);
            } else {
                key[i] = order_key(to_float(v[i]));
                index[i] = e;
            }
        }
    }
    // The ordered bits of a 16-bit float, -0 as +0, over the complement of the index; 0 for -inf and NaNs.
    static __device__ __forceinline__ uint32_t half_key(uint32_t b, int e) {
        constexpr uint32_t kInf = std::is_same_v<T, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
        if (b == 0x8000u) b = 0u;
        const uint32_t k = b & 0x8000u ? 0xffffu & ~b : b | 0x8000u;
        return (b & 0x7fffu) > kInf || b == (0x8000u | kInf) ? 0u : k << 16 | (0xffffu - (uint32_t)e);
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

    // rows that start on a lane's piece are read piece by piece
    constexpr uint32_t kPiece = sizeof(T) * PER < 16 ? sizeof(T) * PER : 16;
    const bool vector = reinterpret_cast<uintptr_t>(a.logits) % kPiece == 0 && a.logits_stride * sizeof(T) % kPiece == 0;
    // N tokens at a time: their rounds run beside one another
    auto select = [&](int t, auto count) {
        constexpr int N = decltype(count)::value;
        Lane<T, PER> l[N];
        float top_value[N], sum[N];
        int my_id[N];
        uint32_t my_key[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = min(t + i * kWarps, n_tokens - 1);  // (past the end: the last token again, not written)
            l[i].load(static_cast<const T*>(a.logits) + (t0 + u) * a.logits_stride, lane, a.experts, vector);
            l[i].sort();
            my_id[i] = -1;
            my_key[i] = 0;
            sum[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, l[i].key[0]);
            top_value[i] = Lane<T, PER>::value(top);
            if (!a.renormalize && top) {
#pragma unroll
                for (int k = 0; k < PER; ++k)
                    if (l[i].key[k]) sum[i] += exp_below(Lane<T, PER>::value(l[i].key[k]), top_value[i]);
                sum[i] = warp_sum(sum[i]);
            }
        }
#pragma unroll 1
        for (int j = 0; j < a.top_k; ++j) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                int e;
                const uint32_t m = l[i].take(e);
                if (lane == j) { my_id[i] = e; my_key[i] = m; }
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = t + i * kWarps;
            if (!my_key[i]) my_id[i] = -1;
            const float w = my_id[i] >= 0 ? exp_below(Lane<T, PER>::value(my_key[i]), top_value[i]) : 0.f;
            if (a.renormalize) sum[i] = warp_sum(w);
            if (lane < a.top_k && u < n_tokens) {
                const int64_t o = (t0 + u) * a.top_k + lane;
                a.ids[o] = my_id[i];
                a.weights[o] = my_id[i] >= 0 ? w / sum[i] : 0.f;
                ids[u * a.top_k + lane] = (int16_t)my_id[i];
                if (my_id[i] >= 0) atomicOr(&mask[my_id[i]][u >> 5], 1u << (u & 31));
            }
        }
    };
    if (PER > 8 || n_tokens <= kWarps)
        for (int t = warp; t < n_tokens; t += kWarps) select(t, std::integral_constant<int, 1>{});
    else
        for (int t = warp; t < n_tokens; t += 2 * kWarps) select(t, std::integral_constant<int, PER <= 8 ? 2 : 1>{});
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
    // this block's assignments on their way while the counts are added
    constexpr int kEach = kRouteTokens * kMaxTopK / kRouteThreads;
    int mine[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = threadIdx.x + j * kRouteThreads;
        mine[j] = i < n_tokens * a.top_k ? a.ids[t0 * a.top_k + i] : -1;
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
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = threadIdx.x + j * kRouteThreads;
        if (i >= n_tokens * a.top_k) break;
        const int t = i / a.top_k;
        ids[i] = (int16_t)mine[j];
        if (mine[j] >= 0) atomicOr(&mask[mine[j]][t >> 5], 1u << (t & 31));
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
    // launched in the plain way: blocks that start while the selecting ones run crowd onto the SMs those leave free (22 us
    // against 14 for 16384 tokens of 128 experts)
    route_place_kernel<<<blocks, kRouteThreads, 0, stream>>>(a, scanned);
    SFB_CUDA_CHECK(cudaGetLastError());
    return SFB_OK;
}

}  // namespace sfb
