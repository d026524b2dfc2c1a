// Every token's weighted sum of its experts' rows: out[t, :] = sum_j weights[t, j] y[positions[t, j], :] + residual[t, :].
//
// A position of -1 (an assignment that the router left empty) adds nothing, whatever its weight.  Sums in fp32 in the
// order of j, one rounding; no atomics, so the same inputs give the same bits.
// Bound by HBM: tokens * top_k rows of y in, a row of out (and of residual) per token.  Rows lie anywhere, so the bandwidth
// hangs on how many of them are in flight: one warp of a thread block issues bulk copies of whole row segments (up to 4 KB)
// into a ring of 18 slots in shared memory, lane j the j-th row of the token, and runs ahead of the warps that sum them by
// as many tokens as the ring holds.  (With 16-byte loads into registers instead, eight rows a lane, the compiler either
// serialised them or left too few warps an SM: 2.3 to 4.5 TB/s at 8192 tokens of 8 rows of 4096.)
// Rows that bulk copies cannot address (not on 16 bytes) go value by value through registers.

#include <algorithm>
#include <type_traits>

#include "linear.cuh"

namespace sfb {
namespace {

constexpr int kSlots = 18, kBatch = 16;  // rows in flight; rows issued together
constexpr int kSegmentBytes = 4096;      // of a row, at most: eight warps of 32 lanes of 16 bytes

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {  // two seconds at most
    uint64_t begun = 0;
    for (;;) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        uint64_t now;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (begun == 0) begun = now;
        if (now - begun > 2000000000) return false;
    }
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// Sixteen bytes of a row <-> fp32, by whole words: taken value by value out of a vector the compiler spends 100 instructions.
template <typename T>
__device__ __forceinline__ void add_scaled(float (&sum)[16 / sizeof(T)], float w, uint4 p) {
    const uint32_t u[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same_v<T, float>) {
            sum[i] = fmaf(w, __uint_as_float(u[i]), sum[i]);
        } else {
            float2 f;
            if constexpr (std::is_same_v<T, __nv_bfloat16>) f = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
            else f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            sum[2 * i] = fmaf(w, f.x, sum[2 * i]);
            sum[2 * i + 1] = fmaf(w, f.y, sum[2 * i + 1]);
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 rounded(const float (&sum)[16 / sizeof(T)]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same_v<T, float>) u[i] = __float_as_uint(sum[i]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(sum[2 * i + 1]), "f"(sum[2 * i]));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(sum[2 * i + 1]), "f"(sum[2 * i]));
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// One token's row numbers, lane j the j-th: -1 where there is none.
struct Rows {
    int row;
    float weight;
};
__device__ __forceinline__ Rows token_rows(const CombineArgs& a, int64_t t, int lane) {
    Rows r{-1, 0.f};
    if (lane < a.top_k) {
        r.row = a.positions[t * a.pos_stride + lane];
        r.weight = a.weights[t * a.weight_stride + lane];
    }
    return r;
}
__device__ __forceinline__ bool inside(const CombineArgs& a, int row) { return row >= 0 && row < (int)a.y_rows; }

// Warp 0 fetches, warps 1 .. blockDim / 32 - 1 sum; a block keeps its segment of the rows and walks the tokens.
template <typename T>
__global__ void __launch_bounds__(288) moe_combine_kernel(const CombineArgs a, int segment_bytes, unsigned segments) {
    constexpr int kVec = 16 / (int)sizeof(T);
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t bars[2 * kSlots];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, summing = (int)(blockDim.x >> 5) - 1;
    const uint32_t full = smem_u32(bars), empty = full + 8 * kSlots, ring0 = smem_u32(ring);
    if (threadIdx.x < kSlots) {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full + 8 * threadIdx.x));
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty + 8 * threadIdx.x), "r"(summing));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    let_next_start();
    wait_for_previous();
    __syncthreads();
    // this block's segment of the rows, its tokens and, one ahead, their rows
    const unsigned first = blockIdx.x / segments, s = blockIdx.x - first * segments, step = gridDim.x / segments, tokens = (unsigned)a.tokens;
    const int64_t at = (int64_t)s * segment_bytes;
    const uint32_t bytes = (uint32_t)min((int64_t)segment_bytes, a.hidden * (int64_t)sizeof(T) - at);
    const char* y = static_cast<const char*>(a.y) + at;
    const char* residual = a.residual ? static_cast<const char*>(a.residual) + at : nullptr;
    char* out = static_cast<char*>(a.out) + at;
    const int64_t y_bytes = a.y_stride * (int64_t)sizeof(T), res_bytes = a.res_stride * (int64_t)sizeof(T), out_bytes = a.out_stride * (int64_t)sizeof(T);
    Rows next = token_rows(a, first, lane);  // the grid has no more blocks than items
    uint32_t slot = 0, phase = 0;            // of the next row
    bool ok = true;
    auto skip = [&](uint32_t n) {  // n <= kSlots rows on
        slot += n;
        if (slot >= kSlots) { slot -= kSlots; phase ^= 1; }
    };
    for (unsigned token = first; token < tokens && ok; token += step) {
        const Rows rows = next;
        if (token + step < tokens) next = token_rows(a, token + step, lane);
        const uint32_t mask = __ballot_sync(0xffffffffu, inside(a, rows.row));
        if (warp == 0) {
            if (s == 0 && a.status && rows.row != -1 && !inside(a, rows.row)) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
            // A batch is no larger than the ring, and no lane begins the next one before every lane is through with this one: each
            // slot that a lane waits for has then been filled before, and the parity it asks for cannot be the one before last
            for (int j0 = 0; j0 < a.top_k; j0 += kBatch) {
                const uint32_t batch = mask >> j0 & ((1u << kBatch) - 1u);
                const int rank = __popc(batch & ((1u << (lane & (kBatch - 1))) - 1u));
                if ((lane & ~(kBatch - 1)) == j0 && (batch >> (lane - j0) & 1u)) {
                    const uint32_t mine = slot + rank < kSlots ? slot + rank : slot + rank - kSlots, p = slot + rank < kSlots ? phase : phase ^ 1;
                    ok = mbar_wait(empty + 8 * mine, p ^ 1);
                    if (ok) bulk_load(ring0 + mine * segment_bytes, y + rows.row * y_bytes, bytes, full + 8 * mine);
                }
                __syncwarp();
                skip(__popc(batch));
            }
            if (residual) {
                if (lane == 0 && (ok = ok && mbar_wait(empty + 8 * slot, phase ^ 1)))
                    bulk_load(ring0 + slot * segment_bytes, residual + token * res_bytes, bytes, full + 8 * slot);
                skip(1);
            }
            ok = __all_sync(0xffffffffu, ok);
            continue;
        }
        const uint32_t mine = ((warp - 1) * 32 + lane) * 16;  // (past the end of a short last segment: adds what the slot holds, stores nothing)
        float sum[kVec] = {};
        const int n = __popc(mask);
        auto row = [&](float w) {
            ok = ok && mbar_wait(full + 8 * slot, phase);
            add_scaled<T>(sum, w, *reinterpret_cast<const uint4*>(ring + slot * segment_bytes + mine));
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty + 8 * slot) : "memory");
            skip(1);
        };
        uint32_t left = mask;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            row(__shfl_sync(0xffffffffu, rows.weight, __ffs(left) - 1));
            left &= left - 1;
        }
        if (residual) row(1.f);
        ok = __all_sync(0xffffffffu, ok);
        if (ok && mine < bytes) *reinterpret_cast<uint4*>(out + token * out_bytes + mine) = rounded<T>(sum);
    }
    if (!ok) settle();
    if (!ok && a.status && lane == 0) atomicOr(a.status, SFB_STATUS_WAIT_TIMEOUT);
}

// A warp for 32 values of one token's row.
template <typename T>
__global__ void __launch_bounds__(256) moe_combine_values_kernel(const CombineArgs a, int segments) {
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), t = unit / segments, s = unit - t * segments, h = s * 32 + lane;
    if (t >= a.tokens) return;
    const Rows rows = token_rows(a, t, lane);
    if (s == 0 && a.status && rows.row != -1 && !inside(a, rows.row)) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
    float sum = 0.f;
    for (int j = 0; j < a.top_k; ++j) {
        const int row = __shfl_sync(0xffffffffu, rows.row, j);
        const float w = __shfl_sync(0xffffffffu, rows.weight, j);
        if (inside(a, row) && h < a.hidden) sum = fmaf(w, to_float(static_cast<const T*>(a.y)[row * a.y_stride + h]), sum);
    }
    if (h >= a.hidden) return;
    if (a.residual) sum += to_float(static_cast<const T*>(a.residual)[t * a.res_stride + h]);
    static_cast<T*>(a.out)[t * a.out_stride + h] = from_float<T>(sum);
}

template <typename T>
int launch(const CombineArgs& a, cudaStream_t stream) {
    constexpr int kVec = 16 / (int)sizeof(T);
    if (a.tokens > 0x7fffffffLL || a.y_rows > 0x7fffffffLL || a.hidden > (1LL << 30)) return fail(SFB_ERR_UNSUPPORTED, "moe_combine: too many rows or columns");
    auto even = [&](const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % kVec == 0; };
    if (!(a.hidden % kVec == 0 && even(a.y, a.y_stride) && even(a.out, a.out_stride) && (!a.residual || even(a.residual, a.res_stride)))) {
        const int64_t segments = ceil_div(a.hidden, (int64_t)32), blocks = ceil_div(a.tokens * segments, (int64_t)8);
        if (blocks > 0x7fffffffLL) return fail(SFB_ERR_UNSUPPORTED, "moe_combine: too many rows or columns");
        moe_combine_values_kernel<T><<<(unsigned)blocks, 256, 0, stream>>>(a, (int)segments);
        SFB_CUDA_CHECK(cudaGetLastError());
        return SFB_OK;
    }
    int dev = 0, sms = 0;
    SFB_CUDA_CHECK(cudaGetDevice(&dev));
    SFB_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const int rc = allow_shared_memory_once(reinterpret_cast<const void*>(moe_combine_kernel<T>), kSlots * kSegmentBytes);
    if (rc != SFB_OK) return rc;
    // segments of whole warps' pieces; short rows leave a block few warps and an SM many blocks
    const int64_t row_bytes = a.hidden * (int64_t)sizeof(T);
    const int segment = (int)std::min<int64_t>(kSegmentBytes, ceil_div(row_bytes, (int64_t)512) * 512);
    const int64_t segments = ceil_div(row_bytes, (int64_t)segment);
    const int threads = 32 * (1 + segment / 512), smem = kSlots * segment;
    const int64_t resident = (int64_t)sms * std::min(2048 / threads, 229376 / (smem + 2048));
    const int64_t blocks = segments * std::max<int64_t>(1, std::min(a.tokens, resident / segments));
    return launch_after(moe_combine_kernel<T>, (unsigned)blocks, (unsigned)threads, smem, 1, stream, a, segment, (unsigned)segments);
}

}  // namespace

int launch_moe_combine(const CombineArgs& a, cudaStream_t stream) {
    if (a.dtype == SFB_F32) return launch<float>(a, stream);
    if (a.dtype == SFB_BF16) return launch<__nv_bfloat16>(a, stream);
    return launch<__half>(a, stream);
}

}  // namespace sfb
