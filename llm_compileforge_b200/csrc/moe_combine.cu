// Every token's weighted sum of its experts' rows: out[t, :] = sum_j weights[t, j] y[positions[t, j], :] + residual[t, :].
//
// A position of -1 (an assignment that the router left empty) adds nothing, whatever its weight.  Sums in fp32 in the
// order of j, one rounding; no atomics, so the same inputs give the same bits.  Bound by HBM: tokens * top_k rows of y
// in, a row of out (and of residual) per token; a thread owns one 16-byte piece of out and has up to eight rows' pieces
// in flight.

#include "linear.cuh"

namespace sfb {
namespace {

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Piece {
    T v[VEC];
};

template <typename T, int VEC>
__global__ void __launch_bounds__(256) moe_combine_kernel(const CombineArgs a) {
    __shared__ int64_t row[kMaxTopK];
    __shared__ float weight[kMaxTopK];
    const int64_t t = blockIdx.x;
    if (threadIdx.x < a.top_k) {
        int64_t p = a.positions[t * a.pos_stride + threadIdx.x];
        if (p < -1 || p >= a.y_rows) {
            if (a.status && blockIdx.y == 0) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
            p = -1;
        }
        row[threadIdx.x] = p < 0 ? -1 : p * a.y_stride;
        weight[threadIdx.x] = a.weights[t * a.weight_stride + threadIdx.x];
    }
    __syncthreads();
    const T* y = static_cast<const T*>(a.y);
    const int64_t h = ((int64_t)blockIdx.y * 256 + threadIdx.x) * VEC;
    if (h >= a.hidden) return;
    float sum[VEC] = {};
    constexpr int kAhead = 8;
    for (int j0 = 0; j0 < a.top_k; j0 += kAhead) {
        Piece<T, VEC> p[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (j0 + j < a.top_k && row[j0 + j] >= 0) p[j] = *reinterpret_cast<const Piece<T, VEC>*>(y + row[j0 + j] + h);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (j0 + j >= a.top_k || row[j0 + j] < 0) continue;
            const float w = weight[j0 + j];
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] = fmaf(w, to_float(p[j].v[i]), sum[i]);
        }
    }
    if (a.residual) {
        const Piece<T, VEC> r = *reinterpret_cast<const Piece<T, VEC>*>(static_cast<const T*>(a.residual) + t * a.res_stride + h);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] += to_float(r.v[i]);
    }
    Piece<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = from_float<T>(sum[i]);
    *reinterpret_cast<Piece<T, VEC>*>(static_cast<T*>(a.out) + t * a.out_stride + h) = o;
}

template <typename T>
int launch(const CombineArgs& a, cudaStream_t stream) {
    constexpr int kVec = 16 / (int)sizeof(T);
    auto even = [&](const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % kVec == 0; };
    // 16-byte pieces where every row allows them, single values otherwise
    const bool wide = a.hidden % kVec == 0 && even(a.y, a.y_stride) && even(a.out, a.out_stride) && (!a.residual || even(a.residual, a.res_stride));
    const int64_t per_block = 256 * (wide ? kVec : 1), parts = ceil_div(a.hidden, per_block);
    if (a.tokens > 0x7fffffffLL || parts > 65535) return fail(SFB_ERR_UNSUPPORTED, "moe_combine: too many tokens or columns");
    const dim3 grid((unsigned)a.tokens, (unsigned)parts);
    if (wide) moe_combine_kernel<T, kVec><<<grid, 256, 0, stream>>>(a);
    else moe_combine_kernel<T, 1><<<grid, 256, 0, stream>>>(a);
    SFB_CUDA_CHECK(cudaGetLastError());
    return SFB_OK;
}

}  // namespace

int launch_moe_combine(const CombineArgs& a, cudaStream_t stream) {
    if (a.dtype == SFB_F32) return launch<float>(a, stream);
    if (a.dtype == SFB_BF16) return launch<__nv_bfloat16>(a, stream);
    return launch<__half>(a, stream);
}

}  // namespace sfb
