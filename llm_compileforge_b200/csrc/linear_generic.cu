// Matrix product with bias, activation, gate and residual, dense or grouped by ragged row ranges: the form for every
// type, size and stride, on the CUDA cores.
//
// out[r, n] = act(sum_k x[i, k] W_e[k, n] + b_e[n]) * (sum_k x[i, k] V_e[k, n] + c_e[n]) + residual[r, n], i = row_index[r]
//
// A thread block owns a 64 x 64 tile of out and walks K in steps of 16 through shared memory; a thread holds 4 x 4
// accumulators (twice that with a gate) in fp32 and sums over k in ascending order.  Bound by the FMA pipes.  It is the
// only path of fp32 and of matrices whose rows TMA cannot address (base or row stride not a multiple of 16 bytes).

#include <algorithm>

#include "linear.cuh"

namespace sfb {
namespace {

constexpr int kTile = 64, kStep = 16, kLine = kTile + 4;

template <typename T, typename TO, bool GATED>
__global__ void __launch_bounds__(256) linear_generic_kernel(const LinearArgs a) {
    __shared__ float xs[kStep][kLine], ws[kStep][kLine], us[GATED ? kStep : 1][kLine];
    __shared__ int64_t x_off[kTile];
    __shared__ int tile_of[4];  // group, first row, end row
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;

    if (tid == 0) {  // row tile blockIdx.x -> its group: groups take ceil(rows / 64) tiles each, one after another
        int left = (int)blockIdx.x, e = 0, lo = 0, hi = (int)a.rows, flag = 0;
        bool found = !a.offsets && (int64_t)left * kTile < a.rows;
        if (a.offsets) {
            hi = group_offset(a.offsets[0], 0, (int)a.rows);
            flag = hi != a.offsets[0];
            for (; e < a.groups && !found; ++e) {
                lo = hi;
                hi = group_offset(a.offsets[e + 1], lo, (int)a.rows);
                flag |= hi != a.offsets[e + 1];
                const int tiles = (hi - lo + kTile - 1) / kTile;
                found = left < tiles;
                if (found) break;
                left -= tiles;
            }
            if (flag && a.status) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
        }
        tile_of[0] = found ? e : -1;
        tile_of[1] = lo + left * kTile;
        tile_of[2] = hi;
    }
    __syncthreads();
    const int e = tile_of[0], row0 = tile_of[1], row_end = tile_of[2];
    if (e < 0) return;
    const int64_t n0 = (int64_t)blockIdx.y * kTile;
    if (tid < kTile) {
        const int r = row0 + tid;
        int64_t i = r < row_end ? r : -1;
        if (i >= 0 && a.row_index) {
            i = a.row_index[r];
            if (i < 0 || i >= a.x_rows) {
                if (a.status && blockIdx.y == 0) atomicOr(a.status, SFB_STATUS_BAD_ROW_INDEX);
                i = 0;
            }
        }
        x_off[tid] = i < 0 ? -1 : i * a.x_stride;
    }
    __syncthreads();

    const T* x = static_cast<const T*>(a.x);
    const T* w = static_cast<const T*>(a.w) + e * a.w_stride[0];
    const T* up = GATED ? static_cast<const T*>(a.up) + e * a.up_stride[0] : nullptr;
    float acc[4][4] = {}, gate[GATED ? 4 : 1][4] = {};
    for (int64_t k0 = 0; k0 < a.K; k0 += kStep) {
#pragma unroll
        for (int j = 0; j < kTile * kStep / 256; ++j) {
            const int i = tid + j * 256;
            const int xk = i % kStep, xr = i / kStep;  // x: k runs fastest
            xs[xk][xr] = x_off[xr] >= 0 && k0 + xk < a.K ? to_float(x[x_off[xr] + k0 + xk]) : 0.f;
            // weights: whichever dimension is contiguous runs fastest
            const int wk = a.w_stride[2] == 1 ? i / kTile : i % kStep, wn = a.w_stride[2] == 1 ? i % kTile : i / kStep;
            const bool in = k0 + wk < a.K && n0 + wn < a.N;
            ws[wk][wn] = in ? to_float(w[(k0 + wk) * a.w_stride[1] + (n0 + wn) * a.w_stride[2]]) : 0.f;
            if constexpr (GATED) us[wk][wn] = in ? to_float(up[(k0 + wk) * a.up_stride[1] + (n0 + wn) * a.up_stride[2]]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            float xv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) xv[i] = xs[k][ty * 4 + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float wv = ws[k][tx + 16 * j];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i][j] = fmaf(xv[i], wv, acc[i][j]);
                if constexpr (GATED) {
                    const float uv = us[k][tx + 16 * j];
#pragma unroll
                    for (int i = 0; i < 4; ++i) gate[i][j] = fmaf(xv[i], uv, gate[i][j]);
                }
            }
        }
        __syncthreads();
    }
    const T* bias = a.bias ? static_cast<const T*>(a.bias) + e * a.bias_stride : nullptr;
    const T* up_bias = GATED && a.up_bias ? static_cast<const T*>(a.up_bias) + e * a.up_bias_stride : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = row0 + ty * 4 + i;
        if (r >= row_end) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (n >= a.N) break;
            float h = activate(acc[i][j] + (bias ? to_float(bias[n]) : 0.f), a.act);
            if constexpr (GATED) h *= gate[i][j] + (up_bias ? to_float(up_bias[n]) : 0.f);
            if (a.residual) h += to_float(static_cast<const TO*>(a.residual)[r * a.res_stride + n]);
            static_cast<TO*>(a.out)[r * a.out_stride + n] = from_float<TO>(h);
        }
    }
}

template <typename T, typename TO>
int launch(const LinearArgs& a, cudaStream_t stream) {
    // every group rounds its rows up to whole tiles: at most one tile more per group than the rows fill, and one that only
    // reads the offsets to their end
    const int64_t row_tiles = ceil_div(a.rows, (int64_t)kTile) + (a.offsets ? std::min(a.groups, a.rows) + 1 : 0);
    const int64_t col_tiles = ceil_div(a.N, (int64_t)kTile);
    if (row_tiles > 0x7fffffffLL || col_tiles > 65535) return fail(SFB_ERR_UNSUPPORTED, "linear: too many tiles");
    const dim3 grid((unsigned)row_tiles, (unsigned)col_tiles);
    if (a.up) linear_generic_kernel<T, TO, true><<<grid, 256, 0, stream>>>(a);
    else linear_generic_kernel<T, TO, false><<<grid, 256, 0, stream>>>(a);
    SFB_CUDA_CHECK(cudaGetLastError());
    return SFB_OK;
}

}  // namespace

int launch_linear_generic(const LinearArgs& a, cudaStream_t stream) {
    const bool wide = a.out_dtype == SFB_F32;
    if (a.dtype == SFB_F32) return launch<float, float>(a, stream);
    if (a.dtype == SFB_BF16) return wide ? launch<__nv_bfloat16, float>(a, stream) : launch<__nv_bfloat16, __nv_bfloat16>(a, stream);
    return wide ? launch<__half, float>(a, stream) : launch<__half, __half>(a, stream);
}

}  // namespace sfb
