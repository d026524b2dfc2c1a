// C-ABI entry points of the feed-forward operators: descriptor validation, error text, dispatch.

#include "linear.cuh"

using namespace sfb;

namespace {

bool float_type(int dt) { return dt == SFB_F32 || dt == SFB_BF16 || dt == SFB_F16; }

// An optional [.., n] vector per group: element stride between groups, size and contiguity checked.
int vector_view(const SFBTensor* t, const char* what, int64_t groups, int64_t n, bool grouped, int elem, const void** base, int64_t* stride) {
    if (!t) return SFB_OK;
    View v;
    const int rank = grouped ? 2 : 1;
    if (const int rc = make_view(t, what, rank, rank, elem, &v)) return rc;
    if (v.size[3] != n || v.size[2] != (grouped ? groups : 1)) return fail(SFB_ERR_INVALID_ARG, "%s: expected %s", what, grouped ? "[E, N]" : "[N]");
    *base = v.base;
    *stride = v.stride[2];
    return SFB_OK;
}

int index_view(const SFBTensor* t, const char* what, int rank, View* v) {
    if (const int rc = make_view(t, what, rank, rank, 4, v)) return rc;
    return SFB_OK;
}

// Whether rows [rows][width bytes], `stride` bytes apart, share memory with others.  Exact for equal strides (column slices of
// one buffer) and where either is one block of memory; two interleaved patterns of different strides are left to the caller.
struct Rows {
    const char* base;
    int64_t rows, stride, width;
    Rows(const void* p, int64_t n, int64_t stride_elements, int64_t columns, int elem)
        : base(static_cast<const char*>(p)), rows(n), stride(n > 1 ? stride_elements * elem : columns * elem), width(columns * elem) {}
    const char* end() const { return base + (rows - 1) * stride + width; }
};
bool share_memory(const Rows& a, const Rows& b) {
    if (a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1 || a.end() <= b.base || b.end() <= a.base) return false;
    for (int i = 0; i < 2; ++i) {
        const Rows &block = i ? b : a, &other = i ? a : b;
        if (block.stride > block.width) continue;
        if (other.stride <= 0) return true;
        // the first row of `other` that ends behind the block's start
        const int64_t before = block.base - other.base - other.width, first = before < 0 ? 0 : before / other.stride + 1;
        return first < other.rows && other.base + first * other.stride < block.end();
    }
    if (a.stride != b.stride) return false;
    const int64_t apart = ((b.base - a.base) % a.stride + a.stride) % a.stride;
    return apart < a.width || apart + b.width > a.stride;
}

// Row and column numbers are 32-bit, those of a tile's end and of a grid stride further on too.
constexpr int64_t kMostRows = 0x7fff0000LL;

// Fills the parts that the dense and the grouped product have in common.
int linear_views(const char* op, const SFBTensor* x, const SFBTensor* weight, const SFBTensor* bias, const SFBTensor* up_weight,
                 const SFBTensor* up_bias, SFBTensor* out, bool grouped, int layout, int dtype, int out_dtype, int activation, LinearArgs* a) {
    if (!float_type(dtype) || (out_dtype != dtype && out_dtype != SFB_F32)) return fail(SFB_ERR_UNSUPPORTED, "%s: fp32, bf16 or fp16 operands, out in the same type or fp32", op);
    if (layout != SFB_WEIGHT_KN && layout != SFB_WEIGHT_NK) return fail(SFB_ERR_INVALID_ARG, "%s: weight layout %d", op, layout);
    if (activation < SFB_ACT_NONE || activation > SFB_ACT_RELU) return fail(SFB_ERR_INVALID_ARG, "%s: activation %d", op, activation);
    if (up_bias && !up_weight) return fail(SFB_ERR_INVALID_ARG, "%s: up_bias without up_weight", op);
    const int e = dtype_size(dtype), rank = grouped ? 3 : 2;
    View vx, vw, vu, vo;
    int rc;
    if ((rc = make_view(x, "x", 2, 2, e, &vx))) return rc;
    if ((rc = make_view(weight, "weight", rank, rank, e, &vw))) return rc;
    if ((rc = make_view(out, "out", 2, 2, dtype_size(out_dtype), &vo))) return rc;
    const bool nk = layout == SFB_WEIGHT_NK;
    a->K = vx.size[3];
    a->N = vo.size[3];
    a->groups = vw.size[1];
    a->rows = vo.size[2];
    a->x_rows = vx.size[2];
    const int64_t d2 = nk ? a->N : a->K, d3 = nk ? a->K : a->N;
    if (vw.size[2] != d2 || vw.size[3] != d3)
        return fail(SFB_ERR_INVALID_ARG, "%s: weight is [.., %lld, %lld], x and out ask for [.., %lld, %lld]", op, (long long)vw.size[2], (long long)vw.size[3], (long long)d2, (long long)d3);
    auto strides = [&](const View& v, int64_t* s) { s[0] = v.stride[1]; s[1] = nk ? 1 : v.stride[2]; s[2] = nk ? v.stride[2] : 1; };
    a->w = vw.base;
    strides(vw, a->w_stride);
    if (up_weight) {
        if ((rc = make_view(up_weight, "up_weight", rank, rank, e, &vu))) return rc;
        for (int i = 1; i < 4; ++i)
            if (vu.size[i] != vw.size[i]) return fail(SFB_ERR_INVALID_ARG, "%s: up_weight must have weight's shape", op);
        a->up = vu.base;
        strides(vu, a->up_stride);
    }
    if ((rc = vector_view(bias, "bias", a->groups, a->N, grouped, e, &a->bias, &a->bias_stride))) return rc;
    if ((rc = vector_view(up_bias, "up_bias", a->groups, a->N, grouped, e, &a->up_bias, &a->up_bias_stride))) return rc;
    if (vo.size[2] > 1 && vo.stride[2] < a->N) return fail(SFB_ERR_INVALID_ARG, "%s: rows of out overlap (stride %lld)", op, (long long)vo.stride[2]);
    a->x = vx.base;
    a->x_stride = vx.stride[2];
    a->out = vo.base;
    a->out_stride = vo.stride[2];
    a->layout = layout;
    a->dtype = dtype;
    a->out_dtype = out_dtype;
    a->act = activation;
    const int64_t most = kMostRows;
    if (a->rows > most || a->x_rows > most || a->K > most || a->N > most) return fail(SFB_ERR_UNSUPPORTED, "%s: dimension too large", op);
    return SFB_OK;
}

// The tensor cores where TMA can address the operands, else the CUDA cores.
int launch_linear(const LinearArgs& a, cudaStream_t stream) {
    const int rc = launch_linear_tcgen05(a, stream);
    return rc == SFB_ERR_UNSUPPORTED ? launch_linear_generic(a, stream) : rc;
}

}  // namespace

extern "C" {

int sfb_fused_linear(const SFBTensor* x, const SFBTensor* weight, const SFBTensor* bias, const SFBTensor* up_weight, const SFBTensor* up_bias,
                     const SFBTensor* residual, SFBTensor* out, int weight_layout, int dtype, int out_dtype, int activation, int32_t* status,
                     void* stream) {
    SFB_TRACE_OP("fused_linear", stream, "dtype %d activation %d gated %d", dtype, activation, up_weight ? 1 : 0);
    LinearArgs a{};
    if (const int rc = linear_views("fused_linear", x, weight, bias, up_weight, up_bias, out, false, weight_layout, dtype, out_dtype, activation, &a)) return rc;
    if (a.x_rows != a.rows) return fail(SFB_ERR_INVALID_ARG, "fused_linear: x [M, K], out [M, N]");
    if (residual) {
        View vr;
        if (const int rc = make_view(residual, "residual", 2, 2, dtype_size(out_dtype), &vr)) return rc;
        if (vr.size[2] != a.rows || vr.size[3] != a.N) return fail(SFB_ERR_INVALID_ARG, "fused_linear: residual must have out's shape");
        a.residual = vr.base;
        a.res_stride = vr.stride[2];
    }
    if (a.rows == 0 || a.N == 0) return SFB_OK;
    if (a.K == 0) return fail(SFB_ERR_INVALID_ARG, "fused_linear: K is zero");
    const Rows o(a.out, a.rows, a.out_stride, a.N, dtype_size(out_dtype));
    if (share_memory(o, Rows(a.x, a.x_rows, a.x_stride, a.K, dtype_size(dtype)))) return fail(SFB_ERR_INVALID_ARG, "fused_linear: out shares memory with x");
    if (a.residual && !(a.residual == a.out && (a.rows == 1 || a.res_stride == a.out_stride)) &&
        share_memory(o, Rows(a.residual, a.rows, a.res_stride, a.N, dtype_size(out_dtype))))
        return fail(SFB_ERR_INVALID_ARG, "fused_linear: out shares memory with the residual, but is not the residual");
    a.status = status;
    return launch_linear(a, static_cast<cudaStream_t>(stream));
}

int64_t sfb_grouped_linear_workspace_bytes(int64_t rows, int64_t K, int64_t groups, int indexed) {
    if (rows < 0 || K < 0 || groups < 1) return SFB_ERR_INVALID_ARG;
    return indexed && rows >= kOrderedRows * groups ? rows * ceil_div(K, (int64_t)8) * 16 : 0;
}

int sfb_grouped_linear(const SFBTensor* x, const SFBTensor* weight, const SFBTensor* bias, const SFBTensor* up_weight, const SFBTensor* up_bias,
                       const SFBTensor* group_offsets, const SFBTensor* row_index, SFBTensor* out, int weight_layout, int dtype, int out_dtype,
                       int activation, int32_t* status, void* workspace, int64_t workspace_bytes, void* stream) {
    SFB_TRACE_OP("grouped_linear", stream, "dtype %d activation %d gated %d", dtype, activation, up_weight ? 1 : 0);
    LinearArgs a{};
    if (const int rc = linear_views("grouped_linear", x, weight, bias, up_weight, up_bias, out, true, weight_layout, dtype, out_dtype, activation, &a)) return rc;
    if (a.groups < 1 || a.groups > kMaxGroups) return fail(SFB_ERR_UNSUPPORTED, "grouped_linear: 1 to %d groups, got %lld", kMaxGroups, (long long)a.groups);
    View vg, vi;
    int rc;
    if ((rc = index_view(group_offsets, "group_offsets", 1, &vg))) return rc;
    if (vg.size[3] != a.groups + 1) return fail(SFB_ERR_INVALID_ARG, "grouped_linear: group_offsets must have E + 1 = %lld entries", (long long)a.groups + 1);
    a.offsets = reinterpret_cast<const int32_t*>(vg.base);
    if (row_index) {
        if ((rc = index_view(row_index, "row_index", 1, &vi))) return rc;
        if (vi.size[3] != a.rows) return fail(SFB_ERR_INVALID_ARG, "grouped_linear: row_index must have one entry for every row of out");
        a.row_index = reinterpret_cast<const int32_t*>(vi.base);
        if (a.rows && !a.x_rows) return fail(SFB_ERR_INVALID_ARG, "grouped_linear: x has no rows to index");
    } else if (a.x_rows != a.rows) {
        return fail(SFB_ERR_INVALID_ARG, "grouped_linear: without row_index x and out have the same rows");
    }
    if (a.rows == 0 || a.N == 0) return SFB_OK;
    if (a.K == 0) return fail(SFB_ERR_INVALID_ARG, "grouped_linear: K is zero");
    if (share_memory(Rows(a.out, a.rows, a.out_stride, a.N, dtype_size(out_dtype)), Rows(a.x, a.x_rows, a.x_stride, a.K, dtype_size(dtype))))
        return fail(SFB_ERR_INVALID_ARG, "grouped_linear: out shares memory with x");
    a.workspace = workspace;
    a.workspace_bytes = workspace ? workspace_bytes : 0;
    a.status = status;
    return launch_linear(a, static_cast<cudaStream_t>(stream));
}

int sfb_linear_plan(int64_t rows, int64_t K, int64_t N, int64_t groups, int gated, int indexed, int has_workspace, int sms, int32_t* plan6) {
    if (rows < 1 || K < 1 || N < 1 || rows > kMostRows || K > kMostRows || N > kMostRows || groups < 0 || groups > kMaxGroups || sms < 1 || !plan6) return fail(SFB_ERR_INVALID_ARG, "linear_plan: bad argument");
    const LinearPlan p = plan_linear(rows, K, N, groups ? groups : 1, groups > 0, gated != 0, groups > 0 && indexed, has_workspace != 0, sms);
    plan6[0] = p.tokens; plan6[1] = p.pair; plan6[2] = p.split; plan6[3] = p.order; plan6[4] = p.blocks_an_sm; plan6[5] = (int32_t)p.feat_tiles;
    return SFB_OK;
}

int64_t sfb_moe_route_workspace_bytes(int64_t tokens, int64_t experts) {
    if (tokens < 0 || experts < 0) return SFB_ERR_INVALID_ARG;
    const int64_t blocks = ceil_div(tokens, (int64_t)kRouteTokens);
    return blocks > 1 ? (blocks + 1) * experts * 4 : 0;
}

int sfb_moe_route(const SFBTensor* logits, SFBTensor* expert_ids, SFBTensor* weights, SFBTensor* group_offsets, SFBTensor* token_rows,
                  SFBTensor* positions, int dtype, int renormalize, void* workspace, int64_t workspace_bytes, void* stream) {
    SFB_TRACE_OP("moe_route", stream, "dtype %d renormalize %d", dtype, renormalize);
    if (!float_type(dtype)) return fail(SFB_ERR_UNSUPPORTED, "moe_route: fp32, bf16 or fp16 logits");
    View vl, vi, vw, vo, vt, vp;
    int rc;
    if ((rc = make_view(logits, "logits", 2, 2, dtype_size(dtype), &vl))) return rc;
    if ((rc = index_view(expert_ids, "expert_ids", 2, &vi))) return rc;
    if ((rc = index_view(weights, "weights", 2, &vw))) return rc;
    if ((rc = index_view(group_offsets, "group_offsets", 1, &vo))) return rc;
    if ((rc = index_view(token_rows, "token_rows", 1, &vt))) return rc;
    if ((rc = index_view(positions, "positions", 2, &vp))) return rc;
    const int64_t T = vl.size[2], E = vl.size[3], k = vi.size[3];
    if (E < 1 || E > kMaxGroups) return fail(SFB_ERR_UNSUPPORTED, "moe_route: 1 to %d experts, got %lld", kMaxGroups, (long long)E);
    if (k < 1 || k > E || k > kMaxTopK) return fail(SFB_ERR_INVALID_ARG, "moe_route: top_k %lld outside 1 .. min(experts, %d)", (long long)k, kMaxTopK);
    for (const View* v : {&vi, &vw, &vp}) {
        if (v->size[2] != T || v->size[3] != k) return fail(SFB_ERR_INVALID_ARG, "moe_route: expert_ids, weights and positions are [T, top_k]");
        if (T > 1 && v->stride[2] != k) return fail(SFB_ERR_INVALID_ARG, "moe_route: expert_ids, weights and positions must be contiguous");
    }
    if (vo.size[3] != E + 1 || vt.size[3] != T * k) return fail(SFB_ERR_INVALID_ARG, "moe_route: group_offsets [E + 1], token_rows [T * top_k]");
    if (T * k > 0x7fffffffLL) return fail(SFB_ERR_UNSUPPORTED, "moe_route: too many assignments");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        SFB_CUDA_CHECK(cudaMemsetAsync(vo.base, 0, (size_t)(E + 1) * 4, st));
        return SFB_OK;
    }
    const int64_t need = sfb_moe_route_workspace_bytes(T, E);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(SFB_ERR_WORKSPACE, "moe_route: workspace of %lld B needed, %lld given", (long long)need, (long long)(workspace ? workspace_bytes : 0));
    if (need > 0 && reinterpret_cast<uintptr_t>(workspace) % 4) return fail(SFB_ERR_INVALID_ARG, "moe_route: workspace must start on 4 bytes (int32 counts)");
    RouteArgs a{};
    a.logits = vl.base; a.logits_stride = vl.stride[2];
    a.ids = reinterpret_cast<int32_t*>(vi.base); a.weights = reinterpret_cast<float*>(vw.base);
    a.offsets = reinterpret_cast<int32_t*>(vo.base); a.token_rows = reinterpret_cast<int32_t*>(vt.base);
    a.positions = reinterpret_cast<int32_t*>(vp.base); a.counts = static_cast<int32_t*>(workspace);
    a.tokens = T; a.experts = (int)E; a.top_k = (int)k; a.renormalize = renormalize != 0; a.dtype = dtype;
    return launch_moe_route(a, st);
}

int sfb_moe_combine(const SFBTensor* y, const SFBTensor* positions, const SFBTensor* weights, const SFBTensor* residual, SFBTensor* out, int dtype,
                    int32_t* status, void* stream) {
    SFB_TRACE_OP("moe_combine", stream, "dtype %d residual %d", dtype, residual ? 1 : 0);
    if (!float_type(dtype)) return fail(SFB_ERR_UNSUPPORTED, "moe_combine: fp32, bf16 or fp16");
    const int e = dtype_size(dtype);
    View vy, vp, vw, vr, vo;
    int rc;
    if ((rc = make_view(y, "y", 2, 2, e, &vy))) return rc;
    if ((rc = index_view(positions, "positions", 2, &vp))) return rc;
    if ((rc = index_view(weights, "weights", 2, &vw))) return rc;
    if ((rc = make_view(out, "out", 2, 2, e, &vo))) return rc;
    const int64_t T = vo.size[2], H = vo.size[3], k = vp.size[3];
    if (vy.size[3] != H) return fail(SFB_ERR_INVALID_ARG, "moe_combine: y [R, H], out [T, H]");
    if (k < 1 || k > kMaxTopK) return fail(SFB_ERR_INVALID_ARG, "moe_combine: %lld rows a token outside 1 .. %d", (long long)k, kMaxTopK);
    if (vp.size[2] != T || vw.size[2] != T || vw.size[3] != k) return fail(SFB_ERR_INVALID_ARG, "moe_combine: positions and weights are [T, k]");
    if (T > 1 && vo.stride[2] < H) return fail(SFB_ERR_INVALID_ARG, "moe_combine: rows of out overlap (stride %lld)", (long long)vo.stride[2]);
    CombineArgs a{};
    if (residual) {
        if ((rc = make_view(residual, "residual", 2, 2, e, &vr))) return rc;
        if (vr.size[2] != T || vr.size[3] != H) return fail(SFB_ERR_INVALID_ARG, "moe_combine: residual must have out's shape");
        a.residual = vr.base;
        a.res_stride = vr.stride[2];
    }
    if (T == 0 || H == 0) return SFB_OK;
    const Rows o(vo.base, T, vo.stride[2], H, e);
    if (share_memory(o, Rows(vy.base, vy.size[2], vy.stride[2], H, e))) return fail(SFB_ERR_INVALID_ARG, "moe_combine: out shares memory with y");
    if (residual && !(a.residual == vo.base && (T == 1 || a.res_stride == vo.stride[2])) && share_memory(o, Rows(vr.base, T, vr.stride[2], H, e)))
        return fail(SFB_ERR_INVALID_ARG, "moe_combine: out shares memory with the residual, but is not the residual");
    a.y = vy.base; a.y_stride = vy.stride[2]; a.y_rows = vy.size[2];
    a.positions = reinterpret_cast<const int32_t*>(vp.base); a.pos_stride = vp.stride[2];
    a.weights = reinterpret_cast<const float*>(vw.base); a.weight_stride = vw.stride[2];
    a.out = vo.base; a.out_stride = vo.stride[2];
    a.tokens = T; a.hidden = H; a.top_k = (int)k; a.dtype = dtype;
    a.status = status;
    return launch_moe_combine(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
