// fp8_capi.cu -- C entry points of the block-scaled FP8 products and the routed
// experts around them (include/gemm_sm100.h): argument checks, then the kernels'
// launchers. No exception leaves an entry point, and the handle's device is
// current while it runs.
#include <new>
#include <string>

#include "gs_fp8.h"

namespace gs {
namespace {

constexpr int kMaxDim = 0x7fffffff - 1024;  // 32-bit coordinates run up to one tile past the end
constexpr int kMaxRow = 1 << 30;            // the element-wise kernels' run up to one block's step past it

class DeviceGuard {
public:
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&prev_) != cudaSuccess || prev_ == device) prev_ = -1;
        else if (cudaSetDevice(device) != cudaSuccess) cudaGetLastError();
    }
    ~DeviceGuard() {
        if (prev_ >= 0) cudaSetDevice(prev_);
    }
    DeviceGuard(const DeviceGuard &) = delete;
    DeviceGuard &operator=(const DeviceGuard &) = delete;

private:
    int prev_ = -1;
};

// A check's answer: null, or why the call is refused.
struct Refusal {
    gs_status status = GS_STATUS_SUCCESS;
    const char *why = nullptr;
};
Refusal invalid(const char *why) { return {GS_STATUS_INVALID_VALUE, why}; }
Refusal unsupported(const char *why) { return {GS_STATUS_NOT_SUPPORTED, why}; }

// Runs `check` (fills a descriptor; sets *empty when nothing is to be done), then `launch`. The arguments are
// checked before the handle, so a refusal is the same without a device.
template <typename Check, typename Launch>
gs_status call(gs_handle h, Check check, Launch launch) noexcept {
    try {
        bool empty = false;
        const Refusal r = check(&empty);
        if (!h) return r.status != GS_STATUS_SUCCESS ? r.status : GS_STATUS_NOT_INITIALIZED;
        Context &ctx = h->ctx;
        ctx.last_kernels = 0;
        ctx.last_error.clear();
        if (r.status != GS_STATUS_SUCCESS) {
            ctx.last_error = r.why;
            return r.status;
        }
        if (empty) return GS_STATUS_SUCCESS;
        DeviceGuard guard(ctx.device);
        const cudaError_t e = launch(ctx);
        if (e == cudaSuccess) return GS_STATUS_SUCCESS;
        cudaGetLastError();
        if (ctx.last_error.empty()) ctx.last_error = std::string("kernel launch: ") + cudaGetErrorString(e);
        return GS_STATUS_EXECUTION_FAILED;
    } catch (const std::bad_alloc &) {
        return GS_STATUS_ALLOC_FAILED;
    } catch (...) {
        return GS_STATUS_INTERNAL_ERROR;
    }
}

bool on(const void *p, size_t align) { return reinterpret_cast<uintptr_t>(p) % align == 0; }
bool float_type(int t) { return t == GS_R_32F || t == GS_R_16F || t == GS_R_16BF; }
bool fp8_type(int t) { return t == GS_R_8F_E4M3 || t == GS_R_8F_E5M2; }
size_t float_size(int t) { return t == GS_R_32F ? 4 : 2; }
int blocks128(int x) { return x / 128 + (x % 128 != 0 ? 1 : 0); }
bool valid_mode(int mode) { return mode == GS_SCALE_VEC128 || mode == GS_SCALE_BLK128; }
int at_least_1(int x) { return x > 1 ? x : 1; }

Refusal check_gemm(int ragged, int transa, int transb, int m, int n, int k, int groups, const int32_t *offsets,
                   const float *alpha, const void *A, int at, int lda, long long stride_a, const float *sa, int mode_a,
                   int ldsa, long long stride_sa, const void *B, int bt, int ldb, const float *sb, int mode_b, int ldsb,
                   const float *beta, void *C, int ct, int ldc, long long stride_c, GemmFp8Desc *d, bool *empty) {
    auto valid_op = [](int op) { return op == GS_OP_N || op == GS_OP_T || op == GS_OP_C; };
    if (!valid_op(transa) || !valid_op(transb)) return invalid("invalid op");
    if (m < 0 || n < 0 || k < 0 || groups < 0) return invalid("negative dimension");
    if (!alpha || !beta) return invalid("alpha or beta is null");
    if (!valid_mode(mode_a) || !valid_mode(mode_b)) return invalid("scale mode must be VEC128 or BLK128");
    const bool ta = transa != GS_OP_N, tb = transb != GS_OP_N;
    if (lda < at_least_1(ta ? k : m)) return invalid("lda too small");
    if (ldb < at_least_1(tb ? n : k)) return invalid("ldb too small");
    if (ldc < at_least_1(m)) return invalid("ldc too small");
    const bool a_vec = mode_a == GS_SCALE_VEC128, b_vec = mode_b == GS_SCALE_VEC128;
    if (ldsa < at_least_1(a_vec ? m : blocks128(ta ? k : m))) return invalid("ldsa too small");
    if (ldsb < at_least_1(b_vec ? n : blocks128(tb ? n : k))) return invalid("ldsb too small");
    const bool ragged_n = groups > 0 && ragged == GS_GROUP_N;
    if (groups > 0) {
        if (ragged != GS_GROUP_N && ragged != GS_GROUP_K) return invalid("ragged must be GS_GROUP_N or GS_GROUP_K");
        if (!offsets || !on(offsets, 4)) return invalid("offsets is null or misaligned");
        if (ragged_n && (stride_a < 0 || stride_sa < 0)) return invalid("negative stride");
        if (!ragged_n && groups > 1 && stride_c < static_cast<long long>(n - 1) * ldc + m && m > 0 && n > 0)
            return invalid("strideC too small: the groups' C would overlap");
    }
    if (!fp8_type(at) || !fp8_type(bt)) return unsupported("A and B must be R_8F_E4M3 or R_8F_E5M2");
    if (!float_type(ct)) return unsupported("C must be R_32F, R_16F or R_16BF");
    if (groups > GS_FP8_MAX_GROUPS) return unsupported("too many groups");
    if (ragged_n && tb) return unsupported("ragged N needs op(B) = N");
    if (ragged_n && !b_vec) return unsupported("ragged N needs B's scales per column (VEC128)");
    if (m == 0 || n == 0) {
        *empty = true;
        return {};
    }
    if (m > kMaxDim || n > kMaxDim || k > kMaxDim) return unsupported("m, n and k are limited to 2^31 - 1025");
    // tiles of the smallest kind, and one more round of them, are counted in 32 bits
    const long long across = n / 32 + (ragged_n ? groups : 1);
    if (across > kMaxDim / blocks128(m) || (groups > 0 && !ragged_n && across * blocks128(m) > kMaxDim / groups)) return unsupported("too many tiles");
    if (!C || !on(C, float_size(ct))) return invalid("C is null or misaligned");
    if (k > 0) {
        if (!A || !B || !sa || !sb) return invalid("null operand or scale");
        if (!on(sa, 4) || !on(sb, 4)) return invalid("misaligned scale");
        if (!on(A, 16) || !on(B, 16) || lda % 16 != 0 || ldb % 16 != 0 || (ragged_n && stride_a % 16 != 0))
            return unsupported("A and B need 16-byte aligned addresses, leading dimensions and strides");
    }
    d->trans_a = ta;
    d->trans_b = tb;
    d->m = m;
    d->n = n;
    d->k = k;
    d->groups = groups;
    d->ragged = ragged;
    d->offsets = offsets;
    d->A = A;
    d->lda = lda;
    d->stride_a = stride_a;
    d->a_e5m2 = at == GS_R_8F_E5M2;
    d->sa = sa;
    d->a_vec = a_vec;
    d->ldsa = ldsa;
    d->stride_sa = stride_sa;
    d->B = B;
    d->ldb = ldb;
    d->b_e5m2 = bt == GS_R_8F_E5M2;
    d->sb = sb;
    d->b_vec = b_vec;
    d->ldsb = ldsb;
    d->C = C;
    d->ldc = ldc;
    d->stride_c = stride_c;
    d->out_kind = ct == GS_R_32F ? OUT_F32 : ct == GS_R_16F ? OUT_F16 : OUT_BF16;
    d->ep = Epilogue{};
    d->ep.alpha_f = *alpha;
    d->ep.beta_f = *beta;
    d->ep.beta_zero = *beta == 0.0f;
    d->ep.identity = *alpha == 1.0f;
    return {};
}

bool route_rows(int tokens, int experts, int top_k, int align, long long *rows) {
    const long long slots = static_cast<long long>(tokens) * top_k;
    *rows = slots + (slots < experts ? slots : experts) * static_cast<long long>(align - 1);
    return *rows <= kMaxDim;
}

// What gs_moe_route and its gradient share.
Refusal check_route(const gs_route_desc *q) {
    if (!q) return invalid("null descriptor");
    if (q->tokens < 0) return invalid("negative dimension");
    if (q->experts < 1 || q->top_k < 1 || q->top_k > q->experts) return invalid("experts and top_k must be positive, top_k at most experts");
    if (q->score != GS_ROUTE_SOFTMAX && q->score != GS_ROUTE_SIGMOID) return invalid("unknown score function");
    if (q->ld_logits < q->experts) return invalid("ld_logits too small");
    if (!float_type(q->logits_type)) return unsupported("logits must be R_32F, R_16F or R_16BF");
    if (q->experts > GS_ROUTE_MAX_EXPERTS || q->top_k > GS_ROUTE_MAX_TOP_K) return unsupported("at most 1024 experts and top_k 32");
    if (static_cast<long long>(q->tokens) * q->top_k > kMaxDim) return unsupported("too many slots");
    if (q->tokens > 0 && (!q->logits || !on(q->logits, float_size(q->logits_type)))) return invalid("logits is null or misaligned");
    return {};
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

gs_status gs_fp8_quantize(gs_handle h, int mode, int axis, int rows, int cols, const void *src, int src_type, int ldsrc,
                          const int32_t *index, int index_div, int src_cols, void *dst, int dst_type, int lddst, float *scale,
                          int ldscale) {
    QuantDesc d{};
    return call(
        h,
        [&](bool *empty) -> Refusal {
            if (!valid_mode(mode)) return invalid("scale mode must be VEC128 or BLK128");
            if (axis != 0 && (axis != 1 || mode == GS_SCALE_BLK128)) return invalid("axis must be 0, or 1 with VEC128");
            if (rows < 0 || cols < 0) return invalid("negative dimension");
            if (ldsrc < at_least_1(rows) || lddst < at_least_1(rows)) return invalid("ldsrc or lddst too small");
            if (ldscale < at_least_1(mode == GS_SCALE_BLK128 ? blocks128(rows) : axis == 0 ? cols : rows)) return invalid("ldscale too small");
            if (index && (index_div < 1 || src_cols < 0)) return invalid("indexDiv must be positive and srcCols not negative");
            if (!float_type(src_type)) return unsupported("src must be R_32F, R_16F or R_16BF");
            if (!fp8_type(dst_type)) return unsupported("dst must be R_8F_E4M3 or R_8F_E5M2");
            if (rows > kMaxRow || cols > kMaxRow) return unsupported("rows and cols are limited to 2^30");
            if (rows == 0 || cols == 0) {
                *empty = true;
                return {};
            }
            const bool no_source = index && src_cols == 0;
            if ((!src && !no_source) || !dst || !scale) return invalid("null pointer");
            if (!on(src, float_size(src_type)) || !on(scale, 4) || !on(index, 4)) return invalid("misaligned pointer");
            d.blk = mode == GS_SCALE_BLK128;
            d.axis = axis;
            d.rows = rows;
            d.cols = cols;
            d.src = src;
            d.src_type = src_type;
            d.ld_src = ldsrc;
            d.src_cols = index ? src_cols : cols;
            d.index = index;
            d.index_div = index ? index_div : 1;
            d.dst = dst;
            d.e5m2 = dst_type == GS_R_8F_E5M2;
            d.ld_dst = lddst;
            d.scale = scale;
            d.ld_scale = ldscale;
            return {};
        },
        [&](Context &ctx) { return launch_quantize(ctx, d); });
}

gs_status gs_gemm_fp8_grouped(gs_handle h, int ragged, int transa, int transb, int m, int n, int k, int groups,
                              const int32_t *offsets, const float *alpha, const void *A, int at, int lda, long long stride_a,
                              const float *sa, int mode_a, int ldsa, long long stride_sa, const void *B, int bt, int ldb,
                              const float *sb, int mode_b, int ldsb, const float *beta, void *C, int ct, int ldc,
                              long long stride_c) {
    GemmFp8Desc d{};
    return call(
        h,
        [&](bool *empty) -> Refusal {
            if (groups < 1) return invalid("groups must be positive");
            return check_gemm(ragged, transa, transb, m, n, k, groups, offsets, alpha, A, at, lda, stride_a, sa, mode_a, ldsa,
                              stride_sa, B, bt, ldb, sb, mode_b, ldsb, beta, C, ct, ldc, stride_c, &d, empty);
        },
        [&](Context &ctx) { return launch_gemm_fp8(ctx, d); });
}

gs_status gs_gemm_fp8(gs_handle h, int transa, int transb, int m, int n, int k, const float *alpha, const void *A, int at,
                      int lda, const float *sa, int mode_a, int ldsa, const void *B, int bt, int ldb, const float *sb,
                      int mode_b, int ldsb, const float *beta, void *C, int ct, int ldc) {
    GemmFp8Desc d{};
    return call(
        h,
        [&](bool *empty) -> Refusal {
            return check_gemm(GS_GROUP_N, transa, transb, m, n, k, 0, nullptr, alpha, A, at, lda, 0, sa, mode_a, ldsa, 0, B, bt,
                              ldb, sb, mode_b, ldsb, beta, C, ct, ldc, 0, &d, empty);
        },
        [&](Context &ctx) { return launch_gemm_fp8(ctx, d); });
}

gs_status gs_plan_gemm_fp8_ex(int ragged, int transa, int transb, int m, int n, int k, int mode_a, int mode_b, int ct,
                              int c_aligned, int groups, int sm_count, int *columns, int *ctas, int *k_slices) {
    if (!columns || !ctas || !k_slices || sm_count < 1 || m < 1 || n < 1 || k < 0 || groups < 0 || groups > GS_FP8_MAX_GROUPS)
        return GS_STATUS_INVALID_VALUE;
    if (groups > 0 && ragged != GS_GROUP_N && ragged != GS_GROUP_K) return GS_STATUS_INVALID_VALUE;
    if (!valid_mode(mode_a) || !valid_mode(mode_b) || !float_type(ct)) return GS_STATUS_INVALID_VALUE;
    GemmFp8Desc d{};
    d.trans_a = transa != GS_OP_N;
    d.trans_b = transb != GS_OP_N;
    d.m = m;
    d.n = n;
    d.k = k;
    d.groups = groups;
    d.ragged = ragged;
    d.a_vec = mode_a == GS_SCALE_VEC128;
    d.b_vec = mode_b == GS_SCALE_VEC128;
    d.out_kind = ct == GS_R_32F ? OUT_F32 : ct == GS_R_16F ? OUT_F16 : OUT_BF16;
    d.ldc = c_aligned ? 16 : 1;  // stands for any that is a multiple of 16 bytes, or is not
    const fp8::Tile t = fp8::choose_tile(d, sm_count);
    *columns = t.bn;
    *ctas = t.cg;
    *k_slices = t.split;
    return GS_STATUS_SUCCESS;
}

gs_status gs_plan_gemm_fp8(int ragged, int transa, int transb, int m, int n, int k, int groups, int sm_count, int *columns,
                           int *ctas, int *k_slices) {
    return gs_plan_gemm_fp8_ex(ragged, transa, transb, m, n, k, GS_SCALE_BLK128, GS_SCALE_VEC128, GS_R_16BF, 1, groups,
                               sm_count, columns, ctas, k_slices);
}

gs_status gs_moe_rows(int tokens, int experts, int top_k, int align, int *rows) {
    long long n = 0;
    if (!rows || tokens < 0 || experts < 1 || top_k < 1 || align < 1) return GS_STATUS_INVALID_VALUE;
    if (!route_rows(tokens, experts, top_k, align, &n)) return GS_STATUS_NOT_SUPPORTED;
    *rows = static_cast<int>(n);
    return GS_STATUS_SUCCESS;
}

gs_status gs_moe_route_workspace(int tokens, int experts, int top_k, size_t *bytes) {
    if (!bytes || tokens < 0 || experts < 1 || top_k < 1) return GS_STATUS_INVALID_VALUE;
    *bytes = static_cast<size_t>(route_blocks(tokens, top_k)) * static_cast<size_t>(experts) * sizeof(int32_t);
    return GS_STATUS_SUCCESS;
}

gs_status gs_moe_route(gs_handle h, const gs_route_desc *q) {
    RouteDesc d{};
    return call(
        h,
        [&](bool *empty) -> Refusal {
            const Refusal r = check_route(q);
            if (r.status != GS_STATUS_SUCCESS) return r;
            if (q->groups < 1 || q->experts % q->groups != 0) return invalid("experts must be a multiple of groups");
            if (q->top_groups < 1 || q->top_groups > q->groups) return invalid("top_groups must lie in 1..groups");
            if (q->top_k > q->experts / q->groups * q->top_groups) return invalid("top_k exceeds the kept groups' experts");
            if (q->align < 1) return invalid("align must be positive");
            if (q->groups > GS_ROUTE_MAX_GROUPS) return unsupported("at most 32 groups");
            if (!on(q->bias, 4) || !on(q->token_count, 4) || !on(q->ids, 4) || !on(q->weights, 4) || !on(q->offsets, 4) ||
                !on(q->slot_row, 4) || !on(q->row_slot, 4) || !on(q->workspace, 4))
                return invalid("misaligned pointer");
            if (q->tokens > 0 && (!q->ids || !q->weights)) return invalid("ids or weights is null");
            if (q->offsets) {
                long long need = 0;
                if (!route_rows(q->tokens, q->experts, q->top_k, q->align, &need)) return unsupported("too many rows");
                if (q->rows < need) return invalid("rows is less than gs_moe_rows");
                if (q->rows > kMaxDim) return unsupported("too many rows");
                if ((q->tokens > 0 && !q->slot_row) || (q->rows > 0 && !q->row_slot)) return invalid("slot_row or row_slot is null");
                const size_t bytes = static_cast<size_t>(route_blocks(q->tokens, q->top_k)) * static_cast<size_t>(q->experts) * 4;
                if (bytes > 0 && (!q->workspace || q->workspace_bytes < bytes)) return invalid("workspace too small");
            } else if (q->tokens == 0) {
                *empty = true;
            }
            d.tokens = q->tokens;
            d.experts = q->experts;
            d.top_k = q->top_k;
            d.logits = q->logits;
            d.type = q->logits_type;
            d.ld = q->ld_logits;
            d.bias = q->bias;
            d.sigmoid = q->score == GS_ROUTE_SIGMOID;
            d.groups = q->groups;
            d.top_groups = q->top_groups;
            d.group_size = q->experts / q->groups;
            d.group_magic = ((1u << 20) + static_cast<uint32_t>(d.group_size) - 1) / static_cast<uint32_t>(d.group_size);
            d.renorm = q->renormalize != 0;
            d.scale = q->scale;
            d.token_count = q->token_count;
            d.align = q->align;
            d.ids = q->ids;
            d.weights = q->weights;
            d.offsets = q->offsets;
            d.slot_row = q->slot_row;
            d.row_slot = q->row_slot;
            d.rows = q->rows;
            d.hist = static_cast<int32_t *>(q->workspace);
            return {};
        },
        [&](Context &ctx) { return launch_route(ctx, d); });
}

gs_status gs_moe_route_backward(gs_handle h, const gs_route_desc *q, const float *dweights, void *dlogits, int dtype, int ldd) {
    RouteBwdDesc d{};
    return call(
        h,
        [&](bool *empty) -> Refusal {
            const Refusal r = check_route(q);
            if (r.status != GS_STATUS_SUCCESS) return r;
            if (ldd < q->experts) return invalid("lddlogits too small");
            if (dtype != q->logits_type && dtype != GS_R_32F) return unsupported("dlogits must have the logits' type or R_32F");
            if (q->tokens == 0) {
                *empty = true;
                return {};
            }
            if (!q->ids || !dweights || !dlogits) return invalid("null pointer");
            if (!on(q->ids, 4) || !on(dweights, 4) || !on(dlogits, float_size(dtype))) return invalid("misaligned pointer");
            d.tokens = q->tokens;
            d.experts = q->experts;
            d.top_k = q->top_k;
            d.logits = q->logits;
            d.type = q->logits_type;
            d.ld = q->ld_logits;
            d.ids = q->ids;
            d.dweights = dweights;
            d.sigmoid = q->score == GS_ROUTE_SIGMOID;
            d.renorm = q->renormalize != 0;
            d.scale = q->scale;
            d.dlogits = dlogits;
            d.dtype = dtype;
            d.ldd = ldd;
            return {};
        },
        [&](Context &ctx) { return launch_route_backward(ctx, d); });
}

static Refusal check_combine(int tokens, int top_k, int hidden, const void *y, int type, int ldy, int rows, const int32_t *slot_row) {
    if (tokens < 0 || hidden < 0 || rows < 0) return invalid("negative dimension");
    if (top_k < 1) return invalid("top_k must be positive");
    if (ldy < at_least_1(hidden)) return invalid("ldy too small");
    if (!float_type(type)) return unsupported("y must be R_32F, R_16F or R_16BF");
    if (static_cast<long long>(tokens) * top_k > kMaxDim || rows > kMaxDim || hidden > kMaxRow) return unsupported("too many slots or rows, or hidden above 2^30");
    if (tokens > 0 && hidden > 0 && rows > 0 && !y) return invalid("y is null");
    if (tokens > 0 && !slot_row) return invalid("slot_row is null");
    if (!on(y, float_size(type)) || !on(slot_row, 4)) return invalid("misaligned pointer");
    return {};
}

gs_status gs_moe_combine(gs_handle h, int tokens, int top_k, int hidden, const void *y, int type, int ldy, int rows,
                         const int32_t *slot_row, const float *weights, void *out, int out_type, int ldout) {
    CombineDesc d{};
    return call(
        h,
        [&](bool *empty) -> Refusal {
            const Refusal r = check_combine(tokens, top_k, hidden, y, type, ldy, rows, slot_row);
            if (r.status != GS_STATUS_SUCCESS) return r;
            if (ldout < at_least_1(hidden)) return invalid("ldout too small");
            if (!float_type(out_type)) return unsupported("out must be R_32F, R_16F or R_16BF");
            if (tokens == 0 || hidden == 0) {
                *empty = true;
                return {};
            }
            if (!out) return invalid("out is null");
            if (!on(out, float_size(out_type)) || !on(weights, 4)) return invalid("misaligned pointer");
            d.tokens = tokens;
            d.top_k = top_k;
            d.hidden = hidden;
            d.rows = rows;
            d.y = y;
            d.type = type;
            d.ldy = ldy;
            d.slot_row = slot_row;
            d.weights = weights;
            d.out = out;
            d.out_type = out_type;
            d.ldo = ldout;
            return {};
        },
        [&](Context &ctx) { return launch_combine(ctx, d); });
}

gs_status gs_moe_combine_backward(gs_handle h, int tokens, int top_k, int hidden, const void *y, int type, int ldy, int rows,
                                  const int32_t *slot_row, const int32_t *row_slot, const float *weights, const void *dout,
                                  int lddout, void *dy, int lddy, float *dweights) {
    CombineDesc d{};
    return call(
        h,
        [&](bool *empty) -> Refusal {
            const Refusal r = check_combine(tokens, top_k, hidden, y, type, ldy, rows, slot_row);
            if (r.status != GS_STATUS_SUCCESS) return r;
            if (lddout < at_least_1(hidden) || lddy < at_least_1(hidden)) return invalid("lddout or lddy too small");
            if (tokens == 0 && rows == 0) {
                *empty = true;
                return {};
            }
            if (rows > 0 && (!row_slot || (hidden > 0 && !dy))) return invalid("row_slot or dy is null");
            if (tokens > 0 && (!weights || !dweights || (hidden > 0 && !dout))) return invalid("weights, dout or dweights is null");
            if (!on(row_slot, 4) || !on(weights, 4) || !on(dweights, 4) || !on(dout, float_size(type)) || !on(dy, float_size(type)))
                return invalid("misaligned pointer");
            d.tokens = tokens;
            d.top_k = top_k;
            d.hidden = hidden;
            d.rows = rows;
            d.y = y;
            d.type = type;
            d.ldy = ldy;
            d.slot_row = slot_row;
            d.row_slot = row_slot;
            d.weights = weights;
            d.dout = dout;
            d.lddo = lddout;
            d.dy = dy;
            d.lddy = lddy;
            d.dweights = dweights;
            return {};
        },
        [&](Context &ctx) { return launch_combine_backward(ctx, d); });
}

}  // extern "C"
