// Entry points of the products with quantized weights: checks of arguments, workspace layout, launches.
#include "host_checks.cuh"
#include "linear_backward.cuh"

namespace qk {

// A float matrix [rows, cols] whose rows are contiguous and a constant stride apart; leading dims are rows too.
struct Matrix {
    void *ptr = nullptr;
    long long rows = 0, cols = 0, stride = 0;
};

static int as_matrix(const QkTensor *t, int dtype, Matrix &m)
{
    const int rc = check_tensor(t, dtype_size(dtype));
    if (rc != QK_OK) return rc;
    m.ptr = t->ptr;
    m.cols = t->shape[t->rank - 1];
    m.rows = 1;
    for (int d = 0; d < t->rank - 1; ++d) m.rows *= t->shape[d];
    m.stride = m.cols;
    if (m.rows == 0 || m.cols == 0) return QK_OK;
    if (!is_contiguous(t) && !is_row_strided(t, &m.stride)) {
        // one row of contiguous elements: its strides are never used
        if (m.rows != 1 || (m.cols != 1 && t->strides[t->rank - 1] != 1)) return QK_ERR_LAYOUT;
    }
    if (m.rows > QK_LINEAR_MAX_ROWS || m.cols >= (1ll << 31)) return QK_ERR_TOO_LARGE;
    return QK_OK;
}

static int same_matrix(const QkTensor *t, int dtype, long long rows, long long cols, Matrix &m)
{
    const int rc = as_matrix(t, dtype, m);
    if (rc != QK_OK) return rc;
    return m.rows == rows && m.cols == cols ? QK_OK : QK_ERR_SHAPE;
}

// [N] or [E, N] of any non-negative strides.
static int check_bias(const QkTensor *t, int dtype, bool grouped, long long e, long long n, bool written, long long *stride, long long *expert)
{
    const int rc = check_tensor(t, dtype_size(dtype));
    if (rc != QK_OK) return rc;
    if (t->rank != (grouped ? 2 : 1) || t->shape[t->rank - 1] != n || (grouped && t->shape[0] != e)) return QK_ERR_SHAPE;
    *stride = n > 1 ? t->strides[t->rank - 1] : 1;
    *expert = grouped && e > 1 ? t->strides[0] : 0;
    if (*stride < 0 || *expert < 0) return QK_ERR_LAYOUT;
    // a gradient must not have two elements in one place
    if (written && ((n > 1 && *stride == 0) || (grouped && e > 1 && *expert < (n - 1) * *stride + 1))) return QK_ERR_LAYOUT;
    return QK_OK;
}

// The weight's part of the arguments.  `values` is [N, K / num_quants] or [E, N, K / num_quants], rows contiguous.
static int fill_weight(LinearArgs &a, const QkTensor *values, const QkTensor *params, const QkScheme *s, bool grouped)
{
    const int nq = num_quants(s);
    const int item = s->store == QK_STORE_U32 ? 4 : 1;
    int rc = check_tensor(values, item);
    if (rc != QK_OK) return rc;
    rc = check_tensor(params, dtype_size(s->param));
    if (rc != QK_OK) return rc;
    const int r = grouped ? 3 : 2;
    if (values->rank != r) return QK_ERR_SHAPE;
    const long long e = grouped ? values->shape[0] : 1, n = values->shape[r - 2], items = values->shape[r - 1], k = items * nq;
    if (grouped && e < 1) return QK_ERR_SHAPE;
    if (n >= QK_LINEAR_MAX_EXTENT || k >= QK_LINEAR_MAX_EXTENT || e > QK_LINEAR_MAX_EXPERTS) return QK_ERR_TOO_LARGE;
    a.experts = (int)e;
    a.n = (int)n;
    a.k = (int)k;
    if (n > 0 && items > 1 && values->strides[r - 1] != 1) return QK_ERR_LAYOUT;
    const long long row = n > 1 ? values->strides[r - 2] : items, expert = grouped && e > 1 ? values->strides[0] : 0;
    if (row < 0 || expert < 0) return QK_ERR_LAYOUT;
    a.codes = static_cast<const uint8_t *>(values->ptr);
    a.code_row = row * item;
    a.code_expert = expert * item;
    const unsigned long long all = reinterpret_cast<uintptr_t>(values->ptr) | (unsigned long long)a.code_row | (unsigned long long)a.code_expert;
    a.code_align = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    a.scales = params->ptr;
    a.param = s->param;
    a.run_scales = 1;
    a.be = 1;
    a.bn = a.bk = make_fastdiv(1);
    a.scale_row = a.scale_col = a.scale_expert = 0;
    if (s->level == QK_LEVEL_TENSOR) {
        long long have = 1;
        for (int d = 0; d < params->rank; ++d) have *= params->shape[d];
        return have == 1 ? QK_OK : QK_ERR_SHAPE;
    }
    if (s->block_rank > r) return QK_ERR_BLOCK_SIZE;
    long long blk[3] = {1, 1, 1};  // experts, rows, columns
    for (int i = 0; i < s->block_rank; ++i) blk[3 - s->block_rank + i] = s->block[i];
    if (blk[2] % nq != 0) return QK_ERR_BLOCK_SIZE;
    if (blk[2] % 8 != 0 && blk[2] < k) return QK_ERR_BLOCK_SIZE;  // the kernels take the scale of 8 neighbouring codes at once
    if (params->rank != r) return QK_ERR_SHAPE;
    const long long dims[3] = {e, n, k};
    long long strides[3] = {0, 0, 0};
    for (int d = 3 - r; d < 3; ++d) {
        const long long want = (dims[d] + blk[d] - 1) / blk[d];
        if (params->shape[d - (3 - r)] != want) return QK_ERR_SHAPE;
        if (want > 1) strides[d] = params->strides[d - (3 - r)];
        if (strides[d] < 0) return QK_ERR_LAYOUT;
    }
    a.be = (unsigned)blk[0];
    a.bn = make_fastdiv((unsigned)blk[1]);
    a.bk = make_fastdiv((unsigned)blk[2]);
    a.scale_expert = strides[0];
    a.scale_row = strides[1];
    a.scale_col = strides[2];
    a.run_scales = blk[2] % 32 == 0 || blk[2] >= k ? 1 : blk[2] % 16 == 0 ? 2 : 4;
    return QK_OK;
}

static int check_common(const QkScheme *s, int activation, int dtype)
{
    if (dtype != QK_F16 && dtype != QK_BF16) return QK_ERR_DTYPE;
    const int rc = check_scheme(s);
    if (rc != QK_OK) return rc;
    return activation >= QK_ACT_IDENTITY && activation <= QK_ACT_SILU ? QK_OK : QK_ERR_UNSUPPORTED_SCHEME;
}

static int check_offsets(const QkTensor *t, int experts, const void **ptr, int *is64)
{
    if (!t) return QK_ERR_NULL;
    if (t->elem_size != 4 && t->elem_size != 8) return QK_ERR_DTYPE;
    const int rc = check_tensor(t, t->elem_size);
    if (rc != QK_OK) return rc;
    if (t->rank != 1 || t->shape[0] != experts + 1) return QK_ERR_SHAPE;
    if (t->strides[0] != 1) return QK_ERR_LAYOUT;
    *ptr = t->ptr;
    *is64 = t->elem_size == 8;
    return QK_OK;
}

static size_t round256(size_t v) { return (v + 255) & ~(size_t)255; }

// Rows of 16-bit elements that start on `bytes`.
static bool rows_on(int bytes, const void *p, long long stride) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * 2 % bytes == 0; }

// Rows of x that do not start on 16 bytes are copied to ones that do (bulk tensor loads need it).
static size_t copied_rows_bytes(long long rows, long long cols) { return round256((size_t)rows * ((cols + 7) / 8 * 8) * 2); }

static int copy_rows(const Matrix &x, int dtype, void *to, long long stride, cudaStream_t stream)
{
    ActBackwardArgs b = {};
    b.grad = x.ptr;
    b.grad_stride = x.stride;
    b.dz = to;
    b.dz_stride = stride;
    b.slices = bias_slices(x.rows, x.cols, 1);
    b.n = (int)x.cols;
    b.rows = (int)x.rows;
    b.experts = 1;
    int launches = 0;
    const cudaError_t e = launch_activation_backward(dtype, b, current_cfg(), stream, &launches);
    count_launch(launches);
    return cuda_status(e);
}

static int run_product(int dtype, const QkScheme *s, bool backward, LinearArgs &a, cudaStream_t stream)
{
    const auto all_on = [&](int bytes) {
        return rows_on(bytes, a.out, a.out_stride) && (!a.residual || rows_on(bytes, a.residual, a.residual_stride)) &&
               (!a.pre || rows_on(bytes, a.pre, a.pre_stride));
    };
    a.pairs = a.feats % 2 == 0 && all_on(4);
    a.wide = all_on(32) ? 32 : all_on(16) ? 16 : 0;
    a.error_flag = stage_error_flag();
    count_launch();
    return cuda_status(launch_linear_product(dtype, kind_of(s), backward, a, current_cfg(), stream));
}

static int linear_forward(const QkTensor *input, const QkTensor *offsets, bool grouped, const QkTensor *values, const QkTensor *params,
                          const QkScheme *scheme, const QkTensor *bias, const QkTensor *residual, int activation, const QkTensor *output,
                          const QkTensor *pre, int dtype, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (!input || !values || !params || !scheme || !output) return QK_ERR_NULL;
    int rc = check_common(scheme, activation, dtype);
    if (rc != QK_OK) return rc;
    LinearArgs a = {};
    if ((rc = fill_weight(a, values, params, scheme, grouped)) != QK_OK) return rc;
    Matrix x, y, r, z;
    if ((rc = as_matrix(input, dtype, x)) != QK_OK) return rc;
    if (x.cols != a.k) return QK_ERR_SHAPE;
    if ((rc = same_matrix(output, dtype, x.rows, a.n, y)) != QK_OK) return rc;
    if (residual && (rc = same_matrix(residual, dtype, x.rows, a.n, r)) != QK_OK) return rc;
    if (pre && (rc = same_matrix(pre, dtype, x.rows, a.n, z)) != QK_OK) return rc;
    if (bias && (rc = check_bias(bias, dtype, grouped, a.experts, a.n, false, &a.bias_stride, &a.bias_expert)) != QK_OK) return rc;
    if (grouped && (rc = check_offsets(offsets, a.experts, &a.offsets, &a.offsets64)) != QK_OK) return rc;
    if (x.rows == 0 || a.n == 0) return QK_OK;
    a.rows = (int)x.rows;
    a.contraction = a.k;
    a.feats = a.n;
    if (!product_tiles_fit(false, a)) return QK_ERR_TOO_LARGE;
    a.x = x.ptr;
    a.x_stride = x.stride;
    if (a.k > 0 && product_needs_aligned_rows(x.rows, x.ptr, x.stride)) {
        if (!workspace || workspace_bytes < copied_rows_bytes(x.rows, x.cols)) return QK_ERR_WORKSPACE;
        if (reinterpret_cast<uintptr_t>(workspace) % 16) return QK_ERR_ALIGN;
        a.x = workspace;
        a.x_stride = (x.cols + 7) / 8 * 8;
        if ((rc = copy_rows(x, dtype, workspace, a.x_stride, stream)) != QK_OK) return rc;
    }
    a.out = y.ptr;
    a.out_stride = y.stride;
    a.bias = bias ? bias->ptr : nullptr;
    a.residual = r.ptr;
    a.residual_stride = r.stride;
    a.pre = z.ptr;
    a.pre_stride = z.stride;
    a.act = activation;
    return run_product(dtype, scheme, false, a, stream);
}

// Workspace of the backward pass: [dz, rows padded to 16 bytes] [partial bias sums], each from a 256-byte boundary.
struct BackwardPlan {
    bool dz;            // the product reads dz from the workspace
    long long dz_stride;
    size_t partial_at, bytes;
    int slices;
};

// `operand_aligned`: what the product would read otherwise, grad_pre or grad_output, can be loaded as it lies.
static BackwardPlan plan_backward(long long rows, long long n, int experts, int activation, bool grad_bias, bool grad_pre, bool operand_aligned)
{
    BackwardPlan p;
    p.dz = (activation != QK_ACT_IDENTITY && !grad_pre) || !operand_aligned;
    p.dz_stride = (n + 7) / 8 * 8;
    size_t at = p.dz ? round256((size_t)rows * p.dz_stride * 2) : 0;
    p.partial_at = at;
    p.slices = bias_slices(rows, n > 0 ? n : 1, experts);
    if (grad_bias && p.slices > 1) at += round256((size_t)experts * p.slices * n * 4);
    p.bytes = at;
    return p;
}

static int linear_backward(const QkTensor *grad_output, const QkTensor *offsets, bool grouped, const QkTensor *values, const QkTensor *params,
                           const QkScheme *scheme, int activation, const QkTensor *pre, const QkTensor *grad_input, const QkTensor *grad_bias,
                           const QkTensor *grad_pre, int dtype, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (!grad_output || !values || !params || !scheme) return QK_ERR_NULL;
    int rc = check_common(scheme, activation, dtype);
    if (rc != QK_OK) return rc;
    if (activation != QK_ACT_IDENTITY && !pre) return QK_ERR_NULL;
    LinearArgs a = {};
    if ((rc = fill_weight(a, values, params, scheme, grouped)) != QK_OK) return rc;
    Matrix g, z, dx, dz;
    if ((rc = as_matrix(grad_output, dtype, g)) != QK_OK) return rc;
    if (g.cols != a.n) return QK_ERR_SHAPE;
    if (pre && (rc = same_matrix(pre, dtype, g.rows, a.n, z)) != QK_OK) return rc;
    if (grad_input && (rc = same_matrix(grad_input, dtype, g.rows, a.k, dx)) != QK_OK) return rc;
    if (grad_pre && (rc = same_matrix(grad_pre, dtype, g.rows, a.n, dz)) != QK_OK) return rc;
    ActBackwardArgs b = {};
    if (grad_bias && (rc = check_bias(grad_bias, dtype, grouped, a.experts, a.n, true, &b.grad_bias_stride, &b.grad_bias_expert)) != QK_OK)
        return rc;
    if (grouped && (rc = check_offsets(offsets, a.experts, &a.offsets, &a.offsets64)) != QK_OK) return rc;
    const Matrix &operand = activation != QK_ACT_IDENTITY && grad_pre ? dz : g;
    const BackwardPlan plan = plan_backward(g.rows, a.n, a.experts, activation, grad_bias != nullptr, grad_pre != nullptr,
                                            !product_needs_aligned_rows(operand.rows, operand.ptr, operand.stride));
    const bool product = grad_input && g.rows > 0 && a.k > 0;
    a.rows = (int)g.rows;
    a.contraction = a.n;
    a.feats = a.k;
    if (product && !product_tiles_fit(true, a)) return QK_ERR_TOO_LARGE;
    const bool needs = plan.bytes > 0 && ((plan.dz && product) || (grad_bias && plan.slices > 1));   // nothing where there are no features
    if (needs && (!workspace || workspace_bytes < plan.bytes)) return QK_ERR_WORKSPACE;
    if (needs && reinterpret_cast<uintptr_t>(workspace) % 16) return QK_ERR_ALIGN;

    const bool staged = plan.dz && product;
    if ((staged || grad_pre || grad_bias) && a.n > 0 && (g.rows > 0 || grad_bias)) {
        b.grad = g.ptr;
        b.grad_stride = g.stride;
        b.pre = z.ptr;
        b.pre_stride = z.stride;
        b.dz = staged ? workspace : nullptr;
        b.dz_stride = plan.dz_stride;
        b.dz2 = dz.ptr;
        b.dz2_stride = dz.stride;
        b.grad_bias = grad_bias ? grad_bias->ptr : nullptr;
        b.partial = grad_bias && plan.slices > 1 ? reinterpret_cast<float *>(static_cast<char *>(workspace) + plan.partial_at) : nullptr;
        b.slices = plan.slices;
        b.n = a.n;
        b.rows = (int)g.rows;
        b.act = activation;
        b.experts = a.experts;
        b.offsets = a.offsets;
        b.offsets64 = a.offsets64;
        const auto vec = [](const void *p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; };
        b.vec = a.n % 8 == 0 && vec(b.grad, b.grad_stride) && (activation == QK_ACT_IDENTITY || vec(b.pre, b.pre_stride)) &&
                (!b.dz2 || vec(b.dz2, b.dz2_stride));
        int launches = 0;
        const cudaError_t e = launch_activation_backward(dtype, b, current_cfg(), stream, &launches);
        count_launch(launches);
        if (e != cudaSuccess) return cuda_status(e);
    }
    if (!product) return QK_OK;
    a.x = staged ? workspace : operand.ptr;
    a.x_stride = staged ? plan.dz_stride : operand.stride;
    a.out = dx.ptr;
    a.out_stride = dx.stride;
    a.act = QK_ACT_IDENTITY;
    return run_product(dtype, scheme, true, a, stream);
}

}  // namespace qk

extern "C" {

int qk_linear(const QkTensor *input, const QkTensor *values, const QkTensor *params, const QkScheme *scheme, const QkTensor *bias,
              const QkTensor *residual, int activation, const QkTensor *output, const QkTensor *pre, int dtype, void *workspace,
              size_t workspace_bytes, void *stream)
{
    return qk::linear_forward(input, nullptr, false, values, params, scheme, bias, residual, activation, output, pre, dtype, workspace,
                              workspace_bytes, static_cast<cudaStream_t>(stream));
}

int qk_grouped_linear(const QkTensor *input, const QkTensor *offsets, const QkTensor *values, const QkTensor *params, const QkScheme *scheme,
                      const QkTensor *bias, const QkTensor *residual, int activation, const QkTensor *output, const QkTensor *pre, int dtype,
                      void *workspace, size_t workspace_bytes, void *stream)
{
    return qk::linear_forward(input, offsets, true, values, params, scheme, bias, residual, activation, output, pre, dtype, workspace,
                              workspace_bytes, static_cast<cudaStream_t>(stream));
}

int qk_linear_backward(const QkTensor *grad_output, const QkTensor *values, const QkTensor *params, const QkScheme *scheme, int activation,
                       const QkTensor *pre, const QkTensor *grad_input, const QkTensor *grad_bias, const QkTensor *grad_pre, int dtype,
                       void *workspace, size_t workspace_bytes, void *stream)
{
    return qk::linear_backward(grad_output, nullptr, false, values, params, scheme, activation, pre, grad_input, grad_bias, grad_pre, dtype,
                               workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int qk_grouped_linear_backward(const QkTensor *grad_output, const QkTensor *offsets, const QkTensor *values, const QkTensor *params,
                               const QkScheme *scheme, int activation, const QkTensor *pre, const QkTensor *grad_input,
                               const QkTensor *grad_bias, const QkTensor *grad_pre, int dtype, void *workspace, size_t workspace_bytes,
                               void *stream)
{
    return qk::linear_backward(grad_output, offsets, true, values, params, scheme, activation, pre, grad_input, grad_bias, grad_pre, dtype,
                               workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

size_t qk_linear_workspace_bytes(const QkTensor *input, const QkTensor *values, const QkScheme *scheme, int dtype)
{
    if (!input || !values || !scheme) return 0;
    qk::Matrix x;
    if ((dtype != QK_F16 && dtype != QK_BF16) || qk::as_matrix(input, dtype, x) != QK_OK || x.rows == 0 || x.cols == 0) return 0;
    return qk::product_needs_aligned_rows(x.rows, x.ptr, x.stride) ? qk::copied_rows_bytes(x.rows, x.cols) : 0;
}

size_t qk_linear_backward_workspace_bytes(const QkTensor *grad_output, const QkTensor *values, const QkScheme *scheme, int activation,
                                          int has_grad_bias, const QkTensor *grad_pre, int dtype)
{
    if (!grad_output || !values || !scheme || !values->shape || values->rank < 2 || values->rank > 3) return 0;
    qk::Matrix g, z;
    if ((dtype != QK_F16 && dtype != QK_BF16) || qk::as_matrix(grad_output, dtype, g) != QK_OK) return 0;
    if (grad_pre && qk::as_matrix(grad_pre, dtype, z) != QK_OK) return 0;
    const long long experts = values->rank == 3 ? values->shape[0] : 1;
    if (experts < 1 || experts > QK_LINEAR_MAX_EXPERTS) return 0;
    const qk::Matrix &operand = activation != QK_ACT_IDENTITY && grad_pre ? z : g;
    return qk::plan_backward(g.rows, g.cols, (int)experts, activation, has_grad_bias != 0, grad_pre != nullptr,
                             !qk::product_needs_aligned_rows(operand.rows, operand.ptr, operand.stride)).bytes;
}

}  // extern "C"
