// Host side of LayerNorm's gradient: argument validation, kernel selection and launch.
#include "layernorm_grad_kernels.cuh"
#include "row_host.h"

#include <algorithm>

using namespace b200pp;

namespace {

// How the rows are dealt out. One-pass kernel: `threads` per row with `values` values each, `groups` rows per CTA, one part per CTA;
// for longer rows (values = 0) the sums over the rows are a kernel of their own.
struct GradPlan
{
    int threads, groups, values, parts;
};

GradPlan plan_layernorm_grad(long long rows, long long cols)
{
    GradPlan g{};
    if (cols <= 8192)
    {
        // a warp per row, or part of one, up to 768 columns; above, whole warps with sixteen values per thread
        if (cols <= 768)
        {
            g.values = cols <= 256 ? 8 : cols <= 512 ? 16 : 24;
            for (g.threads = 4; g.threads < 32 && g.threads * 8 < cols;) g.threads *= 2;
        }
        else
        {
            g.values  = 16;
            g.threads = static_cast<int>((cols + 511) / 512 * 32);
        }
        g.groups              = std::max(1, 256 / g.threads);
        const long long turns = (rows + g.groups - 1) / g.groups;
        const int       ctas  = kSms * std::max(1, kGradResident / (g.threads * g.groups));
        g.parts               = static_cast<int>(std::max(1LL, std::min<long long>(turns, ctas)));
        return g;
    }
    const long long blocks = (cols + 31) / 32;
    g.parts = static_cast<int>(std::max(1LL, std::min({(rows + 31) / 32, (kSms * 8 + blocks - 1) / blocks, 65535LL})));
    return g;
}

size_t grad_workspace(const GradPlan &g, long long cols)
{
    return static_cast<size_t>(g.parts) * 2 * cols * sizeof(float);
}

template<int SRC, int GRAD, int E, int W, bool BLOCK>
int launch_one_pass(const LayerNormGradKParams &p, const GradPlan &g, cudaStream_t stream)
{
    typedef GradRing<SRC, GRAD, E, W>      Ring;
    static std::atomic<unsigned long long> raised{0};
    const int                              threads = g.threads * g.groups;
    const int ring = Ring::kThread * Ring::kStages * threads, sums = p.partials ? 2 * p.cols * static_cast<int>(sizeof(float)) : 0;
    const int smem = std::max(ring, sums);
    if (smem > 32 * 1024) // a launch gets 48 KB unasked, static memory included
        if (int st = raise_smem(layernorm_grad_kernel<SRC, GRAD, E, W, BLOCK>,
                                std::max(Ring::kThread * Ring::kStages * kGradResident, 2 * 8192 * static_cast<int>(sizeof(float))), raised))
            return st;
    layernorm_grad_kernel<SRC, GRAD, E, W, BLOCK><<<p.parts, dim3(g.threads, g.groups), smem, stream>>>(p);
    return check_launch("LayerNormBackward");
}

template<int SRC, int GRAD, int W>
int launch_one_pass(const LayerNormGradKParams &p, const GradPlan &g, cudaStream_t stream)
{
    if (g.values == 8)
        return launch_one_pass<SRC, GRAD, 8, W, false>(p, g, stream);
    if (g.values == 24)
        return launch_one_pass<SRC, GRAD, 24, W, false>(p, g, stream);
    if (g.threads == 32)
        return launch_one_pass<SRC, GRAD, 16, W, false>(p, g, stream);
    return launch_one_pass<SRC, GRAD, 16, W, true>(p, g, stream);
}

template<int SRC, int GRAD>
int launch_one_pass(const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream)
{
    if (width == 8)
        return launch_one_pass<SRC, GRAD, 8>(p, g, stream);
    if (width == 4)
        return launch_one_pass<SRC, GRAD, 4>(p, g, stream);
    if (width == 2)
        return launch_one_pass<SRC, GRAD, 2>(p, g, stream);
    return launch_one_pass<SRC, GRAD, 1>(p, g, stream);
}

// The pairs of element types the one-pass kernel is built for: gradients of the source's type or float32, any for uint8.
// -1: not this pair, or rows too long.
int launch_one_pass(int srcType, const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream)
{
    if (g.values == 0)
        return -1;
    switch (srcType * 16 + p.gradType)
    {
#define B200PP_PAIR(S, G) \
    case S * 16 + G:      \
        return launch_one_pass<S, G>(p, g, width, stream);
        B200PP_PAIR(B200PP_U8, B200PP_F32)
        B200PP_PAIR(B200PP_U8, B200PP_F16)
        B200PP_PAIR(B200PP_U8, B200PP_BF16)
        B200PP_PAIR(B200PP_F16, B200PP_F16)
        B200PP_PAIR(B200PP_F16, B200PP_F32)
        B200PP_PAIR(B200PP_BF16, B200PP_BF16)
        B200PP_PAIR(B200PP_BF16, B200PP_F32)
        B200PP_PAIR(B200PP_F32, B200PP_F32)
#undef B200PP_PAIR
    }
    return -1;
}

template<int SRC>
int launch_two_pass(const LayerNormGradKParams &p, cudaStream_t stream)
{
    // the sums over the rows first: dsrc may be written over grad or src
    if (p.partials)
    {
        const dim3 grid((p.cols + 31u) / 32u, p.parts);
        layernorm_grad_columns_kernel<SRC><<<grid, 256, 0, stream>>>(p);
        if (int st = check_launch("LayerNormBackward"))
            return st;
    }
    if (p.dsrc.base)
    {
        layernorm_grad_row_kernel<SRC><<<std::min(p.rows, 65535u), 256, 0, stream>>>(p);
        return check_launch("LayerNormBackward");
    }
    return B200PP_SUCCESS;
}

} // namespace

extern "C" int b200ppLayerNormBackwardWorkspace(const B200ppRows *src, size_t *bytes)
{
    if (!src || !bytes)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    RowMap    m;
    long long rows = 0;
    B200ppRows t   = *src;
    t.base         = reinterpret_cast<void *>(uintptr_t(256));
    if (int st = take_rows(&t, "Input", false, m, rows))
        return st;
    *bytes = grad_workspace(plan_layernorm_grad(rows, t.cols), t.cols);
    return B200PP_SUCCESS;
}

extern "C" int b200ppLayerNormBackward(const B200ppRows *grad, const B200ppRows *src, const B200ppRows *dsrc,
                                       const B200ppLayerNormGradOp *op, void *workspace, size_t workspaceBytes,
                                       cudaStream_t stream)
{
    if (!grad || !src || !op)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    if (!dsrc && !op->dweight && !op->dbias)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "No gradient is asked for");
    if ((!is_float(src->dtype) && src->dtype != B200PP_U8) || !is_float(grad->dtype) || (dsrc && !is_float(dsrc->dtype)))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType");
    if (src->cols != grad->cols || (dsrc && src->cols != dsrc->cols))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Input and gradient shapes are different");
    LayerNormGradKParams p{};
    long long            rows = 0, gradRows = 0, dsrcRows = 0;
    int                  st;
    if ((st = take_rows(src, "Input", false, p.src, rows)) || (st = take_rows(grad, "Gradient", false, p.grad, gradRows))
        || (dsrc && (st = take_rows(dsrc, "Input gradient", true, p.dsrc, dsrcRows)))
        || (st = check_param(op->weight, op->weightType, "weight"))
        || (st = check_param(op->dweight, op->dweightType, "weight gradient"))
        || (st = check_param(op->dbias, op->dbiasType, "bias gradient")) || (st = check_param(op->mean, B200PP_F32, "mean"))
        || (st = check_param(op->rstd, B200PP_F32, "rstd")))
        return st;
    if (rows != gradRows || (dsrc && rows != dsrcRows))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Input and gradient shapes are different");
    if (rows > 0 && (!op->mean || !op->rstd))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "The backward pass needs the forward pass's mean and rstd");
    p.cols  = static_cast<int>(src->cols);
    const GradPlan plan = plan_layernorm_grad(rows, p.cols);
    p.parts             = plan.parts;
    if (op->dweight || op->dbias)
    {
        if ((st = check_workspace(workspace, workspaceBytes, grad_workspace(plan, p.cols))))
            return st;
        p.partials = static_cast<float *>(workspace);
    }
    p.rows        = static_cast<unsigned>(rows);
    p.gradType    = grad->dtype;
    p.dsrcType    = dsrc ? dsrc->dtype : 0;
    p.weightType  = op->weightType;
    p.dweightType = op->dweightType;
    p.dbiasType   = op->dbiasType;
    p.weight      = static_cast<const uint8_t *>(op->weight);
    p.mean        = op->mean;
    p.rstd        = op->rstd;
    p.fcols       = static_cast<float>(p.cols);
    p.invCols     = 1.0f / p.fcols;
    p.dweight     = static_cast<uint8_t *>(op->dweight);
    p.dbias       = static_cast<uint8_t *>(op->dbias);
    if (rows == 0)
        p.dsrc.base = nullptr;
    VecWidth width(p.cols);
    width.take(p.src, row_elem_size(src->dtype));
    width.take(p.grad, row_elem_size(p.gradType));
    width.take(p.dsrc, row_elem_size(p.dsrcType));
    width.take(p.weight, 0, row_elem_size(p.weightType));
    st = launch_one_pass(src->dtype, p, plan, width.width, stream);
    if (st >= 0)
        ; // done, or refused
    else if (src->dtype == B200PP_U8)
        st = launch_two_pass<B200PP_U8>(p, stream);
    else if (src->dtype == B200PP_F16)
        st = launch_two_pass<B200PP_F16>(p, stream);
    else if (src->dtype == B200PP_BF16)
        st = launch_two_pass<B200PP_BF16>(p, stream);
    else
        st = launch_two_pass<B200PP_F32>(p, stream);
    if (st || !p.partials)
        return st;
    layernorm_grad_join_kernel<<<(2u * p.cols + 31u) / 32u, dim3(32, 32), 0, stream>>>(p);
    return check_launch("LayerNormBackward");
}
