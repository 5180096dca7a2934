// Host side of LayerNorm's gradient: argument validation, kernel selection and launch.
#include "layernorm_grad_launch.cuh"

#include <algorithm>

using namespace b200pp;

namespace {

// The rows of the CTAs of a plan start like one another if row `step` rows on does, and so do those of a warp, which are `warps` apart.
bool rows_start_alike(const GradPlan &g, const RowShift &s)
{
    const bool warp = g.threads < 32;
    return s.valid && g.parts * g.groups * s.step % s.width == 0 && (!warp || g.threads * g.groups / 32 * s.step % s.width == 0);
}

// Rows that a thread adds up one after another where the data does not leave many parts anyway: a float32 sum loses a part of each
// addend that grows with their number (300000 rows of 65537: up to 37500 of them, 0.2 % of the sum).
constexpr long long kGradDepth = 1024;

GradPlan plan_layernorm_grad(long long rows, long long length, int elem)
{
    GradPlan g{};
    if (length <= 8 * 16 * kGradResident)
    {
        g.ctas = 1;
        // room for rows that start anywhere in a vector, unless that takes more CTAs
        while (g.ctas * 16 * kGradResident < length) g.ctas *= 2;
        const long long cols = length % 4 && length + 7 <= g.ctas * 16 * kGradResident ? length + 7 : length;
        if (cols <= 768)
        {
            // as few lanes per row as leave little idle
            static const int table[][3] = {{8, 1, 8},     {16, 2, 8},    {32, 4, 8},    {64, 4, 16},   {96, 4, 24},  {128, 8, 16},
                                           {192, 8, 24},  {256, 16, 16}, {384, 16, 24}, {512, 32, 16}, {768, 32, 24}};
            int              i = 0;
            while (cols > table[i][0]) ++i;
            g.threads = table[i][1];
            g.values  = table[i][2];
        }
        else
        {
            // sixteen values, or 24 where that lets two CTAs share an SM or leaves no more lanes idle (50030 rows of 2051 float16: 176 ->
            // 157 us; 30000 of 1536: 67 -> 60 us). With float32 rows shared memory is too small for two CTAs
            const long long part = (cols + g.ctas - 1) / g.ctas;
            const bool      pair = part > 16 * kGradResident / 2 && part <= 24 * kGradResident / 2;
            g.values             = elem < 4 && (pair || (part + 767) / 768 * 768 <= (part + 511) / 512 * 512) ? 24 : 16;
            g.threads            = static_cast<int>((part + 32 * g.values - 1) / (32 * g.values) * 32);
        }
        g.span = g.threads * g.values;
        // several rows per CTA as long as there are enough for all SMs; whole warps
        g.groups = std::max(1, 256 / g.threads);
        while (g.groups > 1 && g.groups * g.threads > 32 && rows < static_cast<long long>(g.groups) * kSms) g.groups /= 2;
        const long long turns = (rows + g.groups - 1) / g.groups;
        const int       most  = std::max(1, kSms * std::max(1, kGradResident / (g.threads * g.groups)) / g.ctas);
        g.parts               = static_cast<int>(std::max(1LL, std::min<long long>(turns, most)));
        // every eighth row of packed ones starts at the boundary of a vector: as many CTAs that each of them has rows that start alike,
        // unless it takes them another turn
        int apart = 8;
        while (apart > 1 && (length * g.groups * apart / 2) % 8 == 0) apart /= 2;
        const int more = (g.parts + apart - 1) / apart * apart, less = g.parts / apart * apart;
        if (cols != length && more <= most)
            g.parts = more;
        else if (cols != length && less > 0 && (turns + less - 1) / less <= (turns + g.parts - 1) / g.parts + turns / (16LL * g.parts))
            g.parts = less;
        // 37 clusters of four CTAs or eighteen of eight are resident: more of them where each would have too many rows
        if (g.ctas > 2)
            g.parts *= static_cast<int>(std::max(1LL, (turns + kGradDepth * g.parts - 1) / (kGradDepth * g.parts)));
        return g;
    }
    // there are columns enough for all SMs; a warp adds every eighth row of its part
    g.parts = static_cast<int>(std::max(1LL, std::min((rows + 8 * kGradDepth - 1) / (8 * kGradDepth), 65535LL)));
    return g;
}

bool are_few(long long rows, long long cols)
{
    return rows <= kFewRows && cols <= kFewCols;
}

size_t grad_workspace(const GradPlan &g, long long rows, long long cols)
{
    return are_few(rows, cols) ? 0 : static_cast<size_t>(g.parts) * 2 * cols * sizeof(float);
}

// -1: not these types, or rows too long.
int launch_one_pass(int srcType, const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream)
{
    if (g.values == 0)
        return -1;
    switch (srcType)
    {
    case B200PP_U8:
        return layernorm_grad_u8(p, g, width, stream);
    case B200PP_F16:
        return layernorm_grad_f16(p, g, width, stream);
    case B200PP_BF16:
        return layernorm_grad_bf16(p, g, width, stream);
    }
    return layernorm_grad_f32(p, g, width, stream);
}

template<int SRC>
int launch_few(const LayerNormGradKParams &p, cudaStream_t stream)
{
    const unsigned rows = p.dsrc.base ? p.rows : 0, columns = p.dweight || p.dbias ? (p.cols + 31u) / 32u : 0;
    // dsrc over grad or src: the sums over the rows first
    if (rows && columns && (p.dsrc.base == p.grad.base || p.dsrc.base == p.src.base))
    {
        layernorm_grad_few_kernel<SRC><<<columns, kFewThreads, 0, stream>>>(p, 0);
        if (int st = check_launch("LayerNormBackward"))
            return st;
        layernorm_grad_few_kernel<SRC><<<rows, kFewThreads, 0, stream>>>(p, rows);
    }
    else if (rows + columns > 0)
        layernorm_grad_few_kernel<SRC><<<rows + columns, kFewThreads, 0, stream>>>(p, rows);
    return check_launch("LayerNormBackward");
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
    if (!is_float(src->dtype) && src->dtype != B200PP_U8)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType");
    RowMap    m;
    long long rows = 0;
    B200ppRows t   = *src;
    t.base         = reinterpret_cast<void *>(uintptr_t(256));
    if (int st = take_rows(&t, "Input", false, m, rows))
        return st;
    *bytes = grad_workspace(plan_layernorm_grad(rows, t.cols, row_elem_size(t.dtype)), rows, t.cols);
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
    GradPlan plan = plan_layernorm_grad(rows, p.cols, row_elem_size(src->dtype));
    p.parts       = plan.parts;
    if (op->dweight || op->dbias)
    {
        if ((st = check_workspace(workspace, workspaceBytes, grad_workspace(plan, rows, p.cols))))
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
    if (are_few(rows, p.cols))
    {
        if (src->dtype == B200PP_U8)
            return launch_few<B200PP_U8>(p, stream);
        if (src->dtype == B200PP_F16)
            return launch_few<B200PP_F16>(p, stream);
        if (src->dtype == B200PP_BF16)
            return launch_few<B200PP_BF16>(p, stream);
        return launch_few<B200PP_F32>(p, stream);
    }
    VecWidth width(p.cols);
    width.take(p.src, row_elem_size(src->dtype));
    width.take(p.grad, row_elem_size(p.gradType));
    width.take(p.dsrc, row_elem_size(p.dsrcType));
    width.take(p.weight, 0, row_elem_size(p.weightType));
    const int wide = src->dtype == B200PP_F32 || p.gradType == B200PP_F32 ? 4 : 8;
    RowShift  shift(wide);
    shift.take(p.src, row_elem_size(src->dtype), rows);
    shift.take(p.grad, row_elem_size(p.gradType), rows);
    shift.take(p.dsrc, row_elem_size(p.dsrcType), rows);
    // below four vectors per row, the first and the last one cost more than the pairs do
    if (width.width < 4 && plan.values && p.cols >= 4 * wide && p.cols + wide - 1 <= plan.span * plan.ctas && rows_start_alike(plan, shift))
    {
        p.shift0     = shift.start;
        p.shift      = shift.step;
        p.ownWeights = shift.step != 0 && plan.groups > 1;
        // copies of the weights that leave no room for a second CTA are not worth it
        plan.ragged  = !(p.ownWeights && p.weight && wide == 4 && plan.values == 24);
        p.ownWeights = p.ownWeights && plan.ragged;
    }
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
    // as many threads share a column as there are parts for (50176 rows of 768 bfloat16, 296 parts: all in all 44 us with 32 threads, 50 with
    // eight, 107 with one; 600 of 40000 float16, 18 parts: 92, 85 and 91 us)
    const int  share = p.parts >= 64 ? 32 : p.parts >= 8 ? 8 : 1;
    const dim3 block(share == 1 ? 128 : 32, share);
    Launch(dim3((2u * p.cols + block.x - 1) / block.x), block, 0, stream, 1, true).run(layernorm_grad_join_kernel, p);
    return check_launch("LayerNormBackward");
}
