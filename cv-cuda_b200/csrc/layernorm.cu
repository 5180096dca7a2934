// Host side of LayerNorm and its gradient: argument validation, kernel selection and launch.
#include "layernorm_kernels.cuh"
#include "row_host.h"

#include <algorithm>

using namespace b200pp;

namespace {

// Rows longer than this are split into chunks.
constexpr long long kLongRow = 32768;

long long layernorm_chunks(long long cols)
{
    return cols > kLongRow ? (cols + kChunk - 1) / kChunk : 0;
}

template<int SRC, int W>
void launch_layernorm(const LayerNormKParams &p, cudaStream_t stream)
{
    const int cols = p.cols;
    if (p.chunks)
    {
        layernorm_chunk_stats_kernel<SRC, W><<<p.rows * p.chunks, kChunkThreads, 0, stream>>>(p);
        layernorm_chunk_apply_kernel<SRC, W><<<p.rows * p.chunks, kChunkThreads, 0, stream>>>(p);
        return;
    }
    if (cols > 1024 || (cols > 256 && p.rows <= static_cast<unsigned>(kSms)))
    {
        // A CTA per row: sixteen values per thread, thirty-two where that would take more than 512 threads; eight for so few rows
        // that the GPU is not full anyway.
        auto threads = [cols](int e) { return dim3((cols + 32 * e - 1) / (32 * e) * 32); };
        if (cols <= 4096 && p.rows <= static_cast<unsigned>(kSms))
            layernorm_kernel<SRC, 8, W, true><<<p.rows, threads(8), 0, stream>>>(p);
        else if (cols <= 8192)
            layernorm_kernel<SRC, 16, W, true><<<p.rows, threads(16), 0, stream>>>(p);
        else
            layernorm_kernel<SRC, 32, W, true><<<p.rows, threads(32), 0, stream>>>(p);
        return;
    }
    int lanes = 4;
    while (lanes < 32 && lanes * 8 < cols) lanes *= 2;
    const dim3     block(lanes, 256 / lanes);
    const unsigned grid = (p.rows + block.y - 1) / block.y;
    if (cols <= 256)
        layernorm_kernel<SRC, 8, W, false><<<grid, block, 0, stream>>>(p);
    else if (cols <= 512)
        layernorm_kernel<SRC, 16, W, false><<<grid, block, 0, stream>>>(p);
    else if (cols <= 768)
        layernorm_kernel<SRC, 24, W, false><<<grid, block, 0, stream>>>(p);
    else
        layernorm_kernel<SRC, 32, W, false><<<grid, block, 0, stream>>>(p);
}

template<int SRC>
void launch_layernorm(const LayerNormKParams &p, int width, cudaStream_t stream)
{
    if (width == 8)
        launch_layernorm<SRC, 8>(p, stream);
    else if (width == 4)
        launch_layernorm<SRC, 4>(p, stream);
    else if (width == 2)
        launch_layernorm<SRC, 2>(p, stream);
    else
        launch_layernorm<SRC, 1>(p, stream);
}

} // namespace

extern "C" int b200ppLayerNormWorkspace(const B200ppRows *src, size_t *bytes)
{
    if (!src || !bytes)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    RowMap     m;
    long long  rows = 0;
    B200ppRows t    = *src;
    t.base          = reinterpret_cast<void *>(uintptr_t(256));
    if (int st = take_rows(&t, "Input", false, m, rows))
        return st;
    *bytes = static_cast<size_t>(rows) * layernorm_chunks(t.cols) * sizeof(float2);
    return B200PP_SUCCESS;
}

extern "C" int b200ppLayerNorm(const B200ppRows *src, const B200ppRows *dst, const B200ppLayerNormOp *op, void *workspace,
                               size_t workspaceBytes, cudaStream_t stream)
{
    if (!src || !dst || !op)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    if ((!is_float(src->dtype) && src->dtype != B200PP_U8) || !is_float(dst->dtype))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType");
    if (src->cols != dst->cols)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Input and output shapes are different");
    if (!(op->epsilon >= 0.0f))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "epsilon must not be negative");
    LayerNormKParams p{};
    long long        rows = 0, dstRows = 0;
    int              st;
    if ((st = take_rows(src, "Input", false, p.src, rows)) || (st = take_rows(dst, "Output", true, p.dst, dstRows))
        || (st = check_param(op->weight, op->weightType, "weight")) || (st = check_param(op->bias, op->biasType, "bias"))
        || (st = check_param(op->mean, B200PP_F32, "mean")) || (st = check_param(op->rstd, B200PP_F32, "rstd")))
        return st;
    if (rows != dstRows)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Input and output shapes are different");
    const long long chunks = layernorm_chunks(src->cols);
    if ((st = check_workspace(workspace, workspaceBytes, static_cast<size_t>(rows) * chunks * sizeof(float2))))
        return st;
    if (rows * chunks > 0x7fffffffLL)
        return fail(B200PP_ERROR_OVERFLOW, "Input is too large");
    if (rows == 0)
        return B200PP_SUCCESS;
    p.rows       = static_cast<unsigned>(rows);
    p.cols       = static_cast<int>(src->cols);
    p.dstType    = dst->dtype;
    p.weight     = static_cast<const uint8_t *>(op->weight);
    p.bias       = static_cast<const uint8_t *>(op->bias);
    p.weightType = op->weightType;
    p.biasType   = op->biasType;
    p.epsilon    = op->epsilon;
    p.fcols      = static_cast<float>(p.cols);
    p.mean       = op->mean;
    p.rstd       = op->rstd;
    p.chunks     = static_cast<unsigned>(chunks);
    p.partials   = static_cast<float2 *>(workspace);
    VecWidth width(p.cols);
    width.take(p.src, row_elem_size(src->dtype));
    width.take(p.dst, row_elem_size(dst->dtype));
    width.take(p.weight, 0, row_elem_size(p.weightType));
    width.take(p.bias, 0, row_elem_size(p.biasType));
    switch (src->dtype)
    {
    case B200PP_U8:
        launch_layernorm<B200PP_U8>(p, width.width, stream);
        break;
    case B200PP_F16:
        launch_layernorm<B200PP_F16>(p, width.width, stream);
        break;
    case B200PP_BF16:
        launch_layernorm<B200PP_BF16>(p, width.width, stream);
        break;
    default:
        launch_layernorm<B200PP_F32>(p, width.width, stream);
        break;
    }
    return check_launch("LayerNorm");
}

// Parts the rows are divided into for the sums over the rows.
static int layernorm_grad_parts(long long rows, long long cols)
{
    const long long blocks = (cols + 31) / 32;
    return static_cast<int>(std::max(1LL, std::min({(rows + 31) / 32, (kSms * 8 + blocks - 1) / blocks, 65535LL})));
}

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
    *bytes = static_cast<size_t>(layernorm_grad_parts(rows, t.cols)) * 2 * t.cols * sizeof(float);
    return B200PP_SUCCESS;
}

namespace {

template<int SRC>
void launch_layernorm_grad(const LayerNormGradKParams &p, cudaStream_t stream, int &status)
{
    // the sums over the rows first: dsrc may be written over grad or src
    if (p.dweight || p.dbias)
    {
        const dim3 grid((p.cols + 31u) / 32u, p.parts);
        layernorm_grad_columns_kernel<SRC><<<grid, 256, 0, stream>>>(p);
        if ((status = check_launch("LayerNormBackward")))
            return;
        layernorm_grad_join_kernel<<<(p.cols + 255u) / 256u, 256, 0, stream>>>(p);
        if ((status = check_launch("LayerNormBackward")))
            return;
    }
    if (p.dsrc.base)
    {
        layernorm_grad_row_kernel<SRC><<<std::min(p.rows, 65535u), 256, 0, stream>>>(p);
        status = check_launch("LayerNormBackward");
    }
}

} // namespace

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
    p.parts = layernorm_grad_parts(rows, p.cols);
    if (op->dweight || op->dbias)
        if ((st = check_workspace(workspace, workspaceBytes, static_cast<size_t>(p.parts) * 2 * p.cols * sizeof(float))))
            return st;
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
    p.dweight     = static_cast<uint8_t *>(op->dweight);
    p.dbias       = static_cast<uint8_t *>(op->dbias);
    p.partials    = static_cast<float *>(workspace);
    if (rows == 0)
        p.dsrc.base = nullptr;
    int status = B200PP_SUCCESS;
    switch (src->dtype)
    {
    case B200PP_U8:
        launch_layernorm_grad<B200PP_U8>(p, stream, status);
        break;
    case B200PP_F16:
        launch_layernorm_grad<B200PP_F16>(p, stream, status);
        break;
    case B200PP_BF16:
        launch_layernorm_grad<B200PP_BF16>(p, stream, status);
        break;
    default:
        launch_layernorm_grad<B200PP_F32>(p, stream, status);
        break;
    }
    return status;
}

