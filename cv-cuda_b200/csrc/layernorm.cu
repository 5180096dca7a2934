// Host side of LayerNorm: argument validation, kernel selection and launch.
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
    p.invCols    = 1.0f / p.fcols;
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
