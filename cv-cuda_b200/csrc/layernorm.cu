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

template<int SRC, int E, int W>
int launch_warp(const LayerNormKParams &p, int lanes, cudaStream_t stream)
{
    constexpr int                          kRing = RowStage<SRC, W, E / W>::kThread * 256 * kWarpStages;
    static std::atomic<unsigned long long> raised{0};
    if (kRing > 32 * 1024) // a launch gets 48 KB unasked, static memory included
        if (int st = raise_smem(layernorm_warp_kernel<SRC, E, W>, kRing, raised))
            return st;
    const dim3     block(lanes, 256 / lanes);
    const unsigned turns = (p.rows + block.y - 1) / block.y;
    layernorm_warp_kernel<SRC, E, W><<<std::min(turns, static_cast<unsigned>(kSms * kWarpCtas<E>)), block, kRing, stream>>>(p);
    return B200PP_SUCCESS;
}

template<int SRC, int W>
int launch_layernorm(const LayerNormKParams &p, cudaStream_t stream)
{
    const int cols = p.cols;
    if (p.chunks)
    {
        layernorm_chunk_stats_kernel<SRC, W><<<p.rows * p.chunks, kChunkThreads, 0, stream>>>(p);
        layernorm_chunk_apply_kernel<SRC, W><<<p.rows * p.chunks, kChunkThreads, 0, stream>>>(p);
        return B200PP_SUCCESS;
    }
    if (cols > 1024 || (cols > 256 && p.rows <= static_cast<unsigned>(kSms)))
    {
        // A CTA per row: sixteen values per thread, thirty-two where that would take more than 512 threads; eight for so few rows
        // that the GPU is not full anyway.
        auto threads = [cols](int e) { return dim3((cols + 32 * e - 1) / (32 * e) * 32); };
        if (cols <= 4096 && p.rows <= static_cast<unsigned>(kSms))
            layernorm_block_kernel<SRC, 8, W><<<p.rows, threads(8), 0, stream>>>(p);
        else if (cols <= 8192)
            layernorm_block_kernel<SRC, 16, W><<<p.rows, threads(16), 0, stream>>>(p);
        else
            layernorm_block_kernel<SRC, 32, W><<<p.rows, threads(32), 0, stream>>>(p);
        return B200PP_SUCCESS;
    }
    int lanes = 4;
    while (lanes < 32 && lanes * 8 < cols) lanes *= 2;
    if (cols <= 256)
        return launch_warp<SRC, 8, W>(p, lanes, stream);
    if (cols <= 512)
        return launch_warp<SRC, 16, W>(p, lanes, stream);
    if (cols <= 768)
        return launch_warp<SRC, 24, W>(p, lanes, stream);
    return launch_warp<SRC, 32, W>(p, lanes, stream);
}

template<int SRC>
int launch_layernorm(const LayerNormKParams &p, int width, cudaStream_t stream)
{
    if (width == 8)
        return launch_layernorm<SRC, 8>(p, stream);
    if (width == 4)
        return launch_layernorm<SRC, 4>(p, stream);
    if (width == 2)
        return launch_layernorm<SRC, 2>(p, stream);
    return launch_layernorm<SRC, 1>(p, stream);
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
    if (src->dtype == B200PP_U8)
        st = launch_layernorm<B200PP_U8>(p, width.width, stream);
    else if (src->dtype == B200PP_F16)
        st = launch_layernorm<B200PP_F16>(p, width.width, stream);
    else if (src->dtype == B200PP_BF16)
        st = launch_layernorm<B200PP_BF16>(p, width.width, stream);
    else
        st = launch_layernorm<B200PP_F32>(p, width.width, stream);
    if (st)
        return st;
    return check_launch("LayerNorm");
}
