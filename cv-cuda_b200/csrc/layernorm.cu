// Host side of LayerNorm: argument validation, kernel selection and launch.
#include "layernorm_kernels.cuh"
#include "row_host.h"

#include <algorithm>

using namespace b200pp;

namespace {

// How rows of up to 1024 columns are dealt out: `lanes` lanes of a warp with `values` values each, as few lanes as leave little idle.
// What a row costs besides its values -- shuffles, addresses -- is per lane (468750 rows of 64 bfloat16: 24 us with four lanes of
// sixteen values, 31 us with eight of eight).
struct WarpPlan
{
    int lanes, values;
};

WarpPlan plan_warp(int cols)
{
    static const int table[][3] = {{8, 1, 8},    {16, 2, 8},    {32, 4, 8},    {64, 4, 16},   {96, 4, 24},   {128, 8, 16},
                                   {192, 8, 24}, {256, 16, 16}, {384, 16, 24}, {512, 32, 16}, {768, 32, 24}, {1024, 32, 32}};
    int              i = 0;
    while (cols > table[i][0]) ++i;
    return {table[i][1], table[i][2]};
}

int chunk_of(long long cols)
{
    return cols % 8 ? kChunk - 8 : kChunk;
}

// Chunks of a row; 0 for those the other kernels take (no workspace up to 8192 columns, row_ops.h).
long long layernorm_chunks(long long cols)
{
    return cols > kBlockCols ? (cols + chunk_of(cols) - 1) / chunk_of(cols) : 0;
}

template<int SRC, int E, int W, bool RAGGED, bool FULL>
int launch_warp(const LayerNormKParams &p, const WarpPlan &plan, cudaStream_t stream)
{
    static std::atomic<unsigned long long> raised{0};
    const dim3                             block(plan.lanes, 256 / plan.lanes);
    const int                              ring = RowStage<SRC, E, W>::bytes(block.x, block.y) * kWarpStages;
    if (ring > 32 * 1024) // a launch gets 48 KB unasked, static memory included
        if (int st = raise_smem(layernorm_warp_kernel<SRC, E, W, FULL, RAGGED>, 112 * 1024, raised))
            return st;
    const unsigned turns = (p.rows + block.y - 1) / block.y;
    layernorm_warp_kernel<SRC, E, W, FULL, RAGGED><<<std::min(turns, static_cast<unsigned>(kSms * kWarpCtas<E>)), block, ring, stream>>>(p);
    return B200PP_SUCCESS;
}

// RAGGED: with room for rows that start anywhere in a vector.
template<int SRC, int W, bool RAGGED>
int launch_staged(const LayerNormKParams &p, cudaStream_t stream)
{
    const int cols = p.cols + (RAGGED ? W - 1 : 0);
    if (cols > 1024)
    {
        static std::atomic<unsigned long long> raised{0};
        const int                              threads = (cols + 511) / 512 * 32;
        const int                              ring    = RowStage<SRC, 16, W>::bytes(threads, 1) * 3;
        if (ring > 32 * 1024)
            if (int st = raise_smem(layernorm_block_kernel<SRC, W, RAGGED>, 112 * 1024, raised))
                return st;
        unsigned ctas = kSms * (kBlockResident / threads);
        if (RAGGED)
            ctas -= ctas % 8; // the rows of a CTA start alike
        layernorm_block_kernel<SRC, W, RAGGED><<<std::min(p.rows, ctas), threads, ring, stream>>>(p);
        return B200PP_SUCCESS;
    }
    const WarpPlan plan = plan_warp(cols);
    if (plan.values == 8)
        return launch_warp<SRC, 8, W, RAGGED, false>(p, plan, stream);
    if (plan.values == 32)
        return launch_warp<SRC, 32, W, RAGGED, true>(p, plan, stream);
    if (plan.lanes == 32)
        return plan.values == 16 ? launch_warp<SRC, 16, W, RAGGED, true>(p, plan, stream) : launch_warp<SRC, 24, W, RAGGED, true>(p, plan, stream);
    return plan.values == 16 ? launch_warp<SRC, 16, W, RAGGED, false>(p, plan, stream) : launch_warp<SRC, 24, W, RAGGED, false>(p, plan, stream);
}

template<int SRC, int W, bool RAGGED>
int launch_chunks(const LayerNormKParams &p, cudaStream_t stream)
{
    layernorm_chunk_stats_kernel<SRC, W, RAGGED><<<p.rows * p.chunks, kChunkThreads, 0, stream>>>(p);
    Launch(dim3(p.rows * p.chunks), dim3(kChunkThreads), 0, stream, 1, true).run(layernorm_chunk_apply_kernel<SRC, W, RAGGED>, p);
    return B200PP_SUCCESS;
}

template<int SRC, int W>
bool launch_direct(const LayerNormKParams &p, cudaStream_t stream)
{
    if (p.chunks)
    {
        launch_chunks<SRC, W, false>(p, stream);
        return true;
    }
    if (p.cols > 256 && p.cols <= 4096 && p.rows <= static_cast<unsigned>(kSms))
    {
        layernorm_few_kernel<SRC, W><<<p.rows, (p.cols + 255) / 256 * 32, 0, stream>>>(p);
        return true;
    }
    return false;
}

template<int SRC>
int launch_layernorm(LayerNormKParams &p, int width, cudaStream_t stream)
{
    // rows that are no whole vectors of four, but start alike in both tensors
    constexpr int kWide = SRC == B200PP_F32 ? 4 : 8; // of the staged kernels, as below
    const int     wide  = p.chunks ? 8 : kWide;
    RowShift      shift(wide);
    shift.take(p.src, kElemBytes<SRC>, p.rows);
    shift.take(p.dst, row_elem_size(p.dstType), p.rows);
    if (width < 4 && shift.valid)
    {
        p.shift0 = shift.start;
        p.shift  = shift.step;
        if (p.chunks)
        {
            // float32 rows with weights, read eight values apart: 150 of 77777 49 us, value by value 38
            if (p.chunk < kChunk && (SRC != B200PP_F32 || (!p.weight && !p.bias)))
                return launch_chunks<SRC, 8, true>(p, stream);
        }
        // below four vectors per row, the first and the last one cost more than the pairs do
        else if (p.cols >= 4 * wide && !(p.cols > 256 && p.cols <= 4096 && p.rows <= static_cast<unsigned>(kSms)))
            return launch_staged<SRC, kWide, true>(p, stream);
    }
    if (width == 8 ? launch_direct<SRC, 8>(p, stream)
                   : width == 4 ? launch_direct<SRC, 4>(p, stream) : width == 2 ? launch_direct<SRC, 2>(p, stream) : launch_direct<SRC, 1>(p, stream))
        return B200PP_SUCCESS;
    // vectors of 16 bytes at most on the way through shared memory; of four elements at least, otherwise the rows' lines as they are
    if constexpr (SRC != B200PP_F32)
        if (width == 8)
            return launch_staged<SRC, 8, false>(p, stream);
    if (width >= 4)
        return launch_staged<SRC, 4, false>(p, stream);
    return launch_staged<SRC, 0, false>(p, stream);
}

} // namespace

extern "C" int b200ppLayerNormWorkspace(const B200ppRows *src, size_t *bytes)
{
    if (!src || !bytes)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    if (!is_float(src->dtype) && src->dtype != B200PP_U8)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType");
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
    p.chunk      = chunk_of(p.cols);
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
