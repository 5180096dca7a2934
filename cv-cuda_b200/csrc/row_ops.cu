// Host side of the row operators (LayerNorm, embedding lookup): argument validation, kernel selection and launch, and the
// translation unit of their device code.
#include "embedding_kernels.cuh"
#include "host_common.h"
#include "layernorm_kernels.cuh"

#include <algorithm>
#include <atomic>
#include <cstdlib>

using namespace b200pp;

namespace {

constexpr int kSms = 148;

size_t align_up(size_t v)
{
    return (v + 255) & ~static_cast<size_t>(255);
}

int row_elem_size(int dtype)
{
    switch (dtype)
    {
    case B200PP_U8:
        return 1;
    case B200PP_F16:
    case B200PP_BF16:
        return 2;
    case B200PP_F32:
    case B200PP_S32:
        return 4;
    case B200PP_S64:
        return 8;
    }
    return 0;
}

bool is_float(int dtype)
{
    return dtype == B200PP_F16 || dtype == B200PP_BF16 || dtype == B200PP_F32;
}

// Checks a set of rows (its element type is checked by the caller) and works out the kernels' view of it.
int take_rows(const B200ppRows *t, const char *what, bool written, RowMap &m, long long &rows)
{
    const long long limit = 0x7fffffffLL, elem = row_elem_size(t->dtype);
    if (t->cols < 1 || t->cols > limit)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "%s must have 1 to 2^31 - 1 columns", what);
    bool empty = false;
    for (int k = 0; k < 3; ++k)
    {
        if (t->count[k] < 0)
            return fail(B200PP_ERROR_INVALID_ARGUMENT, "%s has a negative number of rows", what);
        empty |= t->count[k] == 0;
    }
    rows = empty ? 0 : 1;
    for (int k = 0; k < 3 && !empty; ++k)
    {
        if (t->count[k] > limit || rows * t->count[k] > limit)
            return fail(B200PP_ERROR_OVERFLOW, "%s has more than 2^31 - 1 rows", what);
        rows *= t->count[k];
    }
    m = RowMap{};
    if (rows == 0)
        return B200PP_SUCCESS;
    if (!t->base)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "%s must be cuda-accessible, pitch-linear memory", what);
    // the dimensions that are left when single ones are dropped and those that continue one another are merged
    long long count[3], stride[3];
    int       n = 0;
    for (int k = 0; k < 3; ++k)
    {
        if (t->count[k] == 1)
            continue;
        if (n > 0 && stride[n - 1] == t->count[k] * t->stride[k])
        {
            count[n - 1] *= t->count[k];
            stride[n - 1] = t->stride[k];
            continue;
        }
        count[n]  = t->count[k];
        stride[n] = t->stride[k];
        ++n;
    }
    long long bits = static_cast<long long>(reinterpret_cast<uintptr_t>(t->base));
    for (int k = 0; k < n; ++k) bits |= stride[k];
    if (bits & (elem - 1))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "%s is not aligned to its element size", what);
    if (written)
    {
        // from the smallest stride up, each step must clear what the smaller ones span
        long long span = t->cols * elem;
        bool      done[3] = {false, false, false};
        for (int k = 0; k < n; ++k)
        {
            int low = -1;
            for (int j = 0; j < n; ++j)
                if (!done[j] && (low < 0 || std::llabs(stride[j]) < std::llabs(stride[low])))
                    low = j;
            done[low] = true;
            if (std::llabs(stride[low]) < span)
                return fail(B200PP_ERROR_INVALID_ARGUMENT, "%s has rows that overlap", what);
            span += std::llabs(stride[low]) * (count[low] - 1);
        }
    }
    m.base = static_cast<uint8_t *>(t->base);
    m.s2   = n > 0 ? stride[n - 1] : 0;
    if (n > 1)
    {
        m.n2 = static_cast<unsigned>(count[n - 1]);
        m.s1 = stride[n - 2];
        m.n1 = static_cast<unsigned>(count[n - 2]);
        m.s0 = n > 2 ? stride[0] : 0;
    }
    return B200PP_SUCCESS;
}

int check_param(const void *ptr, int dtype, const char *what)
{
    if (!ptr)
        return B200PP_SUCCESS;
    if (!is_float(dtype))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType of the %s", what);
    if (reinterpret_cast<uintptr_t>(ptr) & (row_elem_size(dtype) - 1))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "The %s is not aligned to its element size", what);
    return B200PP_SUCCESS;
}

int check_workspace(const void *workspace, size_t have, size_t need)
{
    if (need == 0)
        return B200PP_SUCCESS;
    if (!workspace || have < need)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "The workspace must have %zu bytes", need);
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "The workspace must start on a 16-byte boundary");
    return B200PP_SUCCESS;
}

} // namespace

// ================================================================================================ LayerNorm

extern "C" int b200ppLayerNormWorkspace(const B200ppRows *src, size_t *bytes)
{
    if (!src || !bytes)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    *bytes = 0;
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
    size_t need = 0;
    b200ppLayerNormWorkspace(src, &need);
    if ((st = check_workspace(workspace, workspaceBytes, need)))
        return st;
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
    const dim3 grid(std::min(p.rows, 65535u)), block(256);
    switch (src->dtype)
    {
    case B200PP_U8:
        layernorm_row_kernel<B200PP_U8><<<grid, block, 0, stream>>>(p);
        break;
    case B200PP_F16:
        layernorm_row_kernel<B200PP_F16><<<grid, block, 0, stream>>>(p);
        break;
    case B200PP_BF16:
        layernorm_row_kernel<B200PP_BF16><<<grid, block, 0, stream>>>(p);
        break;
    default:
        layernorm_row_kernel<B200PP_F32><<<grid, block, 0, stream>>>(p);
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

// ================================================================================================ embedding lookup

namespace {

int check_indices(const B200ppRows *indices)
{
    if (indices->dtype != B200PP_U8 && indices->dtype != B200PP_S32 && indices->dtype != B200PP_S64)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Indices must be uint8, int32 or int64");
    if (indices->cols != 1)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Indices must have one column");
    return B200PP_SUCCESS;
}

} // namespace

extern "C" int b200ppEmbedding(const B200ppRows *indices, const B200ppRows *table, const B200ppRows *dst, float scale,
                               cudaStream_t stream)
{
    if (!indices || !table || !dst)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    if (!is_float(table->dtype) || !is_float(dst->dtype))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType");
    if (table->cols != dst->cols)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Table and output have different numbers of columns");
    EmbeddingKParams p{};
    long long        count = 0, dstRows = 0, rows = 0;
    int              st;
    if ((st = check_indices(indices)) || (st = take_rows(indices, "Indices", false, p.indices, count))
        || (st = take_rows(table, "Table", false, p.table, rows)) || (st = take_rows(dst, "Output", true, p.dst, dstRows)))
        return st;
    if (count != dstRows)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Indices and output have different numbers of rows");
    if (count == 0)
        return B200PP_SUCCESS;
    p.indexType = indices->dtype;
    p.tableType = table->dtype;
    p.dstType   = dst->dtype;
    p.count     = static_cast<unsigned>(count);
    p.rows      = static_cast<int>(rows);
    p.cols      = static_cast<int>(dst->cols);
    p.scale     = scale;
    embedding_kernel<<<std::min((p.count + 7u) / 8u, 65535u), 256, 0, stream>>>(p);
    return check_launch("Embedding");
}

namespace {

// Layout of the gradient's workspace.
struct EmbeddingGradPlan
{
    unsigned unit, units;
    size_t   keys[2], order[2], partials, bytes;
};

EmbeddingGradPlan plan_embedding_grad(long long count, long long cols)
{
    EmbeddingGradPlan w{};
    w.unit       = 32;
    w.units      = static_cast<unsigned>((count + w.unit - 1) / w.unit);
    size_t at    = 0;
    const size_t list = align_up(static_cast<size_t>(count) * sizeof(unsigned));
    for (int k = 0; k < 2; ++k)
    {
        w.keys[k] = at;
        at += list;
        w.order[k] = at;
        at += list;
    }
    w.partials = at;
    w.bytes    = at + static_cast<size_t>(w.units) * 2 * cols * sizeof(float);
    return w;
}

// Raises a kernel's dynamic shared-memory limit, once per device.
template<typename K>
int raise_smem(K kernel, int bytes, std::atomic<unsigned long long> &done)
{
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit))
        return B200PP_SUCCESS;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess)
    {
        cudaGetLastError();
        return fail(B200PP_ERROR_INTERNAL, "Cannot raise a kernel's shared memory to %d bytes: %s", bytes, cudaGetErrorString(e));
    }
    done.fetch_or(bit);
    return B200PP_SUCCESS;
}

} // namespace

extern "C" int b200ppEmbeddingBackwardWorkspace(const B200ppRows *grad, size_t *bytes)
{
    if (!grad || !bytes)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    RowMap     m;
    long long  count = 0;
    B200ppRows t     = *grad;
    t.base           = reinterpret_cast<void *>(uintptr_t(256));
    if (int st = take_rows(&t, "Gradient", false, m, count))
        return st;
    *bytes = count > 0 ? plan_embedding_grad(count, t.cols).bytes : 0;
    return B200PP_SUCCESS;
}

extern "C" int b200ppEmbeddingBackward(const B200ppRows *grad, const B200ppRows *indices, const B200ppRows *dtable,
                                       const B200ppEmbeddingGradOp *op, void *workspace, size_t workspaceBytes,
                                       cudaStream_t stream)
{
    if (!grad || !indices || !dtable || !op)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    if (!is_float(grad->dtype) || !is_float(dtable->dtype))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType");
    if (grad->cols != dtable->cols)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Gradient and table have different numbers of columns");
    EmbeddingGradKParams p{};
    long long            count = 0, gradRows = 0, rows = 0;
    int                  st;
    if ((st = check_indices(indices)) || (st = take_rows(indices, "Indices", false, p.indices, count))
        || (st = take_rows(grad, "Gradient", false, p.grad, gradRows)) || (st = take_rows(dtable, "Table gradient", true, p.dtable, rows)))
        return st;
    if (count != gradRows)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Indices and gradient have different numbers of rows");
    if (rows == 0)
        return B200PP_SUCCESS;
    const EmbeddingGradPlan w = plan_embedding_grad(count, grad->cols);
    if (count > 0 && (st = check_workspace(workspace, workspaceBytes, w.bytes)))
        return st;
    uint8_t *ws  = static_cast<uint8_t *>(workspace);
    p.gradType   = grad->dtype;
    p.indexType  = indices->dtype;
    p.dtableType = dtable->dtype;
    p.count      = static_cast<unsigned>(count);
    p.rows       = static_cast<int>(rows);
    p.cols       = static_cast<int>(grad->cols);
    p.scale      = op->scale;
    p.accumulate = op->accumulate != 0;
    p.padding    = op->paddingIndex >= 0 && op->paddingIndex < rows ? static_cast<int>(op->paddingIndex) : -1;
    p.unit       = w.unit;
    if (!p.accumulate)
    {
        embedding_zero_kernel<<<std::min(static_cast<unsigned>(rows), 65535u), 256, 0, stream>>>(p);
        if ((st = check_launch("EmbeddingBackward")))
            return st;
    }
    if (count == 0)
        return B200PP_SUCCESS;
    for (int k = 0; k < 2; ++k)
    {
        p.keys[k]  = reinterpret_cast<unsigned *>(ws + w.keys[k]);
        p.order[k] = reinterpret_cast<unsigned *>(ws + w.order[k]);
    }
    p.partials = reinterpret_cast<float *>(ws + w.partials);
    int bits = 1; // of the largest key, `rows`
    while (bits < 31 && (rows >> bits) != 0) ++bits;
    p.passes    = (bits + kSortMaxBits - 1) / kSortMaxBits;
    p.digitBits = (bits + p.passes - 1) / p.passes;
    const int bins = 1 << p.digitBits;
    static std::atomic<unsigned long long> raised{0};
    if ((st = raise_smem(embedding_sort_kernel, static_cast<int>(sort_smem_words(1 << kSortMaxBits) * sizeof(unsigned)), raised)))
        return st;
    embedding_sort_kernel<<<kSortCtas, kSortThreads, sort_smem_words(bins) * sizeof(unsigned), stream>>>(p);
    if ((st = check_launch("EmbeddingBackward")))
        return st;
    const unsigned           blocks = (p.cols + 255u) / 256u;
    const unsigned long long jobs   = static_cast<unsigned long long>(w.units) * blocks;
    if ((jobs + 7) / 8 > 0x7fffffffull || blocks > 65535u)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Gradient is too large");
    embedding_grad_runs_kernel<<<static_cast<unsigned>((jobs + 7) / 8), 256, 0, stream>>>(p);
    if ((st = check_launch("EmbeddingBackward")))
        return st;
    if (w.units > 1)
    {
        embedding_grad_join_kernel<<<dim3(w.units - 1, blocks), 256, 0, stream>>>(p);
        st = check_launch("EmbeddingBackward");
    }
    return st;
}
