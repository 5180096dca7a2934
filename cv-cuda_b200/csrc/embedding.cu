// Host side of the embedding lookup and its gradient: argument validation, kernel selection and launch.
#include "embedding_grad_direct.cuh"
#include "embedding_kernels.cuh"
#include "row_host.h"

#include <algorithm>

using namespace b200pp;

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

namespace {

template<int C, int R>
void launch_short_rows(const EmbeddingKParams &p, cudaStream_t stream)
{
    const unsigned  tiles = (p.count + 256u * R - 1) / (256u * R);
    const int       lines = 8 * 32 * C * static_cast<int>(sizeof(uint4));
    const long long table = (static_cast<long long>(p.rows) + 1) * kShortStride<C, R> * (16 / R);
    // the copy to shared memory pays from the second index per table row on
    if (table <= kShortTable && p.count >= 2u * p.rows)
        embedding_short_rows_kernel<C, R, true><<<std::min(tiles, kSms * 8u), 256, lines + static_cast<int>(table), stream>>>(p);
    else
        embedding_short_rows_kernel<C, R, false><<<tiles, 256, lines, stream>>>(p);
}

template<int C>
void launch_short_rows(const EmbeddingKParams &p, cudaStream_t stream)
{
    if (p.dstType == B200PP_F32)
        launch_short_rows<C, 4>(p, stream);
    else
        launch_short_rows<C, 8>(p, stream);
}

template<int TABLE, int W, int U>
int launch_embedding(EmbeddingKParams &p, int lanes, cudaStream_t stream)
{
    constexpr int R = kLookupVectors<W> / U;
    p.blocks        = static_cast<unsigned>((static_cast<long long>(p.cols) + lanes * W * U - 1) / (lanes * W * U));
    const dim3               block(lanes, 256 / lanes);
    const unsigned long long ctas = (static_cast<unsigned long long>(p.count) + R * block.y - 1) / (R * block.y) * p.blocks;
    if (ctas > 0x7fffffffull)
        return fail(B200PP_ERROR_OVERFLOW, "Output is too large");
    if (p.dstType == TABLE)
        embedding_kernel<TABLE, TABLE, W, U><<<static_cast<unsigned>(ctas), block, 0, stream>>>(p);
    else
        embedding_kernel<TABLE, -1, W, U><<<static_cast<unsigned>(ctas), block, 0, stream>>>(p);
    return check_launch("Embedding");
}

template<int TABLE, int W>
int launch_embedding(EmbeddingKParams &p, cudaStream_t stream)
{
    // lanes per row: a warp, fewer for rows that would leave half of it idle; as many vectors per lane as the row has
    int lanes = 32;
    while (lanes > 1 && (lanes / 2) * W >= p.cols) lanes /= 2;
    const int vectors = (p.cols + lanes * W - 1) / (lanes * W);
    // so few rows that the GPU is not full: one vector per lane, and as many lanes as there are
    if (vectors == 1 || static_cast<long long>(p.count) * vectors <= kSms * 8)
        return launch_embedding<TABLE, W, 1>(p, lanes, stream);
    if (vectors == 2)
        return launch_embedding<TABLE, W, 2>(p, lanes, stream);
    if constexpr (kLookupVectors<W> == 8)
    {
        // the vectors of a lane's share of the row, rounded up to 4, 6 or 8 (30 million floats in rows of 644: 25.4 us with six, 27.2 with
        // eight, 29.0 with four; of 161: 44.9, 47.0 and 53.0; of 333, two blocks of six or three of four: 43.6, 46.1 and 40.6)
        const int each = (vectors + (vectors + 7) / 8 - 1) / ((vectors + 7) / 8);
        if (each > 4)
            return each > 6 ? launch_embedding<TABLE, W, 8>(p, lanes, stream) : launch_embedding<TABLE, W, 6>(p, lanes, stream);
    }
    return launch_embedding<TABLE, W, 4>(p, lanes, stream);
}

template<int TABLE>
int launch_embedding(EmbeddingKParams &p, int width, cudaStream_t stream)
{
    if (width == 8)
        return launch_embedding<TABLE, 8>(p, stream);
    if (width == 4)
        return launch_embedding<TABLE, 4>(p, stream);
    if (width == 2)
        return launch_embedding<TABLE, 2>(p, stream);
    return launch_embedding<TABLE, 1>(p, stream);
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
    const int elem = row_elem_size(dst->dtype);
    if (p.cols < 8 && p.dst.n2 == 0 && (count == 1 || p.dst.s2 == static_cast<long long>(p.cols) * elem)
        && (reinterpret_cast<uintptr_t>(p.dst.base) & 15) == 0)
    {
        switch (p.cols)
        {
        case 1:
            launch_short_rows<1>(p, stream);
            break;
        case 2:
            launch_short_rows<2>(p, stream);
            break;
        case 3:
            launch_short_rows<3>(p, stream);
            break;
        case 4:
            launch_short_rows<4>(p, stream);
            break;
        case 5:
            launch_short_rows<5>(p, stream);
            break;
        case 6:
            launch_short_rows<6>(p, stream);
            break;
        default:
            launch_short_rows<7>(p, stream);
            break;
        }
        return check_launch("Embedding");
    }
    VecWidth width(p.cols);
    width.take(p.table, row_elem_size(table->dtype));
    width.take(p.dst, elem);
    if (table->dtype == B200PP_F16)
        return launch_embedding<B200PP_F16>(p, width.width, stream);
    if (table->dtype == B200PP_BF16)
        return launch_embedding<B200PP_BF16>(p, width.width, stream);
    return launch_embedding<B200PP_F32>(p, width.width, stream);
}

namespace {

// Layout of the gradient's workspace.
struct EmbeddingGradPlan
{
    unsigned units, groups;
    size_t   entries[2], partials, bytes;
};

EmbeddingGradPlan plan_embedding_grad(long long count, long long cols)
{
    EmbeddingGradPlan w{};
    w.units      = static_cast<unsigned>((count + kGradUnit - 1) / kGradUnit);
    w.groups     = static_cast<unsigned>((count + kShortRun - 1) / kShortRun);
    size_t at    = 0;
    for (int k = 0; k < 2; ++k)
    {
        w.entries[k] = at;
        at += align_up(static_cast<size_t>(count) * sizeof(uint2));
    }
    w.partials = at;
    w.bytes    = at + static_cast<size_t>(w.groups) * 2 * cols * sizeof(float);
    return w;
}

// The workspace query and the call refuse the same sizes, before anything is launched. The largest grid is that of the runs, eight jobs
// per CTA; for vectors that a lane has four values of, blocks of columns are smallest.
int check_grad_size(const EmbeddingGradPlan &w, long long cols)
{
    const unsigned long long jobs = (static_cast<unsigned long long>(w.units) + 2 * w.groups) * ((cols + kGradCols<1> - 1) / kGradCols<1>);
    if ((jobs + 7) / 8 > 0x7fffffffull)
        return fail(B200PP_ERROR_OVERFLOW, "Gradient is too large");
    return B200PP_SUCCESS;
}

template<int GRAD, int W>
int launch_runs(EmbeddingGradKParams &p, cudaStream_t stream)
{
    p.blocks                      = static_cast<unsigned>((static_cast<long long>(p.cols) + kGradCols<W> - 1) / kGradCols<W>);
    const unsigned long long jobs = (static_cast<unsigned long long>(p.units) + 2 * p.groups) * p.blocks;
    Launch(dim3(static_cast<unsigned>((jobs + 7) / 8)), dim3(256), 0, stream, 1, true).run(embedding_grad_runs_kernel<GRAD, W>, p);
    return check_launch("EmbeddingBackward");
}

template<int GRAD>
int launch_runs(EmbeddingGradKParams &p, int width, cudaStream_t stream)
{
    if (width == 8)
        return launch_runs<GRAD, 8>(p, stream);
    if (width == 4)
        return launch_runs<GRAD, 4>(p, stream);
    if (width == 2)
        return launch_runs<GRAD, 2>(p, stream);
    return launch_runs<GRAD, 1>(p, stream);
}

// The sums of the runs of the sorted positions, and the join of the long ones.
int launch_sums(EmbeddingGradKParams &p, cudaStream_t stream)
{
    VecWidth width(p.cols);
    width.take(p.grad, row_elem_size(p.gradType));
    width.take(p.dtable, row_elem_size(p.dtableType));
    width.take(p.partials, p.cols * static_cast<long long>(sizeof(float)), sizeof(float));
    int st;
    if (p.gradType == B200PP_F16)
        st = launch_runs<B200PP_F16>(p, width.width, stream);
    else if (p.gradType == B200PP_BF16)
        st = launch_runs<B200PP_BF16>(p, width.width, stream);
    else
        st = launch_runs<B200PP_F32>(p, width.width, stream);
    if (st || p.groups == 1)
        return st;
    const dim3 grid((p.groups - 1 + 7) / 8, (p.cols + kJoinCols - 1) / kJoinCols);
    Launch(grid, dim3(256), 0, stream, 1, true).run(embedding_grad_join_kernel, p);
    return check_launch("EmbeddingBackward");
}

// CTAs of the cluster that sorts: one for few indices, then eight; sixteen, where the GPU has room for such a cluster, once the
// indices take longer than the exchange between the CTAs (16384 indices: 18 us with eight, 14 us with sixteen; 5003: 10.3 us both).
int sort_ctas(long long count, size_t smem)
{
    if (count <= 2048)
        return 1;
    if (count <= 8192)
        return 8;
    static std::atomic<unsigned long long> wide{0}, asked{0};
    int                                    dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(asked.load() & bit))
    {
        int clusters = 0;
        if (cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess)
        {
            Launch launch(dim3(16), dim3(kSortThreads), static_cast<int>(smem), nullptr, 16, false);
            if (cudaOccupancyMaxActiveClusters(&clusters, embedding_sort_kernel, &launch.cfg) == cudaSuccess && clusters > 0)
                wide.fetch_or(bit);
        }
        cudaGetLastError();
        asked.fetch_or(bit);
    }
    return wide.load() & bit ? 16 : 8;
}

// Few indices: one kernel whose CTAs each read all of them. Tables of so many CTAs' columns and rows that the reading would take longer
// than sorting are left to the others.
bool goes_direct(long long count, long long rows, long long cols)
{
    return count <= kDirectCount && (cols + 31) / 32 * ((rows + kDirectRows - 1) / kDirectRows) <= 4096;
}

} // namespace

extern "C" int b200ppEmbeddingBackwardWorkspace(const B200ppRows *grad, const B200ppRows *dtable, size_t *bytes)
{
    if (!grad || !dtable || !bytes)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Null argument");
    if (!is_float(grad->dtype) || !is_float(dtable->dtype))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType");
    if (grad->cols != dtable->cols)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Gradient and table have different numbers of columns");
    RowMap     m;
    long long  count = 0, rows = 0;
    B200ppRows g = *grad, t = *dtable;
    g.base = t.base = reinterpret_cast<void *>(uintptr_t(256));
    int st;
    if ((st = take_rows(&g, "Gradient", false, m, count)) || (st = take_rows(&t, "Table gradient", true, m, rows)))
        return st;
    *bytes = 0;
    if (count == 0 || goes_direct(count, rows, g.cols))
        return B200PP_SUCCESS;
    const EmbeddingGradPlan w = plan_embedding_grad(count, g.cols);
    if ((st = check_grad_size(w, g.cols)))
        return st;
    *bytes = w.bytes;
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
    if (count == 0 && op->accumulate)
        return B200PP_SUCCESS;
    const int padding = op->paddingIndex >= 0 && op->paddingIndex < rows ? static_cast<int>(op->paddingIndex) : -1;
    if (goes_direct(count, rows, grad->cols))
    {
        EmbeddingDirectKParams d{};
        d.grad       = p.grad;
        d.indices    = p.indices;
        d.dtable     = p.dtable;
        d.gradType   = grad->dtype;
        d.indexType  = indices->dtype;
        d.dtableType = dtable->dtype;
        d.count      = static_cast<unsigned>(count);
        d.rows       = static_cast<int>(rows);
        d.cols       = static_cast<int>(grad->cols);
        d.scale      = op->scale;
        d.accumulate = op->accumulate != 0;
        VecWidth width(d.cols);
        width.take(d.grad, row_elem_size(d.gradType));
        width.take(d.dtable, row_elem_size(d.dtableType));
        return embedding_grad_direct(d, width.width, padding, stream);
    }
    const EmbeddingGradPlan w = plan_embedding_grad(count, grad->cols);
    if (count > 0 && ((st = check_grad_size(w, grad->cols)) || (st = check_workspace(workspace, workspaceBytes, w.bytes))))
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
    p.padding    = padding;
    p.units      = w.units;
    p.groups     = w.groups;
    for (int k = 0; k < 2; ++k) p.entries[k] = reinterpret_cast<uint2 *>(ws + w.entries[k]);
    p.partials = reinterpret_cast<float *>(ws + w.partials);
    int bits = 1; // of the largest key, `rows`
    while (bits < 31 && (rows >> bits) != 0) ++bits;
    p.passes    = (bits + kSortMaxBits - 1) / kSortMaxBits;
    p.digitBits = (bits + p.passes - 1) / p.passes;
    static std::atomic<unsigned long long> raised{0};
    const size_t                           most = sort_smem_words(kSortThreads / 32, 1 << kSortMaxBits) * sizeof(unsigned);
    if ((st = raise_smem(embedding_sort_kernel, static_cast<int>(most), raised)))
        return st;
    if (count > 0)
    {
        // as few warps as hold the indices kSortKeys at a time: each has a table of counts
        const int ctas = sort_ctas(count, most);
        p.sortWarps    = 4;
        while (p.sortWarps < kSortThreads / 32 && static_cast<long long>(p.sortWarps) * 32 * kSortKeys * ctas < count) p.sortWarps *= 2;
        const long long warps = static_cast<long long>(ctas) * p.sortWarps;
        p.span                = static_cast<unsigned>(((count + warps - 1) / warps + 31) / 32 * 32);
        const size_t smem     = sort_smem_words(p.sortWarps, 1 << p.digitBits) * sizeof(unsigned);
        Launch(dim3(ctas), dim3(kSortThreads), static_cast<int>(smem), stream, ctas, false).run(embedding_sort_kernel, p);
        if ((st = check_launch("EmbeddingBackward")))
            return st;
    }
    if (!p.accumulate)
    {
        VecWidth width(p.cols);
        width.take(p.dtable, row_elem_size(p.dtableType));
        p.zeroWidth         = width.width;
        const unsigned ctas = static_cast<unsigned>(std::min<long long>((rows + kZeroThreads / 32 - 1) / (kZeroThreads / 32), kSms * 8));
        Launch(dim3(ctas), dim3(kZeroThreads), 0, stream, 1, count > 0).run(embedding_clear_kernel, p);
        if ((st = check_launch("EmbeddingBackward")))
            return st;
    }
    if (count == 0)
        return st;
    // as many columns at a time as the join's grid has blocks for (blocks in another dimension, or a first column, cost the join 1 us of
    // the 52 for 16384 indices of 32000 x 1024)
    constexpr int kMostCols = 65535 * kJoinCols;
    const int     gradElem = row_elem_size(p.gradType), tableElem = row_elem_size(p.dtableType);
    for (int left = p.cols; left > 0 && !st; left -= p.cols)
    {
        p.cols = std::min(left, kMostCols);
        st     = launch_sums(p, stream);
        p.grad.base += static_cast<long long>(p.cols) * gradElem;
        p.dtable.base += static_cast<long long>(p.cols) * tableElem;
    }
    return st;
}
