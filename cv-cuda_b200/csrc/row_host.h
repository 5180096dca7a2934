// Host helpers of the row operators: argument validation and the choice of vector widths.
#ifndef CVCUDA_B200_ROW_HOST_H
#define CVCUDA_B200_ROW_HOST_H

#include "host_common.h"
#include "row_math.cuh"

#include <algorithm>
#include <atomic>
#include <cstdlib>

namespace b200pp {

constexpr int kSms = 148;

inline size_t align_up(size_t v)
{
    return (v + 255) & ~static_cast<size_t>(255);
}

inline int row_elem_size(int dtype)
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

inline bool is_float(int dtype)
{
    return dtype == B200PP_F16 || dtype == B200PP_BF16 || dtype == B200PP_F32;
}

// Checks a set of rows (its element type is checked by the caller) and works out the kernels' view of it.
inline int take_rows(const B200ppRows *t, const char *what, bool written, RowMap &m, long long &rows)
{
    // columns: room for the vectors behind the last one, whose numbers kernels compute before they leave them out
    const long long limit = 0x7fffffffLL, widest = limit - 0xffff, elem = row_elem_size(t->dtype);
    if (t->cols < 1 || t->cols > widest)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "%s must have 1 to 2^31 - 2^16 columns", what);
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

inline int check_param(const void *ptr, int dtype, const char *what)
{
    if (!ptr)
        return B200PP_SUCCESS;
    if (!is_float(dtype))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "Invalid DataType of the %s", what);
    if (reinterpret_cast<uintptr_t>(ptr) & (row_elem_size(dtype) - 1))
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "The %s is not aligned to its element size", what);
    return B200PP_SUCCESS;
}

inline int check_workspace(const void *workspace, size_t have, size_t need)
{
    if (need == 0)
        return B200PP_SUCCESS;
    if (!workspace || have < need)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "The workspace must have %zu bytes", need);
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return fail(B200PP_ERROR_INVALID_ARGUMENT, "The workspace must start on a 16-byte boundary");
    return B200PP_SUCCESS;
}

// Largest number of elements (8, 4, 2, 1) that can be moved as one vector: it divides the row, and every row of every tensor starts
// on its boundary.
struct VecWidth
{
    int width = 8;

    explicit VecWidth(long long cols)
    {
        while (cols % width) width >>= 1;
    }

    void take(const void *base, long long strides, int elem)
    {
        if (!base)
            return;
        const long long bits = static_cast<long long>(reinterpret_cast<uintptr_t>(base)) | strides;
        while (width > 1 && (bits & (static_cast<long long>(width) * elem - 1))) width >>= 1;
    }

    void take(const RowMap &m, int elem)
    {
        take(m.base, m.s0 | m.s1 | m.s2, elem);
    }
};

// Rows that start anywhere, in vectors of W all the same: how many elements after the boundary of a vector row 0 starts, and how many
// more each row does, modulo W -- if that is the same in all tensors.
struct RowShift
{
    int  width, start = 0, step = 0;
    bool valid = true, first = true;

    explicit RowShift(int w)
        : width(w)
    {
    }

    void take(const RowMap &m, int elem, long long rows)
    {
        if (!m.base)
            return;
        const int a = static_cast<int>(reinterpret_cast<uintptr_t>(m.base) / elem % width);
        const int s = rows > 1 ? static_cast<int>((m.s2 / elem % width + width) % width) : first ? 0 : step;
        if (m.n2 != 0 || (rows > 1 && m.s2 % elem != 0) || (!first && (a != start || s != step)))
            valid = false;
        start = a;
        step  = s;
        first = false;
    }
};

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

// A launch in clusters of `ctas` CTAs (1: none), and/or -- `early` -- one that may begin while the kernel before it on the stream
// is still running, as soon as all CTAs of that one have allowed it: the kernel waits for it itself, before it touches what that one
// writes.
struct Launch
{
    cudaLaunchConfig_t  cfg{};
    cudaLaunchAttribute attrs[2]{};

    Launch(dim3 grid, dim3 block, int smem, cudaStream_t stream, int ctas, bool early)
    {
        cfg.gridDim          = grid;
        cfg.blockDim         = block;
        cfg.dynamicSmemBytes = smem;
        cfg.stream           = stream;
        cfg.attrs            = attrs;
        if (ctas > 1)
        {
            cudaLaunchAttribute &a = attrs[cfg.numAttrs++];
            a.id                   = cudaLaunchAttributeClusterDimension;
            a.val.clusterDim       = {static_cast<unsigned>(ctas), 1, 1};
        }
        if (early)
        {
            cudaLaunchAttribute &a                       = attrs[cfg.numAttrs++];
            a.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
            a.val.programmaticStreamSerializationAllowed = 1;
        }
    }

    Launch(const Launch &) = delete;

    template<typename... P, typename... A>
    void run(void (*kernel)(P...), A... args) // check_launch reports a failure
    {
        cudaLaunchKernelEx(&cfg, kernel, args...);
    }
};

} // namespace b200pp

#endif
