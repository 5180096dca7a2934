// Row addressing, element conversions and reductions shared by the row operators (LayerNorm, embedding lookup).
#ifndef CVCUDA_B200_ROW_MATH_CUH
#define CVCUDA_B200_ROW_MATH_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cvcuda_b200/row_ops.h>

#include <stdint.h>

namespace b200pp {

// Start of row r of a B200ppRows. The host merges dimensions that continue one another; what is left is one stride (the
// usual case: `n2` = 0) or up to three.
struct RowMap
{
    uint8_t  *base;
    long long s0, s1, s2; // bytes
    unsigned  n1, n2;

    __device__ __forceinline__ uint8_t *at(unsigned r) const
    {
        if (n2 == 0)
            return base + static_cast<long long>(r) * s2;
        const unsigned q = r / n2;
        return base + static_cast<long long>(r - q * n2) * s2 + static_cast<long long>(q % n1) * s1 + static_cast<long long>(q / n1) * s0;
    }
};

template<int DT>
struct Elem;
template<>
struct Elem<B200PP_U8>
{
    typedef uint8_t type;
    static __device__ __forceinline__ float up(uint8_t v)
    {
        return static_cast<float>(v);
    }
};
template<>
struct Elem<B200PP_F16>
{
    typedef __half type;
    static __device__ __forceinline__ float up(__half v)
    {
        return __half2float(v);
    }
    static __device__ __forceinline__ __half down(float v)
    {
        return __float2half_rn(v);
    }
};
template<>
struct Elem<B200PP_BF16>
{
    typedef __nv_bfloat16 type;
    static __device__ __forceinline__ float up(__nv_bfloat16 v)
    {
        return __bfloat162float(v);
    }
    static __device__ __forceinline__ __nv_bfloat16 down(float v)
    {
        return __float2bfloat16_rn(v);
    }
};
template<>
struct Elem<B200PP_F32>
{
    typedef float type;
    static __device__ __forceinline__ float up(float v)
    {
        return v;
    }
    static __device__ __forceinline__ float down(float v)
    {
        return v;
    }
};

template<int DT>
__device__ __forceinline__ float load_elem(const uint8_t *row, long long i)
{
    return Elem<DT>::up(reinterpret_cast<const typename Elem<DT>::type *>(row)[i]);
}

template<int DT>
__device__ __forceinline__ void store_elem_as(uint8_t *row, long long i, float v)
{
    reinterpret_cast<typename Elem<DT>::type *>(row)[i] = Elem<DT>::down(v);
}

// Element type chosen at run time (the same for the whole launch, so the branch is uniform).
__device__ __forceinline__ float load_elem(const uint8_t *row, long long i, int dtype)
{
    switch (dtype)
    {
    case B200PP_U8:
        return load_elem<B200PP_U8>(row, i);
    case B200PP_F16:
        return load_elem<B200PP_F16>(row, i);
    case B200PP_BF16:
        return load_elem<B200PP_BF16>(row, i);
    default:
        return load_elem<B200PP_F32>(row, i);
    }
}

__device__ __forceinline__ void store_elem_as(uint8_t *row, long long i, int dtype, float v)
{
    switch (dtype)
    {
    case B200PP_F16:
        store_elem_as<B200PP_F16>(row, i, v);
        break;
    case B200PP_BF16:
        store_elem_as<B200PP_BF16>(row, i, v);
        break;
    default:
        store_elem_as<B200PP_F32>(row, i, v);
        break;
    }
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the block, the same bits in every thread. `scratch`: 32 floats of shared memory; may be reused right away.
__device__ __forceinline__ float block_sum(float v, float *scratch)
{
    v = warp_sum(v);
    const int warps = (blockDim.x + 31) >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
        scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = (threadIdx.x & 31) < warps ? scratch[threadIdx.x & 31] : 0.0f;
    return warp_sum(s);
}

// Index i of a set of indices; -1 if it lies outside [0, rows).
__device__ __forceinline__ int load_index(const RowMap &m, int dtype, unsigned i, int rows)
{
    const uint8_t *p = m.at(i);
    long long      v;
    if (dtype == B200PP_U8)
        v = *p;
    else if (dtype == B200PP_S32)
        v = *reinterpret_cast<const int *>(p);
    else
        v = *reinterpret_cast<const long long *>(p);
    return v >= 0 && v < rows ? static_cast<int>(v) : -1;
}

} // namespace b200pp

#endif
