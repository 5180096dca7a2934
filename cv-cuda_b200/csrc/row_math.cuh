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

// ---- vectors of W neighbouring elements (W * size bytes, on a boundary of as many bytes)

template<int BYTES>
struct RawVec
{
    unsigned w[BYTES / 4];
};
template<>
struct RawVec<2>
{
    unsigned short w[1];
};
template<>
struct RawVec<1>
{
    unsigned char w[1];
};

// Size of an element type in bytes.
template<int DT>
constexpr int kElemBytes = sizeof(typename Elem<DT>::type);

template<int DT, int W>
using Vec = RawVec<kElemBytes<DT> * W>;

// Plain loads (not the read-only path): the operators may be asked to write over what they read.
template<int BYTES>
__device__ __forceinline__ RawVec<BYTES> load_raw(const uint8_t *p)
{
    RawVec<BYTES> r;
    if constexpr (BYTES == 32)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
                     : "l"(p));
    else if constexpr (BYTES == 16)
    {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
    }
    else if constexpr (BYTES == 8)
    {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        r.w[0] = v.x, r.w[1] = v.y;
    }
    else if constexpr (BYTES == 4)
        r.w[0] = *reinterpret_cast<const unsigned *>(p);
    else if constexpr (BYTES == 2)
        r.w[0] = *reinterpret_cast<const unsigned short *>(p);
    else
        r.w[0] = *p;
    return r;
}

template<int BYTES>
__device__ __forceinline__ void store_raw(uint8_t *p, const RawVec<BYTES> &r)
{
    if constexpr (BYTES == 32)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
                     "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
                     : "memory");
    else if constexpr (BYTES == 16)
        *reinterpret_cast<uint4 *>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    else if constexpr (BYTES == 8)
        *reinterpret_cast<uint2 *>(p) = make_uint2(r.w[0], r.w[1]);
    else if constexpr (BYTES == 4)
        *reinterpret_cast<unsigned *>(p) = r.w[0];
    else if constexpr (BYTES == 2)
        *reinterpret_cast<unsigned short *>(p) = r.w[0];
    else
        *p = r.w[0];
}

template<int BYTES>
__device__ __forceinline__ RawVec<BYTES> zero_raw()
{
    RawVec<BYTES> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(r.w) / sizeof(r.w[0])); ++i) r.w[i] = 0;
    return r;
}

template<int DT, int W>
__device__ __forceinline__ void unpack(const Vec<DT, W> &r, float *v)
{
#pragma unroll
    for (int i = 0; i < W; ++i)
    {
        if constexpr (DT == B200PP_F32)
            v[i] = __uint_as_float(r.w[i]);
        else if constexpr (DT == B200PP_U8)
        {
            if constexpr (W >= 4) // the byte becomes the low mantissa bits of 2^23, which is subtracted: exact
                v[i] = __uint_as_float(__byte_perm(r.w[i / 4], 0x4B000000u, 0x7540u + i % 4)) - 8388608.0f;
            else if constexpr (W == 2)
                v[i] = static_cast<float>((r.w[0] >> (8 * i)) & 0xffu);
            else
                v[i] = static_cast<float>(r.w[0]);
        }
        else
        {
            const unsigned bits = W == 1 ? r.w[0] : (i & 1) ? r.w[i / 2] >> 16 : r.w[i / 2] & 0xffffu;
            if constexpr (DT == B200PP_BF16)
                v[i] = __uint_as_float(bits << 16);
            else
                v[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
        }
    }
}

template<int DT, int W>
__device__ __forceinline__ Vec<DT, W> pack(const float *v)
{
    Vec<DT, W> r;
    if constexpr (DT == B200PP_F32)
    {
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = __float_as_uint(v[i]);
    }
    else if constexpr (W == 1)
        r.w[0] = DT == B200PP_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v[0])) : __half_as_ushort(__float2half_rn(v[0]));
    else
    {
#pragma unroll
        for (int i = 0; i < W; i += 2)
        {
            if constexpr (DT == B200PP_BF16)
            {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[i], v[i + 1]);
                r.w[i / 2]             = *reinterpret_cast<const unsigned *>(&h);
            }
            else
            {
                const __half2 h = __floats2half2_rn(v[i], v[i + 1]);
                r.w[i / 2]      = *reinterpret_cast<const unsigned *>(&h);
            }
        }
    }
    return r;
}

template<int DT, int W>
__device__ __forceinline__ void load_vec(const uint8_t *row, long long i, float *v)
{
    unpack<DT, W>(load_raw<kElemBytes<DT> * W>(row + i * kElemBytes<DT>), v);
}

template<int DT, int W>
__device__ __forceinline__ void store_vec(uint8_t *row, long long i, const float *v)
{
    store_raw<kElemBytes<DT> * W>(row + i * kElemBytes<DT>, pack<DT, W>(v));
}

// N neighbouring vectors, `step` elements apart, of float16, bfloat16 or float32 chosen at run time: the type is looked at once for
// all of them. Vectors that start at or after `end` are left out (load: their values are not set).
template<int DT, int W, int N>
__device__ __forceinline__ void load_vecs(const uint8_t *row, int c, int step, int end, float *v)
{
    Vec<DT, W> raw[N];
#pragma unroll
    for (int k = 0; k < N; ++k)
    {
        raw[k] = zero_raw<kElemBytes<DT> * W>();
        if (c + k * step < end)
            raw[k] = load_raw<kElemBytes<DT> * W>(row + static_cast<long long>(c + k * step) * kElemBytes<DT>);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) unpack<DT, W>(raw[k], v + k * W);
}

template<int W, int N>
__device__ __forceinline__ void load_vecs(const uint8_t *row, int dtype, int c, int step, int end, float *v)
{
    if (dtype == B200PP_F32)
        load_vecs<B200PP_F32, W, N>(row, c, step, end, v);
    else if (dtype == B200PP_BF16)
        load_vecs<B200PP_BF16, W, N>(row, c, step, end, v);
    else
        load_vecs<B200PP_F16, W, N>(row, c, step, end, v);
}

template<int DT, int W, int N>
__device__ __forceinline__ void store_vecs(uint8_t *row, int c, int step, int end, const float *v)
{
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (c + k * step < end)
            store_vec<DT, W>(row, c + k * step, v + k * W);
}

template<int W, int N>
__device__ __forceinline__ void store_vecs(uint8_t *row, int dtype, int c, int step, int end, const float *v)
{
    if (dtype == B200PP_F32)
        store_vecs<B200PP_F32, W, N>(row, c, step, end, v);
    else if (dtype == B200PP_BF16)
        store_vecs<B200PP_BF16, W, N>(row, c, step, end, v);
    else
        store_vecs<B200PP_F16, W, N>(row, c, step, end, v);
}

// ---- two float32 values in a 64-bit register: sm_100 adds, multiplies and fuses both with one instruction, each rounded as the
// scalar instruction rounds it. The row operators' kernels issue about as many instructions as HBM gives them time for, so this
// counts.
typedef unsigned long long f32x2;

__device__ __forceinline__ f32x2 make2(float lo, float hi)
{
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ f32x2 both(float v)
{
    return make2(v, v);
}

__device__ __forceinline__ float lo2(f32x2 v)
{
    return __uint_as_float(static_cast<unsigned>(v));
}

__device__ __forceinline__ float hi2(f32x2 v)
{
    return __uint_as_float(static_cast<unsigned>(v >> 32));
}

__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

template<int N>
__device__ __forceinline__ void pairs(const float *v, f32x2 *p)
{
#pragma unroll
    for (int i = 0; i < N / 2; ++i) p[i] = make2(v[2 * i], v[2 * i + 1]);
}

template<int N>
__device__ __forceinline__ void singles(const f32x2 *p, float *v)
{
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[2 * i] = lo2(p[i]), v[2 * i + 1] = hi2(p[i]);
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

// ---- rows on their way through shared memory

template<int BYTES>
__device__ __forceinline__ void copy_async(unsigned dst, const uint8_t *src, int n)
{
    // n bytes of BYTES, zeros after them
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}

__device__ __forceinline__ void copies_commit()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// All but the N latest groups are there.
template<int N>
__device__ __forceinline__ void copies_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Who a thread is: thread t of the `threads` of a row (a power of two below 32, or whole warps), row group g of the CTA; a row's values
// are dealt out as vectors, the thread's first at element c, `step` elements apart.
struct RowThread
{
    int t, threads, g, groups, c, step;
};

// One stage of one tensor for all row groups of a CTA. E values per thread as vectors of W, W dividing the row and everything
// aligned to it: each thread copies its own vectors and reads them back itself, so there is nothing to synchronise and no register
// is held while HBM answers. What lies behind a row's end is set to zero once (`clear`) and never copied over.
template<int DT, int E, int W>
struct RowStage
{
    static constexpr int kVec = kElemBytes<DT> * W, V = E / W; // 4 to 16 bytes

    static __host__ __device__ constexpr int bytes(int threads, int groups)
    {
        return kVec * V * threads * groups;
    }

    // `end`: elements of the row
    static __device__ __forceinline__ void clear(uint8_t *stage, const RowThread &k, int end)
    {
        const int tid = k.g * k.threads + k.t, all = k.threads * k.groups;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (k.c + v * k.step >= end)
                store_raw<kVec>(stage + (v * all + tid) * kVec, zero_raw<kVec>());
    }

    // RAGGED: the row may end inside a vector.
    template<bool RAGGED = false>
    static __device__ __forceinline__ void fetch(unsigned stage, const RowThread &k, const uint8_t *row, int end)
    {
        const int      tid = k.g * k.threads + k.t, all = k.threads * k.groups;
        const uint8_t *at  = row + k.c * kElemBytes<DT>;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (k.c + v * k.step < end)
                copy_async<kVec>(stage + (v * all + tid) * kVec, at + v * k.step * kElemBytes<DT>,
                                 RAGGED ? min(W, end - k.c - v * k.step) * kElemBytes<DT> : kVec);
    }

    // The thread's values, zeros behind the row's end, and before `begin` (which lies in the first vector).
    static __device__ __forceinline__ void take(const uint8_t *stage, const RowThread &k, const uint8_t *, f32x2 *out, int begin = 0)
    {
        const int  tid = k.g * k.threads + k.t, all = k.threads * k.groups;
        Vec<DT, W> raw[V];
        float      f[E];
#pragma unroll
        for (int v = 0; v < V; ++v) raw[v] = load_raw<kVec>(stage + (v * all + tid) * kVec);
#pragma unroll
        for (int v = 0; v < V; ++v) unpack<DT, W>(raw[v], f + v * W);
        if (k.c < begin)
#pragma unroll
            for (int e = 0; e < W; ++e) f[e] = e < begin ? 0.0f : f[e];
        pairs<E>(f, out);
    }
};

// The same for rows that start anywhere (W = 0): the 16-byte lines a row touches are copied as they are, by whichever thread of the
// row, zeros after its end, and each thread picks its pairs of elements out of them. (The first line may begin with bytes before the
// row: those of the row before it, or, before the first row, of the same 16 bytes of memory as its first element.) The threads of a
// row have to meet between the copies' end and `take`, and between `take` and the next copies to the stage.
template<int DT, int E>
struct RowStage<DT, E, 0>
{
    static constexpr int kSize = kElemBytes<DT>;

    static __host__ __device__ constexpr int lines(int threads)
    {
        return (threads * E * kSize + 15 + 15) / 16;
    }

    static __host__ __device__ constexpr int bytes(int threads, int groups)
    {
        return (lines(threads) * 16 + 16) * groups; // a word more for the last pair
    }

    static __device__ __forceinline__ void clear(uint8_t *, const RowThread &, int) {}

    template<bool = false>
    static __device__ __forceinline__ void fetch(unsigned stage, const RowThread &k, const uint8_t *row, int end)
    {
        const int            off   = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
        const int            bytes = off + min(end, k.threads * E) * kSize;
        const unsigned       to    = stage + k.g * bytes_of_group(k.threads);
        const uint8_t *const line  = row - off;
#pragma unroll 4
        for (int q = k.t; q < lines(k.threads); q += k.threads)
        {
            const int n = min(16, max(0, bytes - q * 16));
            copy_async<16>(to + q * 16, n > 0 ? line + q * 16 : line, n);
        }
    }

    static __device__ __forceinline__ void take(const uint8_t *stage, const RowThread &k, const uint8_t *row, f32x2 *out, int = 0)
    {
        // the thread's first pair starts `at` bytes into the lines
        const int       at    = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) + k.c * kSize;
        const int       shift = (at & 3) * 8;
        const unsigned *w     = reinterpret_cast<const unsigned *>(stage + k.g * bytes_of_group(k.threads)) + (at >> 2);
#pragma unroll
        for (int v = 0; v < E / 2; ++v)
        {
            float f[2];
            if constexpr (kSize == 1)
            {
                // vectors are an even number of bytes apart, which need not be whole words
                const int      b = at + v * k.step;
                const unsigned *x = reinterpret_cast<const unsigned *>(stage + k.g * bytes_of_group(k.threads)) + (b >> 2);
                const unsigned  bits = __funnelshift_r(x[0], x[1], (b & 3) * 8);
                f[0]                 = static_cast<float>(bits & 0xffu);
                f[1]                 = static_cast<float>((bits >> 8) & 0xffu);
            }
            else
            {
                const unsigned w0 = w[v * k.step * kSize / 4], w1 = w[v * k.step * kSize / 4 + 1];
                if constexpr (kSize == 4)
                {
                    f[0] = __uint_as_float(w0);
                    f[1] = __uint_as_float(w1);
                }
                else
                {
                    Vec<DT, 2> r;
                    r.w[0] = __funnelshift_r(w0, w1, shift);
                    unpack<DT, 2>(r, f);
                }
            }
            out[v] = make2(f[0], f[1]);
        }
    }

private:
    static __host__ __device__ constexpr int bytes_of_group(int threads)
    {
        return lines(threads) * 16 + 16;
    }
};

// How the threads of a row are laid out over its elements: with `lanes` = 32 or more, warp by warp, 32 E elements each; below, lane
// by lane. W = 0 goes by pairs.
// (WHOLE: whole warps, which lets the compiler know the distance between a thread's vectors.)
template<int E, int W, bool WHOLE>
__device__ __forceinline__ RowThread row_thread(int t, int threads, int g, int groups)
{
    constexpr int kW    = W ? W : 2;
    const int     lanes = WHOLE ? 32 : threads;
    return {t, threads, g, groups, (WHOLE ? (t >> 5) * (32 * E) + (t & 31) * kW : t * kW), lanes * kW};
}

// Eight neighbouring-by-vector values of a parameter (weight, bias), from the thread's vector at element c on.
template<int W>
__device__ __forceinline__ void load_param(const uint8_t *p, int dtype, int c, int step, int end, f32x2 *out)
{
    float f[8];
    if constexpr (W > 0)
        load_vecs<W, 8 / W>(p, dtype, c, step, end, f);
    else
    {
#pragma unroll
        for (int v = 0; v < 4; ++v)
        {
            f[2 * v]     = c + v * step < end ? load_elem(p, c + v * step, dtype) : 0.0f;
            f[2 * v + 1] = c + v * step + 1 < end ? load_elem(p, c + v * step + 1, dtype) : 0.0f;
        }
    }
    pairs<8>(f, out);
}

// N elements of a parameter, all under way at once; where `at` points outside, the nearest one.
template<int DT, int N, typename F>
__device__ __forceinline__ void load_scattered(const uint8_t *p, int count, float *out, F at)
{
    Vec<DT, 1> raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = load_raw<kElemBytes<DT>>(p + static_cast<long long>(min(max(at(i), 0), count - 1)) * kElemBytes<DT>);
#pragma unroll
    for (int i = 0; i < N; ++i) unpack<DT, 1>(raw[i], out + i);
}

template<int N, typename F>
__device__ __forceinline__ void load_scattered(const uint8_t *p, int dtype, int count, float *out, F at)
{
    if (dtype == B200PP_F32)
        load_scattered<B200PP_F32, N>(p, count, out, at);
    else if (dtype == B200PP_BF16)
        load_scattered<B200PP_BF16, N>(p, count, out, at);
    else
        load_scattered<B200PP_F16, N>(p, count, out, at);
}

// A thread's values to its row, which may start anywhere.
template<int DT, int E>
__device__ __forceinline__ void store_pairs(uint8_t *row, int c, int step, int end, const float *f)
{
    const bool whole = (reinterpret_cast<uintptr_t>(row) & (2 * kElemBytes<DT> - 1)) == 0; // pairs start on even elements
    if (c + (E / 2 - 1) * step + 1 < end)
    {
        uint8_t *at = row + c * kElemBytes<DT>;
        if (whole)
        {
#pragma unroll
            for (int v = 0; v < E / 2; ++v) store_vec<DT, 2>(at, v * step, f + 2 * v);
        }
        else
        {
#pragma unroll
            for (int v = 0; v < E / 2; ++v)
            {
                store_elem_as<DT>(at, v * step, f[2 * v]);
                store_elem_as<DT>(at, v * step + 1, f[2 * v + 1]);
            }
        }
        return;
    }
    uint8_t *at = row + c * kElemBytes<DT>;
#pragma unroll
    for (int v = 0; v < E / 2; ++v)
    {
        // past the end for every thread of the row, or for none, but for one vector
        if (c + v * step >= end)
            break;
        if (whole && c + v * step + 1 < end)
            store_vec<DT, 2>(at, v * step, f + 2 * v);
        else
        {
            store_elem_as<DT>(at, v * step, f[2 * v]);
            if (c + v * step + 1 < end)
                store_elem_as<DT>(at, v * step + 1, f[2 * v + 1]);
        }
    }
}

// A thread's values to its row from element `begin`, which lies in the first vector, to `end`, which may lie inside one.
template<int DT, int E, int W>
__device__ __forceinline__ void store_ragged(uint8_t *row, const RowThread &k, int begin, int end, const float *f)
{
#pragma unroll
    for (int v = 0; v < E / W; ++v)
    {
        const int c = k.c + v * k.step;
        if (c >= begin && c + W <= end)
            store_vec<DT, W>(row, c, f + v * W);
        else
        {
#pragma unroll
            for (int e = 0; e < W; ++e)
                if (c + e >= begin && c + e < end)
                    store_elem_as<DT>(row, c + e, f[v * W + e]);
        }
    }
}

template<int E, int W, bool RAGGED = false>
__device__ __forceinline__ void store_row(uint8_t *row, int dtype, const RowThread &k, int end, const f32x2 *x, int begin = 0)
{
    float f[E];
    singles<E>(x, f);
    if constexpr (W > 0 && RAGGED)
    {
        if (dtype == B200PP_F32)
            store_ragged<B200PP_F32, E, W>(row, k, begin, end, f);
        else if (dtype == B200PP_BF16)
            store_ragged<B200PP_BF16, E, W>(row, k, begin, end, f);
        else
            store_ragged<B200PP_F16, E, W>(row, k, begin, end, f);
    }
    else if constexpr (W > 0)
        store_vecs<W, E / W>(row, dtype, k.c, k.step, end, f);
    else if (dtype == B200PP_F32)
        store_pairs<B200PP_F32, E>(row, k.c, k.step, end, f);
    else if (dtype == B200PP_BF16)
        store_pairs<B200PP_BF16, E>(row, k.c, k.step, end, f);
    else
        store_pairs<B200PP_F16, E>(row, k.c, k.step, end, f);
}

// s / n for a count n and inv = 1 / n rounded: one step of division by residual. A sum of n equal values gives the value itself. An
// infinite s has no residual and stays infinite.
__device__ __forceinline__ float divide_count(float s, float n, float inv)
{
    const float q = s * inv;
    return isinf(q) ? q : fmaf(fmaf(-q, n, s), inv, q);
}

template<int DT>
struct Index;
template<>
struct Index<B200PP_U8>
{
    typedef uint8_t type;
};
template<>
struct Index<B200PP_S32>
{
    typedef int type;
};
template<>
struct Index<B200PP_S64>
{
    typedef long long type;
};

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
