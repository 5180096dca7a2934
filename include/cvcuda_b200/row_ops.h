/*
 * Row operators for NVIDIA B200 (sm_100a): plain-C launch layer.
 *
 * LayerNorm and the embedding lookup, each with its gradient: the operators between the tensors the image operators of
 * preproc.h produce (and the indices that come with them: tokens, class labels, label maps) and the first activations of
 * the model they feed. They have no counterpart in the reference. Conventions are those of preproc.h: pointers, sizes and
 * byte strides only; every function is asynchronous with respect to `stream`, allocates nothing and returns an NVCVStatus
 * value (0 = success), whose message b200ppGetLastErrorMessage() keeps. The stream belongs to the current device.
 *
 * Functions that need scratch memory take it from the caller: a ...Workspace function (host only) gives the size, which
 * may be 0. The contents need not be kept or cleared between calls. Calls whose GPU work can overlap -- on two streams, or
 * in two graphs that may replay at the same time -- need a workspace each.
 *
 * Results do not depend on timing: equal inputs of equal alignment give equal bits.
 */
#ifndef CVCUDA_B200_ROW_OPS_H
#define CVCUDA_B200_ROW_OPS_H

#include <cvcuda_b200/preproc.h>

#if defined(__cplusplus)
extern "C"
{
#endif

/* Element types the row operators take besides those of preproc.h. */
enum
{
    B200PP_BF16 = 8, /* bfloat16 */
    B200PP_S64  = 9  /* indices only */
};

/* A set of rows of `cols` adjacent elements each. Row r = (r0 * count[1] + r1) * count[2] + r2 starts
 * r0 * stride[0] + r1 * stride[1] + r2 * stride[2] bytes after base, which expresses a matrix, the pixels of an NHWC tensor
 * with padded rows, or the images of a batch. Strides are multiples of the element size, of any sign; those of a tensor
 * that is written keep its rows apart. At most 2^31 - 1 rows, and at most 2^31 - 2^16 columns. */
typedef struct B200ppRows
{
    void   *base;
    int32_t dtype;
    int64_t cols;
    int64_t count[3];
    int64_t stride[3];
} B200ppRows;

/* LayerNorm: dst = (src - mean) * rstd * weight + bias, row by row, mean and rstd = 1 / sqrt(variance + epsilon) being those
 * of the row (variance: the mean of the squared distances to the mean). src: uint8, float16, bfloat16 or float32; dst:
 * float16, bfloat16 or float32. weight and bias: `cols` adjacent values of float16, bfloat16 or float32, each NULL for 1
 * and 0. mean and rstd: if not NULL, the float32 statistics of the rows, packed, in row order, for the backward pass.
 * Sums are float32 (the variance about the mean, not the difference of two sums), rstd is an approximate reciprocal square
 * root, off by two units in the last place at most. The mean of a row with infinities of one sign is that infinity; its rstd
 * and result, and those of a row with NaN, are NaN. dst may be src if the types agree; apart from that no output may overlap
 * an input or another output. Rows of up to 8192 columns need no workspace. */
typedef struct B200ppLayerNormOp
{
    const void *weight;
    const void *bias;
    int32_t     weightType, biasType;
    float       epsilon; /* >= 0 */
    float      *mean, *rstd;
} B200ppLayerNormOp;

B200PP_PUBLIC int b200ppLayerNormWorkspace(const B200ppRows *src, size_t *bytes);
B200PP_PUBLIC int b200ppLayerNorm(const B200ppRows *src, const B200ppRows *dst, const B200ppLayerNormOp *op, void *workspace,
                                  size_t workspaceBytes, cudaStream_t stream);

/* Gradients of LayerNorm. With h = (src - mean) * rstd and g = grad * weight (g = grad where weight is NULL), row by row:
 *   dsrc    = rstd * (g - mean(g) - h * mean(g * h))
 *   dweight = the sum over the rows of grad * h
 *   dbias   = the sum over the rows of grad
 * grad: float16, bfloat16 or float32, the gradient of the forward pass's dst; src, mean, rstd, weight: as there. dsrc (NULL
 * where it is not wanted; float16, bfloat16 or float32) may be grad, or src, if the types agree; other overlaps are not
 * allowed. dweight and dbias: `cols` adjacent values, NULL where not wanted. All sums are float32, rounded to the output's
 * type once. No rows: zeros. Up to 256 rows of up to 4096 columns, and calls without dweight and dbias, need no workspace. */
typedef struct B200ppLayerNormGradOp
{
    const float *mean, *rstd;
    const void  *weight;
    int32_t      weightType;
    void        *dweight, *dbias;
    int32_t      dweightType, dbiasType;
} B200ppLayerNormGradOp;

B200PP_PUBLIC int b200ppLayerNormBackwardWorkspace(const B200ppRows *src, size_t *bytes);
B200PP_PUBLIC int b200ppLayerNormBackward(const B200ppRows *grad, const B200ppRows *src, const B200ppRows *dsrc,
                                          const B200ppLayerNormGradOp *op, void *workspace, size_t workspaceBytes,
                                          cudaStream_t stream);

/* Embedding lookup: row i of dst = scale * row indices[i] of table. indices: rows of one column, uint8, int32 or int64, as
 * many as dst has rows. An index outside [0, rows of the table) gives a row of zeros, so that a table that holds a part of
 * the rows can be used with indices shifted by its first row. table and dst: float16, bfloat16 or float32, the same number
 * of columns. The product is float32, rounded to dst's type once. dst must not overlap table. */
B200PP_PUBLIC int b200ppEmbedding(const B200ppRows *indices, const B200ppRows *table, const B200ppRows *dst, float scale,
                                  cudaStream_t stream);

/* Gradient of the embedding lookup: row v of dtable = scale * the sum of the rows i of grad with indices[i] = v, in float32,
 * in an order that the indices, the types and the tensors' layout settle; a row no index names is zero. With `accumulate`, the
 * sum is added to what dtable holds, and rows no index names stay as they are. Indices outside the table, and those equal to
 * paddingIndex (a value outside the table: none), take no part. grad and dtable: float16, bfloat16 or float32. dtable must not
 * overlap grad or indices. Up to 8192 indices need no workspace, except with very large tables. */
typedef struct B200ppEmbeddingGradOp
{
    float   scale;
    int32_t accumulate;
    int64_t paddingIndex;
} B200ppEmbeddingGradOp;

B200PP_PUBLIC int b200ppEmbeddingBackwardWorkspace(const B200ppRows *grad, const B200ppRows *dtable, size_t *bytes);
B200PP_PUBLIC int b200ppEmbeddingBackward(const B200ppRows *grad, const B200ppRows *indices, const B200ppRows *dtable,
                                          const B200ppEmbeddingGradOp *op, void *workspace, size_t workspaceBytes,
                                          cudaStream_t stream);

#if defined(__cplusplus)
}
#endif

#endif /* CVCUDA_B200_ROW_OPS_H */
