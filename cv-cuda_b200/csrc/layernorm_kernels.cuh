// LayerNorm and its gradient.
//
// Forward, per row of D values: m = sum(x) / D, v = sum((x - m)^2) / D, r = 1 / sqrt(v + epsilon), y = (x - m) r w + b.
// Backward: h = (x - m) r, g = dy w, dx = r (g - mean(g) - h mean(g h)); dw = sum over rows of dy h, db = sum of dy.
// Bound: HBM (about one operation per byte moved).
#ifndef CVCUDA_B200_LAYERNORM_KERNELS_CUH
#define CVCUDA_B200_LAYERNORM_KERNELS_CUH

#include "row_math.cuh"

namespace b200pp {

struct LayerNormKParams
{
    RowMap         src, dst;
    unsigned       rows;
    int            cols;
    int            dstType, weightType, biasType;
    const uint8_t *weight, *bias;
    float          epsilon, fcols; // fcols: the number of columns
    float         *mean, *rstd;
};

struct LayerNormGradKParams
{
    RowMap         grad, src, dsrc;
    unsigned       rows;
    int            cols;
    int            gradType, dsrcType, weightType, dweightType, dbiasType;
    const uint8_t *weight;
    const float   *mean, *rstd;
    float          fcols;
    uint8_t       *dweight, *dbias;
    float         *partials; // [parts][2][cols]
    int            parts;
};

// One CTA per row, any row length.
template<int SRC>
__global__ void __launch_bounds__(256) layernorm_row_kernel(const LayerNormKParams p)
{
    __shared__ float scratch[32];
    for (unsigned r = blockIdx.x; r < p.rows; r += gridDim.x)
    {
        const uint8_t *x = p.src.at(r);
        uint8_t       *y = p.dst.at(r);
        float          s = 0.0f;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) s += load_elem<SRC>(x, c);
        const float mean = block_sum(s, scratch) / p.fcols;
        float       q    = 0.0f;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x)
        {
            const float d = load_elem<SRC>(x, c) - mean;
            q             = fmaf(d, d, q);
        }
        const float rstd = 1.0f / sqrtf(block_sum(q, scratch) / p.fcols + p.epsilon);
        if (threadIdx.x == 0)
        {
            if (p.mean)
                p.mean[r] = mean;
            if (p.rstd)
                p.rstd[r] = rstd;
        }
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x)
        {
            const float w = p.weight ? load_elem(p.weight, c, p.weightType) : 1.0f;
            const float b = p.bias ? load_elem(p.bias, c, p.biasType) : 0.0f;
            store_elem_as(y, c, p.dstType, fmaf((load_elem<SRC>(x, c) - mean) * rstd, w, b));
        }
    }
}

// dx, one CTA per row, any row length.
template<int SRC>
__global__ void __launch_bounds__(256) layernorm_grad_row_kernel(const LayerNormGradKParams p)
{
    __shared__ float scratch[32];
    for (unsigned r = blockIdx.x; r < p.rows; r += gridDim.x)
    {
        const uint8_t *x = p.src.at(r), *dy = p.grad.at(r);
        uint8_t       *dx   = p.dsrc.at(r);
        const float    mean = p.mean[r], rstd = p.rstd[r];
        float          s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x)
        {
            const float w = p.weight ? load_elem(p.weight, c, p.weightType) : 1.0f;
            const float g = load_elem(dy, c, p.gradType) * w;
            s1 += g;
            s2 = fmaf(g, (load_elem<SRC>(x, c) - mean) * rstd, s2);
        }
        const float c1 = block_sum(s1, scratch) / p.fcols;
        const float c2 = block_sum(s2, scratch) / p.fcols;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x)
        {
            const float w = p.weight ? load_elem(p.weight, c, p.weightType) : 1.0f;
            const float g = load_elem(dy, c, p.gradType) * w;
            const float h = (load_elem<SRC>(x, c) - mean) * rstd;
            store_elem_as(dx, c, p.dsrcType, rstd * (g - c1 - h * c2));
        }
    }
}

// dw and db: a CTA sums one part of the rows for 32 columns; layernorm_grad_join_kernel adds the parts up.
template<int SRC>
__global__ void __launch_bounds__(256) layernorm_grad_columns_kernel(const LayerNormGradKParams p)
{
    __shared__ float sw[8][32], sb[8][32];
    const int        lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long  c    = static_cast<long long>(blockIdx.x) * 32 + lane;
    const unsigned   per  = (p.rows + p.parts - 1) / p.parts;
    const unsigned   r0   = min(p.rows, static_cast<unsigned>(blockIdx.y) * per), r1 = min(p.rows, r0 + per);
    float            dw = 0.0f, db = 0.0f;
    if (c < p.cols)
        for (unsigned r = r0 + warp; r < r1; r += 8)
        {
            const float g = load_elem(p.grad.at(r), c, p.gradType);
            db += g;
            dw = fmaf(g, (load_elem<SRC>(p.src.at(r), c) - p.mean[r]) * p.rstd[r], dw);
        }
    sw[warp][lane] = dw;
    sb[warp][lane] = db;
    __syncthreads();
    if (warp == 0 && c < p.cols)
    {
        for (int k = 1; k < 8; ++k)
        {
            dw += sw[k][lane];
            db += sb[k][lane];
        }
        float *part       = p.partials + static_cast<long long>(blockIdx.y) * 2 * p.cols;
        part[c]           = dw;
        part[p.cols + c]  = db;
    }
}

__global__ void __launch_bounds__(256) layernorm_grad_join_kernel(const LayerNormGradKParams p)
{
    const long long c = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (c >= p.cols)
        return;
    float dw = 0.0f, db = 0.0f;
    for (int k = 0; k < p.parts; ++k)
    {
        dw += p.partials[static_cast<long long>(2 * k) * p.cols + c];
        db += p.partials[static_cast<long long>(2 * k + 1) * p.cols + c];
    }
    if (p.dweight)
        store_elem_as(p.dweight, c, p.dweightType, dw);
    if (p.dbias)
        store_elem_as(p.dbias, c, p.dbiasType, db);
}

} // namespace b200pp

#endif
