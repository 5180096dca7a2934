// Launch of the one-pass LayerNorm gradient kernel. The kernel is compiled in one translation unit per element type of the source
// (layernorm_grad_<type>.cu), for compilation time.
#ifndef CVCUDA_B200_LAYERNORM_GRAD_LAUNCH_CUH
#define CVCUDA_B200_LAYERNORM_GRAD_LAUNCH_CUH

#include "layernorm_grad_kernels.cuh"
#include "row_host.h"

namespace b200pp {

// How the rows are dealt out. One-pass kernel: `threads` per row and CTA with `values` values each, `groups` rows per CTA, a cluster of
// `ctas` CTAs with `span` columns each per row, one part per CTA or cluster; for longer rows (values = 0) the sums over the rows
// are a kernel of their own.
struct GradPlan
{
    int  threads, groups, values, ctas, span, parts;
    bool ragged;
};

// Gradients of the element type p.gradType (float16 sources: not bfloat16, and the other way round): status of the launch, or -1
// for a type there is no kernel for.
int layernorm_grad_u8(const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream);
int layernorm_grad_f16(const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream);
int layernorm_grad_bf16(const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream);
int layernorm_grad_f32(const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream);

template<int SRC, int GRAD, int E, int W, bool RAGGED, bool WARP, bool FULL>
int launch_one_pass(const LayerNormGradKParams &p, const GradPlan &g, cudaStream_t stream)
{
    typedef GradRing<SRC, GRAD, E, W>      Ring;
    static std::atomic<unsigned long long> raised{0};
    const int                              warps = g.threads * g.groups / 32, slots = WARP ? warps : g.groups;
    const int copies = p.ownWeights ? g.groups : 1; // of the weights
    const int ring   = Ring::bytes(g.threads, g.groups) * Ring::kStages + g.threads * copies * E * static_cast<int>(sizeof(float));
    const int sums = p.partials ? slots * 2 * g.span * static_cast<int>(sizeof(float)) : 0;
    const int smem = std::max(ring, sums);
    if (smem > 32 * 1024) // a launch gets 48 KB unasked, static memory included
        if (int st = raise_smem(layernorm_grad_kernel<SRC, GRAD, E, W, WARP, FULL, RAGGED>, 208 * 1024, raised))
            return st;
    Launch(dim3(p.parts * g.ctas), dim3(g.threads, g.groups), smem, stream, g.ctas, false)
        .run(layernorm_grad_kernel<SRC, GRAD, E, W, WARP, FULL, RAGGED>, p, g.span);
    return check_launch("LayerNormBackward");
}

template<int SRC, int GRAD, int W, bool RAGGED>
int launch_one_pass(const LayerNormGradKParams &p, const GradPlan &g, cudaStream_t stream)
{
    if (g.threads > 32)
        return g.values == 16 ? launch_one_pass<SRC, GRAD, 16, W, RAGGED, false, true>(p, g, stream)
                              : launch_one_pass<SRC, GRAD, 24, W, RAGGED, false, true>(p, g, stream);
    if (g.values == 8)
        return launch_one_pass<SRC, GRAD, 8, W, RAGGED, true, false>(p, g, stream);
    if (g.threads == 32)
        return g.values == 16 ? launch_one_pass<SRC, GRAD, 16, W, RAGGED, true, true>(p, g, stream)
                              : launch_one_pass<SRC, GRAD, 24, W, RAGGED, true, true>(p, g, stream);
    return g.values == 16 ? launch_one_pass<SRC, GRAD, 16, W, RAGGED, true, false>(p, g, stream)
                          : launch_one_pass<SRC, GRAD, 24, W, RAGGED, true, false>(p, g, stream);
}

template<int SRC, int GRAD>
int launch_one_pass(const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream)
{
    // vectors of 16 bytes at most on the way through shared memory; of four elements at least, otherwise the rows' lines as they are
    constexpr int kWide = SRC != B200PP_F32 && GRAD != B200PP_F32 ? 8 : 4;
    if (g.ragged)
        return launch_one_pass<SRC, GRAD, kWide, true>(p, g, stream);
    if (width == 8 && kWide == 8)
        return launch_one_pass<SRC, GRAD, kWide, false>(p, g, stream);
    if (width >= 4)
        return launch_one_pass<SRC, GRAD, 4, false>(p, g, stream);
    return launch_one_pass<SRC, GRAD, 0, false>(p, g, stream);
}

} // namespace b200pp

#endif
