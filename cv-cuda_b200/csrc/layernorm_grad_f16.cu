// The one-pass LayerNorm gradient kernels of float16 sources.
#include "layernorm_grad_launch.cuh"

namespace b200pp {

int layernorm_grad_f16(const LayerNormGradKParams &p, const GradPlan &g, int width, cudaStream_t stream)
{
    switch (p.gradType)
    {
    case B200PP_F16:
        return launch_one_pass<B200PP_F16, B200PP_F16>(p, g, width, stream);
    case B200PP_F32:
        return launch_one_pass<B200PP_F16, B200PP_F32>(p, g, width, stream);
    }
    return -1;
}

} // namespace b200pp
