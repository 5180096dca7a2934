// Launch of the embedding gradient's kernel for few indices.
#include "embedding_grad_direct.cuh"
#include "row_host.h"

#include <algorithm>

namespace b200pp {

namespace {

template<int GRAD, int W>
int launch(EmbeddingDirectKParams &p, int padding, cudaStream_t stream)
{
    constexpr int  C      = kDirectLanes<GRAD, W> * W;
    const unsigned blocks = static_cast<unsigned>((static_cast<long long>(p.cols) + C - 1) / C);
    // two CTAs per SM, more for tables of more rows than those keep track of
    const unsigned least = (static_cast<unsigned>(p.rows) + kDirectRows - 1) / kDirectRows;
    p.ranges             = std::min<unsigned>(p.rows, std::max(least, 2 * kSms / blocks));
    p.most               = static_cast<int>((static_cast<unsigned>(p.rows) + p.ranges - 1) / p.ranges);
    p.rest               = static_cast<int>(static_cast<unsigned>(p.rows) - (p.most - 1) * p.ranges);
    p.paddingRange       = padding >= 0 ? padding % p.ranges : p.ranges;
    p.paddingRow         = padding >= 0 ? padding / p.ranges : 0;
    p.twos               = 0;
    while (!(p.ranges >> p.twos & 1)) ++p.twos;
    const unsigned odd = p.ranges >> p.twos;
    p.inverse          = odd; // right in three bits; each step doubles them
    for (int k = 0; k < 4; ++k) p.inverse *= 2 - odd * p.inverse;
    static std::atomic<unsigned long long> raised{0};
    const size_t                           smem = direct_smem(p.count, p.most);
    if (smem > 32 * 1024)
        if (int st = raise_smem(embedding_grad_direct_kernel<GRAD, W>, static_cast<int>(direct_smem(kDirectCount, kDirectRows)), raised))
            return st;
    embedding_grad_direct_kernel<GRAD, W><<<dim3(blocks, p.ranges), kDirectThreads, smem, stream>>>(p);
    return check_launch("EmbeddingBackward");
}

template<int GRAD>
int launch(EmbeddingDirectKParams &p, int width, int padding, cudaStream_t stream)
{
    if constexpr (GRAD != B200PP_F32)
        if (width == 8)
            return launch<GRAD, 8>(p, padding, stream);
    if (width >= 4)
        return launch<GRAD, 4>(p, padding, stream);
    if (width == 2)
        return launch<GRAD, 2>(p, padding, stream);
    return launch<GRAD, 1>(p, padding, stream);
}

} // namespace

int embedding_grad_direct(EmbeddingDirectKParams &p, int width, int padding, cudaStream_t stream)
{
    if (p.gradType == B200PP_F16)
        return launch<B200PP_F16>(p, width, padding, stream);
    if (p.gradType == B200PP_BF16)
        return launch<B200PP_BF16>(p, width, padding, stream);
    return launch<B200PP_F32>(p, width, padding, stream);
}

} // namespace b200pp
