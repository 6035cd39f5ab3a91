// The gated delta rule's backward chain for bf16 tensors.
#include "gated_delta_chain.h"

namespace rka {
namespace delta {

template <>
int launch_chain_backward<bf16>(const Dims& d, const bf16* dout, const float* dstate_out, const int* lengths,
                                 const ChunkData& in, bf16* dv, float* ds0, const BackwardData& bd, hipStream_t stream) {
    return with_chain<bf16>(d, [&](auto ku, auto nc) {
        constexpr int KU = decltype(ku)::value, NC = decltype(nc)::value;
        const long long blocks = chain_blocks(d, NC);
        RKA_RETURN_IF_ERR(check_grid(blocks, kChainThreads, "gated_delta_backward"));
        hipLaunchKernelGGL((chain_backward_kernel<bf16, KU, NC>), dim3((unsigned)blocks), dim3(kChainThreads), 0, stream,
                           d, dout, dstate_out, lengths, in, dv, ds0, bd);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    });
}

}  // namespace delta
}  // namespace rka
