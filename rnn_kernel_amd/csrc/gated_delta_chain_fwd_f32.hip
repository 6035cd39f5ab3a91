// The gated delta rule's forward chain for float tensors (a file per type and
// direction, so that they compile side by side).
#include "gated_delta_chain.h"

namespace rka {
namespace delta {

template <>
int launch_chain_forward<float>(const Dims& d, const float* s0, const int* lengths, const ChunkData& in, float* o,
                                float* state_out, float* states, float* e, hipStream_t stream) {
    return with_chain<float>(d, [&](auto ku, auto nc) {
        constexpr int KU = decltype(ku)::value, NC = decltype(nc)::value;
        const long long blocks = chain_blocks(d, NC);
        RKA_RETURN_IF_ERR(check_grid(blocks, kChainThreads, "gated_delta_forward"));
        hipLaunchKernelGGL((chain_forward_kernel<float, KU, NC>), dim3((unsigned)blocks), dim3(kChainThreads), 0, stream, d,
                           s0, lengths, in, o, state_out, states, e);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    });
}

}  // namespace delta
}  // namespace rka
