// Planned attention over the 8-bit latent cache: the instantiations of latent_attend_kernel.
#include "latent_attend.hpp"

namespace mla {

hipError_t launch_attend_q8(const LatentArgs& a, int dtype, bool rows, hipStream_t stream) {
    return dtype == 0 ? launch_list<F16, true>(a, rows, stream)
                      : launch_list<BF16, true>(a, rows, stream);
}

}  // namespace mla
