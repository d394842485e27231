// f16 instantiations of kv_attend.hpp.
#include "kv_attend.hpp"

namespace mla {

hipError_t launch_kv_attend_f16(const KvArgs& a, bool many, hipStream_t stream) {
    return launch_list<F16>(a, many, stream);
}

}  // namespace mla
