// cf_decay_tc_f16.cu — the chunk kernel of cf_decay_attention for fp16.
#include "cf_decay_launch.cuh"

namespace cf {
namespace decayk {
template int launch_chunks<__half>(bool, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                const DecayArgs&, int, cudaStream_t);
}
}  // namespace cf
