// Attention over the quantised cache for heads of 64 elements.
#include "attention_tiles.cuh"

namespace tf {
template tf_status attend<64, 4>(tf_context*, cudaStream_t, const AttnArgs&, const tf_attention_workspace*, bool);
template tf_status attend<64, 8>(tf_context*, cudaStream_t, const AttnArgs&, const tf_attention_workspace*, bool);
}  // namespace tf
