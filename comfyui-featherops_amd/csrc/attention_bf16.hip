// Attention over many queries in bf16 (attention_tiles.h).
#include "attention_tiles.h"

namespace feather {

int attention_tiles_bf16(const AttnArgs& p, hipStream_t stream) { return attention_tiles<true>(p, stream); }

}  // namespace feather
