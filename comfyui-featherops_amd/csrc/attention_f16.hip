// Attention over many queries in fp16 (attention_tiles.h).
#include "attention_tiles.h"

namespace feather {

int attention_tiles_f16(const AttnArgs& p, hipStream_t stream) { return attention_tiles<false>(p, stream); }

}  // namespace feather
