// Attention in fp16.
#include "attention_launch.h"

namespace feather {

int attention_f16(const AttnArgs& p, const AttnPlan& plan, void* workspace, hipStream_t stream) {
    return attention_of_type<false>(p, plan, workspace, stream);
}

}  // namespace feather
