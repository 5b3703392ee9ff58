// Attention in bf16.
#include "attention_launch.h"

namespace feather {

int attention_bf16(const AttnArgs& p, const AttnPlan& plan, void* workspace, hipStream_t stream) {
    return attention_of_type<true>(p, plan, workspace, stream);
}

}  // namespace feather
