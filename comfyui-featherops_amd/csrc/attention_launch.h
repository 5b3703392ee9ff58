// The instances of the attention kernels for one type of values.
#pragma once

#include "attention_rows.h"
#include "attention_tiles.h"

namespace feather {

template <int kDim, bool kBf16, int kMask>
int launch_attention(const AttnArgs& p, const AttnPlan& plan, void* workspace, hipStream_t stream) {
    if (plan.waves == 0) return launch_attention_tiles<kDim, kBf16, kMask>(p, plan, stream);
    if constexpr (kDim <= 128)
        if (plan.waves == 8) return launch_attention_rows<kDim, kBf16, kMask, 8>(p, plan, workspace, stream);
    return launch_attention_rows<kDim, kBf16, kMask, 4>(p, plan, workspace, stream);
}

template <int kDim, bool kBf16>
int attention_of_mask(const AttnArgs& p, const AttnPlan& plan, void* workspace, hipStream_t stream) {
    switch (p.mask_type) {
        case kMaskNone: return launch_attention<kDim, kBf16, kMaskNone>(p, plan, workspace, stream);
        case kMaskBool: return launch_attention<kDim, kBf16, kMaskBool>(p, plan, workspace, stream);
        case kMaskHalf: return launch_attention<kDim, kBf16, kMaskHalf>(p, plan, workspace, stream);
        default: return launch_attention<kDim, kBf16, kMaskF32>(p, plan, workspace, stream);
    }
}

template <bool kBf16>
int attention_of_type(const AttnArgs& p, const AttnPlan& plan, void* workspace, hipStream_t stream) {
    if (p.dim <= 64) return attention_of_mask<64, kBf16>(p, plan, workspace, stream);
    if (p.dim <= 96) return attention_of_mask<96, kBf16>(p, plan, workspace, stream);
    if (p.dim <= 128) return attention_of_mask<128, kBf16>(p, plan, workspace, stream);
    return attention_of_mask<256, kBf16>(p, plan, workspace, stream);
}

}  // namespace feather
