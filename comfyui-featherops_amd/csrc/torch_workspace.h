// The torch ops' K-split workspace.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <map>
#include <mutex>
#include <utility>

namespace feather {

// Scratch of at least nbytes for a call on `stream`, arrival counters (kCounterBytes at its
// start) zero before the first use; every call leaves them zero. The eager calls of a stream
// share one buffer, which is replaced when a call needs more. A call under stream capture never
// gets that buffer (its address would stay in the graph after a replacement has freed it) and an
// eager call none made under capture (its zero fill runs with the graph's replays only): the
// calls of one capture on one stream share a buffer allocated and zeroed inside that capture,
// whose memory torch keeps for the graph, so graphs share nothing with each other either (the
// tensor itself is held until the stream's next capture, for one that was not begun through
// torch). The caller holds the returned tensor until its kernels are enqueued: a call of
// another thread on this stream may replace the buffer meanwhile.
inline at::Tensor workspace_for(const at::Device& dev, hipStream_t stream, size_t nbytes) {
    constexpr int64_t kCounterBytes = 65536;
    struct Buffers {
        at::Tensor eager, captured;
        unsigned long long capture = 0;
    };
    static std::mutex mu;
    static std::map<std::pair<int, hipStream_t>, Buffers> pool;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(stream, &status, &id) != hipSuccess) {
        (void)hipGetLastError();  // (the legacy stream while another stream captures: not capturing itself)
        status = hipStreamCaptureStatusNone;
    }
    const bool capturing = status == hipStreamCaptureStatusActive;
    const int64_t n = static_cast<int64_t>(nbytes > (size_t(1) << 20) ? nbytes : (size_t(1) << 20));
    const auto options = at::TensorOptions().dtype(at::kByte).device(dev);
    std::lock_guard<std::mutex> lock(mu);
    Buffers& b = pool[{dev.index(), stream}];
    if (!capturing) {
        if (!b.eager.defined() || static_cast<size_t>(b.eager.numel()) < nbytes) b.eager = at::zeros({n}, options);
        return b.eager;
    }
    if (b.capture != id) b.captured.reset();  // of a capture that has ended: its graph's memory alone
    b.capture = id;
    if (!b.captured.defined() || static_cast<size_t>(b.captured.numel()) < nbytes) {
        b.captured = at::empty({n}, options);
        b.captured.narrow(0, 0, kCounterBytes).zero_();
    }
    return b.captured;
}

}  // namespace feather
