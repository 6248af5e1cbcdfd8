// call.h -- what the entry points that take both host and device arrays share: the checks of a caller's pointers and the staging of
// host arrays (CZ_DEVICE_PTRS unset).
#pragma once
#include <deque>

#include "common.h"

namespace cz {

// a pointer handed in as device memory: refused when the runtime knows it as plain host memory or as another GPU's
inline int check_device_ptr(const void *p, const char *what) {
    if (!p) return CZ_OK;
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {  // a mapping the runtime does not track: the caller's word stands
        (void)hipGetLastError();
        return CZ_OK;
    }
    if (a.type == hipMemoryTypeUnregistered) return set_error(CZ_E_INVALID, "%s: host memory handed in with CZ_DEVICE_PTRS", what);
    int dev = 0;
    CZ_HIP(hipGetDevice(&dev));
    if (a.type == hipMemoryTypeDevice && a.device != dev)
        return set_error(CZ_E_INVALID, "%s is on device %d, the library works on device %d", what, a.device, dev);
    return CZ_OK;
}

// host arrays of one synchronous call: copied in before the work, copied back by finish()
class HostStage {
  public:
    explicit HostStage(hipStream_t s) : stream_(s) {}
    template <typename T>
    int in(const T *host, size_t count, const T **dev) {
        void *d = nullptr;
        int rc = place(count * sizeof(T), &d);
        if (rc) return rc;
        if (count) CZ_HIP(hipMemcpyAsync(d, host, count * sizeof(T), hipMemcpyHostToDevice, stream_));
        *dev = static_cast<const T *>(d);
        return CZ_OK;
    }
    template <typename T>
    int out(T *host, size_t count, T **dev) {
        void *d = nullptr;
        int rc = place(count * sizeof(T), &d);
        if (rc) return rc;
        outs_.push_back({host, d, count * sizeof(T)});
        *dev = static_cast<T *>(d);
        return CZ_OK;
    }
    int finish() {
        for (const Out &o : outs_)
            if (o.bytes) CZ_HIP(hipMemcpyAsync(o.host, o.dev, o.bytes, hipMemcpyDeviceToHost, stream_));
        CZ_HIP(hipStreamSynchronize(stream_));
        return CZ_OK;
    }

  private:
    struct Out {
        void *host, *dev;
        size_t bytes;
    };
    int place(size_t bytes, void **d) {
        bufs_.emplace_back();
        CZ_HIP(bufs_.back().alloc(bytes));
        *d = bufs_.back().p;
        return CZ_OK;
    }
    hipStream_t stream_;
    std::deque<DevBuf<uint8_t>> bufs_;
    std::deque<Out> outs_;
};

// the scratch of one call, cut into 256-byte aligned pieces; sizes are added up with base = nullptr first
class Carve {
  public:
    explicit Carve(void *base) : base_(static_cast<uint8_t *>(base)) {}
    template <typename T>
    T *take(size_t count) {
        const size_t at = used_;
        used_ += (count * sizeof(T) + 255) & ~size_t(255);
        return base_ ? reinterpret_cast<T *>(base_ + at) : nullptr;
    }
    size_t used() const { return used_; }

  private:
    uint8_t *base_;
    size_t used_ = 0;
};

// the caller's scratch, or the library's own for this call (`own`; the call then waits before it is freed)
inline int scratch_of(void *ws, uint64_t ws_bytes, size_t need, DevBuf<uint8_t> &own, void **base) {
    if (!ws) {
        CZ_HIP(own.alloc(need));
        *base = own.p;
        return CZ_OK;
    }
    if (reinterpret_cast<uintptr_t>(ws) & 255) return set_error(CZ_E_INVALID, "ws is not 256-byte aligned");
    if (ws_bytes < need) return set_error(CZ_E_INVALID, "ws holds %llu bytes, %llu are needed", (unsigned long long)ws_bytes, (unsigned long long)need);
    *base = ws;
    return check_device_ptr(ws, "ws");
}

}  // namespace cz
