// A device without a GPU, for tests of slc_dispatch's checks: linked with the
// library's own objects (device.cpp, ops.cpp and the launchers) in the place
// of its capture layer. Every command is validated by the library's code and
// then counts as recorded, so nothing is ever launched; buffers have an
// address range that is never touched and, for U32, their host shadow.
#include <string.h>

#include "device_internal.h"

namespace {
uint64_t recorded = 0;
uintptr_t next_address = 1ull << 40;
}  // namespace

int flush_capture(slc_device *) { return SLC_OK; }
void release_capture(slc_device *) {}
void invalidate_capture(slc_device *) {}
int capture_record(slc_device *, const slc_op *, const slc_buffer_ref *, const slc_value *, uint64_t,
                   const slc_buffer_ref *, const slc_value *, uint64_t, const uint32_t *, uint64_t) {
    recorded++;
    return 1;
}

extern "C" __attribute__((visibility("default"))) slc_device *host_device_new() {
    slc_device *d = new slc_device();
    d->capture = reinterpret_cast<CaptureState *>(d);  // set: commands are validated, then recorded
    d->workspace_bytes = 256ull << 20;
    d->workspace = reinterpret_cast<char *>(next_address);
    next_address += d->workspace_bytes;
    return d;
}

extern "C" __attribute__((visibility("default"))) void host_device_free(slc_device *d) { delete d; }

extern "C" __attribute__((visibility("default"))) uint32_t host_buffer(slc_device *d, uint64_t elements,
                                                                       const uint32_t *data) {
    DeviceBuffer b;
    b.alloc = reinterpret_cast<void *>(next_address);
    b.ptr = reinterpret_cast<char *>(next_address);
    next_address += (elements * 4 + 511) / 256 * 256;
    b.elements = elements;
    b.u32 = data != nullptr;
    if (data) b.shadow.assign(data, data + elements);
    d->buffers.push_back(b);
    return (uint32_t)d->buffers.size() - 1;
}

extern "C" __attribute__((visibility("default"))) uint64_t host_recorded() { return recorded; }
