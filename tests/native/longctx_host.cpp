// The host side of the long-context entry points (zh_longctx.cpp) without a device: the HIP calls it makes and
// the launchers are stand-ins, and contexts and buffers are made of numbers.  Memory is never touched.
#include "../../ziggy-llm_amd/csrc/zh_longctx.cpp"

static int launches, current_device;
static struct {
    uintptr_t base;
    size_t size;
    int device;
} allocation = {0x10000000, 0x1000000, 0};

extern "C" {
hipError_t hipGetDevice(int *d) { return *d = current_device, hipSuccess; }
hipError_t hipSetDevice(int d) { return current_device = d, hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t *a, const void *p) {
    if ((uintptr_t)p < allocation.base || (uintptr_t)p >= allocation.base + allocation.size) return hipErrorInvalidValue;
    a->type = hipMemoryTypeDevice;
    a->device = allocation.device;
    return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t *b, size_t *n, hipDeviceptr_t) {
    *b = (hipDeviceptr_t)allocation.base;
    *n = allocation.size;
    return hipSuccess;
}

ZiggyHipContext *fake_context(int device, size_t scratch) {
    ZiggyHipContext *c = new ZiggyHipContext();
    c->device = device;
    c->scratch = (void *)0x1000;
    c->scratch_len = scratch;
    c->info.compute_units = 256;
    return c;
}
ZiggyHipBuffer *fake_buffer(ZiggyHipContext *c, int device, uintptr_t at, size_t len) {
    ZiggyHipBuffer *b = new ZiggyHipBuffer();
    b->ctx = c, b->device = device, b->ptr = (void *)at, b->len = len;
    return b;
}
int fake_launches(void) { return launches; }
int fake_device(void) { return current_device; }
}

namespace zh {
hipError_t launch_rope_rows(const RopeRows &, int, hipStream_t) { return launches++, hipSuccess; }
hipError_t launch_kv8_store(const Kv8Layer &, const float *, const float *, size_t, uint32_t, uint32_t, hipStream_t) {
    return launches++, hipSuccess;
}
hipError_t launch_kv8_load(const Kv8Layer &, float *, float *, uint32_t, uint32_t, hipStream_t) {
    return launches++, hipSuccess;
}
hipError_t launch_kv8_attention(const Kv8Attn &, int, hipStream_t) { return launches++, hipSuccess; }
hipError_t launch_sample_rows(const SampleRows &, hipStream_t) { return launches++, hipSuccess; }
size_t sample_rows_bytes(uint32_t vocab) { return (size_t)vocab * 8; }
}  // namespace zh
