// extern "C" surface declared in include/hayai_hip.h.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>

#include "engine.h"

namespace hh {
const std::string& last_error();
}
hh_status engine_create(int device, hh_engine** out);
void engine_destroy(hh_engine* e);

using namespace hh;

#define HH_NOT_NULL(p, what) \
    if (!(p)) return fail(HH_ERR_INVALID, "%s is NULL", what)

// [off, off + bytes) must lie inside the buffer.
static hh_status check_range(const hh_buf* b, size_t off, size_t bytes, const char* what) {
    if (!b) return fail(HH_ERR_INVALID, "%s: buffer is NULL", what);
    if (off > b->size || bytes > b->size - off)
        return fail(HH_ERR_INVALID, "%s: range [%zu, +%zu) outside a %zu-byte buffer", what, off, bytes, b->size);
    return HH_OK;
}

static hh_status check_engine(hh_engine* e, const hh_buf* b, const char* what) {
    if (b && b->engine != e) return fail(HH_ERR_INVALID, "%s: buffer belongs to another engine", what);
    return HH_OK;
}

struct hh_pending {
    hh_engine* engine;
    void* dx;
    void* dy;
    size_t m;
    hipEvent_t done;
    bool waited;
};

extern "C" {

int hh_abi_version(void) { return HH_ABI_VERSION; }

const char* hh_last_error(void) { return last_error().c_str(); }

const char* hh_status_name(hh_status st) {
    switch (st) {
    case HH_OK: return "HH_OK";
    case HH_ERR_NO_DEVICE: return "HH_ERR_NO_DEVICE";
    case HH_ERR_INVALID: return "HH_ERR_INVALID";
    case HH_ERR_KERNEL_MISSING: return "HH_ERR_KERNEL_MISSING";
    case HH_ERR_RUNTIME: return "HH_ERR_RUNTIME";
    case HH_ERR_OUT_OF_MEMORY: return "HH_ERR_OUT_OF_MEMORY";
    case HH_ERR_UNSUPPORTED_DEVICE: return "HH_ERR_UNSUPPORTED_DEVICE";
    case HH_ERR_IO: return "HH_ERR_IO";
    case HH_ERR_NOT_FOUND: return "HH_ERR_NOT_FOUND";
    }
    return "HH_ERR_UNKNOWN";
}

hh_status hh_row_bytes(int t, size_t n, size_t* out) {
    HH_NOT_NULL(out, "out");
    return row_bytes(t, n, out);
}

hh_status hh_validate_gemv_shape(int t, size_t m, size_t n) { return validate_shape(t, m, n); }

hh_status hh_validate_gemv_weights(int t, size_t m, size_t n, size_t len) { return validate_weights(t, m, n, len); }

hh_status hh_device_count(int* count) {
    HH_NOT_NULL(count, "count");
    *count = 0;
    hipError_t err = hipGetDeviceCount(count);
    if (err == hipErrorNoDevice) {
        *count = 0;
        return HH_OK;
    }
    if (err != hipSuccess) return hip_fail(err, "hipGetDeviceCount");
    return HH_OK;
}

hh_status hh_engine_create(int device, hh_engine** out) {
    HH_NOT_NULL(out, "out");
    try {
        return engine_create(device, out);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

void hh_engine_destroy(hh_engine* e) { engine_destroy(e); }

hh_status hh_engine_info(const hh_engine* e, hh_device_info* out) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(out, "out");
    memset(out, 0, sizeof *out);
    snprintf(out->name, sizeof out->name, "%s", e->props.name);
    snprintf(out->arch, sizeof out->arch, "%s", e->props.gcnArchName);
    out->device_index = e->device;
    out->compute_units = e->props.multiProcessorCount;
    out->wavefront_size = e->props.warpSize;
    out->clock_khz = e->props.clockRate;
    out->memory_clock_khz = e->props.memoryClockRate;
    out->memory_bus_width = e->props.memoryBusWidth;
    out->total_mem = e->props.totalGlobalMem;
    out->lds_per_block = e->props.sharedMemPerBlock;
    out->l2_bytes = (size_t)e->props.l2CacheSize;
    return HH_OK;
}

hh_status hh_engine_sync(hh_engine* e) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->select());
    HH_TRY_HIP(hipStreamSynchronize(e->stream), "hipStreamSynchronize(compute)");
    HH_TRY_HIP(hipStreamSynchronize(e->copy_stream), "hipStreamSynchronize(copy)");
    return e->check_device_error();
}

hh_status hh_engine_stream(hh_engine* e, void** stream) {
    HH_NOT_NULL(stream, "stream");
    *stream = nullptr;
    HH_NOT_NULL(e, "engine");
    *stream = e->stream;
    return HH_OK;
}

uint64_t hh_engine_ffn_calls(const hh_engine* e) { return e ? e->ffn_calls.load() : 0; }

// ---------------------------------------------------------------- buffers ------------

hh_status hh_buf_alloc(hh_engine* e, size_t bytes, int kind, hh_buf** out) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(out, "out");
    *out = nullptr;
    if (kind != HH_BUF_DEVICE && kind != HH_BUF_PINNED_HOST) return fail(HH_ERR_INVALID, "unknown buffer kind %d", kind);
    HH_TRY(e->select());
    void* p = nullptr;
    const size_t sz = std::max<size_t>(bytes, 1);
    if (kind == HH_BUF_DEVICE) {
        HH_TRY_HIP(hipMalloc(&p, sz), "hipMalloc");
    } else {
        HH_TRY_HIP(hipHostMalloc(&p, sz, hipHostMallocDefault), "hipHostMalloc");
    }
    hh_buf* b = new (std::nothrow) hh_buf{e, p, bytes, kind};
    if (!b) {
        if (kind == HH_BUF_DEVICE)
            (void)hipFree(p);
        else
            (void)hipHostFree(p);
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
    *out = b;
    return HH_OK;
}

hh_status hh_buf_wrap(hh_engine* e, void* ptr, size_t bytes, hh_buf** out) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(out, "out");
    *out = nullptr;
    HH_NOT_NULL(ptr, "ptr");
    HH_TRY(e->no_capture("buf_wrap"));
    HH_TRY(e->select());
    hipPointerAttribute_t at{};
    hipDeviceptr_t base = nullptr;
    size_t size = 0;
    if (hipPointerGetAttributes(&at, ptr) != hipSuccess || at.type != hipMemoryTypeDevice || at.device != e->device ||
        hipMemGetAddressRange(&base, &size, ptr) != hipSuccess) {
        (void)hipGetLastError();  // not a fault of the next call
        return fail(HH_ERR_INVALID, "hh_buf_wrap: not device memory of GPU %d", e->device);
    }
    const size_t at_off = (size_t)((char*)ptr - (char*)base);
    if (at_off > size || bytes > size - at_off)
        return fail(HH_ERR_INVALID, "hh_buf_wrap: %zu bytes reach past the allocation's end", bytes);
    hh_buf* b = new (std::nothrow) hh_buf{e, ptr, bytes, HH_BUF_DEVICE, true};
    if (!b) return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    *out = b;
    return HH_OK;
}

void hh_buf_free(hh_buf* b) {
    if (!b) return;
    (void)hipSetDevice(b->engine->device);
    // Work queued on the engine may still read the buffer.
    (void)hipStreamSynchronize(b->engine->stream);
    (void)hipStreamSynchronize(b->engine->copy_stream);
    if (b->borrowed) {
        delete b;
        return;
    }
    if (b->kind == HH_BUF_DEVICE)
        (void)hipFree(b->ptr);
    else
        (void)hipHostFree(b->ptr);
    delete b;
}

size_t hh_buf_size(const hh_buf* b) { return b ? b->size : 0; }

int hh_buf_kind(const hh_buf* b) { return b ? b->kind : -1; }

void* hh_buf_host_ptr(hh_buf* b) { return (b && b->kind == HH_BUF_PINNED_HOST) ? b->ptr : nullptr; }

hh_status hh_buf_write(hh_engine* e, hh_buf* dst, size_t off, const void* src, size_t bytes) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("buf_write"));
    HH_TRY(check_engine(e, dst, "hh_buf_write"));
    HH_TRY(check_range(dst, off, bytes, "hh_buf_write"));
    if (bytes == 0) return HH_OK;
    HH_NOT_NULL(src, "src");
    HH_TRY(e->select());
    HH_TRY_HIP(hipMemcpyAsync((char*)dst->ptr + off, src, bytes, hipMemcpyDefault, e->stream), "hipMemcpyAsync(H2D)");
    HH_TRY_HIP(hipStreamSynchronize(e->stream), "hipStreamSynchronize");
    return HH_OK;
}

hh_status hh_buf_read(hh_engine* e, const hh_buf* src, size_t off, void* dst, size_t bytes) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("buf_read"));
    HH_TRY(check_engine(e, src, "hh_buf_read"));
    HH_TRY(check_range(src, off, bytes, "hh_buf_read"));
    if (bytes == 0) return HH_OK;
    HH_NOT_NULL(dst, "dst");
    HH_TRY(e->select());
    HH_TRY_HIP(hipMemcpyAsync(dst, (const char*)src->ptr + off, bytes, hipMemcpyDefault, e->stream),
               "hipMemcpyAsync(D2H)");
    return e->check_device_error();  // syncs the stream
}

hh_status hh_buf_copy(hh_engine* e, hh_buf* dst, size_t dst_off, const hh_buf* src, size_t src_off, size_t bytes) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("buf_copy"));
    HH_TRY(check_engine(e, dst, "hh_buf_copy"));
    HH_TRY(check_engine(e, src, "hh_buf_copy"));
    HH_TRY(check_range(dst, dst_off, bytes, "hh_buf_copy dst"));
    HH_TRY(check_range(src, src_off, bytes, "hh_buf_copy src"));
    if (bytes == 0) return HH_OK;
    HH_TRY(e->select());
    HH_TRY_HIP(hipMemcpyAsync((char*)dst->ptr + dst_off, (const char*)src->ptr + src_off, bytes, hipMemcpyDefault,
                              e->stream),
               "hipMemcpyAsync(copy)");
    return HH_OK;
}

hh_status hh_buf_fill(hh_engine* e, hh_buf* dst, size_t off, uint8_t value, size_t bytes) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("buf_fill"));
    HH_TRY(check_engine(e, dst, "hh_buf_fill"));
    HH_TRY(check_range(dst, off, bytes, "hh_buf_fill"));
    if (bytes == 0) return HH_OK;
    HH_TRY(e->select());
    HH_TRY_HIP(hipMemsetAsync((char*)dst->ptr + off, value, bytes, e->stream), "hipMemsetAsync");
    return HH_OK;
}

// ---------------------------------------------------------------- GEMV ---------------

hh_status hh_gemv_dev(hh_engine* e, int t, size_t m, size_t n, const hh_buf* w, size_t w_off, const hh_buf* x,
                      size_t x_off, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_shape(t, m, n));
    size_t rb;
    HH_TRY(row_bytes(t, n, &rb));
    HH_TRY(check_engine(e, w, "weights"));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(w, w_off, m * rb, "weights"));
    HH_TRY(check_range(x, x_off, n * sizeof(float), "x"));
    HH_TRY(check_range(y, y_off, m * sizeof(float), "y"));
    HH_TRY(e->select());
    e->ffn_calls++;
    return e->enqueue_gemv(t, m, n, (const uint8_t*)w->ptr + w_off, (const float*)((const char*)x->ptr + x_off),
                           (float*)((char*)y->ptr + y_off));
}

static hh_status gemv_host_io(hh_engine* e, int t, size_t m, size_t n, const uint8_t* wdev, const float* x, float* y) {
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    HH_TRY(e->grow(&e->ws_x, &e->ws_x_cap, n * sizeof(float)));
    HH_TRY(e->grow(&e->ws_y, &e->ws_y_cap, m * sizeof(float)));
    HH_TRY_HIP(hipMemcpyAsync(e->ws_x, x, n * sizeof(float), hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(x)");
    e->ffn_calls++;
    HH_TRY(e->enqueue_gemv(t, m, n, wdev, (const float*)e->ws_x, (float*)e->ws_y));
    HH_TRY_HIP(hipMemcpyAsync(y, e->ws_y, m * sizeof(float), hipMemcpyDeviceToHost, e->stream), "hipMemcpyAsync(y)");
    HH_TRY_HIP(hipStreamSynchronize(e->stream), "hipStreamSynchronize");
    return HH_OK;
}

hh_status hh_gemv_bound(hh_engine* e, int t, size_t m, size_t n, const hh_buf* w, size_t w_off, const float* x,
                        float* y) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_shape(t, m, n));
    size_t rb;
    HH_TRY(row_bytes(t, n, &rb));
    HH_TRY(check_engine(e, w, "weights"));
    HH_TRY(check_range(w, w_off, m * rb, "weights"));
    HH_NOT_NULL(x, "x");
    HH_NOT_NULL(y, "y");
    HH_TRY(e->select());
    return gemv_host_io(e, t, m, n, (const uint8_t*)w->ptr + w_off, x, y);
}

hh_status hh_gemv(hh_engine* e, int t, size_t m, size_t n, const uint8_t* weights, size_t weights_len,
                  const float* x, float* y) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_shape(t, m, n));
    HH_TRY(validate_weights(t, m, n, weights_len));
    HH_NOT_NULL(weights, "weights");
    HH_NOT_NULL(x, "x");
    HH_NOT_NULL(y, "y");
    size_t rb;
    HH_TRY(row_bytes(t, n, &rb));
    HH_TRY(e->select());
    {
        std::lock_guard<std::mutex> lk(e->ws_mutex);
        HH_TRY(e->grow(&e->ws_w, &e->ws_w_cap, m * rb));
        HH_TRY_HIP(hipMemcpyAsync(e->ws_w, weights, m * rb, hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(w)");
    }
    return gemv_host_io(e, t, m, n, (const uint8_t*)e->ws_w, x, y);
}

static hh_status batch_bytes(size_t batch, size_t len, size_t* out) {
    if (len != 0 && batch > SIZE_MAX / (len * sizeof(float))) return fail(HH_ERR_INVALID, "batch size overflow");
    *out = batch * len * sizeof(float);
    return HH_OK;
}

hh_status hh_gemv_batched(hh_engine* e, int t, size_t m, size_t n, const uint8_t* weights, size_t weights_len,
                          const float* inputs, float* outputs, size_t batch) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_shape(t, m, n));
    HH_TRY(validate_weights(t, m, n, weights_len));
    size_t xb, yb, rb;
    HH_TRY(batch_bytes(batch, n, &xb));
    HH_TRY(batch_bytes(batch, m, &yb));
    HH_TRY(row_bytes(t, n, &rb));
    if (batch == 0) return HH_OK;
    HH_NOT_NULL(weights, "weights");
    HH_NOT_NULL(inputs, "inputs");
    HH_NOT_NULL(outputs, "outputs");
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    HH_TRY(e->grow(&e->ws_w, &e->ws_w_cap, m * rb));
    HH_TRY(e->grow(&e->ws_x, &e->ws_x_cap, xb));
    HH_TRY(e->grow(&e->ws_y, &e->ws_y_cap, yb));
    HH_TRY_HIP(hipMemcpyAsync(e->ws_w, weights, m * rb, hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(w)");
    HH_TRY_HIP(hipMemcpyAsync(e->ws_x, inputs, xb, hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(x)");
    HH_TRY(e->enqueue_gemv_batched(t, m, n, (const uint8_t*)e->ws_w, (const float*)e->ws_x, batch, (float*)e->ws_y));
    HH_TRY_HIP(hipMemcpyAsync(outputs, e->ws_y, yb, hipMemcpyDeviceToHost, e->stream), "hipMemcpyAsync(y)");
    return e->check_device_error();
}

hh_status hh_gemv_batched_dev(hh_engine* e, int t, size_t m, size_t n, const hh_buf* w, size_t w_off, const hh_buf* x,
                              size_t x_off, size_t batch, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("gemv_batched_dev"));
    HH_TRY(validate_shape(t, m, n));
    size_t xb, yb, rb;
    HH_TRY(batch_bytes(batch, n, &xb));
    HH_TRY(batch_bytes(batch, m, &yb));
    HH_TRY(row_bytes(t, n, &rb));
    HH_TRY(check_engine(e, w, "weights"));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(w, w_off, m * rb, "weights"));
    HH_TRY(check_range(x, x_off, xb, "x"));
    HH_TRY(check_range(y, y_off, yb, "y"));
    if (((x_off | y_off) & 3u) != 0) return fail(HH_ERR_INVALID, "gemv_batched: x/y offsets must be 4-byte aligned");
    if (batch == 0) return HH_OK;
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_gemv_batched(t, m, n, (const uint8_t*)w->ptr + w_off, (const float*)((const char*)x->ptr + x_off),
                                   batch, (float*)((char*)y->ptr + y_off));
}

hh_status hh_gemv_begin(hh_engine* e, int t, size_t m, size_t n, const hh_buf* w, size_t w_off, const float* x,
                        hh_pending** out) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(out, "out");
    *out = nullptr;
    HH_TRY(validate_shape(t, m, n));
    size_t rb;
    HH_TRY(row_bytes(t, n, &rb));
    HH_TRY(check_engine(e, w, "weights"));
    HH_TRY(check_range(w, w_off, m * rb, "weights"));
    HH_NOT_NULL(x, "x");
    HH_TRY(e->select());
    hh_pending* p = new (std::nothrow) hh_pending{e, nullptr, nullptr, m, nullptr, false};
    if (!p) return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    auto bail = [&](hh_status st) {
        if (p->dx) (void)hipFree(p->dx);
        if (p->dy) (void)hipFree(p->dy);
        if (p->done) (void)hipEventDestroy(p->done);
        delete p;
        return st;
    };
    hipError_t err = hipMalloc(&p->dx, n * sizeof(float));
    if (err == hipSuccess) err = hipMalloc(&p->dy, m * sizeof(float));
    if (err == hipSuccess) err = hipEventCreateWithFlags(&p->done, hipEventDisableTiming);
    if (err == hipSuccess) err = hipMemcpyAsync(p->dx, x, n * sizeof(float), hipMemcpyHostToDevice, e->stream);
    if (err != hipSuccess) return bail(hip_fail(err, "hh_gemv_begin"));
    e->ffn_calls++;
    hh_status st = e->enqueue_gemv(t, m, n, (const uint8_t*)w->ptr + w_off, (const float*)p->dx, (float*)p->dy);
    if (st != HH_OK) {
        (void)hipStreamSynchronize(e->stream);
        return bail(st);
    }
    err = hipEventRecord(p->done, e->stream);
    if (err != hipSuccess) {
        (void)hipStreamSynchronize(e->stream);
        return bail(hip_fail(err, "hipEventRecord"));
    }
    *out = p;
    return HH_OK;
}

hh_status hh_pending_wait(hh_pending* p, float* y, size_t m) {
    HH_NOT_NULL(p, "pending");
    HH_NOT_NULL(y, "y");
    if (m < p->m) return fail(HH_ERR_INVALID, "hh_pending_wait: output holds %zu < %zu floats", m, p->m);
    HH_TRY(p->engine->select());
    HH_TRY_HIP(hipEventSynchronize(p->done), "hipEventSynchronize");
    p->waited = true;
    HH_TRY_HIP(hipMemcpy(y, p->dy, p->m * sizeof(float), hipMemcpyDeviceToHost), "hipMemcpy(y)");
    return HH_OK;
}

void hh_pending_destroy(hh_pending* p) {
    if (!p) return;
    (void)hipSetDevice(p->engine->device);
    (void)hipEventSynchronize(p->done);  // never free buffers a queued kernel still uses
    (void)hipFree(p->dx);
    (void)hipFree(p->dy);
    (void)hipEventDestroy(p->done);
    delete p;
}

// ---------------------------------------------------------------- Q4 LUT GEMV ------

// The reference asserts these (compute.rs:54-58, matmul.rs:61-66); here they are status codes.
static hh_status lut_shape(size_t m, size_t n) {
    if (m == 0 || n == 0) return fail(HH_ERR_INVALID, "lut_matmul_q4: empty shape m=%zu n=%zu", m, n);
    if (n % 2 != 0) return fail(HH_ERR_INVALID, "lut_matmul_q4: N must be even for packed Q4 weights (n=%zu)", n);
    if (m > SIZE_MAX / (n / 2)) return fail(HH_ERR_INVALID, "lut_matmul_q4: weight size overflow");
    return HH_OK;
}

hh_status hh_lut_gemv(hh_engine* e, size_t m, size_t n, const uint8_t* weights_q4, size_t weights_len,
                      const float* lut, const float* x, float* y) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(lut_shape(m, n));
    HH_NOT_NULL(weights_q4, "weights_q4");
    HH_NOT_NULL(lut, "lut");
    HH_NOT_NULL(x, "x");
    HH_NOT_NULL(y, "y");
    const size_t wb = m * (n / 2);
    if (weights_len != wb)
        return fail(HH_ERR_INVALID, "lut_matmul_q4: weights_q4 has %zu bytes, expected m*n/2 = %zu", weights_len, wb);
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    // one staging buffer: [lut 64 B][x n*4 B][weights], x 16-byte aligned
    const size_t xo = 64, wo = xo + ((n * sizeof(float) + 255) / 256) * 256;
    HH_TRY(e->grow(&e->ws_w, &e->ws_w_cap, wo + wb));
    HH_TRY(e->grow(&e->ws_y, &e->ws_y_cap, m * sizeof(float)));
    char* base = (char*)e->ws_w;
    HH_TRY_HIP(hipMemcpyAsync(base, lut, 16 * sizeof(float), hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(lut)");
    HH_TRY_HIP(hipMemcpyAsync(base + xo, x, n * sizeof(float), hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(x)");
    HH_TRY_HIP(hipMemcpyAsync(base + wo, weights_q4, wb, hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(w)");
    HH_TRY(e->enqueue_lut(m, n, (const uint8_t*)(base + wo), (const float*)base, (const float*)(base + xo),
                          (float*)e->ws_y));
    HH_TRY_HIP(hipMemcpyAsync(y, e->ws_y, m * sizeof(float), hipMemcpyDeviceToHost, e->stream), "hipMemcpyAsync(y)");
    HH_TRY_HIP(hipStreamSynchronize(e->stream), "hipStreamSynchronize");
    return HH_OK;
}

hh_status hh_lut_gemv_dev(hh_engine* e, size_t m, size_t n, const hh_buf* w, size_t w_off, const hh_buf* lut,
                          size_t lut_off, const hh_buf* x, size_t x_off, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(lut_shape(m, n));
    HH_TRY(check_engine(e, w, "weights"));
    HH_TRY(check_engine(e, lut, "lut"));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(w, w_off, m * (n / 2), "weights"));
    HH_TRY(check_range(lut, lut_off, 16 * sizeof(float), "lut"));
    HH_TRY(check_range(x, x_off, n * sizeof(float), "x"));
    HH_TRY(check_range(y, y_off, m * sizeof(float), "y"));
    if (lut_off % 4 || x_off % 4 || y_off % 4) return fail(HH_ERR_INVALID, "lut_matmul_q4: f32 offsets must be 4-byte aligned");
    HH_TRY(e->select());
    return e->enqueue_lut(m, n, (const uint8_t*)w->ptr + w_off, (const float*)((const char*)lut->ptr + lut_off),
                          (const float*)((const char*)x->ptr + x_off), (float*)((char*)y->ptr + y_off));
}

hh_status hh_dequant_dev(hh_engine* e, int t, const hh_buf* w, size_t w_off, size_t n, hh_buf* out, size_t out_off) {
    HH_NOT_NULL(e, "engine");
    const Format* f = format_of(t);
    if (!f || t == HH_TYPE_F32) return fail(HH_ERR_KERNEL_MISSING, "no dequant kernel for GGML type %d", t);
    if (t != HH_TYPE_Q4_0 && t != HH_TYPE_Q8_0 && n % f->block != 0)
        return fail(HH_ERR_INVALID, "dequant_%s: n=%zu not a multiple of %u", f->name, n, f->block);
    const size_t nblk = (n + f->block - 1) / f->block;
    HH_TRY(check_engine(e, w, "weights"));
    HH_TRY(check_engine(e, out, "out"));
    HH_TRY(check_range(w, w_off, nblk * f->bytes, "weights"));
    HH_TRY(check_range(out, out_off, n * sizeof(float), "out"));
    if ((w_off & 1u) || (out_off & 3u)) return fail(HH_ERR_INVALID, "dequant_%s: misaligned offsets", f->name);
    if (n == 0) return HH_OK;
    HH_TRY(e->select());
    hipFunction_t fn;
    HH_TRY(e->kernel(std::string("hh_dequant_") + f->name, &fn));
    hh_dequant_args a{(const uint8_t*)w->ptr + w_off, (float*)((char*)out->ptr + out_off), (uint64_t)n};
    const size_t threads = t == HH_TYPE_F16 ? n : nblk;
    return e->launch(fn, (uint32_t)((threads + 255) / 256), 256, a);
}

// ---------------------------------------------------------------- FFN ----------------

static hh_status validate_ffn(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off) {
    HH_NOT_NULL(d, "desc");
    if (d->act != HH_ACT_SILU && d->act != HH_ACT_GELU_TANH) return fail(HH_ERR_INVALID, "ffn: unknown act %d", d->act);
    HH_TRY(validate_shape(d->type_gate, d->d_ff, d->d_model));
    HH_TRY(validate_shape(d->type_up, d->d_ff, d->d_model));
    HH_TRY(validate_shape(d->type_down, d->d_model, d->d_ff));
    size_t rg, ru, rd;
    HH_TRY(row_bytes(d->type_gate, d->d_model, &rg));
    HH_TRY(row_bytes(d->type_up, d->d_model, &ru));
    HH_TRY(row_bytes(d->type_down, d->d_ff, &rd));
    HH_TRY(check_engine(e, pack, "pack"));
    if (pack_off > pack->size) return fail(HH_ERR_INVALID, "ffn: pack offset outside the buffer");
    HH_TRY(check_range(pack, pack_off + d->gate_off, d->d_ff * rg, "ffn gate"));
    HH_TRY(check_range(pack, pack_off + d->up_off, d->d_ff * ru, "ffn up"));
    HH_TRY(check_range(pack, pack_off + d->down_off, d->d_model * rd, "ffn down"));
    return HH_OK;
}

hh_status hh_ffn_dev(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off, const hh_buf* x,
                     size_t x_off, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(x, x_off, d->d_model * sizeof(float), "x"));
    HH_TRY(check_range(y, y_off, d->d_model * sizeof(float), "y"));
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn(d, (const uint8_t*)pack->ptr + pack_off, (const float*)((const char*)x->ptr + x_off),
                          (float*)((char*)y->ptr + y_off));
}

hh_status hh_ffn_dev_noalloc(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off,
                             const hh_buf* x, size_t x_off, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(x, x_off, d->d_model * sizeof(float), "x"));
    HH_TRY(check_range(y, y_off, d->d_model * sizeof(float), "y"));
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn_noalloc(d, (const uint8_t*)pack->ptr + pack_off,
                                  (const float*)((const char*)x->ptr + x_off), (float*)((char*)y->ptr + y_off));
}

hh_status hh_ffn_block_dev(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off,
                           const hh_buf* norm, size_t norm_off, float eps, const hh_buf* x, size_t x_off, hh_buf* y,
                           size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_TRY(check_engine(e, norm, "norm"));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(norm, norm_off, d->d_model * sizeof(float), "norm"));
    HH_TRY(check_range(x, x_off, d->d_model * sizeof(float), "x"));
    HH_TRY(check_range(y, y_off, d->d_model * sizeof(float), "y"));
    if (((norm_off | x_off | y_off) & 3u) != 0)
        return fail(HH_ERR_INVALID, "ffn_block: norm/x/y offsets must be 4-byte aligned");
    if (!(eps >= 0.f) || eps > 1.f) return fail(HH_ERR_INVALID, "ffn_block: eps=%g outside [0, 1]", (double)eps);
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn_block(d, (const uint8_t*)pack->ptr + pack_off,
                                (const float*)((const char*)x->ptr + x_off),
                                (const float*)((const char*)norm->ptr + norm_off), eps,
                                (float*)((char*)y->ptr + y_off));
}

hh_status hh_ffn_block_stack_dev(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off,
                                 size_t layer_stride, size_t n_layers, const hh_buf* norm, size_t norm_off,
                                 size_t norm_stride, float eps, const hh_buf* x, size_t x_off, hh_buf* y,
                                 size_t y_off) {
    HH_NOT_NULL(e, "engine");
    if (n_layers == 0) return fail(HH_ERR_INVALID, "ffn_block_stack: n_layers must be at least 1");
    size_t last_pack, last_norm;
    if (__builtin_mul_overflow(n_layers - 1, layer_stride, &last_pack) ||
        __builtin_add_overflow(last_pack, pack_off, &last_pack) ||
        __builtin_mul_overflow(n_layers - 1, norm_stride, &last_norm) ||
        __builtin_mul_overflow(last_norm, sizeof(float), &last_norm) ||
        __builtin_add_overflow(last_norm, norm_off, &last_norm))
        return fail(HH_ERR_INVALID, "ffn_block_stack: layer offsets overflow");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_TRY(validate_ffn(e, d, pack, last_pack));  // layers lie between the first and the last
    HH_TRY(check_engine(e, norm, "norm"));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(norm, norm_off, d->d_model * sizeof(float), "norm"));
    HH_TRY(check_range(norm, last_norm, d->d_model * sizeof(float), "norm"));
    HH_TRY(check_range(x, x_off, d->d_model * sizeof(float), "x"));
    HH_TRY(check_range(y, y_off, d->d_model * sizeof(float), "y"));
    if (((norm_off | x_off | y_off) & 3u) != 0)
        return fail(HH_ERR_INVALID, "ffn_block_stack: norm/x/y offsets must be 4-byte aligned");
    if (!(eps >= 0.f) || eps > 1.f)
        return fail(HH_ERR_INVALID, "ffn_block_stack: eps=%g outside [0, 1]", (double)eps);
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn_block_stack(d, (const uint8_t*)pack->ptr + pack_off, layer_stride, n_layers,
                                      (const float*)((const char*)norm->ptr + norm_off), norm_stride, eps,
                                      (const float*)((const char*)x->ptr + x_off), (float*)((char*)y->ptr + y_off));
}

hh_status hh_ffn_batched_dev(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off, const hh_buf* x,
                             size_t x_off, size_t batch, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("ffn_batched_dev"));
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    size_t xb;
    HH_TRY(batch_bytes(batch, d->d_model, &xb));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(x, x_off, xb, "x"));
    HH_TRY(check_range(y, y_off, xb, "y"));
    if (((x_off | y_off) & 3u) != 0) return fail(HH_ERR_INVALID, "ffn_batched: x/y offsets must be 4-byte aligned");
    if (batch == 0) return HH_OK;
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn_batched(d, (const uint8_t*)pack->ptr + pack_off, (const float*)((const char*)x->ptr + x_off),
                                  batch, (float*)((char*)y->ptr + y_off));
}

hh_status hh_ffn_batched(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off, const float* x,
                         float* y, size_t batch) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    size_t xb;
    HH_TRY(batch_bytes(batch, d->d_model, &xb));
    if (batch == 0) return HH_OK;
    HH_NOT_NULL(x, "x");
    HH_NOT_NULL(y, "y");
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    HH_TRY(e->grow(&e->ws_x, &e->ws_x_cap, xb));
    HH_TRY(e->grow(&e->ws_y, &e->ws_y_cap, xb));
    HH_TRY_HIP(hipMemcpyAsync(e->ws_x, x, xb, hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(x)");
    HH_TRY(e->enqueue_ffn_batched(d, (const uint8_t*)pack->ptr + pack_off, (const float*)e->ws_x, batch,
                                  (float*)e->ws_y));
    HH_TRY_HIP(hipMemcpyAsync(y, e->ws_y, xb, hipMemcpyDeviceToHost, e->stream), "hipMemcpyAsync(y)");
    return e->check_device_error();
}

hh_status hh_ffn_begin_dev(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off, const hh_buf* x,
                           size_t x_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_range(x, x_off, d->d_model * sizeof(float), "x"));
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn_begin(d, (const uint8_t*)pack->ptr + pack_off, (const float*)((const char*)x->ptr + x_off));
}

hh_status hh_ffn_finish_dev(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off, hh_buf* y,
                            size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(y, y_off, d->d_model * sizeof(float), "y"));
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn_finish(d, (const uint8_t*)pack->ptr + pack_off, (float*)((char*)y->ptr + y_off));
}

hh_status hh_ffn_block_begin_dev(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off,
                                 const hh_buf* norm, size_t norm_off, float eps, const hh_buf* x, size_t x_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_TRY(check_engine(e, norm, "norm"));
    HH_TRY(check_engine(e, x, "x"));
    HH_TRY(check_range(norm, norm_off, d->d_model * sizeof(float), "norm"));
    HH_TRY(check_range(x, x_off, d->d_model * sizeof(float), "x"));
    if (((norm_off | x_off) & 3u) != 0) return fail(HH_ERR_INVALID, "ffn_block_begin: norm/x offsets must be 4-byte aligned");
    if (!(eps >= 0.f) || eps > 1.f) return fail(HH_ERR_INVALID, "ffn_block_begin: eps=%g outside [0, 1]", (double)eps);
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn_begin(d, (const uint8_t*)pack->ptr + pack_off, (const float*)((const char*)x->ptr + x_off),
                                (const float*)((const char*)norm->ptr + norm_off), eps);
}

hh_status hh_ffn_block_finish_dev(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off,
                                  const hh_buf* res, size_t res_off, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_TRY(check_engine(e, res, "res"));
    HH_TRY(check_engine(e, y, "y"));
    HH_TRY(check_range(res, res_off, d->d_model * sizeof(float), "res"));
    HH_TRY(check_range(y, y_off, d->d_model * sizeof(float), "y"));
    if (((res_off | y_off) & 3u) != 0) return fail(HH_ERR_INVALID, "ffn_block_finish: res/y offsets must be 4-byte aligned");
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    return e->enqueue_ffn_finish(d, (const uint8_t*)pack->ptr + pack_off, (float*)((char*)y->ptr + y_off),
                                 (const float*)((const char*)res->ptr + res_off));
}

hh_status hh_ffn(hh_engine* e, const hh_ffn_desc* d, const hh_buf* pack, size_t pack_off, const float* x, float* y) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_ffn(e, d, pack, pack_off));
    HH_NOT_NULL(x, "x");
    HH_NOT_NULL(y, "y");
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    HH_TRY(e->grow(&e->ws_x, &e->ws_x_cap, d->d_model * sizeof(float)));
    HH_TRY(e->grow(&e->ws_y, &e->ws_y_cap, d->d_model * sizeof(float)));
    HH_TRY_HIP(hipMemcpyAsync(e->ws_x, x, d->d_model * sizeof(float), hipMemcpyHostToDevice, e->stream),
               "hipMemcpyAsync(x)");
    HH_TRY(e->enqueue_ffn(d, (const uint8_t*)pack->ptr + pack_off, (const float*)e->ws_x, (float*)e->ws_y));
    HH_TRY_HIP(hipMemcpyAsync(y, e->ws_y, d->d_model * sizeof(float), hipMemcpyDeviceToHost, e->stream),
               "hipMemcpyAsync(y)");
    return e->check_device_error();
}

hh_status hh_gateup_dev(hh_engine* e, int tg, int tu, size_t d_ff, size_t d_model, const hh_buf* wg, size_t wg_off,
                        const hh_buf* wu, size_t wu_off, const hh_buf* x, size_t x_off, hh_buf* h, size_t h_off,
                        int act) {
    HH_NOT_NULL(e, "engine");
    if (act != HH_ACT_SILU && act != HH_ACT_GELU_TANH) return fail(HH_ERR_INVALID, "gateup: unknown act %d", act);
    HH_TRY(validate_shape(tg, d_ff, d_model));
    HH_TRY(validate_shape(tu, d_ff, d_model));
    size_t rg, ru;
    HH_TRY(row_bytes(tg, d_model, &rg));
    HH_TRY(row_bytes(tu, d_model, &ru));
    for (const hh_buf* b : {wg, wu, (const hh_buf*)x, (const hh_buf*)h}) HH_TRY(check_engine(e, b, "gateup"));
    HH_TRY(check_range(wg, wg_off, d_ff * rg, "gate"));
    HH_TRY(check_range(wu, wu_off, d_ff * ru, "up"));
    HH_TRY(check_range(x, x_off, d_model * sizeof(float), "x"));
    HH_TRY(check_range(h, h_off, d_ff * sizeof(float), "h"));
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    e->ffn_calls += 2;
    return e->enqueue_gateup(tg, tu, d_ff, d_model, (const uint8_t*)wg->ptr + wg_off, (const uint8_t*)wu->ptr + wu_off,
                             (const float*)((const char*)x->ptr + x_off), (float*)((char*)h->ptr + h_off), act);
}

// ---------------------------------------------------------------- 8-bit path ---------

static hh_status check_act_type(int type, const char* what) {
    if (!act_type(type)) return fail(HH_ERR_KERNEL_MISSING, "%s: no kernel for activations of GGML type %d", what, type);
    return HH_OK;
}

// A matrix of `rows` rows of `cols` elements of `elem` bytes, *stride elements apart (0: packed,
// filled in), in a device-visible buffer of the engine; whole: the last row has its whole stride too.
static hh_status check_rows(hh_engine* e, const hh_buf* b, size_t off, size_t rows, size_t cols, size_t elem,
                            size_t* stride, const char* what, bool whole = false) {
    HH_TRY(check_engine(e, b, what));
    if (*stride == 0) *stride = cols;
    if (*stride < cols) return fail(HH_ERR_INVALID, "%s: stride %zu < %zu columns", what, *stride, cols);
    if (*stride > SIZE_MAX / elem / (rows ? rows : 1)) return fail(HH_ERR_INVALID, "%s: size overflow", what);
    const size_t bytes = rows ? ((rows - 1) * *stride + (whole ? *stride : cols)) * elem : 0;
    HH_TRY(check_range(b, off, bytes, what));
    if (((uintptr_t)b->ptr + off) % elem) return fail(HH_ERR_INVALID, "%s: offset %zu splits an element", what, off);
    return HH_OK;
}

static hh_status check_vector(hh_engine* e, const hh_buf* b, size_t off, size_t n, const char* what) {
    size_t stride = 0;
    return check_rows(e, b, off, 1, n, 4, &stride, what);
}

// Grids and row indexes are 32 bits; columns are addressed in 32 bits with room for a vector past the end.
static hh_status check_sizes(size_t rows, size_t cols, const char* what) {
    if (cols == 0) return fail(HH_ERR_INVALID, "%s: rows of no columns", what);
    if (rows > INT32_MAX || cols > INT32_MAX)
        return fail(HH_ERR_INVALID, "%s: %zu x %zu exceeds 31-bit sizes", what, rows, cols);
    return HH_OK;
}

static void* at(const hh_buf* b, size_t off) { return b ? (char*)b->ptr + off : nullptr; }

hh_status hh_quant_i8_dev(hh_engine* e, const hh_quant_i8_desc* d, const hh_buf* x, size_t x_off, const hh_buf* up,
                          size_t up_off, hh_buf* q, size_t q_off, hh_buf* scale, size_t scale_off, hh_buf* values,
                          size_t values_off) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(d, "quant_i8 desc");
    HH_TRY(check_act_type(d->type, "quant_i8"));
    HH_TRY(check_sizes(d->rows, d->cols, "quant_i8"));
    if (up && d->act != HH_ACT_SILU && d->act != HH_ACT_GELU_TANH)
        return fail(HH_ERR_INVALID, "quant_i8: unknown act %d", d->act);
    const size_t el = act_type(d->type)->bytes;
    size_t xs = d->x_stride, us = d->up_stride, qs = d->q_stride, vs = 0;
    HH_TRY(check_rows(e, x, x_off, d->rows, d->cols, el, &xs, "quant_i8 x"));
    if (up) HH_TRY(check_rows(e, up, up_off, d->rows, d->cols, el, &us, "quant_i8 up"));
    HH_TRY(check_rows(e, q, q_off, d->rows, d->cols, 1, &qs, "quant_i8 q"));
    HH_TRY(check_vector(e, scale, scale_off, d->rows, "quant_i8 scale"));
    if (values) HH_TRY(check_rows(e, values, values_off, d->rows, d->cols, 4, &vs, "quant_i8 values"));
    if (d->rows == 0) return HH_OK;
    HH_TRY(e->select());
    hh_i8_rows_args a{};
    a.x = at(x, x_off);
    a.b = at(up, up_off);
    a.q = (int8_t*)at(q, q_off);
    a.scale = (float*)at(scale, scale_off);
    a.values = (float*)at(values, values_off);
    a.x_stride = xs;
    a.b_stride = us;
    a.q_stride = qs;
    a.cols = (uint32_t)d->cols;
    a.act = d->act;
    try {
        return e->enqueue_i8_rows(d->type, d->rows, a);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

hh_status hh_rms_norm_i8_dev(hh_engine* e, const hh_rms_norm_i8_desc* d, const hh_buf* x, size_t x_off,
                             const hh_buf* res, size_t res_off, const hh_buf* norm, size_t norm_off, hh_buf* sum,
                             size_t sum_off, hh_buf* q, size_t q_off, hh_buf* scale, size_t scale_off, hh_buf* values,
                             size_t values_off) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(d, "rms_norm_i8 desc");
    HH_TRY(check_act_type(d->type, "rms_norm_i8"));
    HH_TRY(check_sizes(d->rows, d->cols, "rms_norm_i8"));
    if (!(d->eps >= 0.f) || d->eps > 1.f)
        return fail(HH_ERR_INVALID, "rms_norm_i8: eps=%g outside [0, 1]", (double)d->eps);
    if (!res != !sum) return fail(HH_ERR_INVALID, "rms_norm_i8: res and sum come together");
    const size_t el = act_type(d->type)->bytes;
    size_t xs = d->x_stride, rs = d->res_stride, ss = d->sum_stride, qs = d->q_stride, vs = 0;
    HH_TRY(check_rows(e, x, x_off, d->rows, d->cols, el, &xs, "rms_norm_i8 x"));
    if (res) {
        HH_TRY(check_rows(e, res, res_off, d->rows, d->cols, el, &rs, "rms_norm_i8 res"));
        HH_TRY(check_rows(e, sum, sum_off, d->rows, d->cols, el, &ss, "rms_norm_i8 sum"));
    }
    HH_TRY(check_vector(e, norm, norm_off, d->cols, "rms_norm_i8 norm"));
    HH_TRY(check_rows(e, q, q_off, d->rows, d->cols, 1, &qs, "rms_norm_i8 q"));
    HH_TRY(check_vector(e, scale, scale_off, d->rows, "rms_norm_i8 scale"));
    if (values) HH_TRY(check_rows(e, values, values_off, d->rows, d->cols, 4, &vs, "rms_norm_i8 values"));
    if (d->rows == 0) return HH_OK;
    HH_TRY(e->select());
    hh_i8_rows_args a{};
    a.x = at(x, x_off);
    a.b = at(res, res_off);
    a.norm = (const float*)at(norm, norm_off);
    a.sum = at(sum, sum_off);
    a.q = (int8_t*)at(q, q_off);
    a.scale = (float*)at(scale, scale_off);
    a.values = (float*)at(values, values_off);
    a.x_stride = xs;
    a.b_stride = rs;
    a.sum_stride = ss;
    a.q_stride = qs;
    a.cols = (uint32_t)d->cols;
    a.eps = d->eps;
    try {
        return e->enqueue_i8_rows(d->type, d->rows, a);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

hh_status hh_gemm_i8_dev(hh_engine* e, const hh_gemm_i8_desc* d, const hh_buf* w, size_t w_off, const hh_buf* w_scale,
                         size_t w_scale_off, const hh_buf* x, size_t x_off, const hh_buf* x_scale, size_t x_scale_off,
                         const hh_buf* res, size_t res_off, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(d, "gemm_i8 desc");
    HH_TRY(check_act_type(d->type, "gemm_i8"));
    HH_TRY(check_sizes(d->m, d->n, "gemm_i8"));
    if (d->m == 0) return fail(HH_ERR_INVALID, "gemm_i8: empty shape m=0 n=%zu", d->n);
    if (d->n > HH_I8_MAX_N)
        return fail(HH_ERR_INVALID, "gemm_i8: n=%zu > %u, sums could pass 32 bits", d->n, HH_I8_MAX_N);
    HH_TRY(check_sizes(d->tokens, d->m, "gemm_i8"));
    const size_t el = act_type(d->type)->bytes;
    size_t ws = d->w_stride, xs = d->x_stride, rs = d->res_stride, ys = d->y_stride;
    HH_TRY(check_rows(e, w, w_off, d->m, d->n, 1, &ws, "gemm_i8 w", true));
    HH_TRY(check_vector(e, w_scale, w_scale_off, d->m, "gemm_i8 w_scale"));
    HH_TRY(check_rows(e, x, x_off, d->tokens, d->n, 1, &xs, "gemm_i8 x", true));
    HH_TRY(check_vector(e, x_scale, x_scale_off, d->tokens, "gemm_i8 x_scale"));
    if (res) HH_TRY(check_rows(e, res, res_off, d->tokens, d->m, el, &rs, "gemm_i8 res"));
    HH_TRY(check_rows(e, y, y_off, d->tokens, d->m, el, &ys, "gemm_i8 y"));
    if ((((uintptr_t)w->ptr + w_off) | ((uintptr_t)x->ptr + x_off) | ws | xs) % 16)
        return fail(HH_ERR_INVALID, "gemm_i8: rows of codes must start on 16-byte boundaries (strides %zu, %zu)", ws, xs);
    if (d->tokens == 0) return HH_OK;
    HH_TRY(e->select());
    hh_i8_gemm_args a{};
    a.w = (const int8_t*)at(w, w_off);
    a.x = (const int8_t*)at(x, x_off);
    a.ws = (const float*)at(w_scale, w_scale_off);
    a.xs = (const float*)at(x_scale, x_scale_off);
    a.res = at(res, res_off);
    a.y = at(y, y_off);
    a.w_stride = ws;
    a.x_stride = xs;
    a.res_stride = rs;
    a.y_stride = ys;
    a.m = (uint32_t)d->m;
    a.n = (uint32_t)d->n;
    a.t = (uint32_t)d->tokens;
    try {
        std::lock_guard<std::mutex> lk(e->ws_mutex);
        return e->enqueue_i8_gemm(d->type, a);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

hh_status hh_sample_dev(hh_engine* e, const hh_sample_desc* d, const hh_buf* logits, size_t logits_off,
                        const hh_buf* params, size_t params_off, const hh_buf* u, size_t u_off, hh_buf* ids,
                        size_t ids_off, hh_buf* probs, size_t probs_off) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(d, "sample desc");
    HH_TRY(check_act_type(d->type, "sample"));
    HH_TRY(check_sizes(d->rows, d->vocab, "sample"));
    if (d->vocab > HH_SAMPLE_MAX_VOCAB)
        return fail(HH_ERR_INVALID, "sample: vocab=%zu > %u", d->vocab, HH_SAMPLE_MAX_VOCAB);
    size_t stride = d->stride;
    HH_TRY(check_rows(e, logits, logits_off, d->rows, d->vocab, act_type(d->type)->bytes, &stride, "sample logits"));
    HH_TRY(check_vector(e, params, params_off, d->rows * 4, "sample params"));
    HH_TRY(check_vector(e, u, u_off, d->rows, "sample u"));
    HH_TRY(check_vector(e, ids, ids_off, d->rows, "sample ids"));
    if (probs) HH_TRY(check_vector(e, probs, probs_off, d->rows, "sample probs"));
    if (d->rows == 0) return HH_OK;
    HH_TRY(e->select());
    hh_sample_args a{};
    a.x = at(logits, logits_off);
    a.params = at(params, params_off);
    a.u = (const float*)at(u, u_off);
    a.ids = (int32_t*)at(ids, ids_off);
    a.probs = (float*)at(probs, probs_off);
    a.stride = stride;
    a.vocab = (uint32_t)d->vocab;
    try {
        std::lock_guard<std::mutex> lk(e->ws_mutex);
        return e->enqueue_sample(d->type, d->rows, a);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

// ---------------------------------------------------------------- attention ----------

// Whether pages of two of `layers` caches have an element in common: page p of layer l begins at p * stride + l * layer_stride.
static bool layers_meet(size_t stride, size_t page, size_t n_pages, size_t layer_stride, size_t layers) {
    for (size_t l = 1; l < layers; l++) {  // layer l and the first one: every other pair lies like one of these
        const size_t p = l * layer_stride / stride, past = l * layer_stride % stride;
        if (p >= n_pages) return false;
        if (past < page || (p + 1 < n_pages && stride - past < page)) return true;
    }
    return false;
}

// The cache's pages in a device-visible buffer of the engine, `layers` caches *layer_stride elements apart.
static hh_status check_kv(hh_engine* e, const hh_kv_desc* kv, const hh_buf* cache, size_t off, size_t layers,
                          size_t* layer_stride, hh_kv_args* out, const char* what) {
    HH_NOT_NULL(kv, "kv desc");
    HH_TRY(check_act_type(kv->type, what));
    const size_t el = act_type(kv->type)->bytes;
    if (kv->kv_heads < 1 || kv->kv_heads > 1024)
        return fail(HH_ERR_INVALID, "%s: kv_heads=%zu outside 1..1024", what, kv->kv_heads);
    if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8)
        return fail(HH_ERR_INVALID, "%s: head_dim=%zu is no multiple of 8 in 8..256", what, kv->head_dim);
    if (kv->page_size < 16 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1)))
        return fail(HH_ERR_INVALID, "%s: page_size=%zu is no power of two in 16..256", what, kv->page_size);
    if (kv->n_pages < 1 || kv->n_pages > INT32_MAX / kv->page_size)
        return fail(HH_ERR_INVALID, "%s: %zu pages of %zu tokens", what, kv->n_pages, kv->page_size);
    const size_t page = 2 * kv->kv_heads * kv->head_dim * kv->page_size;
    const size_t stride = kv->page_stride ? kv->page_stride : page;
    if (stride < page) return fail(HH_ERR_INVALID, "%s: page_stride %zu < %zu elements of a page", what, stride, page);
    if (stride > SIZE_MAX / el / kv->n_pages) return fail(HH_ERR_INVALID, "%s: size overflow", what);
    if (*layer_stride == 0) *layer_stride = stride * kv->n_pages;
    HH_TRY(check_engine(e, cache, what));
    const size_t last = ((kv->n_pages - 1) * stride + page) * el;
    if (layers > 1 && *layer_stride > (SIZE_MAX - last) / el / (layers - 1))
        return fail(HH_ERR_INVALID, "%s: size overflow", what);
    if (layers_meet(stride, page, kv->n_pages, *layer_stride, layers))
        return fail(HH_ERR_INVALID, "%s: pages of %zu layers %zu elements apart overlap (page_stride %zu)", what, layers, *layer_stride,
                    stride);
    HH_TRY(check_range(cache, off, (layers - 1) * *layer_stride * el + last, what));
    if ((((uintptr_t)cache->ptr + off) | stride * el | (layers > 1 ? *layer_stride * el : 0)) % 16)
        return fail(HH_ERR_INVALID, "%s: pages must start on 16-byte boundaries (strides %zu, %zu)", what, stride,
                    *layer_stride);
    out->base = (uint8_t*)cache->ptr + off;
    out->stride = stride * el;
    out->pages = (uint32_t)kv->n_pages;
    out->shift = (uint32_t)__builtin_ctzll(kv->page_size);
    out->heads = (uint32_t)kv->kv_heads;
    out->dim = (uint32_t)kv->head_dim;
    return HH_OK;
}

static hh_status check_kv_type(int type, const hh_kv_desc* kv, const char* what) {
    HH_NOT_NULL(kv, "kv desc");
    HH_TRY(check_act_type(type, what));
    HH_TRY(check_act_type(kv->type, what));
    if (kv->type != type && type != HH_TYPE_F32)
        return fail(HH_ERR_KERNEL_MISSING, "%s: no kernel for activations of GGML type %d over a cache of type %d", what,
                    type, kv->type);
    return HH_OK;
}

hh_status hh_rope_kv_dev(hh_engine* e, const hh_rope_desc* d, const hh_kv_desc* kv, const hh_buf* q, size_t q_off,
                         const hh_buf* k, size_t k_off, const hh_buf* v, size_t v_off, const hh_buf* positions,
                         size_t positions_off, const hh_buf* slots, size_t slots_off, const hh_buf* factors,
                         size_t factors_off, hh_buf* out, size_t out_off, hh_buf* cache, size_t cache_off) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(d, "rope desc");
    HH_TRY(check_kv_type(d->type, kv, "rope_kv"));
    hh_rope_args a{};
    size_t layer = 0;
    HH_TRY(check_kv(e, kv, cache, cache_off, 1, &layer, &a.kv, "rope_kv cache"));
    if (d->layout != HH_ROPE_HALVES && d->layout != HH_ROPE_PAIRS)
        return fail(HH_ERR_INVALID, "rope_kv: unknown layout %d", d->layout);
    if (d->q_heads > 65535) return fail(HH_ERR_INVALID, "rope_kv: q_heads=%zu > 65535", d->q_heads);
    if (d->rot_dim > kv->head_dim || d->rot_dim % 2)
        return fail(HH_ERR_INVALID, "rope_kv: rot_dim=%zu is not even in 0..%zu", d->rot_dim, kv->head_dim);
    if (!(d->base > 0) || !std::isfinite(d->base) || !std::isfinite(d->mscale))
        return fail(HH_ERR_INVALID, "rope_kv: base=%g mscale=%g", d->base, (double)d->mscale);
    const size_t el = act_type(d->type)->bytes, cols = kv->kv_heads * kv->head_dim, qcols = d->q_heads * kv->head_dim;
    HH_TRY(check_sizes(d->tokens, cols, "rope_kv"));
    size_t qs = d->q_stride, ks = d->k_stride, vs = d->v_stride, os = d->out_stride;
    if (d->q_heads) {
        HH_TRY(check_rows(e, q, q_off, d->tokens, qcols, el, &qs, "rope_kv q"));
        HH_TRY(check_rows(e, out, out_off, d->tokens, qcols, el, &os, "rope_kv out"));
    }
    HH_TRY(check_rows(e, k, k_off, d->tokens, cols, el, &ks, "rope_kv k"));
    HH_TRY(check_rows(e, v, v_off, d->tokens, cols, el, &vs, "rope_kv v"));
    HH_TRY(check_vector(e, positions, positions_off, d->tokens, "rope_kv positions"));
    HH_TRY(check_vector(e, slots, slots_off, d->tokens, "rope_kv slots"));
    if (factors) HH_TRY(check_vector(e, factors, factors_off, d->rot_dim / 2, "rope_kv factors"));
    if (d->tokens == 0) return HH_OK;
    HH_TRY(e->select());
    a.q = at(q, q_off);
    a.k = at(k, k_off);
    a.v = at(v, v_off);
    a.out = at(out, out_off);
    a.positions = (const int32_t*)at(positions, positions_off);
    a.slots = (const int32_t*)at(slots, slots_off);
    a.factors = (const float*)at(factors, factors_off);
    a.q_stride = qs;
    a.k_stride = ks;
    a.v_stride = vs;
    a.out_stride = os;
    a.log2_base = std::log2(d->base);
    a.mscale = d->mscale;
    a.heads = (uint32_t)d->q_heads;
    a.rot = (uint32_t)d->rot_dim;
    try {
        return e->enqueue_rope(d->type, kv->type, d->layout, d->tokens, a);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

hh_status hh_rope_factors(int scaling, size_t rot_dim, double base, double scale, double trained, float* factors,
                          float* mscale) {
    HH_NOT_NULL(factors, "factors");
    if (scaling != HH_ROPE_LINEAR && scaling != HH_ROPE_BY_WAVELENGTH && scaling != HH_ROPE_YARN)
        return fail(HH_ERR_INVALID, "rope_factors: unknown scaling %d", scaling);
    if (rot_dim < 2 || rot_dim > 256 || rot_dim % 2)
        return fail(HH_ERR_INVALID, "rope_factors: rot_dim=%zu is not even in 2..256", rot_dim);
    if (!(base > 1) || !std::isfinite(base) || !(scale >= 1) || !std::isfinite(scale) || !(trained >= 1) ||
        !std::isfinite(trained))
        return fail(HH_ERR_INVALID, "rope_factors: base=%g scale=%g trained=%g", base, scale, trained);
    const double n = (double)(rot_dim / 2), tau = 6.283185307179586476925;
    // the pair that turns `times` times over the trained length
    auto pair_of = [&](double times) { return n * std::log(trained / (times * tau)) / std::log(base); };
    const double lo = std::min(std::max(std::floor(pair_of(32)), 0.0), (double)rot_dim - 1);
    const double hi = std::min(std::max(std::ceil(pair_of(1)), 0.0), (double)rot_dim - 1);
    for (size_t i = 0; i < rot_dim / 2; i++) {
        double f = scale;
        if (scaling == HH_ROPE_BY_WAVELENGTH) {
            const double turns = trained / (tau * std::pow(base, (double)i / n));
            const double s = std::min(std::max((turns - 1) / 3, 0.0), 1.0);
            f = 1 / ((1 - s) / scale + s);
        } else if (scaling == HH_ROPE_YARN) {
            const double r = std::min(std::max(((double)i - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
            f = 1 / ((1 - r) + r / scale);
        }
        factors[i] = (float)f;
    }
    if (mscale) *mscale = scaling == HH_ROPE_YARN ? (float)(1 + 0.1 * std::log(scale)) : 1.f;
    return HH_OK;
}

hh_status hh_kv_copy_dev(hh_engine* e, const hh_kv_desc* kv, size_t layers, size_t layer_stride, hh_buf* cache,
                         size_t cache_off, const hh_buf* moves, size_t moves_off, size_t n) {
    HH_NOT_NULL(e, "engine");
    if (layers < 1 || layers > 65535) return fail(HH_ERR_INVALID, "kv_copy: layers=%zu outside 1..65535", layers);
    hh_kv_copy_args a{};
    HH_TRY(check_kv(e, kv, cache, cache_off, layers, &layer_stride, &a.kv, "kv_copy cache"));
    if (n > INT32_MAX) return fail(HH_ERR_INVALID, "kv_copy: %zu moves exceed 31 bits", n);
    HH_TRY(check_vector(e, moves, moves_off, 2 * n, "kv_copy moves"));
    if (n == 0) return HH_OK;
    HH_TRY(e->select());
    a.moves = (const int32_t*)at(moves, moves_off);
    a.layer_stride = layer_stride * act_type(kv->type)->bytes;
    a.n = (uint32_t)n;
    a.chunks = (uint32_t)(2 * kv->kv_heads * kv->head_dim * kv->page_size * act_type(kv->type)->bytes / 16);
    try {
        return e->enqueue_kv_copy(layers, a);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

// What both attention calls check: heads, scale, activations, tables and lengths.
static hh_status check_attn(hh_engine* e, int type, float scale, size_t rows, size_t seqs, size_t q_heads, size_t entries,
                            const hh_kv_desc* kv, const hh_buf* q, size_t q_off, size_t* q_stride, const hh_buf* out,
                            size_t out_off, size_t* out_stride, const hh_buf* lens, size_t lens_off, const hh_buf* tables,
                            size_t tables_off, const char* what) {
    if (!(scale > 0) || !std::isfinite(scale)) return fail(HH_ERR_INVALID, "%s: scale=%g", what, (double)scale);
    if (q_heads < 1 || q_heads % kv->kv_heads || q_heads / kv->kv_heads > 64)
        return fail(HH_ERR_INVALID, "%s: q_heads=%zu is not 1 to 64 times kv_heads=%zu", what, q_heads, kv->kv_heads);
    const size_t el = act_type(type)->bytes, cols = q_heads * kv->head_dim;
    HH_TRY(check_sizes(rows, cols, what));
    HH_TRY(check_rows(e, q, q_off, rows, cols, el, q_stride, what));
    HH_TRY(check_rows(e, out, out_off, rows, cols, el, out_stride, what));
    HH_TRY(check_sizes(seqs, 1, what));
    if (entries > INT32_MAX) return fail(HH_ERR_INVALID, "%s: table_stride=%zu exceeds 31 bits", what, entries);
    HH_TRY(check_vector(e, lens, lens_off, seqs, what));
    if (entries) HH_TRY(check_vector(e, tables, tables_off, seqs * entries, what));
    return HH_OK;
}

hh_status hh_attn_prompt_dev(hh_engine* e, const hh_attn_prompt_desc* d, const hh_kv_desc* kv, const hh_buf* q,
                             size_t q_off, const hh_buf* cache, size_t cache_off, const hh_buf* starts, size_t starts_off,
                             const hh_buf* lens, size_t lens_off, const hh_buf* tables, size_t tables_off, hh_buf* out,
                             size_t out_off) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(d, "attn_prompt desc");
    HH_TRY(check_kv_type(d->type, kv, "attn_prompt"));
    hh_attn_prompt_args a{};
    size_t layer = 0, qs = d->q_stride, os = d->out_stride;
    HH_TRY(check_kv(e, kv, cache, cache_off, 1, &layer, &a.a.kv, "attn_prompt cache"));
    HH_TRY(check_attn(e, d->type, d->scale, d->tokens, d->seqs, d->q_heads, d->table_stride, kv, q, q_off, &qs, out, out_off,
                      &os, lens, lens_off, tables, tables_off, "attn_prompt"));
    HH_TRY(check_vector(e, starts, starts_off, d->seqs + 1, "attn_prompt starts"));
    if (d->tokens == 0 || d->seqs == 0) return HH_OK;
    HH_TRY(e->select());
    a.a.q = at(q, q_off);
    a.a.out = at(out, out_off);
    a.a.lens = (const int32_t*)at(lens, lens_off);
    a.a.tables = (const int32_t*)at(tables, tables_off);
    a.a.q_stride = qs;
    a.a.out_stride = os;
    a.a.seqs = (uint32_t)d->seqs;
    a.a.entries = (uint32_t)d->table_stride;
    a.a.group = (uint32_t)(d->q_heads / kv->kv_heads);
    a.a.c = (float)((double)d->scale * 1.4426950408889634074);
    a.starts = (const int32_t*)at(starts, starts_off);
    a.tokens = (uint32_t)d->tokens;
    try {
        std::lock_guard<std::mutex> lk(e->ws_mutex);
        return e->enqueue_attn_prompt(d->type, kv->type, a);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

hh_status hh_attn_decode_dev(hh_engine* e, const hh_attn_decode_desc* d, const hh_kv_desc* kv, const hh_buf* q,
                             size_t q_off, const hh_buf* cache, size_t cache_off, const hh_buf* prefix_pages,
                             size_t prefix_pages_off, const hh_buf* lens, size_t lens_off, const hh_buf* tables,
                             size_t tables_off, hh_buf* out, size_t out_off) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(d, "attn_decode desc");
    HH_TRY(check_kv_type(d->type, kv, "attn_decode"));
    hh_attn_decode_args a{};
    size_t layer = 0, qs = d->q_stride, os = d->out_stride;
    HH_TRY(check_kv(e, kv, cache, cache_off, 1, &layer, &a.a.kv, "attn_decode cache"));
    HH_TRY(check_attn(e, d->type, d->scale, d->seqs, d->seqs, d->q_heads, d->table_stride, kv, q, q_off, &qs, out, out_off,
                      &os, lens, lens_off, tables, tables_off, "attn_decode"));
    if (d->prefix > INT32_MAX) return fail(HH_ERR_INVALID, "attn_decode: prefix=%zu exceeds 31 bits", d->prefix);
    const size_t shared = (d->prefix + kv->page_size - 1) / kv->page_size;
    if (shared) HH_TRY(check_vector(e, prefix_pages, prefix_pages_off, shared, "attn_decode prefix_pages"));
    if (d->seqs == 0) return HH_OK;
    HH_TRY(e->select());
    a.a.q = at(q, q_off);
    a.a.out = at(out, out_off);
    a.a.lens = (const int32_t*)at(lens, lens_off);
    a.a.tables = (const int32_t*)at(tables, tables_off);
    a.a.q_stride = qs;
    a.a.out_stride = os;
    a.a.seqs = (uint32_t)d->seqs;
    a.a.entries = (uint32_t)d->table_stride;
    a.a.group = (uint32_t)(d->q_heads / kv->kv_heads);
    a.a.c = (float)((double)d->scale * 1.4426950408889634074);
    a.shared = (const int32_t*)at(prefix_pages, prefix_pages_off);
    a.prefix = (uint32_t)d->prefix;
    a.shared_entries = (uint32_t)shared;
    try {
        std::lock_guard<std::mutex> lk(e->ws_mutex);
        return e->enqueue_attn_decode(d->type, kv->type, a);
    } catch (const std::bad_alloc&) {
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

// ---------------------------------------------------------------- MoE ----------------

static hh_status validate_moe_desc(const hh_moe_desc* d) {
    HH_NOT_NULL(d, "moe desc");
    if (d->type != HH_TYPE_Q4_K)
        return fail(HH_ERR_KERNEL_MISSING, "moe: experts of GGML type %d have no MoE kernel (Q4_K only)", d->type);
    if (d->act != HH_ACT_SILU && d->act != HH_ACT_GELU_TANH) return fail(HH_ERR_INVALID, "moe: unknown act %d", d->act);
    if (d->n_experts < 1 || d->n_experts > 512)
        return fail(HH_ERR_INVALID, "moe: n_experts=%zu outside 1..512", d->n_experts);
    if (d->top_k < 1 || d->top_k > 64) return fail(HH_ERR_INVALID, "moe: top_k=%zu outside 1..64", d->top_k);
    if (d->n_group > 64) return fail(HH_ERR_INVALID, "moe: n_group=%zu > 64", d->n_group);
    return HH_OK;
}

static hh_status validate_moe_experts(hh_engine* e, const hh_moe_desc* d, const hh_buf* experts, size_t off) {
    HH_TRY(validate_shape(d->type, d->d_ff, d->d_model));
    HH_TRY(validate_shape(d->type, d->d_model, d->d_ff));
    size_t rin, rff;
    HH_TRY(row_bytes(d->type, d->d_model, &rin));
    HH_TRY(row_bytes(d->type, d->d_ff, &rff));
    // LDS of the expert kernels holds the digits of x (d_model) and of the k intermediates
    const size_t lds_in = 2 * d->d_model + d->d_model / 4, lds_ff = 2 * d->top_k * d->d_ff + d->top_k * d->d_ff / 4;
    if (lds_in > 65536 || lds_ff > 65536)
        return fail(HH_ERR_INVALID, "moe: d_model=%zu / top_k*d_ff=%zu too large for the expert kernels", d->d_model,
                    d->top_k * d->d_ff);
    HH_TRY(check_engine(e, experts, "experts"));
    const size_t pack_end = std::max({d->gate_off + d->d_ff * rin, d->up_off + d->d_ff * rin,
                                      d->down_off + d->d_model * rff});
    if (d->expert_stride != 0 && d->n_experts - 1 > (SIZE_MAX - pack_end) / d->expert_stride)
        return fail(HH_ERR_INVALID, "moe: expert layout overflows");
    HH_TRY(check_range(experts, off, (d->n_experts - 1) * d->expert_stride + pack_end, "moe experts"));
    if (((uintptr_t)experts->ptr + off) % 16 || d->expert_stride % 16 || d->gate_off % 16 || d->up_off % 16 ||
        d->down_off % 16)
        return fail(HH_ERR_INVALID, "moe: expert packs and tensor offsets must be 16-byte aligned");
    if (d->shared_d_ff) {  // the shared expert: an FFN of d_model x shared_d_ff in the same buffer
        HH_TRY(validate_shape(d->type, d->shared_d_ff, d->d_model));
        HH_TRY(validate_shape(d->type, d->d_model, d->shared_d_ff));
        size_t rsf;
        HH_TRY(row_bytes(d->type, d->shared_d_ff, &rsf));
        const size_t g = d->shared_d_ff * rin, dn = d->d_model * rsf;
        if (d->shared_gate_off > SIZE_MAX - g || d->shared_up_off > SIZE_MAX - g || d->shared_down_off > SIZE_MAX - dn)
            return fail(HH_ERR_INVALID, "moe: shared expert layout overflows");
        HH_TRY(check_range(experts, off, std::max({d->shared_gate_off + g, d->shared_up_off + g, d->shared_down_off + dn}),
                           "moe shared expert"));
    }
    return HH_OK;
}

hh_status hh_route_experts_dev(hh_engine* e, const hh_moe_desc* d, const hh_buf* logits, size_t logits_off,
                               const hh_buf* bias, size_t bias_off, size_t T, hh_buf* ids, size_t ids_off,
                               hh_buf* weights, size_t weights_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("route_experts_dev"));
    HH_TRY(validate_moe_desc(d));
    size_t lb = 0, kb = 0;
    HH_TRY(batch_bytes(T, d->n_experts, &lb));
    HH_TRY(batch_bytes(T, d->top_k, &kb));
    HH_TRY(check_engine(e, logits, "logits"));
    HH_TRY(check_engine(e, ids, "ids"));
    HH_TRY(check_engine(e, weights, "weights"));
    HH_TRY(check_range(logits, logits_off, lb, "logits"));
    HH_TRY(check_range(ids, ids_off, kb, "ids"));
    HH_TRY(check_range(weights, weights_off, kb, "weights"));
    if (bias) {
        HH_TRY(check_engine(e, bias, "bias"));
        HH_TRY(check_range(bias, bias_off, d->n_experts * sizeof(float), "bias"));
    }
    if ((logits_off | ids_off | weights_off | bias_off) & 3u)
        return fail(HH_ERR_INVALID, "route_experts: offsets must be 4-byte aligned");
    if (T == 0) return HH_OK;
    HH_TRY(e->select());
    return e->enqueue_moe_route(d, (const float*)((const char*)logits->ptr + logits_off),
                                bias ? (const float*)((const char*)bias->ptr + bias_off) : nullptr, T,
                                (int32_t*)((char*)ids->ptr + ids_off), (float*)((char*)weights->ptr + weights_off));
}

hh_status hh_route_experts(hh_engine* e, const hh_moe_desc* d, const float* logits, const float* bias, size_t T,
                           int32_t* ids, float* weights) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(validate_moe_desc(d));
    size_t lb = 0, kb = 0;
    HH_TRY(batch_bytes(T, d->n_experts, &lb));
    HH_TRY(batch_bytes(T, d->top_k, &kb));
    if (T == 0) return HH_OK;
    HH_NOT_NULL(logits, "logits");
    HH_NOT_NULL(ids, "ids");
    HH_NOT_NULL(weights, "weights");
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    // x workspace: logits then bias; y workspace: ids then weights
    const size_t bb = bias ? d->n_experts * sizeof(float) : 0;
    HH_TRY(e->grow(&e->ws_x, &e->ws_x_cap, lb + bb));
    HH_TRY(e->grow(&e->ws_y, &e->ws_y_cap, 2 * kb));
    HH_TRY_HIP(hipMemcpyAsync(e->ws_x, logits, lb, hipMemcpyHostToDevice, e->stream), "hipMemcpyAsync(logits)");
    if (bias)
        HH_TRY_HIP(hipMemcpyAsync((char*)e->ws_x + lb, bias, bb, hipMemcpyHostToDevice, e->stream),
                   "hipMemcpyAsync(bias)");
    HH_TRY(e->enqueue_moe_route(d, (const float*)e->ws_x, bias ? (const float*)((char*)e->ws_x + lb) : nullptr, T,
                                (int32_t*)e->ws_y, (float*)((char*)e->ws_y + kb)));
    HH_TRY_HIP(hipMemcpyAsync(ids, e->ws_y, kb, hipMemcpyDeviceToHost, e->stream), "hipMemcpyAsync(ids)");
    HH_TRY_HIP(hipMemcpyAsync(weights, (char*)e->ws_y + kb, kb, hipMemcpyDeviceToHost, e->stream),
               "hipMemcpyAsync(weights)");
    return e->check_device_error();
}

hh_status hh_moe_ffn_dev(hh_engine* e, const hh_moe_desc* d, const hh_buf* experts, size_t experts_off,
                         const hh_buf* x, size_t x_off, size_t T, const hh_buf* ids, size_t ids_off,
                         const hh_buf* weights, size_t weights_off, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("moe_ffn_dev"));
    HH_TRY(validate_moe_desc(d));
    HH_TRY(validate_moe_experts(e, d, experts, experts_off));
    size_t xb = 0, kb = 0;
    HH_TRY(batch_bytes(T, d->d_model, &xb));
    HH_TRY(batch_bytes(T, d->top_k, &kb));
    for (const hh_buf* b : {x, ids, weights, (const hh_buf*)y}) HH_TRY(check_engine(e, b, "moe"));
    HH_TRY(check_range(x, x_off, xb, "x"));
    HH_TRY(check_range(y, y_off, xb, "y"));
    HH_TRY(check_range(ids, ids_off, kb, "ids"));
    HH_TRY(check_range(weights, weights_off, kb, "weights"));
    if ((x_off & 15u) || ((y_off | ids_off | weights_off) & 3u))
        return fail(HH_ERR_INVALID, "moe_ffn: x offset must be 16-byte aligned, y/ids/weights 4-byte");
    if (T == 0) return HH_OK;
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    const uint8_t* ex = (const uint8_t*)experts->ptr + experts_off;
    const float* xp = (const float*)((const char*)x->ptr + x_off);
    float* yp = (float*)((char*)y->ptr + y_off);
    HH_TRY(e->enqueue_moe_ffn(d, ex, xp, T, (int32_t*)((char*)ids->ptr + ids_off),
                              (float*)((char*)weights->ptr + weights_off), yp));
    return e->enqueue_moe_shared(d, ex, xp, T, yp);
}

hh_status hh_moe_dev(hh_engine* e, const hh_moe_desc* d, const hh_buf* experts, size_t experts_off,
                     const hh_buf* logits, size_t logits_off, const hh_buf* bias, size_t bias_off, const hh_buf* x,
                     size_t x_off, size_t T, hh_buf* y, size_t y_off) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->no_capture("moe_dev"));
    HH_TRY(validate_moe_desc(d));
    HH_TRY(validate_moe_experts(e, d, experts, experts_off));
    size_t xb = 0, kb = 0, lb = 0;
    HH_TRY(batch_bytes(T, d->d_model, &xb));
    HH_TRY(batch_bytes(T, d->top_k, &kb));
    HH_TRY(batch_bytes(T, d->n_experts, &lb));
    for (const hh_buf* b : {logits, x, (const hh_buf*)y}) HH_TRY(check_engine(e, b, "moe"));
    HH_TRY(check_range(logits, logits_off, lb, "logits"));
    HH_TRY(check_range(x, x_off, xb, "x"));
    HH_TRY(check_range(y, y_off, xb, "y"));
    if (bias) {
        HH_TRY(check_engine(e, bias, "bias"));
        HH_TRY(check_range(bias, bias_off, d->n_experts * sizeof(float), "bias"));
    }
    if ((x_off & 15u) || ((y_off | logits_off | bias_off) & 3u))
        return fail(HH_ERR_INVALID, "moe: x offset must be 16-byte aligned, y/logits/bias 4-byte");
    if (T == 0) return HH_OK;
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    HH_TRY(e->grow(&e->ws_moe_ids, &e->ws_moe_ids_cap, kb));
    HH_TRY(e->grow(&e->ws_moe_w, &e->ws_moe_w_cap, kb));
    // routing runs inside the gate/up kernel
    const uint8_t* ex = (const uint8_t*)experts->ptr + experts_off;
    const float* xp = (const float*)((const char*)x->ptr + x_off);
    float* yp = (float*)((char*)y->ptr + y_off);
    HH_TRY(e->enqueue_moe_ffn(d, ex, xp, T, (int32_t*)e->ws_moe_ids, (float*)e->ws_moe_w, yp,
                              (const float*)((const char*)logits->ptr + logits_off),
                              bias ? (const float*)((const char*)bias->ptr + bias_off) : nullptr));
    return e->enqueue_moe_shared(d, ex, xp, T, yp);
}

// ---------------------------------------------------------------- events -------------

hh_status hh_event_create(hh_engine* e, hh_event** out) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(out, "out");
    HH_TRY(e->select());
    hh_event* ev = new (std::nothrow) hh_event{nullptr, e->device};
    if (!ev) return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    hipError_t err = hipEventCreate(&ev->ev);
    if (err != hipSuccess) {
        delete ev;
        return hip_fail(err, "hipEventCreate");
    }
    *out = ev;
    return HH_OK;
}

void hh_event_destroy(hh_event* ev) {
    if (!ev) return;
    (void)hipSetDevice(ev->device);
    (void)hipEventDestroy(ev->ev);
    delete ev;
}

hh_status hh_event_record(hh_engine* e, hh_event* ev) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(ev, "event");
    HH_TRY(e->select());
    HH_TRY_HIP(hipEventRecord(ev->ev, e->stream), "hipEventRecord");
    return HH_OK;
}

hh_status hh_event_elapsed_ms(hh_event* a, hh_event* b, float* ms) {
    HH_NOT_NULL(a, "start");
    HH_NOT_NULL(b, "stop");
    HH_NOT_NULL(ms, "ms");
    HH_TRY_HIP(hipEventSynchronize(b->ev), "hipEventSynchronize");
    HH_TRY_HIP(hipEventElapsedTime(ms, a->ev, b->ev), "hipEventElapsedTime");
    return HH_OK;
}

// ---------------------------------------------------------------- graphs -------------

struct hh_graph {
    hh_engine* engine;
    hipGraph_t graph;
    hipGraphExec_t exec;
};

hh_status hh_graph_begin(hh_engine* e) {
    HH_NOT_NULL(e, "engine");
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    if (e->capturing) return fail(HH_ERR_INVALID, "graph_begin: a capture is already open on this engine");
    HH_TRY_HIP(hipStreamBeginCapture(e->stream, hipStreamCaptureModeThreadLocal), "hipStreamBeginCapture");
    e->capturing = true;
    return HH_OK;
}

hh_status hh_graph_end(hh_engine* e, hh_graph** out) {
    HH_NOT_NULL(e, "engine");
    HH_NOT_NULL(out, "out");
    *out = nullptr;
    HH_TRY(e->select());
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    if (!e->capturing) return fail(HH_ERR_INVALID, "graph_end: no capture is open on this engine");
    e->capturing = false;
    hipGraph_t g = nullptr;
    HH_TRY_HIP(hipStreamEndCapture(e->stream, &g), "hipStreamEndCapture");
    hipGraphExec_t x = nullptr;
    hipError_t err = hipGraphInstantiate(&x, g, nullptr, nullptr, 0);
    if (err != hipSuccess) {
        (void)hipGraphDestroy(g);
        return hip_fail(err, "hipGraphInstantiate");
    }
    hh_graph* h = new (std::nothrow) hh_graph{e, g, x};
    if (!h) {
        (void)hipGraphExecDestroy(x);
        (void)hipGraphDestroy(g);
        return fail(HH_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
    e->live_graphs++;
    *out = h;
    return HH_OK;
}

hh_status hh_graph_launch(hh_graph* g) {
    HH_NOT_NULL(g, "graph");
    HH_TRY(g->engine->select());
    std::lock_guard<std::mutex> lk(g->engine->ws_mutex);
    if (g->engine->capturing) return fail(HH_ERR_INVALID, "graph_launch: the engine's stream is being captured");
    HH_TRY_HIP(hipGraphLaunch(g->exec, g->engine->stream), "hipGraphLaunch");
    return HH_OK;
}

void hh_graph_destroy(hh_graph* g) {
    if (!g) return;
    hh_engine* e = g->engine;
    (void)e->select();
    std::lock_guard<std::mutex> lk(e->ws_mutex);
    // a replay may still be running on the stream
    (void)hipStreamSynchronize(e->stream);
    (void)hipGraphExecDestroy(g->exec);
    (void)hipGraphDestroy(g->graph);
    delete g;
    if (--e->live_graphs == 0) e->free_retired();
}

// ---------------------------------------------------------------- synthetic data -----

hh_status hh_synth_weights_dev(hh_engine* e, int t, hh_buf* dst, size_t off, size_t n_blocks, uint64_t seed, float lo,
                               float hi) {
    HH_NOT_NULL(e, "engine");
    const Format* f = format_of(t);
    if (!f) return fail(HH_ERR_KERNEL_MISSING, "no synthetic generator for GGML type %d", t);
    const size_t bytes = n_blocks * f->bytes;
    HH_TRY(check_engine(e, dst, "dst"));
    HH_TRY(check_range(dst, off, bytes, "synth"));
    if (off & 7u) return fail(HH_ERR_INVALID, "synth: offset must be 8-byte aligned");
    if (bytes == 0) return HH_OK;
    HH_TRY(e->select());
    hipFunction_t fb, fs;
    HH_TRY(e->kernel("hh_synth_bytes", &fb));
    HH_TRY(e->kernel("hh_synth_scales", &fs));
    hh_synth_args a{(uint8_t*)dst->ptr + off, (uint64_t)bytes, seed, (uint64_t)n_blocks, t, lo, hi, 0};
    const size_t words = (bytes + 7) / 8;
    const uint32_t grid = (uint32_t)std::min<size_t>((words + 255) / 256, 65536);
    HH_TRY(e->launch(fb, grid, 256, a));
    if (t == HH_TYPE_F32 || t == HH_TYPE_F16) return HH_OK;
    return e->launch(fs, (uint32_t)((n_blocks + 255) / 256), 256, a);
}

}  // extern "C"
