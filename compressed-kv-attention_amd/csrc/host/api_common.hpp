// What the files of the C ABI (kvexp_hip_api.cpp, kvexp_paged_api.cpp) share:
// status and error handling, device buffers and their pool, the context, the
// device guard and the read-back of status words.
#pragma once

#include "kvexp_hip.h"

#include <hip/hip_runtime.h>

#include <mutex>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "../hip/kvexp_types.h"
#include "host_walk.hpp"

namespace kvexp_launch {
hipError_t result(const int64_t *value, const uint32_t *status, int64_t *host, hipStream_t s);
hipError_t esc_start(const kvexp_dev::EscJob *jobs, int n_jobs, uint32_t *status, hipStream_t s);
hipError_t esc_pos(const kvexp_dev::EscJob *jobs, const int2 *blocks, int n_blocks, uint32_t *status, hipStream_t s);
} // namespace kvexp_launch

namespace kvexp_host {

inline thread_local std::string g_error;

inline int set_error(int code, const std::string &msg) {
    g_error = msg;
    return code;
}
inline int ok() {
    g_error.clear();
    return KVEXP_HIP_OK;
}

struct HipFail {
    hipError_t err;
    const char *what;
};

#define HIPX(call)                                                                                                    \
    do {                                                                                                              \
        hipError_t e_ = (call);                                                                                       \
        if (e_ != hipSuccess) throw HipFail{e_, #call};                                                               \
    } while (0)

template <class F> int guarded(F &&fn) {
    try {
        fn();
        return ok();
    } catch (const KvexpFail &f) {
        return set_error(f.code, f.msg);
    } catch (const HipFail &h) {
        return set_error(KVEXP_HIP_DEVICE_ERROR, std::string(h.what) + ": " + hipGetErrorString(h.err));
    } catch (const std::bad_alloc &) {
        return set_error(KVEXP_HIP_DEVICE_ERROR, "host allocation failed");
    } catch (const std::exception &e) {
        return set_error(KVEXP_HIP_LOGIC_ERROR, e.what());
    }
}

// Device buffers kept for reuse by a context: hipFree synchronises the whole
// device, so a call path that allocated and freed on every call would wait
// for every other caller's work. Blocks are kept by size class (four classes
// per power of two), at most kMaxHeld bytes in all, and returned to the
// device when the context is destroyed. Only buffers whose last use is known
// to be finished when they are released go back to a pool.
class DevPool {
  public:
    static size_t size_class(size_t n) {
        size_t c = 256;
        while (c < n) c *= 2;
        if (c <= 256) return c;
        const size_t q = c / 8; // c/2 + q, c/2 + 2q, c/2 + 3q, c
        for (size_t k = 5; k <= 8; ++k)
            if (q * k >= n) return q * k;
        return c;
    }
    void *get(size_t n, size_t &cap) {
        cap = size_class(n);
        {
            std::lock_guard<std::mutex> lock(mu_);
            for (size_t i = 0; i < free_.size(); ++i)
                if (free_[i].first == cap) {
                    void *p = free_[i].second;
                    free_[i] = free_.back();
                    free_.pop_back();
                    held_ -= cap;
                    return p;
                }
        }
        void *p = nullptr;
        HIPX(hipMalloc(&p, cap));
        return p;
    }
    void put(void *p, size_t cap) {
        {
            std::lock_guard<std::mutex> lock(mu_);
            if (held_ + cap <= kMaxHeld) {
                free_.emplace_back(cap, p);
                held_ += cap;
                return;
            }
        }
        (void)hipFree(p);
    }
    ~DevPool() {
        for (auto &f : free_) (void)hipFree(f.second);
    }

  private:
    static constexpr size_t kMaxHeld = size_t(1) << 30;
    std::mutex mu_;
    std::vector<std::pair<size_t, void *>> free_;
    size_t held_ = 0;
};

// Device allocation released on scope exit unless kept: back to its pool
// when it came from one, else to the device.
struct DevBuf {
    void *p = nullptr;
    DevPool *pool = nullptr;
    size_t cap = 0;
    bool part = false;
    DevBuf() = default;
    explicit DevBuf(size_t n) {
        if (n) HIPX(hipMalloc(&p, n));
    }
    DevBuf(DevPool *from, size_t n) {
        if (from == nullptr) {
            if (n) HIPX(hipMalloc(&p, n));
        } else if (n) {
            p = from->get(n, cap);
            pool = from;
        }
    }
    DevBuf(const DevBuf &) = delete;
    DevBuf &operator=(const DevBuf &) = delete;
    DevBuf(DevBuf &&o) noexcept : p(o.p), pool(o.pool), cap(o.cap), part(o.part) { o.p = nullptr; }
    DevBuf &operator=(DevBuf &&o) noexcept {
        std::swap(p, o.p);
        std::swap(pool, o.pool);
        std::swap(cap, o.cap);
        std::swap(part, o.part);
        return *this;
    }
    // A part of another allocation, which outlives it.
    static DevBuf part_of(void *at) {
        DevBuf b;
        b.p = at;
        b.part = true;
        return b;
    }
    ~DevBuf() {
        if (p == nullptr || part) return;
        if (pool) pool->put(p, cap);
        else (void)hipFree(p);
    }
    template <class T> T *as() const { return static_cast<T *>(p); }
};

inline std::string status_message(uint32_t st) {
    using namespace kvexp_dev;
    if (st & kStShort) return "xkv decode ran out of blocks";
    if (st & kStHeader) return "xkv block dimension or length mismatch";
    if (st & kStMode) return "unknown xkv block mode";
    if (st & kStTruncated) return "truncated coded xkv block";
    if (st & kStIndex) return "xkv block index does not match the container";
    if (st & kStEscape) return "xkv escape stream overrun";
    return "xkv container error";
}

// The encoders' status word as an error message.
inline std::string encoder_status_message(uint32_t st) {
    if (st & kvexp_dev::kStLookback) return "one-pass encoder: an earlier block's size never arrived";
    return "escape count drifted from the size model";
}

} // namespace kvexp_host

// ================================================================ context ==
struct kvexp_hip_ctx {
    int device = 0;
    // buffers of the host-pointer entry and of the plans it builds (declared
    // first: destroyed after everything that may return buffers to it)
    kvexp_host::DevPool pool;
    kvexp_host::DevBuf status; // uint32 status word of the encoders and the decoder
    // encoder scratch, grown on demand; `scratch_done` is recorded on the
    // stream of the last launch that used it, so growing it never frees
    // memory that a kernel still in flight reads
    kvexp_host::DevBuf enc_meta, enc_bases, enc_off, enc_first, app_jobs;
    size_t enc_meta_cap = 0, enc_bases_cap = 0, enc_index_cap = 0, app_jobs_cap = 0;
    // look-back entries and ticket counters of the one-pass encoder, the
    // epoch of its last launch, and whether a launch reported a broken
    // look-back (the next one then clears both arrays)
    kvexp_host::DevBuf enc_lb, enc_tk;
    size_t enc_lb_cap = 0, enc_tk_cap = 0;
    uint32_t enc_epoch = 0;
    bool enc_lb_dirty = false;
    hipEvent_t scratch_done = nullptr;
    // stream of the host-pointer entry (kvexp_hip_attention_decode_host): its
    // copies and kernels wait for nothing outside this context
    hipStream_t stream = nullptr;
    int cu_count = 0;
    int enc_modes = int(KVEXP_HIP_MODES_REFERENCE); // coded modes the encoders may choose
    // pinned host staging for the plan builder's reads of block indexes
    void *pinned = nullptr;
    size_t pinned_cap = 0;
    // pinned result slots (two words each, written by result_kernel): leased
    // per call, since plans of one context may be checked from several threads
    static constexpr int kResultSlots = 64;
    std::mutex result_mu;
    int64_t *results = nullptr;
    uint64_t results_used = 0;
    ~kvexp_hip_ctx() {
        if (stream) (void)hipStreamSynchronize(stream);
        if (scratch_done) (void)hipEventSynchronize(scratch_done);
        if (pinned) (void)hipHostFree(pinned);
        if (results) (void)hipHostFree(results);
        if (scratch_done) (void)hipEventDestroy(scratch_done);
        if (stream) (void)hipStreamDestroy(stream);
    }
};

namespace kvexp_host {

struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) {
        HIPX(hipGetDevice(&prev));
        if (prev != dev) HIPX(hipSetDevice(dev));
    }
    ~DeviceGuard() {
        int cur = -1;
        if (hipGetDevice(&cur) == hipSuccess && cur != prev && prev >= 0) (void)hipSetDevice(prev);
    }
};

// The context's pinned staging buffer, at least n bytes (its last use is over:
// every user synchronises its stream before it returns). It grows by half more
// than asked for: a decode loop's rebuilds each need a little more.
inline void *pinned_staging(kvexp_hip_ctx *ctx, size_t n) {
    if (n > ctx->pinned_cap) {
        n += n / 2;
        if (ctx->pinned) HIPX(hipHostFree(ctx->pinned));
        ctx->pinned = nullptr;
        ctx->pinned_cap = 0;
        HIPX(hipHostMalloc(&ctx->pinned, n, hipHostMallocDefault));
        ctx->pinned_cap = n;
    }
    return ctx->pinned;
}

// A leased pinned result slot (p null when all are leased).
struct ResultSlot {
    kvexp_hip_ctx *ctx;
    volatile int64_t *p = nullptr;
    int i = -1;
    explicit ResultSlot(kvexp_hip_ctx *c) : ctx(c) {
        std::lock_guard<std::mutex> lock(c->result_mu);
        if (c->results == nullptr)
            HIPX(hipHostMalloc(reinterpret_cast<void **>(&c->results), kvexp_hip_ctx::kResultSlots * 16,
                               hipHostMallocDefault));
        if (c->results_used == ~uint64_t(0)) return;
        i = __builtin_ctzll(~c->results_used);
        c->results_used |= uint64_t(1) << i;
        p = c->results + 2 * i;
    }
    ResultSlot(const ResultSlot &) = delete;
    ~ResultSlot() {
        if (i < 0) return;
        std::lock_guard<std::mutex> lock(ctx->result_mu);
        ctx->results_used &= ~(uint64_t(1) << i);
    }
};

// Synchronises `s` and returns the status word; *value (nullable) receives
// the device word d_value. Through a pinned slot that the GPU writes (one
// tensor's encode call: 49 us with two copies to pageable memory, 32 so).
inline uint32_t read_result(kvexp_hip_ctx *ctx, const int64_t *d_value, const uint32_t *d_status, int64_t *value,
                     hipStream_t s) {
    ResultSlot slot(ctx);
    if (slot.p == nullptr) { // every slot leased
        int64_t v = 0;
        uint32_t st = 0;
        if (d_value != nullptr) HIPX(hipMemcpyAsync(&v, d_value, sizeof v, hipMemcpyDeviceToHost, s));
        HIPX(hipMemcpyAsync(&st, d_status, sizeof st, hipMemcpyDeviceToHost, s));
        HIPX(hipStreamSynchronize(s));
        if (value != nullptr) *value = v;
        return st;
    }
    HIPX(kvexp_launch::result(d_value, d_status, const_cast<int64_t *>(slot.p), s));
    HIPX(hipStreamSynchronize(s));
    if (value != nullptr) *value = slot.p[0];
    return uint32_t(slot.p[1]);
}

inline void check_status_word(kvexp_hip_ctx *ctx, uint32_t *d_status, hipStream_t s) {
    const uint32_t st = read_result(ctx, nullptr, d_status, nullptr, s);
    if (st != 0u) {
        HIPX(hipMemsetAsync(d_status, 0, sizeof(uint32_t), s));
        HIPX(hipStreamSynchronize(s));
        fail(KVEXP_HIP_FORMAT_ERROR, status_message(st));
    }
}

} // namespace kvexp_host
