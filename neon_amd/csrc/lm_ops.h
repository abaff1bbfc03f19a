// What the language-model operators (layernorm.hip, embedding.hip,
// distill.hip) share on the host side: storage codes, argument checks, the
// device the library was initialised on.
#ifndef NEON_LM_OPS_H
#define NEON_LM_OPS_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "neonhip.h"
#include "device/neon_device.h"

bool nh_internal_ready();
int nh_internal_fail(int code, const char* msg);
int nh_internal_cu_count();
int nh_internal_device();

namespace lm {

// elements of a storage type in one 16-byte access
template <typename T> struct vec { static constexpr int V = 16 / (int)sizeof(T); };

inline size_t align256(size_t x) { return (x + 255) / 256 * 256; }
inline size_t ceil_div(size_t a, size_t b) { return (a + b - 1) / b; }
inline int item_bytes(int dtype) { return dtype == NH_T_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == NH_T_F32 || dtype == NH_T_F16 || dtype == NH_T_BF16; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int refuse(const char* who, const char* why) {
    return nh_internal_fail(NH_EINVAL, (std::string(who) + ": " + why).c_str());
}

// The kernels run on the device nh_init chose, whatever device the calling
// thread has made current since; the thread gets its own back afterwards.
class OnDevice {
  public:
    OnDevice() {
        const int want = nh_internal_device();
        int now = want;
        if (hipGetDevice(&now) == hipSuccess && now != want && hipSetDevice(want) == hipSuccess) back_ = now;
    }
    ~OnDevice() {
        if (back_ >= 0) (void)hipSetDevice(back_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;

  private:
    int back_ = -1;
};

// What an operator launches.  Its body is gone through twice: to see that the
// device can count the threads of every launch -- in 32 bits: 2^24 workgroups of
// 256 threads, 2^22 of 1024 --, and to launch.  So an operator runs as a whole or
// not at all; should a launch fail all the same, none follows it.
class Launches {
  public:
    Launches(const char* who, hipStream_t stream, bool go) : who_(who), stream_(stream), go_(go) {}
    // a grid of (blocks, chunks) workgroups
    template <class... P, class... A>
    void operator()(void (*kernel)(P...), size_t blocks, unsigned chunks, unsigned threads, unsigned lds, const A&... args) {
        if (rc_ == 0 && blocks > 0xFFFFFFFFu / threads) rc_ = refuse(who_, "more threads than one launch counts in 32 bits");
        if (rc_ == 0 && go_) send(kernel, dim3((unsigned)blocks, chunks), dim3(threads), lds, static_cast<P>(args)...);
    }
    int status() const { return rc_; }

  private:
    template <class K, class... P> void send(K kernel, dim3 grid, dim3 block, unsigned lds, P... args) {
        void* list[] = {&args...};
        // (the call's own status: what hipGetLastError holds may be another call's)
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, list, lds, stream_);
        if (e == hipSuccess) return;
        (void)hipGetLastError();
        rc_ = nh_internal_fail((int)e, (std::string(who_) + ": " + hipGetErrorString(e)).c_str());
    }

    const char* who_;
    hipStream_t stream_;
    bool go_;
    int rc_ = 0;
};

template <class F> int run(const char* who, void* stream, F body) {
    Launches look(who, (hipStream_t)stream, false);
    body(look);
    if (look.status()) return look.status();
    if (!nh_internal_ready()) return nh_internal_fail(NH_ENOTINIT, "nh_init has not been called");
    OnDevice here;
    Launches go(who, (hipStream_t)stream, true);
    body(go);
    return go.status();
}

// call f with a value of the storage type `dtype` names
template <class F> void by_dtype(int dtype, F f) {
    if (dtype == NH_T_F32) f(float());
    else if (dtype == NH_T_F16) f(nh_f16());
    else f(nh_bf16());
}

}  // namespace lm

#endif  // NEON_LM_OPS_H
