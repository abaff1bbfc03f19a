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

inline int launched(const char* who) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return nh_internal_fail((int)e, (std::string(who) + ": " + hipGetErrorString(e)).c_str());
    return 0;
}

// call f with a value of the storage type `dtype` names
template <class F> int by_dtype(int dtype, F f) {
    if (dtype == NH_T_F32) return f(float());
    if (dtype == NH_T_F16) return f(nh_f16());
    return f(nh_bf16());
}

constexpr size_t MAX_BLOCKS = 0x7FFFFFFF;

}  // namespace lm

#endif  // NEON_LM_OPS_H
