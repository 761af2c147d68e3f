// Host parts shared by the entry points: messages and devices.
#include "head_common.h"

#include <atomic>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

namespace tkh {

static thread_local char g_message[512];

int fail(int status, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_message, sizeof g_message, fmt, ap);
    va_end(ap);
    return status;
}

int fail_hip(const char* what, hipError_t e) {
    (void)hipGetLastError();  // taken back, so that no later check reports it
    return fail(TKH_E_DEVICE, "%s: %s", what, hipGetErrorString(e));
}

// 0 unknown, 1 gfx950, 2 another architecture
static std::atomic<int> g_arch[64];

static int check_arch(int device) {
    if (device < 0 || device >= 64) return fail(TKH_E_INVALID_ARG, "device %d", device);
    int known = g_arch[device].load(std::memory_order_relaxed);
    if (!known) {
        hipDeviceProp_t prop;
        hipError_t e = hipGetDeviceProperties(&prop, device);
        if (e != hipSuccess) return fail_hip("hipGetDeviceProperties", e);
        known = strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
        g_arch[device].store(known, std::memory_order_relaxed);
    }
    return known == 1 ? TKH_OK : fail(TKH_E_ARCH, "device %d is not a gfx950", device);
}

DeviceScope::DeviceScope(int device) {
    status_ = check_arch(device);
    if (status_ != TKH_OK) return;
    int now = -1;
    hipError_t e = hipGetDevice(&now);
    if (e == hipSuccess && now != device) {
        e = hipSetDevice(device);
        if (e == hipSuccess) prev_ = now;
    }
    if (e != hipSuccess) status_ = fail_hip("device", e);
}

DeviceScope::~DeviceScope() {
    if (prev_ >= 0) (void)hipSetDevice(prev_);
}

}  // namespace tkh

// callers pack these by position
static_assert(TKH_ABI_VERSION == 1 && sizeof(tkh_norm) == 120 && sizeof(tkh_matmul) == 112 &&
                  sizeof(tkh_sample) == 144,
              "other arguments are another TKH_ABI_VERSION");

extern "C" const char* tk_head_last_error(void) { return tkh::g_message; }
extern "C" int tk_head_abi_version(void) { return TKH_ABI_VERSION; }
extern "C" const char* tk_head_sources(void) { return TKH_SOURCES; }
