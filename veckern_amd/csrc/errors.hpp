// Errors of the C ABI: a failure is thrown inside the library, and guarded() turns it into a status code and the calling
// thread's message before it reaches a C caller.
#pragma once

#include <hip/hip_runtime.h>

#include <new>
#include <stdexcept>
#include <string>

#include "veckern/veckern.h"

#define VK_EXPORT extern "C" __attribute__((visibility("default")))

namespace vk {

inline thread_local std::string g_error;

struct Failure {
    int code;
    std::string message;
};

[[noreturn]] inline void fail(int code, const std::string& message) { throw Failure{code, message}; }

inline void require(bool condition, const std::string& message) {
    if (!condition) fail(VK_ERR_RUNTIME, message);
}

inline void hip_check(hipError_t e, const char* what) {
    if (e != hipSuccess)
        fail(e == hipErrorOutOfMemory ? VK_ERR_OUT_OF_MEMORY : VK_ERR_DEVICE,
             std::string(what) + " failed: " + hipGetErrorString(e));
}
#define VK_HIP(call) ::vk::hip_check((call), #call)

template <typename F>
int guarded(F&& body) {
    try {
        body();
        g_error.clear();
        return VK_OK;
    } catch (const Failure& f) {
        g_error = f.message;
        return f.code;
    } catch (const std::bad_alloc&) {
        g_error = "host allocation failed";
        return VK_ERR_OUT_OF_MEMORY;
    } catch (const std::exception& e) {
        g_error = e.what();
        return VK_ERR_RUNTIME;
    } catch (...) {
        g_error = "unknown error";
        return VK_ERR_RUNTIME;
    }
}

}  // namespace vk
