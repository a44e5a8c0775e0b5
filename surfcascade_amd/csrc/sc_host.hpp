// sc_host.hpp -- what the C ABI's translation units share on the host: the
// error convention, device buffers and the device-pointer check.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>
#include <new>
#include <string>

#include "sc_model.hpp"
#include "surfcascade.h"

namespace sc {

// sets the calling thread's sc_last_error message (sc_api.cpp) and returns code
int set_error(int code, const std::string &msg);

#define HIPCHK(expr)                                                                            \
    do {                                                                                        \
        hipError_t e_ = (expr);                                                                 \
        if (e_ != hipSuccess)                                                                   \
            throw sc::Error{SC_ERR_DEVICE, std::string(#expr) + ": " + hipGetErrorString(e_)}; \
    } while (0)

template <class T>
struct DevBuf {
    T *p = nullptr;
    size_t n = 0;
    void ensure(size_t want) {
        if (want <= n) return;
        release();
        HIPCHK(hipMalloc(&p, std::max<size_t>(want, 1) * sizeof(T)));
        n = want;
    }
    void release() {
        if (p) (void)hipFree(p);
        p = nullptr;
        n = 0;
    }
};

// A caller's device pointer must be device memory of GPU `device` (owned by
// `owner`, for the message): a host pointer or another GPU's memory would
// fault in a kernel instead of returning SC_ERR_INVALID.
void check_device_ptr(int device, const char *owner, const void *p, const char *what);

// runs an entry point's body: no C++ exception crosses the ABI
template <class F>
int guarded(F &&f) {
    try {
        return f();
    } catch (const Error &e) {
        return set_error(e.code, e.msg);
    } catch (const std::bad_alloc &) {
        return set_error(SC_ERR_NOMEM, "out of host memory");
    } catch (const std::exception &e) {
        return set_error(SC_ERR_INVALID, e.what());
    }
}

}  // namespace sc
