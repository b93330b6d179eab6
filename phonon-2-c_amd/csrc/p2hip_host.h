/*  p2hip_host.h – what the library's host sources share: the per-thread error message, initialisation, the stream a
 *  call runs on and the device's size. Hidden: none of it is part of the C ABI.
 */
#pragma once

#include "p2hip.h"

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#define P2_HIDDEN __attribute__((visibility("hidden")))

namespace p2host {

/* set this thread's error message and return rc; the runtime's own error, if rc reports one, is thereby taken */
P2_HIDDEN int fail(int rc, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
P2_HIDDEN int ensure_init();
P2_HIDDEN hipStream_t stream_of(void *s);   /* NULL: the calling thread's own stream */
P2_HIDDEN int cu_count();

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

}  // namespace p2host

#define HIPCHK(call)                                                                                            \
    do {                                                                                                        \
        hipError_t e_ = (call);                                                                                 \
        if (e_ != hipSuccess) return p2host::fail(P2H_E_DEVICE, "%s: %s", #call, hipGetErrorString(e_));      \
    } while (0)
