// What the entry points over the caller's device buffers share: their error
// messages and the checks that every call makes before it launches.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <initializer_list>

#include "../../include/llm_b200.h"

namespace llmb {

// Records the message that llmb_last_error(NULL) returns on this thread and returns code.
int op_error(int code, const char *fmt, ...) noexcept __attribute__((format(printf, 2, 3)));

// The current device, with no error pending on the thread (one left by earlier work is the caller's: it is
// reported without being cleared, and nothing is launched).  LLMB_OK or the error's code.
int op_device(const char *what, int *device) noexcept;

struct OpPointer {
    const void *p;
    const char *name;
    int align;      // bytes
    bool optional;  // may be NULL
};

// Each pointer is aligned, and is memory of the device.  LLMB_OK or the error's code.
int op_pointers(const char *what, int device, std::initializer_list<OpPointer> ps) noexcept;

// Alignment and presence alone (no CUDA call), so that bad arguments are refused without a GPU too.
int op_alignment(const char *what, std::initializer_list<OpPointer> ps) noexcept;

// The error of the launch just made (none was pending before it): cleared and reported.
int op_launched(const char *what) noexcept;

// Lets a kernel use that much dynamic shared memory, once per device (the call costs as much as a launch's checks).
template <auto *Kernel>
cudaError_t op_shared(int device, int bytes) noexcept {
    static std::atomic<bool> done[64];
    if (device < 64 && done[device].load(std::memory_order_relaxed)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device < 64) done[device].store(true, std::memory_order_relaxed);
    return e;
}

}  // namespace llmb
