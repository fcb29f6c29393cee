#include "ops.hpp"

#include <cstdarg>
#include <cstdio>

namespace llmb {

// The message buffer of the calling thread (engine.cu: llmb_last_error(NULL)).
void set_thread_error(const char *msg) noexcept;

int op_error(int code, const char *fmt, ...) noexcept {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    set_thread_error(buf);
    return code;
}

int op_device(const char *what, int *device) noexcept {
    cudaError_t e = cudaPeekAtLastError();
    if (e != cudaSuccess)
        return op_error(LLMB_ERR_CUDA, "llm: %s: an earlier CUDA error is pending: %s", what, cudaGetErrorString(e));
    e = cudaGetDevice(device);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return op_error(LLMB_ERR_CUDA, "llm: %s: %s", what, cudaGetErrorString(e));
    }
    return LLMB_OK;
}

int op_alignment(const char *what, std::initializer_list<OpPointer> ps) noexcept {
    for (const OpPointer &q : ps) {
        if (!q.p) {
            if (q.optional) continue;
            return op_error(LLMB_ERR_ARG, "llm: %s: %s is NULL", what, q.name);
        }
        if (reinterpret_cast<uintptr_t>(q.p) % q.align != 0)
            return op_error(LLMB_ERR_ARG, "llm: %s: %s is not aligned to %d bytes", what, q.name, q.align);
    }
    return LLMB_OK;
}

int op_pointers(const char *what, int device, std::initializer_list<OpPointer> ps) noexcept {
    for (const OpPointer &q : ps) {
        if (!q.p) continue;
        cudaPointerAttributes a{};
        const cudaError_t e = cudaPointerGetAttributes(&a, q.p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return op_error(LLMB_ERR_CUDA, "llm: %s: %s: %s", what, q.name, cudaGetErrorString(e));
        }
        if (a.type == cudaMemoryTypeManaged) continue;
        if (a.type != cudaMemoryTypeDevice)
            return op_error(LLMB_ERR_ARG, "llm: %s: %s is not device memory", what, q.name);
        if (a.device != device)
            return op_error(LLMB_ERR_ARG, "llm: %s: %s is memory of device %d, the current device is %d", what, q.name,
                            a.device, device);
    }
    return LLMB_OK;
}

int op_launched(const char *what) noexcept {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LLMB_OK : op_error(LLMB_ERR_CUDA, "llm: %s: %s", what, cudaGetErrorString(e));
}

}  // namespace llmb
