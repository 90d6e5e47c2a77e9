// tb_stream_entry.h -- what the stream-level C entries share (the entries that
// take a cudaStream_t and device pointers, and no context): they run on the
// device that holds the caller's memory, whatever device is current, and their
// kernels report into that device's error word
// (tb_paged_attention_noalloc_status).
#pragma once

#include <atomic>
#include "../../include/tinybrain_cuda.h"
#include "tb_kernels.h"

namespace tb {

// SM count and address of the stream-level entries' error word on device
// `dev`, which must be current.  Safe inside a stream capture.
cudaError_t stream_entry_state(int dev, int* num_sms, int** err);

// Makes the device of `mem` (device memory of the caller) current for the
// lifetime of the object.  `status` is not TB_OK, with the message set, if
// `mem` is not device memory.
class StreamEntry {
public:
    explicit StreamEntry(const void* mem, const char* what) {
        cudaPointerAttributes a{};
        cudaError_t e = cudaPointerGetAttributes(&a, mem);
        if (e != cudaSuccess) {
            cudaGetLastError();  // not left behind for the caller's next check
            status = (tb_status)report_error(e == cudaErrorNoDevice ? TB_ERR_NO_DEVICE : TB_ERR_CUDA, "%s: %s", what,
                                             cudaGetErrorString(e));
            return;
        }
        if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
            status = (tb_status)report_error(TB_ERR_INVALID_ARGUMENT, "%s is not device memory", what);
            return;
        }
        e = cudaGetDevice(&prev_);
        if (e == cudaSuccess && prev_ != a.device) {
            e = cudaSetDevice(a.device);
            if (e == cudaSuccess) switched_ = true;
        }
        if (e == cudaSuccess) e = stream_entry_state(a.device, &num_sms, &err);
        if (e != cudaSuccess)
            status = (tb_status)report_error(TB_ERR_CUDA, "selecting device %d: %s", a.device, cudaGetErrorString(e));
    }
    ~StreamEntry() {
        if (switched_) cudaSetDevice(prev_);
    }
    StreamEntry(const StreamEntry&) = delete;
    StreamEntry& operator=(const StreamEntry&) = delete;

    tb_status status = TB_OK;
    int num_sms = 0;
    int* err = nullptr;

private:
    int prev_ = 0;
    bool switched_ = false;
};

#define TB_ENTRY_CHECK(cond, ...)                                                             \
    do {                                                                                      \
        if (!(cond)) return (tb_status)::tb::report_error(TB_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
    } while (0)

inline tb_status launch_status(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return TB_OK;
    return (tb_status)report_error(e == cudaErrorNotSupported ? TB_ERR_UNSUPPORTED : TB_ERR_CUDA, "%s: %s", what,
                                   cudaGetErrorString(e));
}

// Lets kernel K have `smem` bytes of dynamic shared memory, once per kernel and
// device (the calls cost more than a launch); K names the kernel, each has its own
// record.  regs: the registers of a thread that K must have been built with.
template <auto K>
cudaError_t kernel_attributes(size_t smem, int regs = 0) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done.load(std::memory_order_relaxed) >> dev & 1)) return e;
    e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    if (regs) {
        // setmaxnreg moves registers within what the CTA was launched with: with
        // fewer than planned the warps that ask for more would wait for them
        cudaFuncAttributes a{};
        e = cudaFuncGetAttributes(&a, K);
        if (e != cudaSuccess) return e;
        if (a.numRegs != regs) return cudaErrorNotSupported;
    }
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return cudaSuccess;
}

inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace tb
