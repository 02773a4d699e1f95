// What the translation units of libreels_lowvram.so share on the host side:
// status and message of the C entry points, binding of a buffer's device for
// the length of a call, tensor maps and programmatic launches.  Implemented
// in lowvram.cu, which holds the per-thread and per-device state.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdlib.h>

#include <string>

namespace reels {

// Set the thread's message and return the status (REELS_EINVAL, REELS_EDEVICE, REELS_OK).
int host_fail(const std::string &msg);
int host_fail_dev(const std::string &msg);
int host_ok(int path);
void host_count_launch();

// Makes the device that owns `ptr` current while the object lives and puts
// the caller's context back afterwards.
class HostCall {
  public:
    HostCall() = default;
    ~HostCall();
    HostCall(const HostCall &) = delete;
    HostCall &operator=(const HostCall &) = delete;
    int bind(const void *ptr);  // REELS_OK, or the status to return
    int device = -1;
    int sms = 148;
    unsigned *status = nullptr;  // the device's status word

  private:
    void *scope_ = nullptr;
};

// Tensor map of a 4-d 16-bit array [n3][n2][n1][n0] with byte strides of the
// outer three dimensions, 128-byte swizzle, out-of-range elements read as 0.
int host_tmap_4d(CUtensorMap *tm, const void *base, bool bf16, const uint64_t (&n)[4], const uint64_t (&stride)[3],
                 const uint32_t (&box)[4]);

// Launch with programmatic stream serialization (see griddep_wait in
// common.cuh).  REELS_NO_PDL=1 launches everything in plain stream order.
template <typename... KArgs, typename... Args>
cudaError_t host_launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                            Args... args) {
    static const bool pdl = [] {
        const char *e = getenv("REELS_NO_PDL");
        return !(e && atoi(e) != 0);
    }();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace reels
