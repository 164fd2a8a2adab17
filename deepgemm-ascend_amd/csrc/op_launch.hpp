// Launching of the operators around the GEMMs (moe.hip, mx_quant.hip, linear_xent.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "dg_common.hpp"
#include "../../include/deep_gemm_amd.h"

extern "C" __attribute__((visibility("hidden"))) int dg_set_error(const char* msg);

namespace dg {

// csrc/status.hip: device address of the sticky error words; nullptr if they could not be allocated
uint32_t* status_words();
uint32_t* status_words_if_ready();

// The words for a launch on `st`: a stream being captured allocates nothing.
inline uint32_t* status_words_for(hipStream_t st) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &s) != hipSuccess) (void)hipGetLastError();
    return s == hipStreamCaptureStatusNone ? status_words() : status_words_if_ready();
}

// Extents of the operators: indices of tiles that end past an extent stay within 32 bits.
constexpr int64_t kMaxExtent = int64_t(1) << 30;

inline bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Workgroups [0, grid) of a kernel whose parameters hold the first one of a launch (vbase).  `cus` > 0 (set_num_sms
// below the device's count): at most that many at a time, in launches one after another.
template <typename P>
int launch_op(void (*kernel)(const P), int64_t grid, unsigned threads, P p, hipStream_t st, int cus, unsigned lds = 0) {
    if (grid > 0x7fffffffLL) return dg_set_error("too many workgroups");
    const int64_t most = cus > 0 ? cus : std::max<int64_t>(grid, 1);
    for (int64_t base = 0; base < grid; base += most) {
        p.vbase = (int)base;
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(most, grid - base)), dim3(threads), lds, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            dg_set_error(hipGetErrorString(e));
            return DG_ELAUNCH;
        }
    }
    return DG_OK;
}

}  // namespace dg
