/*
 * Host-side helpers shared by the entry points outside pgqa_decode.cu (defined there).
 */
#ifndef PGQA_HOST_H_
#define PGQA_HOST_H_

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/pgqa.h"

namespace pgqa {

/* Bits of the device error word. */
enum : int32_t {
    kDevErrTimeout = 1, kDevErrBadPage = 2, kDevErrBadSeqlen = 4, kDevErrBadPosition = 8
};

/* The current device, checked to be an sm_100 one; its SM count and shared-memory limit. */
int host_device(int* dev, int* sms, int* smem_optin);

/* Device address of the library's static error word on the current device `dev`: it is
 * never freed, so a captured graph may hold it.  Read by pgqa_check_device_error(NULL). */
int host_error_word(int dev, int32_t** err);

/* Records `st` for pgqa_last_status and returns it. */
int host_set_status(int st);

/* Whether launches are programmatic dependents (PGQA_NO_PDL unset). */
bool host_pdl();

/* cuTensorMapEncodeTiled, or NULL when the driver does not export it. */
void* host_encode_tiled();

/* Allows a kernel `bytes` of dynamic shared memory on device `dev`.  `bytes` is the most that
 * any of its launches takes there, the same in every call, so that neither the order of the
 * calls nor two threads at once can leave a lower limit behind; `done` is the caller's
 * per-kernel table of devices already seen to. */
constexpr int kHostMaxDevices = 64;
typedef std::atomic<bool> HostSmemDone[kHostMaxDevices];
template <typename K>
int host_smem_limit(K kernel, int dev, int bytes, HostSmemDone& done) {
    if (dev < 0 || dev >= kHostMaxDevices) return PGQA_ERR_NO_DEVICE;
    if (done[dev].load(std::memory_order_acquire)) return PGQA_OK;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        cudaGetLastError();
        return PGQA_ERR_CUDA;
    }
    done[dev].store(true, std::memory_order_release);
    return PGQA_OK;
}

/* One launch on `stream`, in clusters of `cluster` CTAs, as a programmatic dependent: every kernel launched through here
 * executes griddepcontrol.wait in all of its CTAs before it touches memory. */
template <typename K, typename... Args>
int host_launch(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, int cluster,
                const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = host_pdl() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)cluster;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        cudaGetLastError();
        return PGQA_ERR_CUDA;
    }
    return PGQA_OK;
}

inline bool host_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

/* log2 of a power of two, else -1 */
inline int32_t host_shift(int64_t P) {
    for (int s = 0; s < 31; ++s)
        if (((int64_t)1 << s) == P) return s;
    return -1;
}

/* The checks every paged operator makes of its pools and table. */
inline int host_check_pages(int64_t B, int64_t Hkv, int64_t D, int64_t P, int64_t num_pages, int64_t bt_stride) {
    if (B <= 0 || Hkv <= 0 || P <= 0 || num_pages <= 0 || bt_stride <= 0 || D <= 0) return PGQA_ERR_BAD_SHAPE;
    if (B > INT32_MAX || Hkv > INT32_MAX || bt_stride > INT32_MAX) return PGQA_ERR_BAD_SHAPE;
    if (D != 128 || P % 16 != 0) return PGQA_ERR_UNSUPPORTED;
    if (num_pages >= ((int64_t)1 << 31) / P) return PGQA_ERR_UNSUPPORTED;  // token slots are 31-bit
    if (bt_stride >= ((int64_t)1 << 31) / P) return PGQA_ERR_UNSUPPORTED;
    return PGQA_OK;
}

}  // namespace pgqa

#endif  // PGQA_HOST_H_
