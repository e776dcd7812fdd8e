// Host-side helpers shared by the translation units of the library (defined in capi.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

typedef CUresult (*CfEncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// the driver's cuTensorMapEncodeTiled, looked up once through the runtime (nullptr if unavailable)
CfEncodeTiledFn cf_host_encode_fn();
// records the thread-local message behind cf_last_error() and returns `code`
int cf_host_fail(int code, const char* fmt, ...);
// CF_ERR_INVALID (with a message naming `what`) while `st` is being captured, CF_OK otherwise
int cf_host_refuse_in_capture(cudaStream_t st, const char* what);
// Whether kernels whose CTAs wait for one another are launched cooperatively, so that the driver checks that all find room: CFB200_COOPERATIVE (0 or 1)
// if it is set, else yes, but for a process that Nsight tools run: ncu ended a cooperative launch of clusters with a GPU fault.  Plain launches
// are as good where nothing else runs on the GPU.
bool cf_host_cooperative();
// status word of the batched Llama path on device `dev` (0 when unused); cleared when it was set
int cf_host_lb_probe_status(int dev, int* status);
// status word of the 4-bit cache's kernels on the current device (0 when unused); cleared when it was set
int cf_host_kv4_probe_status(int* status);
