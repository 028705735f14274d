// A CUDA runtime without a GPU, as far as the page operations' host side calls
// it: allocations are the host's (and can be made to fail), copies and launches
// do nothing.
#include <cuda_runtime_api.h>

#include <cstdlib>

static int allowed = -1;                    // allocations before one fails; below 0: all succeed
static int launches = 0;

static cudaError_t get(void **p, size_t bytes) {
    if (allowed == 0) return cudaErrorMemoryAllocation;
    if (allowed > 0) --allowed;
    *p = std::malloc(bytes);
    return *p ? cudaSuccess : cudaErrorMemoryAllocation;
}

extern "C" {

cudaError_t CUDARTAPI cudaMalloc(void **p, size_t n) { return get(p, n); }
cudaError_t CUDARTAPI cudaHostAlloc(void **p, size_t n, unsigned) { return get(p, n); }
cudaError_t CUDARTAPI cudaFree(void *p) { return std::free(p), cudaSuccess; }
cudaError_t CUDARTAPI cudaFreeHost(void *p) { return std::free(p), cudaSuccess; }
cudaError_t CUDARTAPI cudaEventCreateWithFlags(cudaEvent_t *e, unsigned) { return *e = (cudaEvent_t)1, cudaSuccess; }
cudaError_t CUDARTAPI cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaEventSynchronize(cudaEvent_t) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaGetDevice(int *d) { return *d = 0, cudaSuccess; }
cudaError_t CUDARTAPI cudaSetDevice(int) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaGetLastError(void) { return cudaSuccess; }
const char *CUDARTAPI cudaGetErrorString(cudaError_t) { return "an error of the runtime without a GPU"; }
cudaError_t CUDARTAPI cudaMemcpyAsync(void *, const void *, size_t, cudaMemcpyKind, cudaStream_t) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaLaunchKernelExC(const cudaLaunchConfig_t *, const void *, void **) {
    return ++launches, cudaSuccess;
}
// what the compiler's registration code calls
cudaError_t CUDARTAPI cudaLaunchKernel(const void *, dim3, dim3, void **, size_t, cudaStream_t) { return cudaSuccess; }
void **CUDARTAPI __cudaRegisterFatBinary(void *) { return nullptr; }
void CUDARTAPI __cudaRegisterFatBinaryEnd(void **) {}
void CUDARTAPI __cudaUnregisterFatBinary(void **) {}
void CUDARTAPI __cudaRegisterFunction(void **, const char *, char *, const char *, int, uint3 *, uint3 *, dim3 *, dim3 *,
                                      int *) {}
unsigned CUDARTAPI __cudaPushCallConfiguration(dim3, dim3, size_t, cudaStream_t) { return 0; }
cudaError_t CUDARTAPI __cudaPopCallConfiguration(dim3 *, dim3 *, size_t *, void *) { return cudaSuccess; }
cudaError_t CUDARTAPI __cudaGetKernel(cudaKernel_t *, const void *) { return cudaSuccess; }
cudaError_t CUDARTAPI __cudaLaunchKernel(cudaKernel_t, dim3, dim3, void **, size_t, cudaStream_t) { return cudaSuccess; }
char CUDARTAPI __cudaInitModule(void **) { return 0; }


void host_allow(int n) { allowed = n; }
int host_launches(void) { return launches; }

}  // extern "C"
