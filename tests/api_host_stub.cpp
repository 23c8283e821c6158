/* A host with no GPU for the dispatch layer: the runtime calls plow_moe_create makes, answered from the heap, and the
 * per-device set-up. Linked with plow_amd/csrc/api.hip so that a descriptor's checks run on a CPU; kernel launchers
 * stay undefined (symbols are bound when called, and a refused descriptor calls none). */
#include <hip/hip_runtime.h>

#include <cstdlib>

#include "../plow_amd/csrc/tuning.h"

extern "C" {
hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) { *p = malloc(n); return *p ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void* p) { free(p); return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { *s = (hipStream_t)malloc(1); return hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t s) { free((void*)s); return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { *e = (hipEvent_t)malloc(1); return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t e) { free((void*)e); return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
}
int plow_moe_device_setup(int) { return 0; }
const PlowMoeTuning& plow_moe_tuning() {
    static PlowMoeTuning t;
    return t;
}
