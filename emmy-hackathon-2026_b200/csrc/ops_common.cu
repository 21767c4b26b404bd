#include "ops_common.cuh"

static thread_local char g_error[512];

int ops_fail(int status, const char *format, ...) {
    va_list args;
    va_start(args, format);
    vsnprintf(g_error, sizeof g_error, format, args);
    va_end(args);
    return status;
}

int ops_cuda(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return 0;
    return ops_fail((int)e, "%s: %s", what, cudaGetErrorString(e));
}

int ops_sm_count(int device, int *out) {
    static int counts[64];
    if (device < 0 || device >= 64) return ops_fail(EMMY_RT_EINVAL, "device %d", device);
    int n = __atomic_load_n(&counts[device], __ATOMIC_RELAXED);
    if (!n) {
        cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return ops_cuda(e, "device attribute");
        __atomic_store_n(&counts[device], n, __ATOMIC_RELAXED);
    }
    *out = n;
    return 0;
}

EMMY_EXPORT const char *emmy_ops_last_error(void) { return g_error; }

EMMY_EXPORT int emmy_ops_current_device(int *device) {
    if (!device) return ops_fail(EMMY_RT_EINVAL, "no place for the device");
    return ops_cuda(cudaGetDevice(device), "current device");
}
