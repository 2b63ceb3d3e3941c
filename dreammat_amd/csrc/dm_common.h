// Common helpers for the dreammat HIP library (gfx950 only; no CUDA/HIP dual paths).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define DM_OK 0
#define DM_ERR_ARG (-1)
#define DM_ERR_WORKSPACE (-2)
#define DM_ERR_UNSUPPORTED (-3)

#define DM_HD __host__ __device__ __forceinline__

// hipGetLastError() is per-thread and sticky across libraries: a benign error left behind by another
// component of the process (PyTorch probing a feature, ...) must not be reported as ours, so every
// entry point clears it first (DM_ENTER) and checks only its own launches (DM_LAUNCH_CHECK).
#define DM_ENTER() do { (void)hipGetLastError(); } while (0)

// Launch-check: positive return = hipError_t.
#define DM_LAUNCH_CHECK()                          \
    do {                                           \
        hipError_t e__ = hipGetLastError();        \
        if (e__ != hipSuccess) return (int)e__;    \
    } while (0)

#define DM_HIP(expr)                               \
    do {                                           \
        hipError_t e__ = (expr);                   \
        if (e__ != hipSuccess) return (int)e__;    \
    } while (0)

// More than 64 KB of dynamic LDS for a kernel: asked for once per device (`devices`: the kernel's static record of them, one bit each).
static inline hipError_t dm_dynamic_lds(const void* kernel, int bytes, unsigned long long& devices) {
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (__atomic_load_n(&devices, __ATOMIC_RELAXED) & bit) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) __atomic_fetch_or(&devices, bit, __ATOMIC_RELAXED);
    return e;
}

static inline int dm_div_up(long long a, long long b) { return (int)((a + b - 1) / b); }
