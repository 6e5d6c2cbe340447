/* ckq_int8.hpp - what the int8 rows' kernels share on the host. */
#pragma once
#include <hip/hip_runtime.h>

template <class T> struct i8_as { typedef T type; };

/* A launch in one call of the runtime; <<<>>> makes three (2.45 us of host time each and 2.25), and hipGetLastError would return what an earlier call has left. */
template <class... P>
static inline int i8_launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t s, typename i8_as<P>::type... args)
{
    void *p[] = {(void *)&args...};
    const hipError_t rc = hipLaunchKernel((const void *)kernel, grid, block, p, 0, s);
    if (rc != hipSuccess) (void)hipGetLastError();            /* reported here, not by the caller's next call too */
    return (int)rc;
}
