// Makes a context's GPU current for the duration of a call and puts the caller's current device back afterwards.
#pragma once
#include <cuda_runtime.h>

struct S1DeviceGuard {
    int before = -1;
    bool ok = false;
    explicit S1DeviceGuard(int device) {
        ok = cudaGetDevice(&before) == cudaSuccess;
        if (ok && before != device) ok = cudaSetDevice(device) == cudaSuccess;
        else before = -1;
    }
    ~S1DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
    S1DeviceGuard(const S1DeviceGuard&) = delete;
    S1DeviceGuard& operator=(const S1DeviceGuard&) = delete;
};
