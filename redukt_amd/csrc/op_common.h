// op_common.h — shared by the operators on caller tensors (redukt_ops.h): element types, the
// device of a call, launches.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/redukt_backend.h"
#include "../../include/redukt_ops.h"

namespace rdk {
namespace {

constexpr uint32_t kMaxOpRows = 65536;      // entries or sequences of a call

inline uint32_t op_elem_bytes(uint32_t dtype) { return dtype == REDUKT_OP_F32 ? 4 : 2; }

inline bool op_aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }

// Makes the device that owns `p` the current one until the end of the scope.  ok is false
// where p is no device memory.
class OpDevice {
public:
    explicit OpDevice(const void* p) {
        hipPointerAttribute_t a{};
        if (hipPointerGetAttributes(&a, p) != hipSuccess) {
            (void)hipGetLastError();      // the refusal is this call's answer, not the next call's error
            return;
        }
        if (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged) return;
        if (hipGetDevice(&was_) != hipSuccess) return;
        if (a.device != was_) {
            if (hipSetDevice(a.device) != hipSuccess) return;
            set_ = true;
        }
        ok = true;
    }
    ~OpDevice() {
        if (set_) (void)hipSetDevice(was_);
    }
    OpDevice(const OpDevice&) = delete;
    OpDevice& operator=(const OpDevice&) = delete;
    bool ok = false;

private:
    int was_ = 0;
    bool set_ = false;
};

// Whether a launch of `groups` workgroups of `threads` is one that the runtime takes (threads along a dimension fit 32 bits).
inline bool op_grid_ok(uint64_t groups, uint32_t threads) { return groups <= 0xffffffffull / threads; }

template <typename Args>
inline int32_t op_launch(const void* fn, dim3 grid, dim3 block, size_t lds, void* stream, Args& args) {
    void* p[] = {(void*)&args};
    if (hipLaunchKernel(fn, grid, block, p, lds, (hipStream_t)stream) == hipSuccess) return BACKEND_OK;
    (void)hipGetLastError();
    return BACKEND_FORWARD_FAILED;
}

// N consecutive elements of an activation row as f32; p aligned to their size, 16 bytes at most.
template <typename T, int N>
__device__ __forceinline__ void op_load(const T* p, float (&v)[N]) {
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int kPer = 16 / sizeof(T);
    if constexpr (N % kPer == 0) {
#pragma unroll
        for (int i = 0; i < N / kPer; i++) {
            const vec x = ((const vec*)p)[i];
#pragma unroll
            for (int j = 0; j < kPer; j++) v[i * kPer + j] = (float)x[j];
        }
    } else {
        typedef T part __attribute__((ext_vector_type(N)));
        const part x = *(const part*)p;
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = (float)x[j];
    }
}

}  // namespace
}  // namespace rdk
