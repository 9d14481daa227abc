// Shared by the attention kernels over packed sequences and over a paged cache
// (attn_packed.hip, attn_paged.hip): element types, 16-byte loads, the status
// flag that dgm_end reads.
#pragma once
#include "attn_index.hpp"
#include "common.hpp"

namespace dgm_attn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kNegInf = -__builtin_huge_valf();

// Bits of the device's sequence flag (dgm_gpu::seq_flag).
constexpr uint32_t kBadStarts = 1, kBadPages = 2;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }   // 2^x to about an ulp
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }

// For a scope: the context's device is the current one.
struct OnDevice {
    int before = -1;
    bool moved = false;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) {
            err = hipSetDevice(device);
            moved = err == hipSuccess;
        }
    }
    ~OnDevice() {
        if (moved) (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

inline int type_bytes(int64_t type) { return type == DGM_TYPE_F32 ? 4 : type == DGM_TYPE_BF16 ? 2 : 0; }

// starts[0 .. nseq] is in order and within [0, rows]; else the flag is set. Run by one workgroup.
__device__ inline void check_starts(const int32_t* starts, int64_t nseq, int64_t rows, uint32_t* flag) {
    bool bad = false;
    for (int64_t i = threadIdx.x; i <= nseq; i += blockDim.x) {
        const int32_t s = starts[i];
        bad = bad || s < 0 || s > rows || (i > 0 && s < starts[i - 1]);
    }
    if (bad) atomicOr(flag, kBadStarts);
}

}  // namespace dgm_attn
