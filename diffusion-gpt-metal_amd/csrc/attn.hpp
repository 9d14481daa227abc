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

// Three bf16 pieces of 8 bits each that add up to x exactly, the high one first
// (x's low 16 bits cut off, not rounded, so that none overflows). An infinity or
// NaN is the last piece, which meets the other operand's first one alone.
__device__ __forceinline__ void split3(float x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    const float fin = fabsf(x) < __builtin_huge_valf() ? x : 0.0f;
    hi = __float_as_uint(fin) & 0xffff0000u;
    const float r = fin - __uint_as_float(hi);
    mid = __float_as_uint(r) & 0xffff0000u;
    lo = __float_as_uint(r - __uint_as_float(mid) + (x - fin)) & 0xffff0000u;
}

// 8 values as PIECES bf16 pieces: the value rounded, that and what rounding left, or split3's.
template <int PIECES>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&o)[PIECES]) {
    if constexpr (PIECES < 3) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            o[0][j] = __bf16(x[j]);
            if constexpr (PIECES == 2) o[1][j] = __bf16(x[j] - float(o[0][j]));
        }
    } else {
        u32x4 w[3];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            uint32_t a[3], b[3];
            split3(x[j], a[0], a[1], a[2]);
            split3(x[j + 1], b[0], b[1], b[2]);
#pragma unroll
            for (int p = 0; p < 3; ++p) w[p][j / 2] = __builtin_amdgcn_perm(b[p], a[p], 0x07060302u);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) o[p] = __builtin_bit_cast(bf16x8, w[p]);
    }
}

template <typename IN>
__device__ __forceinline__ void load8(const IN* p, float (&x)[8]) {
    if constexpr (sizeof(IN) == 4) {
        const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    } else {
        const bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = float(a[i]);
    }
}

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
