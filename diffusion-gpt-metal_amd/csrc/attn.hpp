// Shared by the attention kernels over packed sequences and over a paged cache
// (attn_packed.hip, attn_paged.hip): element types, 16-byte loads, what
// dgm_end is told.
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

// Words of the context's report (dgm_gpu::seq_report), which dgm_end reads.
constexpr int kBadStarts = 0, kBadPages = 1, kBadTokens = 2;

__device__ __forceinline__ void report(uint32_t* words, int which) {
    __hip_atomic_store(words + which, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

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

// Three bf16 pieces of 8 bits each (the high halves of the words) that add up to a
// finite x exactly, the high one first: x's low 16 bits cut off, not rounded, so that none overflows.
__device__ __forceinline__ void split3(float x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    hi = __float_as_uint(x);
    const float r = x - __uint_as_float(hi & 0xffff0000u);
    mid = __float_as_uint(r);
    lo = __float_as_uint(r - __uint_as_float(mid & 0xffff0000u));
}

// What split8 makes of an infinity or NaN among values that it takes in three pieces:
// kSpoils: NaN in the later ones. The other two leave it the last piece alone, which
// meets the other operand's first one only: kRare by a branch (fewer
// instructions), kSelect without one (fewer registers).
enum NonFinite { kSpoils, kRare, kSelect };

// 8 values as PIECES bf16 pieces: the value rounded, that and what rounding left, or split3's.
template <int PIECES, NonFinite kAny>
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
            if constexpr (kAny == kSelect) {
                const float y0 = fabsf(x[j]) < __builtin_huge_valf() ? x[j] : 0.0f;
                const float y1 = fabsf(x[j + 1]) < __builtin_huge_valf() ? x[j + 1] : 0.0f;
                split3(y0, a[0], a[1], a[2]);
                split3(y1, b[0], b[1], b[2]);
                a[2] = __float_as_uint(__uint_as_float(a[2]) + (x[j] - y0));
                b[2] = __float_as_uint(__uint_as_float(b[2]) + (x[j + 1] - y1));
            } else {
                split3(x[j], a[0], a[1], a[2]);
                split3(x[j + 1], b[0], b[1], b[2]);
            }
#pragma unroll
            for (int p = 0; p < 3; ++p) w[p][j / 2] = __builtin_amdgcn_perm(b[p], a[p], 0x07060302u);
        }
        if constexpr (kAny == kRare) {
            float t = 0.0f;   // NaN if any value is not finite
#pragma unroll
            for (int j = 0; j < 8; ++j) t = __builtin_fmaf(x[j], 0.0f, t);
            if (t != t) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = x[j];
                    if (fabsf(y) < __builtin_huge_valf()) continue;
                    const uint32_t keep = j % 2 ? 0x0000ffffu : 0xffff0000u;
                    const uint32_t as = y != y ? 0x7fc07fc0u : y > 0.0f ? 0x7f807f80u : 0xff80ff80u;
                    w[0][j / 2] &= keep;
                    w[1][j / 2] &= keep;
                    w[2][j / 2] = (w[2][j / 2] & keep) | (as & ~keep);
                }
            }
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

// starts[0 .. nseq] is in order and within [0, rows]; else it is reported. Run by one workgroup.
__device__ inline void check_starts(const int32_t* starts, int64_t nseq, int64_t rows, uint32_t* words) {
    bool bad = false;
    for (int64_t i = threadIdx.x; i <= nseq; i += blockDim.x) {
        const int32_t s = starts[i];
        bad = bad || s < 0 || s > rows || (i > 0 && s < starts[i - 1]);
    }
    if (bad) report(words, kBadStarts);
}

}  // namespace dgm_attn
