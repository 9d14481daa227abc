// Shared by the operators of a training step around its linears (layer_norm.hip,
// loss.hip, embed_rows.hip, adam_many.hip): rows of any length and alignment in
// 16-byte pieces, and reductions over the lanes that share a row.
#pragma once
#include "attn.hpp"
#include "common.hpp"
#include "dit_rows.hpp"

namespace dgm_step {

using dgm_attn::kBadTokens;
using dgm_attn::kNegInf;
using dgm_attn::OnDevice;
using dgm_attn::report;
using dgm_attn::type_bytes;

// Elements of a 16-byte piece.
template <typename T>
constexpr int kVec = 16 / int(sizeof(T));

// N elements at any address that is aligned to one: the memory system takes 16-byte accesses
// at 2- and 4-byte boundaries, so rows of odd lengths need no other path.
template <typename T, int N>
struct Piece {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
using piece_t = typename Piece<T, N>::type;

// Elements [c, c + N) of a row of `cols`; `fill` behind its end.
template <int N, typename T>
__device__ __forceinline__ void load_piece(const T* row, int c, int cols, float (&x)[N], float fill = 0.0f) {
    if (c + N <= cols) {
        const piece_t<T, N> v = *reinterpret_cast<const piece_t<T, N>*>(row + c);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = float(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = c + j < cols ? float(row[c + j]) : fill;
    }
}

template <int N, typename T>
__device__ __forceinline__ void store_piece(T* row, int c, int cols, const float (&x)[N]) {
    if (c + N <= cols) {
        piece_t<T, N> v;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = T(x[j]);
        *reinterpret_cast<piece_t<T, N>*>(row + c) = v;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c + j < cols) row[c + j] = T(x[j]);
    }
}

// A row of `cols` elements as whole pieces, from its first element at a multiple of 4 bytes on (pieces at
// odd multiples of 2 take more cycles: 8192 bf16 rows of 50257 logits 356 us that way, 304 this), and the up to 8 elements
// before and behind those, one to a lane.
struct Span {
    int head, whole, last;   // elements before the pieces; pieces; this lane's single element, -1 for none
};
template <typename T>
__device__ __forceinline__ Span span_of(const T* row, int cols, int lane) {
    Span s;
    s.head = sizeof(T) == 2 ? int(reinterpret_cast<uintptr_t>(row) >> 1 & 1) : 0;
    s.whole = (cols - s.head) / kVec<T>;
    const int rest = cols - s.head - s.whole * kVec<T>;
    s.last = lane < rest ? s.head + s.whole * kVec<T> + lane : lane == rest && s.head ? 0 : -1;
    return s;
}

__device__ __forceinline__ float wave64_max(float v) {
    v = dgm_rows::row16_max(v);
    const auto r16 = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                      false, false);
    v = fmaxf(__builtin_bit_cast(float, uint32_t(r16[0])), __builtin_bit_cast(float, uint32_t(r16[1])));
    const auto r32 = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                      false, false);
    return fmaxf(__builtin_bit_cast(float, uint32_t(r32[0])), __builtin_bit_cast(float, uint32_t(r32[1])));
}

// Reductions over the TEAM lanes that share a row (16, 64, or a workgroup of TEAM
// threads): every lane gets the same bits, and the order of a sum is fixed. `slot`: TEAM / 64
// floats of LDS of this reduction's own; a workgroup may use it again behind its next other reduction.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* slot) {
    if constexpr (TEAM == 16) return dgm_rows::row16_sum(v);
    v = dgm_rows::wave64_sum(v);
    if constexpr (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < TEAM / 64; ++w) v += slot[w];
    }
    return v;
}
template <int TEAM>
__device__ __forceinline__ float team_max(float v, float* slot) {
    if constexpr (TEAM == 16) return dgm_rows::row16_max(v);
    v = wave64_max(v);
    if constexpr (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < TEAM / 64; ++w) v = fmaxf(v, slot[w]);
    }
    return v;
}

constexpr int threads_of(int team) { return team > 256 ? team : 256; }

}  // namespace dgm_step
