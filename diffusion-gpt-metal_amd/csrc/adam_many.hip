// AdamW over many tensors in one launch, the norm of all their gradients, and
// moments in 8 bits. No counterpart in the reference, which dispatches adam (and quantize)
// once a parameter (src/GPT.swift:193-218) and waits for the norm on the host.
//
// A plan in device memory describes the tensors and cuts them into chunks of kChunk elements, one
// workgroup's work each, a thread 8 elements that follow one another; so groups of codes (8 to 512
// elements) and blocks of 8-bit moments (256) are runs of lanes. Every fp32 operation is rounded on its own
// (fp contraction off), as in adamw: with 32-bit moments the results are dgm_adam's and dgm_adam_quantize's bits.
//
// 8-bit moments, in blocks of 256 elements of a tensor with a scale each:
//   m: code c = -127 .. 127 stands for c |c| sm, sm = max|m| / 127^2
//   v: code c = 0 .. 255 stands for (c^2 rv)^2, rv = sqrt(max v) / 255^2
// The code is that of the nearest root (ties up), decided exactly: c and c + 1 meet where
// |m| 127^2 = max|m| (c + 1/2)^2, whose sides are exact in 64 bits (24 + 14 and 24 + 16 bits), and where
// v 255^4 = max v (c + 1/2)^4 (to 2^-53). A hardware root says which border to ask. A v that is not 0 keeps a
// code of 1 at least, and that a value above 0, so that its steps do not divide by eps alone; but a block whose largest is
// below 2^-120 counts as zeros. An infinity or NaN makes its block's scale NaN.
//
// Nearest codes alone would hold what moves by less than half a code a step, and for good: with b1 = 0.9 an m of c <= 9
// without gradients, whose weight then moves on without end, and a v far below its gradients' squares, whose weight's
// steps stay several times too large. Two codes that stay are therefore moved by one:
//   m toward 0 where |m| shrank and sm did not, nor grew by over an eighth (that moves the codes' places, so that one
//     that stays says nothing), c (1 - b1) < 1 (larger codes follow a decay) and v's code times (1 - b2) is below 4. It is
//     some steps after the last gradient (v decays by rounding to 2 / (1 - b2)), and always where b2 > 0.984. Weights with
//     gradients keep their nearest codes, which a push at every shrinking would draw toward 0.
//   v away from 0 where it grew to over 9 - 8 b2 of itself, as by g^2 > 9 v, and rv did not: a step is then soon at most
//     3 times AdamW's. Nearer ones keep the nearest code: pushed at every growth, v would end at its largest g^2.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "adam_math.hpp"
#include "quant_math.hpp"
#include "step.hpp"

#pragma clang fp contract(off)

namespace {

using namespace dgm_step;
using dgm::AdamArgs;

constexpr int kThreads = 256, kEach = 8, kChunk = kThreads * kEach, kBlock = 256;
constexpr int kNormBlocks = 2048;   // partial sums of the norm
constexpr float kLeast = 0x1p-120f;

// A tensor in the plan, and a chunk: elements [at, at + kChunk) of tensor `tensor`.
struct Tensor {
    float* w;
    const float* g;
    void *m, *v;
    float *ms, *vs;
    void* q;
    float* scale;
    int64_t n, flat;   // elements, and those of the tensors before, each rounded up to a block
    int32_t decay, bits, group, vec;
};
struct Chunk {
    int32_t tensor, index;
};

// The tensors' addresses come out of memory: said to be global ones, or the accesses would be flat.
#define DGM_GLOBAL __attribute__((address_space(1)))
typedef DGM_GLOBAL float gfloat;
typedef DGM_GLOBAL uint8_t gbyte;
typedef dgm_attn::f32x4 f32x4;
typedef dgm_attn::u32x2 u32x2;

// 8 elements from p + at on (`left` of them there are), as 16-byte accesses where `vec`.
__device__ __forceinline__ void get8(const float* base, int64_t at, int64_t left, bool vec, float (&x)[8]) {
    const gfloat* p = (const gfloat*)base + at;
    if (vec && left >= 8) {
        const f32x4 a = *(const DGM_GLOBAL f32x4*)p, b = *(const DGM_GLOBAL f32x4*)(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = a[j];
            x[4 + j] = b[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = j < left ? p[j] : 0.0f;
    }
}
__device__ __forceinline__ void put8(float* base, int64_t at, int64_t left, bool vec, const float (&x)[8]) {
    gfloat* p = (gfloat*)base + at;
    if (vec && left >= 8) {
        *(DGM_GLOBAL f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
        *(DGM_GLOBAL f32x4*)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = x[j];
    }
}
__device__ __forceinline__ u32x2 get_codes(const void* base, int64_t at, int64_t left, bool vec) {
    const gbyte* p = (const gbyte*)base + at;
    if (vec && left >= 8) return *(const DGM_GLOBAL u32x2*)p;
    u32x2 w = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) w[j / 4] |= uint32_t(p[j]) << (8 * (j & 3));
    return w;
}
__device__ __forceinline__ void put_codes(void* base, int64_t at, int64_t left, bool vec, u32x2 c) {
    gbyte* p = (gbyte*)base + at;
    if (vec && left >= 8) {
        *(DGM_GLOBAL u32x2*)p = c;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) p[j] = uint8_t(c[j / 4] >> (8 * (j & 3)));
}
__device__ __forceinline__ int code_of(u32x2 c, int j, bool sign) {
    const uint32_t w = c[j / 4] >> (8 * (j & 3));
    return sign ? int(int8_t(w)) : int(uint8_t(w));
}

__device__ __forceinline__ float m_value(int c, float sm) { return float(c * abs(c)) * sm; }
// At least the smallest number of all where there is a code: squares of roots below 2^-74.5 would be 0. As bits, so that a NaN stays.
__device__ __forceinline__ float v_value(int c, float rv) {
    const float root = float(c * c) * rv;
    return __uint_as_float(max(__float_as_uint(root * root), min(__float_as_uint(root), 1u)));
}
// 8 of them: only scales below 2^-74 need to be looked at.
__device__ __forceinline__ void v_values(u32x2 codes, float rv, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int c = code_of(codes, j, false);
        const float root = float(c * c) * rv;
        v[j] = root * root;
    }
    if (rv < 0x1p-74f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v_value(code_of(codes, j, false), rv);
    }
}

// The bytes of w that are below n (up to 256), as their high bits.
__device__ __forceinline__ u32x2 bytes_below(u32x2 w, uint32_t n) {
    constexpr uint32_t kHigh = 0x80808080u;
    if (n > 128) return (~w | ~((w | kHigh) - (n - 128) * 0x01010101u)) & kHigh;
    return ~(w | ((w | kHigh) - n * 0x01010101u)) & kHigh;
}

// Codes from which on none are held: v's (where (c + 1/2)^4 is c^4 times that growth, and two more for roundings; 255 has no
// next one), v's of moments that are, and those moments' (1 at least).
struct Held {
    uint32_t grown, quiet, small;
    float growth;   // of a v with g^2 = 9 v
};
Held held_of(const AdamArgs& a) {
    Held l{0, 0, 1, std::max(9.0f - 8.0f * a.b2, 1.0f)};
    const double q = l.growth, n = q > 1.0 ? 0.5 / (std::sqrt(std::sqrt(q)) - 1.0) + 2.0 : 255.0;
    l.grown = n < 255.0 ? uint32_t(n) : 255;
    while (l.quiet < 256 && float(l.quiet) * (1.0f - a.b2) < 4.0f) ++l.quiet;
    while (l.small < 128 && float(l.small) * (1.0f - a.b1) < 1.0f) ++l.small;
    return l;
}

// The largest of a block of 32 lanes, as bits: an infinity or NaN is larger than what is finite.
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) x = max(x, uint32_t(__shfl_xor(int(x), off, 64)));
    return x;
}

// The nearest codes of 8 moments of a block whose largest is `top`, and the block's scale.
template <bool SECOND>
__device__ __forceinline__ u32x2 encode(const float (&x)[8], float top, float& scale) {
    constexpr float kMost = SECOND ? 255.0f : 127.0f;
    if (!(top >= kLeast && top < __builtin_huge_valf())) {
        scale = top < kLeast ? 0.0f : __builtin_nanf("");
        return u32x2{0, 0};
    }
    scale = SECOND ? sqrtf(top) * (1.0f / 65025.0f) : top * (1.0f / 16129.0f);
    const float inv = 1.0f / top;
    u32x2 w = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float y = fabsf(x[j]);
        float root = __builtin_amdgcn_sqrtf(y * inv);
        if constexpr (SECOND) root = __builtin_amdgcn_sqrtf(root);
        const float low = fminf(floorf(root * kMost), kMost - 1.0f);
        const double b = double(low) + 0.5, b2 = b * b;
        const bool up = SECOND ? double(y) * 4228250625.0 >= double(top) * (b2 * b2) : double(y) * 16129.0 >= double(top) * b2;
        int c = int(low) + (up ? 1 : 0);
        if (SECOND) c = y > 0.0f && c == 0 ? 1 : c;
        else c = x[j] < 0.0f ? -c : c;
        w[j / 4] |= (uint32_t(c) & 0xFFu) << (8 * (j & 3));
    }
    return w;
}

// Bound by memory: 28 bytes an element with moments of 32 bits, 16 with 8. 353 M elements in 388 tensors 1825 us (5.4
// TB/s) and 1132 (5.0); the character GPT's 0.8 M in 68, 6 us. A workgroup finds its work by two scalar loads, whatever the
// sizes; the 8-bit codes' roots and 64-bit borders stay below the memory's time (without a branch; IEEE roots would not), the
// search for codes that are held adds 5% (b2 0.999, where more may be: 10%). Nontemporal accesses were slower by up to 14% (8 bits)
// or no faster. With the linears' codes, 303 M elements of those: int8 1952 us in groups of 64, 1960 of 8, 1953 of 512 (5.3 TB/s),
// int4 1913; codes that do not lie at multiples of `bits` bytes take all of a tensor's accesses apart, 4360 us.
template <int STATE>
__global__ __launch_bounds__(kThreads) void adam_many_kernel(const Tensor* __restrict__ tensors, const Chunk* __restrict__ chunks,
                                                             const float* __restrict__ factor, AdamArgs a, Held l) {
    const Chunk ch = chunks[blockIdx.x];
    const Tensor t = tensors[ch.tensor];
    const float f = factor ? *factor : 1.0f;
    const int64_t at = int64_t(ch.index) * kChunk + threadIdx.x * kEach, left = t.n - at;   // may be below 0
    const bool vec = t.vec;
    AdamArgs args = a;
    args.wd = t.decay ? a.wd : 0.0f;
    float w[8], g[8], m[8], v[8];
    get8(t.w, at, left, vec, w);
    get8(t.g, at, left, vec, g);
    const int64_t block = at / kBlock;
    u32x2 cm0, cv0;   // what the moments were
    float sm0, rv0;
    if constexpr (STATE == 32) {
        get8(static_cast<const float*>(t.m), at, left, vec, m);
        get8(static_cast<const float*>(t.v), at, left, vec, v);
    } else {
        cm0 = get_codes(t.m, at, left, vec);
        cv0 = get_codes(t.v, at, left, vec);
        sm0 = left > 0 ? ((const gfloat*)t.ms)[block] : 0.0f;
        rv0 = left > 0 ? ((const gfloat*)t.vs)[block] : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = m_value(code_of(cm0, j, true), sm0);
        v_values(cv0, rv0, v);
    }
    if (factor) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = g[j] * f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) dgm::adam_elem(w[j], g[j], m[j], v[j], args);
    put8(t.w, at, left, vec, w);
    if constexpr (STATE == 32) {
        put8(static_cast<float*>(t.m), at, left, vec, m);
        put8(static_cast<float*>(t.v), at, left, vec, v);
    } else {
        uint32_t mm = 0, mv = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // Behind the end all are zeros: 0 / (0 + eps), and with an eps of 0 not a number.
            if (j >= left) m[j] = v[j] = 0.0f;
            mm = max(mm, __float_as_uint(m[j]) & 0x7FFFFFFFu);
            mv = max(mv, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        }
        mm = block_max(mm);
        mv = block_max(mv);
        float sm, rv;
        u32x2 cm = encode<false>(m, __uint_as_float(mm), sm), cv = encode<true>(v, __uint_as_float(mv), rv);
        // Codes that can be held, of 8 at once; then each of a lane that has some.
        u32x2 v_held = rv > 0.0f && rv <= rv0 ? bytes_below(cv ^ cv0, 1) & bytes_below(cv, l.grown) : u32x2{0, 0};
        if (v_held[0] | v_held[1]) {
            u32x2 up = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) up[j / 4] |= v[j] > l.growth * v_value(code_of(cv, j, false), rv0) ? 1u << (8 * (j & 3)) : 0u;
            cv += up & (v_held >> 7);
        }
        u32x2 m_held = sm >= sm0 && sm <= 1.125f * sm0 ? bytes_below(cm ^ cm0, 1) & bytes_below(cv, l.quiet) : u32x2{0, 0};
        if (m_held[0] | m_held[1]) {
            m_held &= bytes_below(cm, l.small) | bytes_below(~cm, l.small - 1);   // c >= 0; |c| - 1 of c < 0
            u32x2 down = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) down[j / 4] |= fabsf(m[j]) < fabsf(m_value(code_of(cm, j, true), sm0)) ? 1u << (8 * (j & 3)) : 0u;
            down &= m_held >> 7;
            // A byte above 0 less 1, one below 0 and 1 (-1: 0, without a carry into the next).
            const u32x2 below0 = cm >> 7 & 0x01010101u;
            cm -= down & ~below0;
            cm = ((cm & 0x7F7F7F7Fu) + (down & below0)) ^ (cm & 0x80808080u);
        }
        put_codes(t.m, at, left, vec, cm);
        put_codes(t.v, at, left, vec, cv);
        if (left > 0 && at % kBlock == 0) {
            ((gfloat*)t.ms)[block] = sm;
            ((gfloat*)t.vs)[block] = rv;
        }
    }
    if (t.bits) {
        // The codes that the linears read, as dgm_adam_quantize has them: groups are runs of group / 8 lanes.
        float mx = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = fabsf(w[j]);
            mx = x >= mx ? x : mx;
        }
        const int lanes = t.group / 8;
        for (int off = lanes / 2; off >= 1; off >>= 1) {
            const float o = __shfl_xor(mx, off, 64);
            mx = o >= mx ? o : mx;
        }
        const float s = dgm::group_scale(mx, t.bits == 4 ? 7.0f : 127.0f);
        if (left > 0) {   // whole groups, so all 8
            if (at % t.group == 0) ((gfloat*)t.scale)[at / t.group] = s;
            if (t.bits == 8) {
                u32x2 c = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) c[j / 4] |= (uint32_t(dgm::quant_code(w[j], s, 127)) & 0xFFu) << (8 * (j & 3));
                put_codes(t.q, at, 8, vec, c);
            } else {
                uint32_t c = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) c |= (uint32_t(dgm::quant_code(w[j], s, 7)) & 0xFu) << (4 * j);
                gbyte* q = (gbyte*)t.q + at / 2;
                if (vec) *(DGM_GLOBAL uint32_t*)q = c;
                else
                    for (int j = 0; j < 4; ++j) q[j] = uint8_t(c >> (8 * j));
            }
        }
    }
}

// Sums of squares in 64 bits, so that the norm is the same fp32 number in whatever order (and 8-bit codes made of gradients
// that it scales too); a workgroup `per` chunks. One read: 353 M elements 291 us (4.9 TB/s); more chunks asked for
// together, or in another order, take the same.
__global__ __launch_bounds__(kThreads) void adam_norm_kernel(const Tensor* __restrict__ tensors, const Chunk* __restrict__ chunks,
                                                             int64_t count, int64_t per, double* __restrict__ part) {
    __shared__ double sums[kThreads / 64];
    double s = 0.0;
    const int64_t to = std::min<int64_t>(count, (blockIdx.x + 1) * per);
    for (int64_t c = blockIdx.x * per; c < to; ++c) {
        const Chunk ch = chunks[c];
        const Tensor& t = tensors[ch.tensor];
        const int64_t at = int64_t(ch.index) * kChunk + threadIdx.x * kEach;
        float g[8];
        get8(t.g, at, t.n - at, t.vec, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += double(g[j]) * double(g[j]);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

__global__ __launch_bounds__(1024) void adam_factor_kernel(const double* __restrict__ part, int count, float clip, float* __restrict__ out) {
    __shared__ double sums[16];
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += 1024) s += part[i];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x > 0) return;
    for (int w = 1; w < 16; ++w) s += sums[w];
    const float norm = float(sqrt(s));
    out[0] = norm;
    // As optimizer_step has it; a norm that is not a number leaves the gradients as they are.
    out[1] = clip > 0.0f && norm > clip ? clip / (norm + 1e-6f) : 1.0f;
}

// The values that 8-bit moments stand for, tensor behind tensor, each rounded up to a block. 353 M elements 607 us (5.8 TB/s).
__global__ __launch_bounds__(kThreads) void adam_states_kernel(const Tensor* __restrict__ tensors, const Chunk* __restrict__ chunks,
                                                               float* __restrict__ m, float* __restrict__ v) {
    const Chunk ch = chunks[blockIdx.x];
    const Tensor& t = tensors[ch.tensor];
    const int64_t at = int64_t(ch.index) * kChunk + threadIdx.x * kEach, left = t.n - at;
    if (left <= 0) return;
    const bool vec = t.vec;
    const u32x2 cm = get_codes(t.m, at, left, vec), cv = get_codes(t.v, at, left, vec);
    const float sm = ((const gfloat*)t.ms)[at / kBlock], rv = ((const gfloat*)t.vs)[at / kBlock];
    float x[8], y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = m_value(code_of(cm, j, true), sm);
    v_values(cv, rv, y);
    put8(m, t.flat + at, left, true, x);
    put8(v, t.flat + at, left, true, y);
}

// ---- host ------------------------------------------------------------------------

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct Sizes {
    int64_t tensors = 0, chunks = 0, flat = 0;
    int64_t partials_at() const { return round_up(tensors * int64_t(sizeof(Tensor)) + chunks * int64_t(sizeof(Chunk)), 16); }
    int64_t bytes() const { return partials_at() + kNormBlocks * int64_t(sizeof(double)); }
};

// Sizes and conditions of a list of tensors, empty ones left out.
int check(dgm_gpu* g, const dgm_adam_tensor* list, int64_t count, int64_t stateBits, Sizes* out) {
    if (count < 0 || (count > 0 && !list)) return dgm::fail(g, DGM_ERR_ARG, "adamMany: null or negative list");
    if (stateBits != 32 && stateBits != 8)
        return dgm::fail(g, DGM_ERR_BITS, "adamMany: moments of %lld bits: 32 or 8", (long long)stateBits);
    for (int64_t i = 0; i < count; ++i) {
        const dgm_adam_tensor& t = list[i];
        if (t.n < 0) return dgm::fail(g, DGM_ERR_ARG, "adamMany: tensor %lld has %lld elements", (long long)i, (long long)t.n);
        if (t.n == 0) continue;
        if (t.n > (int64_t(1) << 40)) return dgm::fail(g, DGM_ERR_UNSUPPORTED, "adamMany: tensor %lld is beyond 2^40 elements", (long long)i);
        if (!t.w || !t.grad || !t.m || !t.v || (stateBits == 8 && (!t.mscale || !t.vscale)))
            return dgm::fail(g, DGM_ERR_ARG, "adamMany: tensor %lld: null buffer", (long long)i);
        if (stateBits == 32 && (t.mscale || t.vscale))
            return dgm::fail(g, DGM_ERR_ARG, "adamMany: tensor %lld has scales of 8-bit moments", (long long)i);
        const size_t e = stateBits == 32 ? 4 : 1;
        if (!dgm::aligned(t.w, 4) || !dgm::aligned(t.grad, 4) || !dgm::aligned(t.m, e) || !dgm::aligned(t.v, e) ||
            !dgm::aligned(t.mscale, 4) || !dgm::aligned(t.vscale, 4) || !dgm::aligned(t.scale, 4))
            return dgm::fail(g, DGM_ERR_UNSUPPORTED, "adamMany: tensor %lld: a buffer is not aligned to its elements", (long long)i);
        if (t.bits != 0) {
            if (t.bits != 4 && t.bits != 8)
                return dgm::fail(g, DGM_ERR_BITS, "adamMany: tensor %lld: codes of %d bits", (long long)i, t.bits);
            if (!t.q || !t.scale) return dgm::fail(g, DGM_ERR_ARG, "adamMany: tensor %lld: null codes or scales", (long long)i);
            if (t.qGroup < 8 || t.qGroup > 512 || (t.qGroup & (t.qGroup - 1)) != 0)
                return dgm::fail(g, DGM_ERR_UNSUPPORTED, "adamMany: tensor %lld: group %d is not a power of two from 8 to 512",
                                 (long long)i, t.qGroup);
            if (t.n % t.qGroup != 0) return dgm::fail(g, DGM_ERR_SHAPE, "adamMany: tensor %lld: elements are not whole groups", (long long)i);
        }
        ++out->tensors;
        out->chunks += (t.n + kChunk - 1) / kChunk;
        out->flat += round_up(t.n, kBlock);
        // A workgroup of kThreads for each chunk, in a launch's bound on threads.
        if (out->chunks > int64_t(UINT32_MAX) / kThreads || out->tensors > INT32_MAX / 2)
            return dgm::fail(g, DGM_ERR_UNSUPPORTED, "adamMany: more than 2^24 chunks of %d elements", kChunk);
    }
    return DGM_OK;
}

typedef std::vector<std::pair<uintptr_t, uintptr_t>> Spans;

// Whether two of the buffers that a step writes overlap (a tensor named twice among them), or one of them a gradient.
bool overlap(Spans& written, const Spans& read) {
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
        if (written[i].first < written[i - 1].second) return true;
    for (const auto& r : read) {
        // Those written lie apart: the last one that begins before r's end is the only one that can reach into r.
        const auto after = std::lower_bound(written.begin(), written.end(), std::make_pair(r.second, uintptr_t(0)));
        if (after != written.begin() && std::prev(after)->second > r.first) return true;
    }
    return false;
}

int fill_plan(dgm_gpu* g, const dgm_adam_tensor* list, int64_t count, int64_t stateBits, const Sizes& s, void* table) {
    std::vector<uint8_t> host(size_t(s.partials_at()));
    Spans spans, grads;
    Tensor* tensors = reinterpret_cast<Tensor*>(host.data());
    Chunk* chunks = reinterpret_cast<Chunk*>(host.data() + s.tensors * int64_t(sizeof(Tensor)));
    int64_t flat = 0;
    int32_t at = 0;
    for (int64_t i = 0; i < count; ++i) {
        const dgm_adam_tensor& t = list[i];
        if (t.n == 0) continue;
        const bool eight = stateBits == 8;
        const size_t e = eight ? 8 : 16;
        const bool vec = dgm::aligned(t.w, 16) && dgm::aligned(t.grad, 16) && dgm::aligned(t.m, e) && dgm::aligned(t.v, e) &&
                         (t.bits == 0 || dgm::aligned(t.q, t.bits));
        tensors[at] = Tensor{t.w, t.grad, t.m, t.v, t.mscale, t.vscale, t.q, t.scale, t.n, flat, t.decay ? 1 : 0, t.bits, t.qGroup, vec};
        const auto span = [&](const void* p, int64_t bytes) {
            spans.emplace_back(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + uintptr_t(bytes));
        };
        span(t.w, 4 * t.n);
        grads.emplace_back(reinterpret_cast<uintptr_t>(t.grad), reinterpret_cast<uintptr_t>(t.grad) + uintptr_t(4 * t.n));
        span(t.m, eight ? t.n : 4 * t.n);
        span(t.v, eight ? t.n : 4 * t.n);
        if (eight) {
            span(t.mscale, 4 * ((t.n + kBlock - 1) / kBlock));
            span(t.vscale, 4 * ((t.n + kBlock - 1) / kBlock));
        }
        if (t.bits) {
            span(t.q, t.n * t.bits / 8);
            span(t.scale, 4 * (t.n / t.qGroup));
        }
        for (int64_t c = 0; c * kChunk < t.n; ++c) *chunks++ = Chunk{at, int32_t(c)};
        flat += round_up(t.n, kBlock);
        ++at;
    }
    if (overlap(spans, grads)) return dgm::fail(g, DGM_ERR_ARG, "adamMany: two of the buffers that a step writes overlap, or one and a gradient");
    hipError_t err = hipMemcpyAsync(table, host.data(), host.size(), hipMemcpyHostToDevice, g->stream);
    if (err == hipSuccess) err = hipStreamSynchronize(g->stream);
    if (err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "adamMany_plan: %s", hipGetErrorString(err));
    return DGM_OK;
}

int check_plan(dgm_gpu* g, const char* name, const dgm_adam_plan* p) {
    if (!p || (p->chunks > 0 && !p->table)) return dgm::fail(g, DGM_ERR_ARG, "%s: null plan", name);
    if (p->tensors < 0 || p->chunks < 0 || p->chunks > int64_t(UINT32_MAX) / kThreads || p->tensors > p->chunks ||
        (p->stateBits != 32 && p->stateBits != 8))
        return dgm::fail(g, DGM_ERR_ARG, "%s: not a plan of dgm_adamMany_plan", name);
    return DGM_OK;
}
const Tensor* tensors_of(const dgm_adam_plan* p) { return static_cast<const Tensor*>(p->table); }
const Chunk* chunks_of(const dgm_adam_plan* p) { return reinterpret_cast<const Chunk*>(tensors_of(p) + p->tensors); }

}  // namespace

extern "C" {

int64_t dgm_adamMany_plan_bytes(const dgm_adam_tensor* tensors, int64_t count, int64_t stateBits) {
    Sizes s;
    return check(nullptr, tensors, count, stateBits, &s) == DGM_OK ? s.bytes() : -1;
}

int dgm_adamMany_plan(dgm_gpu* g, const dgm_adam_tensor* tensors, int64_t count, int64_t stateBits, void* table, int64_t bytes,
                      dgm_adam_plan* plan) {
    if (!g) return DGM_ERR_ARG;
    if (!plan) return dgm::fail(g, DGM_ERR_ARG, "adamMany_plan: null plan");
    *plan = dgm_adam_plan{};
    Sizes s;
    const int rc = check(g, tensors, count, stateBits, &s);
    if (rc) return rc;
    if (!table) return dgm::fail(g, DGM_ERR_ARG, "adamMany_plan: null table");
    if (!dgm::aligned(table, 16)) return dgm::fail(g, DGM_ERR_UNSUPPORTED, "adamMany_plan: the table is not 16-byte aligned");
    if (bytes < s.bytes())
        return dgm::fail(g, DGM_ERR_ARG, "adamMany_plan: table of %lld bytes, %lld needed", (long long)bytes, (long long)s.bytes());
    if (dgm::capturing(g->stream)) return dgm::fail(g, DGM_ERR_UNSUPPORTED, "adamMany_plan: not during a graph capture");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "adamMany_plan: %s", hipGetErrorString(on.err));
    if (s.chunks > 0) {
        try {
            const int filled = fill_plan(g, tensors, count, stateBits, s, table);
            if (filled) return filled;
        } catch (const std::bad_alloc&) {
            return dgm::fail(g, DGM_ERR_ARG, "adamMany_plan: no host memory for %lld chunks", (long long)s.chunks);
        }
    }
    *plan = dgm_adam_plan{table, s.tensors, s.chunks, s.flat, int32_t(stateBits), 0};
    return DGM_OK;
}

int dgm_adamMany_norm(dgm_gpu* g, const dgm_adam_plan* plan, float clip, float* out) {
    int rc = dgm::enter(g, "adam_many_norm");
    if (rc) return rc;
    rc = check_plan(g, "adamMany_norm", plan);
    if (rc) return rc;
    if (!out || !dgm::aligned(out, 4)) return dgm::fail(g, DGM_ERR_ARG, "adamMany_norm: null or unaligned result");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "adamMany_norm: %s", hipGetErrorString(on.err));
    const int64_t per = (plan->chunks + kNormBlocks - 1) / kNormBlocks, blocks = per ? (plan->chunks + per - 1) / per : 0;
    double* part = nullptr;
    if (blocks) {
        const Sizes s{plan->tensors, plan->chunks, 0};
        part = reinterpret_cast<double*>(static_cast<uint8_t*>(plan->table) + s.partials_at());
        adam_norm_kernel<<<dim3(unsigned(blocks)), dim3(kThreads), 0, g->stream>>>(tensors_of(plan), chunks_of(plan), plan->chunks, per, part);
    }
    adam_factor_kernel<<<dim3(1), dim3(1024), 0, g->stream>>>(part, int(blocks), clip, out);
    DGM_LAUNCH_CHECK(g, "adam_many_norm");
    return DGM_OK;
}

int dgm_adamMany(dgm_gpu* g, const dgm_adam_plan* plan, const float* factor, float lr, float b1, float b2, float eps, float wd,
                 float invBC1, float invBC2) {
    int rc = dgm::enter(g, "adam_many");
    if (rc) return rc;
    rc = check_plan(g, "adamMany", plan);
    if (rc) return rc;
    if (!dgm::aligned(factor, 4)) return dgm::fail(g, DGM_ERR_UNSUPPORTED, "adamMany: the factor is not 4-byte aligned");
    if (plan->chunks == 0) return DGM_OK;
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "adamMany: %s", hipGetErrorString(on.err));
    const AdamArgs a{lr, b1, b2, eps, wd, invBC1, invBC2};
    const Held held = plan->stateBits == 8 ? held_of(a) : Held{};
    const dim3 grid{unsigned(plan->chunks)}, block{kThreads};
    if (plan->stateBits == 32) adam_many_kernel<32><<<grid, block, 0, g->stream>>>(tensors_of(plan), chunks_of(plan), factor, a, held);
    else adam_many_kernel<8><<<grid, block, 0, g->stream>>>(tensors_of(plan), chunks_of(plan), factor, a, held);
    DGM_LAUNCH_CHECK(g, "adam_many");
    return DGM_OK;
}

int dgm_adamMany_states(dgm_gpu* g, const dgm_adam_plan* plan, float* m, float* v) {
    int rc = dgm::enter(g, "adam_many_states");
    if (rc) return rc;
    rc = check_plan(g, "adamMany_states", plan);
    if (rc) return rc;
    if (plan->stateBits != 8) return dgm::fail(g, DGM_ERR_BITS, "adamMany_states: the plan's moments are not in 8 bits");
    if (plan->chunks == 0) return DGM_OK;
    if (!m || !v || m == v) return dgm::fail(g, DGM_ERR_ARG, "adamMany_states: null buffer, or one for both");
    if (!dgm::aligned(m, 16) || !dgm::aligned(v, 16)) return dgm::fail(g, DGM_ERR_UNSUPPORTED, "adamMany_states: a buffer is not 16-byte aligned");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "adamMany_states: %s", hipGetErrorString(on.err));
    adam_states_kernel<<<dim3(unsigned(plan->chunks)), dim3(kThreads), 0, g->stream>>>(tensors_of(plan), chunks_of(plan), m, v);
    DGM_LAUNCH_CHECK(g, "adam_many_states");
    return DGM_OK;
}

}  // extern "C"
