// Attention over packed sequences, forward and backward (gfx950).
//
//   S_ij = scale q_i . k_j over the keys of i's own sequence (j <= i if causal)
//   out_i = sum_j softmax_j(S_i) v_j,   lse_i = log2 sum_j 2^(S_ij log2 e)
//
// Design:
//  * Every product keeps its result transposed, S^T = K Q^T: a wave owns 32
//    queries as the columns of 32x32 MFMA tiles, so a query's scores lie in one
//    lane pair (its maximum and sum need one exchange between the halves), and
//    P^T has just the layout that the next product, O^T = V^T P^T, takes as its B
//    operand: the probabilities never leave the registers. The k index of
//    that product follows the order in which a lane holds its scores; V^T is
//    stored to LDS in the same order.
//  * bf16 runs on v_mfma_f32_32x32x16_bf16, with P rounded to bf16 (half a step is
//    2^-9 of each weight, and the roundings of a row's weights are independent, so a
//    row's error stays below that of rounding the row's output once); fp32 runs on
//    v_mfma_f32_32x32x2_f32. Scores, statistics and accumulators are fp32.
//  * Tiles of 64 keys go from memory straight into one of two LDS buffers while
//    the other is computed on (one barrier a tile, no registers on the way).
//    They stay row-major: the A operand of the second product is read transposed
//    (ds_read_b64_tr_b16; for fp32, whose A operand is one element a lane, plainly).
//    16-byte chunks are XOR-swizzled so that both reads are free of bank conflicts.
//  * Rows are found on the device: sequence s owns the tile slots from
//    starts[s] / rows-per-tile + s on, which never overlap, so the grid needs no host
//    copy of the lengths, and a captured graph may be replayed with other lengths.
//  * The running maximum moves only when a score exceeds it by more than 2^8:
//    the factor then stays exact in fp32 and the accumulators are rescaled a few
//    times in a row instead of at every tile.
//  * A masked position takes no part even if its v (or in the backward its k, q
//    or dout) is infinite or NaN, where 0 * inf would spread it over a whole
//    tile: tiles that hold both masked positions and such values are cleaned of them
//    first, and the sums that they belong to spoilt afterwards.
//
// The backward recomputes P from lse; for bf16, dS enters its products as two
// bf16 pieces (rounded once, as P is, dq and dk were 1.5 times as far off as one
// rounding of the result). One kernel owns 32 queries per wave and
// accumulates dq; another owns 32 keys per wave and accumulates dk and dv over all
// query heads of the key head's group, so no gradient is added to by two
// workgroups: no atomics, the same bits every time.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "attn.hpp"

namespace {

using namespace dgm_attn;

constexpr int kTile = 64;   // rows of a staged tile

// ---- tiles in LDS ----------------------------------------------------------------

// 64 rows of D elements, row-major, padded to DP columns. The 16-byte chunk c of
// row r sits at slot c ^ swizzle(r): 16 rows' chunk c (the A operand of mm_rows) and 8
// rows' four chunks (its transposed reads in mm_cols) then lie in different banks.
template <typename T, int DP>
struct Lds {
    static constexpr int EB = sizeof(T), EPC = 16 / EB;       // bytes of an element, elements of a chunk
    static constexpr int RB = DP * EB, CPR = RB / 16;         // bytes and chunks of a row
    static constexpr int RPB = RB >= 256 ? 1 : 256 / RB;      // rows that span all banks
    static constexpr int BYTES = kTile * RB;
    static __device__ __forceinline__ int swizzle(int row) { return (row & 3) / RPB << 2 | (row >> 2 & 3); }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swizzle(row)) << 4); }
};

__device__ __forceinline__ bool nonfinite(u32x4 v, bool half) {
    uint32_t bad = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (half) bad |= ((v[w] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
        else bad |= ((v[w] & 0x7f800000u) + 0x00800000u) & 0x80000000u;
    }
    return bad != 0;
}

// A workgroup's copies of tiles from memory straight into LDS: a wave's
// instruction fills 1 KB in lane order, so that each lane fetches the chunk that belongs in
// its slot. The copies are waited for by tile_ready.
template <typename T, int DP, int NT>
struct Copy {
    using L = Lds<T, DP>;
    static constexpr int N = L::BYTES / 16 / NT, STEP = NT / L::CPR;   // chunks of a thread, rows between them
    static_assert(L::BYTES % (16 * NT) == 0 && NT % L::CPR == 0, "every thread copies whole chunks of one slot");
    int64_t ldb;        // bytes from row to row
    int row, slot, wave;

    __device__ __forceinline__ explicit Copy(int64_t ld)
        : ldb(ld * L::EB), row(int(threadIdx.x) / L::CPR), slot(int(threadIdx.x) % L::CPR),
          wave(__builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6)) {}

    // `rows` rows from `from` on (the first `D` columns); the rest of the tile is zero.
    __device__ __forceinline__ void start(uint8_t* lds, const T* from, int rows, int D) const {
        const uint32_t base = uint32_t(reinterpret_cast<uintptr_t>(lds)) + uint32_t(wave) * 1024u;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(from);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
        if (rows >= kTile && D == DP) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint32_t off = uint32_t(row) * uint32_t(ldb) + uint32_t((slot ^ L::swizzle(row + i * STEP)) << 4);
                asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(base + i * NT * 16), "v"(off),
                             "s"(src + i * STEP * ldb)
                             : "memory", "m0");
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = row + i * STEP, c = slot ^ L::swizzle(r);
                if (r < rows && c * L::EPC < D)
                    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base + i * NT * 16),
                                 "v"(src + r * ldb + c * 16)
                                 : "memory", "m0");
                else
                    *reinterpret_cast<u32x4*>(lds + (i * NT + int(threadIdx.x)) * 16) = u32x4{0, 0, 0, 0};
            }
        }
#pragma clang diagnostic pop
    }
    // Whether this thread's chunks of a tile hold infinities or NaN.
    __device__ __forceinline__ bool bad(const uint8_t* lds) const {
        bool b = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
            b = b || nonfinite(*reinterpret_cast<const u32x4*>(lds + (i * NT + int(threadIdx.x)) * 16), L::EB == 2);
        return b;
    }
};

// Every copy that the workgroup has started is in LDS, and every wave's reads of what the
// next copies overwrite are done.
__device__ __forceinline__ void tile_ready() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- products ------------------------------------------------------------------

// B operand of mm_rows: a wave's 32 rows of q (k, dout, v), one a lane pair.
template <typename T, int DP>
struct Frags {
    using L = Lds<T, DP>;
    static constexpr int NK = L::CPR / 2;
    u32x4 f[NK];
    __device__ __forceinline__ void load(const T* row, bool in, int D, int h) {
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
            const int c = 2 * kk + h;
            f[kk] = u32x4{0, 0, 0, 0};
            if (in && c * L::EPC < D) f[kk] = *reinterpret_cast<const u32x4*>(row + c * L::EPC);
        }
    }
};

template <typename T>
__device__ __forceinline__ void mfma_chunk(f32x16& acc, u32x4 a, u32x4 b) {
    if constexpr (sizeof(T) == 2) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc,
                                                      0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), acc, 0, 0, 0);
    }
}

// out[kb] (32 rows x the wave's 32 columns) = tile rows 32kb .. 32kb+31 times the columns' vectors.
// Element r of a lane: row 32kb + 8(r/4) + 4h + r%4, column lane % 32.
template <typename T, int DP>
__device__ __forceinline__ void mm_rows(f32x16 (&out)[2], const uint8_t* rows, const Frags<T, DP>& b, int lane) {
    using L = Lds<T, DP>;
    const int h = lane >> 5, r = lane & 31;
    out[0] = out[1] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < Frags<T, DP>::NK; ++kk)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
            mfma_chunk<T>(out[kb], *reinterpret_cast<const u32x4*>(rows + L::at(32 * kb + r, 2 * kk + h)), b.f[kk]);
}

__device__ __forceinline__ bf16x8 pack8(const f32x16& p, int at) {
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = __bf16(p[at + j]);
    return o;
}

// A operand of mm_cols for bf16: element j of a lane is column d = 32 dt + lane %
// 32 of row 32 kb + 16 st + 8 (j / 4) + 4h + j % 4, the order in which mm_rows leaves
// a lane's results. The transposed read takes, for each 16 lanes, 4 rows of 16
// columns (4 lanes a row) and gives each lane one column of them.
template <int DP>
__device__ __forceinline__ bf16x8 read_cols(const uint8_t* tile, int kb, int st, int dt, int lane) {
    using L = Lds<__bf16, DP>;
    const int row = 32 * kb + 16 * st + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int chunk = 4 * dt + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), in = (lane & 1) * 8;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* At;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)(tile + L::at(row, chunk) + in));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)(tile + L::at(row + 8, chunk) + in));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// acc[dt] (32 columns d x the wave's 32 columns) += tile^T times p, p as mm_rows
// leaves it; for bf16 in PIECES pieces of 8 bits.
template <typename T, int DP, int PIECES = 1>
__device__ __forceinline__ void mm_cols(f32x16 (&acc)[DP / 32], const uint8_t* tile, const f32x16 (&p)[2], int lane) {
    using L = Lds<T, DP>;
    const int h = lane >> 5, r = lane & 31;
    if constexpr (L::EB == 2) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const bf16x8 b = pack8(p[kb], 8 * st);
                bf16x8 rest;
                if constexpr (PIECES == 2) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) rest[j] = __bf16(p[kb][8 * st + j] - float(b[j]));
                }
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) {
                    const bf16x8 a = read_cols<DP>(tile, kb, st, dt, lane);
                    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc[dt], 0, 0, 0);
                    if constexpr (PIECES == 2)
                        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, rest, acc[dt], 0, 0, 0);
                }
            }
    } else {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = 32 * kb + 8 * (e / 4) + 4 * h + e % 4;
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) {
                    const int d = 32 * dt + r;
                    const float a = *reinterpret_cast<const float*>(tile + L::at(row, d >> 2) + (d & 3) * 4);
                    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[kb][e], acc[dt], 0, 0, 0);
                }
            }
    }
}

// What a tile's infinities and NaN do to sums that masked positions take no part in:
// the tile is cleaned (they become 0, as the weights of masked positions are) and
// for each column d the first (kLast: last) row that holds such a value is
// kept; a query (key) that sees that row has its sum spoilt. Rare, so it may cost barriers.
template <int DP, int KINDS>
struct Marks {
    int row[KINDS][DP];   // kinds: NaN, +inf, -inf; or all of them as one
};

template <typename T, int DP, int NT, int KINDS, bool kLast>
__device__ __forceinline__ void clean_tile(const Copy<T, DP, NT>& c, uint8_t* lds, Marks<DP, KINDS>& marks) {
    using L = Lds<T, DP>;
    for (int i = threadIdx.x; i < KINDS * DP; i += NT) marks.row[i / DP][i % DP] = kLast ? -1 : INT_MAX;
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < Copy<T, DP, NT>::N; ++i) {
        const int r = c.row + i * Copy<T, DP, NT>::STEP, d0 = (c.slot ^ L::swizzle(r)) * L::EPC;
        T* at = reinterpret_cast<T*>(lds + (i * NT + int(threadIdx.x)) * 16);
#pragma unroll 1
        for (int j = 0; j < L::EPC; ++j) {
            const float x = float(at[j]);
            if (fabsf(x) < __builtin_huge_valf()) continue;
            int* m = &marks.row[KINDS == 1 || x != x ? 0 : x > 0.0f ? 1 : 2][d0 + j];
            if (kLast) atomicMax(m, r);
            else atomicMin(m, r);
            at[j] = T(0.0f);
        }
    }
    __syncthreads();
}

// acc after mm_cols on a clean tile. `sees(row)`: whether the lane's column sees a row marked so.
template <int DP, int KINDS, typename Sees>
__device__ __forceinline__ void spoil(f32x16 (&acc)[DP / 32], const Marks<DP, KINDS>& marks, const Sees& sees, int lane) {
    const float inf = __builtin_huge_valf();
    asm volatile("" : "+v"(lane));   // no addresses of this rare path kept through the loop
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int d = 32 * dt + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
            float x = acc[dt][e];
            if constexpr (KINDS == 3) {
                x += sees(marks.row[1][d]) ? inf : 0.0f;
                x += sees(marks.row[2][d]) ? -inf : 0.0f;
            }
            acc[dt][e] = sees(marks.row[0][d]) ? __builtin_nanf("") : x;
        }
}

// ---- rows ----------------------------------------------------------------------

// The sequence and its tile behind slot `slot` of tiles of `per` rows. False where the slot has no rows.
struct Rows {
    int first, len, tile;   // the sequence's first row and length; the tile's number in it
};
__device__ inline bool find_rows(const int32_t* starts, int64_t nseq, int64_t rows, int per, int64_t slot, Rows& out) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, n = nseq;
    while (true) {   // 64 candidates a round
        const int64_t step = (n + 63) / 64, at = lo + lane * step;
        const bool below = lane * step < n && slot_base(clamped(starts, at, rows), at, per) <= slot;
        const int c = __popcll(__ballot(below));
        if (c == 0) return false;
        lo += (c - 1) * step;
        if (step == 1) break;
        n = n - (c - 1) * step < step ? n - (c - 1) * step : step;
    }
    out.first = clamped(starts, lo, rows);
    out.len = clamped(starts, lo + 1, rows) - out.first;
    const int64_t tile = slot - slot_base(out.first, lo, per);
    out.tile = int(tile);
    return tile >= 0 && tile * per < out.len;
}

struct FwdArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;
    const int32_t* starts;
    uint32_t* flag;
    int64_t rows, nseq, ldq, ldk, ldv, ldo, slots;
    int H, KVH, D, causal;
    float c;   // scale * log2 e
};

// Query head of the h'-th workgroup of a slot: consecutive workgroups go to
// different XCDs, so the heads of one group, which read the same k and v, are KVH apart.
__device__ __forceinline__ int head_of(int i, int H, int KVH) { return (i % KVH) * (H / KVH) + i / KVH; }

template <typename T, int DP, int QB, int NW, int NBUF>
__global__ void __launch_bounds__(64 * NW, sizeof(T) == 2 && DP <= 128 && QB == 1 ? 2 : 1)
    attn_packed_fwd_kernel(FwdArgs a) {
    using L = Lds<T, DP>;
    constexpr int NT = 64 * NW, BQ = 32 * QB * NW, DT = DP / 32;
    __shared__ __align__(16) uint8_t lds[NBUF][2][L::BYTES];   // k and v
    __shared__ Marks<DP, 3> marks;
    if (blockIdx.x == 0) check_starts(a.starts, a.nseq, a.rows, a.flag);
    Rows rw;
    // The last tiles of a causal sequence are the longest: they start first.
    if (!find_rows(a.starts, a.nseq, a.rows, BQ, a.slots - 1 - blockIdx.x / a.H, rw)) return;
    const int head = head_of(blockIdx.x % a.H, a.H, a.KVH), kvh = head / (a.H / a.KVH);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int q0 = rw.tile * BQ + wave * 32 * QB;   // the wave's first row in its sequence
    const T* q = static_cast<const T*>(a.q) + int64_t(rw.first) * a.ldq + int64_t(head) * a.D;
    const T* k = static_cast<const T*>(a.k) + int64_t(rw.first) * a.ldk + int64_t(kvh) * a.D;
    const T* v = static_cast<const T*>(a.v) + int64_t(rw.first) * a.ldv + int64_t(kvh) * a.D;
    const Copy<T, DP, NT> ck(a.ldk), cv(a.ldv);
    const auto start = [&](int t) __attribute__((always_inline)) {
        const int key0 = t * kTile;
        ck.start(lds[t % NBUF][0], k + key0 * a.ldk, rw.len - key0, a.D);
        cv.start(lds[t % NBUF][1], v + key0 * a.ldv, rw.len - key0, a.D);
    };
    start(0);

    Frags<T, DP> qf[QB];
    f32x16 o[QB][DT];
    float m[QB], l[QB];
    int last[QB];   // the last key that the lane's query sees
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int row = q0 + 32 * b + (lane & 31);
        qf[b].load(q + int64_t(row) * a.ldq, row < rw.len, a.D, h);
        m[b] = kNegInf;
        l[b] = 0.0f;
        last[b] = a.causal && row < rw.len ? row : rw.len - 1;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[b][t] = f32x16{};
    }
    const int wg_end = min(rw.len, (rw.tile + 1) * BQ), keys = a.causal ? wg_end : rw.len;
    const int tiles = (keys + kTile - 1) / kTile;
    // Tiles from here on hold positions that some query of the workgroup does not see.
    const int masked_from = a.causal ? rw.tile * BQ / kTile : rw.len / kTile;
    const int wave_keys = a.causal ? min(keys, q0 + 32 * QB) : keys;

    const auto step = [&](int t, auto masked) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        const uint8_t* kt = lds[t % NBUF][0];
        uint8_t* vt = lds[t % NBUF][1];
        tile_ready();
        if (NBUF > 1 && t + 1 < tiles) start(t + 1);
        bool dirty = false;
        if (kMasked && a.causal) dirty = __syncthreads_or(cv.bad(vt));
        if (dirty) clean_tile<T, DP, NT, 3, false>(cv, vt, marks);
        const int key0 = t * kTile;
        if (key0 < wave_keys && q0 < rw.len) {
#pragma unroll
            for (int b = 0; b < QB; ++b) {
                f32x16 s[2];
                mm_rows<T, DP>(s, kt, qf[b], lane);
                const int lim = last[b] - key0 - 4 * h;   // element e of block kb is seen up to here
                if constexpr (kMasked) {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            s[kb][e] = 32 * kb + 8 * (e / 4) + e % 4 <= lim ? s[kb][e] : kNegInf;
                }
                float mx = s[0][0];
#pragma unroll
                for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[0][e]);
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[1][e]);
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                if (__any((mx - m[b]) * a.c > 8.0f)) {   // also from -inf; inf - inf is NaN: no move
                    const float to = fmaxf(m[b], mx), f = m[b] == kNegInf ? 0.0f : exp2_hw((m[b] - to) * a.c);
                    l[b] *= f;
#pragma unroll
                    for (int n = 0; n < DT; ++n) o[b][n] *= f;
                    m[b] = to;
                }
                const float mc = m[b] == kNegInf ? 0.0f : m[b] * a.c;
                float sum = 0.0f;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        s[kb][e] = exp2_hw(__builtin_fmaf(s[kb][e], a.c, -mc));
                        sum += s[kb][e];
                    }
                l[b] += sum;
                mm_cols<T, DP>(o[b], vt, s, lane);
                if (dirty) spoil<DP>(o[b], marks, [&](int row) { return row <= last[b] - key0; }, lane);
            }
        }
        if (NBUF == 1 && t + 1 < tiles) {
            __syncthreads();
            start(t + 1);
        }
    };
    int t = 0;
    for (; t < min(masked_from, tiles); ++t) step(t, std::false_type{});
    for (; t < tiles; ++t) step(t, std::true_type{});
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int row = q0 + 32 * b + (lane & 31);
        const float sum = l[b] + __shfl_xor(l[b], 32, 64);
        if (row >= rw.len) continue;
        const float f = 1.0f / sum;
        const int64_t at = int64_t(rw.first) + row;
        if (a.lse && h == 0) a.lse[int64_t(head) * a.rows + at] = (m[b] == kNegInf ? 0.0f : m[b] * a.c) + log2_hw(sum);
        T* out = static_cast<T*>(a.out) + at * a.ldo + int64_t(head) * a.D;
#pragma unroll
        for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * n + 8 * g + 4 * h;
                if (d >= a.D) continue;
                if constexpr (L::EB == 2) {
                    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                    bf16x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = __bf16(o[b][n][4 * g + i] * f);
                    *reinterpret_cast<bf16x4*>(out + d) = w;
                } else {
                    f32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = o[b][n][4 * g + i] * f;
                    *reinterpret_cast<f32x4*>(out + d) = w;
                }
            }
    }
}

// ---- backward ------------------------------------------------------------------

// delta[head][row] = dout . out, one wave a (row, head).
struct DeltaArgs {
    const void *out, *dout;
    float* delta;
    int64_t rows, ldo;
    int H, D;
};
template <typename T>
__global__ void __launch_bounds__(256) attn_packed_delta_kernel(DeltaArgs a) {
    const int64_t at = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (at >= a.rows * a.H) return;
    const int lane = threadIdx.x & 63, head = int(at % a.H);
    const int64_t row = at / a.H, off = row * a.ldo + int64_t(head) * a.D;
    float s = 0.0f;
    for (int d = lane; d < a.D; d += 64)
        s = __builtin_fmaf(float(static_cast<const T*>(a.out)[off + d]), float(static_cast<const T*>(a.dout)[off + d]), s);
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) s += __shfl_xor(s, x, 64);
    if (lane == 0) a.delta[int64_t(head) * a.rows + row] = s;
}

struct BwdArgs {
    const void *q, *k, *v, *dout;
    void *dq, *dk, *dv;
    const float *lse, *delta;
    const int32_t* starts;
    uint32_t* flag;
    int64_t rows, nseq, ldq, ldk, ldv, ldo, slots;
    int H, KVH, D, causal;
    float c, scale;
};

// Rows 32n + 8g + 4h .. +3 of a lane's column, times f, to its row of a gradient.
template <typename T, int DT>
__device__ __forceinline__ void store_grad(T* row, const f32x16 (&acc)[DT], float f, int D, int h) {
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * n + 8 * g + 4 * h;
            if (d >= D) continue;
            if constexpr (sizeof(T) == 2) {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                bf16x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = __bf16(acc[n][4 * g + i] * f);
                *reinterpret_cast<bf16x4*>(row + d) = w;
            } else {
                f32x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = acc[n][4 * g + i] * f;
                *reinterpret_cast<f32x4*>(row + d) = w;
            }
        }
}

// dq: a wave's 32 queries against tiles of 64 keys. dS^T = P^T (dP^T - delta)
// with dP^T = V dout^T; dq^T += K^T dS^T.
template <typename T, int DP, int NW, int NBUF>
__global__ void __launch_bounds__(64 * NW, sizeof(T) == 2 ? 2 : 1) attn_packed_dq_kernel(BwdArgs a) {
    using L = Lds<T, DP>;
    constexpr int NT = 64 * NW, BQ = 32 * NW, DT = DP / 32;
    __shared__ __align__(16) uint8_t lds[NBUF][2][L::BYTES];   // k and v
    __shared__ Marks<DP, 1> marks;
    if (blockIdx.x == 0) check_starts(a.starts, a.nseq, a.rows, a.flag);
    Rows rw;
    if (!find_rows(a.starts, a.nseq, a.rows, BQ, a.slots - 1 - blockIdx.x / a.H, rw)) return;
    const int head = head_of(blockIdx.x % a.H, a.H, a.KVH), kvh = head / (a.H / a.KVH);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int q0 = rw.tile * BQ + wave * 32, row = q0 + (lane & 31);
    const bool in = row < rw.len;
    const int64_t at = int64_t(rw.first) + row;
    const T* k = static_cast<const T*>(a.k) + int64_t(rw.first) * a.ldk + int64_t(kvh) * a.D;
    const T* v = static_cast<const T*>(a.v) + int64_t(rw.first) * a.ldv + int64_t(kvh) * a.D;
    const Copy<T, DP, NT> ck(a.ldk), cv(a.ldv);
    const auto start = [&](int t) __attribute__((always_inline)) {
        const int key0 = t * kTile;
        ck.start(lds[t % NBUF][0], k + key0 * a.ldk, rw.len - key0, a.D);
        cv.start(lds[t % NBUF][1], v + key0 * a.ldv, rw.len - key0, a.D);
    };
    start(0);
    Frags<T, DP> qf, gf;
    qf.load(static_cast<const T*>(a.q) + at * a.ldq + int64_t(head) * a.D, in, a.D, h);
    gf.load(static_cast<const T*>(a.dout) + at * a.ldo + int64_t(head) * a.D, in, a.D, h);
    const float lse = in ? a.lse[int64_t(head) * a.rows + at] : 0.0f;
    const float delta = in ? a.delta[int64_t(head) * a.rows + at] : 0.0f;
    const int last = a.causal && in ? row : rw.len - 1;
    f32x16 acc[DT];
#pragma unroll
    for (int n = 0; n < DT; ++n) acc[n] = f32x16{};

    const int keys = a.causal ? min(rw.len, (rw.tile + 1) * BQ) : rw.len, tiles = (keys + kTile - 1) / kTile;
    const int masked_from = a.causal ? rw.tile * BQ / kTile : rw.len / kTile;
    const int wave_keys = a.causal ? min(keys, q0 + 32) : keys;
    const auto step = [&](int t, auto masked) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        uint8_t* kt = lds[t % NBUF][0];
        const uint8_t* vt = lds[t % NBUF][1];
        tile_ready();
        if (NBUF > 1 && t + 1 < tiles) start(t + 1);
        bool dirty = false;
        if (kMasked && a.causal) dirty = __syncthreads_or(ck.bad(kt));
        const int key0 = t * kTile;
        const bool active = key0 < wave_keys && q0 < rw.len;
        f32x16 s[2], dp[2];
        if (active) {
            mm_rows<T, DP>(s, kt, qf, lane);
            mm_rows<T, DP>(dp, vt, gf, lane);
            const int lim = last - key0 - 4 * h;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float p = exp2_hw(__builtin_fmaf(s[kb][e], a.c, -lse));
                    s[kb][e] = !kMasked || 32 * kb + 8 * (e / 4) + e % 4 <= lim ? p * (dp[kb][e] - delta) : 0.0f;
                }
        }
        if (dirty) {
            __syncthreads();   // the tile has been read as it is
            clean_tile<T, DP, NT, 1, false>(ck, kt, marks);
        }
        if (active) {
            mm_cols<T, DP, 2>(acc, kt, s, lane);
            if (dirty) spoil<DP>(acc, marks, [&](int row) { return row <= last - key0; }, lane);
        }
        if (NBUF == 1 && t + 1 < tiles) {
            __syncthreads();
            start(t + 1);
        }
    };
    int t = 0;
    for (; t < min(masked_from, tiles); ++t) step(t, std::false_type{});
    for (; t < tiles; ++t) step(t, std::true_type{});
    if (in) store_grad<T, DT>(static_cast<T*>(a.dq) + at * a.ldq + int64_t(head) * a.D, acc, a.scale, a.D, h);
}

// dk, dv: a wave's 32 keys as columns against tiles of 64 queries, over the query heads of
// the group one after the other. S = Q K^T, dP = dout V^T; dv^T += dout^T P, dk^T += Q^T dS.
template <typename T, int DP, int NW, int NBUF>
__global__ void __launch_bounds__(64 * NW, sizeof(T) == 2 && DP <= 64 ? 2 : 1) attn_packed_dkv_kernel(BwdArgs a) {
    using L = Lds<T, DP>;
    constexpr int NT = 64 * NW, BK = 32 * NW, DT = DP / 32;
    __shared__ __align__(16) uint8_t lds[NBUF][2][L::BYTES];   // q and dout
    __shared__ __align__(16) float stat[NBUF][2][kTile];       // lse and delta
    __shared__ Marks<DP, 1> marks[2];
    Rows rw;
    if (!find_rows(a.starts, a.nseq, a.rows, BK, blockIdx.x / a.KVH, rw)) return;
    const int kvh = blockIdx.x % a.KVH, G = a.H / a.KVH;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int k0 = rw.tile * BK + wave * 32, row = k0 + (lane & 31);
    const bool in = row < rw.len;
    const int64_t at = int64_t(rw.first) + row;
    const int first = a.causal ? rw.tile * BK / kTile : 0, per_head = (rw.len + kTile - 1) / kTile - first;
    const int steps = per_head * G;
    const Copy<T, DP, NT> cq(a.ldq), cg(a.ldo);
    static_assert(NT >= 2 * kTile, "a thread stages one statistic");
    int head = kvh * G, tile = first;   // of the next copy
    const auto start = [&](int buf) __attribute__((always_inline)) {
        const int row0 = tile * kTile;
        const int64_t r0 = int64_t(rw.first) + row0;
        cq.start(lds[buf][0], static_cast<const T*>(a.q) + r0 * a.ldq + int64_t(head) * a.D, rw.len - row0, a.D);
        cg.start(lds[buf][1], static_cast<const T*>(a.dout) + r0 * a.ldo + int64_t(head) * a.D, rw.len - row0, a.D);
        if (threadIdx.x < 2 * kTile) {
            const int r = threadIdx.x & (kTile - 1);
            const float* from = threadIdx.x < kTile ? a.lse : a.delta;
            stat[buf][threadIdx.x / kTile][r] = row0 + r < rw.len ? from[int64_t(head) * a.rows + r0 + r] : 0.0f;
        }
        if (++tile - first == per_head) {
            tile = first;
            ++head;
        }
    };
    start(0);
    Frags<T, DP> kf, vf;
    kf.load(static_cast<const T*>(a.k) + at * a.ldk + int64_t(kvh) * a.D, in, a.D, h);
    vf.load(static_cast<const T*>(a.v) + at * a.ldv + int64_t(kvh) * a.D, in, a.D, h);
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int n = 0; n < DT; ++n) dk[n] = dv[n] = f32x16{};

    int now = first;   // the tile that is computed on
    const auto step = [&](int t, auto masked, bool hidden) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        const int buf = t % NBUF, row0 = now * kTile;
        uint8_t* qt = lds[buf][0];
        uint8_t* gt = lds[buf][1];
        const float* lse = stat[buf][0];
        const float* delta = stat[buf][1];
        tile_ready();
        if (NBUF > 1 && t + 1 < steps) start((t + 1) % NBUF);
        bool dirty = false;
        if (kMasked && hidden) dirty = __syncthreads_or(cq.bad(qt) || cg.bad(gt));
        const bool active = k0 < rw.len && !(a.causal && row0 + kTile <= k0);
        const int from = (a.causal ? row : 0) - row0;   // the tile's rows that the key sees
        f32x16 p[2], ds[2];
        if (active) {
            mm_rows<T, DP>(p, qt, kf, lane);
            mm_rows<T, DP>(ds, gt, vf, lane);
            // Element e of block kb is row 32kb + 8(e/4) + e%4 + 4h.
            const int lo = from - 4 * h, hi = rw.len - row0 - 4 * h;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int i0 = 32 * kb + 8 * g;
                    const f32x4 ls = *reinterpret_cast<const f32x4*>(lse + i0 + 4 * h);
                    const f32x4 de = *reinterpret_cast<const f32x4*>(delta + i0 + 4 * h);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = 4 * g + i;
                        const bool see = !kMasked || (i0 + i >= lo && i0 + i < hi);
                        const float w = see ? exp2_hw(__builtin_fmaf(p[kb][e], a.c, -ls[i])) : 0.0f;
                        ds[kb][e] = see ? w * (ds[kb][e] - de[i]) : 0.0f;
                        p[kb][e] = w;
                    }
                }
        }
        if (dirty) {
            __syncthreads();   // the tiles have been read as they are
            clean_tile<T, DP, NT, 1, true>(cq, qt, marks[0]);
            clean_tile<T, DP, NT, 1, true>(cg, gt, marks[1]);
        }
        if (active) {
            mm_cols<T, DP>(dv, gt, p, lane);
            mm_cols<T, DP, 2>(dk, qt, ds, lane);
            if (dirty) {
                const auto sees = [&](int row) { return row >= 0 && row >= from; };
                spoil<DP>(dk, marks[0], sees, lane);
                spoil<DP>(dv, marks[1], sees, lane);
            }
        }
        if (NBUF == 1 && t + 1 < steps) {
            __syncthreads();
            start(0);
        }
        if (++now - first == per_head) now = first;
    };
    for (int t = 0; t < steps; ++t) {
        // Positions not seen: queries before the workgroup's last key, or behind the sequence.
        const int row0 = now * kTile;
        const bool hidden = a.causal && row0 < (rw.tile + 1) * BK;
        if (hidden || row0 + kTile > rw.len) step(t, std::true_type{}, hidden);
        else step(t, std::false_type{}, false);
    }
    if (in) {
        store_grad<T, DT>(static_cast<T*>(a.dk) + at * a.ldk + int64_t(kvh) * a.D, dk, a.scale, a.D, h);
        store_grad<T, DT>(static_cast<T*>(a.dv) + at * a.ldv + int64_t(kvh) * a.D, dv, 1.0f, a.D, h);
    }
}

// ---- host ----------------------------------------------------------------------

constexpr int64_t kMaxStride = int64_t(1) << 23;   // a tile's 64 rows within the copies' 32-bit offsets

// Strides of 0 mean rows back to back.
struct Strides {
    int64_t q, k, v, o;
};
Strides strides(const dgm_attn_cfg* c) {
    const int64_t qo = int64_t(c->H) * c->D, kv = int64_t(c->KVH) * c->D;
    return {c->ldq ? c->ldq : qo, c->ldk ? c->ldk : kv, c->ldv ? c->ldv : kv, c->ldo ? c->ldo : qo};
}

int check_cfg(dgm_gpu* g, const char* name, const dgm_attn_cfg* c, int max_d) {
    if (!c) return dgm::fail(g, DGM_ERR_ARG, "%s: null configuration", name);
    if (!type_bytes(c->type)) return dgm::fail(g, DGM_ERR_ARG, "%s: unknown type %d", name, c->type);
    if (c->rows < 0 || c->nseq < 0 || c->H < 1 || c->KVH < 1 || c->D < 1)
        return dgm::fail(g, DGM_ERR_ARG, "%s: bad sizes rows=%lld nseq=%lld H=%d KVH=%d D=%d", name,
                         (long long)c->rows, (long long)c->nseq, c->H, c->KVH, c->D);
    if (!(c->scale > 0.0f) || !std::isfinite(c->scale * kLog2e))
        return dgm::fail(g, DGM_ERR_ARG, "%s: scale must be positive and finite", name);
    if (c->H % c->KVH != 0)
        return dgm::fail(g, DGM_ERR_SHAPE, "%s: %d query heads over %d key heads", name, c->H, c->KVH);
    if (c->D % 8 != 0 || c->D > max_d)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: head dim %d is not a multiple of 8 up to %d", name, c->D, max_d);
    if (c->rows > (int64_t(1) << 30) || c->nseq > (int64_t(1) << 30) || c->H > 65536)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: too many rows, sequences or heads", name);
    const Strides s = strides(c);
    const int64_t qo = int64_t(c->H) * c->D, kv = int64_t(c->KVH) * c->D;
    if (s.q < qo || s.o < qo || s.k < kv || s.v < kv)
        return dgm::fail(g, DGM_ERR_SHAPE, "%s: a row stride is shorter than the row's heads", name);
    if ((s.q | s.k | s.v | s.o) % 8 != 0)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: row strides must be multiples of 8 elements", name);
    if (std::max(std::max(s.q, s.o), std::max(s.k, s.v)) > kMaxStride)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: a row stride beyond %lld elements", name, (long long)kMaxStride);
    return DGM_OK;
}

int slots_of(dgm_gpu* g, const char* name, const dgm_attn_cfg* c, int per, int heads, int threads, int64_t& slots) {
    slots = slot_count(c->rows, c->nseq, per);
    if (slots * heads * threads > int64_t(UINT32_MAX))   // hipLaunchKernel's bound on a grid's threads
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: %lld tiles of %d heads exceed one launch", name,
                         (long long)slots, heads);
    return DGM_OK;
}

template <typename T, int DP, int QB, int NW, int NBUF>
int launch_fwd(dgm_gpu* g, const dgm_attn_cfg* c, FwdArgs a) {
    const int rc = slots_of(g, "attnPackedFwd", c, 32 * QB * NW, c->H, 64 * NW, a.slots);
    if (rc) return rc;
    attn_packed_fwd_kernel<T, DP, QB, NW, NBUF><<<dim3(unsigned(a.slots * c->H)), dim3(64 * NW), 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "attn_packed_fwd");
    return DGM_OK;
}

template <typename T>
int run_fwd(dgm_gpu* g, const dgm_attn_cfg* c, const FwdArgs& a) {
    if (c->D <= 32) return launch_fwd<T, 32, 1, 4, 2>(g, c, a);
    if (c->D <= 64) return launch_fwd<T, 64, 1, 4, 2>(g, c, a);
    if (c->D <= 128) return launch_fwd<T, 128, 1, 4, 2>(g, c, a);
    return launch_fwd<T, 256, 1, 4, sizeof(T) == 2 ? 2 : 1>(g, c, a);
}

template <typename T, int DP, int NW, int NBUF>
int launch_bwd(dgm_gpu* g, const dgm_attn_cfg* c, BwdArgs a) {
    BwdArgs kv = a;
    int rc = slots_of(g, "attnPackedBwd", c, 32 * NW, c->H, 64 * NW, a.slots);
    if (!rc) rc = slots_of(g, "attnPackedBwd", c, 32 * NW, c->KVH, 64 * NW, kv.slots);
    if (rc) return rc;
    attn_packed_dkv_kernel<T, DP, NW, NBUF><<<dim3(unsigned(kv.slots * c->KVH)), dim3(64 * NW), 0, g->stream>>>(kv);
    DGM_LAUNCH_CHECK(g, "attn_packed_dkv");
    attn_packed_dq_kernel<T, DP, NW, NBUF><<<dim3(unsigned(a.slots * c->H)), dim3(64 * NW), 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "attn_packed_dq");
    return DGM_OK;
}

template <typename T>
int run_bwd(dgm_gpu* g, const dgm_attn_cfg* c, const BwdArgs& a, const DeltaArgs& d) {
    const int64_t pairs = c->rows * c->H;
    if (pairs > int64_t(UINT32_MAX) / 64)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "attnPackedBwd: %lld rows of %d heads exceed one launch",
                         (long long)c->rows, c->H);
    attn_packed_delta_kernel<T><<<dim3(dgm::ceil_div(pairs, 4)), dim3(256), 0, g->stream>>>(d);
    DGM_LAUNCH_CHECK(g, "attn_packed_delta");
    if (c->D <= 32) return launch_bwd<T, 32, 4, 2>(g, c, a);
    if (c->D <= 64) return launch_bwd<T, 64, 4, 2>(g, c, a);
    return launch_bwd<T, 128, 4, 1>(g, c, a);
}

constexpr int kMaxD = 256, kMaxDBwd = 128;

int64_t bwd_ws_bytes(const dgm_attn_cfg* c) { return c->rows * c->H * int64_t(sizeof(float)); }

}  // namespace

extern "C" {

int dgm_attnPackedFwd(dgm_gpu* g, const dgm_attn_cfg* cfg, const void* q, const void* k, const void* v,
                      const int32_t* starts, void* out, float* lse) {
    int rc = dgm::enter(g, "attn_packed_fwd");
    if (rc) return rc;
    rc = check_cfg(g, "attnPackedFwd", cfg, kMaxD);
    if (rc) return rc;
    if (cfg->rows == 0 || cfg->nseq == 0) return DGM_OK;
    if (!q || !k || !v || !starts || !out) return dgm::fail(g, DGM_ERR_ARG, "attnPackedFwd: null buffer");
    for (const void* p : {q, k, v, static_cast<const void*>(out)})
        if (!dgm::aligned(p, 16)) return dgm::fail(g, DGM_ERR_UNSUPPORTED, "attnPackedFwd: a buffer is not 16-byte aligned");
    if (!dgm::aligned(starts, 4) || !dgm::aligned(lse, 4))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "attnPackedFwd: starts or lse is not 4-byte aligned");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "attnPackedFwd: %s", hipGetErrorString(on.err));
    const Strides s = strides(cfg);
    FwdArgs a{q, k, v, out, lse, starts, g->seq_flag, cfg->rows, cfg->nseq, s.q, s.k, s.v, s.o, 0, cfg->H, cfg->KVH,
              cfg->D, cfg->causal != 0, cfg->scale * kLog2e};
    g->seq_checks = true;
    return cfg->type == DGM_TYPE_F32 ? run_fwd<float>(g, cfg, a) : run_fwd<__bf16>(g, cfg, a);
}

int64_t dgm_attnPackedBwd_ws_bytes(const dgm_attn_cfg* cfg) {
    if (!cfg || cfg->rows < 0 || cfg->H < 1 || cfg->rows > (int64_t(1) << 30) || cfg->H > 65536) return -1;
    return bwd_ws_bytes(cfg);
}

int dgm_attnPackedBwd(dgm_gpu* g, const dgm_attn_cfg* cfg, const void* q, const void* k, const void* v,
                      const int32_t* starts, const void* out, const float* lse, const void* dout, void* dq, void* dk,
                      void* dv, void* ws, int64_t ws_bytes) {
    int rc = dgm::enter(g, "attn_packed_bwd");
    if (rc) return rc;
    rc = check_cfg(g, "attnPackedBwd", cfg, kMaxDBwd);
    if (rc) return rc;
    if (cfg->rows == 0 || cfg->nseq == 0) return DGM_OK;
    if (!q || !k || !v || !starts || !out || !lse || !dout || !dq || !dk || !dv || !ws)
        return dgm::fail(g, DGM_ERR_ARG, "attnPackedBwd: null buffer");
    if (ws_bytes < bwd_ws_bytes(cfg))
        return dgm::fail(g, DGM_ERR_ARG, "attnPackedBwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
                         (long long)bwd_ws_bytes(cfg));
    for (const void* p : {q, k, v, out, dout, static_cast<const void*>(dq), static_cast<const void*>(dk),
                          static_cast<const void*>(dv), static_cast<const void*>(ws)})
        if (!dgm::aligned(p, 16)) return dgm::fail(g, DGM_ERR_UNSUPPORTED, "attnPackedBwd: a buffer is not 16-byte aligned");
    if (!dgm::aligned(starts, 4) || !dgm::aligned(lse, 4))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "attnPackedBwd: starts or lse is not 4-byte aligned");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "attnPackedBwd: %s", hipGetErrorString(on.err));
    const Strides s = strides(cfg);
    float* delta = static_cast<float*>(ws);
    const BwdArgs a{q, k, v, dout, dq, dk, dv, lse, delta, starts, g->seq_flag, cfg->rows, cfg->nseq, s.q, s.k, s.v,
                    s.o, 0, cfg->H, cfg->KVH, cfg->D, cfg->causal != 0, cfg->scale * kLog2e, cfg->scale};
    const DeltaArgs d{out, dout, delta, cfg->rows, s.o, cfg->H, cfg->D};
    g->seq_checks = true;
    return cfg->type == DGM_TYPE_F32 ? run_bwd<float>(g, cfg, a, d) : run_bwd<__bf16>(g, cfg, a, d);
}

}  // extern "C"
