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
//    that product follows the order in which a lane holds its scores; V is read
//    from LDS in the same order.
//  * The matrix unit runs on bf16 (v_mfma_f32_32x32x16_bf16). bf16 tensors take
//    one product, with P rounded to bf16 (half a step is 2^-9 of a weight's binade, and
//    the roundings of a row's weights are independent, so a row's error stays about that of
//    rounding its output once). fp32 tensors are split into three bf16 pieces of 8
//    bits, exactly, and take the six largest of their nine products: 192 cycles for
//    32x32x16, which v_mfma_f32_32x32x2_f32 does in 512. The pieces are cut and not
//    rounded, so that none overflows; the three products left out are then of the product's
//    sign, up to 2^-21 of it and 2^-24.5 on average. Scores, statistics and accumulators are fp32.
//  * Tiles of 64 (32) keys stay row-major in LDS: the A operand of the second product
//    is read transposed (ds_read_b64_tr_b16), and 16-byte chunks are XOR-swizzled so
//    that both reads are free of bank conflicts. bf16 tiles go from memory straight into
//    one of two buffers while the other is computed on, one barrier a tile; fp32 tiles
//    pass through registers, where they are split.
//  * Rows are found on the device, so that the grid needs no host copy of the lengths, and a
//    captured graph may be replayed with other ones: up to 64 sequences are ranked by a wave, longest
//    work first; of more, sequence s owns the tile slots from
//    starts[s] / rows-per-tile + s on, which never overlap.
//  * The running maximum moves only when a score exceeds it by more than 2^8:
//    the factor then stays exact in fp32 and the accumulators are rescaled a few
//    times in a row instead of at every tile.
//  * A masked position takes no part even if its v (or in the backward its k, q
//    or dout) is infinite or NaN, where 0 * inf would spread it over a whole
//    tile: tiles that hold both masked positions and such values are cleaned of them
//    first, and the sums that they belong to spoilt afterwards.
//
// Long sequences are bound by the matrix unit: a prompt of 8192 (32 heads on 8 of 128,
// bf16) takes 530 us, 1,040 TFLOP/s, where a library product reaches 1,158; four of 640 to 2048 in
// fp32 (16 heads on 4 of 64) 108 us, 151 TFLOP/s, where a library product reaches 153; fp32 heads of 128
// run one wave to a SIMD (256 us, 127 TFLOP/s), and of 256 spill (63 to 70). Short ones
// are a chain of waits: starts, tiles, exponentials, rows out (16 of 64: 6 us).
//
// The backward recomputes P from lse. One kernel owns 32 queries per wave and
// accumulates dq; another owns 32 keys per wave and accumulates dk and dv over all
// query heads of the key head's group, so no gradient is added to by two
// workgroups: no atomics, the same bits every time. Four of 2048 (16 heads on 8 of 128, bf16), back to back: forward 88 us, dq
// 151, dk and dv 186; the matrix unit is busy in half of dq's cycles and in 42% of the other's, whose waves wait for one another
// twice a tile. dq keeps 56 B a lane in scratch there (fp32 heads of 64 in pairs of waves 160, of 128 in narrow blocks 188): addresses
// of copies and query pieces, and a reload waits for every copy asked for before it.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "attn.hpp"

namespace {

using namespace dgm_attn;

// An operand in bf16 pieces: one, or the three of an fp32 value.
template <typename T>
constexpr int kPieces = sizeof(T) == 2 ? 1 : 3;

constexpr int64_t kMaxStride = int64_t(1) << 23;   // elements from row to row: see Feed::start

// ---- tiles in LDS ----------------------------------------------------------------

// A tile: kRows rows of D elements padded to DP columns, one row-major bf16 plane a
// piece. The 16-byte chunk c (8 columns) of row r sits at slot c ^ swizzle(r): 16
// rows' chunk c (the A operand of mm_rows) and 8 rows' four chunks (its transposed reads in
// mm_cols) then lie in different banks.
template <typename T, int DP, int ROWS>
struct Lds {
    static constexpr int kRows = ROWS;
    static constexpr int RB = DP * 2, CPR = RB / 16;          // bytes and chunks of a row
    static constexpr int RPB = RB >= 256 ? 1 : 256 / RB;      // rows that span all banks
    static constexpr int PLANE = kRows * RB, BYTES = kPieces<T> * PLANE;
    // Two buffers where tiles are copied straight from memory, one where they pass through registers.
    static constexpr int NBUF = sizeof(T) == 2 ? 2 : 1;
    static __device__ __forceinline__ int swizzle(int row) { return (row & 3) / RPB << 2 | (row >> 2 & 3); }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swizzle(row)) << 4); }
};

// The value of the first lane, for one that all share: the copies' instructions want it in scalar registers.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return uint32_t(__builtin_amdgcn_readfirstlane(int(x))); }

// A workgroup's way of bringing tiles to LDS. Each thread has N chunks of 8 columns, at
// 16 bytes x its number from the tile's (a plane's) start.
//
// bf16: copies straight into LDS (a wave's instruction fills 1 KB in lane order, so
// each lane fetches the chunk that belongs in its slot) while the other
// buffer is computed on. fp32: loads into registers while the one buffer is
// computed on, split into pieces and stored between two barriers.
//
// DC: the columns that the products read, D and zeros behind it.
template <typename T, int DP, int DC, int NT, int ROWS>
struct Feed {
    using L = Lds<T, DP, ROWS>;
    static constexpr int N = L::PLANE / 16 / NT, STEP = NT / L::CPR;   // STEP: rows between a thread's chunks
    static_assert(L::PLANE % (16 * NT) == 0 && NT % L::CPR == 0, "every thread has whole chunks of one slot");
    int64_t ldb;        // bytes from row to row
    int row, slot, wave;
    u32x4 held[sizeof(T) == 4 ? N : 1][2];

    __device__ __forceinline__ explicit Feed(int64_t ld)
        : ldb(ld * int64_t(sizeof(T))), row(int(threadIdx.x) / L::CPR), slot(int(threadIdx.x) % L::CPR),
          wave(__builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6)) {}

    // `rows` rows from `from` on, their first D columns; the rest of the tile's first DC is zero.
    __device__ __forceinline__ void start(uint8_t* lds, const T* from, int rows, int D) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(from);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = row + i * STEP, c = slot ^ L::swizzle(r);
                held[i][0] = held[i][1] = u32x4{0, 0, 0, 0};
                if (r < rows && c * 8 < D) {
                    const u32x4* p = reinterpret_cast<const u32x4*>(src + r * ldb + c * 32);
                    held[i][0] = p[0];
                    held[i][1] = p[1];
                }
            }
        } else {
            const uint32_t base = uniform(uint32_t(reinterpret_cast<uintptr_t>(lds)) + uint32_t(wave) * 1024u);
            const uint64_t at = reinterpret_cast<uintptr_t>(from);
            const uint8_t* const first = reinterpret_cast<const uint8_t*>(
                uint64_t(uniform(uint32_t(at >> 32))) << 32 | uniform(uint32_t(at)));
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
            static_assert(uint64_t(STEP - 1) * kMaxStride * sizeof(T) + L::RB <= UINT32_MAX,
                          "a thread's first row and slot are a 32-bit offset from the tile's start");
            const auto whole = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t off =
                        uint32_t(row) * uint32_t(ldb) + uint32_t((slot ^ L::swizzle(row + i * STEP)) << 4);
                    asm volatile(DGM_M0 "global_load_lds_dwordx4 %1, %2" ::"s"(base + i * NT * 16),
                                 "v"(off), "s"(first + i * STEP * ldb)
                                 : "memory", "m0");
                }
            };
            constexpr bool kOneChunk = STEP % 16 == 0;   // the same one of every row that a thread has
            if (rows >= L::kRows && D == DP) {
                whole();
            } else if (rows >= L::kRows && kOneChunk) {
                const int c = slot ^ L::swizzle(row);
                if (c * 8 < D)
                    whole();
                else if (c * 8 < DC)
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        *reinterpret_cast<u32x4*>(lds + (i * NT + int(threadIdx.x)) * 16) = u32x4{0, 0, 0, 0};
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int r = row + i * STEP, c = slot ^ L::swizzle(r);
                    if (r < rows && c * 8 < D)
                        asm volatile(DGM_M0 "global_load_lds_dwordx4 %1, off" ::"s"(base + i * NT * 16),
                                     "v"(src + r * ldb + c * 16)
                                     : "memory", "m0");
                    else
                        *reinterpret_cast<u32x4*>(lds + (i * NT + int(threadIdx.x)) * 16) = u32x4{0, 0, 0, 0};
                }
            }
#pragma clang diagnostic pop
        }
    }
    // fp32: the held rows' pieces to the planes.
    __device__ __forceinline__ void store(uint8_t* lds) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(held[i][j / 4][j % 4]);
                bf16x8 o[3];
                split8<3, kRare>(x, o);
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<bf16x8*>(lds + p * L::PLANE + (i * NT + int(threadIdx.x)) * 16) = o[p];
            }
        }
    }
    // Whether this thread's chunks of a tile in LDS hold infinities or NaN, which lie in the last plane.
    __device__ __forceinline__ bool bad(const uint8_t* lds) const {
        uint32_t b = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (DC < DP && (slot ^ L::swizzle(row + i * STEP)) * 8 >= DC) continue;
            const u32x4 v =
                *reinterpret_cast<const u32x4*>(lds + L::BYTES - L::PLANE + (i * NT + int(threadIdx.x)) * 16);
#pragma unroll
            for (int w = 0; w < 4; ++w) b |= ((v[w] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
        }
        return b != 0;
    }
};

// The copies that the workgroup has started are in LDS, and every wave's reads of what
// the next ones overwrite are done.
__device__ __forceinline__ void copies_ready() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Waits for the pair of tiles that was started last, in buffer `now`, and starts the next with `next()`.
template <typename T, int DP, int DC, int NT, int ROWS, typename Next>
__device__ __forceinline__ void turn(Feed<T, DP, DC, NT, ROWS>& a, Feed<T, DP, DC, NT, ROWS>& b,
                                     uint8_t (*now)[Lds<T, DP, ROWS>::BYTES], const Next& next) {
    if constexpr (sizeof(T) == 2) {
        copies_ready();
    } else {
        __syncthreads();
        a.store(now[0]);
        b.store(now[1]);
        __syncthreads();
    }
    next();
}

// ---- products ------------------------------------------------------------------

// B operand of mm_rows: a wave's 32 rows of q (k, dout, v), one a lane pair.
template <typename T, int DC>
struct Frags {
    static constexpr int NK = DC / 16;
    bf16x8 f[kPieces<T>][NK];
    __device__ __forceinline__ void load(const T* row, bool in, int D, int h) {
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
            const int d = 16 * kk + 8 * h;
            if constexpr (sizeof(T) == 2) {
                u32x4 w{0, 0, 0, 0};
                if (in && d < D) w = *reinterpret_cast<const u32x4*>(row + d);
                f[0][kk] = __builtin_bit_cast(bf16x8, w);
            } else {
                float x[8] = {};
                if (in && d < D) load8(row + d, x);
                bf16x8 o[3];
                split8<3, kSelect>(x, o);
#pragma unroll
                for (int p = 0; p < 3; ++p) f[p][kk] = o[p];
            }
        }
    }
    // Waits for the loads here: in a loop the wait would also be one for the copies that the loop starts.
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int p = 0; p < kPieces<T>; ++p)
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) asm volatile("" : "+v"(f[p][kk]));
    }
};

// acc += A B over their pieces: for fp32 the six largest products. kTurned: in the
// order that the product with A and B exchanged takes, for the same bits as it.
template <bool kTurned = false, int PA, int PB>
__device__ __forceinline__ void mfma_pieces(f32x16& acc, const bf16x8 (&a)[PA], const bf16x8 (&b)[PB]) {
#pragma unroll
    for (int s = PA + PB - 2; s >= 0; --s)   // the small ones first
#pragma unroll
        for (int n = 0; n < PA; ++n) {
            const int i = kTurned ? PA - 1 - n : n;
            if (s < 3 && s - i >= 0 && s - i < PB)
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[s - i], acc, 0, 0, 0);
        }
}

constexpr int kRead = 0x100, kMfma = 0x8;   // instruction classes of __builtin_amdgcn_sched_group_barrier

// The order of N operand reads (P pieces each) and their products: some reads ahead of
// the product that takes them. Left alone, the compiler reads into the registers
// that the product before has just taken, and every product waits for its own read
// (a prompt of 8192: 528 us so, 515 with six ahead).
template <int P, int N>
__device__ __forceinline__ void reads_ahead() {
    constexpr int M = P == 1 ? 1 : 6, AHEAD = P == 1 ? 6 : 2;
    if constexpr (N > AHEAD) {
        __builtin_amdgcn_sched_group_barrier(kRead, P * AHEAD, 0);
#pragma unroll
        for (int i = 0; i < N - AHEAD; ++i) {
            __builtin_amdgcn_sched_group_barrier(kMfma, M, 0);
            __builtin_amdgcn_sched_group_barrier(kRead, P, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, M * AHEAD, 0);
    }
}

// out[kb] (32 rows x the wave's 32 columns) = the tile's rows 32kb .. 32kb+31 times the
// columns' vectors. Element r of a lane: row 32kb + 8(r/4) + 4h + r%4, column lane %
// 32. The tile is part of one of ROWS rows.
template <typename T, int DP, int ROWS, int KB, int DC>
__device__ __forceinline__ void mm_rows(f32x16 (&out)[KB], const uint8_t* tile, const Frags<T, DC>& b, int lane) {
    using L = Lds<T, DP, ROWS>;
    constexpr int P = kPieces<T>;
    const int h = lane >> 5, r = lane & 31;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) out[kb] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < DC / 16; ++kk) {
        bf16x8 y[P];
#pragma unroll
        for (int p = 0; p < P; ++p) y[p] = b.f[p][kk];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            bf16x8 x[P];
#pragma unroll
            for (int p = 0; p < P; ++p)
                x[p] = *reinterpret_cast<const bf16x8*>(tile + p * L::PLANE + L::at(32 * kb + r, 2 * kk + h));
            mfma_pieces(out[kb], x, y);
        }
    }
    reads_ahead<P, DC / 16 * KB>();
}

// The same of two tiles and two sets of vectors, for KB blocks from kb0 on; the bits of mm_rows of
// the columns as a tile and the tile as columns.
template <typename T, int DP, int ROWS, int KB, int DC>
__device__ __forceinline__ void mm_rows2(f32x16 (&out)[KB], f32x16 (&out2)[KB], const uint8_t* tile, const uint8_t* tile2,
                                         int kb0, const Frags<T, DC>& b, const Frags<T, DC>& b2, int lane) {
    using L = Lds<T, DP, ROWS>;
    constexpr int P = kPieces<T>;
    const int h = lane >> 5, r = lane & 31;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) out[kb] = out2[kb] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < DC / 16; ++kk) {
        bf16x8 y[P], y2[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            y[p] = b.f[p][kk];
            y2[p] = b2.f[p][kk];
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int at = L::at(32 * (kb0 + kb) + r, 2 * kk + h);
            bf16x8 x[P], x2[P];
#pragma unroll
            for (int p = 0; p < P; ++p) {
                x[p] = *reinterpret_cast<const bf16x8*>(tile + p * L::PLANE + at);
                x2[p] = *reinterpret_cast<const bf16x8*>(tile2 + p * L::PLANE + at);
            }
            mfma_pieces<true>(out[kb], x, y);
            mfma_pieces<true>(out2[kb], x2, y2);
        }
    }
    reads_ahead<P, 2 * (DC / 16) * KB>();
}

// A operand of mm_cols: element j of a lane is column d = 32 dt + lane % 32 of
// row 32 kb + 16 st + 8 (j / 4) + 4h + j % 4, the order in which mm_rows leaves
// a lane's results. The transposed read takes, for each 16 lanes, 4 rows of 16
// columns (4 lanes a row) and gives each lane one column of them.
template <typename T, int DP>
__device__ __forceinline__ bf16x8 read_cols(const uint8_t* plane, int kb, int st, int dt, int lane) {
    using L = Lds<T, DP, 32>;   // the same for any number of rows
    const int row = 32 * kb + 16 * st + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int chunk = 4 * dt + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), in = (lane & 1) * 8;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* At;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)(plane + L::at(row, chunk) + in));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)(plane + L::at(row + 8, chunk) + in));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// acc[dt] (32 columns d x the wave's 32 columns) += tile^T times p, p as mm_rows
// leaves it, taken in PB pieces.
template <typename T, int DP, int PB, int ROWS, int KB, int DT>
__device__ __forceinline__ void mm_cols(f32x16 (&acc)[DT], const uint8_t* tile, const f32x16 (&p)[KB], int lane) {
    constexpr int PA = kPieces<T>;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = p[kb][8 * st + j];
            bf16x8 b[PB];
            split8<PB, kSpoils>(x, b);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                bf16x8 a[PA];
#pragma unroll
                for (int n = 0; n < PA; ++n)
                    a[n] = read_cols<T, DP>(tile + n * Lds<T, DP, ROWS>::PLANE, kb, st, dt, lane);
                mfma_pieces(acc[dt], a, b);
            }
        }
}

// What infinities and NaN do to sums that masked positions take no part in: a
// tile that holds both is cleaned (they become 0, as the weights of masked positions are), and
// for each column d the first (kLast: last) row of the sequence that held such a
// value is kept; a query (key) that sees that row has its sum spoilt in the end.
template <int DP, int KINDS>
struct Marks {
    int row[KINDS][DP];   // kinds: NaN, +inf, -inf; or all of them as one
    __device__ __forceinline__ void init(int none) {
        for (int i = threadIdx.x; i < KINDS * DP; i += blockDim.x) row[i / DP][i % DP] = none;
    }
};

// The tile's first row is row0 of the sequence.
template <typename T, int DP, int DC, int NT, int KINDS, bool kLast, int ROWS>
__device__ __forceinline__ void clean_tile(const Feed<T, DP, DC, NT, ROWS>& c, uint8_t* lds, int row0,
                                           Marks<DP, KINDS>& marks) {
    using F = Feed<T, DP, DC, NT, ROWS>;
    using L = typename F::L;
#pragma unroll 1
    for (int i = 0; i < F::N; ++i) {
        const int r = c.row + i * F::STEP, d0 = (c.slot ^ L::swizzle(r)) * 8;
        if (DC < DP && d0 >= DC) continue;
        __bf16* at = reinterpret_cast<__bf16*>(lds + L::BYTES - L::PLANE + (i * NT + int(threadIdx.x)) * 16);
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
            const float x = float(at[j]);
            if (fabsf(x) < __builtin_huge_valf()) continue;
            int* m = &marks.row[KINDS == 1 || x != x ? 0 : x > 0.0f ? 1 : 2][d0 + j];
            if (kLast) atomicMax(m, row0 + r);
            else atomicMin(m, row0 + r);
            at[j] = __bf16(0.0f);
        }
    }
    __syncthreads();
}

// `sees(row)`: whether the lane's column sees a row marked so.
template <int DP, int DT, int KINDS, typename Sees>
__device__ __forceinline__ void spoil(f32x16 (&acc)[DT], const Marks<DP, KINDS>& marks, int d0, const Sees& sees,
                                      int lane) {
    const float inf = __builtin_huge_valf();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int d = d0 + 32 * dt + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
            float x = acc[dt][e];
            if constexpr (KINDS == 3) {
                x += sees(marks.row[1][d]) ? inf : 0.0f;
                x += sees(marks.row[2][d]) ? -inf : 0.0f;
            }
            acc[dt][e] = sees(marks.row[0][d]) ? __builtin_nanf("") : x;
        }
}

// ---- rows ----------------------------------------------------------------------

// The tile of `per` rows that the n-th workgroup of a head takes. False where it has no rows.
struct Rows {
    int first, len, tile;   // the sequence's first row and length; the tile's number in it
};

// Sum over a wave of values >= 0, by DPP.
__device__ __forceinline__ int wave_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return __builtin_amdgcn_readlane(x, 63);
}

// Up to 64 sequences: the n-th tile in the order of falling tile numbers (kFromEnd: as
// counted from the sequence's end), over all sequences. With a causal mask
// that is the order of falling work, so that the longest workgroups start first.
// sum_s max(0, tiles_s - i) tiles have number i or more; a search by bits finds the n-th's.
template <bool kFromEnd>
__device__ __forceinline__ bool rank_rows(const int32_t* starts, int nseq, int64_t rows, int per, int n, Rows& out) {
    const int lane = threadIdx.x & 63;
    const bool there = lane < nseq;
    const int first = there ? clamped(starts, lane, rows) : 0;
    const int len = there ? max(clamped(starts, lane + 1, rows) - first, 0) : 0;
    const int tiles = (len + per - 1) / per;
    if (wave_sum(tiles) <= n) return false;
    int number = 0, bit = 1;
    while (__ballot(tiles > bit)) bit <<= 1;
    for (; bit; bit >>= 1)
        if (wave_sum(max(tiles - number - bit, 0)) > n) number += bit;
    const int before = wave_sum(max(tiles - number - 1, 0));
    const unsigned long long with = __ballot(tiles > number);
    const int rank = __builtin_amdgcn_mbcnt_hi(uint32_t(with >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(with), 0));
    const unsigned long long mine = __ballot(tiles > number && rank == n - before);
    if (!mine) return false;   // starts out of order, whose tiles add up to more than 32 bits
    const int s = __ffsll(mine) - 1;
    out.first = __builtin_amdgcn_readlane(first, s);
    out.len = __builtin_amdgcn_readlane(len, s);
    out.tile = kFromEnd ? __builtin_amdgcn_readlane(tiles, s) - 1 - number : number;
    return true;
}

// More: in the order of the tile slots (kFromEnd) or against it.
template <bool kFromEnd>
__device__ __forceinline__ bool find_rows(const int32_t* starts, int64_t nseq, int64_t rows, int per, int64_t slots,
                                          int64_t index, Rows& out) {
    if (nseq <= 64) return rank_rows<kFromEnd>(starts, int(nseq), rows, per, int(index), out);
    const int64_t slot = kFromEnd ? index : slots - 1 - index;
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, n = nseq;
    while (n > 64) {   // 64 candidates a round
        const int64_t step = (n + 63) / 64, at = lo + lane * step;
        const bool below = lane * step < n && slot_base(clamped(starts, at, rows), at, per) <= slot;
        const int c = __popcll(__ballot(below));
        if (c == 0) return false;
        lo += (c - 1) * step;
        n = n - (c - 1) * step < step ? n - (c - 1) * step : step;
    }
    // The last round reads the sequences' ends beside their starts: one wait, not two.
    const bool there = lane < n;
    const int first = there ? clamped(starts, lo + lane, rows) : 0, end = there ? clamped(starts, lo + lane + 1, rows) : 0;
    const int c = __popcll(__ballot(there && slot_base(first, lo + lane, per) <= slot));
    if (c == 0) return false;
    out.first = __builtin_amdgcn_readlane(first, c - 1);
    out.len = __builtin_amdgcn_readlane(end, c - 1) - out.first;
    const int64_t tile = slot - slot_base(out.first, lo + c - 1, per);
    out.tile = int(tile);
    return tile >= 0 && tile * per < out.len;
}

struct FwdArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;
    const int32_t* starts;
    uint32_t* report;
    int64_t rows, nseq, ldq, ldk, ldv, ldo, slots;
    int H, KVH, D, causal;
    float c;   // scale * log2 e
};

// Query head of the h'-th workgroup of a slot: consecutive workgroups go to
// different XCDs, so the heads of one group, which read the same k and v, are KVH apart.
__device__ __forceinline__ int head_of(int i, int H, int KVH) { return (i % KVH) * (H / KVH) + i / KVH; }

// Rows 32n + 8g + 4h .. +3 of a lane's column, times f, to columns d0 + .. of its row of the output.
template <typename T, int DT>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&acc)[DT], float f, int d0, int D, int h) {
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = d0 + 32 * n + 8 * g + 4 * h;
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

// Waves of a workgroup: QW blocks of 32 queries, each by KS waves that take every KS-th tile of
// TILE keys and are joined in the end. DP and DC: the columns of a tile, and those computed on (80 and 96 on 96 of 128: prompts of six
// times 1024, 16 heads, fp32 201 us -> 173, bf16 44 -> 40).
template <typename T_, int DP_, int DC_, int QW_, int KS_, int TILE_>
struct Shape {
    typedef T_ T;
    static constexpr int DP = DP_, DC = DC_, QW = QW_, KS = KS_, TILE = TILE_;
    static constexpr int BQ = 32 * QW, NT = 64 * QW * KS, ROWS = KS * TILE, KB = TILE / 32, DT = DC / 32;
    using L = Lds<T, DP, ROWS>;
    using F = Feed<T, DP, DC, NT, ROWS>;
    static constexpr int kTiles = L::NBUF * 2 * L::BYTES;
    template <int N>   // bytes for N floats a lane of every wave but a block's first
    static constexpr int kRoom = kTiles > QW * (KS - 1) * N * 256 ? kTiles : QW * (KS - 1) * N * 256;
};

// The three that there are; kind_of chooses.
enum Kind { kWhole, kPairs, kNarrow };
template <typename T, int DP, int DC>
using Whole = Shape<T, DP, DC, 4, 1, (sizeof(T) == 4 && DP > 64 ? 32 : 64)>;
template <typename T, int DP>
constexpr bool kHasPairs = DP <= (sizeof(T) == 2 ? 128 : 64);
template <typename T, int DP, int DC>
using Pairs = Shape<T, DP, DC, (sizeof(T) == 2 ? 2 : 4), 2, (DP == 128 ? 32 : 64)>;
template <int DP>
constexpr bool kHasNarrow = DP <= 128;
template <typename T, int DP, int DC>
using Narrow = Shape<T, DP, DC, 2, (sizeof(T) == 4 && DP == 128 ? 2 : 4),
                     (DP == 128 || (sizeof(T) == 4 && DP == 64) ? 32 : 64)>;

// Waves to a SIMD that the registers are to leave room for: two, unless tiles leave room for one
// workgroup of four waves to a CU, or the registers would spill.
template <typename S>
constexpr bool kAlone = S::NT == 256 && S::kTiles > 81920;

template <typename S>
__global__ void __launch_bounds__(S::NT, S::DP <= (sizeof(typename S::T) == 2 ? 128 : 64) && !kAlone<S> ? 2 : 1)
    attn_packed_fwd_kernel(FwdArgs a) {
    using T = typename S::T;
    using L = typename S::L;
    constexpr int DP = S::DP, DC = S::DC, QW = S::QW, KS = S::KS, TILE = S::TILE, ROWS = S::ROWS, NT = S::NT, DT = S::DT,
                  KB = S::KB, BQ = S::BQ;
    __shared__ __align__(16) uint8_t room[S::template kRoom<DT * 16 + 2>];
    uint8_t(*lds)[2][L::BYTES] = reinterpret_cast<uint8_t(*)[2][L::BYTES]>(room);   // k and v
    __shared__ Marks<DP, 3> marks;
    marks.init(INT_MAX);
    if (blockIdx.x == gridDim.x - 1) check_starts(a.starts, a.nseq, a.rows, a.report);   // one with little to do
    Rows rw;
    if (!find_rows<false>(a.starts, a.nseq, a.rows, BQ, a.slots, blockIdx.x / a.H, rw)) return;
    const int head = head_of(blockIdx.x % a.H, a.H, a.KVH), kvh = head / (a.H / a.KVH);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, kg = wave / QW;
    const int q0 = rw.tile * BQ + wave % QW * 32, row = q0 + (lane & 31);   // in the sequence
    const bool in = row < rw.len;
    const int64_t at = int64_t(rw.first) + row;
    const T* k = static_cast<const T*>(a.k) + int64_t(rw.first) * a.ldk + int64_t(kvh) * a.D;
    const T* v = static_cast<const T*>(a.v) + int64_t(rw.first) * a.ldv + int64_t(kvh) * a.D;
    typename S::F ck(a.ldk), cv(a.ldv);
    const auto start = [&](int t) __attribute__((always_inline)) {
        const int key0 = t * ROWS;
        ck.start(lds[t % L::NBUF][0], k + key0 * a.ldk, rw.len - key0, a.D);
        cv.start(lds[t % L::NBUF][1], v + key0 * a.ldv, rw.len - key0, a.D);
    };
    start(0);

    Frags<T, DC> qf;
    qf.load(static_cast<const T*>(a.q) + at * a.ldq + int64_t(head) * a.D, in, a.D, h);
    f32x16 o[DT];
#pragma unroll
    for (int n = 0; n < DT; ++n) o[n] = f32x16{};
    float m = kNegInf, l = 0.0f;
    const int last = a.causal && in ? row : rw.len - 1;   // the last key that the lane's query sees
    const int keys = a.causal ? min(rw.len, (rw.tile + 1) * BQ) : rw.len, steps = (keys + ROWS - 1) / ROWS;
    // Steps from here on hold positions that some query of the workgroup does not see.
    const int masked_from = a.causal ? rw.tile * BQ / ROWS : rw.len / ROWS;
    const int wave_keys = a.causal ? min(keys, q0 + 32) : keys;

    qf.settle();
    bool spoilt = false;
    for (int t = 0; t < steps; ++t) {
        turn(ck, cv, lds[t % L::NBUF], [&]() __attribute__((always_inline)) {
            if (t + 1 < steps) start(t + 1);
        });
        const bool masked = t >= masked_from;
        if (masked && a.causal && __syncthreads_or(cv.bad(lds[t % L::NBUF][1]))) {
            clean_tile<T, DP, DC, NT, 3, false>(cv, lds[t % L::NBUF][1], t * ROWS, marks);
            spoilt = true;
        }
        const int key0 = t * ROWS + kg * TILE;
        if (key0 >= wave_keys || q0 >= rw.len) continue;
        const uint8_t* kt = lds[t % L::NBUF][0] + kg * TILE * L::RB;
        const uint8_t* vt = lds[t % L::NBUF][1] + kg * TILE * L::RB;
        f32x16 s[KB];
        mm_rows<T, DP, ROWS>(s, kt, qf, lane);
        if (masked) {
            const int lim = last - key0 - 4 * h;   // element e of block kb is seen up to here
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[kb][e] = 32 * kb + 8 * (e / 4) + e % 4 <= lim ? s[kb][e] : kNegInf;
        }
        float mx = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (__any((mx - m) * a.c > 8.0f)) {   // also from -inf; inf - inf is NaN: no move
            const float to = fmaxf(m, mx), f = m == kNegInf ? 0.0f : exp2_hw((m - to) * a.c);
            l *= f;
#pragma unroll
            for (int n = 0; n < DT; ++n) o[n] *= f;
            m = to;
        }
        const float mc = m == kNegInf ? 0.0f : m * a.c;
        float sum = 0.0f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[kb][e] = exp2_hw(__builtin_fmaf(s[kb][e], a.c, -mc));
                sum += s[kb][e];
            }
        l += sum;
        mm_cols<T, DP, kPieces<T>, ROWS>(o, vt, s, lane);
    }
    if constexpr (KS > 1) {   // the other waves' parts of a block, through LDS
        constexpr int N = (DT * 16 + 2) * 64;
        float* part = reinterpret_cast<float*>(room) + wave % QW * (KS - 1) * N + lane;
        __syncthreads();
        if (kg > 0) {
            part += (kg - 1) * N;
            part[0] = m;
            part[64] = l;
#pragma unroll
            for (int n = 0; n < DT; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) part[(2 + n * 16 + e) * 64] = o[n][e];
        }
        __syncthreads();
        if (kg > 0) return;
        for (int i = 0; i < KS - 1; ++i, part += N) {
            const float m1 = part[0], to = fmaxf(m, m1);
            const float f0 = m == to ? 1.0f : exp2_hw((m - to) * a.c), f1 = m1 == to ? 1.0f : exp2_hw((m1 - to) * a.c);
            m = to;
            l = l * f0 + part[64] * f1;
#pragma unroll
            for (int n = 0; n < DT; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[n][e] = o[n][e] * f0 + part[(2 + n * 16 + e) * 64] * f1;
        }
    }
    if (spoilt) spoil<DP>(o, marks, 0, [&](int r) { return r <= last; }, lane);

    const float sum = l + __shfl_xor(l, 32, 64);
    if (!in) return;
    if (a.lse && h == 0) a.lse[int64_t(head) * a.rows + at] = (m == kNegInf ? 0.0f : m * a.c) + log2_hw(sum);
    store_row<T, DT>(static_cast<T*>(a.out) + at * a.ldo + int64_t(head) * a.D, o, 1.0f / sum, 0, a.D, h);
}

// ---- backward ------------------------------------------------------------------

// Pieces of dS. One would do for bf16 as it does for P, but leaves dq and dk, which are
// rounded once more, 1.5 times as far off as one rounding.
template <typename T>
constexpr int kSlopePieces = sizeof(T) == 2 ? 2 : 3;

// Delta of rows that see kFewKeys keys or less. Over few keys it is as large as dP, and what rounded out, or the sums of
// either, is off by stays in dS. 400 sequences of 128 causal bf16 tokens, heads of 128, dq's error by that of rounding it once:
// median 2.2 and at the worst 420 in the row of two keys, 1.0 and 30 of four, 0.2 and 3 from 65 on; fp32 rows of two keys were
// 1e-6 off. So there it is what it stands for, the sum of P dP by that of P, as a difference from dP of key 0, and
// one key alone leaves exactly 0. It goes by the keys that a row sees and by nothing else, so that neither the rest of the batch
// nor the layout changes a row's delta.
template <typename T>
constexpr int kFewKeys = sizeof(T) == 2 ? 64 : 16;
template <typename T>
constexpr int kFewBlocks = (kFewKeys<T> + 31) / 32;   // of 32 keys

struct FewKeys {
    float ref = 0.0f, sum = 0.0f, weights = 0.0f;
    // Of 32 keys, a query in each lane pair: s and dP as mm_rows leaves them, keys up to element lim are seen. The same
    // order in every kernel, for the same bits.
    __device__ __forceinline__ void add(const f32x16& s, const f32x16& dp, int lim, float c, float lse) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const bool see = 8 * (e / 4) + e % 4 <= lim;
            const float p = see ? exp2_hw(__builtin_fmaf(s[e], c, -lse)) : 0.0f;
            weights += p;
            sum += see ? p * (dp[e] - ref) : 0.0f;
        }
    }
    __device__ __forceinline__ float delta() const {
        return ref + (sum + __shfl_xor(sum, 32, 64)) / (weights + __shfl_xor(weights, 32, 64));
    }
};

struct BwdArgs {
    const void *q, *k, *v, *out, *dout;
    void *dq, *dk, *dv;
    const float* lse;
    float* delta;   // [H, rows]
    float* sums;    // [parts][dk, dv][rows, KVH, D], with several parts
    const int32_t* starts;
    uint32_t* report;
    int64_t rows, nseq, ldq, ldk, ldv, ldo, slots;
    int H, KVH, D, causal, parts, per;   // per: rows of a workgroup that adds parts
    float c, scale;
};

// dq: a wave's 32 queries against tiles of 64 keys. dS^T = P^T (dP^T - delta)
// with dP^T = V dout^T; dq^T += K^T dS^T. delta = dout . out on the way, kept for the next kernel; of rows that see few keys,
// from a first pass over those. (A pass of its own: in the loop it would cost registers, and four of 2048 430 us -> 443.)
template <typename S>
struct DqRoom {
    __align__(16) uint8_t room[S::template kRoom<S::DT * 16>];
    Marks<S::DP, 1> marks;
};

template <typename S>
__device__ __forceinline__ void dq_body(const BwdArgs& a, DqRoom<S>& sh, uint32_t index, bool last_block) {
    using T = typename S::T;
    using L = typename S::L;
    constexpr int DP = S::DP, DC = S::DC, QW = S::QW, KS = S::KS, TILE = S::TILE, ROWS = S::ROWS, NT = S::NT, DT = S::DT,
                  KB = S::KB, BQ = S::BQ;
    uint8_t* const room = sh.room;
    uint8_t(*lds)[2][L::BYTES] = reinterpret_cast<uint8_t(*)[2][L::BYTES]>(room);   // k and v
    Marks<DP, 1>& marks = sh.marks;
    marks.init(INT_MAX);
    if (last_block) check_starts(a.starts, a.nseq, a.rows, a.report);   // one with little to do
    Rows rw;
    if (!find_rows<false>(a.starts, a.nseq, a.rows, BQ, a.slots, index / a.H, rw)) return;
    const int head = head_of(index % a.H, a.H, a.KVH), kvh = head / (a.H / a.KVH);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, kg = wave / QW;
    const int q0 = rw.tile * BQ + wave % QW * 32, row = q0 + (lane & 31);
    const bool in = row < rw.len;
    const int64_t at = int64_t(rw.first) + row;
    const T* k = static_cast<const T*>(a.k) + int64_t(rw.first) * a.ldk + int64_t(kvh) * a.D;
    const T* v = static_cast<const T*>(a.v) + int64_t(rw.first) * a.ldv + int64_t(kvh) * a.D;
    typename S::F ck(a.ldk), cv(a.ldv);
    const auto start = [&](int t) __attribute__((always_inline)) {
        const int key0 = t * ROWS;
        ck.start(lds[t % L::NBUF][0], k + key0 * a.ldk, rw.len - key0, a.D);
        cv.start(lds[t % L::NBUF][1], v + key0 * a.ldv, rw.len - key0, a.D);
    };
    start(0);
    const T* grad = static_cast<const T*>(a.dout) + at * a.ldo + int64_t(head) * a.D;
    const T* out = static_cast<const T*>(a.out) + at * a.ldo + int64_t(head) * a.D;
    Frags<T, DC> qf, gf;
    qf.load(static_cast<const T*>(a.q) + at * a.ldq + int64_t(head) * a.D, in, a.D, h);
    gf.load(grad, in, a.D, h);
    float delta = 0.0f;
#pragma unroll
    for (int d = 8 * h; d < DC; d += 16)
        if (in && d < a.D) {
            float x[8], y[8];
            load8(grad + d, x);
            load8(out + d, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) delta = __builtin_fmaf(x[j], y[j], delta);
        }
    delta += __shfl_xor(delta, 32, 64);
    float lse = in ? a.lse[int64_t(head) * a.rows + at] : 0.0f;
    asm volatile("" : "+v"(lse), "+v"(delta));
    const int last = a.causal && in ? row : rw.len - 1;
    static_assert(ROWS >= kFewKeys<T> && ROWS >= 32 * kFewBlocks<T>, "the first tile holds the few keys");
    if (a.causal ? rw.tile * BQ < kFewKeys<T> : rw.len <= kFewKeys<T>) {
        turn(ck, cv, lds[0], [] {});
        if (q0 < rw.len && (!a.causal || q0 < kFewKeys<T>)) {   // each of a block's waves for itself
            FewKeys few;
#pragma unroll 1   // unrolled, four of 2048 take 4 us more: registers
            for (int kb = 0; kb < kFewBlocks<T>; ++kb) {
                f32x16 s[1], dp[1];
                mm_rows<T, DP, ROWS>(s, lds[0][0] + kb * 32 * L::RB, qf, lane);
                mm_rows<T, DP, ROWS>(dp, lds[0][1] + kb * 32 * L::RB, gf, lane);
                if (kb == 0) few.ref = __shfl(dp[0][0], lane & 31, 64);
                few.add(s[0], dp[0], last - 32 * kb - 4 * h, a.c, lse);
            }
            const float of_few = few.delta();
            delta = last < kFewKeys<T> ? of_few : delta;
        }
    }
    if (in && h == 0 && kg == 0) a.delta[int64_t(head) * a.rows + at] = delta;
    f32x16 acc[DT];
#pragma unroll
    for (int n = 0; n < DT; ++n) acc[n] = f32x16{};

    const int keys = a.causal ? min(rw.len, (rw.tile + 1) * BQ) : rw.len, steps = (keys + ROWS - 1) / ROWS;
    const int masked_from = a.causal ? rw.tile * BQ / ROWS : rw.len / ROWS;
    const int wave_keys = a.causal ? min(keys, q0 + 32) : keys;
    qf.settle();
    gf.settle();
    bool spoilt = false;
    for (int t = 0; t < steps; ++t) {
        turn(ck, cv, lds[t % L::NBUF], [&]() __attribute__((always_inline)) {
            if (t + 1 < steps) start(t + 1);
        });
        const int key0 = t * ROWS + kg * TILE;
        const uint8_t* kt = lds[t % L::NBUF][0] + kg * TILE * L::RB;
        const uint8_t* vt = lds[t % L::NBUF][1] + kg * TILE * L::RB;
        const bool masked = t >= masked_from, active = key0 < wave_keys && q0 < rw.len;
        const bool dirty = masked && a.causal && __syncthreads_or(ck.bad(lds[t % L::NBUF][0]));
        f32x16 s[KB], dp[KB];
        if (active) {
            if constexpr (sizeof(T) == 2) {
                mm_rows2<T, DP, ROWS>(s, dp, kt, vt, 0, qf, gf, lane);
            } else {   // one after the other: there are no registers for reads of both
                mm_rows<T, DP, ROWS>(s, kt, qf, lane);
                mm_rows<T, DP, ROWS>(dp, vt, gf, lane);
            }
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[kb][e] = exp2_hw(__builtin_fmaf(s[kb][e], a.c, -lse)) * (dp[kb][e] - delta);
            if (masked) {
                const int lim = last - key0 - 4 * h;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        s[kb][e] = 32 * kb + 8 * (e / 4) + e % 4 <= lim ? s[kb][e] : 0.0f;
            }
        }
        if (dirty) {
            __syncthreads();   // the tile has been read as it is
            clean_tile<T, DP, DC, NT, 1, false>(ck, lds[t % L::NBUF][0], t * ROWS, marks);
            spoilt = true;
        }
        if (active) mm_cols<T, DP, kSlopePieces<T>, ROWS>(acc, kt, s, lane);
    }
    if constexpr (KS > 1) {
        constexpr int N = DT * 16 * 64;
        float* part = reinterpret_cast<float*>(room) + wave % QW * (KS - 1) * N + lane;
        __syncthreads();
        if (kg > 0)
#pragma unroll
            for (int n = 0; n < DT; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) part[(kg - 1) * N + (n * 16 + e) * 64] = acc[n][e];
        __syncthreads();
        if (kg > 0) return;
        for (int i = 0; i < KS - 1; ++i, part += N)
#pragma unroll
            for (int n = 0; n < DT; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[n][e] += part[(n * 16 + e) * 64];
    }
    if (spoilt) spoil<DP>(acc, marks, 0, [&](int r) { return r <= last; }, lane);
    if (in) store_row<T, DT>(static_cast<T*>(a.dq) + at * a.ldq + int64_t(head) * a.D, acc, a.scale, 0, a.D, h);
}

template <typename S>
__global__ void __launch_bounds__(S::NT, (sizeof(typename S::T) == 2 && !kAlone<S>) || S::NT == 512 ? 2 : 1)
    attn_packed_dq_kernel(BwdArgs a) {
    __shared__ DqRoom<S> room;
    dq_body<S>(a, room, blockIdx.x, blockIdx.x == gridDim.x - 1);
}

// dk, dv: a pair of waves' 32 keys as columns against tiles of 64 queries, over the query heads
// of the group one after the other. S = Q K^T, dP = dout V^T; dv^T += dout^T P, dk^T += Q^T dS.
//
// dk and dv of 32 keys are 128 registers at D = 128, and a wave with them, k, v and the
// scores has room for one on a SIMD, where nothing runs beside its waits and its
// exponentials. So a pair shares the keys: each wave computes P and dS for half of the tile's
// rows, hands them to the other through LDS as the B operands that they are, and
// accumulates half of the columns of dk and dv. Four blocks of 2048 (16 heads on 8
// of 128, bf16), before parts shared the steps: 428 us with whole waves, 336 so.
//
// Where that gives too few workgroups (few key heads, short batches), `parts` of
// them share a key tile's steps and leave fp32 sums in the workspace, which a
// second kernel adds up in order.
template <typename T, int DP>
struct DkvShape {
    // Waves: as many as leave room for the tiles and the handed-over operands (2 KB a piece and wave).
    static constexpr int NW = sizeof(T) == 2 ? (DP == 128 ? 8 : 4) : (DP == 64 ? 8 : 4);
    static constexpr int BK = 16 * NW;   // keys
};

template <typename T, int DP>
struct DkvRoom {
    using L = Lds<T, DP, 64>;
    __align__(16) uint8_t lds[L::NBUF][2][L::BYTES];                                  // q and dout
    bf16x8 hand[DkvShape<T, DP>::NW][kPieces<T> + kSlopePieces<T>][2][64];            // P and dS, by wave, piece, 16 rows
    __align__(16) float stat[2][2][64];                                               // lse and delta, of two tiles
    __align__(16) float few[32];                                                      // delta of rows that see few keys
    Marks<DP, 1> marks[2];
};

// kOwnDelta: delta from out and dout (or of few keys) here, not from the dq kernel.
template <typename T, int DP, int DC, bool kOwnDelta>
__device__ __forceinline__ void dkv_body(const BwdArgs& a, DkvRoom<T, DP>& sh, uint32_t index) {
    using L = Lds<T, DP, 64>;
    constexpr int NW = DkvShape<T, DP>::NW, NT = 64 * NW, BK = DkvShape<T, DP>::BK, TILE = 64;
    constexpr int PP = kPieces<T>, PS = kSlopePieces<T>;
    constexpr bool kSplitD = DC % 64 == 0;              // else the pair's waves take dv and dk, one each
    constexpr int DT = kSplitD ? DC / 64 : DC / 32;     // blocks of 32 columns of a wave
    auto& lds = sh.lds;
    auto& hand = sh.hand;
    auto& stat = sh.stat;
    auto& marks = sh.marks;
    marks[0].init(-1);
    marks[1].init(-1);
    Rows rw;
    const int kvh = index % a.KVH, G = a.H / a.KVH, part = int(index / a.KVH % a.parts);
    if (!find_rows<true>(a.starts, a.nseq, a.rows, BK, a.slots, index / a.KVH / a.parts, rw)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, half = wave & 1;
    const int k0 = rw.tile * BK + wave / 2 * 32, row = k0 + (lane & 31);
    const bool in = row < rw.len;
    const int64_t at = int64_t(rw.first) + row;
    const int first = a.causal ? rw.tile * BK / TILE : 0, per_head = (rw.len + TILE - 1) / TILE - first;
    const int t0 = int(int64_t(per_head) * G * part / a.parts), t1 = int(int64_t(per_head) * G * (part + 1) / a.parts);
    Feed<T, DP, DC, NT, 64> cq(a.ldq), cg(a.ldo);
    static_assert(NT >= 2 * TILE, "a thread stages one statistic");
    int head = kvh * G + t0 / per_head, tile = first + t0 % per_head, now = tile;   // of the next copy; computed on
    struct Raw8 {
        u32x4 w[sizeof(T) / 2];
    };
    float stat_held = 0.0f;
    Raw8 grad_held[kOwnDelta ? DP / 32 : 1], out_held[kOwnDelta ? DP / 32 : 1];
    const auto store_stat = [&](int t) __attribute__((always_inline)) {
        if (threadIdx.x < (kOwnDelta ? TILE : 2 * TILE)) stat[t % 2][threadIdx.x / TILE][threadIdx.x & (TILE - 1)] = stat_held;
        if constexpr (kOwnDelta) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                float x[8], y[8];
                load8(reinterpret_cast<const T*>(&grad_held[i]), x);
                load8(reinterpret_cast<const T*>(&out_held[i]), y);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(x[j], y[j], sum);
            }
            sum += __shfl_xor(sum, 1, 64);
            sum += __shfl_xor(sum, 2, 64);
            if ((threadIdx.x & 3) == 0) stat[t % 2][1][threadIdx.x / 4] = sum;
        }
    };
    const auto start = [&](int t) __attribute__((always_inline)) {
        const int row0 = tile * TILE;
        const int64_t r0 = int64_t(rw.first) + row0;
        // First, and kept in registers until the tile's turn: a wait for these is one for all that was asked for before.
        if (threadIdx.x < (kOwnDelta ? TILE : 2 * TILE)) {
            const int r = threadIdx.x & (TILE - 1);
            const float* from = threadIdx.x < TILE ? a.lse : a.delta;
            stat_held = row0 + r < rw.len ? from[int64_t(head) * a.rows + r0 + r] : 0.0f;
        }
        if constexpr (kOwnDelta) {   // 4 lanes a row
            static_assert(NT == 4 * TILE, "every thread has a quarter of a row");
            const int r = threadIdx.x / 4;
            const int64_t from = (r0 + r) * a.ldo + int64_t(head) * a.D;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const int d = 32 * i + 8 * (threadIdx.x & 3);
                grad_held[i] = out_held[i] = {};
                if (row0 + r < rw.len && d < a.D) {
                    grad_held[i] = *reinterpret_cast<const Raw8*>(static_cast<const T*>(a.dout) + from + d);
                    out_held[i] = *reinterpret_cast<const Raw8*>(static_cast<const T*>(a.out) + from + d);
                }
            }
        }
        cq.start(lds[t % L::NBUF][0], static_cast<const T*>(a.q) + r0 * a.ldq + int64_t(head) * a.D, rw.len - row0, a.D);
        cg.start(lds[t % L::NBUF][1], static_cast<const T*>(a.dout) + r0 * a.ldo + int64_t(head) * a.D, rw.len - row0,
                 a.D);
        if (++tile - first == per_head) {
            tile = first;
            ++head;
        }
    };
    if (t0 < t1) start(t0);
    Frags<T, DC> kf, vf;
    kf.load(static_cast<const T*>(a.k) + at * a.ldk + int64_t(kvh) * a.D, in, a.D, h);
    vf.load(static_cast<const T*>(a.v) + at * a.ldv + int64_t(kvh) * a.D, in, a.D, h);
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int n = 0; n < DT; ++n) dk[n] = dv[n] = f32x16{};

    kf.settle();
    vf.settle();
    bool spoilt = false;
    for (int t = t0; t < t1; ++t) {
        const int row0 = now * TILE;
        uint8_t* qt = lds[t % L::NBUF][0];
        uint8_t* gt = lds[t % L::NBUF][1];
        const float* lse = stat[t % 2][0] + 32 * half + 4 * h;
        const float* delta = stat[t % 2][1] + 32 * half + 4 * h;
        store_stat(t);
        turn(cq, cg, lds[t % L::NBUF], [&]() __attribute__((always_inline)) {
            if (t + 1 < t1) start(t + 1);
        });
        // Positions not seen: queries before the workgroup's last key, or behind the sequence.
        const bool hidden = a.causal && row0 < (rw.tile + 1) * BK;
        const bool active = k0 < rw.len && !(a.causal && row0 + TILE <= k0);
        const bool dirty = hidden && __syncthreads_or(cq.bad(qt) || cg.bad(gt));
        if constexpr (kOwnDelta) {
            // Rows that see few keys are among the first 32, their keys among this wave's: no other one sees those. The
            // dq kernel's products, keys as rows and queries as columns, with the same bits.
            static_assert(kFewKeys<T> <= 32 && kFewBlocks<T> == 1, "one wave has them");
            if (k0 == 0 && half == 0 && row0 == 0 && (a.causal || rw.len <= kFewKeys<T>)) {
                f32x16 s{}, dp{};
#pragma unroll
                for (int kk = 0; kk < DC / 16; ++kk) {
                    bf16x8 kx[PP], vx[PP], x[PP], y[PP];
#pragma unroll
                    for (int p = 0; p < PP; ++p) {
                        const int at = p * L::PLANE + L::at(lane & 31, 2 * kk + h);
                        kx[p] = kf.f[p][kk];
                        vx[p] = vf.f[p][kk];
                        x[p] = *reinterpret_cast<const bf16x8*>(qt + at);
                        y[p] = *reinterpret_cast<const bf16x8*>(gt + at);
                    }
                    mfma_pieces(s, kx, x);
                    mfma_pieces(dp, vx, y);
                }
                const int r = lane & 31, seen = a.causal && r < rw.len ? r : rw.len - 1;   // its last key
                FewKeys few;
                few.ref = __shfl(dp[0], r, 64);
                few.add(s, dp, seen - 4 * h, a.c, stat[t % 2][0][r]);
                const float of_few = few.delta();
                if (h == 0) sh.few[r] = seen < kFewKeys<T> ? of_few : stat[t % 2][1][r];
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                delta = sh.few + 4 * h;
            }
        }
        if (active) {
            f32x16 p1[1], ds1[1];
            mm_rows2<T, DP, 64>(p1, ds1, qt, gt, half, kf, vf, lane);
            f32x16 &p = p1[0], &ds = ds1[0];
            // Element e is row 32 half + 8(e/4) + e%4 + 4h.
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 ls = *reinterpret_cast<const f32x4*>(lse + 8 * g);
                const f32x4 de = *reinterpret_cast<const f32x4*>(delta + 8 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 4 * g + i;
                    p[e] = exp2_hw(__builtin_fmaf(p[e], a.c, -ls[i]));
                    ds[e] = p[e] * (ds[e] - de[i]);
                }
            }
            if (hidden || row0 + TILE > rw.len) {
                const int r0 = row0 + 32 * half + 4 * h, lo = (a.causal ? row : 0) - r0, hi = rw.len - r0;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int i = 8 * (e / 4) + e % 4;
                    const bool see = i >= lo && i < hi;
                    p[e] = see ? p[e] : 0.0f;
                    ds[e] = see ? ds[e] : 0.0f;
                }
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                float x[8], y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[j] = p[8 * st + j];
                    y[j] = ds[8 * st + j];
                }
                bf16x8 px[PP], sx[PS];
                split8<PP, kSpoils>(x, px);
                split8<PS, kSpoils>(y, sx);
#pragma unroll
                for (int n = 0; n < PP; ++n) hand[wave][n][st][lane] = px[n];
#pragma unroll
                for (int n = 0; n < PS; ++n) hand[wave][PP + n][st][lane] = sx[n];
            }
        }
        __syncthreads();
        if (dirty) {   // the tiles have been read as they are
            clean_tile<T, DP, DC, NT, 1, true>(cq, qt, row0, marks[0]);
            clean_tile<T, DP, DC, NT, 1, true>(cg, gt, row0, marks[1]);
            spoilt = true;
        }
        if (active) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    const auto& from = hand[(wave & ~1) + kb];
                    bf16x8 px[PP], sx[PS];
#pragma unroll
                    for (int n = 0; n < PP; ++n) px[n] = from[n][st][lane];
#pragma unroll
                    for (int n = 0; n < PS; ++n) sx[n] = from[PP + n][st][lane];
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const int d = kSplitD ? half * DT + dt : dt;
                        bf16x8 x[PP], y[PP];
#pragma unroll
                        for (int n = 0; n < PP; ++n) {
                            x[n] = read_cols<T, DP>(gt + n * L::PLANE, kb, st, d, lane);
                            y[n] = read_cols<T, DP>(qt + n * L::PLANE, kb, st, d, lane);
                        }
                        if (kSplitD || half == 0) mfma_pieces(dv[dt], x, px);
                        if (kSplitD || half == 1) mfma_pieces(dk[dt], y, sx);
                    }
                }
            if constexpr (sizeof(T) == 2 && kSplitD) {   // as reads_ahead, two reads to a product
                __builtin_amdgcn_sched_group_barrier(kRead, 14, 0);
#pragma unroll
                for (int i = 0; i < 4 * DT * 3; ++i) {
                    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
                }
            }
        }
        if (++now - first == per_head) now = first;
    }
    const int d0 = kSplitD ? half * 32 * DT : 0;
    if (spoilt) {
        const auto sees = [&](int r) { return r >= 0 && r >= row; };
        spoil<DP>(dk, marks[0], d0, sees, lane);
        spoil<DP>(dv, marks[1], d0, sees, lane);
    }
    if (!in) return;
    const bool mine_v = kSplitD || half == 0, mine_k = kSplitD || half == 1;
    if (a.parts > 1) {
        const int64_t r = at * a.KVH + kvh, all = a.rows * a.KVH;
        float* sums = a.sums + (int64_t(part) * 2 * all + r) * a.D;
        if (mine_k) store_row<float, DT>(sums, dk, 1.0f, d0, a.D, h);
        if (mine_v) store_row<float, DT>(sums + all * a.D, dv, 1.0f, d0, a.D, h);
        return;
    }
    if (mine_k) store_row<T, DT>(static_cast<T*>(a.dk) + at * a.ldk + int64_t(kvh) * a.D, dk, a.scale, d0, a.D, h);
    if (mine_v) store_row<T, DT>(static_cast<T*>(a.dv) + at * a.ldv + int64_t(kvh) * a.D, dv, 1.0f, d0, a.D, h);
}

template <typename T, int DP, int DC>
__global__ void __launch_bounds__((64 * DkvShape<T, DP>::NW), (sizeof(T) == 4 && DP == 128 ? 1 : 2))
    attn_packed_dkv_kernel(BwdArgs a) {
    __shared__ DkvRoom<T, DP> room;
    dkv_body<T, DP, DC, false>(a, room, blockIdx.x);
}

// Both in one launch, a workgroup one or the other, for grids that the chip holds at once:
// forward and backward of 16 sequences of 64 (4 heads of 32, fp32) take 16 us so, 22 in three launches.
template <typename T, int DP>
__global__ void __launch_bounds__(256, 2) attn_packed_grads_kernel(BwdArgs a, uint32_t first, int64_t dkv_slots) {
    __shared__ union Room {
        DqRoom<Whole<T, DP, DP>> dq;
        DkvRoom<T, DP> dkv;
        __device__ Room() {}
    } room;
    if (blockIdx.x < first) {
        dq_body<Whole<T, DP, DP>>(a, room.dq, blockIdx.x, blockIdx.x == first - 1);
    } else {
        a.slots = dkv_slots;
        dkv_body<T, DP, DP, true>(a, room.dkv, blockIdx.x - first);
    }
}

// The parts' sums of dk and dv, added in order: a workgroup takes a.per rows of one
// sequence and head, 4 columns a thread; 8 parts are asked for at once, then added
// (one after the other, 8 heads of 128 on one over 400 rows wait 22 us longer).
template <typename T>
__global__ void __launch_bounds__(256) attn_packed_sum_kernel(BwdArgs a) {
    Rows rw;
    const int kvh = blockIdx.x % a.KVH;
    if (!find_rows<true>(a.starts, a.nseq, a.rows, a.per, a.slots, blockIdx.x / a.KVH, rw)) return;
    const int64_t all = a.rows * a.KVH;
    const int quads = a.D / 4;
    for (int i = threadIdx.x; i < 2 * a.per * quads; i += 256) {
        const int which = i / (a.per * quads), r = rw.tile * a.per + i / quads % a.per, d = i % quads * 4;
        if (r >= rw.len) continue;
        const int64_t at = int64_t(rw.first) + r;
        const float* from = a.sums + (which * all + at * a.KVH + kvh) * a.D + d;
        f32x4 sum{0, 0, 0, 0};
        for (int p = 0; p < a.parts; p += 8) {
            f32x4 x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = p + j < a.parts ? *reinterpret_cast<const f32x4*>(from + (p + j) * 2 * all * a.D) : f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += x[j];
        }
        T* to = which ? static_cast<T*>(a.dv) + at * a.ldv + int64_t(kvh) * a.D
                      : static_cast<T*>(a.dk) + at * a.ldk + int64_t(kvh) * a.D;
        const float f = which ? 1.0f : a.scale;
#pragma unroll
        for (int j = 0; j < 4; ++j) to[d + j] = T(sum[j] * f);
    }
}

// ---- host ----------------------------------------------------------------------

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

// A launch of few workgroups waits for its longest, and that is made shorter by more waves for a
// block of queries, each with its share of the keys, and by blocks of fewer
// queries. Both cost: a tile is staged for fewer queries, and the waves of a
// workgroup wait for one another.
//  * kNarrow, 64 queries by 8 waves (4 where fp32 tiles of 128 columns leave no room), while
//    there is no more than one such workgroup to a CU, or two for long sequences:
//    four of 70 to 1500 under 4 heads, fp32 of 64 60 us -> 44 (and the backward 162 -> 125), of 128
//    157 -> 110, bf16 of 128 29.3 -> 24.9. But ten of 300 under 8 heads, bf16: 14.0, 21.4.
//  * kPairs, two waves a block. bf16 (64 queries) gains while four waves' workgroups would be no
//    more than two to a CU (seven of 1 to 1024 under 12 heads of 128: 28.5 -> 24.7; 16 heads of 96, six of
//    1024: 39.8, 47.8); fp32 (128), where two workgroups of four waves leave
//    less overlap, on any grid (16 heads of 64, 2048 and shorter: 129 -> 108), but
//    not in its backward, short of registers (four of 1024: 370, 376).
//  * Sequences of one tile have nothing to share (16 of 64: 6.6, 7.5); lengths differ, and the longest
//    sets the time, so that an average of two is enough (18 of 1 to 745, bf16 of 80, forward and
//    backward 98 -> 88; the call's rows by its sequences, those of none among them; nine of 100, 8 heads of 128: bf16 63, 66, fp32 135 -> 128).
template <typename T>
Kind kind_of(const dgm_attn_cfg* c, bool forward) {
    const int64_t average = c->rows / c->nseq;
    if (average <= 64) return kWhole;
    if (slot_count(c->rows, c->nseq, 64) * c->H <= (average > 512 ? 2 : 1) * dgm::kCus && c->D <= 128) return kNarrow;
    const bool few = slot_count(c->rows, c->nseq, 128) * c->H <= 2 * dgm::kCus;
    return few || (sizeof(T) == 4 && forward) ? kPairs : kWhole;
}

template <typename S>
int launch_fwd(dgm_gpu* g, const dgm_attn_cfg* c, FwdArgs a) {
    const int rc = slots_of(g, "attnPackedFwd", c, S::BQ, c->H, S::NT, a.slots);
    if (rc) return rc;
    attn_packed_fwd_kernel<S><<<dim3(unsigned(a.slots * c->H)), dim3(S::NT), 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "attn_packed_fwd");
    return DGM_OK;
}

template <typename T, int DP, int DC>
int choose_fwd(dgm_gpu* g, const dgm_attn_cfg* c, const FwdArgs& a) {
    const Kind kind = kind_of<T>(c, true);
    if constexpr (kHasNarrow<DP>)
        if (kind == kNarrow) return launch_fwd<Narrow<T, DP, DC>>(g, c, a);
    if constexpr (kHasPairs<T, DP>)
        if (kind == kPairs) return launch_fwd<Pairs<T, DP, DC>>(g, c, a);
    return launch_fwd<Whole<T, DP, DC>>(g, c, a);
}

template <typename T>
int run_fwd(dgm_gpu* g, const dgm_attn_cfg* c, const FwdArgs& a) {
    if (c->D <= 32) return choose_fwd<T, 32, 32>(g, c, a);
    if (c->D <= 64) return choose_fwd<T, 64, 64>(g, c, a);
    if (c->D <= 96) return choose_fwd<T, 128, 96>(g, c, a);
    if (c->D <= 128) return choose_fwd<T, 128, 128>(g, c, a);
    return choose_fwd<T, 256, 256>(g, c, a);
}

// Keys of a workgroup of the dk, dv kernel.
int dkv_keys(const dgm_attn_cfg* c) {
    if (c->type == DGM_TYPE_BF16)
        return c->D <= 32 ? DkvShape<__bf16, 32>::BK : c->D <= 64 ? DkvShape<__bf16, 64>::BK : DkvShape<__bf16, 128>::BK;
    return c->D <= 32 ? DkvShape<float, 32>::BK : c->D <= 64 ? DkvShape<float, 64>::BK : DkvShape<float, 128>::BK;
}

// dq and dk, dv can go in one launch, each with its own delta from out and dout: with as many threads
// to a workgroup, no more workgroups than two to a CU, an exact out (fp32) and more than 32 rows to a sequence on average.
template <typename T, int DP>
constexpr bool kOneLaunch = sizeof(T) == 4 && DP == 32;
bool one_launch(const dgm_attn_cfg* c) {
    return c->type == DGM_TYPE_F32 && c->D <= 32 && c->rows > 32 * c->nseq && slot_count(c->rows, c->nseq, 128) * c->H + slot_count(c->rows, c->nseq, dkv_keys(c)) * c->KVH <=
                       2 * dgm::kCus;
}

// Workgroups that share a key tile's steps, each with a step or more at the sequences' average length (15
// of 1 to 1280, one fp32 head of 128, forward and backward 375 us, with two steps or more each; 301 so):
// as many as give
//  * bf16 of more than 64 columns, whose tiles fill a CU's LDS with one workgroup: one to a CU. In the order of
//    falling work, the longest beside the shortest, more only add sums to write and read
//    (four blocks of 2048, 16 heads on 8 of 128: 410 us whole, 467 in two parts; six of 1024, 16 on 4: 229, 246);
//  * fp32 of more than 32 columns, also one to a CU but with steps six times as long: two (seven of 1 to
//    1024, 12 heads on 4 of 64: 252 us with one, 213 with two, 220 with three);
//  * the others, of which a CU holds two or more: three (24 heads on 8 of 64, six of 283 on average: 80 us,
//    87 with two, 84 with four).
// One launch for dq, dk and dv is worth more than parts of a few steps: dq then runs beside them.
// fp32, 4 heads of 32 over four times 256, 41 us in parts, 28 whole; but 8 query heads on 2 over 900 rows 40 and 50.
int64_t dkv_parts(const dgm_attn_cfg* c) {
    const int64_t tiles = slot_count(c->rows, c->nseq, dkv_keys(c)) * c->KVH;
    const int64_t steps = (c->rows / std::max<int64_t>(c->nseq, 1) + 63) / 64 * (c->H / c->KVH);
    if (steps <= (c->H == c->KVH ? 16 : 4) && one_launch(c)) return 1;
    const int per_cu = c->type == DGM_TYPE_BF16 ? (c->D > 64 ? 1 : 3) : c->D > 32 ? 2 : 3;
    return std::max<int64_t>(1, std::min<int64_t>({16, (per_cu * dgm::kCus + tiles - 1) / std::max<int64_t>(tiles, 1), steps}));
}

template <typename S>
int launch_dq(dgm_gpu* g, const dgm_attn_cfg* c, BwdArgs a) {
    const int rc = slots_of(g, "attnPackedBwd", c, S::BQ, c->H, S::NT, a.slots);
    if (rc) return rc;
    attn_packed_dq_kernel<S><<<dim3(unsigned(a.slots * c->H)), dim3(S::NT), 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "attn_packed_dq");
    return DGM_OK;
}
template <typename T, int DP, int DC>
int choose_dq(dgm_gpu* g, const dgm_attn_cfg* c, const BwdArgs& a) {
    const Kind kind = kind_of<T>(c, false);
    if constexpr (kHasNarrow<DP>)
        if (kind == kNarrow) return launch_dq<Narrow<T, DP, DC>>(g, c, a);
    if constexpr (kHasPairs<T, DP>)
        if (kind == kPairs) return launch_dq<Pairs<T, DP, DC>>(g, c, a);
    return launch_dq<Whole<T, DP, DC>>(g, c, a);
}

template <typename T, int DP, int DC>
int launch_bwd(dgm_gpu* g, const dgm_attn_cfg* c, BwdArgs kv) {
    constexpr int NK = DkvShape<T, DP>::NW;
    int rc = slots_of(g, "attnPackedBwd", c, DkvShape<T, DP>::BK, c->KVH * kv.parts, 64 * NK, kv.slots);
    if (rc) return rc;
    if constexpr (kOneLaunch<T, DP>) {
        if (kv.parts == 1 && one_launch(c)) {
            BwdArgs q = kv;
            q.slots = slot_count(c->rows, c->nseq, Whole<T, DP, DP>::BQ);
            const int64_t first = q.slots * c->H, all = first + kv.slots * c->KVH;
            attn_packed_grads_kernel<T, DP>
                <<<dim3(unsigned(all)), dim3(256), 0, g->stream>>>(q, uint32_t(first), kv.slots);
            DGM_LAUNCH_CHECK(g, "attn_packed_grads");
            return DGM_OK;
        }
    }
    rc = choose_dq<T, DP, DC>(g, c, kv);
    if (rc) return rc;
    attn_packed_dkv_kernel<T, DP, DC>
        <<<dim3(unsigned(kv.slots * c->KVH * kv.parts)), dim3(64 * NK), 0, g->stream>>>(kv);
    DGM_LAUNCH_CHECK(g, "attn_packed_dkv");
    if (kv.parts > 1) {
        // 32 rows where that gives four workgroups to a CU (four blocks of 2048: 31 us, with 8 rows 37), else 8 (12 of
        // 200, 2 heads: 44 us in all, 43).
        kv.per = slot_count(c->rows, c->nseq, 32) * c->KVH >= 4 * dgm::kCus ? 32 : 8;
        rc = slots_of(g, "attnPackedBwd", c, kv.per, c->KVH, 256, kv.slots);
        if (rc) return rc;
        attn_packed_sum_kernel<T><<<dim3(unsigned(kv.slots * c->KVH)), dim3(256), 0, g->stream>>>(kv);
        DGM_LAUNCH_CHECK(g, "attn_packed_sum");
    }
    return DGM_OK;
}

template <typename T>
int run_bwd(dgm_gpu* g, const dgm_attn_cfg* c, const BwdArgs& a) {
    if (c->D <= 32) return launch_bwd<T, 32, 32>(g, c, a);
    if (c->D <= 64) return launch_bwd<T, 64, 64>(g, c, a);
    if (c->D <= 96) return launch_bwd<T, 128, 96>(g, c, a);
    return launch_bwd<T, 128, 128>(g, c, a);
}

constexpr int kMaxD = 256, kMaxDBwd = 128;

// delta, and the parts' sums.
int64_t delta_floats(const dgm_attn_cfg* c) { return (c->rows * c->H + 3) / 4 * 4; }
int64_t bwd_ws_bytes(const dgm_attn_cfg* c) {
    const int64_t parts = dkv_parts(c);
    return (delta_floats(c) + (parts > 1 ? parts * 2 * c->rows * c->KVH * c->D : 0)) * int64_t(sizeof(float));
}

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
    FwdArgs a{q, k, v, out, lse, starts, g->seq_report, cfg->rows, cfg->nseq, s.q, s.k, s.v, s.o, 0, cfg->H, cfg->KVH,
              cfg->D, cfg->causal != 0, cfg->scale * kLog2e};
    return cfg->type == DGM_TYPE_F32 ? run_fwd<float>(g, cfg, a) : run_fwd<__bf16>(g, cfg, a);
}

int64_t dgm_attnPackedBwd_ws_bytes(const dgm_attn_cfg* cfg) {
    if (!cfg || check_cfg(nullptr, "", cfg, kMaxDBwd) != DGM_OK) return -1;
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
    const BwdArgs a{q, k, v, out, dout, dq, dk, dv, lse, delta, delta + delta_floats(cfg), starts, g->seq_report,
                    cfg->rows, cfg->nseq, s.q, s.k, s.v, s.o, 0, cfg->H, cfg->KVH, cfg->D, cfg->causal != 0,
                    int(dkv_parts(cfg)), 0, cfg->scale * kLog2e, cfg->scale};
    return cfg->type == DGM_TYPE_F32 ? run_bwd<float>(g, cfg, a) : run_bwd<__bf16>(g, cfg, a);
}

}  // extern "C"
