// Lookup of token embeddings with scaling, and its gradient by sorted tokens. No
// counterpart in the reference, whose embed / embedBwd (train.hip) add positions to an fp32 or
// quantized table's rows and go through all tokens for every vocabulary row.
//
//   y[r] = scale table[tok[r]];  dtable[v] = (dtable[v] +) scale sum of dy[r] over the rows r with tok[r] = v
//
// The gradient sorts the tokens (stable, by digits of up to 9 bits), so that a token's rows lie together
// and each is read once. A unit, one wave, adds up a segment of the sorted rows in 256 columns; runs within its
// segment it writes, what crosses a segment's end it leaves in the workspace, and a last launch joins those in
// the order of the rows. Few tokens, or a few more of a small vocabulary, are not sorted: a workgroup for each looks
// for its rows itself. Nothing is added to by two workgroups: no atomics on results, the same bits every time.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "step.hpp"

namespace {

using namespace dgm_step;

constexpr uint32_t kNone = 0xFFFFFFFFu;   // no token

// ---- lookup -------------------------------------------------------------------

struct LookupArgs {
    const uint32_t* tokens;
    const void* table;
    void* y;
    uint32_t* words;
    int64_t rows;
    uint32_t V;
    int C;
    float scale;
    int team;   // lanes to a row, a power of two up to 256
};
// Pieces begin at a row's first element, whatever its address: the table's row and y's begin at different ones, so that not both can have
// them at multiples of 4 bytes (8192 bf16 rows of 4097 20.7 us, of 4096 19.5; of 1001 8.1, of 1000 7.6).
// 16-byte pieces that a lane asks for together (8192 rows of 4096, fp32: 41.4 us, with one 42.4, with four from half the lanes
// 41.2; 32768 bf16 rows of 512 9.6, 10.0, 10.4).
constexpr int kPieces = 2;

template <typename W, typename T>
__global__ __launch_bounds__(256) void embed_rows_kernel(LookupArgs a) {
    constexpr int N = kVec<T>;
    const int teams = 256 / a.team, lane = threadIdx.x & (a.team - 1);
    for (int64_t row = int64_t(blockIdx.x) * teams + threadIdx.x / a.team; row < a.rows; row += int64_t(gridDim.x) * teams) {
        const uint32_t tok = a.tokens[row];
        const bool held = tok < a.V;
        if (!held && tok != kNone && lane == 0) report(a.words, kBadTokens);
        const W* from = static_cast<const W*>(a.table) + int64_t(held ? tok : 0) * a.C;
        T* to = static_cast<T*>(a.y) + row * a.C;
        for (int c0 = lane * N; c0 < a.C; c0 += kPieces * a.team * N) {
            float x[kPieces][N];
#pragma unroll
            for (int u = 0; u < kPieces; ++u) load_piece<N>(from, c0 + u * a.team * N, a.C, x[u]);
#pragma unroll
            for (int u = 0; u < kPieces; ++u) {
#pragma unroll
                for (int j = 0; j < N; ++j) x[u][j] = held ? x[u][j] * a.scale : 0.0f;
                store_piece<N>(to, c0 + u * a.team * N, a.C, x[u]);
            }
        }
    }
}

// ---- the tokens in order ----------------------------------------------------------

constexpr int kSortThreads = 1024, kTile = 4096, kBatches = kTile / kSortThreads;
constexpr int kRun = 2048, kRunWave = kRun / 16, kRunBatches = kRunWave / 64;   // of the sort over several workgroups
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kMaxBlocks = 256;   // workgroups of that sort, each with a run of kRun elements or several

struct SortArgs {
    const uint32_t* tokens;               // of the first pass, which makes keys of them: V for rows without one
    const uint32_t *keys, *rows;          // of a later pass
    uint32_t *keys_out, *rows_out;
    uint32_t* hist;                       // [workgroups][bins]
    uint32_t* words;
    int64_t n;
    int64_t per;                          // elements of a workgroup's run
    uint32_t V;
    int passes, shift, bits, blocks;
    float* zero;                          // memory to clear beside the sort's first launch (may be null)
    int64_t zero_n;
};

template <bool FIRST>
__device__ __forceinline__ uint32_t key_of(const SortArgs& a, int64_t i) {
    if constexpr (!FIRST) return a.keys[i];
    const uint32_t t = a.tokens[i];
    if (t >= a.V && t != kNone) report(a.words, kBadTokens);
    return t < a.V ? t : a.V;
}

__device__ void clear(float* p, int64_t n, int64_t thread, int64_t threads) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        const dgm_attn::f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t i = thread; i < n / 4; i += threads) reinterpret_cast<dgm_attn::f32x4*>(p)[i] = none;
        for (int64_t i = (n & ~int64_t(3)) + thread; i < n; i += threads) p[i] = 0.0f;
    } else {
        for (int64_t i = thread; i < n; i += threads) p[i] = 0.0f;
    }
}

__global__ __launch_bounds__(256) void embed_clear_kernel(float* p, int64_t n) {
    clear(p, n, int64_t(blockIdx.x) * 256 + threadIdx.x, int64_t(gridDim.x) * 256);
}

// Up to kTile rows in one workgroup, by the digits, the lowest first, elements of a digit in their order: behind the
// smaller digits, the same digit of the waves before, of the wave's batches before, and of the lanes before. Bound by
// the ballots that find equal digits, about 0.7 us a pass for each 1024 rows, so that more than kTile are sorted sooner by several
// workgroups (5000 rows of 50257 x 512, all of it: 32 us, 43 in one).
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(SortArgs a) {
    __shared__ uint32_t held[kTile];
    __shared__ uint16_t from[kTile];
    __shared__ uint16_t count[16][kMaxBins];
    __shared__ uint32_t base[kMaxBins], sums[16];
    if (blockIdx.x > 0) {   // the others clear
        clear(a.zero, a.zero_n, int64_t(blockIdx.x - 1) * kSortThreads + threadIdx.x, int64_t(gridDim.x - 1) * kSortThreads);
        return;
    }
    const int bins = 1 << a.bits, t = threadIdx.x, lane = t & 63, wave = t >> 6, n = int(a.n);
    const int batches = (n + kSortThreads - 1) / kSortThreads, at0 = wave * batches * 64 + lane;   // each wave has as many in a row
    uint32_t key[kBatches];
    uint16_t row[kBatches];
#pragma unroll
    for (int u = 0; u < kBatches; ++u) {
        if (u >= batches) break;
        const int i = at0 + u * 64;
        key[u] = i < n ? key_of<true>(a, i) : 0;
        row[u] = uint16_t(i);
    }
    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = pass * a.bits;
        for (int d = t; d < 16 * bins; d += kSortThreads) count[d >> a.bits][d & (bins - 1)] = 0;
        __syncthreads();
        uint32_t rank[kBatches];
#pragma unroll
        for (int u = 0; u < kBatches; ++u) {
            if (u >= batches) break;
            const bool in = at0 + u * 64 < n;
            const uint32_t digit = (key[u] >> shift) & (bins - 1);
            uint64_t same = __ballot(in);
            for (int b = 0; b < a.bits; ++b) {
                const bool one = (digit >> b) & 1;
                const uint64_t ones = __ballot(one);
                same &= one ? ones : ~ones;
            }
            const uint32_t under = __builtin_amdgcn_mbcnt_hi(uint32_t(same >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(same), 0));
            const uint32_t had = count[wave][digit];
            // A wave's LDS accesses complete in the order of issue; the fences keep the compiler's.
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (in && under == 0) count[wave][digit] = uint16_t(had + __popcll(same));
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
            rank[u] = had + under;
        }
        __syncthreads();
        // Of each digit: what the waves before have, and all; then a scan over the digits.
        uint32_t total = 0;
        if (t < bins) {
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                const uint32_t c = count[w][t];
                count[w][t] = uint16_t(total);
                total += c;
            }
        }
        uint32_t scan = total;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(scan, off, 64);
            scan += lane >= off ? o : 0;
        }
        if (lane == 63) sums[wave] = scan;
        __syncthreads();
        for (int w = 0; w < wave; ++w) scan += sums[w];
        if (t < bins) base[t] = scan - total;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kBatches; ++u) {
            if (u >= batches || at0 + u * 64 >= n) continue;
            const uint32_t digit = (key[u] >> shift) & (bins - 1);
            const uint32_t to = base[digit] + count[wave][digit] + rank[u];
            held[to] = key[u];
            from[to] = row[u];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kBatches; ++u) {
            if (u >= batches || at0 + u * 64 >= n) continue;
            key[u] = held[at0 + u * 64];
            row[u] = from[at0 + u * 64];
        }
        // The next pass writes counts, which no one reads any more, and these behind two more barriers.
    }
#pragma unroll
    for (int u = 0; u < kBatches; ++u) {
        const int i = at0 + u * 64;
        if (u >= batches || i >= n) continue;
        a.keys_out[i] = key[u];
        a.rows_out[i] = row[u];
    }
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void embed_hist_kernel(SortArgs a) {
    __shared__ uint32_t count[kMaxBins];
    if (int(blockIdx.x) >= a.blocks) {   // the others clear
        clear(a.zero, a.zero_n, int64_t(blockIdx.x - a.blocks) * kSortThreads + threadIdx.x,
              int64_t(gridDim.x - a.blocks) * kSortThreads);
        return;
    }
    const int bins = 1 << a.bits;
    for (int d = threadIdx.x; d < bins; d += kSortThreads) count[d] = 0;
    __syncthreads();
    const int64_t from = int64_t(blockIdx.x) * a.per, to = std::min<int64_t>(a.n, from + a.per);
    for (int64_t i = from + threadIdx.x; i < to; i += kSortThreads)
        atomicAdd(&count[(key_of<FIRST>(a, i) >> a.shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) a.hist[int64_t(blockIdx.x) * bins + d] = count[d];
}

// Places a workgroup's run of elements by the digit, those of a digit in their order: behind the
// smaller digits of all workgroups, the same digit of the workgroups before, of this one's tiles before, of the tile's
// waves before, of the wave's batches before, and of the lanes before.
template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void embed_place_kernel(SortArgs a) {
    __shared__ uint32_t base[kMaxBins];                 // where this workgroup's next element of a digit goes
    __shared__ uint16_t count[16][kMaxBins];
    __shared__ uint32_t sums[16];
    const int bins = 1 << a.bits, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // Digits' totals and, of them, those of the workgroups before; then a scan over the digits.
    uint32_t total = 0, before = 0;
    if (t < bins) {
#pragma unroll 8
        for (int b = 0; b < a.blocks; ++b) {
            const uint32_t c = a.hist[int64_t(b) * bins + t];
            total += c;
            before += b < int(blockIdx.x) ? c : 0;
        }
    }
    uint32_t scan = total;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(scan, off, 64);
        scan += lane >= off ? o : 0;
    }
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    for (int w = 0; w < wave; ++w) scan += sums[w];
    if (t < bins) base[t] = scan - total + before;
    const int64_t from = int64_t(blockIdx.x) * a.per, to = std::min<int64_t>(a.n, from + a.per);
    for (int64_t tile = from; tile < to; tile += kRun) {
        for (int d = t; d < 16 * bins; d += kSortThreads) count[d / bins][d & (bins - 1)] = 0;
        __syncthreads();
        uint32_t key[kRunBatches], row[kRunBatches], rank[kRunBatches];
#pragma unroll
        for (int u = 0; u < kRunBatches; ++u) {
            const int64_t i = tile + wave * kRunWave + u * 64 + lane;
            key[u] = i < to ? key_of<FIRST>(a, i) : 0;
            row[u] = FIRST ? uint32_t(i) : i < to ? a.rows[i] : 0;
        }
#pragma unroll
        for (int u = 0; u < kRunBatches; ++u) {
            const bool in = tile + wave * kRunWave + u * 64 + lane < to;
            const uint32_t digit = (key[u] >> a.shift) & (bins - 1);
            uint64_t same = __ballot(in);
            for (int b = 0; b < a.bits; ++b) {
                const bool one = (digit >> b) & 1;
                const uint64_t ones = __ballot(one);
                same &= one ? ones : ~ones;
            }
            const uint32_t under = __builtin_amdgcn_mbcnt_hi(uint32_t(same >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(same), 0));
            const uint32_t had = count[wave][digit];
            // A wave's LDS accesses complete in the order of issue; the fences keep the compiler's.
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (in && under == 0) count[wave][digit] = uint16_t(had + __popcll(same));
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
            rank[u] = had + under;
        }
        __syncthreads();
        uint32_t all = 0;
        if (t < bins) {
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                const uint32_t c = count[w][t];
                count[w][t] = uint16_t(all);
                all += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kRunBatches; ++u) {
            if (tile + wave * kRunWave + u * 64 + lane >= to) continue;
            const uint32_t digit = (key[u] >> a.shift) & (bins - 1);
            const uint32_t at = base[digit] + count[wave][digit] + rank[u];
            a.keys_out[at] = key[u];
            a.rows_out[at] = row[u];
        }
        __syncthreads();
        if (t < bins) base[t] += all;
    }
}

// ---- sums ---------------------------------------------------------------------------

constexpr int kMaxSeg = 64, kMinSeg = 8;   // sorted rows of a unit
constexpr int kAhead = 8;                  // of them asked for together

// Everything that is added up is read once, and said so to the caches: 32768 bf16 rows of 50257 x 2048 with the lookup 143 us,
// 151 with ordinary loads; 16384 of 300 x 4096 74 and 87.
// Columns of a lane: 4 where rows are whole pieces of 4, else 1, so that no lane's columns are cut by a row's end (8192 rows of
// 50257 x 4096, added, 77 us, of 4097 95; bf16 66 and 85; of 1000 40, of 1001 52). Lanes behind a row's end load its last
// ones and store nothing.
inline int cols_of(int64_t C) { return C % 4 == 0 ? 4 : 1; }
template <int N, typename T>
__device__ __forceinline__ void load_cols(const T* p, float (&x)[N]) {
    const piece_t<T, N> v = __builtin_nontemporal_load(reinterpret_cast<const piece_t<T, N>*>(p));
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = float(v[j]);
}
template <int N>
__device__ __forceinline__ void store_cols(float* p, bool live, const float (&x)[N]) {
    piece_t<float, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = x[j];
    if (live) *reinterpret_cast<piece_t<float, N>*>(p) = v;
}

struct SumArgs {
    const void* dy;
    const uint32_t *keys, *rows;
    float* out;
    float *head, *tail;   // [segments][C]: of a run from the segment before, of one into the next
    int64_t n;
    uint32_t V;
    int C, slabs, add, seg;
    int64_t segs;
    float scale;
};

// A vocabulary row's sum into the gradient; `old` is what it held (0 where it is overwritten).
template <int N>
__device__ __forceinline__ void finish(const SumArgs& a, uint32_t v, int c, bool live, float (&acc)[N], const float (&old)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = old[j] + a.scale * acc[j];
    store_cols<N>(a.out + int64_t(v) * a.C + c, live, acc);
}

// Bound by memory where there is work: 32768 bf16 rows of 2048 columns, 9,900 different tokens, added to fp32 rows, 65 us for the 285 MB
// that move (4.4 TB/s, rows in no order); the sort before takes 22 in its four launches, the join 6.
template <typename T, int N>
__global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= a.segs * a.slabs) return;
    const int64_t seg = unit / a.slabs, p0 = seg * a.seg, p = p0 + lane;
    const int col = (int(unit - seg * a.slabs) * 64 + lane) * N, c = std::min(col, a.C - N);
    const bool live = col < a.C;
    const bool in = lane < a.seg && p < a.n;
    const uint32_t key = in ? a.keys[p] : a.V, row = in ? a.rows[p] : 0;
    const uint32_t prev = p0 > 0 ? a.keys[p0 - 1] : kNone, next = p0 + a.seg < a.n ? a.keys[p0 + a.seg] : kNone;
    const int n = __popcll(__ballot(key < a.V));   // sorted: rows without a token come last
    if (n == 0) return;
    const uint32_t left = __shfl_up(key, 1, 64), right = __shfl_down(key, 1, 64);
    const uint64_t heads = __ballot(key != (lane ? left : prev));   // a run begins
    const uint64_t tails = __ballot(key != (lane + 1 == a.seg ? next : right));   // and ends
    float acc[N] = {};
    for (int i0 = 0; i0 < n; i0 += kAhead) {
        // The rows, and what the runs that end among them are added to, all on their way together.
        float x[kAhead][N], old[kAhead][N] = {};
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u < n ? i0 + u : n - 1;
            const uint32_t r = __builtin_amdgcn_readlane(row, i);
            load_cols<N>(static_cast<const T*>(a.dy) + int64_t(r) * a.C + c, x[u]);
            if (a.add && (tails >> i & 1))
                load_cols<N>(a.out + int64_t(uint32_t(__builtin_amdgcn_readlane(key, i))) * a.C + c, old[u]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u;
            if (i >= n) break;
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] += x[u][j];
            const bool last = tails >> i & 1;
            if (!last && i + 1 < n) continue;
            const bool begun = heads & (~uint64_t(0) >> (63 - i));   // in this segment
            if (begun && last) finish<N>(a, __builtin_amdgcn_readlane(key, i), c, live, acc, old[u]);
            else store_cols<N>((begun ? a.tail : a.head) + seg * a.C + c, live, acc);
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        }
    }
}

// A run that begins in segment `seg` and goes on: its tail there, then the heads of the segments behind it, in four
// shares of the workgroup's waves.
template <int N>
__global__ __launch_bounds__(256) void embed_join_kernel(SumArgs a) {
    __shared__ float sums[4][64 * N];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t seg = blockIdx.x / a.slabs, p0 = seg * a.seg, end = p0 + a.seg;
    if (end >= a.n) return;
    const uint32_t v = a.keys[end - 1], next = a.keys[end], prev = p0 > 0 ? a.keys[p0 - 1] : kNone, first = a.keys[p0];
    if (v >= a.V || next != v) return;
    if (first == v && prev == v) return;   // it began before
    // Segments behind this one that the run reaches: it holds their first row.
    int64_t count = 0;
    for (;; count += 64) {
        const int64_t at = (seg + 1 + count + lane) * a.seg;
        const uint64_t in = __ballot(at < a.n && a.keys[at < a.n ? at : 0] == v);
        if (in != ~uint64_t(0)) {
            count += __builtin_ctzll(~in);
            break;
        }
    }
    const int col = (int(blockIdx.x - seg * a.slabs) * 64 + lane) * N, c = std::min(col, a.C - N);
    const bool live = col < a.C;
    float acc[N] = {}, old[N] = {};
    if (wave == 0) load_cols<N>(a.tail + seg * a.C + c, acc);
    if (wave == 0 && a.add) load_cols<N>(a.out + int64_t(v) * a.C + c, old);
    const int64_t from = seg + 1 + count * wave / 4, to = seg + 1 + count * (wave + 1) / 4;
#pragma unroll 8
    for (int64_t s = from; s < to; ++s) {
        float x[N];
        load_cols<N>(a.head + s * a.C + c, x);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += x[j];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) sums[wave][lane * N + j] = acc[j];
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < 4; ++w)
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += sums[w][lane * N + j];
    finish<N>(a, v, c, live, acc, old);
}

// ---- without a sort ---------------------------------------------------------------------

constexpr int kDirectRows = 4096;

// One token in 64 N columns: the token of each vocabulary row, or (BYROW) that of each row that has it first. The waves
// look through a share of the tokens each and list the rows that they find in their order; then each adds up a share of the
// list. A chain of two loads: 1024 rows of 65 x 128 5.3 us.
template <typename T, int N, int kDirectWaves, bool BYROW>
__global__ __launch_bounds__(64 * kDirectWaves) void embed_direct_kernel(SumArgs a, const uint32_t* __restrict__ tokens, uint32_t* words) {
    __shared__ uint16_t list[kDirectRows];
    __shared__ int found[kDirectWaves];
    __shared__ float sums[kDirectWaves][64 * N];
    constexpr int kTokens = kDirectRows / (64 * kDirectWaves);   // of a lane
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t which = blockIdx.x / a.slabs, v = BYROW ? tokens[which] : which;
    const int col = (int(blockIdx.x - which * a.slabs) * 64 + lane) * N, c = std::min(col, a.C - N);
    const bool live = col < a.C;
    const int each = (int(a.n) + 64 * kDirectWaves - 1) / (64 * kDirectWaves);   // batches of 64 tokens of a wave
    uint64_t hits[kTokens];
    if (BYROW && v >= a.V) {
        if (v != kNone && threadIdx.x == 0) report(words, kBadTokens);
        return;
    }
    int n = 0;
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
        if (u >= each) {
            hits[u] = 0;
            continue;
        }
        const int i = (wave * each + u) * 64 + lane;
        const uint32_t t = i < a.n ? tokens[i] : kNone;
        if (!BYROW && blockIdx.x == 0 && t >= a.V && t != kNone) report(words, kBadTokens);
        hits[u] = __ballot(t == v);
        n += __popcll(hits[u]);
    }
    if (lane == 0) found[wave] = n;
    float old[N] = {};
    if (a.add && wave == 0) load_cols<N>(a.out + int64_t(v) * a.C + c, old);
    __syncthreads();
    int all = 0, at = 0;
#pragma unroll
    for (int w = 0; w < kDirectWaves; ++w) {
        at = w == wave ? all : at;
        all += found[w];
    }
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
        if (hits[u] >> lane & 1)
            list[at + __builtin_amdgcn_mbcnt_hi(uint32_t(hits[u] >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(hits[u]), 0))] =
                uint16_t((wave * each + u) * 64 + lane);
        at += __popcll(hits[u]);
    }
    if (all == 0 && a.add) return;
    __syncthreads();
    if (BYROW && list[0] != which) return;   // a row before has it
    float acc[N] = {};
    const int to = all * (wave + 1) / kDirectWaves;
    for (int i0 = all * wave / kDirectWaves; i0 < to; i0 += kAhead) {
        float x[kAhead][N];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int r = __builtin_amdgcn_readfirstlane(list[i0 + u < to ? i0 + u : to - 1]);
            load_cols<N>(static_cast<const T*>(a.dy) + int64_t(r) * a.C + c, x[u]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (i0 + u < to)
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += x[u][j];
    }
    const int waves = all < kDirectWaves ? all : kDirectWaves;   // with all < 16 some shares in between are empty: zeros
#pragma unroll
    for (int j = 0; j < N; ++j) sums[wave][lane * N + j] = acc[j];
    __syncthreads();
    if (wave) return;
    if (waves)
        for (int w = 1; w < kDirectWaves; ++w)
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] += sums[w][lane * N + j];
    finish<N>(a, v, c, live, acc, old);
}

// ---- host ------------------------------------------------------------------------------

int check(dgm_gpu* g, const char* name, const dgm_rows_cfg* c) {
    if (!c) return dgm::fail(g, DGM_ERR_ARG, "%s: null configuration", name);
    if (!type_bytes(c->type) || !type_bytes(c->tableType))
        return dgm::fail(g, DGM_ERR_ARG, "%s: unknown type %d or %d", name, c->type, c->tableType);
    if (c->rows < 0 || c->C < 1 || c->V < 1 || !std::isfinite(c->scale))
        return dgm::fail(g, DGM_ERR_ARG, "%s: bad sizes or scale", name);
    if (c->rows > (int64_t(1) << 30) || c->V > dgm::kMaxIndex || c->C > (int64_t(1) << 24))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: rows beyond 2^30, a vocabulary beyond 2^31 - 1 or rows of more than 2^24",
                         name);
    return DGM_OK;
}

// Workgroups of token x columns up to which tokens are not sorted, each workgroup looking for its own (us with the lookup,
// added): 1000 rows of 50257 x 512, 2000 workgroups, 11 (sorted 17); 4000 rows of 50257 x 512, 8000, 30 (sorted 26). Up to
// kWideGroups of them have 16 waves: 4000 rows of 200 x 512 18 (22 with four); 2000 workgroups 15 with sixteen.
constexpr int64_t kDirectGroups = 2048, kWideGroups = 512;

// What the gradient's launches need of a configuration.
struct Plan {
    int passes, bits, blocks;
    int64_t per, segs;
    int slabs, seg;
    bool direct, byrow;
    int64_t lists, hist, parts;   // bytes of the workspace's areas
    int64_t bytes() const { return lists + hist + parts; }
};
int64_t round16(int64_t n) { return (n + 15) & ~int64_t(15); }
Plan plan_of(const dgm_rows_cfg* c) {
    Plan p;
    const int64_t wide = 64 * cols_of(c->C);
    p.slabs = int((c->C + wide - 1) / wide);
    const int64_t keys = std::min(c->V, c->rows);
    p.byrow = c->rows < c->V;
    p.direct = c->rows > 0 && c->rows <= kDirectRows && keys * p.slabs <= kDirectGroups;
    if (p.direct) {
        p.lists = p.hist = p.parts = 0;
        return p;
    }
    int width = 1;
    while ((int64_t(1) << width) <= c->V) ++width;   // keys 0 .. V
    p.passes = (width + kMaxBits - 1) / kMaxBits;
    p.bits = (width + p.passes - 1) / p.passes;
    const int64_t runs = (c->rows + kRun - 1) / kRun, each = (runs + kMaxBlocks - 1) / kMaxBlocks;
    p.per = each * kRun;
    p.blocks = c->rows <= kTile ? 0 : int((runs + each - 1) / each);
    p.hist = round16(int64_t(p.blocks) * (4 << p.bits));
    // Shorter segments where there is little work: 8 waves to a CU, if so many can be.
    p.seg = kMaxSeg;
    while (p.seg > kMinSeg && (c->rows + p.seg - 1) / p.seg * p.slabs < 8 * dgm::kCus) p.seg /= 2;
    p.segs = (c->rows + p.seg - 1) / p.seg;
    p.lists = 4 * round16(c->rows * 4);
    p.parts = 2 * round16(p.segs * c->C * 4);
    return p;
}

// f(type of dy, columns of a lane).
template <typename F>
void by_shape(const dgm_rows_cfg* c, const F& f) {
    using four = std::integral_constant<int, 4>;
    using one = std::integral_constant<int, 1>;
    if (c->type == DGM_TYPE_F32) cols_of(c->C) == 4 ? f(float{}, four{}) : f(float{}, one{});
    else cols_of(c->C) == 4 ? f(__bf16{}, four{}) : f(__bf16{}, one{});
}

// Whether a workgroup of 256 for each segment and slab is within a launch's bound on threads.
bool one_launch(const Plan& p) { return p.direct || p.segs * p.slabs <= int64_t(UINT32_MAX) / 256; }

}  // namespace

extern "C" {

int dgm_embedRows(dgm_gpu* g, const dgm_rows_cfg* cfg, const uint32_t* tokens, const void* table, void* y) {
    int rc = dgm::enter(g, "embed_rows");
    if (rc) return rc;
    rc = check(g, "embedRows", cfg);
    if (rc) return rc;
    if (cfg->rows == 0) return DGM_OK;
    if (!tokens || !table || !y) return dgm::fail(g, DGM_ERR_ARG, "embedRows: null buffer");
    if (!dgm::aligned(tokens, 4) || !dgm::aligned(table, size_t(type_bytes(cfg->tableType))) ||
        !dgm::aligned(y, size_t(type_bytes(cfg->type))))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "embedRows: a buffer is not aligned to its elements");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "embedRows: %s", hipGetErrorString(on.err));
    const int n = 16 / type_bytes(cfg->type);
    int team = 1;
    while (team < 256 && int64_t(team) * n * kPieces < cfg->C) team *= 2;
    const LookupArgs a{tokens, table, y, g->seq_report, cfg->rows, uint32_t(cfg->V), int(cfg->C), cfg->scale, team};
    const int teams = 256 / team;
    const dim3 grid(unsigned(std::min<int64_t>((cfg->rows + teams - 1) / teams, 1 << 22)));
    const bool wide = cfg->tableType == DGM_TYPE_F32;
    if (cfg->type == DGM_TYPE_F32)
        wide ? embed_rows_kernel<float, float><<<grid, dim3(256), 0, g->stream>>>(a)
             : embed_rows_kernel<__bf16, float><<<grid, dim3(256), 0, g->stream>>>(a);
    else
        wide ? embed_rows_kernel<float, __bf16><<<grid, dim3(256), 0, g->stream>>>(a)
             : embed_rows_kernel<__bf16, __bf16><<<grid, dim3(256), 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "embed_rows");
    return DGM_OK;
}

int64_t dgm_embedRowsBwd_ws_bytes(const dgm_rows_cfg* cfg) {
    if (check(nullptr, "", cfg) != DGM_OK) return -1;
    const Plan p = plan_of(cfg);
    return one_launch(p) ? p.bytes() : -1;
}

int dgm_embedRowsBwd(dgm_gpu* g, const dgm_rows_cfg* cfg, const uint32_t* tokens, const void* dy, float* dtable,
                     int accumulate, void* ws, int64_t ws_bytes) {
    int rc = dgm::enter(g, "embed_rows_bwd");
    if (rc) return rc;
    rc = check(g, "embedRowsBwd", cfg);
    if (rc) return rc;
    const Plan p = plan_of(cfg);
    if (!dtable || (cfg->rows > 0 && (!tokens || !dy)) || (p.bytes() > 0 && !ws))
        return dgm::fail(g, DGM_ERR_ARG, "embedRowsBwd: null buffer");
    if (ws_bytes < p.bytes())
        return dgm::fail(g, DGM_ERR_ARG, "embedRowsBwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)p.bytes());
    if (!dgm::aligned(tokens, 4) || !dgm::aligned(dy, size_t(type_bytes(cfg->type))) || !dgm::aligned(dtable, 4) || !dgm::aligned(ws, 16))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "embedRowsBwd: a buffer is not aligned to its elements, or the workspace to 16 bytes");
    if (!one_launch(p))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "embedRowsBwd: %lld rows of %lld exceed one launch", (long long)cfg->rows, (long long)cfg->C);
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "embedRowsBwd: %s", hipGetErrorString(on.err));
    SumArgs a{dy, nullptr, nullptr, dtable, nullptr, nullptr, cfg->rows, uint32_t(cfg->V), int(cfg->C), p.slabs, accumulate ? 1 : 0,
              0, 0, cfg->scale};
    if (p.direct) {
        const dim3 grid(unsigned(p.byrow ? cfg->rows : cfg->V) * unsigned(p.slabs));
        if (p.byrow && !accumulate) {
            const int64_t n = cfg->V * cfg->C;
            embed_clear_kernel<<<dim3(unsigned(std::min<int64_t>((n + 4095) / 4096, 2048))), dim3(256), 0, g->stream>>>(dtable, n);
            DGM_LAUNCH_CHECK(g, "embed_clear");
        }
        by_shape(cfg, [&](auto t, auto n) {
            constexpr int N = decltype(n)::value;
            using T = decltype(t);
            if (grid.x <= kWideGroups) {
                if (p.byrow) embed_direct_kernel<T, N, 16, true><<<grid, dim3(1024), 0, g->stream>>>(a, tokens, g->seq_report);
                else embed_direct_kernel<T, N, 16, false><<<grid, dim3(1024), 0, g->stream>>>(a, tokens, g->seq_report);
            } else {
                if (p.byrow) embed_direct_kernel<T, N, 4, true><<<grid, dim3(256), 0, g->stream>>>(a, tokens, g->seq_report);
                else embed_direct_kernel<T, N, 4, false><<<grid, dim3(256), 0, g->stream>>>(a, tokens, g->seq_report);
            }
        });
        DGM_LAUNCH_CHECK(g, "embed_direct");
        return DGM_OK;
    }
    uint8_t* at = static_cast<uint8_t*>(ws);
    uint32_t* lists[4];
    for (auto& l : lists) {
        l = reinterpret_cast<uint32_t*>(at);
        at += p.lists / 4;
    }
    const int64_t zero_n = accumulate ? 0 : cfg->V * cfg->C;
    const unsigned clearing = unsigned(std::min<int64_t>((zero_n + 16 * kSortThreads - 1) / (16 * kSortThreads), 2048));
    SortArgs s{tokens, nullptr, nullptr, lists[0], lists[1], reinterpret_cast<uint32_t*>(at), g->seq_report, cfg->rows, p.per,
               uint32_t(cfg->V), p.passes, 0, p.bits, p.blocks, dtable, zero_n};
    at += p.hist;
    const dim3 block{kSortThreads};
    if (p.blocks == 0) {
        if (cfg->rows + zero_n == 0) return DGM_OK;
        embed_sort_kernel<<<dim3(1 + clearing), block, 0, g->stream>>>(s);
        DGM_LAUNCH_CHECK(g, "embed_sort");
        if (cfg->rows == 0) return DGM_OK;
        s.keys = lists[0];
        s.rows = lists[1];
    } else {
        const dim3 grid{unsigned(p.blocks)};
        embed_hist_kernel<true><<<dim3(unsigned(p.blocks) + clearing), block, 0, g->stream>>>(s);
        embed_place_kernel<true><<<grid, block, 0, g->stream>>>(s);
        for (int i = 1; i < p.passes; ++i) {
            s.shift = i * p.bits;
            s.keys = s.keys_out;
            s.rows = s.rows_out;
            s.keys_out = lists[2 * (i & 1)];
            s.rows_out = lists[2 * (i & 1) + 1];
            embed_hist_kernel<false><<<grid, block, 0, g->stream>>>(s);
            embed_place_kernel<false><<<grid, block, 0, g->stream>>>(s);
        }
        DGM_LAUNCH_CHECK(g, "embed_place");
        s.keys = s.keys_out;
        s.rows = s.rows_out;
    }
    a.keys = s.keys;
    a.rows = s.rows;
    a.head = reinterpret_cast<float*>(at);
    a.tail = a.head + p.parts / 8;
    a.seg = p.seg;
    a.segs = p.segs;
    const dim3 grid(dgm::ceil_div(p.segs * p.slabs, 4));
    by_shape(cfg, [&](auto t, auto n) { embed_sum_kernel<decltype(t), decltype(n)::value><<<grid, dim3(256), 0, g->stream>>>(a); });
    DGM_LAUNCH_CHECK(g, "embed_sum");
    if (p.segs > 1) {
        const dim3 join{unsigned(p.segs * p.slabs)};
        by_shape(cfg, [&](auto, auto n) { embed_join_kernel<decltype(n)::value><<<join, dim3(256), 0, g->stream>>>(a); });
        DGM_LAUNCH_CHECK(g, "embed_join");
    }
    return DGM_OK;
}

}  // extern "C"
