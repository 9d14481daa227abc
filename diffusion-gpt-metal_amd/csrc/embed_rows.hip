// Lookup of token embeddings with scaling, and its gradient by sorted tokens. No
// counterpart in the reference, whose embed / embedBwd (train.hip) add positions to an fp32 or
// quantized table's rows and go through all tokens for every vocabulary row.
//
//   y[r] = scale table[tok[r]];  dtable[v] = (dtable[v] +) scale sum of dy[r] over the rows r with tok[r] = v
//
// The gradient sorts the tokens (stable, by digits of up to 9 bits), so that a token's rows lie together
// and each is read once. A unit, one wave, adds up to kSeg sorted rows of 64 pieces of columns; runs within its
// segment it writes, what crosses a segment's end it leaves in the workspace, and a last launch joins those in
// the order of the rows. Nothing is added to by two waves: no atomics on results, the same bits every time.
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
        for (int c = lane * N; c < a.C; c += a.team * N) {
            float x[N];
            load_piece<N>(from, c, a.C, x);
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = held ? x[j] * a.scale : 0.0f;
            store_piece<N>(to, c, a.C, x);
        }
    }
}

// ---- the tokens in order ----------------------------------------------------------

constexpr int kSortThreads = 1024, kTile = 4096, kPerWave = kTile / 16, kBatches = kPerWave / 64;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kMaxBlocks = 256;   // sorting workgroups, each with a run of tiles

struct SortArgs {
    const uint32_t* tokens;               // of the first pass, which makes keys of them: V for rows without one
    const uint32_t *keys, *rows;          // of a later pass
    uint32_t *keys_out, *rows_out;
    uint32_t* hist;                       // [workgroups][bins]
    uint32_t* words;
    int64_t n;
    int64_t per;                          // elements of a workgroup's run
    uint32_t V;
    int shift, bits, blocks;
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
    for (int64_t tile = from; tile < to; tile += kTile) {
        for (int d = t; d < 16 * bins; d += kSortThreads) count[d / bins][d & (bins - 1)] = 0;
        __syncthreads();
        uint32_t key[kBatches], row[kBatches], rank[kBatches];
#pragma unroll
        for (int u = 0; u < kBatches; ++u) {
            const int64_t i = tile + wave * kPerWave + u * 64 + lane;
            key[u] = i < to ? key_of<FIRST>(a, i) : 0;
            row[u] = FIRST ? uint32_t(i) : i < to ? a.rows[i] : 0;
        }
#pragma unroll
        for (int u = 0; u < kBatches; ++u) {
            const bool in = tile + wave * kPerWave + u * 64 + lane < to;
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
        for (int u = 0; u < kBatches; ++u) {
            if (tile + wave * kPerWave + u * 64 + lane >= to) continue;
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

constexpr int kSeg = 64;     // sorted rows of a unit
constexpr int kAhead = 8;    // of them asked for together

struct SumArgs {
    const void* dy;
    const uint32_t *keys, *rows;
    float* out;
    float *head, *tail;   // [segments][C]: of a run from the segment before, of one into the next
    int64_t n;
    uint32_t V;
    int C, slabs, add;
    int64_t segs;
    float scale;
};

template <int N>
__device__ __forceinline__ void finish(const SumArgs& a, uint32_t v, int c, float (&acc)[N]) {
    float* row = a.out + int64_t(v) * a.C;
    float old[N];
#pragma unroll
    for (int j = 0; j < N; ++j) old[j] = 0.0f;
    if (a.add && c < a.C) load_piece<N>(row, c, a.C, old);
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = a.add ? old[j] + a.scale * acc[j] : a.scale * acc[j];
    store_piece<N>(row, c, a.C, acc);
}

template <typename T>
__global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a) {
    constexpr int N = kVec<T>;
    const int lane = threadIdx.x & 63;
    const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (unit >= a.segs * a.slabs) return;
    const int64_t seg = unit / a.slabs, p0 = seg * kSeg;
    const int c = (int(unit - seg * a.slabs) * 64 + lane) * N;
    const int64_t p = p0 + lane;
    const uint32_t key = p < a.n ? a.keys[p] : a.V, row = p < a.n ? a.rows[p] : 0;
    const uint32_t prev = p0 > 0 ? a.keys[p0 - 1] : kNone, next = p0 + kSeg < a.n ? a.keys[p0 + kSeg] : kNone;
    const int n = __popcll(__ballot(key < a.V));   // sorted: rows without a token come last
    if (n == 0) return;
    const uint32_t left = __shfl_up(key, 1, 64);
    const uint64_t heads = __ballot(key != (lane ? left : prev));   // a run begins
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.0f;
    for (int i0 = 0; i0 < n; i0 += kAhead) {
        float x[kAhead][N];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u < n ? i0 + u : n - 1;
            const uint32_t r = __builtin_amdgcn_readlane(row, i);
            load_piece<N>(static_cast<const T*>(a.dy) + int64_t(r) * a.C, c, a.C, x[u]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u;
            if (i >= n) break;
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] += x[u][j];
            const uint32_t v = __builtin_amdgcn_readlane(key, i);
            const bool last = i + 1 == n ? !(n == kSeg && next == v) : (heads >> (i + 1)) & 1;
            if (!last && i + 1 < n) continue;
            const bool begun = heads & (~uint64_t(0) >> (63 - i));   // in this segment
            if (begun && last) finish<N>(a, v, c, acc);
            else store_piece<N>((begun ? a.tail : a.head) + seg * a.C, c, a.C, acc);
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        }
    }
}

// A run that begins in segment `seg` and goes on: its tail there, then the heads of the segments behind it.
__global__ __launch_bounds__(256) void embed_join_kernel(SumArgs a) {
    constexpr int N = 4;
    const int lane = threadIdx.x & 63;
    const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (unit >= a.segs * a.slabs) return;
    const int64_t seg = unit / a.slabs, p0 = seg * kSeg, end = p0 + kSeg;
    if (end >= a.n) return;
    const uint32_t v = a.keys[end - 1];
    if (v >= a.V || a.keys[end] != v) return;
    if (p0 > 0 && a.keys[p0 - 1] == v) return;   // it began before
    const int c = (int(unit - seg * a.slabs) * 64 + lane) * N;
    float acc[N];
    load_piece<N>(a.tail + seg * a.C, c, a.C, acc);
    for (int64_t s = seg + 1;; s += 64) {
        // Segments s .. s + 63 that this run reaches: it holds their first row.
        const int64_t first = (s + lane) * kSeg;
        const uint64_t in = __ballot(first < a.n && a.keys[first < a.n ? first : 0] == v);
        const int count = in == ~uint64_t(0) ? 64 : __builtin_ctzll(~in);
#pragma unroll 8
        for (int i = 0; i < count; ++i) {
            float x[N];
            load_piece<N>(a.head + (s + i) * a.C, c, a.C, x);
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] += x[j];
        }
        if (count < 64) break;
    }
    finish<N>(a, v, c, acc);
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

// What the gradient's launches need of a configuration.
struct Plan {
    int passes, bits, blocks;
    int64_t per, segs;
    int64_t lists, hist, parts;   // bytes of the workspace's areas
    int64_t bytes() const { return lists + hist + parts; }
};
int64_t round16(int64_t n) { return (n + 15) & ~int64_t(15); }
Plan plan_of(const dgm_rows_cfg* c) {
    Plan p;
    int width = 1;
    while ((int64_t(1) << width) <= c->V) ++width;   // keys 0 .. V
    p.passes = (width + kMaxBits - 1) / kMaxBits;
    p.bits = (width + p.passes - 1) / p.passes;
    const int64_t tiles = (c->rows + kTile - 1) / kTile, each = (tiles + kMaxBlocks - 1) / kMaxBlocks;
    p.per = each * kTile;
    p.blocks = int(each ? (tiles + each - 1) / each : 0);
    p.segs = (c->rows + kSeg - 1) / kSeg;
    p.lists = 4 * round16(c->rows * 4);
    p.hist = round16(int64_t(p.blocks) * (4 << p.bits));
    p.parts = 2 * round16(p.segs * c->C * 4);
    return p;
}

// Waves of `count` units of work fit one launch's bound on threads.
bool fits(int64_t units) { return units <= int64_t(UINT32_MAX) / 64 - 4; }

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
    while (team < 256 && int64_t(team) * n < cfg->C) team *= 2;
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
    return plan_of(cfg).bytes();
}

int dgm_embedRowsBwd(dgm_gpu* g, const dgm_rows_cfg* cfg, const uint32_t* tokens, const void* dy, float* dtable,
                     int accumulate, void* ws, int64_t ws_bytes) {
    int rc = dgm::enter(g, "embed_rows_bwd");
    if (rc) return rc;
    rc = check(g, "embedRowsBwd", cfg);
    if (rc) return rc;
    if (!dtable || (cfg->rows > 0 && (!tokens || !dy || !ws))) return dgm::fail(g, DGM_ERR_ARG, "embedRowsBwd: null buffer");
    const Plan p = plan_of(cfg);
    if (ws_bytes < p.bytes())
        return dgm::fail(g, DGM_ERR_ARG, "embedRowsBwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)p.bytes());
    if (!dgm::aligned(tokens, 4) || !dgm::aligned(dy, size_t(type_bytes(cfg->type))) || !dgm::aligned(dtable, 4) || !dgm::aligned(ws, 16))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "embedRowsBwd: a buffer is not aligned to its elements, or the workspace to 16 bytes");
    const int n = 16 / type_bytes(cfg->type);
    const int64_t slabs = (cfg->C + 64 * n - 1) / (64 * n), join = (cfg->C + 255) / 256;
    if (!fits(p.segs * slabs) || !fits(p.segs * join))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "embedRowsBwd: %lld rows of %lld exceed one launch", (long long)cfg->rows, (long long)cfg->C);
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "embedRowsBwd: %s", hipGetErrorString(on.err));
    uint8_t* at = static_cast<uint8_t*>(ws);
    uint32_t* lists[4];
    for (auto& l : lists) {
        l = reinterpret_cast<uint32_t*>(at);
        at += p.lists / 4;
    }
    SortArgs s{tokens, nullptr, nullptr, nullptr, nullptr, reinterpret_cast<uint32_t*>(at), g->seq_report, cfg->rows, p.per,
               uint32_t(cfg->V), 0, p.bits, p.blocks, accumulate ? nullptr : dtable, accumulate ? 0 : cfg->V * cfg->C};
    at += p.hist;
    const unsigned clearing = unsigned(std::min<int64_t>((s.zero_n + 16 * kSortThreads - 1) / (16 * kSortThreads), 2048));
    if (p.blocks + clearing == 0) return DGM_OK;
    embed_hist_kernel<true><<<dim3(unsigned(p.blocks) + clearing), dim3(kSortThreads), 0, g->stream>>>(s);
    DGM_LAUNCH_CHECK(g, "embed_hist");
    if (p.blocks == 0) return DGM_OK;
    for (int i = 0; i < p.passes; ++i) {
        s.shift = i * p.bits;
        s.keys_out = lists[2 * (i & 1)];
        s.rows_out = lists[2 * (i & 1) + 1];
        const dim3 grid{unsigned(p.blocks)}, block{kSortThreads};
        if (i) embed_hist_kernel<false><<<grid, block, 0, g->stream>>>(s);
        if (i) embed_place_kernel<false><<<grid, block, 0, g->stream>>>(s);
        else embed_place_kernel<true><<<grid, block, 0, g->stream>>>(s);
        DGM_LAUNCH_CHECK(g, "embed_place");
        s.keys = s.keys_out;
        s.rows = s.rows_out;
    }
    float* parts = reinterpret_cast<float*>(at);
    SumArgs a{dy, s.keys, s.rows, dtable, parts, parts + p.parts / 8, cfg->rows, uint32_t(cfg->V), int(cfg->C), int(slabs),
              accumulate ? 1 : 0, p.segs, cfg->scale};
    const dim3 grid(dgm::ceil_div(p.segs * slabs, 4));
    if (cfg->type == DGM_TYPE_F32) embed_sum_kernel<float><<<grid, dim3(256), 0, g->stream>>>(a);
    else embed_sum_kernel<__bf16><<<grid, dim3(256), 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "embed_sum");
    if (p.segs > 1) {
        a.slabs = int(join);
        embed_join_kernel<<<dim3(dgm::ceil_div(p.segs * join, 4)), dim3(256), 0, g->stream>>>(a);
        DGM_LAUNCH_CHECK(g, "embed_join");
    }
    return DGM_OK;
}

}  // extern "C"
