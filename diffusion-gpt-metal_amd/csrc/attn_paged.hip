// A paged cache of keys and values, and the attention of one new token per
// sequence over it (gfx950). HBM-bound: a cached element is used once per query head of its group.
//
// Decode design:
//  * Work is cut over the sequences' lengths as the device finds them: all
//    tiles (128 keys of a bf16 cache, 64 of an fp32 one) of all sequences lie in a row, and
//    each of W workgroups per key head takes an equal run of them, so that 48
//    ragged sequences keep the chip as busy as one long one. A run ends in at most a few sequences;
//    worker w's part of sequence s is slot w + s of the partial results (w and s only
//    grow along the row of tiles, so slots never collide). A sequence inside one
//    run is written out by its worker; the others are joined by a second kernel.
//  * No LDS on the way from HBM to the matrix unit. S^T = K Q^T takes K as it
//    lies in the cache (16 keys x 8 columns of 16 bytes a lane), with the heads of
//    the group as columns; P^T then is in the layout of the B operand of
//    O^T = V^T P^T, whose A operand a lane builds from 8 keys' rows by byte
//    permutes among its own registers. A wave takes 32 keys (16 of an fp32
//    cache) at a time, and asks for those of the next round as soon as the product
//    that took this round's registers is issued: two waves to a SIMD then keep up to 128 KB
//    a CU under way. 48 sequences, 708 MB: 133 us, 5.3 TB/s (with two sets of
//    registers, which spill, 182; with three waves, which spill more, 235).
//  * A bf16 cache meets fp32 queries as three bf16 pieces (8 bits each: all 24),
//    and so do the probabilities, with fp32 sums: nothing of fp32 is lost. bf16
//    queries take one piece each, P rounded to bf16. An fp32 cache runs on fp32 MFMA.
//  * Slots behind a sequence's end, and of pages that are not the cache's, are
//    not read: they count as zero keys with a weight of zero.
#include <algorithm>
#include <climits>
#include <cmath>

#include "attn.hpp"

namespace {

using namespace dgm_attn;

struct Cache {
    const int32_t* pages;
    uint32_t* words;   // the report
    int64_t numPages, maxPages;
    int KVH, D, capacity;   // positions that a sequence's row of the table holds
    Div page;
    // As cache_row; pos below capacity.
    __device__ __forceinline__ int row(int64_t s, uint32_t pos, int h) const {
        return cache_row(pages, page, numPages, maxPages, KVH, s, pos, h);
    }
};

// ---- write ---------------------------------------------------------------------

struct WriteArgs {
    Cache c;
    const void *k, *v;
    void *kc, *vc;
    const int32_t *starts, *lens;
    int64_t rows, nseq, ldk, ldv;
    Div per_row;   // threads of a row
};

template <typename IN, typename CT>
__device__ __forceinline__ void convert8(const IN* from, CT* to) {
    if constexpr (sizeof(IN) == 2 && sizeof(CT) == 2) {
        *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(from);
    } else if constexpr (sizeof(IN) == 4 && sizeof(CT) == 4) {
        const u32x4 a = reinterpret_cast<const u32x4*>(from)[0], b = reinterpret_cast<const u32x4*>(from)[1];
        reinterpret_cast<u32x4*>(to)[0] = a;
        reinterpret_cast<u32x4*>(to)[1] = b;
    } else if constexpr (sizeof(IN) == 4) {
        const f32x4 a = reinterpret_cast<const f32x4*>(from)[0], b = reinterpret_cast<const f32x4*>(from)[1];
        bf16x8 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] = __bf16(a[i]);
            o[4 + i] = __bf16(b[i]);
        }
        *reinterpret_cast<bf16x8*>(to) = o;
    } else {
        const u32x4 a = *reinterpret_cast<const u32x4*>(from);
        u32x4 lo, hi;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lo[2 * i] = a[i] << 16;
            lo[2 * i + 1] = a[i] & 0xffff0000u;
            hi[2 * i] = a[2 + i] << 16;
            hi[2 * i + 1] = a[2 + i] & 0xffff0000u;
        }
        reinterpret_cast<u32x4*>(to)[0] = lo;
        reinterpret_cast<u32x4*>(to)[1] = hi;
    }
}

// A thread moves 8 elements of k and of v of one (row, head). The sequence of the
// workgroup's first row is looked up by whole waves, 64 candidates a round; a thread's own row
// lies in that or a later one, and the ones between are looked at one by one. A write of few rows is a chain of waits: starts,
// lengths, pages, rows (48 rows: 3.5 us); of many, HBM-bound (8 heads of 128, 8162 rows, fp32 to a bf16
// cache, 100 MB: 19 us, 5.3 TB/s).
template <typename IN, typename CT>
__global__ void __launch_bounds__(256) cache_write_kernel(WriteArgs a) {
    const int per_head = a.c.D / 8, per_row = a.c.KVH * per_head;
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    // 32 bits where they hold all of it: a 64-bit division is a call's worth of instructions.
    const int64_t row = a.rows <= INT_MAX / per_row ? int64_t(a.per_row(uint32_t(i))) : i / per_row;
    const int64_t row0 = a.rows <= INT_MAX / per_row ? int64_t(a.per_row(blockIdx.x * 256u)) : int64_t(blockIdx.x) * 256 / per_row;
    int64_t s = row, first = row;
    if (a.starts) {   // the last sequence that starts at or before the row
        const int lane = threadIdx.x & 63;
        int64_t lo = 0, n = a.nseq;
        while (n > 1) {
            const int64_t step = (n + 63) / 64;
            const int c = __popcll(__ballot(lane * step < n && a.starts[lo + lane * step] <= row0));
            const int64_t skip = (c > 0 ? c - 1 : 0) * step;
            lo += skip;
            n = n - skip < step ? n - skip : step;
        }
        if (blockIdx.x == gridDim.x - 1) check_starts(a.starts, a.nseq, a.rows, a.c.words);
        if (row >= a.rows) return;
        first = a.starts[lo];
        int64_t next = a.starts[lo + 1];
        while (next <= row) {
            if (++lo == a.nseq) return;
            first = next;
            next = a.starts[lo + 1];
        }
        if (first > row) return;
        s = lo;
    } else if (row >= a.rows) {
        return;
    }
    const int e = int(i - row * per_row), head = e / per_head, d = e % per_head * 8;
    const int64_t pos = (a.lens ? int64_t(a.lens[s]) : 0) + (row - first);
    const int at = pos >= 0 && pos < a.c.capacity ? a.c.row(s, uint32_t(pos), head) : -1;
    if (at < 0) {
        if (e == 0) report(a.c.words, kBadPages);
        return;
    }
    const int64_t to = int64_t(at) * a.c.D + d;
    convert8(static_cast<const IN*>(a.k) + row * a.ldk + int64_t(head) * a.c.D + d, static_cast<CT*>(a.kc) + to);
    convert8(static_cast<const IN*>(a.v) + row * a.ldv + int64_t(head) * a.c.D + d, static_cast<CT*>(a.vc) + to);
}

// ---- decode --------------------------------------------------------------------

constexpr int kHeads = 16;      // query heads of a workgroup: the columns of an MFMA tile
constexpr int kWorkers = 512;   // workgroups that share the tiles, over all key heads

template <typename CT>
constexpr int kWaveKeys = sizeof(CT) == 2 ? 32 : 16;
template <typename CT>
constexpr int kTileKeys = 4 * kWaveKeys<CT>;   // four waves

struct DecodeArgs {
    Cache c;
    const void *q, *kc, *vc;
    void* out;
    float* part;   // [units][workers + nseq][heads][D]; behind them m and l, [..][heads][2]
    float* stat;
    const int32_t* lens;
    int64_t nseq, ldq, ldo;
    int H, G, heads, parts, workers, units;   // heads of a unit; units of a key head
    float scale2;                             // scale * log2 e
    Div share;                                // by workers
};

__device__ __forceinline__ int length_of(const DecodeArgs& a, int64_t s) {
    const int n = a.lens[s];
    return n < 0 ? 0 : n > a.c.capacity ? a.c.capacity : n;
}

// Inclusive sum over a wave's lanes, by DPP: rows of 16, then across them.
__device__ __forceinline__ int scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}

// What a head's sums come to, its largest score M.
__device__ __forceinline__ float quotient(float x, float sum, float M) {
    return sum == 0.0f ? 0.0f : M == kNegInf ? __builtin_nanf("") : x / sum;
}

// A wave's view of a run of 64 sequences, one a lane: length, tiles, and tiles up to and with this one.
template <int KEYS>
struct Run {
    int64_t first;
    int len, tiles, upto;
    __device__ __forceinline__ void load(const DecodeArgs& a, int64_t s0, int before) {
        const int64_t s = s0 + (threadIdx.x & 63);
        first = s0;
        len = s < a.nseq ? length_of(a, s) : 0;
        tiles = (len + KEYS - 1) / KEYS;
        upto = before + scan(tiles);
    }
    __device__ __forceinline__ int last() const { return __builtin_amdgcn_readlane(upto, 63); }
};

// All tiles of all sequences; `run` is left on the first 64.
template <int KEYS>
__device__ __forceinline__ int total_tiles(const DecodeArgs& a, Run<KEYS>& run) {
    run.load(a, 0, 0);
    int total = run.last();
    for (int64_t s0 = 64; s0 < a.nseq; s0 += 64) {
        Run<KEYS> r;
        r.load(a, s0, total);
        total = r.last();
    }
    return total;
}

// VW consecutive elements of a value row in registers.
template <int BYTES>
struct Piece {
    uint32_t w[BYTES / 4];
};
template <int BYTES>
__device__ __forceinline__ Piece<BYTES> load_piece(const void* p, int bytes) {   // those up to `bytes`
    Piece<BYTES> o{};
    if (bytes > 0) {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                if (i * 16 >= bytes) continue;
                const u32x4 v = static_cast<const u32x4*>(p)[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) o.w[4 * i + j] = v[j];
            }
        } else if constexpr (BYTES == 8) {
            const u32x2 v = *static_cast<const u32x2*>(p);
            o.w[0] = v[0];
            o.w[1] = v[1];
        } else {
            o.w[0] = *static_cast<const uint32_t*>(p);
        }
    }
    return o;
}

// One wave's 32 (16) keys on their way.
template <typename CT, int DP>
struct Round {
    static constexpr int EB = sizeof(CT), KEYS = kWaveKeys<CT>, NB = KEYS / 16;   // blocks of 16 keys
    static constexpr int KC = DP * EB / 64;                          // 16-byte chunks of a key to a lane
    static constexpr int VW = DP / 16, VB = VW * EB;                 // elements and bytes of a value row to a lane
    u32x4 k[NB][KC];
    Piece<VB> v[4 * NB];

    // Rows of key lane % KEYS (-1: none) for the lane's part of the keys, and of the values.
    __device__ __forceinline__ void load_k(const Cache& c, const uint8_t* kc, int row) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const int rb = c.D * EB;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int at = __shfl(row, 16 * b + (lane & 15), 64);
            const uint8_t* p = kc + int64_t(at) * rb + g * 16;
#pragma unroll
            for (int kk = 0; kk < KC; ++kk) {
                k[b][kk] = u32x4{0, 0, 0, 0};
                if (at >= 0 && kk * 64 + g * 16 < rb) k[b][kk] = *reinterpret_cast<const u32x4*>(p + kk * 64);
            }
        }
    }
    __device__ __forceinline__ void load_v(const Cache& c, const uint8_t* vc, int row) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
        const int rb = c.D * EB;
#pragma unroll
        for (int j = 0; j < 4 * NB; ++j) {   // key 16 (j / 4) + 4 g + j % 4
            const int at = __shfl(row, 16 * (j / 4) + 4 * g + j % 4, 64);
            v[j] = load_piece<VB>(vc + int64_t(at) * rb + r * VB, at >= 0 ? rb - r * VB : 0);
        }
    }
};

// The queries of a unit as B operand, columns = heads, in LDS: 16 bytes a lane, chunk and piece.
template <typename IN, typename CT, int DP>
struct Queries {
    static constexpr int PIECES = sizeof(IN) == 4 && sizeof(CT) == 2 ? 3 : 1;
    static constexpr int KC = DP * int(sizeof(CT)) / 64;
    u32x4 f[PIECES][KC][64];
    // Chunk kk by the wave kk % 4; q: of the lane's head.
    __device__ __forceinline__ void load(const IN* q, int D, bool in) {
        const int lane = threadIdx.x & 63, g = lane >> 4, wave = threadIdx.x >> 6;
        for (int kk = wave; kk < KC; kk += 4) {
            if constexpr (sizeof(CT) == 2) {
                const int d = 32 * kk + 8 * g;
                float x[8] = {};
                if (in && d < D) load8(q + d, x);
                bf16x8 o[PIECES];
                split8<PIECES, kSelect>(x, o);
#pragma unroll
                for (int p = 0; p < PIECES; ++p) f[p][kk][lane] = __builtin_bit_cast(u32x4, o[p]);
            } else {
                const int d = 16 * kk + 4 * g;
                f32x4 x = {};
                if (in && d < D) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = float(q[d + i]);
                }
                f[0][kk][lane] = __builtin_bit_cast(u32x4, x);
            }
        }
    }
};

template <typename IN, typename CT, int DP>
__global__ void __launch_bounds__(256, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) attn_paged_decode_kernel(DecodeArgs a) {
    using R = Round<CT, DP>;
    using Q = Queries<IN, CT, DP>;
    constexpr int KEYS = kTileKeys<CT>, WK = kWaveKeys<CT>, NB = R::NB, VW = R::VW;
    __shared__ Q q;
    __shared__ float part[4][kHeads][DP];
    __shared__ float stat[4][kHeads][2];
    const int unit = blockIdx.x % a.units, worker = blockIdx.x / a.units;
    const int kvh = unit / a.parts, h0 = kvh * a.G + unit % a.parts * kHeads;   // first query head
    const int heads = min(kHeads, a.G - unit % a.parts * kHeads);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    Run<KEYS> run;
    const int total = total_tiles(a, run), per = int(a.share(uint32_t(total + a.workers - 1)));
    int at = worker * per;
    const int end = min(at + per, total);
    if (worker == a.workers - 1)
        // Sequences without keys have no tile: their rows are zeros. Lengths beyond the table are reported.
        for (int64_t s0 = 0; s0 < a.nseq; s0 += 64) {
            const bool there = s0 + lane < a.nseq;
            if (there && a.lens[s0 + lane] > a.c.capacity) report(a.c.words, kBadPages);
            unsigned long long none = __ballot(there && length_of(a, s0 + lane) == 0);
            for (; none; none &= none - 1)
                for (int e = threadIdx.x; e < heads * a.c.D; e += 256)
                    static_cast<IN*>(a.out)[(s0 + __ffsll(none) - 1) * a.ldo + int64_t(h0) * a.c.D + e] = IN(0.0f);
        }
    if (at >= end) return;
    // The sequence of the first tile, its length and its own first tile.
    unsigned long long past = __ballot(run.upto > at);
    while (!past) {
        run.load(a, run.first + 64, run.last());
        past = __ballot(run.upto > at);
    }
    const int first = __ffsll(past) - 1;
    int64_t s = run.first + first;
    int len = __builtin_amdgcn_readlane(run.len, first);
    int base = __builtin_amdgcn_readlane(run.upto - run.tiles, first);
    const uint8_t* kc = static_cast<const uint8_t*>(a.kc);
    const uint8_t* vc = static_cast<const uint8_t*>(a.vc);
    while (true) {
        const int tiles = (len + KEYS - 1) / KEYS;
        const int t0 = at - base, t1 = min(tiles, end - base);
        // The page of this lane's key (lane % WK) in tile t, read ahead; its row, -1 for none.
        const int64_t table = s * a.c.maxPages;
        const auto page_of = [&](int t) {
            const int key = t * KEYS + wave * WK + (lane & (WK - 1));
            return t < t1 && key < len ? a.c.pages[table + a.c.page(uint32_t(key))] : -1;
        };
        const auto row_of = [&](int t, int id) {
            const int key = t * KEYS + wave * WK + (lane & (WK - 1));
            if (t >= t1 || key >= len) return -1;
            if (id < 0 || id >= a.c.numPages) {
                report(a.c.words, kBadPages);
                return -1;
            }
            const int page = int(a.c.page.d);
            return (id * a.c.KVH + kvh) * page + key - int(a.c.page(uint32_t(key))) * page;
        };
        int id1 = page_of(t0), id2 = page_of(t0 + 1);
        q.load(static_cast<const IN*>(a.q) + s * a.ldq + int64_t(h0 + col) * a.c.D, a.c.D, col < heads);
        f32x4 o[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) o[i] = f32x4{0, 0, 0, 0};
        float m = kNegInf, l = 0.0f;
        bool seen = false;   // a key
        R now;
        int row = row_of(t0, id1);
        now.load_k(a.c, kc, row);
        now.load_v(a.c, vc, row);
        __syncthreads();   // the queries are there
        for (int t = t0; t < t1; ++t) {
            id1 = id2;
            id2 = page_of(t + 2);
            // Bit i: key i of the wave's is there.
            const uint32_t there = uint32_t(__ballot(row >= 0)) & uint32_t((uint64_t(1) << WK) - 1);
            seen = seen || there;
            f32x4 sc[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) sc[b] = f32x4{0, 0, 0, 0};
            // fp32: four sums, each a quarter as long (heads of 256 over 5000 keys were off by twice what the plain sums are).
            f32x4 quarter[4] = {};
#pragma unroll
            for (int kk = 0; kk < Q::KC; ++kk)
#pragma unroll
                for (int p = Q::PIECES - 1; p >= 0; --p) {
                    const u32x4 y = q.f[p][kk][lane];
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        if constexpr (sizeof(CT) == 2) {
                            sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, now.k[b][kk]),
                                                                            __builtin_bit_cast(bf16x8, y), sc[b], 0, 0, 0);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                quarter[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(now.k[b][kk][i]),
                                                                                  __uint_as_float(y[i]), quarter[i], 0, 0, 0);
                        }
                    }
                }
            if constexpr (sizeof(CT) == 4) sc[0] = (quarter[0] + quarter[1]) + (quarter[2] + quarter[3]);
            // The keys' registers are free for those of the next round.
            row = row_of(t + 1, id1);
            if (t + 1 < t1) now.load_k(a.c, kc, row);
            if (there != uint32_t((uint64_t(1) << WK) - 1)) {
                const uint32_t mine = there >> (4 * g);
#pragma unroll
                for (int j = 0; j < 4 * NB; ++j)
                    sc[j / 4][j % 4] = mine >> (16 * (j / 4) + j % 4) & 1 ? sc[j / 4][j % 4] : kNegInf;
            }
            float mx = kNegInf;
#pragma unroll
            for (int j = 0; j < 4 * NB; ++j) mx = fmaxf(mx, sc[j / 4][j % 4]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (__any((mx - m) * a.scale2 > 8.0f)) {
                const float to = fmaxf(m, mx), f = m == kNegInf ? 0.0f : exp2_hw((m - to) * a.scale2);
                l *= f;
#pragma unroll
                for (int i = 0; i < VW; ++i) o[i] *= f;
                m = to;
            }
            const float mc = m == kNegInf ? 0.0f : m * a.scale2;
            float p[4 * NB];
#pragma unroll
            for (int j = 0; j < 4 * NB; ++j) {
                p[j] = exp2_hw(__builtin_fmaf(sc[j / 4][j % 4], a.scale2, -mc));
                l += p[j];
            }
            if constexpr (sizeof(CT) == 2) {
                bf16x8 w[Q::PIECES];
                split8<Q::PIECES, kSpoils>(p, w);
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
                    u32x4 x;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[j] = __builtin_amdgcn_perm(now.v[2 * j + 1].w[i / 2], now.v[2 * j].w[i / 2], sel);
#pragma unroll
                    for (int n = Q::PIECES - 1; n >= 0; --n)
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), w[n], o[i], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < VW; ++i)
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(now.v[j].w[i]), p[j], o[i], 0, 0, 0);
            }
            if (t + 1 < t1) now.load_v(a.c, vc, row);
        }
        // The four waves' parts, joined: o[i][r] is column (4 g + r) VW + i of head `col`.
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        // Keys whose scores are all -inf: no softmax, and not the zeros of no keys. Beside
        // any other score the factor of this sum is 0.
        if (seen && m == kNegInf && l == 0.0f) l = 1.0f;
        if (g == 0) {
            stat[wave][col][0] = m;
            stat[wave][col][1] = l;
        }
#pragma unroll
        for (int i = 0; i < VW; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[wave][col][(4 * g + r) * VW + i] = o[i][r];
        __syncthreads();
        const bool whole = t0 == 0 && t1 == tiles;
        const int64_t slot = int64_t(unit) * (a.workers + a.nseq) + worker + s;
        for (int e = threadIdx.x; e < heads * DP; e += 256) {
            const int hd = e / DP, d = e % DP;
            float M = kNegInf;
#pragma unroll
            for (int w = 0; w < 4; ++w) M = fmaxf(M, stat[w][hd][0]);
            float sum = 0.0f, x = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {   // a wave without keys has m = -inf, l = 0 and zeros
                const float f = stat[w][hd][0] == M ? 1.0f : exp2_hw((stat[w][hd][0] - M) * a.scale2);
                sum = __builtin_fmaf(stat[w][hd][1], f, sum);
                x = __builtin_fmaf(part[w][hd][d], f, x);
            }
            if (d >= a.c.D) continue;
            if (whole) {
                static_cast<IN*>(a.out)[s * a.ldo + int64_t(h0 + hd) * a.c.D + d] = IN(quotient(x, sum, M));
            } else {
                a.part[(slot * a.heads + hd) * a.c.D + d] = x;
                if (d == 0) {
                    a.stat[(slot * a.heads + hd) * 2] = M;
                    a.stat[(slot * a.heads + hd) * 2 + 1] = sum;
                }
            }
        }
        at = base + t1;
        if (at >= end) break;
        __syncthreads();
        base += tiles;
        do len = length_of(a, ++s);
        while (len == 0);
    }
}

// Joins the parts of the sequences that several workers share: one workgroup a
// (sequence, query head), columns over its threads, parts over the groups of threads that are
// left. A thread asks for its first parts before it knows their factors: the
// kernel is a chain of waits (lengths, maxima and sums, parts) and little else.
// Every workgroup goes through all lengths, 64 at a time, so that the call's time grows with the square of the
// sequences where these are many: 64 keys each, 8 heads on 2 of 64, take 13 us for 256 sequences, 59 for 1024, 517 for 4096
// and 6.7 ms for 16384.
template <typename IN, int KEYS>
__global__ void __launch_bounds__(1024) attn_paged_join_kernel(DecodeArgs a) {
    constexpr int AHEAD = 8;
    __shared__ float factor[kWorkers], sums[1024];
    const int64_t s = blockIdx.x / a.H;
    const int head = blockIdx.x % a.H, kvh = head / a.G, of = head % a.G;
    const int unit = kvh * a.parts + of / kHeads, hd = of % kHeads, lane = threadIdx.x & 63;
    Run<KEYS> run;
    const int total = total_tiles(a, run), per = int(a.share(uint32_t(total + a.workers - 1)));
    while (s >= run.first + 64) run.load(a, run.first + 64, run.last());
    const int tiles = __builtin_amdgcn_readlane(run.tiles, int(s - run.first));
    const int base = __builtin_amdgcn_readlane(run.upto, int(s - run.first)) - tiles;
    if (tiles == 0) return;
    const int w0 = base / per, parts = (base + tiles - 1) / per - w0 + 1;   // at most kWorkers
    if (parts == 1) return;
    const int64_t row0 = (int64_t(unit) * (a.workers + a.nseq) + w0 + s) * a.heads + hd;   // of the first part; heads apart
    const int cols = a.c.D <= 32 ? 32 : a.c.D <= 64 ? 64 : a.c.D <= 128 ? 128 : 256, groups = int(blockDim.x) / cols;
    const int d = threadIdx.x % cols, group = threadIdx.x / cols;
    const float* part = a.part + row0 * a.c.D + d;
    const int64_t step = int64_t(a.heads) * a.c.D;
    float held[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        const int w = group + i * groups;
        held[i] = w < parts && d < a.c.D ? part[w * step] : 0.0f;
    }
    // Every wave: the largest maximum, the parts' factors and their sum.
    const float2* st = reinterpret_cast<const float2*>(a.stat) + row0;
    const float2 mine = lane < parts ? st[int64_t(lane) * a.heads] : float2{kNegInf, 0.0f};
    float M = mine.x;
    for (int w = lane + 64; w < parts; w += 64) M = fmaxf(M, st[int64_t(w) * a.heads].x);
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
    float sum = 0.0f;
    for (int w = lane; w < parts; w += 64) {
        const float2 v = w < 64 ? mine : st[int64_t(w) * a.heads];
        const float f = v.x == M ? 1.0f : exp2_hw((v.x - M) * a.scale2);
        if (threadIdx.x < 64) factor[w] = f;
        sum = __builtin_fmaf(v.y, f, sum);
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x, 64);
    __syncthreads();
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        const int w = group + i * groups;
        if (w < parts) x = __builtin_fmaf(held[i], factor[w], x);
    }
    if (d < a.c.D)
#pragma unroll 8
        for (int w = group + AHEAD * groups; w < parts; w += groups) x = __builtin_fmaf(part[w * step], factor[w], x);
    sums[threadIdx.x] = x;
    __syncthreads();
    if (group > 0 || d >= a.c.D) return;
    for (int i = 1; i < groups; ++i) x += sums[i * cols + d];
    static_cast<IN*>(a.out)[s * a.ldo + int64_t(head) * a.c.D + d] = IN(quotient(x, sum, M));
}

// ---- host ----------------------------------------------------------------------

// Positions that a sequence's row of the table holds; tiles past the end keep within 32 bits.
int64_t capacity_of(const dgm_cache_cfg* c) {
    return std::min<int64_t>(c->maxPages * c->pageSize, INT_MAX - 1024);
}

int check_cache(dgm_gpu* g, const char* name, const dgm_cache_cfg* c, int64_t type, int64_t nseq) {
    if (!c) return dgm::fail(g, DGM_ERR_ARG, "%s: null configuration", name);
    if (!type_bytes(c->type) || !type_bytes(type))
        return dgm::fail(g, DGM_ERR_ARG, "%s: unknown type %d or %lld", name, c->type, (long long)type);
    if (nseq < 0 || c->KVH < 1 || c->D < 1 || c->pageSize < 1 || c->numPages < 0 || c->maxPages < 0)
        return dgm::fail(g, DGM_ERR_ARG, "%s: bad sizes", name);
    if (c->D % 8 != 0 || c->D > 256)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: head dim %d is not a multiple of 8 up to 256", name, c->D);
    if (c->numPages > INT_MAX || c->maxPages > INT_MAX || nseq > 65536 ||
        c->numPages > INT_MAX / (int64_t(c->KVH) * c->pageSize) ||
        nseq * ((capacity_of(c) + 63) / 64) > INT_MAX - kWorkers)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: more than 2^31 cache rows or table positions, or too many sequences",
                         name);
    return DGM_OK;
}

// A workgroup of up to 1024 threads for each, in hipLaunchKernel's bound on a grid's threads.
bool heads_fit(int64_t nseq, int64_t H) { return H <= 65536 && nseq * H <= int64_t(UINT32_MAX) / 1024; }

Cache cache_of(dgm_gpu* g, const dgm_cache_cfg* c, const int32_t* pages) {
    return Cache{pages, g->seq_report, c->numPages, c->maxPages, c->KVH, c->D, int(capacity_of(c)),
                 Div(uint32_t(c->pageSize))};
}

// Workgroups of a key head's unit that share the tiles, and units of a key head.
struct Split {
    int parts, units, workers, heads;
};
Split split_of(const dgm_cache_cfg* c, int64_t H) {
    const int G = int(H / c->KVH), parts = (G + kHeads - 1) / kHeads, units = c->KVH * parts;
    return {parts, units, units < kWorkers ? kWorkers / units : 1, G < kHeads ? G : kHeads};
}
int64_t part_floats(const dgm_cache_cfg* c, int64_t nseq, int64_t H) {
    const Split s = split_of(c, H);
    return int64_t(s.units) * (s.workers + nseq) * s.heads;
}
int64_t decode_ws_bytes(const dgm_cache_cfg* c, int64_t nseq, int64_t H) {
    return part_floats(c, nseq, H) * (c->D + 2) * int64_t(sizeof(float));
}

template <typename IN, typename CT>
int run_decode(dgm_gpu* g, const DecodeArgs& a) {
    const dim3 grid(unsigned(a.units) * unsigned(a.workers)), block(256);
    if (a.c.D <= 32) attn_paged_decode_kernel<IN, CT, 32><<<grid, block, 0, g->stream>>>(a);
    else if (a.c.D <= 64) attn_paged_decode_kernel<IN, CT, 64><<<grid, block, 0, g->stream>>>(a);
    else if (a.c.D <= 128) attn_paged_decode_kernel<IN, CT, 128><<<grid, block, 0, g->stream>>>(a);
    else attn_paged_decode_kernel<IN, CT, 256><<<grid, block, 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "attn_paged_decode");
    // Few sequences have many parts each: 1024 threads ask for more of them at once.
    const dim3 join(a.workers / a.nseq >= 32 ? 1024 : 256);
    attn_paged_join_kernel<IN, kTileKeys<CT>><<<dim3(unsigned(a.nseq * a.H)), join, 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "attn_paged_join");
    return DGM_OK;
}

template <typename IN, typename CT>
int run_write(dgm_gpu* g, const WriteArgs& a) {
    const int64_t blocks = (a.rows * (a.c.KVH * a.c.D / 8) + 255) / 256;
    if (blocks * 256 > int64_t(UINT32_MAX))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "cacheWrite: %lld rows exceed one launch", (long long)a.rows);
    cache_write_kernel<IN, CT><<<dim3(unsigned(blocks)), dim3(256), 0, g->stream>>>(a);
    DGM_LAUNCH_CHECK(g, "cache_write");
    return DGM_OK;
}

}  // namespace

extern "C" {

int dgm_cacheWrite(dgm_gpu* g, const dgm_cache_cfg* cfg, int64_t type, const void* k, const void* v,
                   const int32_t* starts, const int32_t* lens, const int32_t* pages, void* kcache, void* vcache,
                   int64_t rows, int64_t nseq, int64_t ldk, int64_t ldv) {
    int rc = dgm::enter(g, "cache_write");
    if (rc) return rc;
    rc = check_cache(g, "cacheWrite", cfg, type, nseq);
    if (rc) return rc;
    if (rows < 0) return dgm::fail(g, DGM_ERR_ARG, "cacheWrite: rows=%lld", (long long)rows);
    if (!starts && rows != nseq)
        return dgm::fail(g, DGM_ERR_SHAPE, "cacheWrite: %lld rows of %lld sequences without starts", (long long)rows,
                         (long long)nseq);
    const int64_t width = int64_t(cfg->KVH) * cfg->D;
    if (!ldk) ldk = width;
    if (!ldv) ldv = width;
    if (ldk < width || ldv < width)
        return dgm::fail(g, DGM_ERR_SHAPE, "cacheWrite: a row stride is shorter than the row's heads");
    if ((ldk | ldv) % 8 != 0 || ldk > (int64_t(1) << 31) || ldv > (int64_t(1) << 31) || rows > (int64_t(1) << 30) ||
        width > (int64_t(1) << 24))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "cacheWrite: strides must be multiples of 8 elements up to 2^31, "
                                                 "rows up to 2^30");
    if (rows == 0 || nseq == 0) return DGM_OK;
    if (!k || !v || !pages || !kcache || !vcache) return dgm::fail(g, DGM_ERR_ARG, "cacheWrite: null buffer");
    if (!dgm::aligned(k, 16) || !dgm::aligned(v, 16) || !dgm::aligned(kcache, 16) || !dgm::aligned(vcache, 16) ||
        !dgm::aligned(pages, 4) || !dgm::aligned(lens, 4) || !dgm::aligned(starts, 4))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "cacheWrite: a buffer is not 16-byte (starts, lens, pages: 4-byte) aligned");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "cacheWrite: %s", hipGetErrorString(on.err));
    const WriteArgs a{cache_of(g, cfg, pages), k, v, kcache, vcache, starts, lens, rows, nseq, ldk, ldv,
                      Div(uint32_t(width / 8))};
    if (type == DGM_TYPE_F32)
        return cfg->type == DGM_TYPE_F32 ? run_write<float, float>(g, a) : run_write<float, __bf16>(g, a);
    return cfg->type == DGM_TYPE_F32 ? run_write<__bf16, float>(g, a) : run_write<__bf16, __bf16>(g, a);
}

int64_t dgm_attnPagedDecode_ws_bytes(const dgm_cache_cfg* cfg, int64_t nseq, int64_t H) {
    if (!cfg || check_cache(nullptr, "", cfg, cfg->type, nseq) != DGM_OK || H < 1 || !heads_fit(nseq, H) ||
        H % cfg->KVH != 0)
        return -1;
    return decode_ws_bytes(cfg, nseq, H);
}

int dgm_attnPagedDecode(dgm_gpu* g, const dgm_cache_cfg* cfg, int64_t type, const void* q, const void* kcache,
                        const void* vcache, const int32_t* pages, const int32_t* lens, void* out, void* ws,
                        int64_t ws_bytes, int64_t nseq, int64_t H, int64_t ldq, int64_t ldo, float scale) {
    int rc = dgm::enter(g, "attn_paged_decode");
    if (rc) return rc;
    rc = check_cache(g, "attnPagedDecode", cfg, type, nseq);
    if (rc) return rc;
    if (H < 1) return dgm::fail(g, DGM_ERR_ARG, "attnPagedDecode: H=%lld", (long long)H);
    if (!(scale > 0.0f) || !std::isfinite(scale * kLog2e))
        return dgm::fail(g, DGM_ERR_ARG, "attnPagedDecode: scale must be positive and finite");
    if (H % cfg->KVH != 0)
        return dgm::fail(g, DGM_ERR_SHAPE, "attnPagedDecode: %lld query heads over %d key heads", (long long)H, cfg->KVH);
    const int64_t width = H * cfg->D;
    if (!ldq) ldq = width;
    if (!ldo) ldo = width;
    if (ldq < width || ldo < width)
        return dgm::fail(g, DGM_ERR_SHAPE, "attnPagedDecode: a row stride is shorter than the row's heads");
    if (!heads_fit(nseq, H) || (ldq | ldo) % 8 != 0 || ldq > (int64_t(1) << 31) || ldo > (int64_t(1) << 31))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "attnPagedDecode: strides must be multiples of 8 elements up to 2^31, "
                                                 "sequences x heads below 2^22");
    if (nseq == 0) return DGM_OK;
    if (!q || !kcache || !vcache || !pages || !lens || !out || !ws)
        return dgm::fail(g, DGM_ERR_ARG, "attnPagedDecode: null buffer");
    if (ws_bytes < decode_ws_bytes(cfg, nseq, H))
        return dgm::fail(g, DGM_ERR_ARG, "attnPagedDecode: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
                         (long long)decode_ws_bytes(cfg, nseq, H));
    for (const void* p : {q, kcache, vcache, static_cast<const void*>(out), static_cast<const void*>(ws)})
        if (!dgm::aligned(p, 16)) return dgm::fail(g, DGM_ERR_UNSUPPORTED, "attnPagedDecode: a buffer is not 16-byte aligned");
    if (!dgm::aligned(pages, 4) || !dgm::aligned(lens, 4))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "attnPagedDecode: pages or lens is not 4-byte aligned");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "attnPagedDecode: %s", hipGetErrorString(on.err));
    const Split sp = split_of(cfg, H);
    float* part = static_cast<float*>(ws);
    const DecodeArgs a{cache_of(g, cfg, pages), q, kcache, vcache, out, part, part + part_floats(cfg, nseq, H) * cfg->D,
                       lens, nseq, ldq, ldo, int(H), int(H / cfg->KVH), sp.heads, sp.parts, sp.workers, sp.units,
                       scale * kLog2e, Div(uint32_t(sp.workers))};
    if (type == DGM_TYPE_F32)
        return cfg->type == DGM_TYPE_F32 ? run_decode<float, float>(g, a) : run_decode<float, __bf16>(g, a);
    return cfg->type == DGM_TYPE_F32 ? run_decode<__bf16, float>(g, a) : run_decode<__bf16, __bf16>(g, a);
}

}  // extern "C"
