// Index arithmetic of the attention kernels over packed sequences and over a
// paged cache: what turns starts, lengths and page tables, which only the
// device reads, into rows. Plain C++, so that it also runs on the host.
#pragma once
#include <cstdint>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define DGM_HD __host__ __device__ __forceinline__
#else
#define DGM_HD inline
#endif

namespace dgm_attn {

// starts[i] within [0, rows], whatever it holds.
DGM_HD int clamped(const int32_t* starts, int64_t i, int64_t rows) {
    const int64_t s = starts[i];
    return int(s < 0 ? 0 : s > rows ? rows : s);
}

// First tile slot (tiles of `per` rows) of sequence s, which starts at row
// `first`: ceil(len / per) <= (first + len) / per - first / per + 1, so that the
// slots of the next sequence lie behind those of this one.
DGM_HD int64_t slot_base(int first, int64_t s, int per) { return first / per + s; }
inline int64_t slot_count(int64_t rows, int64_t nseq, int per) { return rows / per + nseq; }

// n / d for n < 2^31 by a product: m = floor(2^sh / d) + 1 with sh = 31 +
// ceil(log2 d). m d exceeds 2^sh by at most d <= 2^(sh - 31), which n < 2^31 keeps below the next quotient.
struct Div {
    uint32_t d, m;
    int sh;
    explicit Div(uint32_t d_) : d(d_) {
        int l = 0;
        while ((uint64_t(1) << l) < d) ++l;
        sh = 31 + l;
        m = uint32_t((uint64_t(1) << sh) / d + 1);
    }
    DGM_HD uint32_t operator()(uint32_t n) const { return uint32_t(uint64_t(n) * m >> sh); }
};

// Row of a cache [numPages * KVH * page.d, D] (below 2^31 rows) that holds position
// `pos` (below maxPages * page.d) of sequence s for key head h; -1 for a page
// that the cache does not have.
DGM_HD int cache_row(const int32_t* pages, const Div& page, int64_t numPages, int64_t maxPages, int KVH, int64_t s,
                     uint32_t pos, int h) {
    const uint32_t i = page(pos);
    const int32_t id = pages[s * maxPages + i];
    if (id < 0 || id >= numPages) return -1;
    return (id * KVH + h) * int(page.d) + int(pos - i * page.d);
}

}  // namespace dgm_attn
