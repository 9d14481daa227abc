// Layer norm with the residual sum before it, and its gradients. No counterpart
// among the entry points that mirror the reference's wrappers: rmsFwd / rmsBwd are the DiT's norm,
// this one is the GPT's (its parameters ln1.g, ln1.b, ..., ln_f.b are in the checkpoints).
//
//   h = x + res (rounded to the rows' type: the next layer reads it), mu = mean(h),
//   rstd = 1 / sqrt(mean((h - mu)^2) + eps), y = (h - mu) rstd w + b
//   with g = dy w and xh = (h - mu) rstd:
//   dx = dsum + rstd (g - mean(g) - xh mean(g xh)), dw += sum dy xh, db += sum dy over the rows
#include <algorithm>
#include <type_traits>

#include "step.hpp"

// Products are fused into sums only where it is written: g, which is added up and then less its mean, has to be the same number both
// times (the gradient of a row of one element is 0). In short rows, where dx is what is left of terms that cancel (all but
// eps / variance of it in rows of two), each operation is rounded on its own: no more exact, but the formula's own roundings, so
// that what remains is what the formula in 32 bits leaves. Wide rows: 202 us fused, 213 not (16384 of 4096, bf16).
#pragma clang fp contract(off)

namespace {

using namespace dgm_step;

// a b + c, fused for rows that a wave or more lanes share.
template <int TEAM>
__device__ __forceinline__ float mul_add(float a, float b, float c) {
    return TEAM > 16 ? __builtin_fmaf(a, b, c) : a * b + c;
}

// A lane's share of a row: CH whole pieces of 16 bytes as they came, and one of the elements around those. What the
// row does not have is zeros.
template <typename T, int TEAM, int CH>
struct Share {
    static constexpr int V = kVec<T>;
    piece_t<T, V> piece[CH];
    float last;

    __device__ __forceinline__ void load(const T* row, const Span& w, int lane) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (i * TEAM + lane < w.whole) {
                piece[i] = *reinterpret_cast<const piece_t<T, V>*>(row + w.head + (i * TEAM + lane) * V);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) piece[i][j] = T(0.0f);
            }
        }
        last = w.last >= 0 ? float(row[w.last]) : 0.0f;
    }
    __device__ __forceinline__ void store(T* row, const Span& w, int lane) const {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i * TEAM + lane < w.whole) *reinterpret_cast<piece_t<T, V>*>(row + w.head + (i * TEAM + lane) * V) = piece[i];
        if (w.last >= 0) row[w.last] = T(last);
    }
};

// The same share of a row of fp32 parameters or sums.
template <int V, int TEAM, int CH>
struct Floats {
    float piece[CH][V], last;

    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) piece[i][j] = x;
        last = x;
    }
    __device__ __forceinline__ void load(const float* row, const Span& w, int lane) {
        fill(0.0f);
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i * TEAM + lane < w.whole) {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const piece_t<float, 4> v = *reinterpret_cast<const piece_t<float, 4>*>(row + w.head + (i * TEAM + lane) * V + j);
#pragma unroll
                    for (int k = 0; k < 4; ++k) piece[i][j + k] = v[k];
                }
            }
        if (w.last >= 0) last = row[w.last];
    }
    __device__ __forceinline__ void store(float* row, const Span& w, int lane) const {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i * TEAM + lane < w.whole) {
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    *reinterpret_cast<piece_t<float, 4>*>(row + w.head + (i * TEAM + lane) * V + j) =
                        piece_t<float, 4>{piece[i][j], piece[i][j + 1], piece[i][j + 2], piece[i][j + 3]};
            }
        if (w.last >= 0) row[w.last] = last;
    }
};

struct FwdArgs {
    const void *x, *res;
    const float *w, *b;
    void *sum, *y;
    float *mean, *rstd;
    int64_t rows;
    int cols;
    float eps;
};

// TEAM lanes hold a row, so that it is read once and the variance is that of differences from the mean. Bound by memory:
// 16384 bf16 rows of 4096 with the residual 97 us (5.5 TB/s).
template <typename T, int TEAM, int CH>
__global__ __launch_bounds__(threads_of(TEAM)) void norm_fwd_kernel(FwdArgs a) {
    constexpr int V = kVec<T>, TEAMS = threads_of(TEAM) / TEAM;
    __shared__ float slots[2][16];
    const int lane = threadIdx.x % TEAM;
    const float n = float(a.cols);
    for (int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / TEAM; row < a.rows; row += int64_t(gridDim.x) * TEAMS) {
        const int64_t at = row * a.cols;
        const Span p = span_of(static_cast<const T*>(a.x) + at, a.cols, lane);
        Share<T, TEAM, CH> x;
        x.load(static_cast<const T*>(a.x) + at, p, lane);
        if (a.res) {
            Share<T, TEAM, CH> r;
            r.load(static_cast<const T*>(a.res) + at, p, lane);
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) x.piece[i][j] = T(float(x.piece[i][j]) + float(r.piece[i][j]));
            x.last = float(T(x.last + r.last));
            x.store(static_cast<T*>(a.sum) + at, p, lane);
        }
        float s = x.last;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s += float(x.piece[i][j]);
        const float mean = team_sum<TEAM>(s, slots[0]) / n;
        const float d = p.last >= 0 ? x.last - mean : 0.0f;
        float ss = d * d;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i * TEAM + lane < p.whole)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float e = float(x.piece[i][j]) - mean;
                    ss = mul_add<TEAM>(e, e, ss);
                }
        const float rstd = 1.0f / sqrtf(team_sum<TEAM>(ss, slots[1]) / n + a.eps);
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        Floats<V, TEAM, CH> w, b;
        w.load(a.w, p, lane);
        if (a.b) b.load(a.b, p, lane);
        else b.fill(0.0f);
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                x.piece[i][j] = T(mul_add<TEAM>((float(x.piece[i][j]) - mean) * rstd, w.piece[i][j], b.piece[i][j]));
        x.last = mul_add<TEAM>(d * rstd, w.last, b.last);
        x.store(static_cast<T*>(a.y) + at, p, lane);
    }
}

struct BwdArgs {
    const void *x, *dy, *dsum;
    const float *mean, *rstd, *w;
    void* dx;
    float* part;   // [workgroups][2][cols]: their sums of dy xh and of dy
    int64_t rows;
    int cols, groups;      // workgroups that take rows
    float *dw, *db;        // of the columns' workgroups
};

// The sums of 32 columns over all rows, a share of the rows to each 32 threads. Eight rows are added up by themselves first: they
// are on their way together, and a share of up to 128 rows is 24 additions long at most, not 128.
template <typename T, int THREADS>
__device__ __forceinline__ void norm_columns(const BwdArgs& a, int block) {
    constexpr int SHARES = THREADS / 32;
    __shared__ float sums[2][SHARES][32];
    const int t = threadIdx.x & 31, share = threadIdx.x >> 5, c = block * 32 + t;
    float dw = 0.0f, db = 0.0f;
    if (c < a.cols) {
        const auto add = [&](int r, float& w, float& b) {
            const float x = float(static_cast<const T*>(a.x)[int64_t(r) * a.cols + c]);
            const float y = float(static_cast<const T*>(a.dy)[int64_t(r) * a.cols + c]);
            w = __builtin_fmaf(y, (x - a.mean[r]) * a.rstd[r], w);
            b += y;
        };
        int r = share;
        for (; r + 7 * SHARES < int(a.rows); r += 8 * SHARES) {
            float w = 0.0f, b = 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u) add(r + u * SHARES, w, b);
            dw += w;
            db += b;
        }
        float w = 0.0f, b = 0.0f;
        for (; r < int(a.rows); r += SHARES) add(r, w, b);
        dw += w;
        db += b;
    }
    sums[0][share][t] = dw;
    sums[1][share][t] = db;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    float* out = share ? a.db : a.dw;
    if (!out || c >= a.cols) return;
    float s = sums[share][0][t];
#pragma unroll
    for (int i = 1; i < SHARES; ++i) s += sums[share][i][t];
    out[c] += s;
}

// TEAMS rows at a time in a workgroup, whose lanes keep the sums of their columns over all its rows; with AHEAD the next
// rows are on their way while these are worked on. APART: workgroups behind those of the rows take the columns' sums. Bound
// by memory and the chain of a row's steps: 16384 bf16 rows of 4096 with dsum 122 us (4.4 TB/s; two rows ahead 45 more).
template <typename T, int TEAM, int CH, int TEAMS, int WAVES, bool AHEAD, bool APART>
__global__ __launch_bounds__(TEAM* TEAMS, WAVES) void norm_bwd_kernel(BwdArgs a) {
    constexpr int V = kVec<T>;
    if constexpr (APART) {
        if (int(blockIdx.x) >= a.groups) {
            norm_columns<T, TEAM * TEAMS>(a, int(blockIdx.x) - a.groups);
            return;
        }
    }
    __shared__ float slots[2][TEAMS][2][TEAM > 64 ? TEAM / 64 : 1];
    __shared__ float held[TEAMS > 1 && !APART ? TEAMS : 1][TEAMS > 1 && !APART ? TEAM * CH * V : 1];
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float n = float(a.cols);
    const T *x0 = static_cast<const T*>(a.x), *y0 = static_cast<const T*>(a.dy), *s0 = static_cast<const T*>(a.dsum);
    const int64_t step = int64_t(a.groups) * TEAMS;
    const int64_t first = int64_t(blockIdx.x) * TEAMS;
    // A lane's columns stay the same over its rows: where rows of odd lengths follow at odd distances, all have their pieces
    // from the first element on.
    const bool even = (step & 1) == 0 || (a.cols & 1) == 0;
    const Span p = span_of(even ? x0 + (first + team) * a.cols : x0, a.cols, lane);
    Floats<V, TEAM, CH> w, dw, db;
    w.load(a.w, p, lane);
    dw.fill(0.0f);
    db.fill(0.0f);
    Share<T, TEAM, CH> x, y, s;
    float mean = 0.0f, rstd = 0.0f;
    const auto load = [&](int64_t row) {
        if (row < a.rows) {
            const int64_t at = row * a.cols;
            x.load(x0 + at, p, lane);
            y.load(y0 + at, p, lane);
            if (a.dsum) s.load(s0 + at, p, lane);
            mean = a.mean[row];
            rstd = a.rstd[row];
        }
    };
    if (AHEAD) load(first + team);
    int turn = 0;
    for (int64_t base = first; base < a.rows; base += step, turn ^= 1) {
        const int64_t row = base + team;
        const bool in = row < a.rows;
        if (!AHEAD) load(row);
        Share<T, TEAM, CH> cx = x, cy = y, cs = s;
        const float cmean = mean, crstd = rstd;
        if (AHEAD) load(row + step);
        float s1 = 0.0f, s2 = 0.0f;
        const auto term = [&](float xv, float yv, float wv, float& dwv, float& dbv) {
            const float xh = (xv - cmean) * crstd, g = yv * wv;
            dwv = __builtin_fmaf(yv, xh, dwv);
            dbv += yv;
            s1 += g;
            s2 = mul_add<TEAM>(g, xh, s2);
        };
        if (in) {
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (i * TEAM + lane < p.whole)
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        term(float(cx.piece[i][j]), float(cy.piece[i][j]), w.piece[i][j], dw.piece[i][j], db.piece[i][j]);
            if (p.last >= 0) term(cx.last, cy.last, w.last, dw.last, db.last);
        }
        if constexpr (TEAM == 16) {
            s1 = dgm_rows::row16_sum(s1);
            s2 = dgm_rows::row16_sum(s2);
        } else {
            s1 = dgm_rows::wave64_sum(s1);
            s2 = dgm_rows::wave64_sum(s2);
        }
        if constexpr (TEAM > 64) {
            // Two sets of slots: a row's are read before its barrier's successor, behind which they are written again.
            float(&slot)[2][TEAM / 64] = slots[turn][team];
            if ((lane & 63) == 0) {
                slot[0][lane >> 6] = s1;
                slot[1][lane >> 6] = s2;
            }
            __syncthreads();
            s1 = slot[0][0];
            s2 = slot[1][0];
#pragma unroll
            for (int v = 1; v < TEAM / 64; ++v) {
                s1 += slot[0][v];
                s2 += slot[1][v];
            }
        }
        if (!in) continue;
        s1 /= n;
        s2 /= n;
        const auto slope = [&](float xv, float yv, float wv, float sv) {
            const float xh = (xv - cmean) * crstd;
            return mul_add<TEAM>(crstd, mul_add<TEAM>(-xh, s2, yv * wv - s1), sv);
        };
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                cx.piece[i][j] = T(slope(float(cx.piece[i][j]), float(cy.piece[i][j]), w.piece[i][j], a.dsum ? float(cs.piece[i][j]) : 0.0f));
        cx.last = slope(cx.last, cy.last, w.last, a.dsum ? cs.last : 0.0f);
        cx.store(static_cast<T*>(a.dx) + row * a.cols, p, lane);
    }
    if constexpr (APART) return;
    float* part = a.part + int64_t(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const Floats<V, TEAM, CH>& own = k ? db : dw;
        if constexpr (TEAMS == 1) {
            own.store(part + k * a.cols, p, lane);
        } else {
            __syncthreads();
            own.store(held[team], p, lane);
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += TEAM * TEAMS) {
                float sum = held[0][c];
#pragma unroll
                for (int t = 1; t < TEAMS; ++t) sum += held[t][c];
                part[k * a.cols + c] = sum;
            }
        }
    }
}

// dw += the workgroups' sums, and db: 64 columns a workgroup, a share of the parts to each of its 16 waves.
__global__ __launch_bounds__(1024) void norm_join_kernel(const float* __restrict__ part, float* dw, float* db, int parts, int cols) {
    __shared__ float sums[16][64];
    const int k = blockIdx.y, lane = threadIdx.x & 63, share = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float* out = k ? db : dw;
    if (!out) return;
    float s = 0.0f;
    if (c < cols) {
        const float* p = part + k * cols + c;
#pragma unroll 16
        for (int i = share; i < parts; i += 16) s += p[int64_t(i) * 2 * cols];
    }
    sums[share][lane] = s;
    __syncthreads();
    if (share > 0 || c >= cols) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sums[i][lane];
    out[c] += s;
}

constexpr int kMaxCols = 16384;

int check(dgm_gpu* g, const char* name, const dgm_norm_cfg* c) {
    if (!c) return dgm::fail(g, DGM_ERR_ARG, "%s: null configuration", name);
    if (!type_bytes(c->type)) return dgm::fail(g, DGM_ERR_ARG, "%s: unknown type %d", name, c->type);
    if (c->rows < 0 || c->cols < 1 || !(c->eps >= 0.0f) || c->eps > 1e30f)
        return dgm::fail(g, DGM_ERR_ARG, "%s: bad sizes or eps", name);
    if (c->cols > kMaxCols || c->rows > dgm::kMaxIndex)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "%s: %lld rows of %lld: at most 2^31 - 1 of %d", name, (long long)c->rows,
                         (long long)c->cols, kMaxCols);
    return DGM_OK;
}

// The forward's lanes to a row and elements to a lane: 16 lanes up to 128 elements, a wave up to 2048, a workgroup beyond.
#define DGM_NORM_FWD(X) X(16, 8) X(64, 8) X(64, 16) X(64, 32) X(256, 16) X(256, 32) X(1024, 16)
// The backward's lanes, elements, rows of a workgroup at a time, waves to a SIMD and whether the next rows are asked for ahead,
// by the same widths: sums, parameters and rows have to fit the registers of enough waves (us with the forward, bf16 with the
// residual): 16384 rows of 4096 204 with 512 lanes and ahead, 235 without, 207 with 256 lanes; 16384 of 2048 107, a wave for
// a row 107 (fp32 209 and 315); 32768 of 1024 106 without and 126 ahead (fp32 223 and 348: spills); 8192 of 8192 214, 216
// ahead; 4096 of 16384 240 with 512 lanes, 259 with 1024.
#define DGM_NORM_BWD(X) \
    X(128, 16, 8, 32, 4, true) X(512, 64, 8, 8, 4, true) X(1024, 64, 16, 8, 4, false) X(2048, 256, 8, 1, 4, true) \
    X(4096, 512, 8, 1, 4, true) X(8192, 1024, 8, 1, 4, false) X(16384, 512, 32, 1, 2, false)

int width_of(int64_t cols) {
    for (int w : {128, 512, 1024, 2048, 4096, 8192})
        if (cols <= w) return w;
    return kMaxCols;
}

// f(type, TEAM, pieces of a lane).
template <typename F>
void forward(const dgm_norm_cfg* c, const F& f) {
    const bool wide = c->type == DGM_TYPE_F32;
    switch (width_of(c->cols)) {
#define DGM_NORM(TEAM, E)                                                                              \
    case TEAM * E:                                                                                     \
        wide ? f(float{}, std::integral_constant<int, TEAM>{}, std::integral_constant<int, E / 4>{})   \
             : f(__bf16{}, std::integral_constant<int, TEAM>{}, std::integral_constant<int, E / 8>{}); \
        break;
        DGM_NORM_FWD(DGM_NORM)
#undef DGM_NORM
    }
}

// Rows of a workgroup at a time, its workgroups and whether the columns' sums are workgroups of their own: then there is no
// second launch, but x and dy are read twice (us with the forward, fp32: 1024 rows of 128 15.5, 18.3 with a second launch; of
// 1024 16.2 and 18.8; of 4096 34.5 and 33.0; 4096 rows of 128 24.9 and 19.2).
struct Split {
    int teams, groups;
    bool apart;
};
constexpr int kBwdGroups = 256;
constexpr int64_t kApartRows = 2048, kApartSize = 1 << 20;
Split split_of(const dgm_norm_cfg* c) {
    Split s{1, 0, c->rows <= kApartRows && c->rows * c->cols <= kApartSize};
    switch (width_of(c->cols)) {
#define DGM_NORM(W, TEAM, E, TEAMS, WAVES, AHEAD) \
    case W: s.teams = TEAMS; break;
        DGM_NORM_BWD(DGM_NORM)
#undef DGM_NORM
    }
    const int64_t groups = (c->rows + s.teams - 1) / s.teams;
    s.groups = int(s.apart ? groups : std::min<int64_t>(groups, c->cols <= 2048 && c->cols > 1024 ? 2 * kBwdGroups : kBwdGroups));
    return s;
}

template <typename T, bool APART>
void launch_bwd(dgm_gpu* g, int64_t cols, unsigned grid, const BwdArgs& a) {
    switch (width_of(cols)) {
#define DGM_NORM(W, TEAM, E, TEAMS, WAVES, AHEAD)                                                            \
    case W:                                                                                                  \
        norm_bwd_kernel<T, TEAM, E / kVec<T>, TEAMS, WAVES, AHEAD && !APART, APART>                           \
            <<<dim3(grid), dim3(TEAM * TEAMS), 0, g->stream>>>(a);                                           \
        break;
        DGM_NORM_BWD(DGM_NORM)
#undef DGM_NORM
    }
}

constexpr int64_t kFwdBlocks = 1 << 20;

}  // namespace

extern "C" {

int dgm_layerNormFwd(dgm_gpu* g, const dgm_norm_cfg* cfg, const void* x, const void* res, const float* weight,
                     const float* bias, void* sum, void* y, float* mean, float* rstd) {
    int rc = dgm::enter(g, "layer_norm_fwd");
    if (rc) return rc;
    rc = check(g, "layerNormFwd", cfg);
    if (rc) return rc;
    if (cfg->rows == 0) return DGM_OK;
    if (!x || !weight || !y) return dgm::fail(g, DGM_ERR_ARG, "layerNormFwd: null buffer");
    if (!res != !sum) return dgm::fail(g, DGM_ERR_ARG, "layerNormFwd: a residual and its sum go together");
    if (sum == y || (mean && mean == rstd)) return dgm::fail(g, DGM_ERR_ARG, "layerNormFwd: two results share memory");
    const size_t e = size_t(type_bytes(cfg->type));
    if (!dgm::aligned(x, e) || !dgm::aligned(res, e) || !dgm::aligned(sum, e) || !dgm::aligned(y, e) ||
        !dgm::aligned(weight, 4) || !dgm::aligned(bias, 4) || !dgm::aligned(mean, 4) || !dgm::aligned(rstd, 4))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "layerNormFwd: a buffer is not aligned to its elements");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "layerNormFwd: %s", hipGetErrorString(on.err));
    const FwdArgs a{x, res, weight, bias, sum, y, mean, rstd, cfg->rows, int(cfg->cols), cfg->eps};
    forward(cfg, [&](auto t, auto team, auto ch) {
        constexpr int TEAM = decltype(team)::value, CH = decltype(ch)::value, TEAMS = threads_of(TEAM) / TEAM;
        const int64_t groups = std::min<int64_t>((cfg->rows + TEAMS - 1) / TEAMS, kFwdBlocks);
        norm_fwd_kernel<decltype(t), TEAM, CH><<<dim3(unsigned(groups)), dim3(threads_of(TEAM)), 0, g->stream>>>(a);
    });
    DGM_LAUNCH_CHECK(g, "layer_norm_fwd");
    return DGM_OK;
}

int64_t dgm_layerNormBwd_ws_bytes(const dgm_norm_cfg* cfg) {
    if (check(nullptr, "", cfg) != DGM_OK) return -1;
    const Split s = split_of(cfg);
    return s.apart ? 0 : int64_t(s.groups) * 2 * cfg->cols * int64_t(sizeof(float));
}

int dgm_layerNormBwd(dgm_gpu* g, const dgm_norm_cfg* cfg, const void* x, const float* mean, const float* rstd,
                     const float* weight, const void* dy, const void* dsum, void* dx, float* dweight, float* dbias,
                     void* ws, int64_t ws_bytes) {
    int rc = dgm::enter(g, "layer_norm_bwd");
    if (rc) return rc;
    rc = check(g, "layerNormBwd", cfg);
    if (rc) return rc;
    if (cfg->rows == 0) return DGM_OK;
    if (!x || !mean || !rstd || !weight || !dy || !dx || (!ws && dgm_layerNormBwd_ws_bytes(cfg) > 0))
        return dgm::fail(g, DGM_ERR_ARG, "layerNormBwd: null buffer");
    if (dweight && dweight == dbias) return dgm::fail(g, DGM_ERR_ARG, "layerNormBwd: dweight and dbias share memory");
    if (dx == x || dx == dy) return dgm::fail(g, DGM_ERR_ARG, "layerNormBwd: dx may share memory with dsum alone");
    if (ws_bytes < dgm_layerNormBwd_ws_bytes(cfg))
        return dgm::fail(g, DGM_ERR_ARG, "layerNormBwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
                         (long long)dgm_layerNormBwd_ws_bytes(cfg));
    const size_t e = size_t(type_bytes(cfg->type));
    if (!dgm::aligned(x, e) || !dgm::aligned(dy, e) || !dgm::aligned(dsum, e) || !dgm::aligned(dx, e) ||
        !dgm::aligned(weight, 4) || !dgm::aligned(mean, 4) || !dgm::aligned(rstd, 4) || !dgm::aligned(dweight, 4) ||
        !dgm::aligned(dbias, 4) || !dgm::aligned(ws, 16))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "layerNormBwd: a buffer is not aligned to its elements, or the workspace to 16 bytes");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "layerNormBwd: %s", hipGetErrorString(on.err));
    const Split s = split_of(cfg);
    const bool sums = dweight || dbias;
    const BwdArgs a{x, dy, dsum, mean, rstd, weight, dx, static_cast<float*>(ws), cfg->rows, int(cfg->cols), s.groups, dweight, dbias};
    const bool wide = cfg->type == DGM_TYPE_F32;
    if (s.apart) {
        const unsigned grid = unsigned(s.groups) + (sums ? dgm::ceil_div(cfg->cols, 32) : 0);
        wide ? launch_bwd<float, true>(g, cfg->cols, grid, a) : launch_bwd<__bf16, true>(g, cfg->cols, grid, a);
    } else {
        wide ? launch_bwd<float, false>(g, cfg->cols, unsigned(s.groups), a) : launch_bwd<__bf16, false>(g, cfg->cols, unsigned(s.groups), a);
    }
    DGM_LAUNCH_CHECK(g, "layer_norm_bwd");
    if (!sums || s.apart) return DGM_OK;
    norm_join_kernel<<<dim3(dgm::ceil_div(cfg->cols, 64), 2), dim3(1024), 0, g->stream>>>(a.part, dweight, dbias, s.groups, a.cols);
    DGM_LAUNCH_CHECK(g, "layer_norm_join");
    return DGM_OK;
}

}  // extern "C"
