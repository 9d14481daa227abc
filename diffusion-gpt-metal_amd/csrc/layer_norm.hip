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

namespace {

using namespace dgm_step;

struct FwdArgs {
    const void *x, *res;
    const float *w, *b;
    void *sum, *y;
    float *mean, *rstd;
    int64_t rows;
    int cols;
    float eps;
};

// TEAM lanes hold a row, CH pieces of 16 bytes each, so that it is read once and the
// variance is that of differences from the mean.
template <typename T, int TEAM, int CH>
__global__ __launch_bounds__(threads_of(TEAM)) void norm_fwd_kernel(FwdArgs a) {
    constexpr int V = kVec<T>, TEAMS = threads_of(TEAM) / TEAM;
    __shared__ float slots[2][16];
    const int lane = threadIdx.x % TEAM;
    const float n = float(a.cols);
    for (int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / TEAM; row < a.rows; row += int64_t(gridDim.x) * TEAMS) {
        const int64_t at = row * a.cols;
        float x[CH][V];
#pragma unroll
        for (int i = 0; i < CH; ++i) load_piece<V>(static_cast<const T*>(a.x) + at, (i * TEAM + lane) * V, a.cols, x[i]);
        if (a.res) {
            float r[CH][V];
#pragma unroll
            for (int i = 0; i < CH; ++i) load_piece<V>(static_cast<const T*>(a.res) + at, (i * TEAM + lane) * V, a.cols, r[i]);
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) x[i][j] = float(T(x[i][j] + r[i][j]));
            if (a.sum)
#pragma unroll
                for (int i = 0; i < CH; ++i) store_piece<V>(static_cast<T*>(a.sum) + at, (i * TEAM + lane) * V, a.cols, x[i]);
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s += x[i][j];
        const float mean = team_sum<TEAM>(s, slots[0]) / n;
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[i][j] -= mean;
                if ((i * TEAM + lane) * V + j < a.cols) ss = __builtin_fmaf(x[i][j], x[i][j], ss);
            }
        const float rstd = 1.0f / sqrtf(team_sum<TEAM>(ss, slots[1]) / n + a.eps);
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = (i * TEAM + lane) * V;
            float w[V], b[V];
            load_piece<V>(a.w, c, a.cols, w);
#pragma unroll
            for (int j = 0; j < V; ++j) b[j] = 0.0f;
            if (a.b) load_piece<V>(a.b, c, a.cols, b);
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = __builtin_fmaf(x[i][j] * rstd, w[j], b[j]);
            store_piece<V>(static_cast<T*>(a.y) + at, c, a.cols, x[i]);
        }
    }
}

struct BwdArgs {
    const void *x, *dy, *dsum;
    const float *mean, *rstd, *w;
    void* dx;
    float* part;   // [workgroups][2][cols]: their sums of dy xh and of dy
    int64_t rows;
    int cols;
};

template <typename T, int TEAM, int CH>
__global__ __launch_bounds__(threads_of(TEAM)) void norm_bwd_kernel(BwdArgs a) {
    constexpr int V = kVec<T>, TEAMS = threads_of(TEAM) / TEAM, WIDTH = TEAM * CH * V;
    __shared__ float slots[2][16];
    __shared__ float held[TEAMS > 1 ? TEAMS : 1][TEAMS > 1 ? WIDTH : 1];
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float n = float(a.cols);
    float w[CH][V], dw[CH][V], db[CH][V];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        load_piece<V>(a.w, (i * TEAM + lane) * V, a.cols, w[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
    }
    for (int64_t row = int64_t(blockIdx.x) * TEAMS + team; row < a.rows; row += int64_t(gridDim.x) * TEAMS) {
        const int64_t at = row * a.cols;
        float x[CH][V], dy[CH][V];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            load_piece<V>(static_cast<const T*>(a.x) + at, (i * TEAM + lane) * V, a.cols, x[i]);
            load_piece<V>(static_cast<const T*>(a.dy) + at, (i * TEAM + lane) * V, a.cols, dy[i]);
        }
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // Behind the row's end dy is 0 and takes no part.
                const float xh = (x[i][j] - mean) * rstd, g = dy[i][j] * w[i][j];
                x[i][j] = xh;
                const bool in = (i * TEAM + lane) * V + j < a.cols;
                dw[i][j] = in ? __builtin_fmaf(dy[i][j], xh, dw[i][j]) : 0.0f;
                db[i][j] += dy[i][j];
                s1 += g;
                s2 = in ? __builtin_fmaf(g, xh, s2) : s2;
            }
        s1 = team_sum<TEAM>(s1, slots[0]) / n;
        s2 = team_sum<TEAM>(s2, slots[1]) / n;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = (i * TEAM + lane) * V;
            float d[V];
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = 0.0f;
            if (a.dsum) load_piece<V>(static_cast<const T*>(a.dsum) + at, c, a.cols, d);
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] += rstd * (dy[i][j] * w[i][j] - s1 - x[i][j] * s2);
            store_piece<V>(static_cast<T*>(a.dx) + at, c, a.cols, d);
        }
    }
    float* part = a.part + int64_t(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float(&own)[CH][V] = k ? db : dw;
        if constexpr (TEAMS == 1) {
#pragma unroll
            for (int i = 0; i < CH; ++i) store_piece<V>(part + k * a.cols, (i * TEAM + lane) * V, a.cols, own[i]);
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) held[team][(i * TEAM + lane) * V + j] = own[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += int(blockDim.x)) {
                float s = held[0][c];
#pragma unroll
                for (int t = 1; t < TEAMS; ++t) s += held[t][c];
                part[k * a.cols + c] = s;
            }
        }
    }
}

// dw += the workgroups' sums, and db: 64 columns a workgroup, four shares of the workgroups' rows.
__global__ __launch_bounds__(256) void norm_join_kernel(const float* __restrict__ part, float* dw, float* db, int parts, int cols) {
    __shared__ float sums[4][64];
    const int k = blockIdx.y, lane = threadIdx.x & 63, share = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float* out = k ? db : dw;
    if (!out) return;
    float s = 0.0f;
    if (c < cols) {
        const float* p = part + k * cols + c;
#pragma unroll 8
        for (int i = share; i < parts; i += 4) s += p[int64_t(i) * 2 * cols];
    }
    sums[share][lane] = s;
    __syncthreads();
    if (share == 0 && c < cols) out[c] += ((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane];
}

constexpr int kMaxCols = 32768;

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

// Lanes to a row and pieces to a lane: 16 lanes up to 128 elements, a wave up to 2048, a workgroup beyond.
struct Shape {
    int team, elems;
};
Shape shape_of(int64_t cols) {
    if (cols <= 128) return {16, 8};
    if (cols <= 512) return {64, 8};
    if (cols <= 1024) return {64, 16};
    if (cols <= 2048) return {64, 32};
    if (cols <= 4096) return {256, 16};
    if (cols <= 8192) return {256, 32};
    return {1024, cols <= 16384 ? 16 : 32};
}

// f(T, TEAM, CH) for the configuration's kernel.
template <typename F>
void dispatch(const dgm_norm_cfg* c, const F& f) {
    const Shape s = shape_of(c->cols);
    const int key = s.team * 64 + s.elems;
    const bool wide = c->type == DGM_TYPE_F32;
#define DGM_NORM(TEAM, E)                                                                              \
    case TEAM * 64 + E:                                                                                \
        wide ? f(float{}, std::integral_constant<int, TEAM>{}, std::integral_constant<int, E / 4>{})   \
             : f(__bf16{}, std::integral_constant<int, TEAM>{}, std::integral_constant<int, E / 8>{}); \
        break;
    switch (key) {
        DGM_NORM(16, 8) DGM_NORM(64, 8) DGM_NORM(64, 16) DGM_NORM(64, 32)
        DGM_NORM(256, 16) DGM_NORM(256, 32) DGM_NORM(1024, 16) DGM_NORM(1024, 32)
    }
#undef DGM_NORM
}

int64_t blocks_for(const dgm_norm_cfg* c, int64_t most) {
    const int team = shape_of(c->cols).team, teams = threads_of(team) / team;
    return std::min<int64_t>((c->rows + teams - 1) / teams, most);
}
constexpr int64_t kFwdBlocks = 1 << 20, kBwdBlocks = 512;

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
    const size_t e = size_t(type_bytes(cfg->type));
    if (!dgm::aligned(x, e) || !dgm::aligned(res, e) || !dgm::aligned(sum, e) || !dgm::aligned(y, e) ||
        !dgm::aligned(weight, 4) || !dgm::aligned(bias, 4) || !dgm::aligned(mean, 4) || !dgm::aligned(rstd, 4))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "layerNormFwd: a buffer is not aligned to its elements");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "layerNormFwd: %s", hipGetErrorString(on.err));
    const FwdArgs a{x, res, weight, bias, sum, y, mean, rstd, cfg->rows, int(cfg->cols), cfg->eps};
    dispatch(cfg, [&](auto t, auto team, auto ch) {
        constexpr int TEAM = decltype(team)::value, CH = decltype(ch)::value;
        norm_fwd_kernel<decltype(t), TEAM, CH><<<dim3(unsigned(blocks_for(cfg, kFwdBlocks))), dim3(threads_of(TEAM)), 0, g->stream>>>(a);
    });
    DGM_LAUNCH_CHECK(g, "layer_norm_fwd");
    return DGM_OK;
}

int64_t dgm_layerNormBwd_ws_bytes(const dgm_norm_cfg* cfg) {
    if (check(nullptr, "", cfg) != DGM_OK) return -1;
    return blocks_for(cfg, kBwdBlocks) * 2 * cfg->cols * int64_t(sizeof(float));
}

int dgm_layerNormBwd(dgm_gpu* g, const dgm_norm_cfg* cfg, const void* x, const float* mean, const float* rstd,
                     const float* weight, const void* dy, const void* dsum, void* dx, float* dweight, float* dbias,
                     void* ws, int64_t ws_bytes) {
    int rc = dgm::enter(g, "layer_norm_bwd");
    if (rc) return rc;
    rc = check(g, "layerNormBwd", cfg);
    if (rc) return rc;
    if (cfg->rows == 0) return DGM_OK;
    if (!x || !mean || !rstd || !weight || !dy || !dx || !ws) return dgm::fail(g, DGM_ERR_ARG, "layerNormBwd: null buffer");
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
    const int64_t blocks = blocks_for(cfg, kBwdBlocks);
    const BwdArgs a{x, dy, dsum, mean, rstd, weight, dx, static_cast<float*>(ws), cfg->rows, int(cfg->cols)};
    dispatch(cfg, [&](auto t, auto team, auto ch) {
        constexpr int TEAM = decltype(team)::value, CH = decltype(ch)::value;
        norm_bwd_kernel<decltype(t), TEAM, CH><<<dim3(unsigned(blocks)), dim3(threads_of(TEAM)), 0, g->stream>>>(a);
    });
    DGM_LAUNCH_CHECK(g, "layer_norm_bwd");
    if (!dweight && !dbias) return DGM_OK;
    norm_join_kernel<<<dim3(dgm::ceil_div(cfg->cols, 64), 2), dim3(256), 0, g->stream>>>(a.part, dweight, dbias, int(blocks), a.cols);
    DGM_LAUNCH_CHECK(g, "layer_norm_join");
    return DGM_OK;
}

}  // extern "C"
