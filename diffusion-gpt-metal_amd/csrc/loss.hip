// Softmax cross-entropy of rows of logits with its gradient. No counterpart among
// the entry points that mirror the reference's wrappers.
//
//   lse = m + ln sum_v e^(z_v - m), m = max z;  loss = lse - z_t
//   dz_v = k (e^(z_v - m) / sum - [v = t]), k = scale * rowScale
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "step.hpp"

namespace {

using namespace dgm_step;

constexpr float kLn2 = 0.693147180559945309f;

struct LossArgs {
    const void* z;
    const int32_t* targets;
    const float* row_scale;
    float *loss, *lse;
    void* dz;
    uint32_t* words;
    int64_t rows, ld;
    int V;
    float scale;
};

// e^(z - m) by the hardware's power of two: the difference is exact where it matters (z near
// m), its product with log2 e rounded.
__device__ __forceinline__ float exp_of(float z, float m) { return dgm_attn::exp2_hw((z - m) * dgm_attn::kLog2e); }

// What a row's target asks for.
struct Target {
    int at;      // the target's column, -1: none, the row counts for nothing
    float z;     // its logit
    float k;     // scale of the gradient
};
template <typename T>
__device__ __forceinline__ Target target_of(const LossArgs& a, int64_t row, bool first) {
    const int t = a.targets[row];
    if (t >= a.V && first) report(a.words, kBadTokens);
    const int at = t < a.V ? t : -1;
    Target r{at < 0 ? -1 : at, 0.0f, a.scale};
    if (r.at >= 0) r.z = float(static_cast<const T*>(a.z)[row * a.ld + r.at]);
    if (a.row_scale) r.k *= a.row_scale[row];
    return r;
}

template <int V, typename T>
__device__ __forceinline__ void store_slope(T* row, int c, int cols, const float (&z)[V], float m, float inv, const Target& t) {
    float d[V];
    const float k = t.k * inv;
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = exp_of(z[j], m) * k;
    if (t.at >= c && t.at < c + V) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j == t.at) d[j] = (exp_of(z[j], m) * inv - 1.0f) * t.k;
    }
    if (t.at < 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = 0.0f;
    }
    store_piece<V>(row, c, cols, d);
}

template <typename T>
__device__ __forceinline__ void store_row(const LossArgs& a, int64_t row, const Target& t, float m, float sum) {
    const float lse = m + dgm_attn::log2_hw(sum) * kLn2;
    if (a.lse) a.lse[row] = lse;
    if (a.loss) a.loss[row] = t.at < 0 ? 0.0f : lse - t.z;
}

// TEAM lanes hold a row, CH pieces of 16 bytes each: one read, one write.
template <typename T, int TEAM, int CH>
__global__ __launch_bounds__(threads_of(TEAM)) void loss_kernel(LossArgs a) {
    constexpr int V = kVec<T>, TEAMS = threads_of(TEAM) / TEAM;
    __shared__ float slots[2][16];
    const int lane = threadIdx.x % TEAM;
    for (int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / TEAM; row < a.rows; row += int64_t(gridDim.x) * TEAMS) {
        const T* z = static_cast<const T*>(a.z) + row * a.ld;
        float x[CH][V];
#pragma unroll
        for (int i = 0; i < CH; ++i) load_piece<V>(z, (i * TEAM + lane) * V, a.V, x[i], kNegInf);
        const Target t = target_of<T>(a, row, lane == 0);
        float m = kNegInf;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) m = fmaxf(m, x[i][j]);
        m = team_max<TEAM>(m, slots[0]);
        m = m == kNegInf ? 0.0f : m;   // a row of nothing else: a sum of 0, lse -inf
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s += exp_of(x[i][j], m);
        s = team_sum<TEAM>(s, slots[1]);
        if (lane == 0) store_row<T>(a, row, t, m, s);
        if (a.dz) {
            T* dz = static_cast<T*>(a.dz) + row * a.ld;
            const float inv = 1.0f / s;
#pragma unroll
            for (int i = 0; i < CH; ++i) store_slope<V>(dz, (i * TEAM + lane) * V, a.V, x[i], m, inv, t);
        }
    }
}

// Rows beyond what a workgroup's registers hold: the maximum and the sum that
// belongs to it in one pass, the gradient in a second, from the cache where the row is still there.
template <typename T>
__global__ __launch_bounds__(1024) void loss_long_kernel(LossArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float slots[2][16];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* z = static_cast<const T*>(a.z) + row * a.ld;
        const Target t = target_of<T>(a, row, threadIdx.x == 0);
        float m = kNegInf, s = 0.0f;
        for (int c = threadIdx.x * V; c < a.V; c += 1024 * V) {
            float x[V];
            load_piece<V>(z, c, a.V, x, kNegInf);
            float top = x[0];
#pragma unroll
            for (int j = 1; j < V; ++j) top = fmaxf(top, x[j]);
            if (top > m) {
                s *= exp_of(m, top);
                m = top;
            }
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < a.V && x[j] != kNegInf) s += exp_of(x[j], m);
        }
        const float all = team_max<1024>(m, slots[0]);
        s = team_sum<1024>(m == kNegInf ? s : s * exp_of(m, all), slots[1]);
        if (threadIdx.x == 0) store_row<T>(a, row, t, all, s);
        if (a.dz) {
            T* dz = static_cast<T*>(a.dz) + row * a.ld;
            const float inv = 1.0f / s;
            for (int c = threadIdx.x * V; c < a.V; c += 1024 * V) {
                float x[V];
                load_piece<V>(z, c, a.V, x, kNegInf);
                store_slope<V>(dz, c, a.V, x, all, inv, t);
            }
        }
    }
}

template <typename T>
void launch(dgm_gpu* g, const LossArgs& a) {
    constexpr int V = kVec<T>;
    const auto blocks = [&](int teams) { return dim3(unsigned(std::min<int64_t>((a.rows + teams - 1) / teams, 1 << 20))); };
    const int n = (a.V + V - 1) / V;   // pieces
    if (n <= 16) loss_kernel<T, 16, 1><<<blocks(16), dim3(256), 0, g->stream>>>(a);
    else if (n <= 32) loss_kernel<T, 16, 2><<<blocks(16), dim3(256), 0, g->stream>>>(a);
    else if (n <= 128) loss_kernel<T, 64, 2><<<blocks(4), dim3(256), 0, g->stream>>>(a);
    else if (n <= 256) loss_kernel<T, 64, 4><<<blocks(4), dim3(256), 0, g->stream>>>(a);
    else if (n <= 1024) loss_kernel<T, 256, 4><<<blocks(1), dim3(256), 0, g->stream>>>(a);
    else if (n <= 2048) loss_kernel<T, 256, 8><<<blocks(1), dim3(256), 0, g->stream>>>(a);
    else if (n <= 4096) loss_kernel<T, 1024, 4><<<blocks(1), dim3(1024), 0, g->stream>>>(a);
    else if (n <= 8192) loss_kernel<T, 1024, 8><<<blocks(1), dim3(1024), 0, g->stream>>>(a);
    else loss_long_kernel<T><<<blocks(1), dim3(1024), 0, g->stream>>>(a);
}

}  // namespace

extern "C" int dgm_crossEntropy(dgm_gpu* g, const dgm_loss_cfg* cfg, const void* logits, const int32_t* targets,
                                const float* rowScale, float* loss, float* lse, void* dlogits) {
    int rc = dgm::enter(g, "cross_entropy");
    if (rc) return rc;
    if (!cfg) return dgm::fail(g, DGM_ERR_ARG, "crossEntropy: null configuration");
    if (!type_bytes(cfg->type)) return dgm::fail(g, DGM_ERR_ARG, "crossEntropy: unknown type %d", cfg->type);
    const int64_t ld = cfg->ld ? cfg->ld : cfg->V;
    if (cfg->rows < 0 || cfg->V < 1 || !std::isfinite(cfg->scale)) return dgm::fail(g, DGM_ERR_ARG, "crossEntropy: bad sizes or scale");
    if (ld < cfg->V) return dgm::fail(g, DGM_ERR_SHAPE, "crossEntropy: a row stride is shorter than the vocabulary");
    if (cfg->rows > dgm::kMaxIndex || ld > dgm::kMaxIndex / 2)
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "crossEntropy: rows beyond 2^31 - 1 or a row stride beyond 2^30");
    if (cfg->rows == 0 || (!loss && !lse && !dlogits)) return DGM_OK;
    if (!logits || !targets) return dgm::fail(g, DGM_ERR_ARG, "crossEntropy: null buffer");
    const size_t e = size_t(type_bytes(cfg->type));
    if (!dgm::aligned(logits, e) || !dgm::aligned(dlogits, e) || !dgm::aligned(targets, 4) || !dgm::aligned(rowScale, 4) ||
        !dgm::aligned(loss, 4) || !dgm::aligned(lse, 4))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "crossEntropy: a buffer is not aligned to its elements");
    OnDevice on(g->device);
    if (on.err != hipSuccess) return dgm::fail(g, DGM_ERR_HIP, "crossEntropy: %s", hipGetErrorString(on.err));
    const LossArgs a{logits, targets, rowScale, loss, lse, dlogits, g->seq_report, cfg->rows, ld, int(cfg->V), cfg->scale};
    if (cfg->type == DGM_TYPE_F32) launch<float>(g, a);
    else launch<__bf16>(g, a);
    DGM_LAUNCH_CHECK(g, "cross_entropy");
    return DGM_OK;
}
