// Softmax cross-entropy of rows of logits with its gradient. No counterpart among
// the entry points that mirror the reference's wrappers.
//
//   lse = m + ln sum_v e^(z_v - m), m = max z;  loss = lse - z_t = (m - z_t) + ln sum
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

// A piece of a row's gradient, from column c on, of its e^(z - m): k / sum times those, `hot` at the target.
template <typename T, int V>
__device__ __forceinline__ void store_slopes(T* dz, int c, float (&e)[V], float k, const Target& t, float hot) {
    piece_t<T, V> d;
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] *= k;
    if (uint32_t(t.at - c) < uint32_t(V)) {
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = c + j == t.at ? hot : e[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = T(e[j]);
    *reinterpret_cast<piece_t<T, V>*>(dz + c) = d;
}

// The gradient of a row that counts for nothing, whatever it holds.
template <typename T, int V>
__device__ __forceinline__ void store_zeros(T* dz, int cols, int lane, int lanes) {
    const Span w = span_of(dz, cols, lane);
    piece_t<T, V> d;
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = T(0.0f);
    for (int c = lane; c < w.whole; c += lanes) *reinterpret_cast<piece_t<T, V>*>(dz + w.head + c * V) = d;
    if (w.last >= 0) dz[w.last] = T(0.0f);
}

template <typename T>
__device__ __forceinline__ void store_row(const LossArgs& a, int64_t row, const Target& t, float m, float sum) {
    // The loss from its own terms: lse is rounded at the size of the logits, which may be far above a small loss.
    const float ln = dgm_attn::log2_hw(sum) * kLn2;
    if (a.lse) a.lse[row] = m + ln;
    if (a.loss) a.loss[row] = t.at < 0 ? 0.0f : (m - t.z) + ln;
}

// Bound by memory: one read, one write; 8192 bf16 rows of 50257 304 us (5.4 TB/s), 4096 fp32 rows of 32000 191 (5.5).
// TEAM lanes hold a row in registers as it came, CH pieces of 16 bytes each and one element behind the last
// whole piece: one read, one write.
template <typename T, int TEAM, int CH, int WAVES>
__global__ __launch_bounds__(threads_of(TEAM), WAVES) void loss_kernel(LossArgs a) {
    constexpr int V = kVec<T>, TEAMS = threads_of(TEAM) / TEAM;
    __shared__ float slots[2][16];
    const int lane = threadIdx.x % TEAM;
    for (int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / TEAM; row < a.rows; row += int64_t(gridDim.x) * TEAMS) {
        const T* z = static_cast<const T*>(a.z) + row * a.ld;
        const Span w = span_of(z, a.V, lane);
        piece_t<T, V> x[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (i * TEAM + lane < w.whole) {
                x[i] = *reinterpret_cast<const piece_t<T, V>*>(z + w.head + (i * TEAM + lane) * V);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) x[i][j] = T(kNegInf);
            }
        }
        float last = w.last >= 0 ? float(z[w.last]) : kNegInf;
        const Target t = target_of<T>(a, row, lane == 0);
        float m = last;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i * TEAM < w.whole)
#pragma unroll
                for (int j = 0; j < V; ++j) m = fmaxf(m, float(x[i][j]));
        m = team_max<TEAM>(m, slots[0]);
        m = m == kNegInf ? 0.0f : m;   // a row of nothing else: a sum of 0, lse -inf
        last = exp_of(last, m);
        float s = last;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i * TEAM < w.whole)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float e = exp_of(float(x[i][j]), m);
                    s += e;
                    if constexpr (sizeof(T) == 4) x[i][j] = e;
                }
        s = team_sum<TEAM>(s, slots[1]);
        if (lane == 0) store_row<T>(a, row, t, m, s);
        if (!a.dz) continue;
        T* dz = static_cast<T*>(a.dz) + row * a.ld;
        if (t.at < 0) {
            store_zeros<T, V>(dz, a.V, lane, TEAM);
            continue;
        }
        const float inv = 1.0f / s, k = t.k * inv, hot = (exp_of(t.z, m) * inv - 1.0f) * t.k;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (i * TEAM + lane < w.whole) {
                float e[V];
#pragma unroll
                for (int j = 0; j < V; ++j) e[j] = sizeof(T) == 4 ? float(x[i][j]) : exp_of(float(x[i][j]), m);
                store_slopes<T, V>(dz, w.head + (i * TEAM + lane) * V, e, k, t, hot);
            }
        }
        if (w.last >= 0) dz[w.last] = T(w.last == t.at ? hot : last * k);
    }
}

// Rows beyond what a workgroup's registers hold: the maximum and the sum that
// belongs to it in one pass, the gradient in a second, from the cache where the row is still there. Workgroups of one
// row (grid's y) share the second.
template <typename T>
__global__ __launch_bounds__(1024, 8) void loss_long_kernel(LossArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float slots[2][16];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* z = static_cast<const T*>(a.z) + row * a.ld;
        const Target t = target_of<T>(a, row, blockIdx.y == 0 && threadIdx.x == 0);
        const Span w = span_of(z, a.V, threadIdx.x);
        const float last = w.last >= 0 ? float(z[w.last]) : kNegInf;
        float m = last, s = last == kNegInf ? 0.0f : exp_of(last, m);
        for (int c = threadIdx.x; c < w.whole; c += 1024) {
            const piece_t<T, V> x = *reinterpret_cast<const piece_t<T, V>*>(z + w.head + c * V);
            float top = float(x[0]);
#pragma unroll
            for (int j = 1; j < V; ++j) top = fmaxf(top, float(x[j]));
            if (top > m) {
                s *= exp_of(m, top);
                m = top;
            }
            const float base = m == kNegInf ? 0.0f : m;   // -inf is e^-inf from any base but itself
#pragma unroll
            for (int j = 0; j < V; ++j) s += exp_of(float(x[j]), base);
        }
        const float all = team_max<1024>(m, slots[0]);
        s = team_sum<1024>(m == kNegInf ? s : s * exp_of(m, all), slots[1]);
        if (blockIdx.y == 0 && threadIdx.x == 0) store_row<T>(a, row, t, all, s);
        if (!a.dz) continue;
        T* dz = static_cast<T*>(a.dz) + row * a.ld;
        if (t.at < 0) {
            if (blockIdx.y == 0) store_zeros<T, V>(dz, a.V, threadIdx.x, 1024);
            continue;
        }
        const float inv = 1.0f / s, k = t.k * inv, hot = (exp_of(t.z, all) * inv - 1.0f) * t.k;
        const int part = int(int64_t(w.whole) * blockIdx.y / gridDim.y), end = int(int64_t(w.whole) * (blockIdx.y + 1) / gridDim.y);
        for (int c = part + threadIdx.x; c < end; c += 1024) {
            const piece_t<T, V> x = *reinterpret_cast<const piece_t<T, V>*>(z + w.head + c * V);
            float e[V];
#pragma unroll
            for (int j = 0; j < V; ++j) e[j] = exp_of(float(x[j]), all);
            store_slopes<T, V>(dz, w.head + c * V, e, k, t, hot);
        }
        if (blockIdx.y == 0 && w.last >= 0) dz[w.last] = T(w.last == t.at ? hot : exp_of(last, all) * k);
    }
}

template <typename T>
void launch(dgm_gpu* g, const LossArgs& a) {
    constexpr int V = kVec<T>;
    const auto blocks = [&](int teams) { return dim3(unsigned(std::min<int64_t>((a.rows + teams - 1) / teams, 1 << 20))); };
    const int n = a.V / V;   // whole pieces
    // Lanes to a row. Several rows have to be on a CU at once, some of them being loaded while others are summed and
    // stored, so registers bound the choice (us, gradients): 4096 fp32 rows of 8000 pieces 192 with 1024 lanes (one
    // workgroup), 212 with 512 (two); 8192 bf16 rows of 6282, whose elements are unpacked and raised twice, 356 with
    // 512 and 455 with 1024; 16384 fp32 rows of 2000 192 (512 lanes, 207 with 256), of 250 28 (a wave, 29 with 256); 16384
    // bf16 rows of 937 90 (256 lanes, 102 with 512). Losses alone need no row held: 517 fp32 rows of
    // 8000 15 in the loop below, 18 in registers; 16384 of 1250 111 and 56. bf16 rows of 16032 228 in registers, 258 in the loop.
    // Few long rows: workgroups share a row's gradient, each after the whole row's sum (that of one workgroup is bound by its exponentials,
    // 200,000 fp32 logits 28 us in one, 16 shared; 32 rows of 100,000 20 and 17, 128 of 50,000 12.6 and 13.8). Not where
    // the gradient replaces the logits, which the others still read.
    if (a.dz && a.dz != a.z && n > 4096 && a.rows <= 32) {
        const unsigned parts = unsigned(std::min<int64_t>(dgm::kCus / a.rows, (n + 1023) / 1024));
        loss_long_kernel<T><<<dim3(unsigned(a.rows), parts), dim3(1024), 0, g->stream>>>(a);
        return;
    }
    if (n <= 16) loss_kernel<T, 16, 1, 8><<<blocks(16), dim3(256), 0, g->stream>>>(a);
    else if (n <= 32) loss_kernel<T, 16, 2, 8><<<blocks(16), dim3(256), 0, g->stream>>>(a);
    else if (n <= 128) loss_kernel<T, 64, 2, 8><<<blocks(4), dim3(256), 0, g->stream>>>(a);
    else if (n <= 256) loss_kernel<T, 64, 4, 8><<<blocks(4), dim3(256), 0, g->stream>>>(a);
    else if (n <= 1024) loss_kernel<T, 256, 4, 8><<<blocks(1), dim3(256), 0, g->stream>>>(a);
    else if ((!a.dz && n > 4096) || n > 16384) loss_long_kernel<T><<<blocks(1), dim3(1024), 0, g->stream>>>(a);
    else if (n <= 2048) loss_kernel<T, 256, 8, 6><<<blocks(1), dim3(256), 0, g->stream>>>(a);
    else if (n <= 4096) loss_kernel<T, 512, 8, 6><<<blocks(1), dim3(512), 0, g->stream>>>(a);
    else if (n <= 8192 && sizeof(T) == 4) loss_kernel<T, 1024, 8, 4><<<blocks(1), dim3(1024), 0, g->stream>>>(a);
    else if (n <= 8192) loss_kernel<T, 512, 16, 4><<<blocks(1), dim3(512), 0, g->stream>>>(a);
    else loss_kernel<T, 1024, 16, 4><<<blocks(1), dim3(1024), 0, g->stream>>>(a);
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
    if (cfg->rows > dgm::kMaxIndex || ld > (int64_t(1) << 30))
        return dgm::fail(g, DGM_ERR_UNSUPPORTED, "crossEntropy: rows beyond 2^31 - 1 or a row stride beyond 2^30");
    if (cfg->rows == 0 || (!loss && !lse && !dlogits)) return DGM_OK;
    if (!logits || !targets) return dgm::fail(g, DGM_ERR_ARG, "crossEntropy: null buffer");
    if (loss && loss == lse) return dgm::fail(g, DGM_ERR_ARG, "crossEntropy: loss and lse share memory");
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
