/*
 * dgm_quant.h — C ABI of the MI355X (gfx950) group-quantized linear path.
 *
 * Drop-in for the reference's quantize / group-quant GEMM / STE backward
 * dispatch surface (githubpradeep/diffusion-gpt-metal, paths relative to the
 * reference root). Plain pointers and sizes only: every buffer is device
 * memory owned by the caller, nothing here allocates caller-visible memory,
 * and every call returns an int status (0 = DGM_OK).
 *
 * Layouts are the reference's, unchanged:
 *   W   fp32 master weights [N, K] row-major (output rows x input cols)
 *   Q8  int8 codes [N*K], one byte per weight, codes in [-127, 127]
 *   Q4  int4 codes [N*K/2] bytes, two signed nibbles per byte, even k in the
 *       low nibble, codes in [-7, 7]
 *   S   fp32 scales [N, K/G] row-major, one per (row, group of G along K)
 *   X [M,K], Y [M,N], dY [M,N], dX [M,K], dW [N,K]: fp32 row-major
 *
 * Ordering: one HIP stream per context. Calls are enqueued in issue order
 * (the reference puts a full buffer barrier between dispatches,
 * src/GPU.swift:182-198, which an in-order stream already gives).
 */
#ifndef DGM_QUANT_H
#define DGM_QUANT_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes -------------------------------------------------------- */
#define DGM_OK              0
#define DGM_ERR_ARG         1   /* null pointer / negative size / bad enum     */
#define DGM_ERR_SHAPE       2   /* a reference precondition failed, e.g.
                                   K % qGroup != 0 (src/GPU.swift:229,247) or
                                   odd group for int4 (src/Params.swift:171)  */
#define DGM_ERR_NOT_BEGUN   3   /* dispatch outside begin()/end()
                                   (src/GPU.swift:183)                        */
#define DGM_ERR_HIP         4   /* HIP launch or execution error              */
#define DGM_ERR_BITS        5   /* bits not in {32, 8, 4} (src/GPU.swift:241) */
#define DGM_ERR_UNSUPPORTED 6   /* size beyond what a kernel indexes (2^31)   */

/* ---- math modes (dgm_set_math) ------------------------------------------ */
/* FP32 (default): every result is within max relative error 1e-5 of the
 * float64 product. Quantized forwards of a few rows (M <= 4, and up to
 * M = 16 for weights large enough to split K over the CUs) run on int8 MFMA
 * over an exact split of the activations into four int8 pieces against a
 * power of two per row and k-range (2^-27 of its maximum); other forwards up
 * to M = 64 on f16 MFMA over two f16 pieces per activation against a power
 * of two per (row, 128-k block) (2^-22 of each element; with groups of 32, and
 * int4 groups of 64, also of an element 2^27 below its block's largest, 2^-20
 * at 2^31, and a row of which more than a sixteenth of a block lies below that
 * runs on fp32 operands); large products (from
 * about 0.6 * 2^30 on: the forward, dX and dW) take two f16 pieces of every
 * operand element against a power of two per row of the contraction (2^-23 of
 * each element, and 2^-22 of each product; 2^-20 of an element 2^31 below its
 * row's largest; rows with more than a sixteenth of their nonzero elements
 * below that, or with an infinity or NaN, run on fp32 operands); the rest
 * accumulate fp32 products of fp32 operands.
 * BF16: the int8-piece kernels take two pieces (up to M = 8 when K is
 * split); otherwise up to M = 64, int4 codes
 * meet bf16(x) and int8 codes one f16 piece; larger M (with K % 128 == 0 and
 * qGroup % 32 == 0) runs on bf16 MFMA with activations rounded to bf16 and
 * weights dequantized to bf16 in LDS, fp32 accumulate. Max relative error
 * <= 1e-2. dX and dW are fp32 in both modes. */
#define DGM_MATH_FP32 0
#define DGM_MATH_BF16 1

/* ---- parameter blocks: src/Params.swift:7-23, metal/kernels.metal:22-29 -- */
typedef struct dgm_GemmP {
    uint32_t M, N, K, hasBias, qGroup, pad0, pad1, pad2;
} dgm_GemmP;                                   /* 32 bytes (src/GPU.swift:455) */

typedef struct dgm_QuantP {
    uint32_t rows, cols;
    float qmax;                                /* 127 (int8) or 7 (int4)       */
    uint32_t qGroup;
} dgm_QuantP;                                  /* 16 bytes (src/GPU.swift:456) */

/* ---- context: src/GPU.swift:91-198 (class GPU) --------------------------- */
typedef struct dgm_gpu dgm_gpu;

/* GPU.init (src/GPU.swift:118-156): binds the current HIP device and creates
 * the context's own stream. */
int dgm_gpu_create(dgm_gpu** out);
/* Waits for the work queued on the context's own stream and on every stream
 * it was set to (so those must still exist; after more than 16 distinct
 * streams, for the whole device), then frees its workspace. Graphs captured
 * from calls on the context read that workspace: they must not be replayed
 * after the context is destroyed. Other streams are not synchronized, so a
 * capture in progress elsewhere is undisturbed. */
void dgm_gpu_destroy(dgm_gpu* g);
/* Use a caller-owned stream (e.g. a framework's current stream) instead of the
 * context's own; NULL restores the context's stream. */
int dgm_gpu_set_stream(dgm_gpu* g, void* hip_stream);
void* dgm_gpu_stream(const dgm_gpu* g);
/* The context's device, -1 without one. */
int dgm_gpu_device(const dgm_gpu* g);
int dgm_set_math(dgm_gpu* g, int mode);
int dgm_get_math(const dgm_gpu* g);

/* GPU.begin (src/GPU.swift:158-166): opens a dispatch region. */
int dgm_begin(dgm_gpu* g);
/* GPU.end (src/GPU.swift:168-180): waits for the region's work and returns the
 * first error of the region (the reference prints it with lastKernel and
 * exits; callers turn a nonzero status into their own fatal error). This
 * includes DGM_ERR_HIP when a decode kernel of the region gave up one of its
 * bounded in-workgroup waits, whose results are then not valid (the flag is
 * per device: with several contexts on one device, the first end() that
 * follows reports it). */
int dgm_end(dgm_gpu* g);
/* GPU.lastKernel (src/GPU.swift:99): name of the last dispatched kernel. */
const char* dgm_last_kernel(const dgm_gpu* g);
/* Human-readable text of the context's last error ("" when none). */
const char* dgm_last_error(const dgm_gpu* g);

/* ---- kernel-level entry points: buffer slot order of metal/kernels.metal -- */

/* quant_i8 (metal/kernels.metal:79-98): W f32 -> Q i8 codes, S f32 scales. */
int dgm_quant_i8(dgm_gpu* g, const float* W, int8_t* Q, float* scale,
                 const dgm_QuantP* p);
/* quant_i4 (metal/kernels.metal:100-124): W f32 -> packed nibbles, S. */
int dgm_quant_i4(dgm_gpu* g, const float* W, uint8_t* Q, float* scale,
                 const dgm_QuantP* p);

/* gemm_nt_f32 (metal/kernels.metal:128-150): Y = X W^T (+bias). */
int dgm_gemm_nt_f32(dgm_gpu* g, const float* W, const float* X,
                    const float* bias, float* Y, const dgm_GemmP* p);
/* gemm_nt_i8 (metal/kernels.metal:152-178): Y = X dequant(Q8,S)^T (+bias). */
int dgm_gemm_nt_i8(dgm_gpu* g, const int8_t* W, const float* scale,
                   const float* X, const float* bias, float* Y,
                   const dgm_GemmP* p);
/* gemm_nt_i4 (metal/kernels.metal:180-209): Y = X dequant(Q4,S)^T (+bias). */
int dgm_gemm_nt_i4(dgm_gpu* g, const uint8_t* W, const float* scale,
                   const float* X, const float* bias, float* Y,
                   const dgm_GemmP* p);

/* gemm_dx_f32 (metal/kernels.metal:211-224): dX = dY W. */
int dgm_gemm_dx_f32(dgm_gpu* g, const float* W, const float* dY, float* dX,
                    const dgm_GemmP* p);
/* gemm_dx_i8 (metal/kernels.metal:226-246): STE dX = dY dequant(Q8,S). */
int dgm_gemm_dx_i8(dgm_gpu* g, const int8_t* W, const float* scale,
                   const float* dY, float* dX, const dgm_GemmP* p);
/* gemm_dx_i4 (metal/kernels.metal:248-268): STE dX = dY dequant(Q4,S). */
int dgm_gemm_dx_i4(dgm_gpu* g, const uint8_t* W, const float* scale,
                   const float* dY, float* dX, const dgm_GemmP* p);

/* gemm_dw (metal/kernels.metal:270-283): dW = dY^T X, overwrite. */
int dgm_gemm_dw(dgm_gpu* g, const float* dY, const float* X, float* dW,
                const dgm_GemmP* p);
/* gemm_dw_acc (metal/kernels.metal:1014-1027): dW += dY^T X. */
int dgm_gemm_dw_acc(dgm_gpu* g, const float* dY, const float* X, float* dW,
                    const dgm_GemmP* p);

/* ---- host call surface: src/GPU.swift:220-272 ----------------------------
 * Same names and argument meaning as the Swift wrappers. Sizes are Swift Int
 * (int64_t). q is int8_t* for bits 8, uint8_t* for bits 4; w is read only
 * when bits == 32. bias may be NULL (the reference binds a dummy buffer and
 * sets hasBias = 0). */

/* GPU.quantize (src/GPU.swift:220-225): qmax = 7 for bits 4, else 127. */
int dgm_quantize(dgm_gpu* g, const float* w, void* q, float* scale,
                 int64_t rows, int64_t cols, int64_t bits, int64_t qGroup);
/* GPU.gemmNT (src/GPU.swift:227-243). */
int dgm_gemmNT(dgm_gpu* g, int64_t bits, const float* w, const void* q,
               const float* scale, const float* x, const float* bias, float* y,
               int64_t M, int64_t N, int64_t K, int64_t qGroup);
/* No counterpart in the reference: dgm_gemmNT for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). Same arguments, kernels and results
 * (bitwise; where dgm_gemmNT takes the f16 pieces of large products, or cuts
 * a long K at 17 to 64 rows into slices whose sums do not fit the scratch,
 * this entry takes the kernels without that staging, within the same 1e-5)
 * as dgm_gemmNT, but every staging buffer (the decode kernels'
 * activation pieces, the bf16 copy of X of the reduced-precision prefill
 * path) comes from a static device scratch of DGM_NOALLOC_SCRATCH_BYTES per
 * GPU, held from library load until the process ends; nothing is allocated.
 * A call that would need more scratch returns DGM_ERR_UNSUPPORTED before
 * launching anything (dgm_gemmNT_workspace_bound gives the most a call can
 * need: at most 260 * K + 512 bytes at M <= 64, the K-sliced path's partial
 * sums up to all of the scratch at M <= 16, the bf16 prefill path 2 * M * K
 * bytes). Every such call on one GPU shares
 * that scratch, which keeps the last call's contents (no kernel relies on it
 * starting at zero): calls that overlap in time on one GPU (other streams,
 * other contexts, other threads) race and must be serialized by the caller. */
#define DGM_NOALLOC_SCRATCH_BYTES (8u << 20)
int dgm_gemmNT_noalloc(dgm_gpu* g, int64_t bits, const float* w, const void* q,
                       const float* scale, const float* x, const float* bias, float* y,
                       int64_t M, int64_t N, int64_t K, int64_t qGroup);
/* No counterpart in the reference, whose buffers are all allocated at setup
 * (src/GPU.swift:31-88; its kernels never allocate). dgm_gemmNT's staging
 * buffers (activation pieces of the decode-shaped kernels, partial sums of the
 * K-sliced kernel, the bf16 copy of X of the prefill path) come from a
 * workspace of the context that is otherwise allocated by the first call that
 * needs it; the f16 pieces of large products (dX and dW among them) from a
 * second buffer of the context, which calls under graph capture do not use
 * (they, and calls for which no memory is left, take the kernels that stage
 * nothing). A call on another stream than the last one to use that buffer
 * waits for that one. dgm_gemmNT_workspace_bound returns bytes that cover what
 * a dgm_gemmNT call of that shape cannot do without, on any path, in either
 * math mode; dgm_gemm_staging_bound (never less) also what makes it, and
 * dgm_gemmDX, dgm_gemmDW and dgm_gemmBwd of the shape, faster: the f16 pieces of large
 * products and, at up to 64 rows, the sums of slices of K (both -1 for negative
 * sizes). dgm_gpu_reserve grows both buffers to at least `bytes` now, and then
 * they grow by a reserve only, but for staging that a call cannot do without:
 * later calls whose bound it covers allocate nothing, and those whose staging
 * bound it covers run the kernels that they run on a context without a reserve;
 * the others take kernels that stage less (for large products the fp32 ones,
 * several times slower). A reserve that cannot grow a buffer leaves the context as it
 * was: DGM_ERR_UNSUPPORTED during a graph capture, DGM_ERR_HIP without the
 * memory; one of 0 bytes does nothing. dgm_gpu_workspace_bytes returns the size
 * of the larger buffer (0 before anything was allocated). */
int64_t dgm_gemmNT_workspace_bound(int64_t M, int64_t N, int64_t K);
int64_t dgm_gemm_staging_bound(int64_t M, int64_t N, int64_t K);
int dgm_gpu_reserve(dgm_gpu* g, int64_t bytes);
int64_t dgm_gpu_workspace_bytes(const dgm_gpu* g);
/* GPU.gemmDX (src/GPU.swift:245-260). */
int dgm_gemmDX(dgm_gpu* g, int64_t bits, const float* w, const void* q,
               const float* scale, const float* dy, float* dx,
               int64_t M, int64_t N, int64_t K, int64_t qGroup);
/* GPU.gemmDW (src/GPU.swift:262-266). */
int dgm_gemmDW(dgm_gpu* g, const float* dy, const float* x, float* dw,
               int64_t M, int64_t N, int64_t K);
/* GPU.gemmDWAcc (src/GPU.swift:268-272). */
int dgm_gemmDWAcc(dgm_gpu* g, const float* dy, const float* x, float* dw,
                  int64_t M, int64_t N, int64_t K);

/* GPU.gemmDW (accumulate = 0) or GPU.gemmDWAcc (accumulate != 0) followed by
 * GPU.gemmDX with the same dY: the pair the reference's backward issues back
 * to back for every linear (src/GPT.swift:374-376, 384-420). One launch when
 * the shapes allow (the dX and dW tiles run side by side), else the two
 * calls; either way dx and dw are bitwise what the two calls produce on the
 * same context at the same time (under capture, or under a reserve that has no
 * room for operand pieces, those differ from an eager call's). */
int dgm_gemmBwd(dgm_gpu* g, int64_t bits, const float* w, const void* q, const float* scale,
                const float* dy, const float* x, float* dx, float* dw, int64_t M, int64_t N,
                int64_t K, int64_t qGroup, int accumulate);

/* ---- looped DiT block forward: the non-GEMM wrappers it calls -------------
 * Same names, buffer order and sizes as the Swift wrappers; fp32 buffers in
 * device memory. Layouts: activations [B,T,H,D] (rows of H*D), scores/probs
 * [B,H,T,T], RoPE tables [T,D]. */

/* GPU.rmsFwd (src/GPU.swift:364-367; rmsnorm_fwd, metal/kernels.metal:807-825):
 * y = x * rsqrt(mean(x^2) + eps) * weight per row; rstd[row] = that rsqrt
 * (rstd may be NULL). */
int dgm_rmsFwd(dgm_gpu* g, const float* x, float* y, float* rstd, const float* weight,
               int64_t rows, int64_t cols, float eps);
/* GPU.ropeFwd (src/GPU.swift:375-378; rope_fwd, metal/kernels.metal:871-889):
 * rotate-half RoPE; D must be even. */
int dgm_ropeFwd(dgm_gpu* g, const float* x, float* y, const float* cos_t, const float* sin_t,
                int64_t B, int64_t T, int64_t H, int64_t D);
/* GPU.repeatHeads (src/GPU.swift:407-410; repeat_heads, metal/kernels.metal:980-993):
 * dst[b,t,h,:] = src[b,t,:]. */
int dgm_repeatHeads(dgm_gpu* g, const float* src, float* dst, int64_t B, int64_t T, int64_t H,
                    int64_t D);
/* GPU.attnFwd (src/GPU.swift:302-310; attn_scores/attn_softmax/attn_av,
 * metal/kernels.metal:443-506), one fused kernel: scores = q.k / sqrt(D)
 * (masked to -1e30 above the diagonal when causal), probs = row softmax,
 * av = probs.v. Needs (2*T*D + 16*D + 16*T)*4 bytes <= 160 KiB of LDS. */
int dgm_attnFwd(dgm_gpu* g, const float* q, const float* k, const float* v, float* scores,
                float* probs, float* av, int64_t B, int64_t T, int64_t H, int64_t D, int causal);
/* GPU.swigluFwd (src/GPU.swift:385-387; swiglu_fwd, metal/kernels.metal:911-930):
 * y = gate * sigmoid(gate) * up. */
int dgm_swigluFwd(dgm_gpu* g, const float* gate, const float* up, float* y, int64_t n);
/* GPU.add (src/GPU.swift:211-213; add_f, metal/kernels.metal:419-427): y = a + b. */
int dgm_add(dgm_gpu* g, const float* a, const float* b, float* y, int64_t n);
/* GPU.mix (src/GPU.swift:393-396; mix_f, metal/kernels.metal:951-959): y = ca*a + cb*b. */
int dgm_mix(dgm_gpu* g, const float* a, const float* b, float* y, int64_t n, float ca, float cb);
/* GPU.copy (src/GPU.swift:398-400; copy_f, metal/kernels.metal:961-968): y = x. */
int dgm_copy(dgm_gpu* g, const float* x, float* y, int64_t n);

/* ropeTables (src/Macro.swift:509-530), host side: fills cos_t/sin_t, each
 * maxT*dim floats of HOST memory, with cos/sin(t * theta^(-2i/dim)) for
 * i < dim/2, repeated in both halves of each row. dim must be even. */
int dgm_ropeTables(int64_t maxT, int64_t dim, float theta, float* cos_t, float* sin_t);

/* The DiT block configuration the loop body reads (src/DiT.swift:9-41):
 * B sequences of T tokens, embd C = H*D, SwiGLU width F, one KV head of
 * width D repeated to H heads. bits 8 / 4 route every linear through the
 * group-quantized forward (group `group`); bits 32 uses the fp32 weights. */
typedef struct dgm_dit_cfg {
    int32_t B, T, C, F, H, D, loops, group, bits;
    float eps, mix;
    int32_t pad;
} dgm_dit_cfg;

/* One linear: fp32 weight w [N,K] (bits 32) or codes q + scales (bits 8/4). */
typedef struct dgm_dit_linear {
    const float* w;
    const void* q;
    const float* scale;
} dgm_dit_linear;

/* The block's parameters (src/DiT.swift:242-253): wq [C,C], wk/wv [D,C],
 * wo [C,C], wgate/wup [F,C], wdown [C,F]; RMSNorm weights of C floats. */
typedef struct dgm_dit_weights {
    dgm_dit_linear wq, wk, wv, wo, wgate, wup, wdown;
    const float *n1, *n1b, *n2, *n2b, *nf;
} dgm_dit_weights;

/* Floats of device workspace for dgm_dit_forward of cfg (-1 for NULL): what
 * it needs and, where a linear of the block is a large product, room behind
 * that for its operand pieces (a workspace without the room is accepted: those
 * linears then run on the fp32 kernels). dgm_dit_acts_floats and
 * dgm_dit_backward_ws_floats count the same way. */
int64_t dgm_dit_workspace_floats(const dgm_dit_cfg* cfg);
/* The looped block forward (src/DiT.swift:520-550): x holds xs[0] [B*T, C] on
 * entry and xs[loops] on exit. cos_t/sin_t are device copies of
 * ropeTables(T, D, theta). ws: device workspace of at least
 * dgm_dit_workspace_floats(cfg) floats; on exit it holds the last loop's
 * intermediates (projections, scores and probs [B,H,T,T], attention output,
 * residual stream, SwiGLU input and output). When wq, wk, wv (and wgate,
 * wup) are laid out back to back in memory (codes and scales, or fp32
 * weights), each group runs as one GEMM. RoPE, the value-residual mix and the
 * KV-head broadcast are applied inside the attention kernel, and each
 * RMSNorm + residual chain is one row kernel; every element is computed as
 * the standalone wrappers compute it. Needs T and D multiples of 16 and
 * C <= 1024 (DGM_ERR_UNSUPPORTED otherwise); x, ws and the tables 16-byte
 * aligned. Enqueued on the context's
 * stream; graph-capturable (no host sync, and no allocation for more than 64
 * tokens in all in the fp32 mode; fewer tokens and the reduced-precision mode
 * stage through the context's workspace, as dgm_gemmNT of these shapes does). */
int dgm_dit_forward(dgm_gpu* g, const dgm_dit_cfg* cfg, const dgm_dit_weights* w,
                    const float* cos_t, const float* sin_t, float* x, float* ws,
                    int64_t ws_floats);

/* ---- looped DiT block backward (src/DiT.swift:558-626) ---------------------
 * The wrappers the backward loop calls, with the Swift names and buffer
 * order, then a forward that saves every loop's activations and the block
 * backward. */

/* GPU.rmsBwd (src/GPU.swift:369-373; rmsnorm_bwd_dx / rmsnorm_bwd_dw,
 * metal/kernels.metal:827-868): dx per row from the saved rstd, and
 * dweight[c] += sum over rows of dy*x*rstd (the weight is shared by every
 * loop). eps is accepted for the signature and unused, as in the reference. */
int dgm_rmsBwd(dgm_gpu* g, const float* x, const float* rstd, const float* weight, const float* dy,
               float* dx, float* dweight, int64_t rows, int64_t cols, float eps);
/* GPU.attnBwd (src/GPU.swift:312-322; attn_bwd_dv, attn_bwd_dp,
 * attn_softmax_bwd, attn_bwd_dq, attn_bwd_dk, metal/kernels.metal:508-612):
 * q, k, v, dout, dq, dk, dv [B,T,H,D]; probs, dprobs, dscores [B,H,T,T]. */
int dgm_attnBwd(dgm_gpu* g, const float* q, const float* k, const float* v, const float* probs,
                const float* dout, float* dq, float* dk, float* dv, float* dprobs, float* dscores,
                int64_t B, int64_t T, int64_t H, int64_t D);
/* GPU.ropeBwd (src/GPU.swift:380-383; rope_bwd, metal/kernels.metal:891-909). */
int dgm_ropeBwd(dgm_gpu* g, const float* dy, float* dx, const float* cos_t, const float* sin_t,
                int64_t B, int64_t T, int64_t H, int64_t D);
/* GPU.swigluBwd (src/GPU.swift:389-391; swiglu_bwd, metal/kernels.metal:932-949). */
int dgm_swigluBwd(dgm_gpu* g, const float* gate, const float* up, const float* dy, float* dgate,
                  float* dup, int64_t n);
/* GPU.sumHeads (src/GPU.swift:412-415; sum_heads, metal/kernels.metal:995-1010):
 * dst[b,t,:] = sum over h of src[b,t,h,:]. */
int dgm_sumHeads(dgm_gpu* g, const float* src, float* dst, int64_t B, int64_t T, int64_t H, int64_t D);
/* GPU.acc / GPU.accScale (src/GPU.swift:216-218, 402-405; acc_f, acc_scale_f,
 * metal/kernels.metal:429-436, 970-977): a += b, a += s*b. */
int dgm_acc(dgm_gpu* g, float* a, const float* b, int64_t n);
int dgm_accScale(dgm_gpu* g, float* a, const float* b, int64_t n, float s);

/* Gradients of the block's parameters, fp32, accumulated (+=): the seven
 * linears [N,K] as in dgm_dit_weights and the five RMSNorm weights [C]. */
typedef struct dgm_dit_grads {
    float *wq, *wk, *wv, *wo, *wgate, *wup, *wdown;
    float *n1, *n1b, *n2, *n2b, *nf;
} dgm_dit_grads;

/* Floats of the activation buffer dgm_dit_forward_train fills (-1 for NULL). */
int64_t dgm_dit_acts_floats(const dgm_dit_cfg* cfg);
/* Floats of workspace dgm_dit_backward needs (-1 for NULL). */
int64_t dgm_dit_backward_ws_floats(const dgm_dit_cfg* cfg);
/* The loop body of DiT.forward (src/DiT.swift:520-550) with every loop's
 * activations saved in acts (the reference's Acts): x holds xs[0] on entry
 * and xs[loops] on exit. Linears as in dgm_dit_forward (bits 32: fp32
 * weights; bits 8 / 4: codes + scales). */
int dgm_dit_forward_train(dgm_gpu* g, const dgm_dit_cfg* cfg, const dgm_dit_weights* w,
                          const float* cos_t, const float* sin_t, float* x, float* acts,
                          int64_t acts_floats);
/* The loop part of DiT.backward (src/DiT.swift:566-626) over the activations
 * of dgm_dit_forward_train: gx holds dL/dxs[loops] on entry and dL/dxs[0] on
 * exit; the parameter gradients are added into *grads. bits 32 runs dX on
 * the fp32 weights, as the reference does; bits 8 / 4 run it through the
 * dequantized codes (straight-through estimator) and dW into the fp32
 * gradients. ws: dgm_dit_backward_ws_floats(cfg) floats. */
int dgm_dit_backward(dgm_gpu* g, const dgm_dit_cfg* cfg, const dgm_dit_weights* w,
                     const dgm_dit_grads* grads, const float* cos_t, const float* sin_t,
                     const float* acts, int64_t acts_floats, float* gx, float* ws,
                     int64_t ws_floats);

/* ---- training step around the path: optimizer, re-quantize, embedding ----
 * GPT.step (src/GPT.swift:183-220) zeroes the grads, runs the backward, sums
 * the squared grads for clipping, scales them, applies AdamW to every master
 * weight and re-quantizes the quantized ones; the quantized GPT's token
 * embedding is the other consumer of the codes (src/GPT.swift:332-336,
 * 371-376, 425-429). Parameter blocks are the reference's (src/Params.swift). */

typedef struct dgm_AdamP {                     /* src/Params.swift:138-147      */
    uint32_t n;
    float lr, b1, b2, eps, wd, invBC1, invBC2;
} dgm_AdamP;                                   /* 32 bytes (src/GPU.swift:469)  */
typedef struct dgm_EmbP { uint32_t B, T, C, qGroup; } dgm_EmbP;       /* :78-83   */
typedef struct dgm_EmbBwdP { uint32_t B, T, C, V; } dgm_EmbBwdP;      /* :85-90   */
typedef struct dgm_PosP { uint32_t B, T, C, pad; } dgm_PosP;          /* :92-97   */
typedef struct dgm_BiasP { uint32_t M, N, pad0, pad1; } dgm_BiasP;    /* :46-51   */
typedef struct dgm_ReduceP { uint32_t n, slot, pad0, pad1; } dgm_ReduceP; /* :106-111 */
typedef struct dgm_ScaleP { uint32_t n; float s; uint32_t pad0, pad1; } dgm_ScaleP; /* :39-44 */
typedef struct dgm_UnaryP { uint32_t n, pad0, pad1, pad2; } dgm_UnaryP; /* :32-37  */

/* adamw (metal/kernels.metal:786-802), per element i < n:
 *   m = b1*m + (1-b1)*g;  v = b2*v + (1-b2)*g*g;
 *   w -= lr * ((m*invBC1) / (sqrt(v*invBC2) + eps) + wd*w)
 * each operation rounded to fp32 separately (no fused multiply-add). */
int dgm_adamw(dgm_gpu* g, float* w, const float* grad, float* m, float* v, const dgm_AdamP* p);
/* GPU.adam (src/GPU.swift:425-429). */
int dgm_adam(dgm_gpu* g, float* w, const float* grad, float* m, float* v, int64_t n,
             float lr, float b1, float b2, float eps, float wd, float invBC1, float invBC2);
/* GPU.adam followed by GPU.quantize of the same master (the quantized
 * parameters of src/GPT.swift:214-217 then quantizeAll, 441-447), in one pass
 * over the [rows, cols] master when cols % qGroup == 0 and qGroup is a power
 * of two in [8, 512]: w, m, v, q and scale come out bit-identical to the two
 * calls (which run instead for any other shape). No single reference
 * counterpart; it replaces that pair of dispatches. */
int dgm_adam_quantize(dgm_gpu* g, float* w, const float* grad, float* m, float* v, void* q,
                      float* scale, int64_t rows, int64_t cols, int64_t bits, int64_t qGroup,
                      float lr, float b1, float b2, float eps, float wd, float invBC1,
                      float invBC2);

/* reduce_sumsq (metal/kernels.metal:749-768): out[slot] = sum of x[i]^2,
 * i < n. The sum is taken in a fixed order of this library's own (per-block
 * partial sums over contiguous ranges, then a tree), so repeated calls give
 * identical bits; it agrees with the reference's 256-lane order to fp32
 * rounding, not bitwise. */
int dgm_reduce_sumsq(dgm_gpu* g, const float* x, float* out, const dgm_ReduceP* p);
/* GPU.reduceSumsq (src/GPU.swift:420-422). */
int dgm_reduceSumsq(dgm_gpu* g, const float* x, float* into, int64_t n, int64_t slot);
/* zero_f / scale_f (metal/kernels.metal:770-784); GPU.zero / GPU.scale
 * (src/GPU.swift:200-209). */
int dgm_zero_f(dgm_gpu* g, float* x, const dgm_UnaryP* p);
int dgm_scale_f(dgm_gpu* g, float* x, const dgm_ScaleP* p);
int dgm_zero(dgm_gpu* g, float* x, int64_t n);
int dgm_scale(dgm_gpu* g, float* x, int64_t n, float s);

/* embed_f32 / embed_i8 / embed_i4 (metal/kernels.metal:616-663):
 * y[bt, c] = wte[tok, c] + wpe[bt % T, c], with wte dequantized as
 * code * scale[tok, c / qGroup] for the quantized forms (rounded, then
 * added). tokens are uint32 ids < the table's rows (not checked). */
int dgm_embed_f32(dgm_gpu* g, const uint32_t* tokens, const float* wte, const float* wpe,
                  float* y, const dgm_EmbP* p);
int dgm_embed_i8(dgm_gpu* g, const uint32_t* tokens, const int8_t* wte, const float* scale,
                 const float* wpe, float* y, const dgm_EmbP* p);
int dgm_embed_i4(dgm_gpu* g, const uint32_t* tokens, const uint8_t* wte, const float* scale,
                 const float* wpe, float* y, const dgm_EmbP* p);
/* GPU.embed (src/GPU.swift:324-338): bits selects the kernel; wte is read
 * for bits 32, q and scale for bits 8 / 4. */
int dgm_embed(dgm_gpu* g, int64_t bits, const uint32_t* tokens, const float* wte, const void* q,
              const float* scale, const float* wpe, float* y, int64_t B, int64_t T, int64_t C,
              int64_t qGroup);
/* embed_bwd (metal/kernels.metal:665-682): dwe[v, c] += sum over bt with
 * tokens[bt] == v of dx[bt, c], summed in increasing bt (the reference's
 * order, so results are bitwise the reference's). Every row v < V is
 * rewritten. */
int dgm_embed_bwd(dgm_gpu* g, const uint32_t* tokens, const float* dx, float* dwe,
                  const dgm_EmbBwdP* p);
/* GPU.embedBwd (src/GPU.swift:340-344). */
int dgm_embedBwd(dgm_gpu* g, const uint32_t* tokens, const float* dx, float* dwe, int64_t B,
                 int64_t T, int64_t C, int64_t V);
/* pos_bwd (metal/kernels.metal:684-697): dwp[t, c] = sum over b (increasing)
 * of dx[b*T + t, c]; overwrites. */
int dgm_pos_bwd(dgm_gpu* g, const float* dx, float* dwp, const dgm_PosP* p);
/* GPU.posBwd (src/GPU.swift:346-350). */
int dgm_posBwd(dgm_gpu* g, const float* dx, float* dwp, int64_t B, int64_t T, int64_t C);
/* bias_grad (metal/kernels.metal:285-295): db[n] = sum over m (increasing) of
 * dY[m, n]; overwrites. */
int dgm_bias_grad(dgm_gpu* g, const float* dY, float* db, const dgm_BiasP* p);
/* GPU.biasGrad (src/GPU.swift:274-277). */
int dgm_biasGrad(dgm_gpu* g, const float* dy, float* db, int64_t M, int64_t N);

/* ---- attention over packed sequences, and over a paged cache ----------------
 * No counterpart in the reference, whose attention (dgm_attnFwd, dgm_attnBwd)
 * takes equal lengths and heads and writes out [B,H,T,T] scores. Here
 * sequences of any lengths lie back to back, H query heads share KVH key and value
 * heads (query head h reads key head h / (H / KVH)), no score reaches memory, and
 * keys and values of past tokens can be kept in pages.
 *
 * Types: DGM_TYPE_F32 or DGM_TYPE_BF16. Scores, softmax statistics and sums
 * are fp32 for both; for bf16 the probabilities are rounded to bf16 between the
 * two products. dgm_set_math does not change these calls.
 *
 * Sequence starts, lengths and page tables are read on the device only, so that
 * captured graphs can be replayed with other ones. Where they are wrong (starts out of
 * order or beyond the rows, a page that the cache does not have, a length beyond
 * the page table) nothing outside the buffers is touched, and the context's next
 * dgm_end (after a replay of a graph captured with the context, too) returns DGM_ERR_SHAPE.
 *
 * Buffers 16-byte aligned (starts, lengths, pages, lse: 4), row strides
 * multiples of 8 elements and at least the row's heads, 0 for rows back to back;
 * D a multiple of 8 up to 256 (DGM_ERR_UNSUPPORTED otherwise). DGM_ERR_UNSUPPORTED
 * too beyond 2^30 rows, for packed rows beyond 2^23 elements apart, other rows beyond 2^31, for
 * caches of 2^31 rows (page x key head x slot) or more, beyond 65536 sequences in a cache or
 * 2^22 of its sequences x query heads, and where one launch cannot hold the work. Outputs must
 * not overlap inputs or one another, except that strided rows may interleave
 * (q, k, v of one fused projection, dq, dk, dv of its gradient). Nothing is allocated, and
 * every call can be captured. Results are the same bits every time. */
#define DGM_TYPE_F32  0
#define DGM_TYPE_BF16 1

typedef struct dgm_attn_cfg {
    int32_t type;                  /* DGM_TYPE_* of q, k, v, out and gradients  */
    int32_t H, KVH, D;             /* H % KVH == 0                              */
    int32_t causal;                /* query i of a sequence sees keys 0 .. i    */
    float scale;                   /* of the scores, > 0 (1 / sqrt(D))          */
    int64_t rows, nseq;
    int64_t ldq, ldk, ldv, ldo;    /* row strides in elements; dq, dk, dv have
                                      those of q, k, v, and dout that of out    */
} dgm_attn_cfg;

/* out[r, h, :] = softmax(scale * q[r, h] . k[j, h']) v[j, h'] over the keys j of
 * row r's sequence (up to r when causal). starts: int32 [nseq + 1], sequence s
 * is rows starts[s] .. starts[s + 1] - 1 (none when they are equal); rows before the first
 * and behind the last sequence are left as they were. lse (may be NULL; the
 * backward reads it): float [H, rows], the base-2 logarithm of the row's sum
 * of 2^(score * log2 e). A masked position takes no part whatever its
 * values; an infinity or NaN elsewhere makes what it enters infinite or NaN. */
int dgm_attnPackedFwd(dgm_gpu* g, const dgm_attn_cfg* cfg, const void* q, const void* k, const void* v,
                      const int32_t* starts, void* out, float* lse);
/* The gradients of dgm_attnPackedFwd from its out and lse and from dout = dL/dout:
 * dq [rows, H, D], dk and dv [rows, KVH, D] (summed over the query heads of a key
 * head), overwritten where a sequence has rows. D up to 128. ws: device memory
 * of at least dgm_attnPackedBwd_ws_bytes(cfg) bytes (-1 for sizes that are
 * refused), 16-byte aligned; calls that overlap in time need one each. */
int64_t dgm_attnPackedBwd_ws_bytes(const dgm_attn_cfg* cfg);
int dgm_attnPackedBwd(dgm_gpu* g, const dgm_attn_cfg* cfg, const void* q, const void* k, const void* v,
                      const int32_t* starts, const void* out, const float* lse, const void* dout, void* dq,
                      void* dk, void* dv, void* ws, int64_t ws_bytes);

/* A cache of keys and one of values, each [numPages, KVH, pageSize, D]. Sequence
 * s keeps position p at slot p % pageSize of page pages[s * maxPages + p / pageSize]
 * (int32; entries that no position needs are not read). */
typedef struct dgm_cache_cfg {
    int32_t type;                  /* DGM_TYPE_* of the caches                  */
    int32_t KVH, D, pageSize;
    int64_t numPages, maxPages;    /* pages of the cache; columns of the table  */
} dgm_cache_cfg;

/* Writes rows of k and v [rows, KVH, D] of type `type` into the caches (rounded
 * to the nearest, ties to even, where those are bf16): row r of sequence s
 * becomes position lens[s] + r - starts[s]. lens (int32 [nseq], tokens that s
 * had before) may be NULL for all 0; starts as above, or NULL for one row per
 * sequence (rows == nseq). Rows whose position the table does not hold are left
 * out (and reported by dgm_end). No two rows of a call may meet in one slot (a page
 * named twice): its elements could be of either. */
int dgm_cacheWrite(dgm_gpu* g, const dgm_cache_cfg* cfg, int64_t type, const void* k, const void* v,
                   const int32_t* starts, const int32_t* lens, const int32_t* pages, void* kcache, void* vcache,
                   int64_t rows, int64_t nseq, int64_t ldk, int64_t ldv);
/* One new token per sequence over its cache: out[s, h, :] = softmax(scale *
 * q[s, h] . k_j) v_j over positions j < lens[s] (the new token's own, already
 * written, among them); zeros where none is left. q, out [nseq, H, D] of type
 * `type`. Positions that the table does not hold are left out (and
 * reported by dgm_end). ws: device memory of at least
 * dgm_attnPagedDecode_ws_bytes bytes (-1 for sizes that are refused), 16-byte
 * aligned; calls that overlap in time need one each. */
int64_t dgm_attnPagedDecode_ws_bytes(const dgm_cache_cfg* cfg, int64_t nseq, int64_t H);
int dgm_attnPagedDecode(dgm_gpu* g, const dgm_cache_cfg* cfg, int64_t type, const void* q, const void* kcache,
                        const void* vcache, const int32_t* pages, const int32_t* lens, void* out, void* ws,
                        int64_t ws_bytes, int64_t nseq, int64_t H, int64_t ldq, int64_t ldo, float scale);

/* ---- a training step around its linears ---------------------------------------
 * No counterpart among the reference's wrappers: what a language model's step
 * needs between its linears and attention. Rows lie back to back and may have any
 * length; buffers are aligned to their elements (workspaces and plans: 16 bytes).
 * Types: DGM_TYPE_F32 or DGM_TYPE_BF16; sums, statistics and parameters are fp32.
 * Tokens, targets and plans are read on the device only; a token or target beyond
 * the vocabulary is left out, and the context's next dgm_end returns
 * DGM_ERR_SHAPE. Outputs must not overlap inputs or one another unless said so.
 * Nothing is allocated, every call but dgm_adamMany_plan can be captured, and
 * results are the same bits every time. Calls that overlap in time need a
 * workspace each. DGM_ERR_UNSUPPORTED for sizes beyond those named, and where one
 * launch cannot hold the work. */

typedef struct dgm_norm_cfg {
    int32_t type;                  /* DGM_TYPE_* of the rows                    */
    float eps;                     /* >= 0                                      */
    int64_t rows, cols;            /* rows up to 2^31 - 1, cols up to 16384     */
} dgm_norm_cfg;

/* sum = x + res (rounded to the rows' type; res and sum may both be NULL: x
 * itself), y = (sum - mean) * rstd * weight + bias with each row's mean and rstd
 * = 1 / sqrt(variance + eps). bias, mean and rstd (float [rows], for a backward)
 * may be NULL. sum may be x or res itself, and y what is read no more. */
int dgm_layerNormFwd(dgm_gpu* g, const dgm_norm_cfg* cfg, const void* x, const void* res, const float* weight,
                     const float* bias, void* sum, void* y, float* mean, float* rstd);
/* From the rows that were normalised (x, or sum) and their mean and rstd: dx =
 * dsum + the gradient through the norm (dsum: what reaches the sum by another
 * way, may be NULL, may be dx itself), dweight += and dbias += (either may be
 * NULL). ws: at least dgm_layerNormBwd_ws_bytes(cfg) bytes (-1 for sizes that are
 * refused). */
int64_t dgm_layerNormBwd_ws_bytes(const dgm_norm_cfg* cfg);
int dgm_layerNormBwd(dgm_gpu* g, const dgm_norm_cfg* cfg, const void* x, const float* mean, const float* rstd,
                     const float* weight, const void* dy, const void* dsum, void* dx, float* dweight, float* dbias,
                     void* ws, int64_t ws_bytes);

typedef struct dgm_loss_cfg {
    int32_t type;                  /* DGM_TYPE_* of logits and their gradient   */
    float scale;                   /* of the gradient (1 / rows that count)     */
    int64_t rows, V, ld;           /* row stride in elements, 0 for V; up to 2^30 */
} dgm_loss_cfg;

/* Softmax cross-entropy: loss[r] = lse[r] - logits[r, targets[r]], lse the
 * natural logarithm of the row's sum of e^logit, and dlogits[r, v] = scale *
 * rowScale[r] * (softmax - [v = target]). Targets are int32; a row with a
 * negative one has a loss of 0 and a gradient of zeros, whatever its logits.
 * rowScale (float [rows]) may be NULL for ones, and each of loss, lse and
 * dlogits; dlogits may be logits itself. Elements behind V of a row are neither
 * read nor written. A logit of -inf has probability 0; a row of nothing else has
 * lse -inf and a loss and gradient that are not numbers, as has one with a NaN or
 * +inf. The loss is not taken from the rounded lse: what is added to all logits
 * of a row does not change it. */
int dgm_crossEntropy(dgm_gpu* g, const dgm_loss_cfg* cfg, const void* logits, const int32_t* targets,
                     const float* rowScale, float* loss, float* lse, void* dlogits);

typedef struct dgm_rows_cfg {
    int32_t type, tableType;       /* DGM_TYPE_* of y and dy, and of the table  */
    float scale;
    int32_t pad;
    int64_t rows, C, V;            /* up to 2^30, 2^24, 2^31 - 1                */
} dgm_rows_cfg;

/* y[r, :] = scale * table[tokens[r], :], rounded once. Token 0xFFFFFFFF (-1) is
 * none: a row of zeros, without a report. */
int dgm_embedRows(dgm_gpu* g, const dgm_rows_cfg* cfg, const uint32_t* tokens, const void* table, void* y);
/* dtable[v, :] = scale * the sum of dy[r, :] over the rows of token v, zeros for
 * a token without rows; accumulate != 0: added to dtable, whose other rows are
 * not touched. The sums are fp32, over a token's rows in a fixed order. ws: at
 * least dgm_embedRowsBwd_ws_bytes(cfg) bytes (-1 for sizes that are refused). */
int64_t dgm_embedRowsBwd_ws_bytes(const dgm_rows_cfg* cfg);
int dgm_embedRowsBwd(dgm_gpu* g, const dgm_rows_cfg* cfg, const uint32_t* tokens, const void* dy, float* dtable,
                     int accumulate, void* ws, int64_t ws_bytes);

/* One parameter tensor of n elements: master w, gradient, moments m and v (float
 * [n]; in 8 bits: int8 and uint8 codes [n], with a scale for each 256 elements,
 * float [ceil(n / 256)]), and where its linear reads codes, those and their
 * scales (bits 8 or 4 as in dgm_quantize of rows of whole groups; qGroup a power
 * of two from 8 to 512; bits 0: none). A moment in 8 bits is c |c| mscale (c =
 * -127 .. 127) or (c^2 vscale)^2 (c = 0 .. 255; 2^-149 at least where c > 0), and
 * all zeros stand for zeros. Moments of 256 whose largest is below 2^-120 count
 * as 0; an infinity or NaN among them makes their scale, and so all their moments
 * from then on, NaN. The code is the nearest one (of the roots), but for moments
 * that rounding would hold: an m that shrank while its code stays and the scale
 * does not shrink, nor grow by over an eighth, goes one code down where c (1 -
 * b1) < 1 and v's code times (1 - b2) is below 4; a v whose code stays while the
 * scale does not grow goes one up where it grew to over 9 - 8 b2 of itself (a
 * gradient's square of over 9 times it). So weights without gradients come to
 * rest as with 32-bit moments. Moments far below the largest of their 256 are
 * coarse: of steady gradients below 1.5e-4 of the largest m stays 0, and a v that
 * decays by less than half a code a step (c < 2 / (1 - b2)) keeps its code, so
 * that such weights' steps are smaller than AdamW's. */
typedef struct dgm_adam_tensor {
    float* w;
    const float* grad;
    void *m, *v;
    float *mscale, *vscale;
    void* q;
    float* scale;
    int64_t n;
    int32_t decay;                 /* whether wd holds for it                   */
    int32_t bits, qGroup, pad;
} dgm_adam_tensor;
typedef struct dgm_adam_plan {     /* filled in by dgm_adamMany_plan            */
    void* table;
    int64_t tensors, chunks, elements;
    int32_t stateBits, pad;
} dgm_adam_plan;

/* Lays a list of tensors (host memory; those of 0 elements are left out) out for
 * the calls below, in `table`: device memory of at least dgm_adamMany_plan_bytes
 * bytes (-1 for a list that is refused), kept as long as the plan is used.
 * stateBits: 32 or 8. Waits for the context's stream; not during a graph capture
 * (DGM_ERR_UNSUPPORTED). DGM_ERR_ARG where buffers that a step writes overlap (a
 * tensor named twice), or one and a gradient. Needs no open region. A plan holds
 * addresses and sizes, nothing else of the tensors: it is made once, and again
 * where a buffer moves (68 tensors 0.5 ms on the host, 388 2.5 ms with the Python
 * wrappers), so gradients should keep their buffers from step to step. */
int64_t dgm_adamMany_plan_bytes(const dgm_adam_tensor* tensors, int64_t count, int64_t stateBits);
int dgm_adamMany_plan(dgm_gpu* g, const dgm_adam_tensor* tensors, int64_t count, int64_t stateBits, void* table,
                      int64_t bytes, dgm_adam_plan* plan);
/* out[0] = the norm of all gradients, out[1] = the factor that brings it down to
 * clip: clip / (norm + 1e-6) where clip > 0 and norm > clip, else 1 (device
 * memory). The squares are summed in 64 bits. Calls on one plan must not overlap
 * in time. */
int dgm_adamMany_norm(dgm_gpu* g, const dgm_adam_plan* plan, float clip, float* out);
/* dgm_adam of every tensor, wd 0 for those without decay, in one launch; with
 * bits, dgm_adam_quantize. factor (device memory, may be NULL): one float that
 * the gradients are multiplied by on the way (they are not written). With 32-bit
 * moments the results are those calls' bits. lr, the corrections and the others
 * are taken by value: a captured graph repeats those of its capture. Where they
 * change from step to step, capture what comes before and make this call between
 * the replays. */
int dgm_adamMany(dgm_gpu* g, const dgm_adam_plan* plan, const float* factor, float lr, float b1, float b2, float eps,
                 float wd, float invBC1, float invBC2);
/* The values of a plan's 8-bit moments (for a checkpoint): m and v [elements],
 * 16-byte aligned, tensor behind tensor, each from the next multiple of 256; what
 * lies between is not written. */
int dgm_adamMany_states(dgm_gpu* g, const dgm_adam_plan* plan, float* m, float* v);

/* ---- checkpoints (host code, no context) ----------------------------------
 * The reference's checkpoint files: a little-endian header, then every
 * parameter's fp32 master in the model's creation order. These validate a
 * file image in host memory and describe each parameter; the caller uploads
 * the masters and re-quantizes the quantized ones (GPT.load calls
 * quantizeAll, src/GPT.swift:318-322). Return DGM_ERR_SHAPE for a wrong magic
 * or version, an invalid configuration, or a length that does not match the
 * model (the reference's preconditions). */
typedef struct dgm_tgmt_header {   /* GPT.save (src/GPT.swift:265-281) */
    uint32_t version, bits, vocab, block, layers, heads, embd, qGroup;
} dgm_tgmt_header;
typedef struct dgm_tdit_header {   /* DiT.save (src/DiT.swift:396-411) */
    uint32_t version, side, patch, names, loops, heads, kvHeads, embd, intermediate, freqDim,
        diffusionSteps;
    float lastAlpha, valueMix;      /* version 1 files carry no lastAlpha: 0.01 */
    uint32_t header_bytes;          /* where the first parameter starts       */
} dgm_tdit_header;
typedef struct dgm_param_info {
    char name[32];                  /* the reference's parameter name          */
    int64_t rows, cols;
    int32_t quantized, decay;       /* Param.quantized / Param.decay           */
    int64_t offset;                 /* byte offset of its fp32 data in the file */
} dgm_param_info;

/* GPT.load (src/GPT.swift:283-324): header, itos at *itos_offset (vocab
 * bytes), then 2 + 16*layers + 2 parameters (wte, wpe, per layer ln1.g ...
 * proj.b, ln_f.g, ln_f.b; src/GPT.swift:44-64, 118-131). */
int dgm_tgmt_parse(const void* data, int64_t len, dgm_tgmt_header* hdr, int64_t* itos_offset,
                   int64_t* nparams);
int dgm_tgmt_param(const dgm_tgmt_header* hdr, int64_t i, dgm_param_info* out);
/* DiT.load (src/DiT.swift:413-451): 17 parameters, wpatch ... wdown, n1 ... nf
 * (src/DiT.swift:233-250). */
int dgm_tdit_parse(const void* data, int64_t len, dgm_tdit_header* hdr, int64_t* nparams);
int dgm_tdit_param(const dgm_tdit_header* hdr, int64_t i, dgm_param_info* out);

/* ---- measurement ----------------------------------------------------------
 * No counterpart in the reference: the achievable HBM read rate of one
 * launch, for the bench's roofline. Reads `bytes` (a multiple of 1024) from
 * `src` (16-byte aligned) in contiguous shares over `workgroups` workgroups
 * (0: one per CU), mode 0 with 16-byte loads into registers, mode 1 with
 * 16-byte direct-to-LDS loads, and stores one word per workgroup to `sink`
 * (device memory of at least 4 * workgroups bytes). */
int dgm_probe_read(dgm_gpu* g, const void* src, int64_t bytes, int64_t mode, int64_t workgroups,
                   uint32_t* sink);
/* No counterpart in the reference: a wave-reduction VALU GEMV over int4 codes
 * (Y[M,N] = X[M,K] . dequant(Wq)^T, fp32 FMAs, no bias), the design the
 * library's MFMA decode kernels are measured against. M is 1 or 16; K and
 * qGroup are multiples of 32; Wq and X 16-byte aligned. */
int dgm_probe_gemv_valu(dgm_gpu* g, const uint8_t* Wq, const float* scale, const float* X, float* Y, int64_t M,
                        int64_t N, int64_t K, int64_t qGroup);

/* ---- test hook -------------------------------------------------------------
 * No counterpart in the reference: bounds every in-workgroup hand-over wait of
 * the decode kernels to `spins` rounds (0 restores the default), so that a
 * test can force a wait to give up and check that dgm_end reports it. The
 * kernels still run to their end; only their results are invalid. */
int dgm_debug_wait_limit(int64_t spins);

#ifdef __cplusplus
}
#endif

#endif /* DGM_QUANT_H */
