/*
 * Kernel-level entry points of the B200 alignment backend.
 *
 * These take DEVICE pointers (already resident in HBM) and a CUDA stream, and
 * run one hot-path kernel each.  They exist so that each kernel can be
 * parity-tested and timed on its own; the reference has no counterpart at this
 * granularity (its kernels are WGSL dispatches inside src/decoder.rs and
 * src/audio_encoder_gpu.rs), so each declaration names the reference stage it
 * computes instead.
 *
 * All functions return 0 on success or a QA_ERR_* code (see qa_b200.h).  They
 * launch on the current device, which has to be the buffers' and the stream's.
 * 16-bit element buffers are f16 when `bf16 == 0`, bf16 otherwise.
 */
#ifndef QA_B200_KERNELS_H
#define QA_B200_KERNELS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Epilogue selectors for qa_k_gemm (values match the library's EpiMode). */
#define QA_EPI_STORE16 0
#define QA_EPI_RESID16 1
#define QA_EPI_RESID32 2
#define QA_EPI_SWIGLU16 3
#define QA_EPI_STORE32 4
#define QA_EPI_ARGMAX 5

/*
 * D = A · Bᵀ on the tcgen05 tensor cores (TMEM accumulator, TMA-fed).
 * A [M, K] (row stride lda), B [N, K] (row stride ldb), 16-bit.
 * `mode`/`act`/`bias`/`out`/`ldo`/`row_map`/`pe`/`keys` select the fused
 * epilogue.  Stands in for every `prefill_gemm*` dispatch of the reference
 * (src/shaders.rs:1817-2077; src/decoder.rs:1321-1657) and for the host
 * projections of src/audio_encoder.rs and src/align_inference.rs:789-790.
 * `status` (device, may be NULL) receives timeout bits.  `force_bn`: 0 = the
 * library's tile choice, -1 = 256-row tiles on CTA pairs, > 0 = one CTA per
 * 128-row tile of that width (128, 224, 240 or 256).
 */
int qa_k_gemm(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K,
              int bf16, int mode, int act, void* out, long long ldo, const float* bias,
              const int* row_map, const float* pe, int pe_period, unsigned long long* keys,
              unsigned* status, int force_bn, void* stream);

/*
 * The decoder's fused QKV projection: qkv = A · Bᵀ (B = [q|k|v] rows), with
 * the epilogue of cpu_decoder.rs:305-321 per 128-column head: q and k heads
 * are rounded, RMS-normalised (gains qn / kn), rotated by RoPE at the row's
 * position (cos_t / sin_t [max_seq][64] in the storage format); q is written
 * to q_out (row stride ldo), k and v are appended to the paged caches kc / vc
 * [page][nkv][64][128] at (block_tab[clip_of[row]][pos / 64], pos % 64) with
 * pos = pos_of[row].  N = (nq + 2 nkv) * 128.
 */
int qa_k_gemm_qkv_rope(const void* A, long long lda, const void* B, long long ldb, int M, int N,
                       int K, int bf16, void* q_out, long long ldo, const int* pos_of,
                       const int* clip_of, const int* block_tab, int max_pages, void* kc, void* vc,
                       const void* cos_t, const void* sin_t, const float* qn, const float* kn,
                       float eps, int nq, int nkv, unsigned* status, int force_bn, void* stream);

/*
 * Implicit-GEMM conv2d, 3x3 / stride 2 / pad 1, on the tcgen05 tensor cores:
 * x NHWC [n][h][w][c] 16-bit, wt [c_out][9c] (k = (kh*3 + kw)*c + ic),
 * output [n*ho*wo][c_out] through the same epilogues as qa_k_gemm (rows in
 * (oh, ow) order, or (ow, oh) when time_major).  Stands in for the conv2 /
 * conv3 levels of CpuConvStem::conv_block_stages (src/audio_encoder.rs:361-447)
 * and the GPU tower's im2col + GEMM (src/audio_encoder_gpu.rs:1714-1795).
 */
int qa_k_conv3x3s2(const void* x, int n, int h, int w, int c, const void* wt, int c_out,
                   int time_major, int bf16, int mode, int act, void* out, long long ldo,
                   const float* bias, unsigned* status, void* stream);

/*
 * First conv level of the audio tower: conv2d(1 -> c_out, 3x3, stride 2,
 * pad 1) + bias + erf-GELU over mel chunks [n][h][w] (f32), output NHWC
 * [n][ho][wo][c_out] 16-bit (CpuConvStem::conv_block_stages level 1,
 * src/audio_encoder.rs:361-447).  wt [c_out][9] f32, bias [c_out] f32.
 * c_out a multiple of 32 (up to 512) runs on the tensor cores with split f16
 * operands (f32-grade products); other channel counts on CUDA cores.
 */
int qa_k_conv1(const float* mel, int n, int h, int w, const float* wt, const float* bias,
               int c_out, void* out, int bf16, void* stream);

/*
 * Causal GQA attention of the decoder prefill over the paged K/V cache
 * (src/cpu_decoder.rs:327-412; the reference GPU path's
 * prefill_attention_paged dispatch, src/decoder.rs:1463-1520), on the
 * persistent tcgen05/TMEM kernel the pipeline runs.
 * qkv [q_rows][ldq] 16-bit with query head h at column h*128; kpool/vpool
 * [kv_pages][nkvh][64][128]; tiles [n_tiles][4] = (clip, q0, tok0, len), one
 * per 128 query positions of a clip; block_tab [clips][max_pages] page ids;
 * out [q_rows][nqh*128].  GQA groups of two (nqh == 2 * nkvh, the model's
 * geometry); other head counts give QA_ERR_CUDA.
 */
int qa_k_causal_attention(const void* qkv, long long ldq, long long q_rows, int nqh, int nkvh,
                          const int* tiles, int n_tiles, const int* block_tab, int max_pages,
                          const void* kpool, const void* vpool, int kv_pages, void* out, int bf16,
                          unsigned* status, void* stream);

/*
 * The audio tower's windowed self-attention (src/audio_encoder.rs:574-627;
 * the reference GPU tower's window attention, src/audio_encoder_gpu.rs:
 * 1497-1547) on the tcgen05 tensor cores: every query of a window attends to
 * every key of the same window.  qkv [T][3*dm] 16-bit (q | k | v, head h at
 * columns h*64 of each), out [T][dm] with dm = 64 * nh; windows [n_windows][2]
 * = (first token, length), 1 <= length <= max_window <= 128, inside [0, T).
 * A pipeline wait that runs out sets bit 1 of *status (may be NULL).
 */
int qa_k_window_attention(const void* qkv, long long T, int dm, int nh, const int* windows,
                          int n_windows, int max_window, void* out, int bf16, unsigned* status,
                          void* stream);

/*
 * The three entry points below serve sessions that grow: a few new tokens for
 * each of many sequences, against what their caches already hold.  They have no
 * counterpart in the reference, which prefills a whole clip at once.
 *
 * New tokens are packed: sequence s owns rows [q_start[s], q_start[s + 1]) of
 * every [T]-row buffer, at most max_q of them (0 is allowed; a max_q above T
 * counts as T), and its cache holds kv_len[s] tokens, the new ones among them.  q_start [n_seqs + 1],
 * kv_len [n_seqs] and block_tab [n_seqs][max_pages] are device data; they are
 * checked on the device, and what contradicts the sizes given here (a sequence
 * outside [0, T) or longer than max_q or than its table, a page id outside
 * [0, kv_pages)) sets bit 2 of *status (may be NULL) and is neither read nor
 * written.  Row strides (ld*) are in elements; head h of a row starts at h * hd,
 * hd is 64 or 128, nq a multiple of nkv.  Sizes of zero are allowed and do
 * nothing.
 */

/*
 * Rotates q [T][nq * hd] into q_out (which may be q) and appends k (rotated)
 * and v [T][nkv * hd] to the paged cache at cache indices kv_len[s] - n_s + i.
 * Pools are [kv_pages][nkv][64][hd].
 *
 * Cache format: with kscale / vscale [kv_pages][nkv] (both or neither) the
 * pools hold e4m3 codes of value code * scale, and a page's scale is the least
 * power of two (>= 2^-64) that brings its largest finite value to at most 448;
 * appending to a page that has tokens keeps the larger scale and rescales the
 * older codes when it grows.  Values that are not finite become NaN codes.
 * Without scales the pools hold the 16-bit type (what qa_k_causal_attention
 * reads).  Sequences may share pages that are full, not the page they append to.
 *
 * Rotation: cos_t / sin_t [table_rows][hd / 2] f32 (NULL: none), the halves of a
 * head paired (j, j + hd / 2).  Positions: pos [n_axes][pos_stride], NULL for the
 * cache index; with tables and n_axes > 1 (at most 4), axis_of [hd / 2] names
 * each frequency's axis.  A position outside the tables or an axis outside
 * [0, n_axes) sets bit 2 of *status and counts as 0.  qn / kn [hd] (both or
 * neither): RMSNorm of each head before the rotation, with eps.  Arithmetic in
 * f32, rounded once.  kpool, vpool, cos_t and sin_t are 16-byte aligned.
 */
int qa_k_kv_append(const void* q, long long ldq, const void* k, long long ldk, const void* v,
                   long long ldv, void* q_out, long long ldqo, long long T, int nq, int nkv, int hd,
                   const int* q_start, const int* kv_len, int n_seqs, int max_q,
                   const int* block_tab, int max_pages, void* kpool, void* vpool, int kv_pages,
                   float* kscale, float* vscale, const float* cos_t, const float* sin_t,
                   int table_rows, const int* pos, long long pos_stride, int n_axes,
                   const int* axis_of, const float* qn, const float* kn, float eps, int bf16,
                   unsigned* status, void* stream);

/*
 * Attention of q [T][nq * hd] over the e4m3 cache: query head h reads K/V head
 * h / (nq / nkv).  Query i of a sequence sees cache indices below
 * kv_len - n_s + i + 1 (causal) or kv_len; scores are scale * (q . k).  A row
 * that sees nothing gets zeros and lse -inf; what lies past a sequence's length
 * in its last page is never used, whatever it holds.  A page id outside the pool
 * sets bit 2 of *status and its tokens are left out.  lse [T][nq] f32 (natural
 * logarithm of the sum of exponentials) may be NULL.
 *
 * max_kv (the longest kv_len, as far as the caller knows; above 64 * max_pages it
 * counts as that) sizes the launch; a smaller or larger value gives the same
 * results up to the order of sums.
 *
 * workspace: device memory, 16-byte aligned, of the size that
 * qa_k_cache_attention_workspace gives for these arguments (0: none is needed);
 * what it holds does not matter, and two calls that may run at the same time
 * need one each.  With less of it, or NULL, the last or all sequences are not
 * split over CTAs, which is slow for few long caches.  More than 1 GiB is never
 * asked for: of the sequences past it the same holds.
 *
 * The others of the batch bear on a sequence's result only through max_q, which
 * chooses the kernel and its tiles of rows (other sums, within rounding), and
 * where they leave it no place in the workspace.
 */
int64_t qa_k_cache_attention_workspace(int nq, int nkv, int hd, int n_seqs, int max_q, int max_kv);
int qa_k_cache_attention(const void* q, long long ldq, long long T, int nq, int nkv, int hd,
                         const int* q_start, const int* kv_len, int n_seqs, int max_q, int max_kv,
                         const int* block_tab, int max_pages, const void* kpool, const void* vpool,
                         int kv_pages, const float* kscale, const float* vscale, float scale,
                         int causal, void* out, long long ldo, float* lse, void* workspace,
                         long long workspace_bytes, int bf16, unsigned* status, void* stream);

/*
 * out [M][N] = x [M][K] . W^T (+ bias [N] f32), the weights in 4 bits:
 * W[n][k] = scales[n][k / group] * (code[n][k] - zeros[n][k / group]), zeros any
 * byte, 8 when NULL.  wq [N] rows of K / 2 bytes, ldw bytes apart, the even k of a pair
 * in the low nibble; scales [N][K / group] in x's type; group 32, 64 or 128, K a
 * multiple of it.  f32 sums, one rounding; M and N bear on their order.  Built
 * for few rows, where the weights are what has to be read; any M is taken.
 */
int qa_k_w4_linear(const void* x, long long ldx, int M, int K, const uint8_t* wq, long long ldw,
                   int N, int group, const void* scales, const uint8_t* zeros, const float* bias,
                   void* out, long long ldo, int bf16, void* stream);

/*
 * The same three calls with their arguments in the same order in an array, but for
 * the one float (pointers as integers): for callers through an interpreter, where
 * passing 36 arguments one by one takes longer than the kernel.
 */
int qa_k_kv_append_v(const long long* args, float eps);
int qa_k_cache_attention_v(const long long* args, float scale);
int qa_k_w4_linear_v(const long long* args);

#ifdef __cplusplus
}
#endif

#endif /* QA_B200_KERNELS_H */
