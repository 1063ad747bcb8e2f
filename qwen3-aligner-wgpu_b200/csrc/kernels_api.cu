// extern "C" wrappers for the kernel-level entry points (include/qa_b200_kernels.h).
#include "qa_b200.h"
#include "qa_b200_kernels.h"

#include "gemm_tc.cuh"
#include "kernels.cuh"

using namespace qa;

extern "C" int qa_k_gemm(const void* A, long long lda, const void* B, long long ldb, int M, int N,
                         int K, int bf16, int mode, int act, void* out, long long ldo,
                         const float* bias, const int* row_map, const float* pe, int pe_period,
                         unsigned long long* keys, unsigned* status, int force_bn, void* stream) {
  EpiParams ep;
  ep.mode = mode;
  ep.act = act;
  ep.out = out;
  ep.ldo = ldo;
  ep.bias = bias;
  ep.row_map = row_map;
  ep.pe = pe;
  ep.pe_period = pe_period > 0 ? pe_period : 1;
  ep.keys = keys;
  ep.status = status;
  int rc = gemm_tc(A, lda, B, ldb, M, N, K, bf16 != 0, ep, static_cast<cudaStream_t>(stream),
                   force_bn);
  return rc == 0 ? QA_OK : QA_ERR_CUDA;
}

extern "C" int qa_k_gemm_qkv_rope(const void* A, long long lda, const void* B, long long ldb,
                                  int M, int N, int K, int bf16, void* q_out, long long ldo,
                                  const int* pos_of, const int* clip_of, const int* block_tab,
                                  int max_pages, void* kc, void* vc, const void* cos_t,
                                  const void* sin_t, const float* qn, const float* kn, float eps,
                                  int nq, int nkv, unsigned* status, int force_bn, void* stream) {
  if (!A || !B || !q_out || !pos_of || !clip_of || !block_tab || !kc || !vc || !cos_t || !sin_t ||
      !qn || !kn || nq <= 0 || nkv <= 0 || N != (nq + 2 * nkv) * 128)
    return QA_ERR_ARG;
  EpiParams ep;
  ep.mode = EPI_QKV_ROPE;
  ep.out = q_out;
  ep.ldo = ldo;
  ep.status = status;
  ep.rk.pos_of = pos_of;
  ep.rk.clip_of = clip_of;
  ep.rk.block_tab = block_tab;
  ep.rk.max_pages = max_pages;
  ep.rk.page_size = 64;
  ep.rk.kc = kc;
  ep.rk.vc = vc;
  ep.rk.cos_t = cos_t;
  ep.rk.sin_t = sin_t;
  ep.rk.qn = qn;
  ep.rk.kn = kn;
  ep.rk.eps = eps;
  ep.rk.nq = nq;
  ep.rk.nkv = nkv;
  int rc = gemm_tc(A, lda, B, ldb, M, N, K, bf16 != 0, ep, static_cast<cudaStream_t>(stream),
                   force_bn);
  return rc == 0 ? QA_OK : QA_ERR_CUDA;
}

extern "C" int qa_k_conv3x3s2(const void* x, int n, int h, int w, int c, const void* wt, int c_out,
                              int time_major, int bf16, int mode, int act, void* out, long long ldo,
                              const float* bias, unsigned* status, void* stream) {
  EpiParams ep;
  ep.mode = mode;
  ep.act = act;
  ep.out = out;
  ep.ldo = ldo;
  ep.bias = bias;
  ep.status = status;
  int rc = conv3x3s2_tc(x, n, h, w, c, wt, c_out, time_major != 0, bf16 != 0, ep,
                        static_cast<cudaStream_t>(stream));
  return rc == 0 ? QA_OK : QA_ERR_CUDA;
}

extern "C" int qa_k_causal_attention(const void* qkv, long long ldq, long long q_rows, int nqh,
                                     int nkvh, const int* tiles, int n_tiles, const int* block_tab,
                                     int max_pages, const void* kpool, const void* vpool,
                                     int kv_pages, void* out, int bf16, unsigned* status,
                                     void* stream) {
  if (!qkv || !tiles || !block_tab || !kpool || !vpool || !out || n_tiles < 0 || kv_pages <= 0)
    return QA_ERR_ARG;
  PagedKV kv{const_cast<void*>(kpool), const_cast<void*>(vpool), 64};
  const AttnTile* t = reinterpret_cast<const AttnTile*>(tiles);
  const int rc = causal_attention_tc(qkv, ldq, q_rows, nqh, nkvh, 128, t, n_tiles, block_tab,
                                     max_pages, kv, kv_pages, out, bf16 != 0, status,
                                     static_cast<cudaStream_t>(stream));
  return rc == 0 ? QA_OK : QA_ERR_CUDA;
}

extern "C" int qa_k_window_attention(const void* qkv, long long T, int dm, int nh,
                                     const int* windows, int n_windows, int max_window, void* out,
                                     int bf16, unsigned* status, void* stream) {
  if (!qkv || !out || (n_windows > 0 && !windows) || n_windows < 0 || T <= 0 || nh <= 0 ||
      dm != 64 * nh || max_window <= 0 || max_window > 128)
    return QA_ERR_ARG;
  const int rc = window_attention(qkv, T, dm, nh, 64, reinterpret_cast<const int2*>(windows),
                                  n_windows, max_window, out, bf16 != 0, status,
                                  static_cast<cudaStream_t>(stream));
  return rc == 0 ? QA_OK : QA_ERR_CUDA;
}

extern "C" int qa_k_conv1(const float* mel, int n, int h, int w, const float* wt,
                          const float* bias, int c_out, void* out, int bf16, void* stream) {
  if (!mel || !wt || !bias || !out || n < 0 || h <= 0 || w <= 0) return QA_ERR_ARG;
  const int rc = conv1_direct(mel, n, h, w, wt, bias, c_out, c_out, out, bf16 != 0, nullptr,
                              static_cast<cudaStream_t>(stream));
  return rc == 0 ? QA_OK : QA_ERR_CUDA;
}

namespace {

// What both cache entry points ask of their sequences and pools.
bool cache_args_ok(int nq, int nkv, const int* q_start, const int* kv_len, int n_seqs, int max_q,
                   const int* block_tab, int max_pages, const void* kpool, const void* vpool,
                   int kv_pages) {
  return q_start && kv_len && block_tab && kpool && vpool && n_seqs >= 0 && max_q >= 0 &&
         max_pages > 0 && kv_pages > 0 && nq > 0 && nkv > 0 && nq % nkv == 0;
}

// The answer to a launch.  A failed one's error is taken off the runtime's record, or
// the next call of anybody in the process would be told of it.
int answer(int rc) {
  if (rc == 0) return QA_OK;
  cudaGetLastError();
  return QA_ERR_CUDA;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

extern "C" int qa_k_kv_append(const void* q, long long ldq, const void* k, long long ldk,
                              const void* v, long long ldv, void* q_out, long long ldqo,
                              long long T, int nq, int nkv, int hd, const int* q_start,
                              const int* kv_len, int n_seqs, int max_q, const int* block_tab,
                              int max_pages, void* kpool, void* vpool, int kv_pages, float* kscale,
                              float* vscale, const float* cos_t, const float* sin_t, int table_rows,
                              const int* pos, long long pos_stride, int n_axes, const int* axis_of,
                              const float* qn, const float* kn, float eps, int bf16,
                              unsigned* status, void* stream) {
  if (T == 0 || n_seqs == 0) return QA_OK;
  if (!cache_args_ok(nq, nkv, q_start, kv_len, n_seqs, max_q, block_tab, max_pages, kpool, vpool,
                     kv_pages) ||
      !q || !k || !v || !q_out || T < 0 || T > 0x7FFFFFFFll || !kscale != !vscale ||
      !cos_t != !sin_t || (cos_t && table_rows <= 0) || n_axes < 1 || n_axes > 4 ||
      (n_axes > 1 && cos_t && (!pos || !axis_of)) || !qn != !kn)
    return QA_ERR_ARG;
  if ((hd != 64 && hd != 128) || ldq < static_cast<long long>(nq) * hd ||
      ldqo < static_cast<long long>(nq) * hd || ldk < static_cast<long long>(nkv) * hd ||
      ldv < static_cast<long long>(nkv) * hd)
    return QA_ERR_SHAPE;
  if (!aligned16(kpool) || !aligned16(vpool) || !aligned16(cos_t) || !aligned16(sin_t))
    return QA_ERR_ARG;
  const SeqMap seqs{q_start, kv_len, n_seqs, block_tab, max_pages, max_q};
  const RopeAxes rope{cos_t, sin_t, table_rows, pos, pos_stride, n_axes, axis_of};
  const int rc = kv_append(q, ldq, k, ldk, v, ldv, q_out, ldqo, T, nq, nkv, hd, seqs, max_q,
                           PagedKV{kpool, vpool, 64}, kv_pages, kscale, vscale, rope, qn, kn, eps,
                           bf16 != 0, status, static_cast<cudaStream_t>(stream));
  return answer(rc);
}

extern "C" int qa_k_cache_attention(const void* q, long long ldq, long long T, int nq, int nkv,
                                    int hd, const int* q_start, const int* kv_len, int n_seqs,
                                    int max_q, int max_kv, const int* block_tab, int max_pages,
                                    const void* kpool, const void* vpool, int kv_pages,
                                    const float* kscale, const float* vscale, float scale,
                                    int causal, void* out, long long ldo, float* lse,
                                    void* workspace, long long workspace_bytes, int bf16,
                                    unsigned* status, void* stream) {
  if (T == 0 || n_seqs == 0) return QA_OK;
  if (!cache_args_ok(nq, nkv, q_start, kv_len, n_seqs, max_q, block_tab, max_pages, kpool, vpool,
                     kv_pages) ||
      !q || !kscale || !vscale || !out || T < 0 || T > 0x7FFFFFFFll || max_kv < 0 ||
      !(scale - scale == 0.0f) || workspace_bytes < 0 || !aligned16(workspace))
    return QA_ERR_ARG;
  if ((hd != 64 && hd != 128) || ldq < static_cast<long long>(nq) * hd ||
      ldo < static_cast<long long>(nq) * hd)
    return QA_ERR_SHAPE;
  if (!aligned16(kpool) || !aligned16(vpool)) return QA_ERR_ARG;
  const SeqMap seqs{q_start, kv_len, n_seqs, block_tab, max_pages, max_q};
  const int rc = cache_attention(q, ldq, T, nq, nkv, hd, seqs, max_q, max_kv, kpool, vpool,
                                 kv_pages, kscale, vscale, scale, causal != 0, out, ldo, lse,
                                 workspace, workspace_bytes, bf16 != 0, status, static_cast<cudaStream_t>(stream));
  return answer(rc);
}

extern "C" int64_t qa_k_cache_attention_workspace(int nq, int nkv, int hd, int n_seqs, int max_q,
                                                  int max_kv) {
  return cache_attention_workspace(nq, nkv, hd, n_seqs, max_q, max_kv);
}

extern "C" int qa_k_w4_linear(const void* x, long long ldx, int M, int K, const uint8_t* wq,
                              long long ldw, int N, int group, const void* scales,
                              const uint8_t* zeros, const float* bias, void* out, long long ldo,
                              int bf16, void* stream) {
  if (M == 0 || N == 0) return QA_OK;
  if (!x || !wq || !scales || !out || M < 0 || N < 0) return QA_ERR_ARG;
  if ((group != 32 && group != 64 && group != 128) || K <= 0 || K % group != 0 || ldx < K ||
      ldw < K / 2 || ldo < N)
    return QA_ERR_SHAPE;
  const int rc = w4_linear(x, ldx, M, K, wq, ldw, N, group, scales, zeros, bias, out, ldo,
                           bf16 != 0, static_cast<cudaStream_t>(stream));
  return answer(rc);
}

namespace {

template <typename T>
T* as_ptr(long long v) {
  return reinterpret_cast<T*>(static_cast<uintptr_t>(v));
}

}  // namespace

extern "C" int qa_k_kv_append_v(const long long* a, float eps) {
  if (!a) return QA_ERR_ARG;
  return qa_k_kv_append(as_ptr<void>(a[0]), a[1], as_ptr<void>(a[2]), a[3], as_ptr<void>(a[4]), a[5],
                        as_ptr<void>(a[6]), a[7], a[8], (int)a[9], (int)a[10], (int)a[11],
                        as_ptr<int>(a[12]), as_ptr<int>(a[13]), (int)a[14], (int)a[15],
                        as_ptr<int>(a[16]), (int)a[17], as_ptr<void>(a[18]), as_ptr<void>(a[19]),
                        (int)a[20], as_ptr<float>(a[21]), as_ptr<float>(a[22]), as_ptr<float>(a[23]),
                        as_ptr<float>(a[24]), (int)a[25], as_ptr<int>(a[26]), a[27], (int)a[28],
                        as_ptr<int>(a[29]), as_ptr<float>(a[30]), as_ptr<float>(a[31]), eps,
                        (int)a[32], as_ptr<unsigned>(a[33]), as_ptr<void>(a[34]));
}

extern "C" int qa_k_cache_attention_v(const long long* a, float scale) {
  if (!a) return QA_ERR_ARG;
  return qa_k_cache_attention(as_ptr<void>(a[0]), a[1], a[2], (int)a[3], (int)a[4], (int)a[5],
                              as_ptr<int>(a[6]), as_ptr<int>(a[7]), (int)a[8], (int)a[9], (int)a[10],
                              as_ptr<int>(a[11]), (int)a[12], as_ptr<void>(a[13]),
                              as_ptr<void>(a[14]), (int)a[15], as_ptr<float>(a[16]),
                              as_ptr<float>(a[17]), scale, (int)a[18], as_ptr<void>(a[19]), a[20],
                              as_ptr<float>(a[21]), as_ptr<void>(a[22]), a[23], (int)a[24],
                              as_ptr<unsigned>(a[25]), as_ptr<void>(a[26]));
}

extern "C" int qa_k_w4_linear_v(const long long* a) {
  if (!a) return QA_ERR_ARG;
  return qa_k_w4_linear(as_ptr<void>(a[0]), a[1], (int)a[2], (int)a[3], as_ptr<uint8_t>(a[4]), a[5],
                        (int)a[6], (int)a[7], as_ptr<void>(a[8]), as_ptr<uint8_t>(a[9]),
                        as_ptr<float>(a[10]), as_ptr<void>(a[11]), a[12], (int)a[13],
                        as_ptr<void>(a[14]));
}
