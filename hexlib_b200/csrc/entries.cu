// entries.cu -- the kernel_api.h-shaped C entry points of libhexlib_b200.
//
// One function per kernels/<k>/kernel_api.h signature, with a trailing stream
// and an int status. They validate their scalar arguments, then call the same
// launcher the batch dispatcher uses, with one image.
#include <cuda_runtime.h>

#include <initializer_list>
#include <mutex>

#include "../../include/hexlib_b200.h"
#include "hb_kernels.h"

namespace hb {

int memory_kernels_init();
int gemm_kernels_init();
int quant_kernels_init();
int attention_kernels_init();
int diag_kernels_init();

namespace {
constexpr int kMaxDevices = 64;
std::once_flag g_dev_once[kMaxDevices];
int g_dev_status[kMaxDevices];
std::once_flag g_word_once;
int g_word_status = HEXLIB_B200_ERR_INTERNAL;
int* g_err_host = nullptr;
int* g_err_dev = nullptr;
}  // namespace

// Function attributes (the dynamic shared memory each kernel may take) belong
// to the device that is current when they are set, so every device a process
// uses runs this once, with that device current. It allocates nothing.
int kernels_init_device() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  std::call_once(g_dev_once[dev], [dev] {
    int rc = memory_kernels_init();
    if (rc == HEXLIB_B200_OK) rc = gemm_kernels_init();
    if (rc == HEXLIB_B200_OK) rc = quant_kernels_init();
    if (rc == HEXLIB_B200_OK) rc = attention_kernels_init();
    if (rc == HEXLIB_B200_OK) rc = diag_kernels_init();
    if (rc == HEXLIB_B200_OK) rc = e4m3_kernels_init();
    if (rc == HEXLIB_B200_OK) rc = gemm_e4m3_kernels_init();
    if (rc == HEXLIB_B200_OK) rc = edge_kernels_init();
    if (rc == HEXLIB_B200_OK) rc = rope_pos_kernels_init();
    if (rc != HEXLIB_B200_OK) cudaGetLastError();
    g_dev_status[dev] = rc;
  });
  return g_dev_status[dev];
}

// The per-kernel entries' error word: one int of mapped, portable host memory
// that every device can write (a bounded wait that expires sets it to 1) and
// the host reads after the stream has drained (hexlib_b200_stream_status).
int kernels_init() {
  const int rc = kernels_init_device();
  if (rc != HEXLIB_B200_OK) return rc;
  std::call_once(g_word_once, [] {
    int st = HEXLIB_B200_ERR_CUDA;
    int* host = nullptr;
    if (cudaHostAlloc(reinterpret_cast<void**>(&host), sizeof(int),
                      cudaHostAllocMapped | cudaHostAllocPortable) == cudaSuccess) {
      *host = 0;
      if (cudaHostGetDevicePointer(reinterpret_cast<void**>(&g_err_dev), host, 0) ==
          cudaSuccess) {
        g_err_host = host;
        st = HEXLIB_B200_OK;
      }
    }
    if (st != HEXLIB_B200_OK) cudaGetLastError();
    g_word_status = st;
  });
  return g_word_status;
}

// Reads and clears the per-kernel entries' error word; true if it was set.
bool take_default_error() {
  if (!g_err_host) return false;
  volatile int* e = g_err_host;
  const bool set = *e != 0;
  *e = 0;
  return set;
}

int* default_error_word() { return g_err_dev; }

}  // namespace hb

using hb::kernels_init;

#define HB_ENTRY_INIT()                              \
  do {                                               \
    const int _rc = kernels_init();                  \
    if (_rc != HEXLIB_B200_OK) return _rc;           \
  } while (0)

static inline cudaStream_t as_stream(void* s) {
  return reinterpret_cast<cudaStream_t>(s);
}

static inline bool misaligned(const void* p, uintptr_t n) {
  return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0;
}

extern "C" {

int hexlib_b200_add_fp16(const void* a, const void* b, void* y, int n,
                         void* stream) {
  HB_ENTRY_INIT();
  if (n < 0 || (n > 0 && (!a || !b || !y))) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_add_f16(a, b, y, n, n > 0 ? n : 1, as_stream(stream));
}

int hexlib_b200_add_fp16_f32(const void* a, const float* b, void* y, int n,
                             void* stream) {
  HB_ENTRY_INIT();
  if (n < 0 || (n > 0 && (!a || !b || !y))) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_add_f16_f32(a, b, y, n, n > 0 ? n : 1, as_stream(stream));
}

int hexlib_b200_cast_f32_f16(const float* x, void* y, int n, void* stream) {
  HB_ENTRY_INIT();
  if (n < 0 || (n > 0 && (!x || !y))) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_cast_f32_f16(x, y, n, as_stream(stream));
}

int hexlib_b200_scale_fp16(const void* x, void* y, int n, float factor,
                           void* stream) {
  HB_ENTRY_INIT();
  if (n < 0 || (n > 0 && (!x || !y))) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_scale_f16(x, y, n, factor, as_stream(stream));
}

int hexlib_b200_layernorm_fp16(const void* x, const float* w, const float* b,
                               void* y, int R, int C, float eps,
                               void* stream) {
  HB_ENTRY_INIT();
  if (R < 0 || C <= 0 || (R > 0 && (!x || !w || !b || !y)))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_layernorm_f16(x, w, b, y, R, C, eps, as_stream(stream));
}

int hexlib_b200_rmsnorm_fp16(const void* x, const void* w, void* y, int R,
                             int C, float eps, void* stream) {
  HB_ENTRY_INIT();
  if (R < 0 || C <= 0 || (R > 0 && (!x || !w || !y)))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_rmsnorm_f16(x, w, y, R, C, eps, as_stream(stream));
}

int hexlib_b200_softmax_fp16(const void* x, void* y, int R, int C,
                             void* stream) {
  HB_ENTRY_INIT();
  if (R < 0 || C <= 0 || (R > 0 && (!x || !y)))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_softmax_f16(x, y, R, C, as_stream(stream));
}

int hexlib_b200_rope_2d_fp16(const void* x, const float* costab,
                             const float* sintab, void* y, int T, int H, int D,
                             void* stream) {
  HB_ENTRY_INIT();
  if (T < 0 || H <= 0 || D <= 0 || (D & 1) ||
      (T > 0 && (!x || !costab || !sintab || !y)))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (T == 0) return HEXLIB_B200_OK;
  return hb::launch_rope_f16(x, costab, sintab, y, T, H, D, T,
                             as_stream(stream));
}

int hexlib_b200_transpose_th_fp16(const void* x, void* y, int T, int H, int D,
                                  void* stream) {
  HB_ENTRY_INIT();
  if (T <= 0 || H <= 0 || D <= 0 || !x || !y)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_transpose_th_f16(x, y, 1, T, H, D, as_stream(stream));
}

int hexlib_b200_transpose_hd_fp16(const void* x, void* y, int B, int T, int D,
                                  void* stream) {
  HB_ENTRY_INIT();
  if (B < 0 || T <= 0 || D <= 0 || (B > 0 && (!x || !y)))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_transpose_hd_f16(x, y, B, T, D, as_stream(stream));
}

int hexlib_b200_patchify_fp32(const float* img, float* out, int C, int T,
                              int H, int W, int patch, int merge, int grid_h,
                              int grid_w, void* stream) {
  HB_ENTRY_INIT();
  if (!img || !out) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_patchify_f32(img, out, 1, C, T, H, W, patch, merge, grid_h,
                                 grid_w, as_stream(stream));
}

int hexlib_b200_patchify_fp16(const float* img, void* out, int C, int T, int H, int W,
                              int patch, int merge, int grid_h, int grid_w, void* stream) {
  HB_ENTRY_INIT();
  return hb::launch_patchify_f32_f16(img, out, 1, C, T, H, W, patch, merge, grid_h, grid_w,
                                     as_stream(stream));
}

int hexlib_b200_matmul_fp16(const void* A, const void* B, void* C, int Bn,
                            int M, int K, int N, void* stream) {
  HB_ENTRY_INIT();
  if (Bn < 0 || M < 0 || K <= 0 || N <= 0) return HEXLIB_B200_ERR_INVAL_PARAMS;
  hb::GemmDesc g{};
  g.A = A;
  g.B = B;
  g.out = C;
  g.batch = Bn;
  g.M = M;
  g.K = K;
  g.N = N;
  g.b_shared = false;
  g.act = 0;
  return hb::launch_gemm(g, hb::default_error_word(), as_stream(stream));
}

int hexlib_b200_matmul_epilogue_fp16(const void* a, const void* w,
                                     const float* bias, void* out, int M,
                                     int K, int N, int act, void* stream) {
  HB_ENTRY_INIT();
  if (M < 0 || K <= 0 || N <= 0 || act < 0 || act > 2 || !bias)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  hb::GemmDesc g{};
  g.A = a;
  g.B = w;
  g.bias = bias;
  g.out = out;
  g.batch = 1;
  g.M = M;
  g.K = K;
  g.N = N;
  g.b_shared = true;
  g.act = act;
  return hb::launch_gemm(g, hb::default_error_word(), as_stream(stream));
}

int hexlib_b200_dequant_q4_0_fp16(const void* w, void* out, int K, int N, void* stream) {
  HB_ENTRY_INIT();
  if (K < 0 || N < 0) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_dequant_f16(hb::QTYPE_Q4_0, w, out, K, N, as_stream(stream));
}

int hexlib_b200_dequant_q8_0_fp16(const void* w, void* out, int K, int N, void* stream) {
  HB_ENTRY_INIT();
  if (K < 0 || N < 0) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_dequant_f16(hb::QTYPE_Q8_0, w, out, K, N, as_stream(stream));
}

static int matmul_epilogue_quant(int qtype, const void* a, const void* w, const float* bias,
                                 void* out, int M, int K, int N, int act, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
  if (M < 0 || K <= 0 || N <= 0 || N % 32 || act < 0 || act > 2 || !bias || !w)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  hb::GemmDesc g{};
  g.A = a;
  g.B = w;
  g.bias = bias;
  g.out = out;
  g.batch = 1;
  g.M = M;
  g.K = K;
  g.N = N;
  g.b_shared = true;
  g.act = act;
  return hb::launch_gemm_quant(g, qtype, workspace, workspace_bytes, hb::default_error_word(),
                               as_stream(stream));
}

int hexlib_b200_matmul_epilogue_q4_0(const void* a, const void* w, const float* bias,
                                     void* out, int M, int K, int N, int act, void* workspace,
                                     uint64_t workspace_bytes, void* stream) {
  HB_ENTRY_INIT();
  return matmul_epilogue_quant(hb::QTYPE_Q4_0, a, w, bias, out, M, K, N, act, workspace,
                               workspace_bytes, stream);
}

int hexlib_b200_matmul_epilogue_q8_0(const void* a, const void* w, const float* bias,
                                     void* out, int M, int K, int N, int act, void* workspace,
                                     uint64_t workspace_bytes, void* stream) {
  HB_ENTRY_INIT();
  return matmul_epilogue_quant(hb::QTYPE_Q8_0, a, w, bias, out, M, K, N, act, workspace,
                               workspace_bytes, stream);
}

int hexlib_b200_matmul_epilogue_residual_fp16(const void* a, const void* w,
                                              const float* bias, const void* r,
                                              void* out, int M, int K, int N,
                                              int act, void* stream) {
  HB_ENTRY_INIT();
  if (M < 0 || K <= 0 || N <= 0 || act < 0 || act > 2 || !bias || !r)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  hb::GemmDesc g{};
  g.A = a;
  g.B = w;
  g.bias = bias;
  g.resid = r;
  g.out = out;
  g.batch = 1;
  g.M = M;
  g.K = K;
  g.N = N;
  g.b_shared = true;
  g.act = act;
  return hb::launch_gemm(g, hb::default_error_word(), as_stream(stream));
}

int hexlib_b200_matmul_epilogue_rope_fp16(const void* a, const void* w, const float* bias,
                                          const float* seg_cos, const float* seg_sin,
                                          const int* seg_idx, int n_seg, void* out, int M,
                                          int K, int N, int act, int rope_cols, int T,
                                          void* stream) {
  HB_ENTRY_INIT();
  if (M < 0 || K <= 0 || N <= 0 || act < 0 || act > 2 || !bias || !seg_cos || !seg_sin ||
      !seg_idx || n_seg <= 0 || rope_cols <= 0 || T <= 0 || (M % T) != 0)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  hb::GemmDesc g{};
  g.A = a;
  g.B = w;
  g.bias = bias;
  g.out = out;
  g.batch = 1;
  g.M = M;
  g.K = K;
  g.N = N;
  g.b_shared = true;
  g.act = act;
  g.rope_cos = seg_cos;
  g.rope_sin = seg_sin;
  g.rope_idx = seg_idx;
  g.rope_nseg = n_seg;
  g.rope_T = T;
  g.rope_cols = rope_cols;
  return hb::launch_gemm(g, hb::default_error_word(), as_stream(stream));
}

int hexlib_b200_ln_stats_fp16(const void* x, float* stats, int R, int C, float eps,
                              void* stream) {
  HB_ENTRY_INIT();
  return hb::launch_ln_stats_f16(x, stats, R, C, eps, as_stream(stream));
}

static int matmul_ln(const void* x, const void* w, const float* cols, const float* stats,
                     const float* segtab, const int* seg_idx, int n_seg, void* out, int M,
                     int K, int N, int act, int rope_cols, int T, void* stream) {
  if (M < 0 || K <= 0 || N <= 0 || act < 0 || act > 2 || !cols || !stats)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  hb::GemmDesc g{};
  g.A = x;
  g.B = w;
  g.bias = cols;
  g.ln_colsum = cols + N;
  g.ln_stats = stats;
  g.out = out;
  g.batch = 1;
  g.M = M;
  g.K = K;
  g.N = N;
  g.b_shared = true;
  g.act = act;
  if (segtab) {
    if (!seg_idx || n_seg <= 0 || rope_cols <= 0 || T <= 0 || (M % T) != 0)
      return HEXLIB_B200_ERR_INVAL_PARAMS;
    g.rope_cos = segtab;
    g.rope_sin = segtab + 16;
    g.rope_stride = 32;
    g.rope_idx = seg_idx;
    g.rope_nseg = n_seg;
    g.rope_T = T;
    g.rope_cols = rope_cols;
  }
  return hb::launch_gemm(g, hb::default_error_word(), as_stream(stream));
}

int hexlib_b200_matmul_epilogue_ln_fp16(const void* x, const void* w, const float* cols,
                                        const float* stats, void* out, int M, int K, int N,
                                        int act, void* stream) {
  HB_ENTRY_INIT();
  return matmul_ln(x, w, cols, stats, nullptr, nullptr, 0, out, M, K, N, act, 0, 0, stream);
}

int hexlib_b200_matmul_epilogue_ln_rope_fp16(const void* x, const void* w, const float* cols,
                                             const float* stats, const float* segtab,
                                             const int* seg_idx, int n_seg, void* out, int M,
                                             int K, int N, int act, int rope_cols, int T,
                                             void* stream) {
  HB_ENTRY_INIT();
  if (!segtab) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return matmul_ln(x, w, cols, stats, segtab, seg_idx, n_seg, out, M, K, N, act, rope_cols, T,
                   stream);
}

int hexlib_b200_rope_qk_fp16(const void* qkv, const float* costab, const float* sintab,
                             void* out, int rows, int H, int D, int T, void* stream) {
  HB_ENTRY_INIT();
  if (rows < 0 || T <= 0 || !qkv || !out || !costab || !sintab)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_rope_qk_f16(qkv, costab, sintab, out, rows, H, D, T, as_stream(stream));
}

int hexlib_b200_attention_qkv_fp16(const void* qkv, void* ctx, int B, int T, int H, int D,
                                   float scale, void* stream) {
  HB_ENTRY_INIT();
  return hb::launch_attention_qkv(qkv, ctx, B, T, H, D, scale, hb::default_error_word(),
                                  as_stream(stream));
}

int hexlib_b200_attention_fp16(const void* q, const void* k, const void* v,
                               void* ctx, int Bn, int T, int D, float scale,
                               void* stream) {
  HB_ENTRY_INIT();
  if (Bn < 0 || T <= 0 || D <= 0 || (Bn > 0 && (!q || !k || !v || !ctx)))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  return hb::launch_attention(q, k, v, ctx, Bn, T, D, scale,
                              hb::default_error_word(), as_stream(stream));
}

// Most rows and columns of the operators below: their tiles and padded widths are ints.
constexpr int kMostExtent = 1 << 30;

// The operators of a transformer block in 8-bit floating point. Their refusals
// come before the initialisation, so that a refused call needs no device.

int hexlib_b200_quantize_e4m3_fp16(const void* x, void* codes, void* scales, int R, int K,
                                   void* stream) {
  if (R < 0 || K <= 0 || R > kMostExtent || K > kMostExtent) return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (R == 0) return HEXLIB_B200_OK;
  if (!x || !codes || !scales || misaligned(x, 2) || misaligned(codes, 16) ||
      misaligned(scales, 4))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  HB_ENTRY_INIT();
  return hb::launch_quantize_e4m3(x, codes, scales, R, K, as_stream(stream));
}

int hexlib_b200_quantize_weight_e4m3_fp16(const void* w, void* codes, void* scales, int K, int N,
                                          void* stream) {
  if (K <= 0 || N <= 0 || K > kMostExtent || N > kMostExtent || !w || !codes || !scales || misaligned(w, 2) ||
      misaligned(codes, 16) || misaligned(scales, 4))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  HB_ENTRY_INIT();
  return hb::launch_quantize_weight_e4m3(w, codes, scales, K, N, as_stream(stream));
}

int hexlib_b200_dequant_e4m3_fp16(const void* codes, const void* scales, void* out, int R, int K,
                                  void* stream) {
  if (R < 0 || K <= 0 || R > kMostExtent || K > kMostExtent) return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (R == 0) return HEXLIB_B200_OK;
  if (!codes || !scales || !out || misaligned(codes, 16) || misaligned(scales, 4) ||
      misaligned(out, 2))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  HB_ENTRY_INIT();
  return hb::launch_dequant_e4m3(codes, scales, out, R, K, as_stream(stream));
}

static int matmul_e4m3(const void* a_codes, const void* a_scales, const void* w_codes,
                       const void* w_scales, const float* bias, const void* r, void* out, int M,
                       int K, int N, int act, void* stream) {
  if (M < 0 || K <= 0 || N <= 0 || M > kMostExtent || K > kMostExtent || N > kMostExtent || act < 0 ||
      act > 2)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (M == 0) return HEXLIB_B200_OK;
  if (!a_codes || !a_scales || !w_codes || !w_scales || !out || misaligned(a_codes, 16) ||
      misaligned(a_scales, 4) || misaligned(w_codes, 16) || misaligned(w_scales, 4) ||
      misaligned(bias, 4) || misaligned(r, 2) || misaligned(out, 2))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  HB_ENTRY_INIT();
  hb::GemmE4m3Desc g{};
  g.a = a_codes;
  g.a_scales = static_cast<const uint32_t*>(a_scales);
  g.w = w_codes;
  g.w_scales = static_cast<const uint32_t*>(w_scales);
  g.bias = bias;
  g.resid = r;
  g.out = out;
  g.M = M;
  g.K = K;
  g.N = N;
  g.act = act;
  return hb::launch_gemm_e4m3(g, hb::default_error_word(), as_stream(stream));
}

int hexlib_b200_matmul_epilogue_e4m3(const void* a_codes, const void* a_scales,
                                     const void* w_codes, const void* w_scales,
                                     const float* bias, void* out, int M, int K, int N, int act,
                                     void* stream) {
  return matmul_e4m3(a_codes, a_scales, w_codes, w_scales, bias, nullptr, out, M, K, N, act,
                     stream);
}

int hexlib_b200_matmul_epilogue_residual_e4m3(const void* a_codes, const void* a_scales,
                                              const void* w_codes, const void* w_scales,
                                              const float* bias, const void* r, void* out, int M,
                                              int K, int N, int act, void* stream) {
  if (M > 0 && !r) return HEXLIB_B200_ERR_INVAL_PARAMS;
  return matmul_e4m3(a_codes, a_scales, w_codes, w_scales, bias, r, out, M, K, N, act, stream);
}

static int edge(hb::EdgeDesc& d, bool e4m3, void* stream) {
  if (d.R < 0 || d.C <= 0 || d.R > kMostExtent || d.C > kMostExtent ||
      (d.norm != HEXLIB_B200_NORM_RMS && d.norm != HEXLIB_B200_NORM_LAYER) ||
      !(d.eps >= 0.f) || d.gate_act < HEXLIB_B200_GATE_NONE || d.gate_act > HEXLIB_B200_GATE_TANH)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (d.R == 0) return HEXLIB_B200_OK;
  if (e4m3 && (!d.h_codes != !d.h_scales)) return HEXLIB_B200_ERR_INVAL_PARAMS;
  const bool has_h = e4m3 ? d.h_codes != nullptr : d.h != nullptr;
  if (!d.x || has_h != (d.pre_w != nullptr) || (!d.pre_w && d.pre_b) || (!d.post_w && d.post_b))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (d.y ? !d.x_out : (d.post_w || d.gate || d.x_out || !has_h))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (d.gate ? (d.gate_rows <= 0 || d.R % d.gate_rows != 0) : (d.gate_rows != 0 || d.gate_act != 0))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (misaligned(d.x, 2) || misaligned(d.y, 2) || misaligned(d.x_out, 2) || misaligned(d.h, 2) ||
      misaligned(d.gate, 2) || misaligned(d.pre_w, 4) || misaligned(d.pre_b, 4) ||
      misaligned(d.post_w, 4) || misaligned(d.post_b, 4) || misaligned(d.h_codes, 16) ||
      misaligned(d.h_scales, 4))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  // in place: x_out on x or y, h on y; no other output shares
  auto shares = [](const void* p, std::initializer_list<const void*> with) {
    for (const void* q : with)
      if (p && p == q) return true;
    return false;
  };
  if (shares(d.h, {d.x, d.x_out}) || shares(d.h_codes, {d.x, d.y, d.x_out, d.h_scales}) ||
      shares(d.h_scales, {d.x, d.y, d.x_out}))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  for (const void* p : {d.gate, (const void*)d.pre_w, (const void*)d.pre_b, (const void*)d.post_w,
                        (const void*)d.post_b})
    if (shares(p, {d.x_out, d.h, d.h_codes, d.h_scales})) return HEXLIB_B200_ERR_INVAL_PARAMS;
  HB_ENTRY_INIT();
  d.err = hb::default_error_word();
  return hb::launch_edge(d, as_stream(stream));
}

static hb::EdgeDesc edge_desc(const void* x, const void* y, const float* post_w,
                              const float* post_b, const void* gate, int gate_rows, int gate_act,
                              float x_scale, float y_scale, void* x_out, const float* pre_w,
                              const float* pre_b, int R, int C, int norm, float eps) {
  hb::EdgeDesc d{};
  d.x = x;
  d.y = y;
  d.post_w = post_w;
  d.post_b = post_b;
  d.gate = gate;
  d.gate_rows = gate_rows;
  d.gate_act = gate_act;
  d.x_scale = x_scale;
  d.y_scale = y_scale;
  d.x_out = x_out;
  d.pre_w = pre_w;
  d.pre_b = pre_b;
  d.R = R;
  d.C = C;
  d.norm = norm;
  d.eps = eps;
  return d;
}

int hexlib_b200_norm_gate_residual_fp16(const void* x, const void* y, const float* post_w,
                                        const float* post_b, const void* gate, int gate_rows,
                                        int gate_act, float x_scale, float y_scale, void* x_out,
                                        const float* pre_w, const float* pre_b, void* h, int R,
                                        int C, int norm, float eps, void* stream) {
  hb::EdgeDesc d = edge_desc(x, y, post_w, post_b, gate, gate_rows, gate_act, x_scale, y_scale,
                             x_out, pre_w, pre_b, R, C, norm, eps);
  d.h = h;
  return edge(d, false, stream);
}

int hexlib_b200_norm_gate_residual_e4m3(const void* x, const void* y, const float* post_w,
                                        const float* post_b, const void* gate, int gate_rows,
                                        int gate_act, float x_scale, float y_scale, void* x_out,
                                        const float* pre_w, const float* pre_b, void* h_codes,
                                        void* h_scales, int R, int C, int norm, float eps,
                                        void* stream) {
  hb::EdgeDesc d = edge_desc(x, y, post_w, post_b, gate, gate_rows, gate_act, x_scale, y_scale,
                             x_out, pre_w, pre_b, R, C, norm, eps);
  d.h_codes = h_codes;
  d.h_scales = h_scales;
  return edge(d, true, stream);
}

int hexlib_b200_rope_pos_fp16(const void* x, int64_t x_stride, const int* positions, int n_axes,
                              const uint64_t* table, const int* axis, float mscale, void* y,
                              int64_t y_stride, int T, int H, int D, int rot, int layout,
                              void* stream) {
  if (T < 0 || H <= 0 || D <= 0 || T > kMostExtent || H > kMostExtent || D > kMostExtent || rot <= 0 ||
      (rot & 1) || rot > D || rot > hb::kRopePosMostRot || n_axes < 1 || n_axes > 4 ||
      (layout != HEXLIB_B200_ROPE_HALF && layout != HEXLIB_B200_ROPE_INTERLEAVED) ||
      x_stride < (int64_t)H * D || y_stride < (int64_t)H * D)
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  if (T == 0) return HEXLIB_B200_OK;
  if (!x || !y || !positions || !table || (x == y && x_stride != y_stride) || misaligned(x, 2) ||
      misaligned(y, 2) || misaligned(positions, 4) || misaligned(table, 8) || misaligned(axis, 4))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  HB_ENTRY_INIT();
  hb::RopePosDesc d{};
  d.x = x;
  d.x_stride = x_stride;
  d.positions = positions;
  d.n_axes = n_axes;
  d.table = table;
  d.axis = axis;
  d.mscale = mscale;
  d.y = y;
  d.y_stride = y_stride;
  d.T = T;
  d.H = H;
  d.D = D;
  d.rot = rot;
  d.layout = layout;
  return hb::launch_rope_pos(d, as_stream(stream));
}

int hexlib_b200_stream_status(void* stream) {
  if (cudaStreamSynchronize(as_stream(stream)) != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  bool noalloc_set = false;
  const int rc = hb::noalloc_take_error(&noalloc_set);
  const bool default_set = hb::take_default_error();
  if (rc != HEXLIB_B200_OK) return rc;
  return (default_set || noalloc_set) ? HEXLIB_B200_ERR_TIMEOUT : HEXLIB_B200_OK;
}

int hexlib_b200_diag_wait_timeout_stream(uint32_t limit_us, void* stream) {
  HB_ENTRY_INIT();
  return hb::launch_wait_timeout_probe(hb::default_error_word(), limit_us, as_stream(stream));
}

}  // extern "C"
