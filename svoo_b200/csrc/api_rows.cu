// extern "C" entry points of the token-wise operators: argument checks and launches.
#include "rows_common.cuh"

namespace svoo {
int64_t norm_backward_bytes(int64_t batch, int64_t rows, int groups, int C);
cudaError_t launch_layer_norm(int type, const NormArgs& a, cudaStream_t st);
cudaError_t launch_layer_norm_backward(int type, const NormArgs& a, int groups, void* dgain, void* doffset, cudaStream_t st);
cudaError_t launch_column_sum(const float* partial, int64_t parts, int64_t C, void* out, int out_type, cudaStream_t st);
cudaError_t launch_quantize_rows(int type, const void* x, int64_t M, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, float* scale,
                                 int64_t scale_pitch, cudaStream_t st);
cudaError_t launch_quantize_columns(int type, const void* x, int64_t M, int64_t K, int64_t row_stride, void* qt, int64_t qt_pitch,
                                    float* scale, int64_t scale_pitch, float* column_sum, cudaStream_t st);
cudaError_t launch_quantize_both(int type, const void* x, int64_t M, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, float* scale,
                                 int64_t scale_pitch, void* qt, int64_t qt_pitch, float* scale_t, int64_t scale_t_pitch, float* column_sum,
                                 cudaStream_t st);
cudaError_t launch_quantize_blocks(int type, const void* w, int64_t N, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, void* qt,
                                   int64_t qt_pitch, float* scale, cudaStream_t st);
cudaError_t launch_linear(const void* a, int64_t a_pitch, const float* sa, int64_t sa_pitch, const void* b, int64_t b_pitch, const float* sb,
                             int64_t sb_n, int64_t sb_k, bool row_scales, const void* bias, int bias_type, int64_t M, int64_t N, int64_t K,
                             bool gelu, int out_type, void* out, int64_t out_pitch, float* out_scale, int64_t out_scale_pitch, cudaStream_t st);
bool linear_few_rows(int64_t M, int64_t K, int out_type);
cudaError_t launch_linear_few_rows(int x_type, const void* x, int64_t x_row, const void* b, int64_t b_pitch, const float* sb, int64_t sb_n,
                                   int64_t sb_k, const void* bias, int bias_type, int64_t M, int64_t N, int64_t K, bool gelu, int out_type,
                                   void* out, int64_t out_pitch, cudaStream_t st);
cudaError_t read_linear_status(int32_t* out, cudaStream_t st);
}  // namespace svoo

using namespace svoo;

namespace {
constexpr int64_t kMaxRows = 1 << 26;            // rows and columns of a matrix: tile coordinates are 32-bit ints
bool aligned(const void* p, int to) { return (uintptr_t)p % to == 0; }
bool element(int type) { return type == SVOO_TYPE_BF16 || type == SVOO_TYPE_FP16 || type == SVOO_TYPE_FP32; }

int check_norm(int32_t x_type, int64_t batch, int64_t rows, int64_t C, int64_t x_batch, int64_t x_row, int32_t param_type, bool per_sample) {
  if (!element(x_type) || (param_type != SVOO_TYPE_FP32 && param_type != x_type)) return SVOO_ERR_TYPE;
  if (batch < 0 || rows < 0 || C < 1 || C > SVOO_MAX_NORM_COLUMNS || x_batch < 0 || x_row < 0) return SVOO_ERR_SHAPE;
  if (rows > kMaxRows || batch > kMaxRows || batch * rows > (int64_t)INT32_MAX - (1 << 20) || (per_sample && batch > 65535)) return SVOO_ERR_SHAPE;
  return SVOO_OK;
}
int check_quant(const void* x, int32_t type, int64_t M, int64_t K, int64_t x_row, const void* q, int64_t q_pitch, int64_t q_cols, const float* scale) {
  if (!element(type)) return SVOO_ERR_TYPE;
  if (M < 0 || K < 1 || M > kMaxRows || K > kMaxRows || x_row < 0 || q_pitch < q_cols || q_pitch % 16) return SVOO_ERR_SHAPE;
  if (M * ceil_div64(K, 128) > (int64_t)INT32_MAX - 1024) return SVOO_ERR_SHAPE;     // blocks are counted in 32 bits
  if (M == 0) return SVOO_OK;
  if (!x || !q || !scale) return SVOO_ERR_NULL;
  if (!aligned(q, 16) || !aligned(x, elem_bytes(type)) || !aligned(scale, 4)) return SVOO_ERR_ALIGN;
  return SVOO_OK;
}
int check_mm(const void* a, int64_t a_pitch, const float* a_scale, int64_t a_scale_pitch, const void* b, int64_t b_pitch, const float* b_scale,
             int64_t b_scale_n, int64_t b_scale_k, int32_t b_scale_rows, const void* bias, int32_t bias_type, int64_t M, int64_t N, int64_t K,
             int32_t activation, void* out, int32_t out_type, int64_t out_pitch, float* out_scale, int64_t out_scale_pitch) {
  const bool quantised = out_type == SVOO_TYPE_E4M3, gelu = activation == SVOO_ACT_GELU_TANH;
  if (!element(out_type) && !quantised) return SVOO_ERR_TYPE;
  if ((bias && !element(bias_type)) || (!gelu && activation != SVOO_ACT_NONE)) return SVOO_ERR_TYPE;
  if (b_scale_rows && (bias || gelu || quantised)) return SVOO_ERR_TYPE;
  if (M < 0 || N < 1 || K < 1 || M > kMaxRows || N > kMaxRows || K > kMaxRows) return SVOO_ERR_SHAPE;
  if (ceil_div64(M, 128) * ceil_div64(N, 128) > (int64_t)INT32_MAX / 2) return SVOO_ERR_SHAPE;
  if (a_pitch < K || b_pitch < K || a_pitch % 16 || b_pitch % 16 || a_scale_pitch < M || b_scale_n < 0 || b_scale_k < 0 || out_pitch < N)
    return SVOO_ERR_SHAPE;
  if (b_scale_rows && (b_scale_k < N || b_scale_k % 4)) return SVOO_ERR_SHAPE;
  if (quantised && (out_pitch % 16 || out_scale_pitch < M)) return SVOO_ERR_SHAPE;
  if (M == 0) return SVOO_OK;
  if (!a || !a_scale || !b || !b_scale || !out || (quantised && !out_scale)) return SVOO_ERR_NULL;
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(a_scale, 4) || !aligned(b_scale, b_scale_rows ? 16 : 4) ||
      !aligned(out, quantised ? 16 : elem_bytes(out_type)) || !aligned(out_scale, 4) || (bias && !aligned(bias, elem_bytes(bias_type))))
    return SVOO_ERR_ALIGN;
  return SVOO_OK;
}
// the byte behind the last element of a tensor [batch, rows, C]
const void* end_of(const void* p, int64_t batch, int64_t rows, int64_t C, int64_t batch_stride, int64_t row_stride, int e) {
  return static_cast<const char*>(p) + ((batch - 1) * batch_stride + (rows - 1) * row_stride + C) * e;
}
int64_t norm_groups(int64_t batch, int32_t per_sample) { return per_sample && batch > 1 ? batch : 1; }
// Where a training step keeps things: offsets in `saved`, in forward's and in backward's scratch.
struct TrainLayout {
  int64_t mp, np, kp, mb, nb, kb, xs, ys;        // rows in bytes, blocks, pitches of the column scales
  int64_t wt, w_scale, xt, xt_scale, saved;
  int64_t w_q, x_q, x_scale, forward;
  int64_t g_q, g_scale, gt, gt_scale, part, backward;
  TrainLayout(int64_t M, int64_t N, int64_t K, bool keep_x, bool keep_w) {
    mp = align_up(M, 16), np = align_up(N, 16), kp = align_up(K, 16);
    mb = ceil_div64(M, 128), nb = ceil_div64(N, 128), kb = ceil_div64(K, 128), xs = align_up(K, 4), ys = align_up(N, 4);
    int64_t at = 0;
    auto take = [&at](int64_t bytes) { const int64_t here = at; at += align_up(bytes, 256); return here; };
    wt = take(keep_x ? K * np : 0), w_scale = take(nb * kb * 4), xt = take(keep_w ? K * mp : 0), xt_scale = take(keep_w ? mb * xs * 4 : 0);
    saved = at, at = 0;
    w_q = take(N * kp), x_q = take(M * kp), x_scale = take(kb * M * 4);
    forward = at, at = 0;
    g_q = take(M * np), g_scale = take(nb * M * 4), gt = take(N * mp), gt_scale = take(mb * ys * 4), part = take(mb * N * 4);
    backward = at;
  }
};
int check_train(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1 || M > kMaxRows || N > kMaxRows || K > kMaxRows) return SVOO_ERR_SHAPE;
  const int64_t mb = ceil_div64(M, 128), nb = ceil_div64(N, 128), kb = ceil_div64(K, 128);
  if (mb > 65535 || nb > 65535 || M * kb > (int64_t)INT32_MAX - 1024 || M * nb > (int64_t)INT32_MAX - 1024 || mb * nb > INT32_MAX / 2 ||
      mb * kb > INT32_MAX / 2 || nb * kb > INT32_MAX / 2)
    return SVOO_ERR_SHAPE;
  return SVOO_OK;
}
#define SVOO_CUDA(expr) do { cudaError_t _e = (expr); if (_e != cudaSuccess) return (int)_e; } while (0)
#define SVOO_TRY(expr) do { int _rc = (expr); if (_rc != SVOO_OK) return _rc; } while (0)
}  // namespace

extern "C" {

int svoo_b200_layer_norm(const void* x, int32_t x_type, int64_t batch, int64_t rows, int64_t C, int64_t x_batch, int64_t x_row,
                         const void* gain, int64_t gain_batch, const void* offset, int64_t offset_batch, int32_t param_type,
                         int32_t gain_plus_one, float eps, void* y, float* mean, float* rstd, void* stream) {
  SVOO_TRY(check_norm(x_type, batch, rows, C, x_batch, x_row, param_type, gain_batch != 0 || offset_batch != 0));
  if (batch * rows == 0) return SVOO_OK;
  if (!x || !y || !mean != !rstd) return SVOO_ERR_NULL;
  if (gain_batch < 0 || offset_batch < 0) return SVOO_ERR_SHAPE;
  const int e = elem_bytes(x_type), pe = elem_bytes(param_type);
  if (!aligned(x, e) || !aligned(y, e) || !aligned(gain, pe) || !aligned(offset, pe)) return SVOO_ERR_ALIGN;
  NormArgs a = {};
  a.x = x, a.y = y, a.gain = gain, a.offset = offset, a.mean = mean, a.rstd = rstd;
  a.x_batch = batch == 1 ? 0 : x_batch, a.x_row = x_row, a.gain_batch = gain_batch, a.offset_batch = offset_batch;
  a.batch = batch, a.rows = rows, a.C = (int)C, a.params_fp32 = param_type == SVOO_TYPE_FP32, a.plus_one = gain_plus_one != 0, a.eps = eps;
  a.x_end = end_of(x, batch, rows, C, a.x_batch, x_row, e);
  if (!(a.status = rows_status_word())) return (int)cudaErrorInvalidDevice;
  return (int)launch_layer_norm(x_type, a, (cudaStream_t)stream);
}

int svoo_b200_layer_norm_workspace_bytes(int64_t batch, int64_t rows, int64_t C, int32_t per_sample, int64_t* bytes_out) {
  if (!bytes_out) return SVOO_ERR_NULL;
  SVOO_TRY(check_norm(SVOO_TYPE_FP32, batch, rows, C, 0, 0, SVOO_TYPE_FP32, per_sample != 0));
  const int64_t groups = norm_groups(batch, per_sample);
  *bytes_out = norm_backward_bytes(batch, rows, (int)groups, (int)C);
  return SVOO_OK;
}

int svoo_b200_layer_norm_backward(const void* dy, int64_t dy_batch, int64_t dy_row, const void* x, int32_t x_type, int64_t batch,
                                  int64_t rows, int64_t C, int64_t x_batch, int64_t x_row, const float* mean, const float* rstd,
                                  const void* gain, int64_t gain_batch, int32_t param_type, int32_t gain_plus_one,
                                  int32_t per_sample, void* dx, void* dgain, void* doffset, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const bool own_gain = batch > 1 && gain_batch != 0;       // a gain for every sample, as the forward call has it
  SVOO_TRY(check_norm(x_type, batch, rows, C, x_batch, x_row, param_type, per_sample != 0 || own_gain));
  if (own_gain && !per_sample && dgain) return SVOO_ERR_SHAPE;
  if (dy_batch < 0 || dy_row < 0 || gain_batch < 0) return SVOO_ERR_SHAPE;
  if (!dgain != !doffset || (dgain && !workspace)) return SVOO_ERR_NULL;
  if (batch == 0) return SVOO_OK;                          // no sample, no sums of one; shared sums are the caller's to clear
  if (batch * rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return SVOO_ERR_NULL;
  if (batch * rows == 0 && !dgain) return SVOO_OK;
  const int e = elem_bytes(x_type), pe = elem_bytes(param_type);
  if (!aligned(x, e) || !aligned(dy, e) || !aligned(dx, e) || !aligned(gain, pe) || !aligned(dgain, pe) || !aligned(doffset, pe) ||
      !aligned(workspace, 4) || !aligned(mean, 4) || !aligned(rstd, 4))
    return SVOO_ERR_ALIGN;
  const int64_t groups = norm_groups(batch, per_sample || own_gain);
  if (dgain && workspace_bytes < norm_backward_bytes(batch, rows, (int)groups, (int)C)) return SVOO_ERR_WORKSPACE;
  NormArgs a = {};
  a.x = x, a.dy = dy, a.dx = dx, a.gain = gain, a.mean_in = mean, a.rstd_in = rstd, a.partial = dgain ? (float*)workspace : nullptr;
  a.x_batch = batch == 1 ? 0 : x_batch, a.x_row = x_row, a.dy_batch = batch == 1 ? 0 : dy_batch, a.dy_row = dy_row;
  a.gain_batch = groups > 1 ? gain_batch : 0;
  a.batch = batch, a.rows = rows, a.C = (int)C, a.params_fp32 = param_type == SVOO_TYPE_FP32, a.plus_one = gain_plus_one != 0;
  a.x_end = end_of(x, batch, rows, C, a.x_batch, x_row, e);
  a.dy_end = end_of(dy, batch, rows, C, a.dy_batch, dy_row, e);
  if (!(a.status = rows_status_word())) return (int)cudaErrorInvalidDevice;
  return (int)launch_layer_norm_backward(x_type, a, (int)groups, dgain, doffset, (cudaStream_t)stream);
}

int svoo_b200_quantize_rows(const void* x, int32_t x_type, int64_t M, int64_t K, int64_t x_row, void* q, int64_t q_pitch, float* scale,
                            int64_t scale_pitch, void* stream) {
  SVOO_TRY(check_quant(x, x_type, M, K, x_row, q, q_pitch, K, scale));
  if (scale_pitch < M) return SVOO_ERR_SHAPE;
  if (M == 0) return SVOO_OK;
  return (int)launch_quantize_rows(x_type, x, M, K, x_row, q, q_pitch, scale, scale_pitch, (cudaStream_t)stream);
}

int svoo_b200_quantize_columns(const void* x, int32_t x_type, int64_t M, int64_t K, int64_t x_row, void* q, int64_t q_pitch,
                               float* scale, int64_t scale_pitch, float* column_sums, void* stream) {
  SVOO_TRY(check_quant(x, x_type, M, K, x_row, q, q_pitch, M, scale));
  if (scale_pitch < K || ceil_div64(M, 128) > 65535) return SVOO_ERR_SHAPE;
  if (column_sums && !aligned(column_sums, 4)) return SVOO_ERR_ALIGN;
  if (M == 0) return SVOO_OK;
  return (int)launch_quantize_columns(x_type, x, M, K, x_row, q, q_pitch, scale, scale_pitch, column_sums, (cudaStream_t)stream);
}

int svoo_b200_quantize_blocks(const void* x, int32_t x_type, int64_t M, int64_t K, int64_t x_row, void* q, int64_t q_pitch, void* qt,
                              int64_t qt_pitch, float* scale, void* stream) {
  SVOO_TRY(check_quant(x, x_type, M, K, x_row, q, q_pitch, K, scale));
  if (ceil_div64(M, 128) > 65535 || (qt && (qt_pitch < M || qt_pitch % 16))) return SVOO_ERR_SHAPE;
  if (qt && !aligned(qt, 16)) return SVOO_ERR_ALIGN;
  if (M == 0) return SVOO_OK;
  return (int)launch_quantize_blocks(x_type, x, M, K, x_row, q, q_pitch, qt, qt_pitch, scale, (cudaStream_t)stream);
}

int svoo_b200_quantize_both(const void* x, int32_t x_type, int64_t M, int64_t K, int64_t x_row, void* q, int64_t q_pitch, float* scale,
                            int64_t scale_pitch, void* qt, int64_t qt_pitch, float* scale_t, int64_t scale_t_pitch, float* column_sums,
                            void* stream) {
  SVOO_TRY(check_quant(x, x_type, M, K, x_row, q, q_pitch, K, scale));
  SVOO_TRY(check_quant(x, x_type, M, K, x_row, qt, qt_pitch, M, scale_t));
  if (scale_pitch < M || scale_t_pitch < K || ceil_div64(M, 128) > 65535) return SVOO_ERR_SHAPE;
  if (column_sums && !aligned(column_sums, 4)) return SVOO_ERR_ALIGN;
  if (M == 0) return SVOO_OK;
  return (int)launch_quantize_both(x_type, x, M, K, x_row, q, q_pitch, scale, scale_pitch, qt, qt_pitch, scale_t, scale_t_pitch, column_sums,
                                   (cudaStream_t)stream);
}

int svoo_b200_column_sum(const float* partial, int64_t parts, int64_t C, void* out, int32_t out_type, void* stream) {
  if (!element(out_type)) return SVOO_ERR_TYPE;
  if (parts < 0 || parts > INT32_MAX || C < 1 || C > kMaxRows) return SVOO_ERR_SHAPE;
  if ((parts && !partial) || !out) return SVOO_ERR_NULL;
  if (!aligned(partial, 4) || !aligned(out, elem_bytes(out_type))) return SVOO_ERR_ALIGN;
  return (int)launch_column_sum(partial, parts, C, out, out_type, (cudaStream_t)stream);
}

int svoo_b200_mm_fp8(const void* a, int64_t a_pitch, const float* a_scale, int64_t a_scale_pitch, const void* b, int64_t b_pitch,
                     const float* b_scale, int64_t b_scale_n, int64_t b_scale_k, int32_t b_scale_rows, const void* bias,
                     int32_t bias_type, int64_t M, int64_t N, int64_t K, int32_t activation, void* out, int32_t out_type,
                     int64_t out_pitch, float* out_scale, int64_t out_scale_pitch, void* stream) {
  SVOO_TRY(check_mm(a, a_pitch, a_scale, a_scale_pitch, b, b_pitch, b_scale, b_scale_n, b_scale_k, b_scale_rows, bias, bias_type, M, N, K,
                    activation, out, out_type, out_pitch, out_scale, out_scale_pitch));
  if (M == 0) return SVOO_OK;
  return (int)launch_linear(a, a_pitch, a_scale, a_scale_pitch, b, b_pitch, b_scale, b_scale_n, b_scale_k, b_scale_rows != 0, bias,
                               bias_type, M, N, K, activation == SVOO_ACT_GELU_TANH, out_type, out, out_pitch, out_scale, out_scale_pitch,
                            (cudaStream_t)stream);
}

int svoo_b200_linear_fp8_workspace_bytes(int64_t M, int64_t K, int32_t out_type, int64_t* bytes_out) {
  if (!bytes_out) return SVOO_ERR_NULL;
  if (M < 0 || K < 1 || M > kMaxRows || K > kMaxRows) return SVOO_ERR_SHAPE;
  *bytes_out = linear_few_rows(M, K, out_type) ? 0 : align_up(M * align_up(K, 16), 256) + ceil_div64(K, 128) * M * 4;
  return SVOO_OK;
}

int svoo_b200_linear_fp8(const void* x, int32_t x_type, int64_t M, int64_t K, int64_t x_row, const void* b, int64_t b_pitch,
                         const float* b_scale, int64_t b_scale_n, int64_t b_scale_k, const void* bias, int32_t bias_type, int64_t N,
                         int32_t activation, void* out, int32_t out_type, int64_t out_pitch, float* out_scale,
                         int64_t out_scale_pitch, void* workspace, int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  SVOO_TRY(svoo_b200_linear_fp8_workspace_bytes(M, K, out_type, &need));
  if (need && !workspace) return SVOO_ERR_NULL;
  if (workspace_bytes < need) return SVOO_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return SVOO_ERR_ALIGN;
  const int64_t pitch = align_up(K, 16);
  // the product's arguments are checked before anything is launched; without a workspace b stands in for the rows in it
  const void* rows = need ? workspace : b;
  float* scale = need ? reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up(M * pitch, 256)) : nullptr;
  const float* any_scale = need ? scale : b_scale;
  SVOO_TRY(check_quant(x, x_type, M, K, x_row, rows, pitch, K, any_scale));
  SVOO_TRY(check_mm(rows, pitch, any_scale, M, b, b_pitch, b_scale, b_scale_n, b_scale_k, 0, bias, bias_type, M, N, K, activation, out,
                    out_type, out_pitch, out_scale, out_scale_pitch));
  if (M == 0) return SVOO_OK;
  const bool gelu = activation == SVOO_ACT_GELU_TANH;
  if (!need)
    return (int)launch_linear_few_rows(x_type, x, x_row, b, b_pitch, b_scale, b_scale_n, b_scale_k, bias, bias_type, M, N, K, gelu, out_type,
                                       out, out_pitch, (cudaStream_t)stream);
  const cudaError_t e = launch_quantize_rows(x_type, x, M, K, x_row, workspace, pitch, scale, M, (cudaStream_t)stream);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_linear(workspace, pitch, scale, M, b, b_pitch, b_scale, b_scale_n, b_scale_k, false, bias, bias_type, M, N, K, gelu,
                            out_type, out, out_pitch, out_scale, out_scale_pitch, (cudaStream_t)stream);
}

int svoo_b200_linear_train_bytes(int64_t M, int64_t N, int64_t K, int32_t keep_x_grad, int32_t keep_w_grad, int64_t* bytes_out) {
  if (!bytes_out) return SVOO_ERR_NULL;
  SVOO_TRY(check_train(M, N, K));
  const TrainLayout l(M, N, K, keep_x_grad != 0, keep_w_grad != 0);
  bytes_out[0] = l.saved, bytes_out[1] = l.forward, bytes_out[2] = l.backward;
  return SVOO_OK;
}

int svoo_b200_linear_train_forward(const void* x, int32_t x_type, int64_t M, int64_t K, int64_t x_row, const void* w, int32_t w_type,
                                   int64_t N, int64_t w_row, const void* bias, int32_t bias_type, int32_t keep_x_grad,
                                   int32_t keep_w_grad, void* y, void* saved, int64_t saved_bytes, void* scratch,
                                   int64_t scratch_bytes, void* stream) {
  if (!element(x_type) || !element(w_type) || (bias && !element(bias_type))) return SVOO_ERR_TYPE;
  SVOO_TRY(check_train(M, N, K));
  if (x_row < 0 || w_row < 0) return SVOO_ERR_SHAPE;
  if (!x || !w || !y || !saved || !scratch) return SVOO_ERR_NULL;
  const TrainLayout l(M, N, K, keep_x_grad != 0, keep_w_grad != 0);
  if (saved_bytes < l.saved || scratch_bytes < l.forward) return SVOO_ERR_WORKSPACE;
  if (!aligned(x, elem_bytes(x_type)) || !aligned(w, elem_bytes(w_type)) || !aligned(y, elem_bytes(x_type)) || !aligned(saved, 16) ||
      !aligned(scratch, 16) || (bias && !aligned(bias, elem_bytes(bias_type))))
    return SVOO_ERR_ALIGN;
  char *k = static_cast<char*>(saved), *t = static_cast<char*>(scratch);
  float *w_scale = (float*)(k + l.w_scale), *x_scale = (float*)(t + l.x_scale);
  const cudaStream_t st = (cudaStream_t)stream;
  SVOO_CUDA(launch_quantize_blocks(w_type, w, N, K, w_row, t + l.w_q, l.kp, keep_x_grad ? k + l.wt : nullptr, l.np, w_scale, st));
  if (keep_w_grad)
    SVOO_CUDA(launch_quantize_both(x_type, x, M, K, x_row, t + l.x_q, l.kp, x_scale, M, k + l.xt, l.mp, (float*)(k + l.xt_scale), l.xs, nullptr, st));
  else
    SVOO_CUDA(launch_quantize_rows(x_type, x, M, K, x_row, t + l.x_q, l.kp, x_scale, M, st));
  return (int)launch_linear(t + l.x_q, l.kp, x_scale, M, t + l.w_q, l.kp, w_scale, l.kb, 1, false, bias, bias_type, M, N, K, false, x_type, y, N,
                            nullptr, 0, st);
}

int svoo_b200_linear_train_backward(const void* dy, int32_t x_type, int64_t M, int64_t N, int64_t K, int64_t dy_row, const void* saved,
                                    int64_t saved_bytes, int32_t keep_x_grad, int32_t keep_w_grad, void* dx, void* dw,
                                    int32_t w_type, void* db, int32_t bias_type, void* scratch, int64_t scratch_bytes,
                                    void* stream) {
  if (!element(x_type) || (dw && !element(w_type)) || (db && !element(bias_type))) return SVOO_ERR_TYPE;
  SVOO_TRY(check_train(M, N, K));
  if (dy_row < 0) return SVOO_ERR_SHAPE;
  if (!dy || !saved || !scratch || (dx && !keep_x_grad) || (dw && !keep_w_grad)) return SVOO_ERR_NULL;
  if (!dx && !dw && !db) return SVOO_OK;
  const TrainLayout l(M, N, K, keep_x_grad != 0, keep_w_grad != 0);
  if (saved_bytes < l.saved || scratch_bytes < l.backward) return SVOO_ERR_WORKSPACE;
  if (!aligned(dy, elem_bytes(x_type)) || !aligned(saved, 16) || !aligned(scratch, 16) || !aligned(dx, elem_bytes(x_type)) ||
      (dw && !aligned(dw, elem_bytes(w_type))) || (db && !aligned(db, elem_bytes(bias_type))))
    return SVOO_ERR_ALIGN;
  const char* k = static_cast<const char*>(saved);
  char* t = static_cast<char*>(scratch);
  const float* w_scale = (const float*)(k + l.w_scale);
  float *g_scale = (float*)(t + l.g_scale), *gt_scale = (float*)(t + l.gt_scale), *part = db ? (float*)(t + l.part) : nullptr;
  const cudaStream_t st = (cudaStream_t)stream;
  if (dx && (dw || db))
    SVOO_CUDA(launch_quantize_both(x_type, dy, M, N, dy_row, t + l.g_q, l.np, g_scale, M, t + l.gt, l.mp, gt_scale, l.ys, part, st));
  else if (dx)
    SVOO_CUDA(launch_quantize_rows(x_type, dy, M, N, dy_row, t + l.g_q, l.np, g_scale, M, st));
  else
    SVOO_CUDA(launch_quantize_columns(x_type, dy, M, N, dy_row, t + l.gt, l.mp, gt_scale, l.ys, part, st));
  if (db) SVOO_CUDA(launch_column_sum(part, l.mb, N, db, bias_type, st));
  if (dx)
    SVOO_CUDA(launch_linear(t + l.g_q, l.np, g_scale, M, k + l.wt, l.np, w_scale, 1, l.kb, false, nullptr, 0, M, K, N, false, x_type, dx, K, nullptr,
                            0, st));
  if (dw)
    SVOO_CUDA(launch_linear(t + l.gt, l.mp, gt_scale, l.ys, k + l.xt, l.mp, (const float*)(k + l.xt_scale), 1, l.xs, true, nullptr, 0, N, K, M,
                            false, w_type, dw, K, nullptr, 0, st));
  return SVOO_OK;
}

int svoo_b200_linear_status(int32_t* status, void* stream) {
  if (!status) return SVOO_ERR_NULL;
  return (int)read_linear_status(status, (cudaStream_t)stream);
}

}  // extern "C"
