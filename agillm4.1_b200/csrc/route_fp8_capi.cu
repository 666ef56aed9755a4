// C ABI of general expert routing and of the block-scaled 8-bit path: argument
// checks, workspace layout and launch sequences.
#include <algorithm>
#include <string>

#include "fp8.cuh"
#include "kernels.h"

namespace {

int fail(int code, const std::string& msg) {
  agm::set_last_error(msg);
  return code;
}

int done(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return AGM_OK;
  return fail(AGM_ERR_CUDA, std::string(where) + ": " + cudaGetErrorString(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool known_dtype(int dtype) { return dtype == AGM_F32 || dtype == AGM_BF16 || dtype == AGM_F16; }

int num_sms() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!cached[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cached[dev] = n;
  }
  return cached[dev];
}

int check_route(int dtype, int64_t n, int E, int k, int score) {
  if (!known_dtype(dtype)) return fail(AGM_ERR_ARG, "dtype must be AGM_F32, AGM_BF16 or AGM_F16");
  if (n < 0) return fail(AGM_ERR_ARG, "n_tokens < 0");
  if (E < 1 || E > AGM_ROUTE_MAX_EXPERTS) return fail(AGM_ERR_UNSUPPORTED, "number of experts must be in [1, 512]");
  if (k < 1 || k > E) return fail(AGM_ERR_ARG, "top_k must be in [1, n_experts]");
  if (k > AGM_ROUTE_MAX_TOPK) return fail(AGM_ERR_UNSUPPORTED, "top_k must be at most 32");
  if (score != AGM_ROUTE_SOFTMAX && score != AGM_ROUTE_SIGMOID)
    return fail(AGM_ERR_ARG, "score must be AGM_ROUTE_SOFTMAX or AGM_ROUTE_SIGMOID");
  return AGM_OK;
}

int check_block_matrix(int64_t rows, int width) {
  if (rows < 0) return fail(AGM_ERR_ARG, "negative number of rows");
  if (width <= 0 || width % 16) return fail(AGM_ERR_UNSUPPORTED, "width must be a positive multiple of 16");
  return AGM_OK;
}

struct Carver {
  uint8_t* base;
  size_t off = 0;
  template <typename P>
  P* take(size_t bytes) {
    off = (off + 255) & ~size_t(255);
    P* p = reinterpret_cast<P*>(base ? base + off : nullptr);
    off += bytes;
    return p;
  }
};

// Rows of the padded segments: every expert that can have rows may leave 127 unused.
int64_t segment_rows(int64_t slots, int E) {
  return (slots + std::min<int64_t>(E, slots) * 127 + 127) / 128 * 128;
}

struct ExpertsLayout {
  int* err;
  int32_t* block_hist;
  int32_t* counts;
  int32_t* seg_start;
  int32_t* row_of;
  int32_t* sync;  // ticket, then finished units per 128-row block (few rows per expert)
  int n_sync;
  uint8_t* xq;
  uint8_t* xs;
  uint8_t* hq;
  uint8_t* hs;
  void* y;
  size_t bytes;
};

ExpertsLayout carve(void* ws, int64_t n, int d, int E, int k, int H) {
  Carver c{static_cast<uint8_t*>(ws)};
  ExpertsLayout L;
  const int64_t rows = segment_rows(n * k, E);
  L.err = c.take<int>(sizeof(int));
  L.block_hist = c.take<int32_t>(sizeof(int32_t) * agm_dispatch_blocks(n) * E);
  L.counts = c.take<int32_t>(sizeof(int32_t) * E);
  L.seg_start = c.take<int32_t>(sizeof(int32_t) * (E + 1));
  L.row_of = c.take<int32_t>(sizeof(int32_t) * n * k);
  L.n_sync = agm::fp8_rows_pay(n * k, E) ? 0 : 1 + static_cast<int>(rows / 128);
  L.sync = c.take<int32_t>(sizeof(int32_t) * L.n_sync);
  L.xq = c.take<uint8_t>(static_cast<size_t>(rows) * d);
  L.xs = c.take<uint8_t>(agm_fp8_scale_bytes(rows, d));
  L.hq = c.take<uint8_t>(static_cast<size_t>(rows) * H);
  L.hs = c.take<uint8_t>(agm_fp8_scale_bytes(rows, H));
  L.y = c.take<void>(static_cast<size_t>(rows) * d * 2);
  L.bytes = (c.off + 255) & ~size_t(255);
  return L;
}

}  // namespace

extern "C" {

int agm_route_experts(const void* logits, int dtype, int64_t n_tokens, int n_experts, int top_k, int score,
                      const float* bias, int n_groups, int top_groups, int renormalize, float scale, int32_t* idx,
                      float* weights, void* stream) {
  if (int rc = check_route(dtype, n_tokens, n_experts, top_k, score)) return rc;
  if (n_groups < 1 || n_groups > 32 || n_experts % n_groups)
    return fail(AGM_ERR_ARG, "n_groups must be in [1, 32] and divide n_experts");
  if (top_groups < 1 || top_groups > n_groups) return fail(AGM_ERR_ARG, "top_groups must be in [1, n_groups]");
  if (n_tokens == 0) return AGM_OK;
  if (!logits || !idx || !weights) return fail(AGM_ERR_ARG, "null pointer argument");
  const agm::RouteArgs a{n_tokens, n_experts, top_k, score, n_groups, top_groups, renormalize != 0, scale, bias};
  return done(agm::route_experts(dtype, logits, a, idx, weights, num_sms(), static_cast<cudaStream_t>(stream)),
              "route_experts");
}

int agm_route_experts_backward(const float* dweights, const void* logits, int dtype, int64_t n_tokens, int n_experts,
                               int top_k, const int32_t* idx, int score, int renormalize, float scale, void* dlogits,
                               void* stream) {
  if (int rc = check_route(dtype, n_tokens, n_experts, top_k, score)) return rc;
  if (n_tokens == 0) return AGM_OK;
  if (!dweights || !logits || !idx || !dlogits) return fail(AGM_ERR_ARG, "null pointer argument");
  const agm::RouteArgs a{n_tokens, n_experts, top_k, score, 1, 1, renormalize != 0, scale, nullptr};
  return done(agm::route_experts_backward(dtype, dweights, logits, idx, a, dlogits, num_sms(),
                                          static_cast<cudaStream_t>(stream)),
              "route_experts_backward");
}

size_t agm_fp8_scale_bytes(int64_t rows, int width) {
  if (rows <= 0 || width <= 0) return 0;
  return static_cast<size_t>((rows + 127) / 128) * agm::scale_k4(width) * agm::kScaleTile;
}

int agm_quantize_fp8(const void* x, int dtype, int64_t rows, int width, void* q, void* scales, void* stream) {
  if (!known_dtype(dtype)) return fail(AGM_ERR_ARG, "dtype must be AGM_F32, AGM_BF16 or AGM_F16");
  if (int rc = check_block_matrix(rows, width)) return rc;
  if (rows == 0) return AGM_OK;
  if (!x || !q || !scales) return fail(AGM_ERR_ARG, "null pointer argument");
  if (!aligned16(x) || !aligned16(q) || !aligned16(scales)) return fail(AGM_ERR_ARG, "x, q and scales must be 16-byte aligned");
  return done(agm::quantize_fp8_rows(dtype, x, rows, width, q, scales, num_sms(), static_cast<cudaStream_t>(stream)),
              "quantize_fp8");
}

int agm_quantize_fp8_weight(const void* w, int dtype, int64_t groups, int n, int width, void* q, void* scales,
                            void* stream) {
  if (!known_dtype(dtype)) return fail(AGM_ERR_ARG, "dtype must be AGM_F32, AGM_BF16 or AGM_F16");
  if (int rc = check_block_matrix(n, width)) return rc;
  if (groups < 0) return fail(AGM_ERR_ARG, "groups < 0");
  if (groups == 0 || n == 0) return AGM_OK;
  if (groups > 65535 || (n + 127) / 128 > 65535) return fail(AGM_ERR_UNSUPPORTED, "too many groups or rows");
  if (!w || !q || !scales) return fail(AGM_ERR_ARG, "null pointer argument");
  if (!aligned16(w) || !aligned16(q) || !aligned16(scales)) return fail(AGM_ERR_ARG, "w, q and scales must be 16-byte aligned");
  return done(agm::quantize_fp8_weight(dtype, w, groups, n, width, q, scales, static_cast<cudaStream_t>(stream)),
              "quantize_fp8_weight");
}

int agm_dequantize_fp8(const void* q, const void* scales, int64_t groups, int64_t rows, int width, int dtype, void* out,
                       void* stream) {
  if (!known_dtype(dtype)) return fail(AGM_ERR_ARG, "dtype must be AGM_F32, AGM_BF16 or AGM_F16");
  if (int rc = check_block_matrix(rows, width)) return rc;
  if (groups < 0) return fail(AGM_ERR_ARG, "groups < 0");
  if (groups == 0 || rows == 0) return AGM_OK;
  if (!q || !scales || !out) return fail(AGM_ERR_ARG, "null pointer argument");
  if (!aligned16(q) || !aligned16(scales) || !aligned16(out))
    return fail(AGM_ERR_ARG, "q, scales and out must be 16-byte aligned");
  return done(agm::dequantize_fp8(dtype, q, scales, groups, rows, width, out, num_sms(),
                                  static_cast<cudaStream_t>(stream)),
              "dequantize_fp8");
}

int agm_grouped_gemm_fp8(const void* a, const void* a_scales, int64_t a_rows, const void* w, const void* w_scales,
                         const float* bias, int groups, int n_out, int k_in, const int32_t* seg_start,
                         const int32_t* counts, int relu, int mode, void* c, int c_dtype, void* c_scales, int* err,
                         void* stream) {
  if (!c_scales && c_dtype != AGM_BF16 && c_dtype != AGM_F16)
    return fail(AGM_ERR_ARG, "c_dtype must be AGM_BF16 or AGM_F16 (or c_scales given)");
  if (mode != AGM_FP8_AUTO && mode != AGM_FP8_ROWS && mode != AGM_FP8_WEIGHTS)
    return fail(AGM_ERR_ARG, "mode must be AGM_FP8_AUTO, AGM_FP8_ROWS or AGM_FP8_WEIGHTS");
  if (groups < 1 || groups > AGM_ROUTE_MAX_EXPERTS) return fail(AGM_ERR_UNSUPPORTED, "groups must be in [1, 512]");
  if (!seg_start != !counts) return fail(AGM_ERR_ARG, "seg_start and counts go together");
  if (!counts && groups != 1) return fail(AGM_ERR_ARG, "several groups need seg_start and counts");
  if (int rc = check_block_matrix(a_rows, k_in)) return rc;
  if (n_out <= 0 || n_out % 16) return fail(AGM_ERR_UNSUPPORTED, "n_out must be a positive multiple of 16");
  if (a_rows > INT32_MAX - 256) return fail(AGM_ERR_UNSUPPORTED, "too many rows for int32 indices");
  if (a_rows == 0) return AGM_OK;
  if (!a || !a_scales || !w || !w_scales || !c) return fail(AGM_ERR_ARG, "null pointer argument");
  const void* ptrs[] = {a, a_scales, w, w_scales, c, bias, c_scales};
  for (const void* p : ptrs)
    if (!aligned16(p)) return fail(AGM_ERR_ARG, "all tensors must be 16-byte aligned");
  agm::Fp8GemmArgs g;
  g.a = a;
  g.a_scales = a_scales;
  g.a_rows = a_rows;
  g.w = w;
  g.w_scales = w_scales;
  g.bias = bias;
  g.groups = groups;
  g.n = n_out;
  g.k = k_in;
  g.seg_start = seg_start;
  g.counts = counts;
  // The counts are on the device: of every segment's last tile, take half as padding.
  g.live_rows = counts ? std::max<int64_t>(1, a_rows - 64 * static_cast<int64_t>(groups)) : a_rows;
  g.relu = relu != 0;
  g.zero_pad = counts != nullptr;
  g.c = c;
  g.c_scales = c_scales;
  g.err = err;
  return done(agm::grouped_gemm_fp8(c_dtype, g, mode, num_sms(), static_cast<cudaStream_t>(stream)),
              "grouped_gemm_fp8");
}

size_t agm_moe_experts_fp8_workspace_bytes(int64_t n_tokens, int d, int n_experts, int top_k, int hidden) {
  if (n_tokens < 0 || d <= 0 || n_experts < 1 || top_k < 1 || hidden <= 0) return 0;
  return carve(nullptr, n_tokens, d, n_experts, top_k, hidden).bytes;
}

int agm_moe_experts_fp8(const void* x, int dtype, int64_t n_tokens, int d, int n_experts, int top_k, int hidden,
                        const int32_t* idx, const float* weights, const void* w1, const void* s1, const float* b1,
                        const void* w2, const void* s2, const float* b2, const void* residual, void* out,
                        void* workspace, size_t workspace_bytes, void* stream) {
  return agm_moe_experts_fp8_shared(x, dtype, n_tokens, d, n_experts, top_k, hidden, idx, weights, w1, s1, b1, w2, s2,
                                    b2, residual, nullptr, 0, out, workspace, workspace_bytes, stream);
}

int agm_moe_experts_fp8_shared(const void* x, int dtype, int64_t n_tokens, int d, int n_experts, int top_k, int hidden,
                               const int32_t* idx, const float* weights, const void* w1, const void* s1,
                               const float* b1, const void* w2, const void* s2, const float* b2, const void* residual,
                               const void* shared, int n_shared, void* out, void* workspace, size_t workspace_bytes,
                               void* stream_) {
  if (dtype != AGM_BF16 && dtype != AGM_F16) return fail(AGM_ERR_UNSUPPORTED, "dtype must be AGM_BF16 or AGM_F16");
  if (n_tokens < 0) return fail(AGM_ERR_ARG, "n_tokens < 0");
  if (d <= 0 || d % 16 || hidden <= 0 || hidden % 16)
    return fail(AGM_ERR_UNSUPPORTED, "d and hidden must be positive multiples of 16");
  if (n_experts < 1 || n_experts > AGM_ROUTE_MAX_EXPERTS)
    return fail(AGM_ERR_UNSUPPORTED, "number of experts must be in [1, 512]");
  if (top_k < 1 || top_k > AGM_ROUTE_MAX_TOPK) return fail(AGM_ERR_ARG, "top_k must be in [1, 32]");
  if (n_shared < 0) return fail(AGM_ERR_ARG, "n_shared < 0");
  if (!workspace) return fail(AGM_ERR_ARG, "null pointer argument");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (n_tokens > INT32_MAX / top_k || segment_rows(n_tokens * top_k, n_experts) > INT32_MAX - 256)
    return fail(AGM_ERR_UNSUPPORTED, "too many rows for int32 indices");
  const ExpertsLayout L = carve(workspace, n_tokens, d, n_experts, top_k, hidden);
  if (L.bytes > workspace_bytes) return fail(AGM_ERR_WORKSPACE, "workspace too small");
  if (n_tokens > 0 && (!x || !idx || !weights || !w1 || !s1 || !b1 || !w2 || !s2 || !b2 || !out || (n_shared && !shared)))
    return fail(AGM_ERR_ARG, "null pointer argument");
  const void* ptrs[] = {x, w1, s1, b1, w2, s2, b2, residual, shared, out, workspace};
  for (const void* p : ptrs)
    if (!aligned16(p)) return fail(AGM_ERR_ARG, "all tensors must be 16-byte aligned");
  if (n_tokens == 0) return done(cudaMemsetAsync(L.err, 0, sizeof(int), stream), "memset");
  const int sms = num_sms();
  agm::Fp8Dispatch dsp;
  dsp.x = x;
  dsp.idx = idx;
  dsp.n = n_tokens;
  dsp.d = d;
  dsp.k = top_k;
  dsp.n_experts = n_experts;
  dsp.max_rows = segment_rows(n_tokens * top_k, n_experts);
  dsp.block_hist = L.block_hist;
  dsp.counts = L.counts;
  dsp.seg_start = L.seg_start;
  dsp.row_of = L.row_of;
  dsp.q = L.xq;
  dsp.scales = L.xs;
  dsp.err = L.err;
  dsp.zero = L.sync;
  dsp.n_zero = L.n_sync;
  cudaError_t e = agm::dispatch_fp8(dtype, dsp, sms, stream);  // clears the error word first
  if (e != cudaSuccess) return done(e, "dispatch_fp8");
  agm::Fp8GemmArgs g;
  g.a = L.xq;
  g.a_scales = L.xs;
  g.a_rows = dsp.max_rows;
  g.w = w1;
  g.w_scales = s1;
  g.bias = b1;
  g.groups = n_experts;
  g.n = hidden;
  g.k = d;
  g.seg_start = L.seg_start;
  g.counts = L.counts;
  g.live_rows = n_tokens * top_k;
  g.relu = true;
  g.c = L.hq;
  g.c_scales = L.hs;
  g.err = L.err;
  agm::Fp8GemmArgs h = g;
  h.a = L.hq;
  h.a_scales = L.hs;
  h.w = w2;
  h.w_scales = s2;
  h.bias = b2;
  h.n = d;
  h.k = hidden;
  h.relu = false;
  h.c = L.y;
  h.c_scales = nullptr;
  if (L.n_sync) {
    e = agm::expert_products_fp8(dtype, g, h, L.sync, L.sync + 1, sms, stream);
    if (e != cudaSuccess) return done(e, "expert_products_fp8");
  } else {
    e = agm::grouped_gemm_fp8(dtype, g, AGM_FP8_ROWS, sms, stream);
    if (e != cudaSuccess) return done(e, "grouped_gemm_fp8 fc1");
    e = agm::grouped_gemm_fp8(dtype, h, AGM_FP8_ROWS, sms, stream);
    if (e != cudaSuccess) return done(e, "grouped_gemm_fp8 fc2");
  }
  return done(agm::combine_weighted(dtype, L.y, L.row_of, weights, n_tokens, d, top_k, residual, shared, n_shared, out,
                                    sms, stream),
              "combine_weighted");
}

}  // extern "C"
