// torch custom operators over the C ABI of libtaomate_w8a8.so.
//
// Registers torch.ops.taomate_w8a8.* with the argument order of the vLLM
// out-variant operators the reference calls through torch.ops._C
// (src/taomate_hd/inference/w8a8.py:22-35, :71-72).  Only a CUDA kernel is
// registered: CPU tensors raise (no CPU fallback).  Every op validates
// dtype/device/layout with TORCH_CHECK (RuntimeError in Python), launches on
// the current CUDA stream.  The only allocation is the split-K workspace of
// cutlass_scaled_mm / scaled_mm_i8_ex (cached per device and stream, from
// torch's caching allocator) for shapes that use split-K.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <utility>

#include "../../include/taomate_w8a8.h"

namespace {

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return TM_DTYPE_BF16;
    case at::kHalf: return TM_DTYPE_FP16;
    case at::kFloat: return TM_DTYPE_FP32;
    default: return -1;
  }
}

void check_status(int status, const char* op) {
  TORCH_CHECK(status == TM_OK, "taomate_w8a8.", op, " failed: ", tm_status_string(status),
              " (status ", status, ")");
}

void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

void check_cuda(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == ref.device(), name, " must be on ", ref.device());
}

// Treat `input` as [rows, cols] with unit inner stride and a row stride.
void as_rows(const at::Tensor& input, int64_t* rows, int64_t* cols, int64_t* ld) {
  TORCH_CHECK(input.dim() >= 1, "input must have at least one dimension");
  *cols = input.size(-1);
  if (input.dim() == 2 && input.stride(1) == 1) {
    *rows = input.size(0);
    *ld = input.size(0) > 1 ? input.stride(0) : *cols;
    return;
  }
  TORCH_CHECK(input.is_contiguous(), "input must be contiguous");
  *rows = *cols == 0 ? 0 : input.numel() / *cols;
  *ld = *cols;
}

void dynamic_scaled_int8_quant(at::Tensor& out, const at::Tensor& input, at::Tensor& scales,
                               const std::optional<at::Tensor>& azp) {
  check_cuda(input, input, "input");
  check_cuda(out, input, "result");
  check_cuda(scales, input, "scale");
  TORCH_CHECK(!azp.has_value(), "asymmetric int8 quantisation (azp) is not supported");
  const int dt = dtype_code(input);
  TORCH_CHECK(dt >= 0, "input dtype must be bfloat16, float16 or float32");
  TORCH_CHECK(out.scalar_type() == at::kChar && out.is_contiguous(), "result must be contiguous int8");
  TORCH_CHECK(out.numel() == input.numel(), "result must have the shape of input");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.is_contiguous(),
              "scale must be contiguous float32");
  int64_t rows, cols, ld;
  as_rows(input, &rows, &cols, &ld);
  TORCH_CHECK(scales.numel() == rows, "scale must hold one value per token");
  const c10::cuda::CUDAGuard guard(input.device());
  check_status(tm_dynamic_scaled_int8_quant(out.data_ptr<int8_t>(), input.data_ptr(), dt,
                                            scales.data_ptr<float>(), nullptr, rows, cols, ld,
                                            stream_of(input)),
               "dynamic_scaled_int8_quant");
}

void static_scaled_int8_quant(at::Tensor& out, const at::Tensor& input, const at::Tensor& scale,
                              const std::optional<at::Tensor>& azp) {
  check_cuda(input, input, "input");
  check_cuda(out, input, "result");
  check_cuda(scale, input, "scale");
  TORCH_CHECK(!azp.has_value(), "asymmetric int8 quantisation (azp) is not supported");
  const int dt = dtype_code(input);
  TORCH_CHECK(dt >= 0, "input dtype must be bfloat16, float16 or float32");
  TORCH_CHECK(out.scalar_type() == at::kChar && out.is_contiguous(), "result must be contiguous int8");
  TORCH_CHECK(out.numel() == input.numel(), "result must have the shape of input");
  TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.numel() == 1,
              "static scale must be one float32 value");
  int64_t rows, cols, ld;
  as_rows(input, &rows, &cols, &ld);
  const c10::cuda::CUDAGuard guard(input.device());
  check_status(tm_static_scaled_int8_quant(out.data_ptr<int8_t>(), input.data_ptr(), dt,
                                           scale.data_ptr<float>(), nullptr, rows, cols, ld,
                                           stream_of(input)),
               "static_scaled_int8_quant");
}

// Split-K workspace per (device, stream): zeroed when allocated, grown on
// demand, reused by every call on that stream (calls on one stream never
// overlap).  The kernels leave its counters at zero after each call.
at::Tensor splitk_workspace(const at::Tensor& like, uint64_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, cudaStream_t>, at::Tensor> cache;
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream(like.device().index()).stream();
  const std::pair<int, cudaStream_t> key{like.device().index(), stream};
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(key);
  if (it == cache.end() || static_cast<uint64_t>(it->second.numel()) < bytes) {
    at::Tensor ws = at::zeros({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
    cache[key] = ws;
    return ws;
  }
  return it->second;
}

void scaled_mm_common(at::Tensor& out, const at::Tensor& a, const at::Tensor& b,
                      const at::Tensor& a_scales, const at::Tensor& b_scales,
                      const std::optional<at::Tensor>& bias, int64_t epilogue,
                      const std::optional<at::Tensor>& acc_debug, int64_t tile_n,
                      const char* op) {
  check_cuda(a, a, "a");
  check_cuda(b, a, "b");
  check_cuda(out, a, "out");
  check_cuda(a_scales, a, "a_scales");
  check_cuda(b_scales, a, "b_scales");
  TORCH_CHECK(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar,
              "a and b must be int8");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && out.dim() == 2, "a, b and out must be 2-D");
  const int64_t m = a.size(0), k = a.size(1), n = b.size(1);
  TORCH_CHECK(b.size(0) == k, "a and b inner dimensions differ: ", k, " vs ", b.size(0));
  // SwiGLU: n interleaved (gate, up) columns in, n / 2 out
  const int64_t out_n = (epilogue & TM_EPI_SWIGLU) ? n / 2 : n;
  TORCH_CHECK(out.size(0) == m && out.size(1) == out_n, "out must be [", m, ", ", out_n, "]");
  TORCH_CHECK(a.stride(1) == 1, "a must be row-major");
  TORCH_CHECK(b.stride(0) == 1, "b must be column-major (pass weight.t())");
  TORCH_CHECK(out.stride(1) == 1, "out must be row-major");
  const int out_dt = dtype_code(out);
  TORCH_CHECK(out_dt == TM_DTYPE_BF16 || out_dt == TM_DTYPE_FP16, "out must be bfloat16 or float16");
  TORCH_CHECK(a_scales.scalar_type() == at::kFloat && b_scales.scalar_type() == at::kFloat,
              "scales must be float32");
  TORCH_CHECK(a_scales.is_contiguous() && b_scales.is_contiguous(), "scales must be contiguous");
  TORCH_CHECK(a_scales.numel() == 1 || a_scales.numel() == m, "a_scales must be per-tensor or per-token");
  TORCH_CHECK(b_scales.numel() == 1 || b_scales.numel() == n, "b_scales must be per-tensor or per-channel");
  const void* bias_ptr = nullptr;
  if (bias.has_value()) {
    check_cuda(*bias, a, "bias");
    TORCH_CHECK(bias->scalar_type() == out.scalar_type(), "bias must have the output dtype");
    TORCH_CHECK(bias->numel() == n && bias->is_contiguous(), "bias must be contiguous [n]");
    bias_ptr = bias->data_ptr();
  }
  int32_t* acc_ptr = nullptr;
  if (acc_debug.has_value()) {
    check_cuda(*acc_debug, a, "acc_debug");
    TORCH_CHECK(acc_debug->scalar_type() == at::kInt && acc_debug->is_contiguous() &&
                    acc_debug->numel() == m * n,
                "acc_debug must be a contiguous int32 [m, n]");
    acc_ptr = acc_debug->data_ptr<int32_t>();
  }
  const int64_t lda = m > 1 ? a.stride(0) : k;
  const int64_t ldb = n > 1 ? b.stride(1) : k;
  const int64_t ldo = m > 1 ? out.stride(0) : out_n;
  const c10::cuda::CUDAGuard guard(a.device());
  int status;
  if (tile_n != 0) {
    status = tm_scaled_mm_i8_tile(out.data_ptr(), out_dt, a.data_ptr<int8_t>(),
                                  b.data_ptr<int8_t>(), a_scales.data_ptr<float>(),
                                  a_scales.numel(), b_scales.data_ptr<float>(), b_scales.numel(),
                                  bias_ptr, m, n, k, lda, ldb, ldo,
                                  static_cast<uint32_t>(epilogue), acc_ptr,
                                  static_cast<int>(tile_n), stream_of(a));
  } else {
    uint64_t ws_bytes = 0;
    status = m > 0 ? tm_scaled_mm_i8_workspace_size(m, n, k, &ws_bytes) : TM_OK;
    if (status == TM_OK && ws_bytes > 0) {
      at::Tensor ws = splitk_workspace(a, ws_bytes);
      status = tm_scaled_mm_i8_ws(out.data_ptr(), out_dt, a.data_ptr<int8_t>(),
                                  b.data_ptr<int8_t>(), a_scales.data_ptr<float>(),
                                  a_scales.numel(), b_scales.data_ptr<float>(), b_scales.numel(),
                                  bias_ptr, m, n, k, lda, ldb, ldo,
                                  static_cast<uint32_t>(epilogue), acc_ptr, ws.data_ptr(),
                                  static_cast<uint64_t>(ws.numel()), stream_of(a));
    } else if (status == TM_OK) {
      status = tm_scaled_mm_i8_ex(out.data_ptr(), out_dt, a.data_ptr<int8_t>(),
                                  b.data_ptr<int8_t>(), a_scales.data_ptr<float>(),
                                  a_scales.numel(), b_scales.data_ptr<float>(), b_scales.numel(),
                                  bias_ptr, m, n, k, lda, ldb, ldo,
                                  static_cast<uint32_t>(epilogue), acc_ptr, stream_of(a));
    }
  }
  check_status(status, op);
}

void cutlass_scaled_mm(at::Tensor& out, const at::Tensor& a, const at::Tensor& b,
                       const at::Tensor& a_scales, const at::Tensor& b_scales,
                       const std::optional<at::Tensor>& bias) {
  scaled_mm_common(out, a, b, a_scales, b_scales, bias, 0, std::nullopt, 0, "cutlass_scaled_mm");
}

void scaled_mm_i8_ex(at::Tensor& out, const at::Tensor& a, const at::Tensor& b,
                     const at::Tensor& a_scales, const at::Tensor& b_scales,
                     const std::optional<at::Tensor>& bias, int64_t epilogue,
                     const std::optional<at::Tensor>& acc_debug, int64_t tile_n) {
  scaled_mm_common(out, a, b, a_scales, b_scales, bias, epilogue, acc_debug, tile_n,
                   "scaled_mm_i8_ex");
}

// W8A8 GEMM with the BF16 LoRA delta added in the epilogue:
// out = epi(dequant(a b) (+bias) + lora_t lora_b^T); lora_t = x A^T [m, r],
// lora_b = scale * B [n, r], both bf16 with unit inner stride, r <= 64.
void scaled_mm_i8_lora(at::Tensor& out, const at::Tensor& a, const at::Tensor& b,
                       const at::Tensor& a_scales, const at::Tensor& b_scales,
                       const std::optional<at::Tensor>& bias, const at::Tensor& lora_t,
                       const at::Tensor& lora_b, int64_t epilogue) {
  check_cuda(a, a, "a");
  check_cuda(b, a, "b");
  check_cuda(out, a, "out");
  check_cuda(a_scales, a, "a_scales");
  check_cuda(b_scales, a, "b_scales");
  check_cuda(lora_t, a, "lora_t");
  check_cuda(lora_b, a, "lora_b");
  TORCH_CHECK(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar,
              "a and b must be int8");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && out.dim() == 2, "a, b and out must be 2-D");
  const int64_t m = a.size(0), k = a.size(1), n = b.size(1);
  TORCH_CHECK(b.size(0) == k, "a and b inner dimensions differ: ", k, " vs ", b.size(0));
  TORCH_CHECK(out.size(0) == m && out.size(1) == n, "out must be [", m, ", ", n, "]");
  TORCH_CHECK(a.stride(1) == 1, "a must be row-major");
  TORCH_CHECK(b.stride(0) == 1, "b must be column-major (pass weight.t())");
  TORCH_CHECK(out.stride(1) == 1, "out must be row-major");
  const int out_dt = dtype_code(out);
  TORCH_CHECK(out_dt == TM_DTYPE_BF16 || out_dt == TM_DTYPE_FP16, "out must be bfloat16 or float16");
  TORCH_CHECK(a_scales.scalar_type() == at::kFloat && b_scales.scalar_type() == at::kFloat,
              "scales must be float32");
  TORCH_CHECK(a_scales.is_contiguous() && b_scales.is_contiguous(), "scales must be contiguous");
  TORCH_CHECK(a_scales.numel() == 1 || a_scales.numel() == m, "a_scales must be per-tensor or per-token");
  TORCH_CHECK(b_scales.numel() == 1 || b_scales.numel() == n, "b_scales must be per-tensor or per-channel");
  TORCH_CHECK(lora_t.scalar_type() == at::kBFloat16 && lora_b.scalar_type() == at::kBFloat16,
              "lora_t and lora_b must be bfloat16");
  TORCH_CHECK(lora_t.dim() == 2 && lora_b.dim() == 2 && lora_t.stride(1) == 1 &&
                  lora_b.stride(1) == 1,
              "lora_t and lora_b must be 2-D row-major");
  const int64_t r = lora_t.size(1);
  TORCH_CHECK(lora_t.size(0) == m && lora_b.size(0) == n && lora_b.size(1) == r,
              "lora_t must be [m, r] and lora_b [n, r]");
  const void* bias_ptr = nullptr;
  if (bias.has_value()) {
    check_cuda(*bias, a, "bias");
    TORCH_CHECK(bias->scalar_type() == out.scalar_type(), "bias must have the output dtype");
    TORCH_CHECK(bias->numel() == n && bias->is_contiguous(), "bias must be contiguous [n]");
    bias_ptr = bias->data_ptr();
  }
  const int64_t lda = m > 1 ? a.stride(0) : k;
  const int64_t ldb = n > 1 ? b.stride(1) : k;
  const int64_t ldo = m > 1 ? out.stride(0) : n;
  const int64_t ldt = m > 1 ? lora_t.stride(0) : r;
  const int64_t ldlb = n > 1 ? lora_b.stride(0) : r;
  const c10::cuda::CUDAGuard guard(a.device());
  check_status(tm_scaled_mm_i8_lora(out.data_ptr(), out_dt, a.data_ptr<int8_t>(),
                                    b.data_ptr<int8_t>(), a_scales.data_ptr<float>(),
                                    a_scales.numel(), b_scales.data_ptr<float>(),
                                    b_scales.numel(), bias_ptr, lora_t.data_ptr(), ldt,
                                    lora_b.data_ptr(), ldlb, static_cast<int>(r), m, n, k, lda,
                                    ldb, ldo, static_cast<uint32_t>(epilogue), stream_of(a)),
               "scaled_mm_i8_lora");
}

// LoRA down-projection t = x a^T (tm_lora_down_proj): x bf16 [m, k],
// a bf16 [r, k], t bf16 [m, r]; rows contiguous, any row strides.
void lora_down_proj(at::Tensor& t, const at::Tensor& x, const at::Tensor& a) {
  check_cuda(x, x, "x");
  check_cuda(a, x, "a");
  check_cuda(t, x, "t");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 && a.scalar_type() == at::kBFloat16 &&
                  t.scalar_type() == at::kBFloat16,
              "x, a and t must be bfloat16");
  TORCH_CHECK(x.dim() == 2 && a.dim() == 2 && t.dim() == 2, "x, a and t must be 2-D");
  const int64_t m = x.size(0), k = x.size(1), r = a.size(0);
  TORCH_CHECK(a.size(1) == k, "x and a inner dimensions differ: ", k, " vs ", a.size(1));
  TORCH_CHECK(t.size(0) == m && t.size(1) == r, "t must be [", m, ", ", r, "]");
  TORCH_CHECK(x.stride(1) == 1 && a.stride(1) == 1 && t.stride(1) == 1,
              "x, a and t must be row-major");
  const int64_t ldx = m > 1 ? x.stride(0) : k;
  const int64_t lda = r > 1 ? a.stride(0) : k;
  const int64_t ldt = m > 1 ? t.stride(0) : r;
  const c10::cuda::CUDAGuard guard(x.device());
  check_status(tm_lora_down_proj(t.data_ptr(), ldt, x.data_ptr(), ldx, a.data_ptr(), lda,
                                 static_cast<int>(r), m, k, stream_of(x)),
               "lora_down_proj");
}

// Merged QKV projection into the Ulysses all-to-all send buffer
// send [world, 3, m, ceil(heads / world) * head_dim] (tm_scaled_mm_i8_ulysses_send;
// padded head slots are zeroed).
void scaled_mm_i8_ulysses_send(at::Tensor& send, const at::Tensor& a, const at::Tensor& b,
                               const at::Tensor& a_scales, const at::Tensor& b_scales,
                               const std::optional<at::Tensor>& bias, int64_t num_heads,
                               int64_t head_dim, int64_t world) {
  check_cuda(a, a, "a");
  check_cuda(b, a, "b");
  check_cuda(send, a, "send");
  check_cuda(a_scales, a, "a_scales");
  check_cuda(b_scales, a, "b_scales");
  TORCH_CHECK(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar,
              "a and b must be int8");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2, "a and b must be 2-D");
  const int64_t m = a.size(0), k = a.size(1), n = b.size(1);
  TORCH_CHECK(b.size(0) == k, "a and b inner dimensions differ");
  TORCH_CHECK(world > 0 && num_heads > 0, "heads and the Ulysses degree must be positive");
  TORCH_CHECK(n == 3 * num_heads * head_dim, "b must have 3 x heads x head_dim columns");
  const int64_t local = (num_heads + world - 1) / world;
  TORCH_CHECK(send.is_contiguous() && send.numel() == world * 3 * m * local * head_dim,
              "send must be a contiguous [world, 3, m, ceil(heads / world) * head_dim] buffer");
  TORCH_CHECK(a.stride(1) == 1 && b.stride(0) == 1, "a row-major, b column-major (weight.t())");
  const int out_dt = dtype_code(send);
  TORCH_CHECK(out_dt == TM_DTYPE_BF16 || out_dt == TM_DTYPE_FP16, "send must be bf16 or fp16");
  TORCH_CHECK(a_scales.scalar_type() == at::kFloat && b_scales.scalar_type() == at::kFloat &&
                  a_scales.is_contiguous() && b_scales.is_contiguous(),
              "scales must be contiguous float32");
  const void* bias_ptr = nullptr;
  if (bias.has_value()) {
    check_cuda(*bias, a, "bias");
    TORCH_CHECK(bias->scalar_type() == send.scalar_type() && bias->numel() == n &&
                    bias->is_contiguous(),
                "bias must be contiguous [n] in the output dtype");
    bias_ptr = bias->data_ptr();
  }
  const int64_t lda = m > 1 ? a.stride(0) : k;
  const int64_t ldb = n > 1 ? b.stride(1) : k;
  const c10::cuda::CUDAGuard guard(a.device());
  check_status(tm_scaled_mm_i8_ulysses_send(send.data_ptr(), out_dt, a.data_ptr<int8_t>(),
                                            b.data_ptr<int8_t>(), a_scales.data_ptr<float>(),
                                            a_scales.numel(), b_scales.data_ptr<float>(),
                                            b_scales.numel(), bias_ptr, m, n, k, lda, ldb,
                                            static_cast<int>(num_heads),
                                            static_cast<int>(head_dim), static_cast<int>(world),
                                            stream_of(a)),
               "scaled_mm_i8_ulysses_send");
}

void quantize_weight_int8(at::Tensor& q, at::Tensor& scales, const at::Tensor& w) {
  check_cuda(w, w, "weight");
  check_cuda(q, w, "q");
  check_cuda(scales, w, "scales");
  const int dt = dtype_code(w);
  TORCH_CHECK(dt >= 0, "weight dtype must be bfloat16, float16 or float32");
  TORCH_CHECK(w.dim() == 2 && w.is_contiguous(), "weight must be a contiguous 2-D tensor");
  TORCH_CHECK(q.scalar_type() == at::kChar && q.is_contiguous() && q.sizes() == w.sizes(),
              "q must be contiguous int8 with the weight's shape");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.is_contiguous() &&
                  scales.numel() == w.size(0),
              "scales must be contiguous float32 [n]");
  const c10::cuda::CUDAGuard guard(w.device());
  check_status(tm_quantize_weight_int8(q.data_ptr<int8_t>(), scales.data_ptr<float>(), w.data_ptr(),
                                       dt, w.size(0), w.size(1), stream_of(w)),
               "quantize_weight_int8");
}

struct ModulateArgs {
  int64_t rows, cols, table_stride;
  const int64_t* index;
  void* hidden;
};

ModulateArgs check_modulate_inputs(const std::optional<at::Tensor>& hidden_out,
                                   const at::Tensor& x, const at::Tensor& shift,
                                   const at::Tensor& scale,
                                   const std::optional<at::Tensor>& index) {
  check_cuda(x, x, "x");
  check_cuda(shift, x, "shift");
  check_cuda(scale, x, "scale");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 && x.is_contiguous(), "x must be contiguous bfloat16");
  ModulateArgs r{};
  r.cols = x.size(-1);
  r.rows = r.cols == 0 ? 0 : x.numel() / r.cols;
  TORCH_CHECK(shift.scalar_type() == at::kBFloat16 && scale.scalar_type() == at::kBFloat16,
              "shift/scale must be bfloat16");
  TORCH_CHECK(shift.dim() == 2 && scale.dim() == 2 && shift.sizes() == scale.sizes(),
              "shift/scale must be 2-D tables of equal shape");
  TORCH_CHECK(shift.stride(1) == 1 && scale.stride(1) == 1 && shift.stride(0) == scale.stride(0),
              "shift/scale must be row-major with equal row strides");
  TORCH_CHECK(shift.size(1) == r.cols, "shift/scale width must equal x's last dimension");
  r.table_stride = shift.stride(0);
  if (index.has_value()) {
    check_cuda(*index, x, "index");
    TORCH_CHECK(index->scalar_type() == at::kLong && index->is_contiguous() &&
                    index->numel() == r.rows,
                "index must be contiguous int64 [rows]");
    r.index = index->data_ptr<int64_t>();
  } else {
    TORCH_CHECK(shift.size(0) == r.rows, "without index, shift/scale need one row per token");
  }
  if (hidden_out.has_value()) {
    check_cuda(*hidden_out, x, "hidden_out");
    TORCH_CHECK(hidden_out->scalar_type() == at::kBFloat16 && hidden_out->is_contiguous() &&
                    hidden_out->numel() == x.numel(),
                "hidden_out must be contiguous bfloat16 with x's shape");
    r.hidden = hidden_out->data_ptr();
  }
  return r;
}

// The int8 producers: their outputs, then the common inputs.
ModulateArgs check_modulate(at::Tensor& out, at::Tensor& scales,
                            const std::optional<at::Tensor>& hidden_out, const at::Tensor& x,
                            const at::Tensor& shift, const at::Tensor& scale,
                            const std::optional<at::Tensor>& index) {
  check_cuda(x, x, "x");
  check_cuda(out, x, "out");
  check_cuda(scales, x, "scales");
  const ModulateArgs r = check_modulate_inputs(hidden_out, x, shift, scale, index);
  TORCH_CHECK(out.scalar_type() == at::kChar && out.is_contiguous() && out.numel() == x.numel(),
              "out must be contiguous int8 with x's shape");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.is_contiguous() &&
                  scales.numel() == r.rows,
              "scales must be contiguous float32 [rows]");
  return r;
}

void check_norm_weight(const at::Tensor& weight, const at::Tensor& x, int64_t cols) {
  check_cuda(weight, x, "weight");
  TORCH_CHECK(weight.scalar_type() == at::kBFloat16 && weight.is_contiguous() &&
                  weight.numel() == cols,
              "norm weight must be contiguous bfloat16 [cols]");
}

void check_residual_gate(const at::Tensor& residual_out, const at::Tensor& residual,
                         const at::Tensor& branch, const at::Tensor& gate,
                         const at::Tensor& shift) {
  check_cuda(branch, residual, "branch");
  check_cuda(gate, residual, "gate");
  check_cuda(residual_out, residual, "residual_out");
  TORCH_CHECK(branch.scalar_type() == at::kBFloat16 && branch.is_contiguous() &&
                  branch.sizes() == residual.sizes(),
              "branch must be contiguous bfloat16 with the residual's shape");
  TORCH_CHECK(residual_out.scalar_type() == at::kBFloat16 && residual_out.is_contiguous() &&
                  residual_out.numel() == residual.numel(),
              "residual_out must be contiguous bfloat16 with the residual's shape");
  TORCH_CHECK(gate.scalar_type() == at::kBFloat16 && gate.sizes() == shift.sizes() &&
                  gate.stride(1) == 1 && gate.stride(0) == shift.stride(0),
              "gate must be a bfloat16 table shaped and strided like shift/scale");
}

void modulate_int8_quant(at::Tensor& out, at::Tensor& scales,
                         const std::optional<at::Tensor>& hidden_out, const at::Tensor& x,
                         const at::Tensor& shift, const at::Tensor& scale,
                         const std::optional<at::Tensor>& index) {
  const ModulateArgs r = check_modulate(out, scales, hidden_out, x, shift, scale, index);
  const c10::cuda::CUDAGuard guard(x.device());
  check_status(tm_modulate_int8_quant(out.data_ptr<int8_t>(), scales.data_ptr<float>(), r.hidden,
                                      x.data_ptr(), shift.data_ptr(), scale.data_ptr(), r.index,
                                      r.table_stride, r.rows, r.cols, stream_of(x)),
               "modulate_int8_quant");
}

void rms_norm_modulate_int8_quant(at::Tensor& out, at::Tensor& scales,
                                  const std::optional<at::Tensor>& hidden_out,
                                  const at::Tensor& x, const at::Tensor& weight, double eps,
                                  const at::Tensor& shift, const at::Tensor& scale,
                                  const std::optional<at::Tensor>& index) {
  const ModulateArgs r = check_modulate(out, scales, hidden_out, x, shift, scale, index);
  check_norm_weight(weight, x, r.cols);
  const c10::cuda::CUDAGuard guard(x.device());
  check_status(tm_rms_norm_modulate_int8_quant(out.data_ptr<int8_t>(), scales.data_ptr<float>(),
                                               r.hidden, x.data_ptr(), weight.data_ptr(),
                                               static_cast<float>(eps), shift.data_ptr(),
                                               scale.data_ptr(), r.index, r.table_stride, r.rows,
                                               r.cols, stream_of(x)),
               "rms_norm_modulate_int8_quant");
}

void residual_gate_rms_norm_modulate_int8_quant(
    at::Tensor& out, at::Tensor& scales, at::Tensor& residual_out,
    const std::optional<at::Tensor>& hidden_out, const at::Tensor& residual,
    const at::Tensor& branch, const at::Tensor& gate, const at::Tensor& weight, double eps,
    const at::Tensor& shift, const at::Tensor& scale, const std::optional<at::Tensor>& index) {
  const ModulateArgs r = check_modulate(out, scales, hidden_out, residual, shift, scale, index);
  check_norm_weight(weight, residual, r.cols);
  check_residual_gate(residual_out, residual, branch, gate, shift);
  const c10::cuda::CUDAGuard guard(residual.device());
  check_status(tm_residual_gate_rms_norm_modulate_int8_quant(
                   out.data_ptr<int8_t>(), scales.data_ptr<float>(), residual_out.data_ptr(),
                   r.hidden, residual.data_ptr(), branch.data_ptr(), gate.data_ptr(),
                   weight.data_ptr(), static_cast<float>(eps), shift.data_ptr(),
                   scale.data_ptr(), r.index, r.table_stride, r.rows, r.cols,
                   stream_of(residual)),
               "residual_gate_rms_norm_modulate_int8_quant");
}

// ---- 4-bit block formats ----
// The format is the dtype of the block scales: float8_e4m3fn (TM_FP4_NV) or
// float8_e8m0fnu (TM_FP4_MX).
int fp4_format(const at::Tensor& block_scales, const char* name) {
  const auto t = block_scales.scalar_type();
  TORCH_CHECK(t == at::kFloat8_e4m3fn || t == at::kFloat8_e8m0fnu, name,
              " must be float8_e4m3fn (blocks of 16) or float8_e8m0fnu (blocks of 32)");
  return t == at::kFloat8_e4m3fn ? TM_FP4_NV : TM_FP4_MX;
}

// Block scales of a [rows, cols] tensor: the whole padded tile buffer.
uint8_t* fp4_blocks(const at::Tensor& t, const at::Tensor& ref, int64_t rows, int64_t cols,
                    int format, const char* name) {
  check_cuda(t, ref, name);
  TORCH_CHECK(fp4_format(t, name) == format, name, " must be in the other operand's format");
  uint64_t bytes = 0;
  TORCH_CHECK(tm_fp4_block_scales_size(rows, cols, format, &bytes) == TM_OK,
              "4-bit rows must be a positive multiple of 32 elements wide, got ", cols);
  TORCH_CHECK(t.is_contiguous() && static_cast<uint64_t>(t.numel()) == bytes, name,
              " must be contiguous with ", bytes, " elements for [", rows, ", ", cols, "]");
  return static_cast<uint8_t*>(t.data_ptr());
}

uint8_t* fp4_codes(const at::Tensor& q, const at::Tensor& ref, int64_t rows, int64_t cols,
                   const char* name) {
  check_cuda(q, ref, name);
  TORCH_CHECK(q.scalar_type() == at::kByte && q.is_contiguous() && q.numel() == rows * (cols / 2),
              name, " must be contiguous uint8 with two codes a byte");
  return q.data_ptr<uint8_t>();
}

// Outer scales written by a quantising call: one a row (TM_FP4_NV), none (TM_FP4_MX).
float* fp4_row_scales(const std::optional<at::Tensor>& scales, const at::Tensor& ref, int64_t rows,
                      int format) {
  if (!scales.has_value()) return nullptr;
  check_cuda(*scales, ref, "scales");
  TORCH_CHECK(format == TM_FP4_NV, "blocks of 32 take no fp32 scales");
  TORCH_CHECK(scales->scalar_type() == at::kFloat && scales->is_contiguous() &&
                  scales->numel() == rows,
              "scales must be contiguous float32, one per row");
  return scales->data_ptr<float>();
}

void scaled_fp4_quant(at::Tensor& q, at::Tensor& block_scales,
                      const std::optional<at::Tensor>& scales, const at::Tensor& input,
                      const std::optional<at::Tensor>& given_scale) {
  check_cuda(input, input, "input");
  const int dt = dtype_code(input);
  TORCH_CHECK(dt >= 0, "input dtype must be bfloat16, float16 or float32");
  int64_t rows, cols, ld;
  as_rows(input, &rows, &cols, &ld);
  const int format = fp4_format(block_scales, "block_scales");
  uint8_t* blocks = fp4_blocks(block_scales, input, rows, cols, format, "block_scales");
  uint8_t* codes = fp4_codes(q, input, rows, cols, "q");
  float* row_scales = fp4_row_scales(scales, input, rows, format);
  const float* given = nullptr;
  if (given_scale.has_value()) {
    check_cuda(*given_scale, input, "scale");
    TORCH_CHECK(format == TM_FP4_NV, "blocks of 32 take no fp32 scale");
    TORCH_CHECK(given_scale->scalar_type() == at::kFloat && given_scale->numel() == 1,
                "a given scale must be one float32 value");
    given = given_scale->data_ptr<float>();
  }
  TORCH_CHECK(format == TM_FP4_MX || scales.has_value() != given_scale.has_value(),
              "blocks of 16 need either scales to write or a given scale");
  const c10::cuda::CUDAGuard guard(input.device());
  check_status(tm_scaled_fp4_quant(codes, blocks, row_scales, given, input.data_ptr(), dt, format,
                                   rows, cols, ld, stream_of(input)),
               "scaled_fp4_quant");
}

void dequantize_fp4(at::Tensor& out, const at::Tensor& q, const at::Tensor& block_scales,
                    const std::optional<at::Tensor>& scales) {
  check_cuda(q, q, "q");
  check_cuda(out, q, "out");
  const int dt = dtype_code(out);
  TORCH_CHECK(dt >= 0, "out dtype must be bfloat16, float16 or float32");
  TORCH_CHECK(out.dim() >= 1 && out.is_contiguous(), "out must be contiguous");
  const int64_t cols = out.size(-1);
  const int64_t rows = cols == 0 ? 0 : out.numel() / cols;
  const int format = fp4_format(block_scales, "block_scales");
  const uint8_t* blocks = fp4_blocks(block_scales, q, rows, cols, format, "block_scales");
  const uint8_t* codes = fp4_codes(q, q, rows, cols, "q");
  const float* s = nullptr;
  if (scales.has_value()) {
    check_cuda(*scales, q, "scales");
    TORCH_CHECK(format == TM_FP4_NV, "blocks of 32 take no fp32 scales");
    TORCH_CHECK(scales->scalar_type() == at::kFloat && scales->is_contiguous() &&
                    (scales->numel() == 1 || scales->numel() == rows),
                "scales must be contiguous float32, one or one per row");
    s = scales->data_ptr<float>();
  }
  TORCH_CHECK(format == TM_FP4_MX || s != nullptr, "blocks of 16 need their fp32 scales");
  const c10::cuda::CUDAGuard guard(q.device());
  check_status(tm_dequantize_fp4(out.data_ptr(), dt, codes, blocks, s,
                                 scales.has_value() ? scales->numel() : 0, format, rows, cols,
                                 stream_of(q)),
               "dequantize_fp4");
}

struct Fp4Out {
  uint8_t* codes;
  uint8_t* blocks;
  float* scales;
  int format;
};

Fp4Out check_fp4_out(const at::Tensor& q, const at::Tensor& block_scales,
                     const std::optional<at::Tensor>& scales, const at::Tensor& x,
                     const ModulateArgs& r) {
  Fp4Out o;
  o.format = fp4_format(block_scales, "block_scales");
  o.blocks = fp4_blocks(block_scales, x, r.rows, r.cols, o.format, "block_scales");
  o.codes = fp4_codes(q, x, r.rows, r.cols, "q");
  o.scales = fp4_row_scales(scales, x, r.rows, o.format);
  TORCH_CHECK(o.format == TM_FP4_MX || o.scales != nullptr, "blocks of 16 need scales to write");
  return o;
}

void modulate_fp4_quant(at::Tensor& q, at::Tensor& block_scales,
                        const std::optional<at::Tensor>& scales,
                        const std::optional<at::Tensor>& hidden_out, const at::Tensor& x,
                        const at::Tensor& shift, const at::Tensor& scale,
                        const std::optional<at::Tensor>& index) {
  const ModulateArgs r = check_modulate_inputs(hidden_out, x, shift, scale, index);
  const Fp4Out o = check_fp4_out(q, block_scales, scales, x, r);
  const c10::cuda::CUDAGuard guard(x.device());
  check_status(tm_modulate_fp4_quant(o.codes, o.blocks, o.scales, r.hidden, x.data_ptr(),
                                     shift.data_ptr(), scale.data_ptr(), r.index, r.table_stride,
                                     o.format, r.rows, r.cols, stream_of(x)),
               "modulate_fp4_quant");
}

void rms_norm_modulate_fp4_quant(at::Tensor& q, at::Tensor& block_scales,
                                 const std::optional<at::Tensor>& scales,
                                 const std::optional<at::Tensor>& hidden_out, const at::Tensor& x,
                                 const at::Tensor& weight, double eps, const at::Tensor& shift,
                                 const at::Tensor& scale, const std::optional<at::Tensor>& index) {
  const ModulateArgs r = check_modulate_inputs(hidden_out, x, shift, scale, index);
  const Fp4Out o = check_fp4_out(q, block_scales, scales, x, r);
  check_norm_weight(weight, x, r.cols);
  const c10::cuda::CUDAGuard guard(x.device());
  check_status(tm_rms_norm_modulate_fp4_quant(o.codes, o.blocks, o.scales, r.hidden, x.data_ptr(),
                                              weight.data_ptr(), static_cast<float>(eps),
                                              shift.data_ptr(), scale.data_ptr(), r.index,
                                              r.table_stride, o.format, r.rows, r.cols,
                                              stream_of(x)),
               "rms_norm_modulate_fp4_quant");
}

void residual_gate_rms_norm_modulate_fp4_quant(
    at::Tensor& q, at::Tensor& block_scales, const std::optional<at::Tensor>& scales,
    at::Tensor& residual_out, const std::optional<at::Tensor>& hidden_out,
    const at::Tensor& residual, const at::Tensor& branch, const at::Tensor& gate,
    const at::Tensor& weight, double eps, const at::Tensor& shift, const at::Tensor& scale,
    const std::optional<at::Tensor>& index) {
  const ModulateArgs r = check_modulate_inputs(hidden_out, residual, shift, scale, index);
  const Fp4Out o = check_fp4_out(q, block_scales, scales, residual, r);
  check_norm_weight(weight, residual, r.cols);
  check_residual_gate(residual_out, residual, branch, gate, shift);
  const c10::cuda::CUDAGuard guard(residual.device());
  check_status(tm_residual_gate_rms_norm_modulate_fp4_quant(
                   o.codes, o.blocks, o.scales, residual_out.data_ptr(), r.hidden,
                   residual.data_ptr(), branch.data_ptr(), gate.data_ptr(), weight.data_ptr(),
                   static_cast<float>(eps), shift.data_ptr(), scale.data_ptr(), r.index,
                   r.table_stride, o.format, r.rows, r.cols, stream_of(residual)),
               "residual_gate_rms_norm_modulate_fp4_quant");
}

const float* fp4_outer(const std::optional<at::Tensor>& t, const at::Tensor& ref, int64_t n,
                       int format, const char* name) {
  TORCH_CHECK(t.has_value() == (format == TM_FP4_NV), name,
              format == TM_FP4_NV ? " is needed with blocks of 16" : " must be None with blocks of 32");
  if (!t.has_value()) return nullptr;
  check_cuda(*t, ref, name);
  TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() &&
                  (t->numel() == 1 || t->numel() == n),
              name, " must be contiguous float32 with 1 or ", n, " values");
  return t->data_ptr<float>();
}

void scaled_mm_fp4(at::Tensor& out, const at::Tensor& a, const at::Tensor& b,
                   const at::Tensor& block_scales_a, const at::Tensor& block_scales_b,
                   const std::optional<at::Tensor>& scales_a,
                   const std::optional<at::Tensor>& scales_b,
                   const std::optional<at::Tensor>& bias, int64_t epilogue, int64_t tile,
                   int64_t splits) {
  check_cuda(a, a, "a");
  check_cuda(b, a, "b");
  check_cuda(out, a, "out");
  TORCH_CHECK(a.scalar_type() == at::kByte && b.scalar_type() == at::kByte,
              "a and b must be uint8 (two codes a byte)");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && out.dim() == 2, "a, b and out must be 2-D");
  const int64_t m = a.size(0), k = 2 * a.size(1), n = b.size(1);
  TORCH_CHECK(2 * b.size(0) == k, "a and b inner dimensions differ: ", a.size(1), " vs ", b.size(0),
              " bytes");
  const int64_t out_n = (epilogue & TM_EPI_SWIGLU) ? n / 2 : n;
  TORCH_CHECK(out.size(0) == m && out.size(1) == out_n, "out must be [", m, ", ", out_n, "]");
  TORCH_CHECK(a.stride(1) == 1, "a must be row-major");
  TORCH_CHECK(b.stride(0) == 1, "b must be column-major (pass weight.t())");
  TORCH_CHECK(out.stride(1) == 1, "out must be row-major");
  const int out_dt = dtype_code(out);
  TORCH_CHECK(out_dt == TM_DTYPE_BF16 || out_dt == TM_DTYPE_FP16, "out must be bfloat16 or float16");
  const int format = fp4_format(block_scales_a, "block_scales_a");
  const uint8_t* blocks_a = fp4_blocks(block_scales_a, a, m, k, format, "block_scales_a");
  const uint8_t* blocks_b = fp4_blocks(block_scales_b, a, n, k, format, "block_scales_b");
  const float* sa = fp4_outer(scales_a, a, m, format, "scales_a");
  const float* sb = fp4_outer(scales_b, a, n, format, "scales_b");
  const void* bias_ptr = nullptr;
  if (bias.has_value()) {
    check_cuda(*bias, a, "bias");
    TORCH_CHECK(bias->scalar_type() == out.scalar_type(), "bias must have the output dtype");
    TORCH_CHECK(bias->numel() == n && bias->is_contiguous(), "bias must be contiguous [n]");
    bias_ptr = bias->data_ptr();
  }
  const int64_t lda = m > 1 ? a.stride(0) : k / 2;
  const int64_t ldb = n > 1 ? b.stride(1) : k / 2;
  const int64_t ldo = m > 1 ? out.stride(0) : (out_n + 7) / 8 * 8;
  const c10::cuda::CUDAGuard guard(a.device());
  const int64_t na = scales_a.has_value() ? scales_a->numel() : 0;
  const int64_t nb = scales_b.has_value() ? scales_b->numel() : 0;
  const int status =
      tile == 0 ? tm_scaled_mm_fp4(out.data_ptr(), out_dt, a.data_ptr<uint8_t>(),
                                   b.data_ptr<uint8_t>(), blocks_a, blocks_b, sa, na, sb, nb,
                                   bias_ptr, format, m, n, k, lda, ldb, ldo,
                                   static_cast<uint32_t>(epilogue), stream_of(a))
                : tm_scaled_mm_fp4_tile(out.data_ptr(), out_dt, a.data_ptr<uint8_t>(),
                                        b.data_ptr<uint8_t>(), blocks_a, blocks_b, sa, na, sb, nb,
                                        bias_ptr, format, m, n, k, lda, ldb, ldo,
                                        static_cast<uint32_t>(epilogue), static_cast<int>(tile),
                                        static_cast<int>(splits), stream_of(a));
  check_status(status, "scaled_mm_fp4");
}

// ---- the allocating forms, one dispatcher call each (the Python API) ----
// Contiguous and uninitialised, from the caching allocator without another
// pass through the dispatcher.
at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}

struct Fp4Tensors {
  at::Tensor q, blocks;
  std::optional<at::Tensor> scales;
};

Fp4Tensors empty_fp4(const at::Tensor& like, bool mx, bool row_scales) {
  TORCH_CHECK(like.dim() >= 1, "input must have at least one dimension");
  const int64_t cols = like.size(-1);
  TORCH_CHECK(cols > 0 && cols % 32 == 0,
              "4-bit rows must be a positive multiple of 32 elements wide, got ", cols);
  const int64_t rows = like.numel() / cols;
  Fp4Tensors t;
  at::DimVector sizes(like.sizes());
  sizes.back() = cols / 2;
  t.q = empty_on(like, sizes, at::kByte);
  const int64_t blocks = cols / (mx ? 32 : 16);
  t.blocks = empty_on(like, {(rows + 127) / 128 * 128, (blocks + 3) / 4 * 4},
                      mx ? at::kFloat8_e8m0fnu : at::kFloat8_e4m3fn);
  if (row_scales && !mx) t.scales = empty_on(like, {rows, 1}, at::kFloat);
  return t;
}

using Fp4Result = std::tuple<at::Tensor, at::Tensor, std::optional<at::Tensor>>;

Fp4Result scaled_fp4_quant_new(const at::Tensor& input, const std::optional<at::Tensor>& scale,
                               bool mx) {
  TORCH_CHECK(!mx || !scale.has_value(), "blocks of 32 take no fp32 scale");
  const c10::cuda::CUDAGuard guard(input.device());
  Fp4Tensors t = empty_fp4(input, mx, !scale.has_value());
  // rows may be any distance apart, but not overlap (an expanded or windowed view)
  const bool rows = input.dim() == 2 && input.stride(1) == 1 &&
                    (input.size(0) <= 1 || input.stride(0) >= input.size(1));
  scaled_fp4_quant(t.q, t.blocks, t.scales, rows ? input : input.contiguous(), scale);
  return {t.q, t.blocks, t.scales};  // none where a scale is given: the schema's outputs are fresh
}

at::Tensor dequantize_fp4_new(const at::Tensor& q, const at::Tensor& block_scales,
                              const std::optional<at::Tensor>& scales, at::ScalarType dtype) {
  TORCH_CHECK(q.dim() >= 1, "q must have at least one dimension");
  const c10::cuda::CUDAGuard guard(q.device());
  at::DimVector sizes(q.sizes());
  sizes.back() *= 2;
  at::Tensor out = empty_on(q, sizes, dtype);
  dequantize_fp4(out, q.contiguous(), block_scales, scales);
  return out;
}

at::Tensor scaled_mm_fp4_new(const at::Tensor& a, const at::Tensor& b,
                             const at::Tensor& block_scales_a, const at::Tensor& block_scales_b,
                             const std::optional<at::Tensor>& scales_a,
                             const std::optional<at::Tensor>& scales_b, at::ScalarType dtype,
                             const std::optional<at::Tensor>& bias, int64_t epilogue) {
  TORCH_CHECK(a.dim() >= 1 && a.size(-1) > 0, "a must be [..., K / 2] with K > 0");
  TORCH_CHECK(b.dim() == 2, "b must be 2-D");
  const c10::cuda::CUDAGuard guard(a.device());
  const at::Tensor a2 = a.dim() == 2 ? a : a.reshape({a.numel() / a.size(-1), a.size(-1)});
  const int64_t cols = (epilogue & TM_EPI_SWIGLU) ? b.size(1) / 2 : b.size(1);
  at::Tensor out = empty_on(a, {a2.size(0), cols}, dtype);
  scaled_mm_fp4(out, a2, b, block_scales_a, block_scales_b, scales_a, scales_b, bias, epilogue, 0,
                1);
  if (a.dim() == 2) return out;
  at::DimVector sizes(a.sizes());
  sizes.back() = cols;
  return out.view(sizes);
}

using Fp4Hidden =
    std::tuple<at::Tensor, at::Tensor, std::optional<at::Tensor>, std::optional<at::Tensor>>;

std::optional<at::Tensor> empty_hidden(const at::Tensor& x, bool wanted) {
  return wanted ? std::optional<at::Tensor>(at::empty_like(x)) : std::nullopt;
}

Fp4Hidden modulate_fp4_quant_new(const at::Tensor& x, const at::Tensor& shift,
                                 const at::Tensor& scale, const std::optional<at::Tensor>& index,
                                 bool mx, bool hidden) {
  const c10::cuda::CUDAGuard guard(x.device());
  Fp4Tensors t = empty_fp4(x, mx, true);
  const std::optional<at::Tensor> h = empty_hidden(x, hidden);
  modulate_fp4_quant(t.q, t.blocks, t.scales, h, x, shift, scale, index);
  return {t.q, t.blocks, t.scales, h};
}

Fp4Hidden rms_norm_modulate_fp4_quant_new(const at::Tensor& x, const at::Tensor& weight, double eps,
                                          const at::Tensor& shift, const at::Tensor& scale,
                                          const std::optional<at::Tensor>& index, bool mx,
                                          bool hidden) {
  const c10::cuda::CUDAGuard guard(x.device());
  Fp4Tensors t = empty_fp4(x, mx, true);
  const std::optional<at::Tensor> h = empty_hidden(x, hidden);
  rms_norm_modulate_fp4_quant(t.q, t.blocks, t.scales, h, x, weight, eps, shift, scale, index);
  return {t.q, t.blocks, t.scales, h};
}

std::tuple<at::Tensor, at::Tensor, std::optional<at::Tensor>, at::Tensor, std::optional<at::Tensor>>
residual_gate_rms_norm_modulate_fp4_quant_new(const at::Tensor& residual, const at::Tensor& branch,
                                              const at::Tensor& gate, const at::Tensor& weight,
                                              double eps, const at::Tensor& shift,
                                              const at::Tensor& scale,
                                              const std::optional<at::Tensor>& index, bool mx,
                                              bool hidden) {
  const c10::cuda::CUDAGuard guard(residual.device());
  Fp4Tensors t = empty_fp4(residual, mx, true);
  const std::optional<at::Tensor> h = empty_hidden(residual, hidden);
  at::Tensor residual_out = at::empty_like(residual);
  residual_gate_rms_norm_modulate_fp4_quant(t.q, t.blocks, t.scales, residual_out, h, residual,
                                            branch, gate, weight, eps, shift, scale, index);
  return {t.q, t.blocks, t.scales, residual_out, h};
}

}  // namespace

TORCH_LIBRARY(taomate_w8a8, m) {
  m.def("dynamic_scaled_int8_quant(Tensor(a!) result, Tensor input, Tensor(b!) scale, Tensor? azp) -> ()");
  m.def("static_scaled_int8_quant(Tensor(a!) result, Tensor input, Tensor scale, Tensor? azp) -> ()");
  m.def(
      "cutlass_scaled_mm(Tensor(a!) out, Tensor a, Tensor b, Tensor a_scales, Tensor b_scales, "
      "Tensor? bias) -> ()");
  m.def(
      "scaled_mm_i8_ex(Tensor(a!) out, Tensor a, Tensor b, Tensor a_scales, Tensor b_scales, "
      "Tensor? bias, int epilogue, Tensor(b!)? acc_debug, int tile_n) -> ()");
  m.def(
      "scaled_mm_i8_lora(Tensor(a!) out, Tensor a, Tensor b, Tensor a_scales, Tensor b_scales, "
      "Tensor? bias, Tensor lora_t, Tensor lora_b, int epilogue) -> ()");
  m.def(
      "scaled_mm_i8_ulysses_send(Tensor(a!) send, Tensor a, Tensor b, Tensor a_scales, "
      "Tensor b_scales, Tensor? bias, int num_heads, int head_dim, int world) -> ()");
  m.def("quantize_weight_int8(Tensor(a!) q, Tensor(b!) scales, Tensor w) -> ()");
  m.def("lora_down_proj(Tensor(a!) t, Tensor x, Tensor a) -> ()");
  m.def(
      "modulate_int8_quant(Tensor(a!) out, Tensor(b!) scales, Tensor(c!)? hidden_out, Tensor x, "
      "Tensor shift, Tensor scale, Tensor? index) -> ()");
  m.def(
      "rms_norm_modulate_int8_quant(Tensor(a!) out, Tensor(b!) scales, Tensor(c!)? hidden_out, "
      "Tensor x, Tensor weight, float eps, Tensor shift, Tensor scale, Tensor? index) -> ()");
  m.def(
      "residual_gate_rms_norm_modulate_int8_quant(Tensor(a!) out, Tensor(b!) scales, "
      "Tensor(c!) residual_out, Tensor(d!)? hidden_out, Tensor residual, Tensor branch, "
      "Tensor gate, Tensor weight, float eps, Tensor shift, Tensor scale, Tensor? index) -> ()");
  m.def(
      "scaled_fp4_quant(Tensor(a!) q, Tensor(b!) block_scales, Tensor(c!)? scales, Tensor input, "
      "Tensor? given_scale) -> ()");
  m.def(
      "dequantize_fp4(Tensor(a!) out, Tensor q, Tensor block_scales, Tensor? scales) -> ()");
  m.def(
      "modulate_fp4_quant(Tensor(a!) q, Tensor(b!) block_scales, Tensor(c!)? scales, "
      "Tensor(d!)? hidden_out, Tensor x, Tensor shift, Tensor scale, Tensor? index) -> ()");
  m.def(
      "rms_norm_modulate_fp4_quant(Tensor(a!) q, Tensor(b!) block_scales, Tensor(c!)? scales, "
      "Tensor(d!)? hidden_out, Tensor x, Tensor weight, float eps, Tensor shift, Tensor scale, "
      "Tensor? index) -> ()");
  m.def(
      "residual_gate_rms_norm_modulate_fp4_quant(Tensor(a!) q, Tensor(b!) block_scales, "
      "Tensor(c!)? scales, Tensor(d!) residual_out, Tensor(e!)? hidden_out, Tensor residual, "
      "Tensor branch, Tensor gate, Tensor weight, float eps, Tensor shift, Tensor scale, "
      "Tensor? index) -> ()");
  m.def(
      "scaled_mm_fp4(Tensor(a!) out, Tensor a, Tensor b, Tensor block_scales_a, "
      "Tensor block_scales_b, Tensor? scales_a, Tensor? scales_b, Tensor? bias, int epilogue, "
      "int tile, int splits) -> ()");
  m.def(
      "scaled_fp4_quant_new(Tensor input, Tensor? scale, bool mx) -> (Tensor, Tensor, Tensor?)");
  m.def(
      "dequantize_fp4_new(Tensor q, Tensor block_scales, Tensor? scales, ScalarType dtype) -> "
      "Tensor");
  m.def(
      "scaled_mm_fp4_new(Tensor a, Tensor b, Tensor block_scales_a, Tensor block_scales_b, "
      "Tensor? scales_a, Tensor? scales_b, ScalarType dtype, Tensor? bias, int epilogue) -> "
      "Tensor");
  m.def(
      "modulate_fp4_quant_new(Tensor x, Tensor shift, Tensor scale, Tensor? index, bool mx, "
      "bool hidden) -> (Tensor, Tensor, Tensor?, Tensor?)");
  m.def(
      "rms_norm_modulate_fp4_quant_new(Tensor x, Tensor weight, float eps, Tensor shift, "
      "Tensor scale, Tensor? index, bool mx, bool hidden) -> (Tensor, Tensor, Tensor?, Tensor?)");
  m.def(
      "residual_gate_rms_norm_modulate_fp4_quant_new(Tensor residual, Tensor branch, Tensor gate, "
      "Tensor weight, float eps, Tensor shift, Tensor scale, Tensor? index, bool mx, bool hidden) "
      "-> (Tensor, Tensor, Tensor?, Tensor, Tensor?)");
}

TORCH_LIBRARY_IMPL(taomate_w8a8, CUDA, m) {
  m.impl("dynamic_scaled_int8_quant", &dynamic_scaled_int8_quant);
  m.impl("static_scaled_int8_quant", &static_scaled_int8_quant);
  m.impl("cutlass_scaled_mm", &cutlass_scaled_mm);
  m.impl("scaled_mm_i8_ex", &scaled_mm_i8_ex);
  m.impl("scaled_mm_i8_lora", &scaled_mm_i8_lora);
  m.impl("scaled_mm_i8_ulysses_send", &scaled_mm_i8_ulysses_send);
  m.impl("quantize_weight_int8", &quantize_weight_int8);
  m.impl("lora_down_proj", &lora_down_proj);
  m.impl("modulate_int8_quant", &modulate_int8_quant);
  m.impl("rms_norm_modulate_int8_quant", &rms_norm_modulate_int8_quant);
  m.impl("residual_gate_rms_norm_modulate_int8_quant",
         &residual_gate_rms_norm_modulate_int8_quant);
  m.impl("scaled_fp4_quant", &scaled_fp4_quant);
  m.impl("dequantize_fp4", &dequantize_fp4);
  m.impl("modulate_fp4_quant", &modulate_fp4_quant);
  m.impl("rms_norm_modulate_fp4_quant", &rms_norm_modulate_fp4_quant);
  m.impl("residual_gate_rms_norm_modulate_fp4_quant", &residual_gate_rms_norm_modulate_fp4_quant);
  m.impl("scaled_mm_fp4", &scaled_mm_fp4);
  m.impl("scaled_fp4_quant_new", &scaled_fp4_quant_new);
  m.impl("dequantize_fp4_new", &dequantize_fp4_new);
  m.impl("scaled_mm_fp4_new", &scaled_mm_fp4_new);
  m.impl("modulate_fp4_quant_new", &modulate_fp4_quant_new);
  m.impl("rms_norm_modulate_fp4_quant_new", &rms_norm_modulate_fp4_quant_new);
  m.impl("residual_gate_rms_norm_modulate_fp4_quant_new",
         &residual_gate_rms_norm_modulate_fp4_quant_new);
}
