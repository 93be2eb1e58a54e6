// torch bindings of the block operators: rms_norm_quant, linear_fp8, rope_axes, cross_attention.
// As in bindings.cpp every rule that keeps a launch inside its buffers is checked here, so a bad call
// raises a Python exception instead of reaching the GPU.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>

#include "kernels.h"

namespace {

int elem_type(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return ds::kBF16;
    case at::kHalf: return ds::kFP16;
    case at::kFloat: return ds::kFP32;
    default: TORCH_CHECK(false, name, " must be bfloat16, float16 or float32");
  }
}

void check_rows(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device());
  TORCH_CHECK(t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1), name, " must be 2-D with unit column stride");
}

// an output's rows must not overlap each other
void check_output(const at::Tensor& t, const at::Tensor& like, const char* name) {
  check_rows(t, like, name);
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " must have rows that do not overlap");
}

void check_vector(const at::Tensor& t, const at::Tensor& like, int64_t n, at::ScalarType type, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device());
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n && t.scalar_type() == type, name, " must be ", type, " [", n, "]");
}

void rms_norm_quant(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                    const c10::optional<at::Tensor>& residual, c10::optional<at::Tensor> h, at::Tensor& q,
                    at::Tensor& scale, double eps) {
  check_rows(x, x, "x");
  ds::NormQuantArgs a;
  a.type = elem_type(x, "x");
  check_output(q, x, "out");
  TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn && q.sizes() == x.sizes(), "out must be float8_e4m3fn of x's shape");
  check_vector(scale, x, x.size(0), at::kFloat, "scale_out");
  TORCH_CHECK(residual.has_value() == h.has_value(), "rms_norm_quant: a residual needs its output and the reverse");
  if (residual.has_value()) {
    check_rows(*residual, x, "residual");
    check_output(*h, x, "residual_out");
    TORCH_CHECK(residual->sizes() == x.sizes() && h->sizes() == x.sizes() &&
                    residual->scalar_type() == x.scalar_type() && h->scalar_type() == x.scalar_type(),
                "residual and residual_out must have x's shape and type");
    a.residual = residual->data_ptr();
    a.r_stride = residual->stride(0);
    a.h = h->data_ptr();
    a.h_stride = h->stride(0);
  }
  if (weight.has_value()) {
    check_vector(*weight, x, x.size(1), x.scalar_type(), "weight");
    TORCH_CHECK(weight->stride(0) == 1 || weight->size(0) == 1, "weight must be contiguous");
    a.weight = weight->data_ptr();
  }
  TORCH_CHECK(x.size(1) > 0 && x.size(1) < (int64_t{1} << 30), "rms_norm_quant: bad row length");
  const c10::cuda::CUDAGuard guard(x.device());
  a.x = x.data_ptr();
  a.x_stride = x.stride(0);
  a.q = reinterpret_cast<uint8_t*>(q.data_ptr());
  a.q_stride = q.stride(0);
  a.scale = scale.data_ptr<float>();
  a.scale_stride = scale.stride(0);
  a.rows = x.size(0);
  a.dim = static_cast<int>(x.size(1));
  a.eps = static_cast<float>(eps);
  ds::launch_norm_quant(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void linear_fp8(const at::Tensor& x, const at::Tensor& sx, const at::Tensor& w, const at::Tensor& sw, at::Tensor& y,
                const c10::optional<at::Tensor>& bias, bool gelu, const c10::optional<at::Tensor>& residual,
                const c10::optional<at::Tensor>& gate, int64_t rows_per_batch,
                const c10::optional<at::Tensor>& row_batch, const at::Tensor& status) {
  check_rows(x, x, "xq");
  check_rows(w, x, "wq");
  TORCH_CHECK(x.scalar_type() == at::kFloat8_e4m3fn && w.scalar_type() == at::kFloat8_e4m3fn,
              "xq and wq must be float8_e4m3fn");
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK(w.size(1) == K, "linear_fp8: K mismatch");
  TORCH_CHECK(K > 0 && K <= (1 << 30) && M <= (1 << 30) && N <= (1 << 30), "linear_fp8: sizes out of range");
  for (const at::Tensor* t : {&x, &w})
    TORCH_CHECK(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0 &&
                    (t->size(0) <= 1 || (t->stride(0) % 16 == 0 && t->stride(0) >= K)),
                "xq and wq must have rows that start on 16 bytes");
  check_vector(sx, x, M, at::kFloat, "x_scale");
  check_vector(sw, x, N, at::kFloat, "w_scale");
  check_output(y, x, "out");
  TORCH_CHECK(y.size(0) == M && y.size(1) == N, "linear_fp8: out must be [", M, ", ", N, "]");
  ds::LinearFp8Args a;
  a.out_type = elem_type(y, "out");
  if (bias.has_value()) {
    check_vector(*bias, x, N, y.scalar_type(), "bias");
    TORCH_CHECK(bias->stride(0) == 1 || N == 1, "bias must be contiguous");
    a.bias = bias->data_ptr();
  }
  if (residual.has_value()) {
    check_rows(*residual, x, "residual");
    TORCH_CHECK(residual->sizes() == y.sizes() && residual->scalar_type() == y.scalar_type(),
                "residual must have out's shape and type");
    a.residual = residual->data_ptr();
    a.ldr = residual->stride(0);
  }
  if (gate.has_value()) {
    check_rows(*gate, x, "gate");
    TORCH_CHECK(residual.has_value(), "linear_fp8: a gate needs a residual");
    TORCH_CHECK(gate->scalar_type() == at::kFloat && gate->size(1) == N && gate->size(0) >= 1, "gate must be fp32 [B, N]");
    a.gate = gate->data_ptr<float>();
    a.gate_stride = gate->stride(0);
    a.batches = static_cast<int>(gate->size(0));
    TORCH_CHECK(rows_per_batch > 0, "rows_per_batch must be positive");
    a.rows_per_batch = static_cast<int>(std::min<int64_t>(rows_per_batch, 1 << 30));
    if (row_batch.has_value()) {
      check_vector(*row_batch, x, M, at::kInt, "row_batch");
      TORCH_CHECK(row_batch->stride(0) == 1 || M == 1, "row_batch must be contiguous");
      a.row_batch = row_batch->data_ptr<int>();
    } else {
      TORCH_CHECK((M + rows_per_batch - 1) / rows_per_batch <= gate->size(0), "gate has too few rows");
    }
  }
  TORCH_CHECK(status.is_cuda() && status.device() == x.device() && status.scalar_type() == at::kInt && status.numel() >= 2,
              "status must be int32 with 2 elements on ", x.device());
  const c10::cuda::CUDAGuard guard(x.device());
  a.x = reinterpret_cast<const uint8_t*>(x.data_ptr());
  a.ldx = M > 1 ? x.stride(0) : (K + 15) / 16 * 16;
  a.w = reinterpret_cast<const uint8_t*>(w.data_ptr());
  a.ldw = N > 1 ? w.stride(0) : (K + 15) / 16 * 16;
  a.sx = sx.data_ptr<float>();
  a.sx_stride = sx.stride(0);
  a.sw = sw.data_ptr<float>();
  a.sw_stride = sw.stride(0);
  a.y = y.data_ptr();
  a.ldy = y.stride(0);
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.gelu = gelu ? 1 : 0;
  a.status = status.data_ptr<int>();
  ds::launch_linear_fp8(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void rope_axes(const at::Tensor& x, at::Tensor& y, const c10::optional<at::Tensor>& k, c10::optional<at::Tensor> ky,
               const at::Tensor& pos, const std::vector<int64_t>& dims, const std::vector<double>& theta,
               int64_t head_dim, bool half, bool inverse) {
  ds::RopeAxesArgs a;
  a.type = elem_type(x, "x");
  TORCH_CHECK(head_dim > 0 && head_dim <= (1 << 20), "rope_axes: bad head_dim");
  const int64_t rows = x.size(0);
  auto fill = [&](ds::RopeTensor& t, const at::Tensor& in, const at::Tensor& out, const char* name) {
    check_rows(in, x, name);
    check_output(out, x, "out");
    TORCH_CHECK(in.scalar_type() == x.scalar_type() && out.scalar_type() == x.scalar_type() && in.size(0) == rows &&
                    out.sizes() == in.sizes(),
                "rope_axes: ", name, " and its output must agree in rows, shape and type");
    TORCH_CHECK(in.size(1) % head_dim == 0 && in.size(1) < (int64_t{1} << 30), name, " must hold whole heads");
    t.x = in.data_ptr();
    t.x_stride = in.stride(0);
    t.y = out.data_ptr();
    t.y_stride = out.stride(0);
    t.heads = static_cast<int>(in.size(1) / head_dim);
  };
  fill(a.t[0], x, y, "x");
  TORCH_CHECK(k.has_value() == ky.has_value(), "rope_axes: k needs its output and the reverse");
  if (k.has_value()) fill(a.t[1], *k, *ky, "k");
  TORCH_CHECK(pos.is_cuda() && pos.device() == x.device() && pos.dim() == 2, "positions must be [P, axes] on ", x.device());
  TORCH_CHECK(dims.size() >= 1 && dims.size() <= ds::kRopeMaxAxes && dims.size() == theta.size() &&
                  pos.size(1) == static_cast<int64_t>(dims.size()),
              "rope_axes: one to ", ds::kRopeMaxAxes, " axes, each with its dims, theta and position");
  TORCH_CHECK(rows == 0 || (pos.size(0) > 0 && rows % pos.size(0) == 0), "rope_axes: rows must be a multiple of positions");
  switch (pos.scalar_type()) {
    case at::kLong: a.pos_type = 0; break;
    case at::kInt: a.pos_type = 1; break;
    case at::kFloat: a.pos_type = 2; break;
    case at::kDouble: a.pos_type = 3; break;
    default: TORCH_CHECK(false, "positions must be int64, int32, float32 or float64");
  }
  int pairs = 0;
  for (size_t i = 0; i < dims.size(); ++i) {
    TORCH_CHECK(dims[i] > 0 && dims[i] % 2 == 0 && dims[i] <= head_dim && pairs + dims[i] / 2 <= ds::kRopeMaxPairs,
                "rope_axes: dims must be positive, even, and at most ", 2 * ds::kRopeMaxPairs, " together");
    for (int64_t j = 0; j < dims[i] / 2; ++j, ++pairs) {
      a.axis[pairs] = static_cast<uint8_t>(i);
      a.turns[pairs] = std::pow(theta[i], -2.0 * static_cast<double>(j) / static_cast<double>(dims[i])) / (2.0 * M_PI);
    }
  }
  TORCH_CHECK(2 * pairs <= head_dim, "rope_axes: dims exceed head_dim");
  const c10::cuda::CUDAGuard guard(x.device());
  a.rows = rows;
  a.head_dim = static_cast<int>(head_dim);
  a.pairs = pairs;
  a.half = half ? 1 : 0;
  a.inverse = inverse ? 1 : 0;
  a.pos = pos.data_ptr();
  a.pos_rows = pos.size(0);
  a.pos_stride = pos.stride(0);
  a.axis_stride = pos.stride(1);
  ds::launch_rope_axes(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void cross_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& o,
                     c10::optional<at::Tensor> lse, const c10::optional<at::Tensor>& kv_lens,
                     const c10::optional<at::Tensor>& key_mask, int64_t heads, int64_t heads_kv, int64_t head_dim,
                     double scale, const at::Tensor& status) {
  ds::CrossAttnArgs a;
  a.type = elem_type(q, "q");
  TORCH_CHECK(q.is_cuda() && q.dim() == 3, "q must be a CUDA tensor [B, Sq, heads * head_dim]");
  const int64_t B = q.size(0), Sq = q.size(1), Sk = k.dim() == 3 ? k.size(1) : -1;
  TORCH_CHECK(heads > 0 && heads_kv > 0 && heads % heads_kv == 0, "cross_attention: heads must be a multiple of heads_kv");
  TORCH_CHECK(B <= 65535 && heads_kv <= 65535 && Sk > 0 && Sk < (int64_t{1} << 30) &&
                  Sq * (heads / heads_kv) < (int64_t{1} << 30) && heads * head_dim < (int64_t{1} << 30),
              "cross_attention: sizes out of range");
  auto check = [&](const at::Tensor& t, int64_t rows, int64_t width, const char* name, bool output) {
    TORCH_CHECK(t.is_cuda() && t.device() == q.device() && t.scalar_type() == q.scalar_type(), name,
                " must have q's device and type");
    TORCH_CHECK(t.dim() == 3 && t.size(0) == B && t.size(1) == rows && t.size(2) == width, name, " must be [", B, ", ",
                rows, ", ", width, "]");
    TORCH_CHECK(t.stride(2) == 1 && t.stride(1) % 8 == 0 && t.stride(0) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
                name, " must have rows that start on 16 bytes");
    if (output)
      TORCH_CHECK((rows <= 1 || t.stride(1) >= width) && (B <= 1 || t.stride(0) >= width), name,
                  " must have rows that do not overlap");
  };
  check(q, Sq, heads * head_dim, "q", false);
  check(k, Sk, heads_kv * head_dim, "k", false);
  check(v, Sk, heads_kv * head_dim, "v", false);
  check(o, Sq, heads * head_dim, "out", true);
  if (lse.has_value()) {
    TORCH_CHECK(lse->is_cuda() && lse->device() == q.device() && lse->scalar_type() == at::kFloat && lse->is_contiguous() &&
                    lse->numel() == B * heads * Sq,
                "lse must be contiguous fp32 [B, heads, Sq]");
    a.lse = lse->data_ptr<float>();
  }
  at::Tensor lens;
  if (kv_lens.has_value()) {
    check_vector(*kv_lens, q, B, at::kInt, "kv_lens");
    lens = kv_lens->contiguous();
    a.kv_lens = lens.data_ptr<int>();
  }
  if (key_mask.has_value()) {
    TORCH_CHECK(key_mask->is_cuda() && key_mask->device() == q.device() && key_mask->scalar_type() == at::kBool &&
                    key_mask->dim() == 2 && key_mask->size(0) == B && key_mask->size(1) == Sk,
                "key_mask must be bool [", B, ", ", Sk, "]");
    a.key_mask = reinterpret_cast<const uint8_t*>(key_mask->data_ptr());
    a.mask_row = key_mask->stride(0);
    a.mask_col = key_mask->stride(1);
  }
  TORCH_CHECK(status.is_cuda() && status.device() == q.device() && status.scalar_type() == at::kInt && status.numel() >= 2,
              "status must be int32 with 2 elements on ", q.device());
  const c10::cuda::CUDAGuard guard(q.device());
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.o = o.data_ptr();
  a.q_batch = q.stride(0), a.q_row = q.stride(1);
  a.k_batch = k.stride(0), a.k_row = k.stride(1);
  a.v_batch = v.stride(0), a.v_row = v.stride(1);
  a.o_batch = o.stride(0), a.o_row = o.stride(1);
  a.batch = static_cast<int>(B);
  a.seq_q = static_cast<int>(Sq);
  a.seq_k = static_cast<int>(Sk);
  a.heads = static_cast<int>(heads);
  a.heads_kv = static_cast<int>(heads_kv);
  a.head_dim = static_cast<int>(head_dim);
  a.scale = static_cast<float>(scale);
  a.status = status.data_ptr<int>();
  ds::launch_cross_attention(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace

void bind_block_ops(pybind11::module_& m) {
  m.def("rms_norm_quant", &rms_norm_quant, "residual addition + RMS norm + e4m3 rows with scales");
  m.def("linear_fp8", &linear_fp8, "linear layer on e4m3 operands with row scales");
  m.def("rope_axes", &rope_axes, "rotary positions with several axes");
  m.def("cross_attention", &cross_attention, "attention to padded, masked encoder states");
}
