// Entry points of the operators on 8-bit floating-point blocks over device pointers, and the dense
// product of float x, whose codes live in pool memory for the length of the call (the pool is
// ordered by the backend's stream, so the block may be handed out again once the product is queued).
#include <algorithm>
#include <string>

#include "mxrt_internal.h"

namespace mx {
namespace {

bool f32_or_bf16(int dt) { return dt == MX_DTYPE_FLOAT32 || dt == MX_DTYPE_BFLOAT16; }
int64_t blocks(int64_t n) { return (n + MX_F8_BLOCK - 1) / MX_F8_BLOCK; }

bool misaligned(const void* p, int dt) { return p && (uintptr_t)p % (uintptr_t)(dtype_bits(dt) / 8) != 0; }

int check_dims(const char* op, int64_t M, int64_t K, int64_t N) {
  constexpr int64_t kMost = (int64_t)1 << 30;  // kernels index a tile past the last row or column in 32 bits
  if (M < 0 || K < 0 || N < 0)
    return set_error(MX_ERR_INVALID, "%s: negative size", op);
  if (M >= kMost || K >= kMost || N >= kMost)
    return set_error(MX_ERR_INVALID, "%s: rows and columns must be < 2^30", op);
  constexpr int64_t kArray = (int64_t)1 << 45;  // more values than any device holds; sizes in bytes stay in 64 bits
  if (M * K > kArray || K * N > kArray || M * N > kArray)
    return set_error(MX_ERR_INVALID, "%s: an array of more than 2^45 values", op);
  return MX_OK;
}

int check_float(const char* op, const char* what, int dt) {
  if (!f32_or_bf16(dt))
    return set_error(MX_ERR_NOT_IMPLEMENTED, "%s: %s must be Float32 or BFloat16, got %s", op, what, dtype_name(dt));
  return MX_OK;
}

int null_pointer(const char* op) { return set_error(MX_ERR_INVALID, "%s: NULL data pointer", op); }
int bad_alignment(const char* op) {
  return set_error(MX_ERR_INVALID, "%s: float32 data must be 4-byte aligned and bfloat16 data 2-byte aligned", op);
}

// Whether [p, p + n) and [q, q + m) share a byte.
bool overlap(const void* p, int64_t n, const void* q, int64_t m) {
  const uintptr_t a = (uintptr_t)p, c = (uintptr_t)q;
  return p && q && n > 0 && m > 0 && a < c + (uintptr_t)m && c < a + (uintptr_t)n;
}
int overlapping(const char* op) { return set_error(MX_ERR_INVALID, "%s: an output overlaps another array", op); }

// The backend's device is current for the length of the call.
class OnDevice {
 public:
  explicit OnDevice(mx_backend* b) {
    if (hipGetDevice(&before_) != hipSuccess) before_ = b->device;
    if (before_ != b->device) rc_ = hipSetDevice(b->device);
    changed_ = before_ != b->device;
  }
  ~OnDevice() {
    if (changed_) (void)hipSetDevice(before_);
  }
  hipError_t status() const { return rc_; }

 private:
  int before_ = 0;
  bool changed_ = false;
  hipError_t rc_ = hipSuccess;
};

template <typename F>
int on_backend(mx_backend* b, F&& fn) {
  std::lock_guard<std::recursive_mutex> lk(b->mu);
  OnDevice dev(b);
  MX_CHECK_HIP(dev.status());
  return fn();
}

int validate(const mx_f8_quantize_args* a, F8QuantizeDesc* d) {
  const char* op = "F8Quantize";
  if (!a) return set_error(MX_ERR_INVALID, "%s: args is NULL", op);
  MX_TRY(check_float(op, "x", a->x_dtype));
  if (a->block_rows != 1 && a->block_rows != MX_F8_BLOCK)
    return set_error(MX_ERR_NOT_IMPLEMENTED, "%s: block_rows must be 1 or %d, got %d", op, MX_F8_BLOCK, a->block_rows);
  MX_TRY(check_dims(op, a->M, a->K, 0));
  if (a->M > 0 && a->K > 0) {
    if (!a->x || !a->codes || !a->scale) return null_pointer(op);
    const int64_t n = a->M * a->K, nx = n * dtype_bits(a->x_dtype) / 8;
    const int64_t ns = 4 * (a->block_rows == 1 ? a->M : blocks(a->M)) * blocks(a->K);
    if (overlap(a->codes, n, a->x, nx) || overlap(a->scale, ns, a->x, nx) || overlap(a->codes, n, a->scale, ns))
      return overlapping(op);
  }
  if (misaligned(a->x, a->x_dtype) || misaligned(a->scale, MX_DTYPE_FLOAT32)) return bad_alignment(op);
  *d = F8QuantizeDesc{a->x, (uint8_t*)a->codes, a->scale, a->M, a->K, a->x_dtype, a->block_rows};
  return MX_OK;
}

int validate(const mx_f8_dense_args* a, F8DenseDesc* d) {
  const char* op = "F8Dense";
  if (!a) return set_error(MX_ERR_INVALID, "%s: args is NULL", op);
  const bool codes = a->x_dtype == MX_DTYPE_F8E4M3FN;
  if (!codes && !f32_or_bf16(a->x_dtype))
    return set_error(MX_ERR_NOT_IMPLEMENTED, "%s: x must be F8E4M3FN, Float32 or BFloat16, got %s", op, dtype_name(a->x_dtype));
  if (!codes && a->x_scale) return set_error(MX_ERR_INVALID, "%s: x in %s takes no scales", op, dtype_name(a->x_dtype));
  if (a->bias) MX_TRY(check_float(op, "bias", a->bias_dtype));
  MX_TRY(check_float(op, "out", a->out_dtype));
  if (a->weight_layout != MX_DENSE_LAYOUT_INPUT_OUTPUTS && a->weight_layout != MX_DENSE_LAYOUT_OUTPUTS_INPUT)
    return set_error(MX_ERR_INVALID, "%s: unknown weight_layout %d", op, a->weight_layout);
  if (a->activation < MX_ACT_NONE || a->activation > MX_ACT_TANH)
    return set_error(MX_ERR_INVALID, "%s: unknown activation %d", op, a->activation);
  MX_TRY(check_dims(op, a->M, a->K, a->N));
  if (a->M > 0 && a->N > 0) {
    if (!a->out || (a->K > 0 && (!a->x || !a->w || !a->w_scale || (codes && !a->x_scale)))) return null_pointer(op);
    const int64_t n = a->M * a->N * dtype_bits(a->out_dtype) / 8;
    if (overlap(a->out, n, a->x, a->M * a->K * dtype_bits(a->x_dtype) / 8) || overlap(a->out, n, a->w, a->K * a->N) ||
        overlap(a->out, n, a->x_scale, 4 * a->M * blocks(a->K)) || overlap(a->out, n, a->w_scale, 4 * blocks(a->K) * blocks(a->N)) ||
        (a->bias && overlap(a->out, n, a->bias, a->N * dtype_bits(a->bias_dtype) / 8)))
      return overlapping(op);
  }
  if (misaligned(a->x, a->x_dtype) || misaligned(a->x_scale, MX_DTYPE_FLOAT32) || misaligned(a->w_scale, MX_DTYPE_FLOAT32) ||
      (a->bias && misaligned(a->bias, a->bias_dtype)) || misaligned(a->out, a->out_dtype))
    return bad_alignment(op);
  *d = F8DenseDesc{a->x, a->x_scale, (const uint8_t*)a->w, a->w_scale, a->bias, a->out, a->M, a->K, a->N,
                   a->x_dtype, a->bias ? a->bias_dtype : 0, a->out_dtype, a->activation,
                   a->weight_layout == MX_DENSE_LAYOUT_OUTPUTS_INPUT};
  return MX_OK;
}

int validate(const mx_f8_weight_grad_args* a, F8WGradDesc* d) {
  const char* op = "F8WeightGradient";
  if (!a) return set_error(MX_ERR_INVALID, "%s: args is NULL", op);
  MX_TRY(check_float(op, "dy", a->dy_dtype));
  MX_TRY(check_float(op, "out", a->out_dtype));
  if (a->weight_layout != MX_DENSE_LAYOUT_INPUT_OUTPUTS && a->weight_layout != MX_DENSE_LAYOUT_OUTPUTS_INPUT)
    return set_error(MX_ERR_INVALID, "%s: unknown weight_layout %d", op, a->weight_layout);
  MX_TRY(check_dims(op, a->M, a->K, a->N));
  if (a->K > 0 && a->N > 0) {
    if (!a->out || (a->M > 0 && (!a->x || !a->x_scale || !a->dy))) return null_pointer(op);
    const int64_t n = a->K * a->N * dtype_bits(a->out_dtype) / 8;
    if (overlap(a->out, n, a->x, a->M * a->K) || overlap(a->out, n, a->x_scale, 4 * a->M * blocks(a->K)) ||
        overlap(a->out, n, a->dy, a->M * a->N * dtype_bits(a->dy_dtype) / 8))
      return overlapping(op);
  }
  if (misaligned(a->x_scale, MX_DTYPE_FLOAT32) || misaligned(a->dy, a->dy_dtype) || misaligned(a->out, a->out_dtype))
    return bad_alignment(op);
  *d = F8WGradDesc{(const uint8_t*)a->x, a->x_scale, a->dy, a->out, a->M, a->K, a->N, a->dy_dtype, a->out_dtype,
                   a->weight_layout == MX_DENSE_LAYOUT_OUTPUTS_INPUT};
  return MX_OK;
}

int validate(const mx_f8_act_grad_args* a, F8ActGradDesc* d) {
  const char* op = "F8ActivationGradient";
  if (!a) return set_error(MX_ERR_INVALID, "%s: args is NULL", op);
  MX_TRY(check_float(op, "dy", a->dy_dtype));
  if (a->activation < MX_ACT_NONE || a->activation > MX_ACT_TANH)
    return set_error(MX_ERR_INVALID, "%s: unknown activation %d", op, a->activation);
  MX_TRY(check_dims(op, a->M, 0, a->N));
  if (a->M > 0 && a->N > 0) {
    if ((a->up != nullptr) != (a->up_scale != nullptr) || (a->up != nullptr) != (a->dup != nullptr))
      return set_error(MX_ERR_INVALID, "%s: up, up_scale and dup come together", op);
    if (!a->z || !a->z_scale || !a->dy || !a->dz) return null_pointer(op);
    const int64_t n = a->M * a->N, nf = n * dtype_bits(a->dy_dtype) / 8, ns = 4 * a->M * blocks(a->N);
    auto hits = [&](const void* o) {
      return overlap(o, nf, a->z, n) || overlap(o, nf, a->up, n) || overlap(o, nf, a->z_scale, ns) || overlap(o, nf, a->up_scale, ns);
    };
    if (hits(a->dz) || hits(a->dup) || overlap(a->dup, nf, a->dz, nf) || overlap(a->dup, nf, a->dy, nf) ||
        (a->dz != a->dy && overlap(a->dz, nf, a->dy, nf)))
        return overlapping(op);
  }
  if (misaligned(a->z_scale, MX_DTYPE_FLOAT32) || misaligned(a->up_scale, MX_DTYPE_FLOAT32) || misaligned(a->dy, a->dy_dtype) ||
      misaligned(a->dz, a->dy_dtype) || misaligned(a->dup, a->dy_dtype))
    return bad_alignment(op);
  *d = F8ActGradDesc{(const uint8_t*)a->z, a->z_scale, (const uint8_t*)a->up, a->up_scale, a->dy, a->dz, a->dup, a->M, a->N,
                     a->dy_dtype, a->activation};
  return MX_OK;
}

int copy_name(const std::string& s, char* buf, size_t buflen) {
  if (buf && buflen) {
    const size_t n = std::min(buflen - 1, s.size());
    memcpy(buf, s.data(), n);
    buf[n] = 0;
  }
  return MX_OK;
}

}  // namespace

// Whether the product of float x takes codes that are made first.
static bool makes_codes(const F8DenseDesc& d) { return d.x_dt != MX_DTYPE_F8E4M3FN && d.K != 0 && !f8_product_takes_float(d); }

// The product over codes in memory of the call's own.
static F8DenseDesc over_codes(F8DenseDesc d, void* codes, float* scale) {
  d.x = codes;
  d.x_scale = scale;
  d.x_dt = MX_DTYPE_F8E4M3FN;
  return d;
}

int f8_dense_run(mx_backend* b, const F8DenseDesc& d) {
  if (d.M == 0 || d.N == 0) return MX_OK;
  if (!makes_codes(d)) return f8_product_run(b, d);
  // Codes, then scales on a 256-byte boundary, in one block.
  const size_t codes = ((size_t)d.M * d.K + 255) & ~(size_t)255;
  void* mem = nullptr;
  MX_TRY(dev_alloc(b, codes + (size_t)4 * d.M * blocks(d.K), &mem));
  const F8DenseDesc p = over_codes(d, mem, (float*)((char*)mem + codes));
  int rc = f8_quantize_run(b, F8QuantizeDesc{d.x, (uint8_t*)mem, (float*)p.x_scale, d.M, d.K, d.x_dt, 1});
  if (rc == MX_OK) rc = f8_product_run(b, p);
  dev_free(b, mem);
  return rc;
}

}  // namespace mx

extern "C" {

int mx_f8_quantize(mx_backend* b, const mx_f8_quantize_args* args) {
  mx::clear_error();
  MX_TRY(mx::check_device(b));
  mx::F8QuantizeDesc d;
  MX_TRY(mx::validate(args, &d));
  return mx::on_backend(b, [&] { return mx::f8_quantize_run(b, d); });
}

int mx_f8_dense(mx_backend* b, const mx_f8_dense_args* args) {
  mx::clear_error();
  MX_TRY(mx::check_device(b));
  mx::F8DenseDesc d;
  MX_TRY(mx::validate(args, &d));
  return mx::on_backend(b, [&] { return mx::f8_dense_run(b, d); });
}

int mx_f8_dense_plan(mx_backend* b, const mx_f8_dense_args* args, char* buf, size_t buflen) {
  mx::clear_error();
  if (!b) return mx::set_error(MX_ERR_INVALID, "backend is NULL");
  mx::F8DenseDesc d;
  MX_TRY(mx::validate(args, &d));
  if (mx::makes_codes(d)) d = mx::over_codes(d, nullptr, nullptr);  // (pool memory is aligned, as NULL is)
  return mx::copy_name(mx::f8_product_plan(d), buf, buflen);
}

int mx_f8_weight_gradient(mx_backend* b, const mx_f8_weight_grad_args* args) {
  mx::clear_error();
  MX_TRY(mx::check_device(b));
  mx::F8WGradDesc d;
  MX_TRY(mx::validate(args, &d));
  return mx::on_backend(b, [&] { return mx::f8_wgrad_run(b, d); });
}

int mx_f8_weight_gradient_plan(mx_backend* b, const mx_f8_weight_grad_args* args, char* buf, size_t buflen) {
  mx::clear_error();
  if (!b) return mx::set_error(MX_ERR_INVALID, "backend is NULL");
  mx::F8WGradDesc d;
  MX_TRY(mx::validate(args, &d));
  return mx::copy_name(mx::f8_wgrad_plan(d), buf, buflen);
}

int mx_f8_activation_gradient(mx_backend* b, const mx_f8_act_grad_args* args) {
  mx::clear_error();
  MX_TRY(mx::check_device(b));
  mx::F8ActGradDesc d;
  MX_TRY(mx::validate(args, &d));
  return mx::on_backend(b, [&] { return mx::f8_act_grad_run(b, d); });
}

}  // extern "C"
