// C entry points of the operators on device buffers (include/flowedge_b200.h,
// part 3): argument checks and errors in the manner of the engine's, then the
// launch functions of ops.h.  Host C++23, no CUDA headers.
#include "ops.h"

#include <cmath>
#include <cstddef>
#include <cstring>
#include <exception>
#include <string>

namespace {

constexpr std::uint64_t kMaxRows = std::uint64_t(1) << 30;
constexpr std::uint64_t kMaxWidth = std::uint64_t(1) << 20;

// Collects the first complaint of a call.
class Checks {
 public:
  explicit Checks(const char* call) : call_(call) {}
  void need(bool ok, const char* what) {
    if (ok_ && !ok) {
      ok_ = false;
      what_ = what;
    }
  }
  // FE_STATUS_OK, or the error recorded
  int done() const {
    if (ok_) return FE_STATUS_OK;
    feb::set_last_error(std::string(call_) + ": " + what_);
    return FE_STATUS_INVALID_ARGUMENT;
  }

 private:
  const char* call_;
  const char* what_ = "";
  bool ok_ = true;
};

std::uint64_t dtype_bytes(std::uint32_t dtype) {
  return dtype == FE_DTYPE_F32 ? 4 : dtype == FE_DTYPE_BF16 || dtype == FE_DTYPE_F16 ? 2 : 0;
}

bool aligned(const void* p, std::uint64_t bytes) { return reinterpret_cast<std::uintptr_t>(p) % bytes == 0; }

// A matrix of `rows` rows of `width` elements, `ld` elements apart.
struct Matrix {
  const void* p;
  std::uint64_t rows, width;
  std::int64_t ld;
  std::uint64_t esz;
  [[nodiscard]] std::uintptr_t begin() const { return reinterpret_cast<std::uintptr_t>(p); }
  [[nodiscard]] std::uintptr_t end() const {
    return begin() + ((rows - 1) * static_cast<std::uint64_t>(ld) + width) * esz;
  }
};

// Whether the two share a byte (true where that is not plain to see): apart,
// or columns beside one another of rows with one pitch.
bool overlap(const Matrix& a, const Matrix& b) {
  if (a.p == nullptr || b.p == nullptr || a.rows == 0 || b.rows == 0) return false;
  if (a.end() <= b.begin() || b.end() <= a.begin()) return false;
  const std::uint64_t pitch = static_cast<std::uint64_t>(a.ld) * a.esz;
  if (pitch != static_cast<std::uint64_t>(b.ld) * b.esz) return true;
  const bool first = a.begin() <= b.begin();
  const Matrix &lo = first ? a : b, &hi = first ? b : a;
  const std::uint64_t shift = (hi.begin() - lo.begin()) % pitch;
  return shift < lo.width * lo.esz || shift + hi.width * hi.esz > pitch;
}

bool row_ld(std::int64_t ld, std::uint64_t width) {
  return ld >= static_cast<std::int64_t>(width) && ld <= (std::int64_t(1) << 40);
}

// The checks that conv and scan share.
template <typename Args>
void check_sequences(Checks& c, const Args& a, const float* state, std::uint64_t per_slot) {
  c.need(a.rows <= kMaxRows && a.n_seq <= kMaxRows, "rows and n_seq are at most 2^30");
  c.need(a.n_slots <= kMaxRows, "n_slots is at most 2^30");
  c.need(a.d_inner >= 1 && a.d_inner <= kMaxWidth, "d_inner is from 1 to 2^20");
  c.need(a.offsets != nullptr || a.n_seq == a.rows, "without offsets n_seq equals rows");
  c.need(dtype_bytes(a.dtype) != 0, "unknown dtype");
  c.need(a.device >= -1, "unknown device");
  c.need(aligned(a.offsets, 4) && aligned(a.slots, 4) && aligned(a.status, 4) && aligned(state, 4),
         "offsets, slots, status and states are 4-byte aligned");
  if (state != nullptr) {
    c.need(a.n_slots >= 1, "a state needs n_slots");
    c.need(a.slots != nullptr || a.n_slots >= a.n_seq, "without slots n_slots is at least n_seq");
    c.need(a.slots == nullptr || a.n_seq <= feb::kMaxSlotSequences, "a call with slots has at most 2^16 sequences");
    c.need(a.slot_stride >= static_cast<std::int64_t>(per_slot) && a.slot_stride <= (std::int64_t(1) << 40),
           "slot_stride is at least one slot's state");
  }
}

int check_conv(const fe_conv_args* args) {
  Checks c("fe_causal_conv_device");
  c.need(args != nullptr && args->struct_size >= sizeof(fe_conv_args), "args are missing or of another size");
  if (int rc = c.done(); rc != 0) return rc;
  const fe_conv_args& a = *args;
  c.need(a.d_conv >= 1 && a.d_conv <= 8, "d_conv is from 1 to 8");
  if (int rc = c.done(); rc != 0) return rc;
  check_sequences(c, a, a.window, a.d_inner * a.d_conv);
  if (int rc = c.done(); rc != 0) return rc;
  const std::uint64_t e = dtype_bytes(a.dtype);
  c.need(a.w != nullptr && a.b != nullptr && aligned(a.w, 4) && aligned(a.b, 4), "w and b are required, 4-byte aligned");
  c.need(a.rows == 0 || (a.x != nullptr && a.u != nullptr), "x and u are required");
  c.need(aligned(a.x, e) && aligned(a.u, e), "x and u are aligned to their elements");
  c.need(row_ld(a.x_ld, a.d_inner) && row_ld(a.u_ld, a.d_inner), "x_ld and u_ld are at least d_inner");
  if (int rc = c.done(); rc != 0) return rc;
  c.need(!overlap({a.x, a.rows, a.d_inner, a.x_ld, e}, {a.u, a.rows, a.d_inner, a.u_ld, e}), "u overlaps x");
  return c.done();
}

int check_scan(const fe_scan_args* args, const char* call, bool sizes_only) {
  Checks c(call);
  c.need(args != nullptr && args->struct_size >= sizeof(fe_scan_args), "args are missing or of another size");
  if (int rc = c.done(); rc != 0) return rc;
  const fe_scan_args& a = *args;
  c.need(a.d_state >= 1 && a.d_state <= 32, "d_state is from 1 to 32");
  c.need(a.dt_rank >= 1 && a.dt_rank <= 512, "dt_rank is from 1 to 512");
  if (int rc = c.done(); rc != 0) return rc;
  check_sequences(c, a, sizes_only ? nullptr : a.state, a.d_inner * a.d_state);
  if (int rc = c.done(); rc != 0 || sizes_only) return rc;
  const std::uint64_t e = dtype_bytes(a.dtype), wd = a.dt_rank + 2 * std::uint64_t(a.d_state);
  c.need(a.a != nullptr && a.d != nullptr && a.dt_w != nullptr && a.dt_b != nullptr, "a, d, dt_w and dt_b are required");
  c.need(aligned(a.a, 4) && aligned(a.d, 4) && aligned(a.dt_w, 4) && aligned(a.dt_b, 4), "weights are 4-byte aligned");
  c.need(a.rows == 0 || (a.u != nullptr && a.proj != nullptr && a.y != nullptr), "u, proj and y are required");
  c.need(aligned(a.u, e) && aligned(a.proj, e) && aligned(a.z, e) && aligned(a.y, e),
         "u, proj, z and y are aligned to their elements");
  c.need(row_ld(a.u_ld, a.d_inner) && row_ld(a.y_ld, a.d_inner), "u_ld and y_ld are at least d_inner");
  c.need(row_ld(a.proj_ld, wd), "proj_ld is at least dt_rank + 2 d_state");
  c.need(a.z == nullptr || row_ld(a.z_ld, a.d_inner), "z_ld is at least d_inner");
  if (int rc = c.done(); rc != 0) return rc;
  const Matrix y{a.y, a.rows, a.d_inner, a.y_ld, e};
  c.need(!overlap(y, {a.u, a.rows, a.d_inner, a.u_ld, e}), "y overlaps u");
  c.need(!overlap(y, {a.z, a.rows, a.d_inner, a.z == nullptr ? 1 : a.z_ld, e}), "y overlaps z");
  c.need(!overlap(y, {a.proj, a.rows, wd, a.proj_ld, e}), "y overlaps proj");
  return c.done();
}

// Reads the caller's structure into `a` (one that ends before the layout has
// it zero) and checks it.
int check_w4(const fe_w4_args* args, fe_w4_args& a, const char* call, bool reads_x, bool writes_y, bool per_row) {
  constexpr std::size_t kFirst = offsetof(fe_w4_args, layout);
  Checks c(call);
  c.need(args != nullptr && args->struct_size >= kFirst, "args are missing or of another size");
  if (int rc = c.done(); rc != 0) return rc;
  a = {};
  std::memcpy(&a, args, args->struct_size < sizeof(a) ? kFirst : sizeof(a));
  const std::uint64_t e = dtype_bytes(a.dtype);
  const std::uint64_t x_rows = per_row ? a.rows : a.m, y_rows = per_row ? a.rows : a.m, y_width = per_row ? a.m : a.k;
  c.need(e != 0, "unknown dtype");
  c.need(a.device >= -1, "unknown device");
  c.need(a.group == 32 || a.group == 64 || a.group == 128, "group is 32, 64 or 128");
  c.need(a.m >= 1 && a.m <= kMaxWidth && a.k >= 1 && a.k <= kMaxWidth, "m and k are from 1 to 2^20");
  c.need(a.m * a.k <= std::uint64_t(1) << 38, "m k is at most 2^38");
  c.need(!per_row || a.rows <= kMaxWidth, "rows is at most 2^20");
  c.need(a.layout <= FE_W4_ROWS && a.reserved == 0, "unknown layout");
  c.need(a.packed != nullptr && aligned(a.packed, 16), "packed is required, 16-byte aligned");
  c.need(a.scales != nullptr && aligned(a.scales, 2), "scales are required, aligned to their elements");
  if (int rc = c.done(); rc != 0) return rc;
  const bool some = !per_row || a.rows > 0;
  if (reads_x && some) {
    c.need(a.x != nullptr && aligned(a.x, e), "x is required, aligned to its elements");
    c.need(row_ld(a.x_ld, a.k), "x_ld is at least k");
  }
  if (writes_y && some) {
    c.need(a.y != nullptr && aligned(a.y, e), "y is required, aligned to its elements");
    c.need(row_ld(a.y_ld, y_width), "y_ld is at least y's width");
  }
  if (int rc = c.done(); rc != 0) return rc;
  if (reads_x && writes_y)
    c.need(!overlap({a.x, x_rows, a.k, a.x_ld, e}, {a.y, y_rows, y_width, a.y_ld, e}), "y overlaps x");
  return c.done();
}

int check_norm(const fe_norm_args* args) {
  Checks c("fe_residual_norm_device");
  c.need(args != nullptr && args->struct_size >= sizeof(fe_norm_args), "args are missing or of another size");
  if (int rc = c.done(); rc != 0) return rc;
  const fe_norm_args& a = *args;
  const std::uint64_t e = dtype_bytes(a.dtype), r = dtype_bytes(a.residual_dtype);
  c.need(e != 0, "unknown dtype");
  c.need(r != 0 && (a.residual_dtype == a.dtype || a.residual_dtype == FE_DTYPE_F32),
         "residual_dtype is fp32 or dtype");
  c.need(a.device >= -1, "unknown device");
  c.need(a.rows <= kMaxRows, "rows is at most 2^30");
  c.need(a.dim >= 1 && a.dim <= 16384, "dim is from 1 to 16384");
  c.need(std::isfinite(a.scale), "scale is finite");
  c.need(a.eps >= 0.0f && std::isfinite(a.eps), "eps is finite and not negative");
  c.need(a.weight != nullptr && aligned(a.weight, 4) && aligned(a.post_weight, 4), "weight is required, 4-byte aligned");
  if (int rc = c.done(); rc != 0 || a.rows == 0) return rc;
  c.need(a.x != nullptr && a.residual != nullptr && a.out != nullptr, "x, residual and out are required");
  c.need(aligned(a.x, e) && aligned(a.gate, e) && aligned(a.out, e) && aligned(a.residual, r),
         "x, gate, residual and out are aligned to their elements");
  c.need(row_ld(a.x_ld, a.dim) && row_ld(a.residual_ld, a.dim) && row_ld(a.out_ld, a.dim),
         "x_ld, residual_ld and out_ld are at least dim");
  c.need(a.gate == nullptr || a.gate_ld == 0 || row_ld(a.gate_ld, a.dim), "gate_ld is 0 or at least dim");
  if (int rc = c.done(); rc != 0) return rc;
  const Matrix x{a.x, a.rows, a.dim, a.x_ld, e}, out{a.out, a.rows, a.dim, a.out_ld, e};
  const Matrix res{a.residual, a.rows, a.dim, a.residual_ld, r};
  const Matrix gate = a.gate_ld == 0 ? Matrix{a.gate, 1, a.dim, static_cast<std::int64_t>(a.dim), e}
                                     : Matrix{a.gate, a.rows, a.dim, a.gate_ld, e};
  c.need(!overlap(out, x) && !overlap(out, res) && !overlap(out, gate), "out overlaps another argument");
  c.need(!overlap(res, x) && !overlap(res, gate), "the residual overlaps another argument");
  return c.done();
}

// The launch's result as a status.
int launched(int code, const char* call) {
  if (code == 0) return FE_STATUS_OK;
  feb::set_last_error(std::string(call) + ": " + feb::cuda_error_text(code));
  return FE_STATUS_RESOURCE_EXHAUSTED;
}

// Runs `body` with the call's error handling: nothing is thrown across the C
// boundary.
template <typename F>
int guarded(F body) noexcept {
  try {
    feb::clear_last_error();
    return body();
  } catch (const std::exception&) {
    feb::set_last_error_text("out of host memory");
    return FE_STATUS_RESOURCE_EXHAUSTED;
  }
}

int on_device(int device, const char* call, auto launch) {
  const feb::DeviceScope scope(device);
  if (!scope.ok()) {
    feb::set_last_error(std::string(call) + ": the device cannot be used");
    return FE_STATUS_INVALID_ARGUMENT;
  }
  return launched(launch(), call);
}

}  // namespace

extern "C" {

int fe_causal_conv_device(const fe_conv_args* args, void* stream) {
  constexpr const char* kCall = "fe_causal_conv_device";
  return guarded([&] {
    if (int rc = check_conv(args); rc != 0) return rc;
    if (args->n_seq == 0) return static_cast<int>(FE_STATUS_OK);
    return on_device(args->device, kCall, [&] { return feb::launch_causal_conv(*args, stream); });
  });
}

size_t fe_selective_scan_workspace(const fe_scan_args* args) {
  constexpr const char* kCall = "fe_selective_scan_workspace";
  std::size_t bytes = 0;
  guarded([&] {
    if (int rc = check_scan(args, kCall, true); rc != 0) return rc;
    return on_device(args->device, kCall, [&] {
      bytes = feb::selective_scan_workspace(*args);
      return 0;
    });
  });
  return bytes;
}

int fe_selective_scan_device(const fe_scan_args* args, void* stream) {
  constexpr const char* kCall = "fe_selective_scan_device";
  return guarded([&] {
    if (int rc = check_scan(args, kCall, false); rc != 0) return rc;
    if (args->n_seq == 0) return static_cast<int>(FE_STATUS_OK);
    const feb::DeviceScope scope(args->device);
    Checks c(kCall);
    c.need(scope.ok(), "the device cannot be used");
    if (int rc = c.done(); rc != 0) return rc;
    const std::size_t need = feb::selective_scan_workspace(*args);
    c.need(need <= args->workspace_bytes, "the workspace is too small");
    c.need(need == 0 || (args->workspace != nullptr && aligned(args->workspace, 16)),
           "the workspace is required, 16-byte aligned");
    if (int rc = c.done(); rc != 0) return rc;
    return launched(feb::launch_selective_scan(*args, stream), kCall);
  });
}

int fe_w4_matvec_device(const fe_w4_args* args, void* stream) {
  constexpr const char* kCall = "fe_w4_matvec_device";
  return guarded([&] {
    fe_w4_args a;
    if (int rc = check_w4(args, a, kCall, true, true, true); rc != 0) return rc;
    if (a.rows == 0) return static_cast<int>(FE_STATUS_OK);
    return on_device(a.device, kCall, [&] { return feb::launch_w4_matvec(a, stream); });
  });
}

int fe_w4_quantize_device(const fe_w4_args* args, void* stream) {
  constexpr const char* kCall = "fe_w4_quantize_device";
  return guarded([&] {
    fe_w4_args a;
    if (int rc = check_w4(args, a, kCall, true, false, false); rc != 0) return rc;
    return on_device(a.device, kCall, [&] { return feb::launch_w4_quantize(a, stream); });
  });
}

int fe_w4_dequantize_device(const fe_w4_args* args, void* stream) {
  constexpr const char* kCall = "fe_w4_dequantize_device";
  return guarded([&] {
    fe_w4_args a;
    if (int rc = check_w4(args, a, kCall, false, true, false); rc != 0) return rc;
    return on_device(a.device, kCall, [&] { return feb::launch_w4_dequantize(a, stream); });
  });
}

int fe_residual_norm_device(const fe_norm_args* args, void* stream) {
  constexpr const char* kCall = "fe_residual_norm_device";
  return guarded([&] {
    if (int rc = check_norm(args); rc != 0) return rc;
    if (args->rows == 0) return static_cast<int>(FE_STATUS_OK);
    return on_device(args->device, kCall, [&] { return feb::launch_residual_norm(*args, stream); });
  });
}

}  // extern "C"
