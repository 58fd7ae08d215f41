// Operators on device buffers (include/flowedge_b200.h, part 3): the launch
// functions behind the C entry points of ops.cc.  No CUDA types appear here;
// `stream` is a cudaStream_t.  The entry points have checked every size,
// pointer and stride before a launch function runs, and have made the buffers'
// device current.  Each returns 0 or a CUDA error code of the launch.
#pragma once

#include <cstddef>
#include <cstdint>
#include <string>

#include "../../include/flowedge_b200.h"

namespace feb {

// Sequences of a call with states in slots: every CTA searches the slots before
// its own for the same one, which is a small part of the call up to some 8192
// and grows with the square (131072 prompts of one row x 256: scan 42 ms, 4
// without slots).
constexpr std::uint64_t kMaxSlotSequences = 1 << 16;

int launch_causal_conv(const fe_conv_args& a, void* stream) noexcept;

// Rows that a tile of prompts has, for tests, with `across` CTAs over the channels.
int causal_conv_chunk(std::size_t rows, std::size_t n_seq, std::size_t across) noexcept;

std::size_t selective_scan_workspace(const fe_scan_args& a) noexcept;
// At least selective_scan_workspace() of any call of up to `rows` rows and
// `n_seq` sequences on the current device.
std::size_t selective_scan_workspace_most(std::size_t rows, std::size_t n_seq, std::size_t d_inner,
                                          std::size_t d_state) noexcept;
int launch_selective_scan(const fe_scan_args& a, void* stream) noexcept;

int launch_w4_quantize(const fe_w4_args& a, void* stream) noexcept;
int launch_w4_dequantize(const fe_w4_args& a, void* stream) noexcept;
int launch_w4_matvec(const fe_w4_args& a, void* stream) noexcept;

int launch_residual_norm(const fe_norm_args& a, void* stream) noexcept;

// Last error of this thread (fe_engine_last_error); defined with the engine.
void set_last_error(std::string message);
void set_last_error_text(const char* message) noexcept;  // a literal
void clear_last_error() noexcept;

// Multiprocessors of the current device (looked up once per device).
int current_sm_count() noexcept;

// Makes `device` current for a scope (-1: leaves the current one).
class DeviceScope {
 public:
  explicit DeviceScope(int device) noexcept;
  ~DeviceScope();
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  [[nodiscard]] bool ok() const noexcept { return ok_; }

 private:
  int before_ = -1;
  bool ok_ = true;
};

const char* cuda_error_text(int code) noexcept;

}  // namespace feb
