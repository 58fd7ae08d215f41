// The residual between two blocks and the norms around it in one pass
// (include/flowedge_b200.h, fe_residual_norm_device): a row is read once, held
// in registers through both reductions, and written once.
//
// A row belongs to TPR threads (a power of two from 32 to 512), each with up
// to NV vectors of VEC elements.  Bound by memory: 2 to 5 matrices of the
// row's width per call.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "convert.cuh"
#include "ops.h"

namespace feb {
namespace {

struct NormParams {
  const void *x, *gate;
  const float *post, *weight;
  void *residual, *out;
  long long rows, x_ld, residual_ld, gate_ld, out_ld;
  int dim, tpr;
  float scale, eps, inv_dim;
};

template <typename T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Pack {
  T v[VEC];
};

// Sum over the row's threads, the same in each of them.  Every thread of the
// CTA calls it; `red` holds one float per warp.
__device__ __forceinline__ float row_sum(float v, int tpr, float* red) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if (tpr == 32) return v;
  const int warp = threadIdx.x >> 5, per = tpr >> 5;
  __syncthreads();  // an earlier sum has been read
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  float sum = 0.0f;
  for (int w = warp / per * per, end = w + per; w < end; ++w) sum += red[w];
  return sum;
}

template <typename T, typename R, int VEC, int NV>
__global__ void __launch_bounds__(512, 1) residual_norm_kernel(const NormParams p) {
  __shared__ float red[32];
  const long long row = blockIdx.x * static_cast<long long>(blockDim.x / p.tpr) + threadIdx.x / p.tpr;
  const int lane = threadIdx.x & (p.tpr - 1);
  const bool live = row < p.rows;
  const long long rr = live ? row : 0;
  const T* x = static_cast<const T*>(p.x) + rr * p.x_ld;
  const T* gate = p.gate == nullptr ? nullptr : static_cast<const T*>(p.gate) + rr * p.gate_ld;
  R* res = static_cast<R*>(p.residual) + rr * p.residual_ld;
  T* out = static_cast<T*>(p.out) + rr * p.out_ld;
  // the gate is asked for together with x, but not where that takes the registers of a long row
  constexpr bool kEarly = NV * VEC <= 16;
  float t[NV][VEC], y[NV][VEC], gv[kEarly ? NV : 1][VEC];  // x, then what it adds; the residual
  const int c0 = lane * VEC, step = p.tpr * VEC;
  auto read = [](float(&to)[VEC], const auto* from) {
    using E = std::remove_cv_t<std::remove_pointer_t<decltype(from)>>;
    const Pack<E, VEC> v = *reinterpret_cast<const Pack<E, VEC>*>(from);
#pragma unroll
    for (int e = 0; e < VEC; ++e) to[e] = to_f32(v.v[e]);
  };
  auto write = [](auto* to, const float(&from)[VEC]) {
    using E = std::remove_pointer_t<decltype(to)>;
    Pack<E, VEC> v;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v.v[e] = from_f32<E>(from[e]);
    *reinterpret_cast<Pack<E, VEC>*>(to) = v;
  };
  if constexpr (VEC > 2) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + i * step;
      if (c < p.dim) {
        read(t[i], x + c);
        read(y[i], res + c);
        if (kEarly && gate != nullptr) read(gv[kEarly ? i : 0], gate + c);
      }
    }
  } else {
    // many short requests: all of them first (behind the row's end the last
    // vector again, so that no branch parts them), only then the conversions,
    // each of which waits (16384 x 2047 in bf16: 145 us, as above 370)
    Pack<T, VEC> xr[NV], gr[kEarly ? NV : 1];
    Pack<R, VEC> rr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = min(c0 + i * step, p.dim - VEC);
      xr[i] = *reinterpret_cast<const Pack<T, VEC>*>(x + c);
      rr[i] = *reinterpret_cast<const Pack<R, VEC>*>(res + c);
      if (kEarly && gate != nullptr) gr[kEarly ? i : 0] = *reinterpret_cast<const Pack<T, VEC>*>(gate + c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        t[i][e] = to_f32(xr[i].v[e]);
        y[i][e] = to_f32(rr[i].v[e]);
        if (kEarly && gate != nullptr) gv[kEarly ? i : 0][e] = to_f32(gr[kEarly ? i : 0].v[e]);
      }
  }
  float mul = p.scale;
  if (p.post != nullptr) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (c0 + i * step < p.dim)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss = fmaf(t[i][e], t[i][e], ss);
    mul = p.scale * rsqrtf(fmaf(row_sum(ss, p.tpr, red), p.inv_dim, p.eps));
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * step;
    if (c < p.dim) {
      float pw[VEC];
      if (p.post != nullptr) read(pw, p.post + c);
      if (!kEarly && gate != nullptr) read(gv[0], gate + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float v = t[i][e] * mul;
        if (p.post != nullptr) v *= pw[e];
        if (gate != nullptr) v *= gv[kEarly ? i : 0][e];
        y[i][e] += v;
        ss = fmaf(y[i][e], y[i][e], ss);
      }
      if (live) write(res + c, y[i]);
    }
  }
  const float norm = rsqrtf(fmaf(row_sum(ss, p.tpr, red), p.inv_dim, p.eps));
  if (!live) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * step;
    if (c < p.dim) {
      float w[VEC];
      read(w, p.weight + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] *= y[i][e] * norm;
      write(out + c, w);
    }
  }
}

template <typename T, typename R>
int norm_typed(NormParams p, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);  // 16 bytes of the 16- or 32-bit matrices
  // rows that start on `vec` elements, up to 16 bytes
  const auto starts = [&](int vec) {
    const auto fits = [&](const void* q, long long ld, std::size_t e) {
      const std::size_t bytes = std::min<std::size_t>(16, vec * e);
      return reinterpret_cast<std::uintptr_t>(q) % bytes == 0 && ld * e % bytes == 0;
    };
    return p.dim % vec == 0 && fits(p.x, p.x_ld, sizeof(T)) && fits(p.out, p.out_ld, sizeof(T)) &&
           fits(p.residual, p.residual_ld, sizeof(R)) && (p.gate == nullptr || fits(p.gate, p.gate_ld, sizeof(T))) &&
           fits(p.weight, 0, 4) && fits(p.post, 0, 4);
  };
  const int vec = starts(kVec) ? kVec : starts(2) ? 2 : 1, vecs = p.dim / vec;
  // few rows: as many threads to a row as it has vectors; many rows: about 16
  // elements to a thread, which leaves several rows on an SM at a time (16384 x
  // 2048 gated in bf16: 84.5 us, 8 elements 90.2; 16384 x 2047 with 512 threads
  // to a row, one row on an SM: 540 us)
  const int per = p.rows < 2 * current_sm_count() ? 1 : 16 / vec;
  p.tpr = 32;
  while (p.tpr < 512 && p.tpr * per < vecs) p.tpr *= 2;
  const int threads = std::max(p.tpr, 128), nv = (vecs + p.tpr - 1) / p.tpr;
  const unsigned grid = static_cast<unsigned>((p.rows + threads / p.tpr - 1) / (threads / p.tpr));
  // up to 2, 8, 16 or 32 elements to a thread (at most 16384 on 512 threads)
  const auto launch = [&](auto width) {
    constexpr int V = decltype(width)::value;
    if (nv * V <= 2 || nv == 1)
      residual_norm_kernel<T, R, V, (V < 2 ? 2 : 1)><<<grid, threads, 0, st>>>(p);
    else if (nv * V <= 8)
      residual_norm_kernel<T, R, V, (V < 8 ? 8 / V : 1)><<<grid, threads, 0, st>>>(p);
    else if (nv * V <= 16)
      residual_norm_kernel<T, R, V, 16 / V><<<grid, threads, 0, st>>>(p);
    else
      residual_norm_kernel<T, R, V, 32 / V><<<grid, threads, 0, st>>>(p);
  };
  if (vec == kVec)
    launch(std::integral_constant<int, kVec>{});
  else if (vec == 2)
    launch(std::integral_constant<int, 2>{});
  else
    launch(std::integral_constant<int, 1>{});
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

int launch_residual_norm(const fe_norm_args& a, void* stream) noexcept {
  const NormParams p{a.x, a.gate, a.post_weight, a.weight, a.residual, a.out, static_cast<long long>(a.rows),
                     a.x_ld, a.residual_ld, a.gate_ld, a.out_ld, static_cast<int>(a.dim), 32, a.scale, a.eps, 1.0f / static_cast<float>(a.dim)};
  const auto st = static_cast<cudaStream_t>(stream);
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.residual_dtype == FE_DTYPE_F32 ? norm_typed<T, float>(p, st) : norm_typed<T, T>(p, st);
  });
}

}  // namespace feb
