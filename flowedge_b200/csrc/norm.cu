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
__global__ void __launch_bounds__(512) residual_norm_kernel(const NormParams p) {
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
  Pack<T, VEC> xv[NV], gv[kEarly ? NV : 1];
  Pack<R, VEC> rv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + i * p.tpr) * VEC;
    if (c < p.dim) {
      xv[i] = *reinterpret_cast<const Pack<T, VEC>*>(x + c);
      rv[i] = *reinterpret_cast<const Pack<R, VEC>*>(res + c);
      if (kEarly && gate != nullptr) gv[kEarly ? i : 0] = *reinterpret_cast<const Pack<T, VEC>*>(gate + c);
    }
  }
  float mul = p.scale;
  if (p.post != nullptr) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((lane + i * p.tpr) * VEC < p.dim)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float v = to_f32(xv[i].v[e]);
          ss = fmaf(v, v, ss);
        }
    mul = p.scale * rsqrtf(fmaf(row_sum(ss, p.tpr, red), p.inv_dim, p.eps));
  }
  float y[NV][VEC];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + i * p.tpr) * VEC;
    if (c < p.dim) {
      Pack<R, VEC> keep;
      Pack<float, VEC> pw;
      if (p.post != nullptr) pw = *reinterpret_cast<const Pack<float, VEC>*>(p.post + c);
      if (!kEarly && gate != nullptr) gv[0] = *reinterpret_cast<const Pack<T, VEC>*>(gate + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float t = to_f32(xv[i].v[e]) * mul;
        if (p.post != nullptr) t *= pw.v[e];
        if (gate != nullptr) t *= to_f32(gv[kEarly ? i : 0].v[e]);
        const float v = to_f32(rv[i].v[e]) + t;
        keep.v[e] = from_f32<R>(v);
        y[i][e] = v;
        ss = fmaf(v, v, ss);
      }
      if (live) *reinterpret_cast<Pack<R, VEC>*>(res + c) = keep;
    }
  }
  const float norm = rsqrtf(fmaf(row_sum(ss, p.tpr, red), p.inv_dim, p.eps));
  if (!live) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + i * p.tpr) * VEC;
    if (c < p.dim) {
      Pack<T, VEC> o;
      const Pack<float, VEC> w = *reinterpret_cast<const Pack<float, VEC>*>(p.weight + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.v[e] = from_f32<T>(y[i][e] * norm * w.v[e]);
      *reinterpret_cast<Pack<T, VEC>*>(out + c) = o;
    }
  }
}

template <typename T, typename R>
int norm_typed(NormParams p, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);  // 16 bytes of the 16- or 32-bit matrices
  const auto fits = [&](const void* q, long long ld, std::size_t e) {
    return reinterpret_cast<std::uintptr_t>(q) % 16 == 0 && ld * static_cast<long long>(e) % 16 == 0;
  };
  const bool wide = p.dim % kVec == 0 && fits(p.x, p.x_ld, sizeof(T)) && fits(p.out, p.out_ld, sizeof(T)) &&
                    fits(p.residual, p.residual_ld, sizeof(R)) && (p.gate == nullptr || fits(p.gate, p.gate_ld, sizeof(T))) && fits(p.weight, 0, 4) && fits(p.post, 0, 4);
  const int vecs = wide ? p.dim / kVec : p.dim;
  // few rows: as many threads to a row as it has vectors; many rows: about two
  // vectors to a thread (16384 x 2048 gated in bf16: 84.5 us, one vector 90.2)
  const int per = p.rows < 2 * current_sm_count() ? 1 : 2;
  p.tpr = 32;
  while (p.tpr < 512 && p.tpr * per < vecs) p.tpr *= 2;
  const int threads = std::max(p.tpr, 128), nv = (vecs + p.tpr - 1) / p.tpr;
  const unsigned grid = static_cast<unsigned>((p.rows + threads / p.tpr - 1) / (threads / p.tpr));
  if (wide) {
    if (nv <= 1)
      residual_norm_kernel<T, R, kVec, 1><<<grid, threads, 0, st>>>(p);
    else if (nv <= 2)
      residual_norm_kernel<T, R, kVec, 2><<<grid, threads, 0, st>>>(p);
    else
      residual_norm_kernel<T, R, kVec, 32 / kVec><<<grid, threads, 0, st>>>(p);  // 32 elements to a thread at most
  } else {
    if (nv <= 2)
      residual_norm_kernel<T, R, 1, 2><<<grid, threads, 0, st>>>(p);
    else
      residual_norm_kernel<T, R, 1, 32><<<grid, threads, 0, st>>>(p);
  }
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
