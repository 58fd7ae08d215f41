// Causal convolution and selective scan over ragged sequences whose state
// lives in slots (kernels_scalar.cc:10-27, 133-169; mamba.cc:317-382 for the
// single-token forms).  A sequence is a run of rows [offsets[s], offsets[s+1]);
// without offsets every row is a sequence of one token.  Its state is slot
// slots[s] (without slots, slot s); a negative slot skips the sequence and
// leaves its rows as they were.
//
// Prompts are cut into tiles of `chunk` rows.  Tile indices are spread so that
// no list of tiles has to be built: sequence s owns the indices from
// offsets[s] / chunk + s on, which leaves room for every tile of it (an empty
// sequence keeps one), and a CTA finds its sequence from its tile index by a
// search over the offsets.  The grid is rows / chunk + n_seq tiles, whatever
// the lengths, so the host never reads them.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "convert.cuh"
#include "ops.h"

namespace feb {
namespace {

struct SeqParams {
  const int* offsets;            // [n_seq + 1], or null: one token per row
  const int* slots;              // [n_seq], or null: slot s
  const unsigned char* fresh;    // [n_seq], or null: no sequence starts from zero
  int* status;                   // FE_SEQ_* bits, or null
  long long rows;
  int n_seq, n_slots;
  bool stateful;                 // a state buffer is read and written
};

struct Seq {
  long long begin;
  int len;
  int slot, bad;
  bool fresh, live;
};

// The sequence that owns tile index `tile` (see the file comment), or -1: a
// 32-way search, every warp on its own.  The indices found are within
// [0, n_seq) whatever the offsets hold.
__device__ int find_sequence(const SeqParams& q, long long tile, int chunk) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = q.n_seq;
  for (;;) {
    const int step = (n + 31) / 32;
    const int k = lane * step;
    const bool below = k < n && static_cast<long long>(q.offsets[lo + k]) / chunk + lo + k <= tile;
    const unsigned m = __ballot_sync(0xffffffffu, below);
    if (m == 0) return -1;
    const int top = 31 - __clz(m);
    lo += top * step;
    n = min(step, n - top * step);
    if (step == 1) return lo;
  }
}

// Bounds, slot and flags of sequence s.  live is false for a sequence that is
// skipped: a negative slot, or a fault (offsets outside the rows, a slot
// outside the pool), whose status bits are in bad.
__device__ __forceinline__ Seq resolve(const SeqParams& q, int s) {
  Seq r;
  r.bad = 0;
  if (q.offsets != nullptr) {
    const int b = q.offsets[s], e = q.offsets[s + 1];
    if (b < 0 || e < b || e > q.rows) r.bad |= FE_SEQ_BAD_OFFSETS;
    r.begin = b;
    r.len = e - b;
  } else {
    r.begin = s;
    r.len = 1;
  }
  r.slot = q.slots != nullptr ? q.slots[s] : s;
  if (q.stateful && r.slot >= q.n_slots) r.bad |= FE_SEQ_BAD_SLOT;
  r.fresh = q.fresh != nullptr && q.fresh[s] != 0;
  r.live = r.bad == 0 && r.slot >= 0;
  return r;
}

// The last test before anything is written: a sequence whose slot an earlier
// one of the call has is skipped (kMaxSlotSequences bounds the search).  Every thread of the CTA calls it; `report`
// writes the sequence's faults to the status.
__device__ __forceinline__ bool writes(const SeqParams& q, int s, Seq& r, bool report) {
  if (q.stateful && q.slots != nullptr && r.slot >= 0) {
    int dup = 0;
    for (int i = threadIdx.x; i < s; i += blockDim.x) dup |= q.slots[i] == r.slot;
    if (__syncthreads_or(dup)) r.bad |= FE_SEQ_DUPLICATE_SLOT;
  }
  if (report && r.bad != 0 && q.status != nullptr && threadIdx.x == 0) atomicOr(q.status, r.bad);
  return r.bad == 0 && r.slot >= 0;
}

// The first CTA of a grid also reports offsets that no tile can be found by:
// a decreasing pair hides sequences from the search.
__device__ void report_offsets(const SeqParams& q) {
  if (q.status == nullptr || blockIdx.x != 0 || blockIdx.y != 0) return;
  int bad = 0;
  for (int i = threadIdx.x; i < q.n_seq; i += blockDim.x) {
    const int b = q.offsets[i], e = q.offsets[i + 1];
    bad |= b < 0 || e < b || e > q.rows;
  }
  if (bad) atomicOr(q.status, FE_SEQ_BAD_OFFSETS);
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// SiLU of a pair: x / (1 + 2^(-x log2 e)) by the hardware's power and
// reciprocal (relative error a few steps of fp32, and one more for every unit
// of |x|; -0 below -88, the limit)
__device__ __forceinline__ float2 silu2(float2 x) {
  const float2 t = __fmul2_rn(x, splat(-1.4426950408889634f));
  const float2 d = __fadd2_rn(make_float2(ex2_approx(t.x), ex2_approx(t.y)), splat(1.0f));
  return __fmul2_rn(x, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
}
__device__ __forceinline__ float silu1(float x) {
  return x * rcp_approx(1.0f + ex2_approx(x * -1.4426950408889634f));
}

template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T v[V];
};

// --- causal convolution -------------------------------------------------------

struct ConvParams {
  SeqParams q;
  const void* x;
  const float* w;  // [di][dc]
  const float* b;  // [di]
  void* u;
  float* window;  // [slot][di][dc], the last dc inputs, newest last
  long long x_ld, u_ld, slot_stride;
  int di, dc, chunk;
};

// One thread per (token, channel): shift the window, append x, dot, SiLU.
// Bound by the window's bytes (512 x 2048 in bf16: 8.4 us, 0.70 of the measured
// copy rate).  FOUR: four taps and windows on 16-byte boundaries, one load and
// one store each.
template <typename T, bool FOUR>
__global__ void __launch_bounds__(128) conv_token_kernel(const ConvParams p) {
  const int s = blockIdx.x;
  Seq q = resolve(p.q, s);
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  const bool on = c < p.di && q.live;
  float* win = p.window == nullptr || !on ? nullptr : p.window + q.slot * p.slot_stride + static_cast<long long>(c) * p.dc;
  const bool held = win != nullptr && !q.fresh;
  const int dc = FOUR ? 4 : p.dc;
  float v[8], xv = 0.0f;  // v[j]: tap j's input, the newest (x) last
  if constexpr (FOUR) {
    const float4 o = held ? *reinterpret_cast<const float4*>(win) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    v[0] = o.y;
    v[1] = o.z;
    v[2] = o.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = held && j + 1 < dc ? win[j + 1] : 0.0f;
  }
  if (on) xv = to_f32(static_cast<const T*>(p.x)[s * p.x_ld + c]);
  if (!writes(p.q, s, q, blockIdx.y == 0) || !on) return;
  const float* w = p.w + static_cast<long long>(c) * dc;
  float acc = p.b[c];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= dc) break;
    if (j == dc - 1) v[j] = xv;
    acc = fmaf(w[j], v[j], acc);
  }
  static_cast<T*>(p.u)[s * p.u_ld + c] = from_f32<T>(silu1(acc));
  if (win == nullptr) return;
  if constexpr (FOUR) {
    *reinterpret_cast<float4*>(win) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < dc) win[j] = v[j];
  }
}

// One thread walks V channels of a tile's rows, two and two (V 1: a pair with
// an idle half), with their last DC (d_conv) inputs in registers, kAhead rows
// requested before their arithmetic.  Each tap count is a kernel of its own: a
// surplus tap of weight zero would make NaN of an infinite input.  The first tile of a sequence reads the old window and
// writes the new one from the sequence's last rows, so no other tile touches
// it.  Bound by x and u, read and written once (a tile reads DC - 1 rows
// before its own again, from L2), and in front of that by the chain of a tile:
// search, slot, rows, stores (96 prompts, 12289 x 1024 in bf16: 21 us, 8 of
// them the bytes).
template <typename T, int DC, int V>
__global__ void __launch_bounds__(128, 5) conv_prompt_kernel(const ConvParams p) {
  constexpr int kPairs = (V + 1) / 2, kAhead = 8;
  constexpr int kLines = (32 * V * static_cast<int>(sizeof(T)) + 127) / 128;  // of a row, for a warp
  const int lane = threadIdx.x & 31;
  report_offsets(p.q);
  const int s = find_sequence(p.q, blockIdx.x, p.chunk);
  if (s < 0) return;
  Seq q = resolve(p.q, s);
  const long long k = blockIdx.x - (q.begin / p.chunk + s);
  if (!q.live && q.bad == 0) return;                         // a padded sequence
  if (q.bad == 0 && k > 0 && k * p.chunk >= q.len) return;  // no such tile
  const int t0 = static_cast<int>(k * p.chunk);
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  const bool on = c < p.di && q.live;
  const T* x = static_cast<const T*>(p.x) + q.begin * p.x_ld + c;
  float* win = p.window == nullptr ? nullptr : p.window + q.slot * p.slot_stride + static_cast<long long>(c) * DC;
  const int t1 = on ? min(t0 + p.chunk, q.len) : t0;
  using Row = Vec<T, V>;
  auto pair = [](const Row& r, int e) {
    return make_float2(to_f32(r.v[2 * e]), 2 * e + 1 < V ? to_f32(r.v[V > 1 ? 2 * e + 1 : 0]) : 0.0f);
  };
  Row ahead[kAhead];
  const T* next = x + t0 * p.x_ld;
  auto request = [&](int t) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (t + i < t1) ahead[i] = *reinterpret_cast<const Row*>(next + i * p.x_ld);
    next += kAhead * p.x_ld;
  };
  request(t0);
  // the rows after these into L2: a lane one line of one row
  for (int e = lane; e < (t1 - t0 - kAhead) * kLines; e += 32) {
    const int at = c + (e % kLines * (128 / static_cast<int>(sizeof(T))) - lane * V);
    if (at < p.di) prefetch_l2(static_cast<const T*>(p.x) + (q.begin + t0 + kAhead + e / kLines) * p.x_ld + at);
  }
  float2 wk[DC][kPairs], in[DC][kPairs], bias[kPairs];
  float w[DC][2 * kPairs];
  if (on) {
#pragma unroll
    for (int e = 0; e < 2 * kPairs; ++e) {
      const int ce = e < V ? c + e : c;
      const float* src = p.w + static_cast<long long>(ce) * DC;
      (e & 1 ? bias[e / 2].y : bias[e / 2].x) = p.b[ce];
      if constexpr (V > 1 && DC == 4) {  // on 16 bytes (conv_prompts)
        const float4 w4 = *reinterpret_cast<const float4*>(src);
        w[0][e] = w4.x;
        w[1][e] = w4.y;
        w[2][e] = w4.z;
        w[3][e] = w4.w;
      } else {
#pragma unroll
        for (int j = 0; j < DC; ++j) w[j][e] = src[j];
      }
    }
  }
  Row halo[DC];
#pragma unroll
  for (int j = 1; j < DC; ++j)
    if (on && t0 >= DC) halo[j] = *reinterpret_cast<const Row*>(x + (t0 - DC + j) * p.x_ld);
  // every request is on its way: only now the test that waits
  if (!writes(p.q, s, q, blockIdx.y == 0) || !on) return;
#pragma unroll
  for (int j = 0; j < DC; ++j) {
    // place j holds the input t0 - DC + j before row t0; place 0 is shifted out unused
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      wk[j][e] = make_float2(w[j][2 * e], w[j][2 * e + 1]);
      in[j][e] = j > 0 && t0 >= DC ? pair(halo[j], e) : splat(0.0f);
    }
    // (a tile's first row is a multiple of the chunk, so that t0 is 0 or at least DC)
    if (j > 0 && t0 == 0 && win != nullptr && !q.fresh) {
#pragma unroll
      for (int e = 0; e < V; ++e) (e & 1 ? in[j][e / 2].y : in[j][e / 2].x) = win[e * DC + j];
    }
  }
  if (k == 0 && win != nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      for (int j = 0; j < DC; ++j) {
        const int t = q.len - DC + j;
        win[e * DC + j] = t >= 0 ? to_f32(x[t * p.x_ld + e]) : (q.fresh ? 0.0f : win[e * DC + DC + t]);
      }
  }
  T* u = static_cast<T*>(p.u) + (q.begin + t0) * p.u_ld + c;
  for (int t = t0; t < t1; t += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (t + i >= t1) break;
      Row out;
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
#pragma unroll
        for (int j = 0; j + 1 < DC; ++j) in[j][e] = in[j + 1][e];
        in[DC - 1][e] = pair(ahead[i], e);
        float2 acc = bias[e];
#pragma unroll
        for (int j = 0; j < DC; ++j) acc = __ffma2_rn(wk[j][e], in[j][e], acc);
        acc = silu2(acc);
        out.v[2 * e] = from_f32<T>(acc.x);
        if (2 * e + 1 < V) out.v[V > 1 ? 2 * e + 1 : 0] = from_f32<T>(acc.y);
      }
      *reinterpret_cast<Row*>(u + i * p.u_ld) = out;
    }
    u += kAhead * p.u_ld;
    request(t + kAhead);
  }
}

// Rows of a conv tile: as few as let every tile be resident at once (five CTAs
// to an SM; half of the sequences' last tiles are extra), from 8 to 64.
// `across` CTAs go over the channels.  Measured at 96 prompts of 12289 rows x
// 1024: 16 rows 25.0 us, 24 23.8, 40 (this rule) 21.1, 64 25.8
int conv_chunk(long long rows, long long n_seq, long long across) {
  const long long resident = std::max(1LL, 5LL * current_sm_count() / across - n_seq / 2);
  return static_cast<int>(std::clamp((rows / resident + 7) / 8 * 8, 8LL, 64LL));
}

template <typename T, int DC>
int conv_prompts(ConvParams p, cudaStream_t st) {
  // 16 bytes of a row to a thread where its rows allow it (at most four
  // channels, and two of more than four taps, which take the registers)
  constexpr int kVec = DC > 4 ? 2 : 4;
  const auto fits = [&](const void* q, long long ld) {
    return reinterpret_cast<std::uintptr_t>(q) % (kVec * sizeof(T)) == 0 && ld % kVec == 0;
  };
  const bool wide = p.di % kVec == 0 && fits(p.x, p.x_ld) && fits(p.u, p.u_ld) &&
                    reinterpret_cast<std::uintptr_t>(p.w) % 16 == 0;
  const int threads = wide ? p.di / kVec : p.di;  // for a row
  const unsigned block = static_cast<unsigned>(std::min(128, (threads + 31) / 32 * 32));
  const long long across = (threads + block - 1) / block;
  p.chunk = conv_chunk(p.q.rows, p.q.n_seq, across);
  const dim3 grid(static_cast<unsigned>(p.q.rows / p.chunk + p.q.n_seq), static_cast<unsigned>(across));
  if (wide)
    conv_prompt_kernel<T, DC, kVec><<<grid, block, 0, st>>>(p);
  else
    conv_prompt_kernel<T, DC, 1><<<grid, block, 0, st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int conv_typed(const ConvParams& p, cudaStream_t st) {
  if (p.q.offsets != nullptr) {
    switch (p.dc) {
      case 1: return conv_prompts<T, 1>(p, st);
      case 2: return conv_prompts<T, 2>(p, st);
      case 3: return conv_prompts<T, 3>(p, st);
      case 4: return conv_prompts<T, 4>(p, st);
      case 5: return conv_prompts<T, 5>(p, st);
      case 6: return conv_prompts<T, 6>(p, st);
      case 7: return conv_prompts<T, 7>(p, st);
      default: return conv_prompts<T, 8>(p, st);
    }
  }
  const dim3 grid(static_cast<unsigned>(p.q.n_seq), static_cast<unsigned>((p.di + 127) / 128));
  if (p.dc == 4 && reinterpret_cast<std::uintptr_t>(p.window) % 16 == 0 && p.slot_stride % 4 == 0)
    conv_token_kernel<T, true><<<grid, 128, 0, st>>>(p);
  else
    conv_token_kernel<T, false><<<grid, 128, 0, st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

// --- selective scan -----------------------------------------------------------

struct ScanParams {
  SeqParams q;
  const void *u, *proj, *z;
  const float *a, *d, *dt_w, *dt_b;  // a [ds][di], dt_w [dr][di]
  void* y;
  float* state;  // [slot][ds][di]
  float* steps;  // [rows][di], dt of every row (prompts)
  float* ws;     // [tile][1 + ds][di]: sum of dt, then the tile's state (its end from zero; later its start)
  long long u_ld, proj_ld, z_ld, y_ld, slot_stride;
  int di, ds, dr, chunk;
};

// softplus of a pair to a few ulp of the result: e = exp(-|x|) with the
// rounding error of |x| log2(e) carried into the exponential, log(1 + e) =
// 2 atanh(e / (2 + e)) by its series (the argument s is at most 1/3; the first
// term left out is below 2^-26 of the sum).  log(1 + e) as it stands would
// lose dt's relative precision for the small steps that the scan lives on.
__device__ __forceinline__ float2 softplus_rel2(float2 x) {
  constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.9259629911e-8f;
  const float2 ax = make_float2(min_nan(fabsf(x.x), 120.0f), min_nan(fabsf(x.y), 120.0f));
  const float2 hi = __fmul2_rn(ax, splat(-kLog2e));
  const float2 off = __ffma2_rn(ax, splat(kLog2eLow), __ffma2_rn(ax, splat(kLog2e), hi));  // the exponent is hi - off
  const float2 e2 = make_float2(ex2_approx(hi.x), ex2_approx(hi.y));
  const float2 e = __ffma2_rn(__fmul2_rn(e2, splat(-0.69314718f)), off, e2);
  const float2 den = __fadd2_rn(e, splat(2.0f));
  const float2 s = __fmul2_rn(e, make_float2(rcp_approx(den.x), rcp_approx(den.y))), s2 = __fmul2_rn(s, s);
  float2 r = __ffma2_rn(s2, splat(1.0f / 15.0f), splat(1.0f / 13.0f));
  r = __ffma2_rn(r, s2, splat(1.0f / 11.0f));
  r = __ffma2_rn(r, s2, splat(1.0f / 9.0f));
  r = __ffma2_rn(r, s2, splat(1.0f / 7.0f));
  r = __ffma2_rn(r, s2, splat(1.0f / 5.0f));
  r = __ffma2_rn(r, s2, splat(1.0f / 3.0f));
  r = __ffma2_rn(__fmul2_rn(r, s2), s, s);
  return __ffma2_rn(r, splat(2.0f), make_float2(max_nan(x.x, 0.0f), max_nan(x.y, 0.0f)));
}
__device__ __forceinline__ float softplus_rel(float x) { return softplus_rel2(splat(x)).x; }

// 2^x for a pair of x <= 0 on the FMA pipe.  x = k + r with k whole and r in
// [-1/2, 1/2] (k by adding and taking away 1.5 * 2^23), 2^r = 1 + r q(r) with
// q the degree-5 Chebyshev interpolant of (2^r - 1) / r, times 2^k, whose bits
// are k + 127 in the exponent field (k = -127, which x below it takes too, is
// 0).  A NaN stays one through the sum.  The leading 1 is exact and the error
// is that of the last addition (at most 7.2e-8, mean 3e-10), so that a decay
// near 1 keeps its distance from 1 over thousands of steps.
__device__ __forceinline__ float2 exp2_neg2(float2 x) {
  constexpr float kRound = 12582912.0f;
  x.x = max_nan(x.x, -127.0f);
  x.y = max_nan(x.y, -127.0f);
  const float2 t = __fadd2_rn(x, make_float2(kRound, kRound));
  const float2 k = __fadd2_rn(t, make_float2(-kRound, -kRound));
  const float2 r = __ffma2_rn(k, make_float2(-1.0f, -1.0f), x);
  float2 p = __ffma2_rn(make_float2(1.5453163e-4f, 1.5453163e-4f), r, make_float2(1.3390863e-3f, 1.3390863e-3f));
  p = __ffma2_rn(p, r, make_float2(9.6180830e-3f, 9.6180830e-3f));
  p = __ffma2_rn(p, r, make_float2(5.5503570e-2f, 5.5503570e-2f));
  p = __ffma2_rn(p, r, make_float2(2.4022651e-1f, 2.4022651e-1f));
  p = __ffma2_rn(p, r, make_float2(6.9314718e-1f, 6.9314718e-1f));
  p = __ffma2_rn(p, r, make_float2(1.0f, 1.0f));
  return __fmul2_rn(p, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3F800000),
                                   __int_as_float((__float_as_int(t.y) << 23) + 0x3F800000)));
}

// Lets a kernel have `bytes` of shared memory, at most 200 KB (always the same
// limit, so that calls on several threads do not change each other's).
template <typename K>
cudaError_t allow_smem(K kernel, int bytes) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  return cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize,
                              200 * 1024);
}

// --- the steps dt of a prompt call's rows --------------------------------------
//
// dt[t][c] = softplus(dt_b[c] + sum_r dt_in[t][r] dt_w[r][c]) for every row, into
// the workspace: a matrix product once per call, on the warp's matrix
// instruction, instead of dt_rank products per row and channel on the FMA pipe
// in each of the scan's passes.  The products are those of fp32: every operand
// is a sum of bf16 terms (dt_w of three; dt_in of one, two or three as it is
// bf16, fp16 or fp32: 8, 11 or 24 bits), and all pairs of terms are multiplied
// whose product is above 2^-25 of the whole, smallest first.  Terms of an
// infinity or of a value that bf16 rounds to one do not add up to it (infinity
// times terms of two signs, or of zero, is NaN): a sum that is not finite is
// made again from the operands.  16384 x 2048, dt rank 64, bf16: 74 us, 21 of
// them the bytes of dt.
template <typename T>
constexpr int kDtTerms = std::is_same_v<T, float> ? 3 : std::is_same_v<T, __half> ? 2 : 1;

// the next bf16 term of a pair, packed; the rest stays in a and b
__device__ __forceinline__ uint32_t take_bf16(float& a, float& b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const float2 f = __bfloat1622float2(h);
  a = isinf(f.x) ? 0.0f : a - f.x;
  b = isinf(f.y) ? 0.0f : b - f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A row's steps from the operands themselves, for sums that the terms cannot
// give: columns c, c + 1, c + 8, c + 9 .. below `end`, those of a fragment's lane.
template <typename T>
__device__ __noinline__ void step_row(const T* row, const float* dt_w, const float* dt_b, float* to, int dr, int di, int c,
                                      int end) {
  for (; c < end; c += c & 1 ? 7 : 1) {
    float sum = dt_b[c];
    const float* w = dt_w + c;
    for (int r = 0; r < dr; ++r, w += di) sum = fmaf(to_f32(row[r]), *w, sum);
    to[c] = softplus_rel(sum);
  }
}

// A warp takes 16 rows x COLS channels at a time and walks the rows; dt_in goes from memory into fragments (the next 16 columns asked for before
// the products), the weights' terms sit in shared memory for the whole kernel:
// [term][16 of dt_rank][t][channel][2], t and the pair being the fragment's, a
// lane's two words side by side and the lanes of a half warp on different
// banks.  (Two row tiles a warp, to read the weights' fragments half as often,
// take the registers of a third CTA: 425 against 422 us for the whole scan of
// 16384 rows x 2048 in bf16, 188 against 186 for 96 prompts x 1024 in fp32.)
constexpr int kDtWarps = 8;
constexpr int dt_stride(int cols) { return 2 * cols + 8; }
constexpr int kDtRows = 16, kDtCtas = 3;  // rows of a warp, CTAs resident on an SM

template <typename T, int COLS>
__global__ void __launch_bounds__(kDtWarps * 32, kDtCtas) scan_steps_kernel(const ScanParams p) {
  constexpr int kTerms = kDtTerms<T>, kStride = dt_stride(COLS);
  extern __shared__ __align__(16) uint32_t sb[];
  __shared__ float sbias[COLS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int c0 = blockIdx.y * COLS, nk = (p.dr + 15) / 16;
  const bool pairs = p.di % 2 == 0;
  for (int i = threadIdx.x; i < nk * 8 * COLS; i += kDtWarps * 32) {
    const int n = i % COLS, k2 = i / COLS, r = 2 * k2, c = c0 + n;
    float a = c < p.di && r < p.dr ? p.dt_w[static_cast<long long>(r) * p.di + c] : 0.0f;
    float b = c < p.di && r + 1 < p.dr ? p.dt_w[static_cast<long long>(r + 1) * p.di + c] : 0.0f;
#pragma unroll
    for (int m = 0; m < 3; ++m)
      sb[((m * nk + k2 / 8) * 4 + k2 % 4) * kStride + 2 * n + k2 % 8 / 4] = take_bf16(a, b);
  }
  for (int n = threadIdx.x; n < COLS; n += kDtWarps * 32) sbias[n] = c0 + n < p.di ? p.dt_b[c0 + n] : 0.0f;
  __syncthreads();
  griddep_launch();
  // two neighbours of a row in one load, where rows start on such pairs
  const bool even = p.proj_ld % 2 == 0 && reinterpret_cast<std::uintptr_t>(p.proj) % (2 * sizeof(T)) == 0;
  const long long step = static_cast<long long>(gridDim.x) * kDtWarps * kDtRows;
  for (long long row0 = (static_cast<long long>(blockIdx.x) * kDtWarps + warp) * kDtRows; row0 < p.q.rows; row0 += step) {
    float acc[COLS / 8][4] = {};
    const T* base = static_cast<const T*>(p.proj) + (row0 + g) * p.proj_ld + 2 * t;
    const int have = static_cast<int>(min(static_cast<long long>(kDtRows), p.q.rows - row0)) - g;  // rows g + 8 i, 8 i < have
    Vec<T, 2> raw[4];  // fragment words: (g, 2t), (g + 8, 2t), (g, 2t + 8), (g + 8, 2t + 8)
    auto request = [&](int k) {
      const bool whole = even && 16 * (k + 1) <= p.dr;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int row = 8 * (w & 1), r = 16 * k + 4 * (w & 2);
        const T* src = base + row * p.proj_ld + r;
        raw[w] = Vec<T, 2>{{from_f32<T>(0.0f), from_f32<T>(0.0f)}};
        if (whole) {
          if (row < have) raw[w] = *reinterpret_cast<const Vec<T, 2>*>(src);
        } else {
          const int more = row < have ? p.dr - r - 2 * t : 0;  // columns of dt_in from here on
          if (more > 0) raw[w].v[0] = src[0];
          if (more > 1) raw[w].v[1] = src[1];
        }
      }
    };
    request(0);
    for (int k = 0; k < nk; ++k) {
      uint32_t fa[kTerms][4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float a = to_f32(raw[w].v[0]), b = to_f32(raw[w].v[1]);
#pragma unroll
        for (int q = 0; q < kTerms; ++q) fa[q][w] = take_bf16(a, b);
      }
      if (k + 1 < nk) request(k + 1);
      // several tiles at a time, so that the products in flight have sums of their own
      constexpr int kTogether = COLS / 8 < 8 ? COLS / 8 : 8;
#pragma unroll
      for (int n0 = 0; n0 < COLS / 8; n0 += kTogether) {
#pragma unroll
        for (int m = 2; m >= 0; --m) {
          uint2 b[kTogether];
#pragma unroll
          for (int n = 0; n < kTogether; ++n)
            b[n] = *reinterpret_cast<const uint2*>(sb + ((m * nk + k) * 4 + t) * kStride + 2 * (8 * (n0 + n) + g));
#pragma unroll
          for (int q = kTerms - 1; q >= 0; --q)
            if (q + m <= 2)
#pragma unroll
              for (int n = 0; n < kTogether; ++n) mma_bf16(acc[n0 + n], fa[q], b[n].x, b[n].y);
        }
      }
    }
    float* to = p.steps + (row0 + g) * p.di + c0 + 2 * t;
    const long long below = 8LL * p.di;
    float2 finite[2] = {};  // of both rows, zero times every sum: NaN where one is not
#pragma unroll
    for (int n = 0; n < COLS / 8; ++n, to += 8) {
      const int c = c0 + 8 * n + 2 * t;
      const bool c_lo = c < p.di, c_hi = c + 1 < p.di;
      const float2 bias = make_float2(sbias[8 * n + 2 * t], sbias[8 * n + 2 * t + 1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // (the bias joins here: the instruction's sums drop bits below the
        // largest term's last, and the bias is the largest)
        const float2 sum = make_float2(acc[n][2 * i] + bias.x, acc[n][2 * i + 1] + bias.y);
        finite[i] = __ffma2_rn(sum, splat(0.0f), finite[i]);
        const float2 v = softplus_rel2(sum);
        float* at = to + i * below;
        if (pairs) {
          if (8 * i < have && c_hi) *reinterpret_cast<float2*>(at) = v;
        } else {
          if (8 * i < have && c_lo) at[0] = v.x;
          if (8 * i < have && c_hi) at[1] = v.y;
        }
      }
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      if ((i == 0 ? finite[0].x + finite[0].y : finite[1].x + finite[1].y) == 0.0f || 8 * i >= have) continue;
      const long long row = row0 + g + 8 * i;
      step_row(static_cast<const T*>(p.proj) + row * p.proj_ld, p.dt_w, p.dt_b, p.steps + row * p.di, p.dr, p.di, c0 + 2 * t,
               min(p.di, c0 + COLS));
    }
  }
}

// Channels to a CTA: 64 (sums and fragments then leave room for three CTAs to
// an SM), or 32 where the weights' terms of 64 do not fit the shared memory
// (dt_rank above 256).
template <typename T, int COLS>
int steps_launch_cols(const ScanParams& p, cudaStream_t st) {
  const int smem = 4 * 3 * ((p.dr + 15) / 16) * 4 * dt_stride(COLS);
  if (const cudaError_t rc = allow_smem(scan_steps_kernel<T, COLS>, smem); rc != cudaSuccess) return static_cast<int>(rc);
  const long long tiles = (p.q.rows + kDtRows - 1) / kDtRows, cols = (p.di + COLS - 1) / COLS;
  const long long ctas =
      std::max(1LL, std::min((tiles + kDtWarps - 1) / kDtWarps, static_cast<long long>(kDtCtas) * current_sm_count() / cols));
  scan_steps_kernel<T, COLS><<<dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(cols)), kDtWarps * 32,
                               static_cast<std::size_t>(smem), st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int steps_launch(const ScanParams& p, cudaStream_t st) {
  if (p.q.rows == 0) return 0;
  return p.dr <= 256 ? steps_launch_cols<T, 64>(p, st) : steps_launch_cols<T, 32>(p, st);
}

// --- the scan of single tokens -----------------------------------------------------

// One token for a sequence.  DS / 8 threads of a warp share V neighbouring
// channels (a pair; V 1: the second is idle), eight of their states each: a
// thread requests its states first, which are the kernel's bytes; the rest of
// its work comes while they do.  Arithmetic on the two channels at once
// (FFMA2).  GIVEN: dt is in the workspace (many sequences: dt_w would be read
// again for every one of them), else the CTA makes it.  PADDED: fewer states
// than DS; those that do not exist stay out of y (an infinite u or dt makes NaN
// of them).  Bound by the states'
// bytes and their latency: 475 of 512 x 2048, 16 states, bf16: 38 us with the
// dt before it, 0.53 of the measured copy rate.
constexpr int kTokenStates = 8;  // of a thread

template <typename T, int DS, int V, bool GIVEN, bool PADDED>
__global__ void __launch_bounds__(128) scan_token_kernel(const ScanParams p) {
  constexpr int kSplit = DS / kTokenStates, kPairs = 32 / kSplit;  // threads of a channel pair, pairs of a warp
  extern __shared__ float sdt[];                  // dt_in [dr], not GIVEN
  __shared__ __align__(16) float sbc[2 * DS];     // [B (DS) | C (DS)], zero behind ds
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / kPairs;
  const int s = blockIdx.x, c = ((blockIdx.y * 4 + warp) * kPairs + lane % kPairs) * V;
  const int ds = p.ds, dr = p.dr, n0 = sub * kTokenStates;
  const bool on = c < p.di;
  const int cc = on ? c : 0;
  auto load2 = [](const float* at) {
    if constexpr (V == 2)
      return *reinterpret_cast<const float2*>(at);
    else
      return make_float2(*at, 0.0f);
  };
  auto read2 = [](const void* base, long long at) {
    const T* q = static_cast<const T*>(base) + at;
    if constexpr (V == 2) {
      const Vec<T, 2> v = *reinterpret_cast<const Vec<T, 2>*>(q);
      return make_float2(to_f32(v.v[0]), to_f32(v.v[1]));
    } else {
      return make_float2(to_f32(*q), 0.0f);
    }
  };
  Seq q = resolve(p.q, s);
  float* const st = q.live && p.state != nullptr ? p.state + q.slot * p.slot_stride + static_cast<long long>(n0) * p.di + cc
                                                 : nullptr;
  const bool held = st != nullptr && !q.fresh;
  float2 h[kTokenStates];
  {
    const float* from = st;
#pragma unroll
    for (int n = 0; n < kTokenStates; ++n, from += p.di) h[n] = held && n0 + n < ds ? load2(from) : splat(0.0f);
  }
  const float2 uv = read2(p.u, s * p.u_ld + cc);
  const float2 zv = p.z != nullptr && sub == 0 ? read2(p.z, s * p.z_ld + cc) : splat(0.0f);
  const T* row = static_cast<const T*>(p.proj) + s * p.proj_ld;
  if (!GIVEN)
    for (int e = threadIdx.x; e < dr; e += 128) sdt[e] = to_f32(row[e]);
  for (int e = threadIdx.x; e < 2 * DS; e += 128) {
    const int n = e % DS;
    sbc[e] = n < ds ? to_f32(row[dr + (e < DS ? n : ds + n)]) : 0.0f;
  }
  float2 an[kTokenStates];
  {
    const float* a = p.a + static_cast<long long>(n0) * p.di + cc;
#pragma unroll
    for (int n = 0; n < kTokenStates; ++n, a += p.di)
      an[n] = n0 + n < ds ? __fmul2_rn(load2(a), splat(1.4426950408889634f)) : splat(0.0f);
  }
  const float2 dk = load2(p.d + cc);
  const bool runs = writes(p.q, s, q, blockIdx.y == 0);
  if constexpr (GIVEN) griddep_wait();
  __syncthreads();  // dt_in, B and C
  auto across = [](float2 v) {  // summed over the channels' threads, the same in each
#pragma unroll
    for (int off = kPairs; off < 32; off *= 2) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, off);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, off);
    }
    return v;
  };
  float2 dt;
  if constexpr (GIVEN) {
    dt = load2(p.steps + static_cast<long long>(s) * p.di + cc);
  } else {
    // every kSplit-th term here, the rest in the channels' other threads
    float2 acc = sub == 0 ? load2(p.dt_b + cc) : splat(0.0f);
    const float* w = p.dt_w + static_cast<long long>(sub) * p.di + cc;
#pragma unroll 8
    for (int r = sub; r < dr; r += kSplit, w += static_cast<long long>(kSplit) * p.di)
      acc = __ffma2_rn(load2(w), splat(sdt[r]), acc);
    dt = softplus_rel2(across(acc));
  }
  const float2 dtu = __fmul2_rn(dt, uv);
  float2 y = sub == 0 ? __fmul2_rn(dk, uv) : splat(0.0f);
#pragma unroll
  for (int n = 0; n < kTokenStates; n += 4) {
    const float4 bq = *reinterpret_cast<const float4*>(sbc + n0 + n);
    const float4 cq = *reinterpret_cast<const float4*>(sbc + DS + n0 + n);
    const float bn[4] = {bq.x, bq.y, bq.z, bq.w}, cn[4] = {cq.x, cq.y, cq.z, cq.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 e = __fmul2_rn(dt, an[n + i]);
      h[n + i] = __ffma2_rn(make_float2(ex2_approx(e.x), ex2_approx(e.y)), h[n + i], __fmul2_rn(dtu, splat(bn[i])));
      if (!PADDED || n0 + n + i < ds) y = __ffma2_rn(h[n + i], splat(cn[i]), y);
    }
  }
  y = across(y);
  if (!runs || !on) return;
  if (st != nullptr) {
    float* to = st;
#pragma unroll
    for (int n = 0; n < kTokenStates; ++n, to += p.di)
      if (n0 + n < ds) {
        if constexpr (V == 2)
          *reinterpret_cast<float2*>(to) = h[n];
        else
          *to = h[n].x;
      }
  }
  if (sub != 0) return;  // one of the channels' threads writes the row
  if (p.z != nullptr) y = __fmul2_rn(y, silu2(zv));
  T* out = static_cast<T*>(p.y) + s * p.y_ld + c;
  if constexpr (V == 2)
    *reinterpret_cast<Vec<T, 2>*>(out) = Vec<T, 2>{{from_f32<T>(y.x), from_f32<T>(y.y)}};
  else
    *out = from_f32<T>(y.x);
}

// --- the scan of prompts ----------------------------------------------------------

constexpr int kScanWarps = 4;  // warps of a CTA, 32 channels each
constexpr int kStage = 16;     // rows whose B and C are in shared memory at a time
constexpr int kTok = 4;        // rows whose dt, u and z are requested ahead
// State pairs whose exponentials go to the FMA pipe, the first ones (where a
// grows with n, as it does at the start of training, the slowest states, which
// gain from its exactness near 1).  A row's exponentials take the MUFU unit 8
// cycles each, the FMA pipe 20 a pair beside 6 (summary) or 8 for the pair's
// products, so few pairs gain.  Measured at 16384 rows x 2048 channels and at 96
// prompts of 12289 x 1024, DS 16: no pair 421.6 and 183.8 us, one of eight
// 417.7 and 184.9; at 64 prompts of 8192 x 1024, DS 32: none 216.8, one of
// sixteen 218.9, two 213.4.
template <int DS>
constexpr int kPolyPairs = DS / 16;

// One thread per channel, the states in registers, over the rows of one tile.
// SUMMARY: the tile's sum of dt and its state from a zero start, for the tiles
// whose sequence goes on (the recurrence over a tile is h -> exp(A sum dt) h +
// end, so the sum of dt stands for the product of decays).  Otherwise: from
// the state that enters the tile, with y.
//
// Bound by arithmetic: per row and channel DS exponentials, which MUFU and FMA
// pipe share, and 4 DS products; dt, u, z and y pass through once.  The rows'
// B and C sit in shared memory (every channel reads them), the next kStage
// rows' are requested before the arithmetic; dt, u and z are requested kTok
// rows ahead.  All arithmetic on pairs (FFMA2): states two and two.  16384 rows
// x 2048, 16 states, bf16: the main pass adds 191 us to the call, the summaries
// 140.  Four CTAs on an SM: three 466 us for the whole scan, four 420, five 469
// (with two state pairs on the FMA pipe in the summaries).  DS is d_state
// rounded up to a multiple of four; PADDED: the last states do not exist and
// stay out of y, as for single tokens.
template <typename T, int DS, bool SUMMARY, bool PADDED>
__global__ void __launch_bounds__(kScanWarps * 32, DS <= 16 ? 4 : 3) scan_prompt_kernel(const ScanParams p) {
  __shared__ __align__(16) float sbc[2][kStage][2 * DS];
  if (!SUMMARY) report_offsets(p.q);
  // (the call's own inputs may be read before the kernel it waits for is
  // done; every thread passes the wait, so that the kernels follow in order)
  const int s = find_sequence(p.q, blockIdx.x, p.chunk);
  Seq q = resolve(p.q, s < 0 ? 0 : s);
  // (a summary is its sequence's own, whoever else has the slot)
  const bool mine = SUMMARY ? q.live : writes(p.q, s < 0 ? 0 : s, q, s >= 0 && blockIdx.y == 0);
  griddep_launch();
  griddep_wait();
  if (s < 0 || !mine) return;
  const long long k = blockIdx.x - (q.begin / p.chunk + s);
  if (k > 0 && k * p.chunk >= q.len) return;
  const int t0 = static_cast<int>(k * p.chunk);
  const bool last = t0 + p.chunk >= q.len;
  if (SUMMARY && last) return;
  const int rows = min(p.chunk, q.len - t0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.y * (kScanWarps * 32) + threadIdx.x;
  const bool on = c < p.di;
  const int cc = on ? c : p.di - 1;
  const int ds = p.ds;
  float* st = p.state == nullptr ? nullptr : p.state + q.slot * p.slot_stride + cc;
  float* ws = p.ws == nullptr ? nullptr : p.ws + static_cast<long long>(blockIdx.x) * (1 + ds) * p.di + cc;
  const long long row0 = q.begin + t0;
  const T* bc = static_cast<const T*>(p.proj) + row0 * p.proj_ld + p.dr;
  const float* dt = p.steps + row0 * p.di + cc;
  const T* u = static_cast<const T*>(p.u) + row0 * p.u_ld + cc;
  const T* z = SUMMARY || p.z == nullptr ? nullptr : static_cast<const T*>(p.z) + row0 * p.z_ld + cc;
  T* y = static_cast<T*>(p.y) + row0 * p.y_ld + cc;

  // B and C: a warp brings four rows of a stage, a lane the columns lane + 32 m
  // of [B (DS) | C (DS)], zero behind ds and behind the last row
  constexpr int kPieces = (2 * DS + 31) / 32, kMine = kStage / kScanWarps;
  T pn[kMine][kPieces];
  auto request = [&](int t) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int j = t + kMine * warp + i;
#pragma unroll
      for (int m = 0; m < kPieces; ++m) {
        const int e = lane + 32 * m, n = e % DS;
        pn[i][m] = from_f32<T>(0.0f);
        if (e < 2 * DS && n < ds && j < rows) pn[i][m] = bc[j * p.proj_ld + (e < DS ? n : ds + n)];
      }
    }
  };
  auto settle = [&](int b) {
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
      for (int m = 0; m < kPieces; ++m)
        if (lane + 32 * m < 2 * DS) sbc[b][kMine * warp + i][lane + 32 * m] = to_f32(pn[i][m]);
  };
  // dt, u and z of the next kTok rows; the pointers stand behind the last
  // whole step requested
  float dn[kTok];
  T un[kTok], zn[kTok];
  const bool gated = z != nullptr;
  auto request_row = [&](int j) {
    dn[j] = dt[j * static_cast<long long>(p.di)];
    un[j] = u[j * p.u_ld];
    if (gated) zn[j] = z[j * p.z_ld];
  };
  auto advance = [&] {
    dt += kTok * static_cast<long long>(p.di);
    u += kTok * p.u_ld;
    if (gated) z += kTok * p.z_ld;
  };
  // the stage after the next one into L2: a lane its row's line of this warp
  auto prefetch = [&](int t) {
    const int j = t + lane;
    if (lane < kStage && j < rows) {
      const long long row = row0 + j;
      const int cw = min(c - lane, p.di - 1);
      prefetch_l2(p.steps + row * p.di + cw);
      prefetch_l2(static_cast<const T*>(p.u) + row * p.u_ld + cw);
      if (gated) prefetch_l2(static_cast<const T*>(p.z) + row * p.z_ld + cw);
    }
  };
  request(0);
#pragma unroll
  for (int j = 0; j < kTok; ++j)
    if (j < rows) request_row(j);
  advance();
  prefetch(kTok);
  float2 h[DS / 2], an[DS / 2];
  auto load_state = [&](int n) {
    if (SUMMARY || n >= ds) return 0.0f;
    if (k > 0 || !last) return ws[static_cast<long long>(1 + n) * p.di];
    return st != nullptr && !q.fresh ? st[static_cast<long long>(n) * p.di] : 0.0f;
  };
  auto load_a = [&](int n) { return n < ds ? p.a[static_cast<long long>(n) * p.di + cc] * 1.4426950408889634f : 0.0f; };
#pragma unroll
  for (int n = 0; n < DS / 2; ++n) {
    an[n] = make_float2(load_a(2 * n), load_a(2 * n + 1));
    h[n] = make_float2(load_state(2 * n), load_state(2 * n + 1));
  }
  const float dk = p.d[cc];
  float total = 0.0f;
  float sum_dt = 0.0f;  // summed apart: fewer roundings than one long sum
  auto one_row = [&](const float* row, float d, float uv, float zv) {
    const float dtu = d * uv;
    const float2 d2 = splat(d), dtu2 = splat(dtu);
    float2 y0, y1;
    if (SUMMARY) sum_dt += d;
#pragma unroll
    for (int n = 0; n < DS / 2; n += 2) {
      const float4 bq = *reinterpret_cast<const float4*>(row + 2 * n);
      const float2 e0 = __fmul2_rn(d2, an[n]), e1 = __fmul2_rn(d2, an[n + 1]);
      const float2 a0 = n < kPolyPairs<DS> ? exp2_neg2(e0) : make_float2(ex2_approx(e0.x), ex2_approx(e0.y));
      const float2 a1 = n + 1 < kPolyPairs<DS> ? exp2_neg2(e1) : make_float2(ex2_approx(e1.x), ex2_approx(e1.y));
      h[n] = __ffma2_rn(a0, h[n], __fmul2_rn(dtu2, make_float2(bq.x, bq.y)));
      h[n + 1] = __ffma2_rn(a1, h[n + 1], __fmul2_rn(dtu2, make_float2(bq.z, bq.w)));
      if (!SUMMARY) {
        const float4 cq = *reinterpret_cast<const float4*>(row + DS + 2 * n);
        const float2 c0 = make_float2(cq.x, cq.y), c1 = make_float2(cq.z, cq.w);
        float2 h0 = h[n], h1 = h[n + 1];
        if (PADDED && n == DS / 2 - 2) {
          h0.y = DS - 3 < ds ? h0.y : 0.0f;
          h1.x = DS - 2 < ds ? h1.x : 0.0f;
          h1.y = 0.0f;
        }
        y0 = n == 0 ? __fmul2_rn(h0, c0) : __ffma2_rn(h0, c0, y0);
        y1 = n == 0 ? __fmul2_rn(h1, c1) : __ffma2_rn(h1, c1, y1);
      }
    }
    if (SUMMARY) return 0.0f;
    const float2 sum = __fadd2_rn(y0, y1);
    const float yv = fmaf(dk, uv, sum.x + sum.y);
    return gated ? yv * silu1(zv) : yv;
  };
  settle(0);
  for (int t = 0, b = 0; t < rows; t += kStage, b ^= 1) {
    __syncthreads();  // this stage is written, the other one has been read
    const bool more = t + kStage < rows;
    if (more) {
      request(t + kStage);
      prefetch(t + kStage + kTok);
    }
    const int stop = min(kStage, rows - t);
    int i = 0;
    for (; i + kTok <= stop; i += kTok) {
      const int left = rows - t - i - kTok;  // rows behind this step
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        const float d = dn[j], uv = to_f32(un[j]), zv = gated ? to_f32(zn[j]) : 0.0f;
        if (j < left) request_row(j);
        const float yv = one_row(sbc[b][i + j], d, uv, zv);
        if (!SUMMARY && on) y[j * p.y_ld] = from_f32<T>(yv);
      }
      advance();
      y += kTok * p.y_ld;
      total += sum_dt;
      sum_dt = 0.0f;
    }
    for (; i < stop; ++i) {  // the last rows of the tile, fewer than kTok
      const float yv = one_row(sbc[b][i], dn[0], to_f32(un[0]), gated ? to_f32(zn[0]) : 0.0f);
      if (!SUMMARY && on) *y = from_f32<T>(yv);
      y += p.y_ld;
#pragma unroll
      for (int j = 0; j + 1 < kTok; ++j) {
        dn[j] = dn[j + 1];
        un[j] = un[j + 1];
        zn[j] = zn[j + 1];
      }
    }
    total += sum_dt;
    sum_dt = 0.0f;
    if (more) settle(b ^ 1);
  }
  if (!on) return;
  auto store = [&](float* to) {
#pragma unroll
    for (int n = 0; n < DS / 2; ++n) {
      if (2 * n < ds) to[static_cast<long long>(2 * n) * p.di] = h[n].x;
      if (2 * n + 1 < ds) to[static_cast<long long>(2 * n + 1) * p.di] = h[n].y;
    }
  };
  if (SUMMARY) {
    ws[0] = total;
    store(ws + p.di);
  } else if (last && st != nullptr) {
    store(st);
  }
}

// The state that enters each tile of a sequence of several, in place of the
// tile's own end: one thread per channel and kCarryStates states walks the
// tiles, the next kCarryAhead of them requested at a time (16384 rows x
// 2048 channels: adds 12 us, a latency chain).
constexpr int kCarryStates = 2, kCarryAhead = 8, kCarryThreads = 256;
__global__ void __launch_bounds__(kCarryThreads) scan_carry_kernel(const ScanParams p) {
  const int s = blockIdx.x, n0 = blockIdx.z * kCarryStates;
  const Seq q = resolve(p.q, s);
  griddep_launch();
  griddep_wait();
  const int c = blockIdx.y * kCarryThreads + threadIdx.x;
  if (!q.live || q.len <= p.chunk || c >= p.di) return;
  const int tiles = (q.len + p.chunk - 1) / p.chunk;
  const long long step = static_cast<long long>(1 + p.ds) * p.di;
  float* ws = p.ws + (q.begin / p.chunk + s) * step + c;
  float an[kCarryStates], h[kCarryStates];
#pragma unroll
  for (int i = 0; i < kCarryStates; ++i) {
    const long long at = static_cast<long long>(min(n0 + i, p.ds - 1)) * p.di;
    an[i] = p.a[at + c] * 1.4426950408889634f;
    h[i] = p.state == nullptr || q.fresh ? 0.0f : p.state[q.slot * p.slot_stride + at + c];
  }
  for (int k = 0; k < tiles; k += kCarryAhead) {
    float dt[kCarryAhead], e[kCarryAhead][kCarryStates];
#pragma unroll
    for (int j = 0; j < kCarryAhead; ++j) {
      const bool more = k + j + 1 < tiles;  // the last tile has no summary
      dt[j] = more ? ws[j * step] : 0.0f;
#pragma unroll
      for (int i = 0; i < kCarryStates; ++i)
        e[j][i] = more && n0 + i < p.ds ? ws[j * step + static_cast<long long>(1 + n0 + i) * p.di] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kCarryAhead; ++j) {
      if (k + j >= tiles) break;
#pragma unroll
      for (int i = 0; i < kCarryStates; ++i) {
        if (n0 + i < p.ds) ws[j * step + static_cast<long long>(1 + n0 + i) * p.di] = h[i];
        // (a tile's decay may be below float32's range though no row's is: an
        // infinite state stays infinite)
        const float x = dt[j] * an[i], decay = ex2_approx(x);
        h[i] = fmaf(x > -INFINITY ? max_nan(decay, 1.4e-45f) : decay, h[i], e[j][i]);
      }
    }
    ws += kCarryAhead * step;
  }
}

// Rows of a tile, a power of two: as many tiles as keep about kFillThreads
// threads (one per channel) on every SM.
constexpr int kMinChunk = 16, kMaxChunk = 2048, kFillThreads = 768;

int scan_chunk(long long rows, int di) {
  const long long want = rows * di / (static_cast<long long>(kFillThreads) * current_sm_count());
  int chunk = kMinChunk;
  while (chunk < kMaxChunk && chunk * 2 <= want) chunk *= 2;
  return chunk;
}

// Whether dt of single tokens is made for all of them beforehand: from as many
// as fill the GPU.  Fewer take dt_w from L2 faster than another kernel starts.
bool tokens_given(long long n_seq, long long di) { return n_seq * di >= 512LL * current_sm_count() && n_seq >= 16; }

template <typename T, int DS, bool PADDED>
int scan_tokens(const ScanParams& p, cudaStream_t st) {
  const auto even = [](const void* q, long long ld, std::size_t e) {
    return reinterpret_cast<std::uintptr_t>(q) % (2 * e) == 0 && ld % 2 == 0;
  };
  // pairs of channels where the matrices and slots allow it
  const bool pairs = p.di % 2 == 0 && even(p.u, p.u_ld, sizeof(T)) && even(p.y, p.y_ld, sizeof(T)) &&
                     even(p.z, p.z_ld, sizeof(T)) && even(p.state, p.slot_stride, 4) && even(p.a, 0, 4) &&
                     even(p.d, 0, 4) && even(p.dt_w, 0, 4) && even(p.dt_b, 0, 4);
  const int channels = 128 / (DS / kTokenStates) * (pairs ? 2 : 1);  // of a CTA
  const dim3 grid(static_cast<unsigned>(p.q.n_seq), static_cast<unsigned>((p.di + channels - 1) / channels));
  const dim3 block(128);
  if (tokens_given(p.q.n_seq, p.di)) {
    if (const int rc = steps_launch<T>(p, st); rc != 0) return rc;
    pairs ? launch_pdl(scan_token_kernel<T, DS, 2, true, PADDED>, grid, block, 0, st, p)
          : launch_pdl(scan_token_kernel<T, DS, 1, true, PADDED>, grid, block, 0, st, p);
  } else {
    const std::size_t smem = static_cast<std::size_t>(p.dr) * sizeof(float);
    pairs ? scan_token_kernel<T, DS, 2, false, PADDED><<<grid, block, smem, st>>>(p)
          : scan_token_kernel<T, DS, 1, false, PADDED><<<grid, block, smem, st>>>(p);
  }
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int DS, bool PADDED>
int scan_prompts(const ScanParams& p, cudaStream_t st) {
  const unsigned cb = static_cast<unsigned>((p.di + 127) / 128);
  const dim3 grid(static_cast<unsigned>(p.q.rows / p.chunk + p.q.n_seq), cb);
  if (const int rc = steps_launch<T>(p, st); rc != 0) return rc;
  if (p.q.rows > p.chunk) {
    launch_pdl(scan_prompt_kernel<T, DS, true, false>, grid, dim3(kScanWarps * 32), 0, st, p);
    launch_pdl(scan_carry_kernel,
               dim3(static_cast<unsigned>(p.q.n_seq), static_cast<unsigned>((p.di + kCarryThreads - 1) / kCarryThreads),
                    static_cast<unsigned>((p.ds + kCarryStates - 1) / kCarryStates)),
               dim3(kCarryThreads), 0, st, p);
  }
  if (p.q.rows > 0)
    launch_pdl(scan_prompt_kernel<T, DS, false, PADDED>, grid, dim3(kScanWarps * 32), 0, st, p);
  else  // behind no kernel of this call: the caller's writes have to be seen
    scan_prompt_kernel<T, DS, false, PADDED><<<grid, kScanWarps * 32, 0, st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int DS = 4>
int scan_prompts_sized(const ScanParams& p, cudaStream_t st) {
  if constexpr (DS < 32)
    if (p.ds > DS) return scan_prompts_sized<T, DS + 4>(p, st);
  return p.ds < DS ? scan_prompts<T, DS, true>(p, st) : scan_prompts<T, DS, false>(p, st);
}

template <typename T, int DS>
int scan_tokens_sized(const ScanParams& p, cudaStream_t st) {
  return p.ds < DS ? scan_tokens<T, DS, true>(p, st) : scan_tokens<T, DS, false>(p, st);
}

template <typename T>
int scan_sized(const ScanParams& p, cudaStream_t st) {
  if (p.q.offsets != nullptr) return scan_prompts_sized<T>(p, st);
  if (p.ds <= 8) return scan_tokens_sized<T, 8>(p, st);
  if (p.ds <= 16) return scan_tokens_sized<T, 16>(p, st);
  return scan_tokens_sized<T, 32>(p, st);
}

SeqParams sequences(const std::int32_t* offsets, const std::int32_t* slots, const std::uint8_t* fresh,
                    std::int32_t* status, std::uint64_t rows, std::uint64_t n_seq, std::uint64_t n_slots,
                    bool stateful) {
  return SeqParams{offsets, slots, fresh, status, static_cast<long long>(rows), static_cast<int>(n_seq),
                   static_cast<int>(n_slots), stateful};
}

}  // namespace

DeviceScope::DeviceScope(int device) noexcept {
  int now = 0;
  if (device < 0) return;
  ok_ = cudaGetDevice(&now) == cudaSuccess;
  if (!ok_ || now == device) return;
  ok_ = cudaSetDevice(device) == cudaSuccess;
  if (ok_)
    before_ = now;
  else
    cudaGetLastError();
}

DeviceScope::~DeviceScope() {
  if (before_ >= 0) cudaSetDevice(before_);
}

const char* cuda_error_text(int code) noexcept { return cudaGetErrorString(static_cast<cudaError_t>(code)); }

int current_sm_count() noexcept {
  static std::atomic<int> counts[64];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 148;
  int v = counts[device].load(std::memory_order_relaxed);
  if (v == 0) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || v <= 0) return 148;
    counts[device].store(v, std::memory_order_relaxed);
  }
  return v;
}

int causal_conv_chunk(std::size_t rows, std::size_t n_seq, std::size_t across) noexcept {
  return conv_chunk(static_cast<long long>(rows), static_cast<long long>(n_seq), static_cast<long long>(across));
}

int launch_causal_conv(const fe_conv_args& a, void* stream) noexcept {
  ConvParams p{sequences(a.offsets, a.slots, a.fresh, a.status, a.rows, a.n_seq, a.n_slots, a.window != nullptr),
               a.x, a.w, a.b, a.u, a.window, a.x_ld, a.u_ld, a.slot_stride, static_cast<int>(a.d_inner),
               static_cast<int>(a.d_conv), 0};
  const auto st = static_cast<cudaStream_t>(stream);
  return with_dtype(a.dtype, [&](auto t) { return conv_typed<decltype(t)>(p, st); });
}

namespace {

// Bytes of the rows' steps, a whole number of 256 bytes.
std::size_t steps_bytes(std::size_t rows, std::size_t d_inner) {
  return (rows * d_inner * sizeof(float) + 255) / 256 * 256;
}

}  // namespace

std::size_t selective_scan_workspace(const fe_scan_args& a) noexcept {
  const std::size_t steps = steps_bytes(a.rows, a.d_inner);
  if (a.offsets == nullptr)
    return tokens_given(static_cast<long long>(a.n_seq), static_cast<long long>(a.d_inner)) ? steps : 0;
  const int chunk = scan_chunk(static_cast<long long>(a.rows), static_cast<int>(a.d_inner));
  if (a.rows <= static_cast<std::uint64_t>(chunk)) return steps;
  return steps + (a.rows / static_cast<std::uint64_t>(chunk) + a.n_seq) * (1 + a.d_state) * a.d_inner * sizeof(float);
}

std::size_t selective_scan_workspace_most(std::size_t rows, std::size_t n_seq, std::size_t d_inner,
                                          std::size_t d_state) noexcept {
  // the most tiles of rows cut by each chunk that scan_chunk gives for fewer
  std::size_t tiles = 0;
  for (std::size_t chunk = kMinChunk; chunk <= kMaxChunk; chunk *= 2) {
    std::size_t most = rows;
    if (chunk < kMaxChunk) most = std::min(most, 2 * chunk * kFillThreads * current_sm_count() / d_inner + 1);
    tiles = std::max(tiles, most / chunk);
  }
  return steps_bytes(rows, d_inner) + (tiles + n_seq) * (1 + d_state) * d_inner * sizeof(float);
}

int launch_selective_scan(const fe_scan_args& a, void* stream) noexcept {
  ScanParams p{sequences(a.offsets, a.slots, a.fresh, a.status, a.rows, a.n_seq, a.n_slots, a.state != nullptr),
               a.u, a.proj, a.z, a.a, a.d, a.dt_w, a.dt_b, a.y, a.state, static_cast<float*>(a.workspace),
               static_cast<float*>(a.workspace), a.u_ld, a.proj_ld, a.z_ld, a.y_ld, a.slot_stride, static_cast<int>(a.d_inner),
               static_cast<int>(a.d_state), static_cast<int>(a.dt_rank), 0};
  if (a.offsets != nullptr) {
    p.chunk = scan_chunk(p.q.rows, p.di);
    p.ws = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + steps_bytes(a.rows, a.d_inner));
  }
  const auto st = static_cast<cudaStream_t>(stream);
  return with_dtype(a.dtype, [&](auto t) { return scan_sized<decltype(t)>(p, st); });
}

}  // namespace feb
