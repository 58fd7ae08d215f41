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
#include <cstdint>

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
  int slot;
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

// Bounds, slot and flags of sequence s; every thread of the CTA calls it.
// live is false for a sequence that is skipped: a negative slot, or one of the
// faults that set a status bit (offsets outside the rows, a slot outside the
// pool, a slot that an earlier sequence of the call has).
__device__ Seq resolve(const SeqParams& q, int s, bool report) {
  Seq r;
  int bad = 0;
  if (q.offsets != nullptr) {
    const int b = q.offsets[s], e = q.offsets[s + 1];
    if (b < 0 || e < b || e > q.rows) bad |= FE_SEQ_BAD_OFFSETS;
    r.begin = b;
    r.len = e - b;
  } else {
    r.begin = s;
    r.len = 1;
  }
  r.slot = q.slots != nullptr ? q.slots[s] : s;
  if (q.stateful && r.slot >= q.n_slots) bad |= FE_SEQ_BAD_SLOT;
  r.fresh = q.fresh != nullptr && q.fresh[s] != 0;
  int dup = 0;
  if (q.stateful && q.slots != nullptr && r.slot >= 0) {
    for (int i = threadIdx.x; i < s; i += blockDim.x) dup |= q.slots[i] == r.slot;
    dup = __syncthreads_or(dup);
  }
  if (dup) bad |= FE_SEQ_DUPLICATE_SLOT;
  r.live = bad == 0 && r.slot >= 0;
  if (report && bad != 0 && q.status != nullptr && threadIdx.x == 0) atomicOr(q.status, bad);
  return r;
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
// Bound by the window's bytes.
template <typename T>
__global__ void __launch_bounds__(128) conv_token_kernel(const ConvParams p) {
  const int s = blockIdx.x;
  const Seq q = resolve(p.q, s, blockIdx.y == 0);
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  if (!q.live || c >= p.di) return;
  const float xv = to_f32(static_cast<const T*>(p.x)[s * p.x_ld + c]);
  const float* w = p.w + static_cast<long long>(c) * p.dc;
  float* win = p.window == nullptr ? nullptr : p.window + q.slot * p.slot_stride + static_cast<long long>(c) * p.dc;
  float acc = p.b[c];
  for (int k = 0; k + 1 < p.dc; ++k) {
    const float v = win == nullptr || q.fresh ? 0.0f : win[k + 1];
    if (win != nullptr) win[k] = v;
    acc = fmaf(w[k], v, acc);
  }
  if (win != nullptr) win[p.dc - 1] = xv;
  acc = fmaf(w[p.dc - 1], xv, acc);
  static_cast<T*>(p.u)[s * p.u_ld + c] = from_f32<T>(silu_f(acc));
}

// One thread per channel walks the tile's rows with the last DC inputs in
// registers (right-aligned: taps before the first of dc carry weight zero).
// The first tile of a sequence reads the old window and writes the new one
// from the sequence's last rows, so no other tile touches it.
template <typename T, int DC>
__global__ void __launch_bounds__(128) conv_prompt_kernel(const ConvParams p) {
  report_offsets(p.q);
  const int s = find_sequence(p.q, blockIdx.x, p.chunk);
  if (s < 0) return;
  const Seq q = resolve(p.q, s, blockIdx.y == 0);
  const long long k = blockIdx.x - (q.begin / p.chunk + s);
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  if (!q.live || c >= p.di || (k > 0 && k * p.chunk >= q.len)) return;
  const int t0 = static_cast<int>(k * p.chunk);
  const T* x = static_cast<const T*>(p.x) + q.begin * p.x_ld + c;
  T* u = static_cast<T*>(p.u) + q.begin * p.u_ld + c;
  float* win = p.window == nullptr ? nullptr : p.window + q.slot * p.slot_stride + static_cast<long long>(c) * p.dc;
  float wk[DC], in[DC];
#pragma unroll
  for (int j = 0; j < DC; ++j) {
    const int tap = j - (DC - p.dc);
    wk[j] = tap >= 0 ? p.w[static_cast<long long>(c) * p.dc + tap] : 0.0f;
    const int t = t0 - DC + j;  // the input that slot j holds before row t0
    in[j] = 0.0f;
    if (t >= 0)
      in[j] = to_f32(x[t * p.x_ld]);
    else if (win != nullptr && !q.fresh && p.dc + t >= 0)
      in[j] = win[p.dc + t];
  }
  const float bias = p.b[c];
  if (k == 0 && win != nullptr) {
    for (int j = 0; j < p.dc; ++j) {
      const int t = q.len - p.dc + j;
      win[j] = t >= 0 ? to_f32(x[t * p.x_ld]) : (q.fresh ? 0.0f : win[p.dc + t]);
    }
  }
  const int t1 = min(t0 + p.chunk, q.len);
  constexpr int kAhead = 8;
  for (int t = t0; t < t1; t += kAhead) {
    float v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = t + i < t1 ? to_f32(x[(t + i) * p.x_ld]) : 0.0f;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
#pragma unroll
      for (int j = 0; j + 1 < DC; ++j) in[j] = in[j + 1];
      in[DC - 1] = v[i];
      float acc = bias;
#pragma unroll
      for (int j = 0; j < DC; ++j) acc = fmaf(wk[j], in[j], acc);
      if (t + i < t1) u[(t + i) * p.u_ld] = from_f32<T>(silu_f(acc));
    }
  }
}

template <typename T>
int conv_typed(const ConvParams& p, cudaStream_t st) {
  const unsigned cb = static_cast<unsigned>((p.di + 127) / 128);
  if (p.q.offsets == nullptr) {
    conv_token_kernel<T><<<dim3(static_cast<unsigned>(p.q.n_seq), cb), 128, 0, st>>>(p);
    return static_cast<int>(cudaGetLastError());
  }
  const dim3 grid(static_cast<unsigned>(p.q.rows / p.chunk + p.q.n_seq), cb);
  if (p.dc <= 4)
    conv_prompt_kernel<T, 4><<<grid, 128, 0, st>>>(p);
  else
    conv_prompt_kernel<T, 8><<<grid, 128, 0, st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

// --- selective scan -----------------------------------------------------------

struct ScanParams {
  SeqParams q;
  const void *u, *proj, *z;
  const float *a, *d, *dt_w, *dt_b;  // a [ds][di], dt_w [dr][di]
  void* y;
  float* state;  // [slot][ds][di]
  float* ws;     // [tile][1 + ds][di]: sum of dt, then the tile's state (its end from zero; later its start)
  long long u_ld, proj_ld, z_ld, y_ld, slot_stride;
  int di, ds, dr, chunk;
};

// softplus(x) to a few ulp of the result: e = exp(-|x|) with the rounding error
// of x log2(e) carried into the exponential, log(1 + e) = 2 atanh(e / (2 + e))
// by its series (the argument is at most 1/3; the first term left out is
// below 2^-26 of the sum).  log(1 + e) as it stands would lose dt's relative
// precision for the small steps that the scan lives on.
__device__ __forceinline__ float softplus_rel(float x) {
  constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.9259629911e-8f;
  const float ax = fminf(fabsf(x), 120.0f);
  const float hi = -ax * kLog2e;
  const float lo = fmaf(-ax, kLog2e, -hi) - ax * kLog2eLow;
  const float e2 = ex2_approx(hi);
  const float e = fmaf(e2 * 0.69314718f, lo, e2);
  const float s = __fdividef(e, 2.0f + e), s2 = s * s;
  float r = fmaf(s2, 1.0f / 15.0f, 1.0f / 13.0f);
  r = fmaf(r, s2, 1.0f / 11.0f);
  r = fmaf(r, s2, 1.0f / 9.0f);
  r = fmaf(r, s2, 1.0f / 7.0f);
  r = fmaf(r, s2, 1.0f / 5.0f);
  r = fmaf(r, s2, 1.0f / 3.0f);
  r = fmaf(r * s2, s, s);
  const float sp = fmaf(2.0f, r, fmaxf(x, 0.0f));
  return x != x ? x : sp;
}

// One token for each of up to RT sequences, one thread per channel.  The dt
// projection's weights are read once for the RT tokens; then each sequence's
// ds states are read, stepped and written (the kernel's bytes).
template <typename T, int DS, int RT>
__global__ void __launch_bounds__(128) scan_token_kernel(const ScanParams p) {
  extern __shared__ float sp[];  // [RT][dr + 2 ds]
  __shared__ int sdup;
  const int s0 = blockIdx.x * RT, c = blockIdx.y * 128 + threadIdx.x;
  const int wd = p.dr + 2 * p.ds;
  int slot[RT], bad[RT];
  bool fresh[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    const int s = s0 + j;
    slot[j] = s >= p.q.n_seq ? -1 : (p.q.slots != nullptr ? p.q.slots[s] : s);
    fresh[j] = s < p.q.n_seq && p.q.fresh != nullptr && p.q.fresh[s] != 0;
    bad[j] = p.q.stateful && slot[j] >= p.q.n_slots ? FE_SEQ_BAD_SLOT : 0;
  }
  if (threadIdx.x == 0) sdup = 0;
  for (int i = threadIdx.x; i < RT * wd; i += 128) {
    const int j = i / wd;
    if (s0 + j < p.q.n_seq)
      sp[i] = to_f32(static_cast<const T*>(p.proj)[(s0 + j) * p.proj_ld + (i - j * wd)]);
  }
  __syncthreads();
  if (p.q.stateful && p.q.slots != nullptr) {
    int dup = 0;
    for (int i = threadIdx.x; i < min(s0 + RT, p.q.n_seq); i += 128) {
      const int v = p.q.slots[i];
#pragma unroll
      for (int j = 0; j < RT; ++j)
        if (i < s0 + j && v == slot[j] && v >= 0) dup |= 1 << j;
    }
    if (dup != 0) atomicOr(&sdup, dup);
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    if (sdup >> j & 1) bad[j] |= FE_SEQ_DUPLICATE_SLOT;
    if (bad[j] != 0 && p.q.status != nullptr && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(p.q.status, bad[j]);
    if (bad[j] != 0) slot[j] = -1;
  }
  if (c >= p.di) return;
  float acc[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) acc[j] = 0.0f;
#pragma unroll 8
  for (int r = 0; r < p.dr; ++r) {
    const float w = p.dt_w[static_cast<long long>(r) * p.di + c];
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[j] = fmaf(sp[j * wd + r], w, acc[j]);
  }
  float an[DS];
#pragma unroll
  for (int n = 0; n < DS; ++n) an[n] = n < p.ds ? p.a[static_cast<long long>(n) * p.di + c] * 1.4426950408889634f : 0.0f;
  const float bdt = p.dt_b[c], dk = p.d[c];
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    if (slot[j] < 0) continue;
    float* st = p.state == nullptr ? nullptr : p.state + slot[j] * p.slot_stride + c;
    float h[DS];
#pragma unroll
    for (int n = 0; n < DS; ++n)
      h[n] = st != nullptr && !fresh[j] && n < p.ds ? st[static_cast<long long>(n) * p.di] : 0.0f;
    const float uv = to_f32(static_cast<const T*>(p.u)[(s0 + j) * p.u_ld + c]);
    const float dt = softplus_rel(acc[j] + bdt), dtu = dt * uv;
    const float* row = sp + j * wd + p.dr;
    float y = dk * uv;
#pragma unroll
    for (int n = 0; n < DS; ++n) {
      if (n >= p.ds) break;
      h[n] = fmaf(ex2_approx(dt * an[n]), h[n], dtu * row[n]);
      y = fmaf(h[n], row[p.ds + n], y);
      if (st != nullptr) st[static_cast<long long>(n) * p.di] = h[n];
    }
    if (p.z != nullptr) {
      const float zv = to_f32(static_cast<const T*>(p.z)[(s0 + j) * p.z_ld + c]);
      y *= silu_f(zv);
    }
    static_cast<T*>(p.y)[(s0 + j) * p.y_ld + c] = from_f32<T>(y);
  }
}

// 2^x for a pair of x <= 0 on the FMA pipe.  x = k + r with k whole and r in
// [-1/2, 1/2] (k by adding and taking away 1.5 * 2^23), 2^r = 1 + r q(r) with
// q the degree-5 Chebyshev interpolant of (2^r - 1) / r, 2^k added to the
// exponent field; below 2^-125 the result stays there.  The leading 1 is exact
// and the error is that of the last addition (at most 7.2e-8, mean 3e-10), so
// that a decay near 1 keeps its distance from 1 over thousands of steps.
__device__ __forceinline__ float2 exp2_neg2(float2 x) {
  constexpr float kRound = 12582912.0f;
  x.x = fmaxf(x.x, -125.0f);
  x.y = fmaxf(x.y, -125.0f);
  const float2 t = __fadd2_rn(x, make_float2(kRound, kRound));
  const float2 k = __fadd2_rn(t, make_float2(-kRound, -kRound));
  const float2 r = __ffma2_rn(k, make_float2(-1.0f, -1.0f), x);
  float2 p = __ffma2_rn(make_float2(1.5453163e-4f, 1.5453163e-4f), r, make_float2(1.3390863e-3f, 1.3390863e-3f));
  p = __ffma2_rn(p, r, make_float2(9.6180830e-3f, 9.6180830e-3f));
  p = __ffma2_rn(p, r, make_float2(5.5503570e-2f, 5.5503570e-2f));
  p = __ffma2_rn(p, r, make_float2(2.4022651e-1f, 2.4022651e-1f));
  p = __ffma2_rn(p, r, make_float2(6.9314718e-1f, 6.9314718e-1f));
  p = __ffma2_rn(p, r, make_float2(1.0f, 1.0f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}

// softplus_rel for a pair
__device__ __forceinline__ float2 softplus_rel2(float2 x) {
  return make_float2(softplus_rel(x.x), softplus_rel(x.y));
}

constexpr int kTok = 8;        // rows of a step of the prompt kernel
constexpr int kScanWarps = 4;  // warps of its CTA, 32 channels each
constexpr int kAhead = 4;      // 32-column pieces of a proj row that are requested a step ahead
// State pairs whose exponentials go to the FMA pipe: the MUFU unit then has
// 2 (DS - 2 kPolyPairs) / 2 + 4 results per row and channel to make, the FMA
// pipe about 4 per state and 12 per exponential; DS / 8 of the pairs balance
// them.
template <int DS>
constexpr int kPolyPairs = DS / 8;

// The shared memory of a step: dt_in of its rows [dr][kTok], then per row
// [B (DS) | C (DS)], zero behind ds.
__host__ __device__ constexpr int scan_stage(int dr, int ds_padded) { return kTok * (dr + 2 * ds_padded); }

// One thread per channel, the states in registers, over the rows of one tile.
// SUMMARY: the tile's sum of dt and its state from a zero start, for the tiles
// whose sequence goes on (the recurrence over a tile is h -> exp(A sum dt) h +
// end, so the sum of dt stands for the product of decays).  Otherwise: from
// the state that enters the tile, with y.
//
// Bound by arithmetic: per row and channel DS exponentials (MUFU and FMA pipe
// share them), dr products for dt and 4 DS for the states; u, z, y and proj
// pass through once.  Rows go in steps of kTok: the step's proj rows sit in
// shared memory (read by every channel), the next step's proj, u and z are
// requested before the arithmetic.  All arithmetic on pairs (FFMA2): states
// two and two, dt rows two and two.
template <typename T, int DS, bool SUMMARY>
__global__ void __launch_bounds__(kScanWarps * 32) scan_prompt_kernel(const ScanParams p) {
  extern __shared__ __align__(16) float sp[];  // two stages
  if (!SUMMARY) report_offsets(p.q);
  const int s = find_sequence(p.q, blockIdx.x, p.chunk);
  if (s < 0) return;
  const Seq q = resolve(p.q, s, !SUMMARY && blockIdx.y == 0);
  const long long k = blockIdx.x - (q.begin / p.chunk + s);
  if (!q.live || (k > 0 && k * p.chunk >= q.len)) return;
  const int t0 = static_cast<int>(k * p.chunk);
  const bool last = t0 + p.chunk >= q.len;
  if (SUMMARY && last) return;
  const int t1 = min(t0 + p.chunk, q.len);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.y * (kScanWarps * 32) + threadIdx.x;
  const bool on = c < p.di;
  const int cc = on ? c : p.di - 1;
  const int ds = p.ds, dr = p.dr, wd = dr + 2 * ds;
  const int stage = scan_stage(dr, DS);
  float* st = p.state == nullptr ? nullptr : p.state + q.slot * p.slot_stride + cc;
  float* ws = p.ws == nullptr ? nullptr : p.ws + static_cast<long long>(blockIdx.x) * (1 + ds) * p.di + cc;
  const T* proj = static_cast<const T*>(p.proj) + (q.begin + t0) * p.proj_ld;
  const T* u = static_cast<const T*>(p.u) + (q.begin + t0) * p.u_ld + cc;
  const T* z = SUMMARY || p.z == nullptr ? nullptr : static_cast<const T*>(p.z) + (q.begin + t0) * p.z_ld + cc;
  T* y = static_cast<T*>(p.y) + (q.begin + t0) * p.y_ld + cc;
  const int rows = t1 - t0;
  // a warp brings two rows of a step: rows 2 warp and 2 warp + 1, a lane
  // their columns lane + 32 m; column e goes to place(e) + its row's distance
  auto place = [&](int e, int j) {
    if (e < dr) return e * kTok + j;
    const int b = e - dr;
    return dr * kTok + j * 2 * DS + (b < ds ? b : DS + b - ds);
  };
  T pn[2][kAhead];
  auto request = [&](int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = t + 2 * warp + i;
#pragma unroll
      for (int m = 0; m < kAhead; ++m) {
        const int e = lane + 32 * m;
        pn[i][m] = from_f32<T>(0.0f);
        if (e < wd && j < rows) pn[i][m] = proj[j * p.proj_ld + e];
      }
    }
  };
  auto settle = [&](int t, float* to) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = 2 * warp + i;
#pragma unroll
      for (int m = 0; m < kAhead; ++m) {
        const int e = lane + 32 * m;
        if (e < wd) to[place(e, j)] = to_f32(pn[i][m]);
      }
      for (int e = lane + 32 * kAhead; e < wd; e += 32)
        to[place(e, j)] = t + j < rows ? to_f32(proj[(t + j) * p.proj_ld + e]) : 0.0f;
    }
  };
  T un[kTok], zn[kTok];
  auto request_uz = [&](int t) {
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      un[j] = zn[j] = from_f32<T>(0.0f);
      if (t + j < rows) {
        un[j] = u[(t + j) * p.u_ld];
        if (z != nullptr) zn[j] = z[(t + j) * p.z_ld];
      }
    }
  };
  if (rows > 0) {
    request(0);
    request_uz(0);
  }
  if (ds < DS)
    for (int i = threadIdx.x; i < 2 * kTok * 2 * DS; i += kScanWarps * 32) {
      const int b = i / (kTok * 2 * DS), e = i % (kTok * 2 * DS);
      if (e % DS >= ds) sp[b * stage + dr * kTok + e] = 0.0f;
    }
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
  const float bdt = p.dt_b[cc], dk = p.d[cc];
  const float* dt_w = p.dt_w + cc;
  float total = 0.0f;
  if (rows > 0) settle(0, sp);
  for (int t = 0, b = 0; t < rows; t += kTok, b ^= 1) {
    __syncthreads();  // this step's stage is written, the other one has been read
    const float* now = sp + b * stage;
    float uv[kTok], zv[kTok];
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      uv[j] = to_f32(un[j]);
      zv[j] = to_f32(zn[j]);
    }
    const bool more = t + kTok < rows;
    if (more) {
      request(t + kTok);
      request_uz(t + kTok);
    }
    float2 dt[kTok / 2];
#pragma unroll
    for (int j = 0; j < kTok / 2; ++j) dt[j] = make_float2(bdt, bdt);
#pragma unroll 8
    for (int r = 0; r < dr; ++r) {
      const float w = __ldg(dt_w + static_cast<long long>(r) * p.di);
      const float4 v0 = *reinterpret_cast<const float4*>(now + r * kTok);
      const float4 v1 = *reinterpret_cast<const float4*>(now + r * kTok + 4);
      const float2 w2 = make_float2(w, w);
      dt[0] = __ffma2_rn(make_float2(v0.x, v0.y), w2, dt[0]);
      dt[1] = __ffma2_rn(make_float2(v0.z, v0.w), w2, dt[1]);
      dt[2] = __ffma2_rn(make_float2(v1.x, v1.y), w2, dt[2]);
      dt[3] = __ffma2_rn(make_float2(v1.z, v1.w), w2, dt[3]);
    }
#pragma unroll
    for (int j = 0; j < kTok / 2; ++j) {
      dt[j] = softplus_rel2(dt[j]);
      // rows behind the tile's last leave the state: a step of zero
      if (t + 2 * j >= rows) dt[j].x = 0.0f;
      if (t + 2 * j + 1 >= rows) dt[j].y = 0.0f;
    }
    if (SUMMARY) {
      const float2 sum = __fadd2_rn(__fadd2_rn(dt[0], dt[1]), __fadd2_rn(dt[2], dt[3]));
      total += sum.x + sum.y;
    }
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      const float d = j & 1 ? dt[j / 2].y : dt[j / 2].x;
      const float dtu = d * uv[j];
      const float2 d2 = make_float2(d, d), dtu2 = make_float2(dtu, dtu);
      const float* bc = now + dr * kTok + j * 2 * DS;
      float2 y0 = make_float2(dk * uv[j], 0.0f), y1 = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int n = 0; n < DS / 2; n += 2) {
        const float4 bq = *reinterpret_cast<const float4*>(bc + 2 * n);
        const float2 e0 = __fmul2_rn(d2, an[n]), e1 = __fmul2_rn(d2, an[n + 1]);
        const float2 a0 = n < kPolyPairs<DS> ? exp2_neg2(e0) : make_float2(ex2_approx(e0.x), ex2_approx(e0.y));
        const float2 a1 = n + 1 < kPolyPairs<DS> ? exp2_neg2(e1) : make_float2(ex2_approx(e1.x), ex2_approx(e1.y));
        h[n] = __ffma2_rn(a0, h[n], __fmul2_rn(dtu2, make_float2(bq.x, bq.y)));
        h[n + 1] = __ffma2_rn(a1, h[n + 1], __fmul2_rn(dtu2, make_float2(bq.z, bq.w)));
        if (!SUMMARY) {
          const float4 cq = *reinterpret_cast<const float4*>(bc + DS + 2 * n);
          y0 = __ffma2_rn(h[n], make_float2(cq.x, cq.y), y0);
          y1 = __ffma2_rn(h[n + 1], make_float2(cq.z, cq.w), y1);
        }
      }
      if (!SUMMARY) {
        float yv = (y0.x + y1.x) + (y0.y + y1.y);
        if (z != nullptr) yv *= silu_fast(zv[j]);
        if (on && t + j < rows) y[(t + j) * p.y_ld] = from_f32<T>(yv);
      }
    }
    if (more) settle(t + kTok, sp + (b ^ 1) * stage);
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
// tile's own end: one thread per (channel, state) walks the tiles.
__global__ void __launch_bounds__(128) scan_carry_kernel(const ScanParams p) {
  const int s = blockIdx.x, n = blockIdx.z;
  const Seq q = resolve(p.q, s, false);
  const int c = blockIdx.y * 128 + threadIdx.x;
  if (!q.live || q.len <= p.chunk || c >= p.di) return;
  const int tiles = (q.len + p.chunk - 1) / p.chunk;
  float* ws = p.ws + (q.begin / p.chunk + s) * (1 + p.ds) * p.di + c;
  const float an = p.a[static_cast<long long>(n) * p.di + c] * 1.4426950408889634f;
  float h = p.state == nullptr || q.fresh ? 0.0f : p.state[q.slot * p.slot_stride + static_cast<long long>(n) * p.di + c];
  const long long step = static_cast<long long>(1 + p.ds) * p.di;
  for (int k = 0; k < tiles; ++k, ws += step) {
    float* end = ws + static_cast<long long>(1 + n) * p.di;
    const bool more = k + 1 < tiles;
    const float dt = more ? ws[0] : 0.0f, e = more ? *end : 0.0f;
    *end = h;
    h = fmaf(ex2_approx(dt * an), h, e);
  }
}

// Rows of a tile, a power of two: as many tiles as keep about kFillThreads
// threads (one per channel) on every SM.
constexpr int kMinChunk = 16, kMaxChunk = 2048, kFillThreads = 512;

int scan_chunk(long long rows, int di) {
  const long long want = rows * di / (static_cast<long long>(kFillThreads) * current_sm_count());
  int chunk = kMinChunk;
  while (chunk < kMaxChunk && chunk * 2 <= want) chunk *= 2;
  return chunk;
}

template <typename T, int DS>
int scan_typed(const ScanParams& p, cudaStream_t st) {
  const unsigned cb = static_cast<unsigned>((p.di + 127) / 128);
  const std::size_t row = static_cast<std::size_t>(p.dr + 2 * p.ds) * sizeof(float);
  if (p.q.offsets == nullptr) {
    if (static_cast<long long>(p.q.n_seq) * cb >= 8LL * current_sm_count())
      scan_token_kernel<T, DS, 4><<<dim3(static_cast<unsigned>((p.q.n_seq + 3) / 4), cb), 128, 4 * row, st>>>(p);
    else
      scan_token_kernel<T, DS, 1><<<dim3(static_cast<unsigned>(p.q.n_seq), cb), 128, row, st>>>(p);
    return static_cast<int>(cudaGetLastError());
  }
  const dim3 grid(static_cast<unsigned>(p.q.rows / p.chunk + p.q.n_seq), cb);
  const std::size_t smem = 2 * static_cast<std::size_t>(scan_stage(p.dr, DS)) * sizeof(float);
  if (p.q.rows > p.chunk) {
    scan_prompt_kernel<T, DS, true><<<grid, kScanWarps * 32, smem, st>>>(p);
    scan_carry_kernel<<<dim3(static_cast<unsigned>(p.q.n_seq), cb, static_cast<unsigned>(p.ds)), 128, 0, st>>>(p);
  }
  scan_prompt_kernel<T, DS, false><<<grid, kScanWarps * 32, smem, st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int scan_sized(const ScanParams& p, cudaStream_t st) {
  if (p.ds <= 8) return scan_typed<T, 8>(p, st);
  if (p.ds <= 16) return scan_typed<T, 16>(p, st);
  return scan_typed<T, 32>(p, st);
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
  static int counts[64];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 148;
  if (counts[device] == 0) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || v <= 0) return 148;
    counts[device] = v;
  }
  return counts[device];
}

int launch_causal_conv(const fe_conv_args& a, void* stream) noexcept {
  ConvParams p{sequences(a.offsets, a.slots, a.fresh, a.status, a.rows, a.n_seq, a.n_slots, a.window != nullptr),
               a.x, a.w, a.b, a.u, a.window, a.x_ld, a.u_ld, a.slot_stride, static_cast<int>(a.d_inner),
               static_cast<int>(a.d_conv), 32};
  const auto st = static_cast<cudaStream_t>(stream);
  return with_dtype(a.dtype, [&](auto t) { return conv_typed<decltype(t)>(p, st); });
}

std::size_t selective_scan_workspace(const fe_scan_args& a) noexcept {
  if (a.offsets == nullptr) return 0;
  const int chunk = scan_chunk(static_cast<long long>(a.rows), static_cast<int>(a.d_inner));
  if (a.rows <= static_cast<std::uint64_t>(chunk)) return 0;
  return (a.rows / static_cast<std::uint64_t>(chunk) + a.n_seq) * (1 + a.d_state) * a.d_inner * sizeof(float);
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
  return (tiles + n_seq) * (1 + d_state) * d_inner * sizeof(float);
}

int launch_selective_scan(const fe_scan_args& a, void* stream) noexcept {
  ScanParams p{sequences(a.offsets, a.slots, a.fresh, a.status, a.rows, a.n_seq, a.n_slots, a.state != nullptr),
               a.u, a.proj, a.z, a.a, a.d, a.dt_w, a.dt_b, a.y, a.state, static_cast<float*>(a.workspace),
               a.u_ld, a.proj_ld, a.z_ld, a.y_ld, a.slot_stride, static_cast<int>(a.d_inner),
               static_cast<int>(a.d_state), static_cast<int>(a.dt_rank), 0};
  if (a.offsets != nullptr) p.chunk = scan_chunk(p.q.rows, p.di);
  const auto st = static_cast<cudaStream_t>(stream);
  return with_dtype(a.dtype, [&](auto t) { return scan_sized<decltype(t)>(p, st); });
}

}  // namespace feb
