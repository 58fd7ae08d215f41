// Products of a few rows with 4-bit weights under group scales, and the
// conversions to and from the packed form (include/flowedge_b200.h,
// fe_w4_args).
//
// y = x W^T on the warp's matrix instruction (16 weight rows x 8 rows of x x
// 16 elements of k): its cost does not grow up to 8 rows of x, and the weights'
// whole numbers -8 .. 7 are exact in either 16-bit type, so the products are
// exact and the sums fp32.  A group's sum is scaled when it is complete; no
// weight is ever rounded.  x enters as it is (16-bit types) or as three bf16
// terms that add up to its 24 bits (fp32).
//
// Two layouts of the packed words (FE_W4_BLOCKS, FE_W4_ROWS) differ in what a
// lane reads: a fragment's four lanes must hold words of one group.  In blocks
// a lane's four words, one of each piece of 32 elements, lie side by side.  In
// rows it reads as many side by side as a group has pieces (16, 8 or 4 bytes
// at a time), and the eights of x are staged in the order in which it does.
// One bf16 row x 16384 x 8192: groups of 128 25 us in either, of 64 27 in
// blocks and 30 in rows, of 32 34 and 46.
//
// Bound by the weights' bytes for few rows; a warp reads 16 weight rows x 64
// bytes per block of k, and the blocks are dealt out to several warps where
// there are too few rows of weights to fill the GPU.  16384 x 8192 in groups
// of 128, one bf16 row: 25 us, 0.43 of the measured copy rate (a copy without the
// unpacking took 22 us); 32 rows 78 us.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "convert.cuh"
#include "ops.h"

namespace feb {
namespace {

constexpr int kBlock = 128;  // elements of a packed block of 64 bytes

struct W4Params {
  const void* x;
  const uint32_t* packed;  // [m][words]
  const __half* scales;
  void* y;
  long long x_ld, y_ld;
  int rows, m, k, blocks, groups;
  int words;   // of a row: 16 to a block, or four to every 32 elements (rows)
  int kw;      // warps that share a tile of 16 weight rows, each with part of k
  int stage;   // blocks of x staged in shared memory at a time
};

// D += A B, fp32 accumulators; A 16 x 16 and B 16 x 8 of fp16 or bf16
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight nibbles -> four pairs of exact q - 8.  A nibble under the exponent of
// 2^10 (fp16) or 2^7 (bf16) reads as that power plus q.
template <bool BF16>
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      const uint32_t b = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
      __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&b);
      h = __hsub2(h, __nv_bfloat162(__float2bfloat16_rn(136.0f), __float2bfloat16_rn(136.0f)));
      v[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const uint32_t b = ((w >> (4 * i)) & 0x000F000Fu) | 0x64006400u;
      __half2 h = *reinterpret_cast<const __half2*>(&b);
      h = __hsub2(h, __floats2half2_rn(1032.0f, 1032.0f));
      v[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
}

// Where the eight elements from 8 i on of a block are staged: place 4 j + t for
// those that lane t multiplies with its word j.
template <int GROUP, bool ROWS>
__device__ __forceinline__ int staged_eight(int i) {
  if constexpr (!ROWS || GROUP == 32) return i;
  if constexpr (GROUP == 64) return (i & 8) | (i & 1) << 2 | (i >> 1 & 3);
  return (i & 3) << 2 | i >> 2;
}

// Stages rows r0 .. r0 + n - 1, columns of `blocks` packed blocks from block
// b0 on, as TERMS planes of [n][stride] 16-bit values, the eights of a block in
// their staged order; zero behind column k.
// A warp a row, a lane four columns at a time (16 or 8 bytes where rows start
// on as many), kAhead of those requested together.
template <typename T, int TERMS, int GROUP, bool ROWS>
__device__ __forceinline__ void stage_x(const W4Params& p, int r0, int n, int b0, int blocks, unsigned short* sx, int stride) {
  constexpr int kAhead = 4;
  const auto place = [](int c) { return (c & ~(kBlock - 1)) | staged_eight<GROUP, ROWS>(c >> 3 & 15) << 3 | (c & 7); };
  if constexpr (TERMS == 1) {
    // whole 16 bytes as they are, where rows start on them and k ends there
    if (p.k % 8 == 0 && p.x_ld % 8 == 0 && reinterpret_cast<std::uintptr_t>(p.x) % 16 == 0) {
      const int pieces = blocks * (kBlock / 8);
      for (int i = threadIdx.x; i < n * pieces; i += blockDim.x) {
        const int r = i / pieces, c = (i - r * pieces) * 8;
        const T* src = static_cast<const T*>(p.x) + (r0 + r) * p.x_ld + b0 * kBlock + c;
        *reinterpret_cast<uint4*>(sx + r * stride + place(c)) =
            b0 * kBlock + c < p.k ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
      }
      return;
    }
  }
  struct alignas(4 * sizeof(T)) Four {
    T v[4];
  };
  const int width = blocks * kBlock, first = b0 * kBlock, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const bool whole = p.x_ld % 4 == 0 && reinterpret_cast<std::uintptr_t>(p.x) % sizeof(Four) == 0;
  // (few rows: several warps share one, each with a part of its columns)
  const int share = max(1, warps / n), part = (threadIdx.x >> 5) % share;
  for (int r = (threadIdx.x >> 5) / share; r < n; r += warps / share) {
    const T* src = static_cast<const T*>(p.x) + (r0 + r) * p.x_ld + first;
    const int have = p.k - first;  // columns of x from here on
    for (int c0 = 4 * lane + 128 * part; c0 < width; c0 += 128 * share * kAhead) {
      Four v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int c = c0 + 128 * share * i;
        if (whole && c + 4 <= have) {
          v[i] = *reinterpret_cast<const Four*>(src + c);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i].v[e] = c + e < have ? src[c + e] : from_f32<T>(0.0f);
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int c = c0 + 128 * share * i;
        if (c >= width) break;
        unsigned short* dst = sx + r * stride + place(c);
        if constexpr (TERMS == 1) {
          *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(&v[i]);
        } else {
          // the leading bits as bf16, then the rest's: 8 + 8 + 8 bits, nothing lost (a sum has a NaN's
          // payload in its leading bits, which alone would read as an infinity where they are zero)
          float f[4] = {v[i].v[0] + 0.0f, v[i].v[1] + 0.0f, v[i].v[2] + 0.0f, v[i].v[3] + 0.0f};
#pragma unroll
          for (int t = 0; t < TERMS; ++t) {
            float h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = __uint_as_float(__float_as_uint(f[e]) & 0xFFFF0000u);
            *reinterpret_cast<uint2*>(dst + t * n * stride) =
                make_uint2(__byte_perm(__float_as_uint(h[0]), __float_as_uint(h[1]), 0x7632),
                           __byte_perm(__float_as_uint(h[2]), __float_as_uint(h[3]), 0x7632));
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = isinf(h[e]) ? 0.0f : f[e] - h[e];
          }
        }
      }
    }
  }
}

// 16-bit elements between staged rows: 64 bytes over a multiple of 128, so
// that the eight rows of a fragment fall into different banks
__host__ __device__ constexpr int stage_stride(int blocks) { return blocks * kBlock + 32; }

// A CTA has 4 or 8 warps: p.kw of them share a tile of 16 weight rows, each with
// a run of the blocks of k, and join their sums through shared memory in
// order.  A warp has kSet blocks in its arithmetic and the next kSet on their
// way; a last odd block and one whose last groups or words do not exist come
// one by one.
template <typename T, int NT, int GROUP, bool ROWS>
__global__ void __launch_bounds__(256, 2) w4_matvec_kernel(const W4Params p) {
  constexpr bool kBf16 = !std::is_same_v<T, __half>;
  constexpr int kTerms = std::is_same_v<T, float> ? 3 : 1;
  constexpr int kPer = kBlock / GROUP, kPieces = 4 / kPer;  // groups of a block, 32-element pieces of a group
  constexpr int kSet = NT == 1 ? 2 : 1;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
  const int rw = warps / p.kw, wk = warp % p.kw, wr = warp / p.kw;
  const int m0 = (blockIdx.x * rw + wr) * 16;
  const int r0 = blockIdx.y * NT * 8, n = min(NT * 8, p.rows - r0);
  unsigned short* sx = reinterpret_cast<unsigned short*>(smem);
  const int stride = stage_stride(p.stage);
  // weight rows behind the last read the last one, columns of x behind the
  // last the last one: their sums are not written
  const int ra = min(m0 + g, p.m - 1), rb = min(m0 + g + 8, p.m - 1);
  float acc[NT][4] = {};
  struct Block {
    uint4 a, b;
    __half sa[kPer], sb[kPer];
  };
  for (int b0 = 0; b0 < p.blocks; b0 += p.stage) {
    // this warp's blocks of the stage: [first, end), with all of their groups and words up to `whole`
    const int nb = min(p.stage, p.blocks - b0), share = (nb + p.kw - 1) / p.kw;
    const int first = min(wk * share, nb), end = min(first + share, nb);
    const int whole = max(first, min(end, min(p.groups / kPer, p.words / 16) - b0));
    const uint32_t* wa = p.packed + static_cast<long long>(ra) * p.words + (b0 + first) * 16;
    const uint32_t* wb = p.packed + static_cast<long long>(rb) * p.words + (b0 + first) * 16;
    const __half* sa = p.scales + static_cast<long long>(ra) * p.groups + (b0 + first) * kPer;
    const __half* sb = p.scales + static_cast<long long>(rb) * p.groups + (b0 + first) * kPer;
    // this lane's words of a block of which `words` exist (a multiple of four); the rest are zero weights
    auto words_of = [&](const uint32_t* w, int words) {
      constexpr uint32_t kZero = 0x88888888u;
      if constexpr (!ROWS || GROUP == 128) {
        return !ROWS || 4 * t < words ? __ldg(reinterpret_cast<const uint4*>(w) + t) : make_uint4(kZero, kZero, kZero, kZero);
      } else if constexpr (GROUP == 64) {
        const uint2 none = make_uint2(kZero, kZero), *at = reinterpret_cast<const uint2*>(w) + t;
        const uint2 lo = 2 * t < words ? __ldg(at) : none, hi = 8 + 2 * t < words ? __ldg(at + 4) : none;
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
      } else {
        return make_uint4(__ldg(w + t), 4 < words ? __ldg(w + 4 + t) : kZero, 8 < words ? __ldg(w + 8 + t) : kZero,
                          12 < words ? __ldg(w + 12 + t) : kZero);
      }
    };
    auto request = [&](Block& blk, int i, int groups, int words) {  // block i from the pointers
      blk.a = words_of(wa + i * 16, words);
      blk.b = words_of(wb + i * 16, words);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        blk.sa[j] = j < groups ? sa[i * kPer + j] : __half(0.0f);
        blk.sb[j] = j < groups ? sb[i * kPer + j] : __half(0.0f);
      }
    };
    const unsigned short* xs[NT];
#pragma unroll
    for (int q = 0; q < NT; ++q) xs[q] = sx + min(q * 8 + g, n - 1) * stride + first * kBlock + t * 8;
    auto consume = [&](const Block& blk, int i) {
      const uint32_t ua[4] = {blk.a.x, blk.a.y, blk.a.z, blk.a.w}, ub[4] = {blk.b.x, blk.b.y, blk.b.z, blk.b.w};
      // the leading terms' sums and those of the rest, apart: the latter's
      // roundings are then 2^-8 of the former's
      float part[NT][4], rest[NT][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j % kPieces == 0)
#pragma unroll
          for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[q][e] = rest[q][e] = 0.0f;
        uint32_t va[4], vb[4];
        unpack8<kBf16>(ua[j], va);
        unpack8<kBf16>(ub[j], vb);
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
          for (int term = 0; term < kTerms; ++term) {
            const uint4 xb = *reinterpret_cast<const uint4*>(xs[q] + term * n * stride + i * kBlock + j * 32);
            float(&sum)[4] = term == 0 ? part[q] : rest[q];
            mma_16816<kBf16>(sum, va[0], vb[0], va[1], vb[1], xb.x, xb.y);
            mma_16816<kBf16>(sum, va[2], vb[2], va[3], vb[3], xb.z, xb.w);
          }
        if (j % kPieces == kPieces - 1) {
          const float fa = __half2float(blk.sa[j / kPieces]), fb = __half2float(blk.sb[j / kPieces]);
#pragma unroll
          for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[q][e] = fmaf(e < 2 ? fa : fb, kTerms > 1 ? part[q][e] + rest[q][e] : part[q][e], acc[q][e]);
        }
      }
    };
    auto advance = [&](int blocks) {
      wa += blocks * 16;
      wb += blocks * 16;
      sa += blocks * kPer;
      sb += blocks * kPer;
#pragma unroll
      for (int q = 0; q < NT; ++q) xs[q] += blocks * kBlock;
    };
    Block one[kSet], two[kSet];
    int sets = (whole - first) / kSet;
    if (sets > 0)
#pragma unroll
      for (int i = 0; i < kSet; ++i) request(one[i], i, kPer, 16);
    if (b0 > 0) __syncthreads();
    stage_x<T, kTerms, GROUP, ROWS>(p, r0, n, b0, nb, sx, stride);
    __syncthreads();
    for (; sets > 0; sets -= 2) {
      if (sets > 1)
#pragma unroll
        for (int i = 0; i < kSet; ++i) request(two[i], kSet + i, kPer, 16);
#pragma unroll
      for (int i = 0; i < kSet; ++i) consume(one[i], i);
      if (sets > 2)
#pragma unroll
        for (int i = 0; i < kSet; ++i) request(one[i], 2 * kSet + i, kPer, 16);
      if (sets > 1)
#pragma unroll
        for (int i = 0; i < kSet; ++i) consume(two[i], kSet + i);
      advance(min(sets, 2) * kSet);
    }
    for (int b = first + (whole - first) / kSet * kSet; b < end; ++b) {
      request(one[0], 0, min(kPer, p.groups - (b0 + b) * kPer), min(16, p.words - (b0 + b) * 16));
      consume(one[0], 0);
      advance(1);
    }
  }
  // the warps' parts of k, joined in order: [warp][16][NT * 8 + 1]
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
  constexpr int kCols = NT * 8 + 1;
  float* mine = red + warp * 16 * kCols;
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    mine[g * kCols + q * 8 + 2 * t] = acc[q][0];
    mine[g * kCols + q * 8 + 2 * t + 1] = acc[q][1];
    mine[(g + 8) * kCols + q * 8 + 2 * t] = acc[q][2];
    mine[(g + 8) * kCols + q * 8 + 2 * t + 1] = acc[q][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rw * 16 * n; i += blockDim.x) {
    const int r = i / (rw * 16), o = i - r * (rw * 16);
    const int m = blockIdx.x * rw * 16 + o;
    if (m >= p.m) continue;
    float sum = 0.0f;
    for (int w = 0; w < p.kw; ++w) sum += red[((o >> 4) * p.kw + w) * 16 * kCols + (o & 15) * kCols + r];
    static_cast<T*>(p.y)[(r0 + r) * p.y_ld + m] = from_f32<T>(sum);
  }
}

template <typename T, int NT, int GROUP, bool ROWS>
int matvec_launch(W4Params p, cudaStream_t st) {
  constexpr int kTerms = std::is_same_v<T, float> ? 3 : 1;
  const int n = std::min(p.rows, NT * 8);
  // warps over k until there are about 12 on every SM, of 16 weight rows each;
  // small CTAs, so that all of them are resident and share the SMs evenly.
  // Every CTA stages x; more than 8 rows of 16 bits make that dear: then eight
  // warps, most of them over weight rows, and more of x at a time (16384 x
  // 8192, group 64: 8 fp32 rows 54 us against 86, 16 bf16 rows 56 against 93).
  const int tiles = (p.m + 15) / 16;
  const bool dear = n * kTerms > 8;
  const int fill = dear ? 8 : 12, widest = dear ? 4 : 8, room = (dear ? 96 : 32) * 1024 / (kTerms * n * 2);
  p.kw = 1;
  while (p.kw < widest && p.kw * 2 <= p.blocks && tiles * p.kw < fill * current_sm_count()) p.kw *= 2;
  const int warps = dear ? 8 : std::max(4, p.kw), rw = warps / p.kw;
  p.stage = std::max(1, std::min(p.blocks, (room - 32) / kBlock));
  const std::size_t xs = static_cast<std::size_t>(kTerms) * n * stage_stride(p.stage) * 2;
  const std::size_t rs = static_cast<std::size_t>(warps) * 16 * (NT * 8 + 1) * 4;
  const dim3 grid(static_cast<unsigned>((tiles + rw - 1) / rw), static_cast<unsigned>((p.rows + NT * 8 - 1) / (NT * 8)));
  if (std::max(xs, rs) > 48 * 1024) {
    const cudaError_t rc = cudaFuncSetAttribute(w4_matvec_kernel<T, NT, GROUP, ROWS>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (rc != cudaSuccess) return static_cast<int>(rc);
  }
  w4_matvec_kernel<T, NT, GROUP, ROWS><<<grid, static_cast<unsigned>(warps * 32), std::max(xs, rs), st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int GROUP, bool ROWS>
int matvec_rows(const W4Params& p, cudaStream_t st) {
  if (p.rows <= 8) return matvec_launch<T, 1, GROUP, ROWS>(p, st);
  if (p.rows <= 16) return matvec_launch<T, 2, GROUP, ROWS>(p, st);
  return matvec_launch<T, 4, GROUP, ROWS>(p, st);
}

template <typename T, bool ROWS>
int matvec_group(const W4Params& p, std::uint32_t group, cudaStream_t st) {
  if (group == 32) return matvec_rows<T, 32, ROWS>(p, st);
  if (group == 64) return matvec_rows<T, 64, ROWS>(p, st);
  return matvec_rows<T, 128, ROWS>(p, st);
}

// Place in its row of the word that holds element c.
__device__ __forceinline__ int word_of(int c, bool in_rows) {
  return in_rows ? c / 8 : c / kBlock * 16 + c % 32 / 8 * 4 + c % kBlock / 32;
}

// One warp per group: the scale, then the group's words.
template <typename T>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const T* __restrict__ w, long long ld, int m, int k, int group,
                                                          int groups, int blocks, int words, bool in_rows,
                                                          uint32_t* packed, __half* scales) {
  const int lane = threadIdx.x & 31;
  const long long id = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) >> 5;
  const int per = kBlock / group;
  if (id >= static_cast<long long>(m) * blocks * per) return;  // whole warps
  const int row = static_cast<int>(id / (blocks * per)), grp = static_cast<int>(id - static_cast<long long>(row) * blocks * per);
  const T* src = w + row * ld + static_cast<long long>(grp) * group;
  const int have = min(group, k - grp * group);  // none behind the last group
  float big = 0.0f;
  for (int i = lane; i < have; i += 32) big = fmaxf(big, fabsf(to_f32(src[i])));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
  const __half scale = __float2half_rn(fminf(big / 7.0f, 65504.0f));
  const float s = __half2float(scale);
  if (lane == 0 && grp < groups) scales[static_cast<long long>(row) * groups + grp] = scale;
  // word i of the group holds its elements 8 i .. 8 i + 7
  if (lane < group / 8) {
    uint32_t word = 0;
    for (int e = 0; e < 8; ++e) {
      int q = 8;
      if (lane * 8 + e < have && s > 0.0f) {
        const float v = fminf(fmaxf(rintf(to_f32(src[lane * 8 + e]) / s), -8.0f), 7.0f);
        q = static_cast<int>(v) + 8;
      }
      word |= static_cast<uint32_t>(q) << (4 * ((e >> 1) + (e & 1) * 4));
    }
    const int at = word_of(grp * group + lane * 8, in_rows);
    if (at < words) packed[static_cast<long long>(row) * words + at] = word;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(const uint32_t* __restrict__ packed,
                                                            const __half* __restrict__ scales, int m, int k, int group,
                                                            int groups, int words, bool in_rows, T* w, long long ld) {
  const long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  if (i >= static_cast<long long>(m) * k) return;
  const int row = static_cast<int>(i / k), c = static_cast<int>(i - static_cast<long long>(row) * k);
  const int e = c % 8;
  const uint32_t word = packed[static_cast<long long>(row) * words + word_of(c, in_rows)];
  const int q = static_cast<int>(word >> (4 * ((e >> 1) + (e & 1) * 4)) & 15u) - 8;
  w[row * ld + c] = from_f32<T>(static_cast<float>(q) * __half2float(scales[static_cast<long long>(row) * groups + c / group]));
}

int blocks_of(const fe_w4_args& a) { return static_cast<int>((a.k + kBlock - 1) / kBlock); }
int words_of(const fe_w4_args& a) {
  return a.layout == FE_W4_ROWS ? static_cast<int>((a.k + 31) / 32 * 4) : blocks_of(a) * 16;
}
int groups_of(const fe_w4_args& a) { return static_cast<int>((a.k + a.group - 1) / a.group); }

}  // namespace

int launch_w4_matvec(const fe_w4_args& a, void* stream) noexcept {
  const W4Params p{a.x, static_cast<const uint32_t*>(a.packed), static_cast<const __half*>(a.scales), a.y, a.x_ld, a.y_ld,
                   static_cast<int>(a.rows), static_cast<int>(a.m), static_cast<int>(a.k), blocks_of(a), groups_of(a),
                   words_of(a), 1, 1};
  const auto st = static_cast<cudaStream_t>(stream);
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.layout == FE_W4_ROWS ? matvec_group<T, true>(p, a.group, st) : matvec_group<T, false>(p, a.group, st);
  });
}

int launch_w4_quantize(const fe_w4_args& a, void* stream) noexcept {
  const long long warps = static_cast<long long>(a.m) * blocks_of(a) * (kBlock / static_cast<int>(a.group));
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    w4_quantize_kernel<T><<<static_cast<unsigned>((warps + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(a.x), a.x_ld, static_cast<int>(a.m), static_cast<int>(a.k), static_cast<int>(a.group),
        groups_of(a), blocks_of(a), words_of(a), a.layout == FE_W4_ROWS, static_cast<uint32_t*>(a.packed),
        static_cast<__half*>(a.scales));
    return static_cast<int>(cudaGetLastError());
  });
}

int launch_w4_dequantize(const fe_w4_args& a, void* stream) noexcept {
  const long long total = static_cast<long long>(a.m) * static_cast<long long>(a.k);
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    w4_dequantize_kernel<T><<<static_cast<unsigned>((total + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint32_t*>(a.packed), static_cast<const __half*>(a.scales), static_cast<int>(a.m),
        static_cast<int>(a.k), static_cast<int>(a.group), groups_of(a), words_of(a), a.layout == FE_W4_ROWS, static_cast<T*>(a.y),
        a.y_ld);
    return static_cast<int>(cudaGetLastError());
  });
}

}  // namespace feb
