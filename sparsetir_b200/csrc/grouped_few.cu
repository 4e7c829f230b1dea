// Grouped products for groups of a few rows (a decoding step) of few features: what costs is reading the weights once.  The pairs
// of blocks of grouped.cu set up tensor memory, barriers and a ring for tiles of 256 features, and a few such tiles leave
// most of the memory system idle; here the weights go straight from global memory into the registers of the matrix instructions
// (m16n8k16, m16n8k32 for 8-bit integers: 16 features, 8 rows of x), by as many warps as it takes to keep it busy: the
// warps of a block share its features and, where these are few, the depth, and their sums meet in shared memory in a fixed order.
// Which element of a step of K plays which k is free as long as both operands agree, so every lane loads 16 (8) bytes of W.
// One row of 8-bit integers, 4096 -> 8192: 33.6 MB in 8.2 us out of HBM, 5.0 out of L2; prefetch sizes of 128 and 256 bytes at the
// loads changed nothing and cost up to a third.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gate.cuh"
#include "grouped.h"
#include "launch.cuh"
#include "lowp.cuh"

namespace sptir {
namespace {

constexpr int kMaxWarps = 16;

// d += a * b for operands of type T
template <class T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_fp8_e4m3>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                   uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <class T>
__device__ __forceinline__ void mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <class T> struct SumOf { using type = float; };
template <> struct SumOf<int8_t> { using type = int; };

// 16 or 8 bytes, or zeros; behind chain_wait() like ld_global
__device__ __forceinline__ void load_if(uint4& v, const char* p, bool in) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"(static_cast<int>(in)));
}
__device__ __forceinline__ void load_if(uint2& v, const char* p, bool in) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t"
      "@p ld.global.v2.b32 {%0, %1}, [%2];\n\t}"
      : "=&r"(v.x), "=&r"(v.y)
      : "l"(p), "r"(static_cast<int>(in)));
}

// W contiguous along K.  A step is 64 bytes of K of 32 features and 8 NT rows: lane l has 16 bytes, at 16 (l % 4), of
// features l / 4 + 8 i and of rows l / 4 + 8 h; registers 0, 1 of them make one instruction, 2, 3 another.
// Gated: the 32 are 16 of the gate (i = 0, 1) and the same 16 of the other projection.
template <class T, int NT, bool GATED = false>
struct AlongK {
  static constexpr int kFeatures = 32, kStepBytes = 64, kRows = 8 * NT;
  static constexpr bool kGated = GATED;
  using Args = std::conditional_t<GATED, FewGatedArgs, FewArgs>;
  using Sum = typename SumOf<T>::type;
  Sum acc[2][NT][4];
  struct Step { uint4 w[4], x[NT]; };

  // Features and rows that are not there take the place of one that is: their sums go nowhere.
  const char *wp[4], *xp[NT];
  int at, bytes;  // of K
  __device__ __forceinline__ void start(const FewArgs& p, int group, int feat0, int row0, int live, int k0, int k1, int lane) {
    at = k0 + 16 * (lane & 3);
    bytes = k1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = feat0 + lane / 4 + 8 * (GATED ? i & 1 : i);
      size_t r = static_cast<size_t>(group) * (GATED ? 2 : 1) * p.fo + min(f, p.fo - 1);
      if (GATED && i >= 2) r += p.fo;
      wp[i] = static_cast<const char*>(p.w) + r * p.w_pitch + at;
    }
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      xp[h] = static_cast<const char*>(p.x) + static_cast<size_t>(row0 + min(lane / 4 + 8 * h, live - 1)) * p.x_pitch + at;
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[0][h][c] = acc[1][h][c] = 0;
    }
  }
  __device__ __forceinline__ void load(Step& s) {
    const bool in = at < bytes;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      load_if(s.w[i], wp[i], in);
      wp[i] += kStepBytes;
    }
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      load_if(s.x[h], xp[h], in);
      xp[h] += kStepBytes;
    }
    at += kStepBytes;
  }
  __device__ __forceinline__ void multiply(const Step& s) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        mma<T>(acc[m][h], s.w[2 * m].x, s.w[2 * m + 1].x, s.w[2 * m].y, s.w[2 * m + 1].y, s.x[h].x, s.x[h].y);
        mma<T>(acc[m][h], s.w[2 * m].z, s.w[2 * m + 1].z, s.w[2 * m].w, s.w[2 * m + 1].w, s.x[h].z, s.x[h].w);
      }
  }
  __device__ __forceinline__ void put(Sum (*to)[kFeatures], int lane) const {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) to[8 * h + 2 * (lane & 3) + (c & 1)][16 * m + lane / 4 + 8 * (c >> 1)] = acc[m][h][c];
  }
};

// The same for 8-bit floating point: the sums of a step, half of a block of K that shares scales, are scaled and added to those of the steps
// before it.  The scales of a block's rows of x and W, for all of the depth, are in shared memory: in registers with the steps
// ahead they were spilled (48 rows, 8 groups, 1024 -> 2 x 2048, weights in L2: 17.2 us where now 8.6).  With 16 rows at a time 52 bytes of a
// thread's registers are spilled all the same, 72 in the gated form.
template <int NT, bool GATED>
struct Scaled : AlongK<__nv_fp8_e4m3, NT, GATED> {
  using Base = AlongK<__nv_fp8_e4m3, NT, GATED>;
  static constexpr int kW = GATED ? 3 : 1;  // of W: gated: the gate's, and two of the other projection's, whose rows may lie in two blocks
  float sum[2][NT][4];
  const float *xs, *ws;  // of the lane's rows: [blocks][kRows]; of the warp's features: [blocks][kW]
  int at;                // of K, of the next step to be multiplied
  __device__ __forceinline__ static int blocks(const FewArgs& p) { return (p.fi + SPARSETIR_F8_BLOCK - 1) / SPARSETIR_F8_BLOCK; }
  static size_t scale_bytes(const FewArgs& p) {
    return static_cast<size_t>((p.fi + SPARSETIR_F8_BLOCK - 1) / SPARSETIR_F8_BLOCK) * (Base::kRows + p.feature_warps * kW) * sizeof(float);
  }
  // By all threads of a block, into `to`; a barrier follows.
  __device__ __forceinline__ static void stage(const FewArgs& p, float* to, int group, int block_feat0, int row0, int live, int tid, int threads) {
    const int n = blocks(p);
    for (int i = tid; i < n * Base::kRows; i += threads) {
      const int b = i / Base::kRows, r = i % Base::kRows;
      to[i] = r < live ? ld_global(p.x_scale + static_cast<size_t>(b) * p.rows + row0 + r) : 0.f;
    }
    to += n * Base::kRows;
    const int of_w = ((GATED ? 2 : 1) * p.fo + SPARSETIR_F8_BLOCK - 1) / SPARSETIR_F8_BLOCK;
    for (int i = tid; i < n * p.feature_warps * kW; i += threads) {
      const int j = i % kW, b = i / kW % n, fw = i / kW / n;
      int f = block_feat0 + fw * (GATED ? 16 : 32) + (j == 2 ? 15 : 0);
      f = (j > 0 ? p.fo : 0) + min(f, p.fo - 1);
      to[i] = ld_global(p.w_scale + (static_cast<size_t>(group) * of_w + f / SPARSETIR_F8_BLOCK) * n + b);
    }
  }
  bool second[2];  // gated: the lane's features lane / 4, and 8 further on, have the other projection's second scale
  __device__ __forceinline__ void scales(const FewArgs& p, const float* from, int fw, int feat0, int k0, int lane) {
    const int n = blocks(p);
    xs = from + 2 * (lane & 3);
    ws = from + n * Base::kRows + fw * n * kW;
    at = k0;
    const int first = (p.fo + min(feat0, p.fo - 1)) / SPARSETIR_F8_BLOCK;
#pragma unroll
    for (int c = 0; c < 2; ++c) second[c] = GATED && (p.fo + min(feat0 + lane / 4 + 8 * c, p.fo - 1)) / SPARSETIR_F8_BLOCK != first;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[m][h][c] = 0.f;
  }
  __device__ __forceinline__ void multiply(const typename Base::Step& s) {
    if (at >= this->bytes) return;
    Base::multiply(s);
    const int b = at / SPARSETIR_F8_BLOCK;
    at += Base::kStepBytes;
    const float* const w = ws + b * kW;
    const float w0 = w[0], u0 = GATED ? (second[0] ? w[2] : w[1]) : w0, u1 = GATED ? (second[1] ? w[2] : w[1]) : w0;
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      const float2 x = *reinterpret_cast<const float2*>(xs + b * Base::kRows + 8 * h);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float by = (c & 1) == 0 ? x.x : x.y;
          sum[m][h][c] = fmaf(this->acc[m][h][c], by * (m == 0 ? w0 : c < 2 ? u0 : u1), sum[m][h][c]);
          this->acc[m][h][c] = 0.f;
        }
    }
  }
  __device__ __forceinline__ void put(float (*to)[Base::kFeatures], int lane) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) this->acc[m][h][c] = sum[m][h][c];
    Base::put(to, lane);
  }
};
template <class Operand> struct IsScaled { static constexpr bool value = false; };
template <int NT, bool GATED> struct IsScaled<Scaled<NT, GATED>> { static constexpr bool value = true; };

// W contiguous along the features (16-bit elements).  A step is 32 of K of 32 features: lane l has 4 features from 4 (l / 4) on of the
// eight rows of W from 8 (l % 4) on, and eight elements of its rows of x; instruction j takes the j-th and the (j + 2)-th
// feature of every lane's four, four rows at a time.  (With 8 features to a lane, 64 to a warp, there are half as many
// warps: 1 row, 4096 -> 2000 12.6 us where now 7.9, 64 rows in 8 groups, 1024 -> 1024 8.1 where now 6.4; along K 5.0 and 4.8.)
template <class T, int NT>
struct AlongFeatures {
  static constexpr int kFeatures = 32, kStepBytes = 64, kRows = 8 * NT;  // bytes of K in x
  static constexpr bool kGated = false;
  using Args = FewArgs;
  using Sum = float;
  float acc[2][NT][4];
  struct Step { uint2 w[8]; uint4 x[NT]; };

  const char *wp, *xp[NT];
  int at, last;  // elements of K
  size_t pitch;
  __device__ __forceinline__ void start(const FewArgs& p, int group, int feat0, int row0, int live, int k0, int k1, int lane) {
    const int f = feat0 + 4 * (lane / 4);
    pitch = p.w_pitch;
    at = k0 / 2 + 8 * (lane & 3);
    last = k1 / 2;
    wp = static_cast<const char*>(p.w) + (static_cast<size_t>(group) * p.fi + at) * pitch + static_cast<size_t>(f < p.fo ? f : 0) * 2;
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      xp[h] = static_cast<const char*>(p.x) + static_cast<size_t>(row0 + min(lane / 4 + 8 * h, live - 1)) * p.x_pitch + static_cast<size_t>(at) * 2;
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[0][h][c] = acc[1][h][c] = 0.f;
    }
  }
  __device__ __forceinline__ void load(Step& s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) load_if(s.w[i], wp + i * pitch, at + i < last);
    wp += 32 * pitch;
#pragma unroll
    for (int h = 0; h < NT; ++h) {  // a row of x that does not end at a multiple of eight elements is followed by zeros
      load_if(s.x[h], xp[h], at < last);
      xp[h] += 64;
    }
    at += 32;
  }
  __device__ __forceinline__ void multiply(const Step& s) {
    // words of four rows that hold the lane's features 0 and 1 (lo), and 2 and 3 (hi)
    auto two = [&](const uint2& r0, const uint2& r1, const uint2& r2, const uint2& r3, int h, uint32_t x0, uint32_t x1) {
      mma<T>(acc[0][h], __byte_perm(r0.x, r1.x, 0x5410), __byte_perm(r0.y, r1.y, 0x5410), __byte_perm(r2.x, r3.x, 0x5410),
             __byte_perm(r2.y, r3.y, 0x5410), x0, x1);
      mma<T>(acc[1][h], __byte_perm(r0.x, r1.x, 0x7632), __byte_perm(r0.y, r1.y, 0x7632), __byte_perm(r2.x, r3.x, 0x7632),
             __byte_perm(r2.y, r3.y, 0x7632), x0, x1);
    };
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      two(s.w[0], s.w[1], s.w[2], s.w[3], h, s.x[h].x, s.x[h].y);
      two(s.w[4], s.w[5], s.w[6], s.w[7], h, s.x[h].z, s.x[h].w);
    }
  }
  __device__ __forceinline__ void put(float (*to)[kFeatures], int lane) const {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) to[8 * h + 2 * (lane & 3) + (c & 1)][4 * (lane / 4) + j + 2 * (c >> 1)] = acc[j][h][c];
  }
};

// Block = (rows, features); `splits` of its warps share the depth of the same features.  Blocks y < groups have the first kRows rows
// of group y; one more block for every further kRows rows of the operand has what lies in them of the rest of a group: of
// the one that their first row belongs to, since the rest of a group that begins among them lies behind them.  They come last and
// find the weights in L2.  With a group's rows walked by its own few blocks, a batch that met in a few groups waited for
// these (256 rows, 64 groups, 2048 -> 1024, W along the depth, us, spread evenly / a quarter in one group / all in one:
// 50 / 175 / 437, this way 50 / 50 / 28; the kernel of grouped.cu 47 / 46 / 15).
template <class Operand, class OutT>
__global__ void __launch_bounds__(32 * kMaxWarps, 1) few_rows_kernel(const __grid_constant__ typename Operand::Args p) {
  using Sum = typename Operand::Sum;
  constexpr int F = Operand::kFeatures, kRows = Operand::kRows;
  constexpr int O = Operand::kGated ? F / 2 : F;  // features of the result to a warp
  extern __shared__ __align__(16) unsigned char smem[];
  Sum(*const part)[kRows][F] = reinterpret_cast<Sum(*)[kRows][F]>(smem);  // of every warp
  chain_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int group = blockIdx.y, from = 0;
  const bool rest = group >= p.groups;
  if (__builtin_expect(rest, 0)) {
    from = (group - p.groups + 1) * kRows;
    group = p.indptr != nullptr ? group_of_row(p.indptr, p.groups, from, lane) : 0;
  }
  int row0 = 0, end = p.rows;
  if (p.indptr != nullptr) {
    row0 = min(max(ld_global(p.indptr + group), 0), p.rows);
    end = min(ld_global(p.indptr + group + 1), p.rows);
  }
  if (rest) row0 = max(row0 + kRows, from);
  end = min(end, (rest ? from : row0) + kRows);
  const int fw = warp / p.splits, ks = warp - fw * p.splits;
  const int block_feats = p.feature_warps * O;
  const int block_feat0 = blockIdx.x * block_feats;
  const int k0 = ks * p.split_bytes, k1 = min(k0 + p.split_bytes, p.k_bytes);
  // Once.  Without the loop the compiler moves what is behind the steps ahead of them and spills 70 bytes of registers (one row,
  // 4096 -> 8192 in 8 bits, quantised: 10.0 us where now 8.7).
  for (; row0 < end; row0 += kRows) {
    const int live = end - row0;
    Operand op;
    op.start(p, group, block_feat0 + fw * O, row0, live, k0, k1, lane);
    const int steps = (k1 - k0 + Operand::kStepBytes - 1) / Operand::kStepBytes;  // <= 0: nothing of the depth left
    // two or three steps requested ahead of the one that is multiplied
    typename Operand::Step a, b, c;
    op.load(a);
    op.load(b);
    if constexpr (IsScaled<Operand>::value) {
      float* const scales = reinterpret_cast<float*>(smem) + (blockDim.x >> 5) * (kRows * F);
      Operand::stage(p, scales, group, block_feat0, row0, live, tid, static_cast<int>(blockDim.x));
      __syncthreads();
      op.scales(p, scales, fw, block_feat0 + fw * O, k0, lane);
    }
    for (int s = 0; s < steps; s += 3) {
      op.load(c);
      op.multiply(a);
      op.load(a);
      op.multiply(b);
      op.load(b);
      op.multiply(c);
    }
    op.put(part[warp], lane);
    __syncthreads();
    for (int i = tid; i < block_feats * live; i += static_cast<int>(blockDim.x)) {
      const int r = i / block_feats, f = i - r * block_feats;
      const int feat = block_feat0 + f;
      if (feat >= p.fo) continue;
      Sum sum = 0;
      for (int q = 0; q < p.splits; ++q) sum += part[f / O * p.splits + q][r][f % O];
      if constexpr (Operand::kGated) {
        float up = 0.f;
        for (int q = 0; q < p.splits; ++q) up += part[f / O * p.splits + q][r][O + f % O];
        static_cast<OutT*>(p.y)[static_cast<size_t>(row0 + r) * p.fo + feat] = from_float<OutT>(p.gate.act(sum, up));
        if (p.hidden != nullptr) {
          OutT* const h = static_cast<OutT*>(p.hidden) + static_cast<size_t>(row0 + r) * 2 * p.fo + feat;
          h[0] = from_float<OutT>(sum);
          h[p.fo] = from_float<OutT>(up);
        }
        continue;
      }
      float v = static_cast<float>(sum);
      if constexpr (std::is_same<Sum, int>::value)
        v *= ld_global(p.x_scale + row0 + r) * ld_global(p.w_scale + static_cast<size_t>(group) * p.fo + feat);
      static_cast<OutT*>(p.y)[static_cast<size_t>(row0 + r) * p.fo + feat] = from_float<OutT>(v);
    }
    __syncthreads();
  }
}

template <class Operand, class OutT>
int launch(typename Operand::Args p, cudaStream_t st) {
  // as many warps as keep the memory busy: the depth is split where the features of the groups are too few, into parts of four
  // steps at least.  Eight warps to a block, fewer where blocks would not be found on every SM.
  const int used = std::min(p.groups, p.rows);
  constexpr int O = Operand::kGated ? Operand::kFeatures / 2 : Operand::kFeatures;
  const long long warps = static_cast<long long>(ceil_div(p.fo, O)) * used;
  int splits = 1;
  while (splits < kMaxWarps && 2 * warps * splits <= kNumSMs * kMaxWarps && p.k_bytes / splits > 4 * Operand::kStepBytes) splits *= 2;
  p.feature_warps = std::max(1, 8 / splits);
  while (p.feature_warps > 1 && warps / p.feature_warps < kNumSMs) p.feature_warps /= 2;
  p.splits = splits;
  p.split_bytes = (ceil_div(p.k_bytes, splits) + 127) / 128 * 128;
  const dim3 grid(ceil_div(p.fo, p.feature_warps * O), p.groups + (p.rows - 1) / Operand::kRows);
  const int block_warps = p.feature_warps * splits;
  int smem = block_warps * Operand::kRows * Operand::kFeatures * 4, most = kMaxWarps * Operand::kRows * Operand::kFeatures * 4;
  if constexpr (IsScaled<Operand>::value) {
    smem += static_cast<int>(Operand::scale_bytes(p));
    most += kFewF8Depth / SPARSETIR_F8_BLOCK * (Operand::kRows + 8 * 3) * 4;
  }
  static thread_local int configured_device = -1;
  int dev = 0;
  SPTIR_CUDA_OK(cudaGetDevice(&dev));
  if (configured_device != dev) {
    SPTIR_CUDA_OK(cudaFuncSetAttribute(few_rows_kernel<Operand, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       most));
    configured_device = dev;
  }
  launch_chained(few_rows_kernel<Operand, OutT>, grid, 32 * block_warps, smem, st, p);
  SPTIR_LAUNCH_OK("few_rows_kernel");
  return 0;
}

template <class T, int NT, class OutT>
int launch_layout(const FewArgs& p, bool along_k, cudaStream_t st) {
  if constexpr (!std::is_same<T, int8_t>::value)
    if (!along_k) return launch<AlongFeatures<T, NT>, OutT>(p, st);
  return launch<AlongK<T, NT>, OutT>(p, st);
}

// f(integral constant NT): 8 rows at a time, up to `each` rows to a group, or 16
template <class F>
int with_rows(const FewArgs& p, int each, F&& f) {
  if (p.rows <= static_cast<long long>(each) * std::min(p.groups, p.rows)) return f(std::integral_constant<int, 1>{});
  return f(std::integral_constant<int, 2>{});
}
// Of the gated products and those of 8-bit floating point.  Us, weights out of HBM, 8 rows at a time / 16.  Even groups: 8 groups of 4, 6 and 8
// rows, 1024 -> 2 x 2048 14.0 / 13.9, 14.5 / 14.5, 14.6 / 14.6, in 8 bits 10.3 / 12.3, 10.8 / 12.8, 10.9 / 12.9; one group of 10 rows, 4096 -> 2 x 4096
// 20.1 / 14.0, 4096 -> 8192 in 8 bits 15.8 / 12.3: beyond 8 rows the weights are read again.  So they are for the larger ones of ragged groups: 40
// and 64 rows over 8 groups, the same sizes, 18.7 / 14.5 and 20.3 / 15.0, in 8 bits 10.8 / 13.2 and 16.5 / 13.2.
constexpr int kRowsEach = 6;

template <class T>
int launch_type(const FewArgs& p, int y_type, bool along_k, cudaStream_t st) {
  return with_type(y_type, [&](auto o) {
    using O = decltype(o);
    return with_rows(p, 4, [&](auto nt) { return launch_layout<T, nt.value, O>(p, along_k, st); });
  });
}

}  // namespace

int few_rows(const FewArgs& p, int type, int y_type, bool along_k, cudaStream_t st) {
  if (type < 0) return launch_type<int8_t>(p, y_type, along_k, st);
  if (type == SPARSETIR_F16) return launch_type<__half>(p, y_type, along_k, st);
  return launch_type<__nv_bfloat16>(p, y_type, along_k, st);
}

int few_rows_gated(const FewGatedArgs& p, int type, cudaStream_t st) {
  return with_rows(p, kRowsEach, [&](auto nt) {
    if (type == SPARSETIR_F16) return launch<AlongK<__half, nt.value, true>, __half>(p, st);
    return launch<AlongK<__nv_bfloat16, nt.value, true>, __nv_bfloat16>(p, st);
  });
}

int few_rows_f8(const FewGatedArgs& p, int y_type, bool gated, cudaStream_t st) {
  return with_rows(p, kRowsEach, [&](auto nt) {
    return with_type(y_type, [&](auto o) {
      using O = decltype(o);
      if constexpr (!std::is_same<O, float>::value)
        if (gated) return launch<Scaled<nt.value, true>, O>(p, st);
      return launch<Scaled<nt.value, false>, O>(p, st);
    });
  });
}

}  // namespace sptir
