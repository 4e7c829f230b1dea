// Grouped products for groups of a few rows (a decoding step) of few features: what costs is reading the weights once.  The pairs
// of blocks of grouped.cu set up tensor memory, barriers and a ring for tiles of 256 features, and a few such tiles leave
// most of the memory system idle; here the weights go straight from global memory into the registers of the matrix instructions
// (m16n8k16, m16n8k32 for 8-bit integers: 16 features, 8 rows of x), by as many warps as it takes to keep it busy: the
// warps of a block share its features and, where these are few, the depth, and their sums meet in shared memory in a fixed order.
// Which element of a step of K plays which k is free as long as both operands agree, so every lane loads 16 (8) bytes of W.
// One row of 8-bit integers, 4096 -> 8192: 33.6 MB in 8.2 us out of HBM, 5.0 out of L2; prefetch sizes of 128 and 256 bytes at the
// loads changed nothing and cost up to a third.
#include <algorithm>
#include <type_traits>

#include "common.h"
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
template <class T, int NT>
struct AlongK {
  static constexpr int kFeatures = 32, kStepBytes = 64, kRows = 8 * NT;
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
      const int f = feat0 + lane / 4 + 8 * i;
      wp[i] = static_cast<const char*>(p.w) + (static_cast<size_t>(group) * p.fo + min(f, p.fo - 1)) * p.w_pitch + at;
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

// W contiguous along the features (16-bit elements).  A step is 32 of K of 32 features: lane l has 4 features from 4 (l / 4) on of the
// eight rows of W from 8 (l % 4) on, and eight elements of its rows of x; instruction j takes the j-th and the (j + 2)-th
// feature of every lane's four, four rows at a time.  (With 8 features to a lane, 64 to a warp, there are half as many
// warps: 1 row, 4096 -> 2000 12.6 us where now 7.9, 64 rows in 8 groups, 1024 -> 1024 8.1 where now 6.4; along K 5.0 and 4.8.)
template <class T, int NT>
struct AlongFeatures {
  static constexpr int kFeatures = 32, kStepBytes = 64, kRows = 8 * NT;  // bytes of K in x
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
__global__ void __launch_bounds__(32 * kMaxWarps, 1) few_rows_kernel(const __grid_constant__ FewArgs p) {
  using Sum = typename Operand::Sum;
  constexpr int F = Operand::kFeatures, kRows = Operand::kRows;
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
  const int block_feats = p.feature_warps * F;
  const int block_feat0 = blockIdx.x * block_feats;
  const int k0 = ks * p.split_bytes, k1 = min(k0 + p.split_bytes, p.k_bytes);
  // Once.  Without the loop the compiler moves what is behind the steps ahead of them and spills 70 bytes of registers (one row,
  // 4096 -> 8192 in 8 bits, quantised: 10.0 us where now 8.7).
  for (; row0 < end; row0 += kRows) {
    const int live = end - row0;
    Operand op;
    op.start(p, group, block_feat0 + fw * F, row0, live, k0, k1, lane);
    const int steps = (k1 - k0 + Operand::kStepBytes - 1) / Operand::kStepBytes;  // <= 0: nothing of the depth left
    // two or three steps requested ahead of the one that is multiplied
    typename Operand::Step a, b, c;
    op.load(a);
    op.load(b);
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
      for (int q = 0; q < p.splits; ++q) sum += part[f / F * p.splits + q][r][f % F];
      float v = static_cast<float>(sum);
      if constexpr (std::is_same<Sum, int>::value)
        v *= ld_global(p.x_scale + row0 + r) * ld_global(p.w_scale + static_cast<size_t>(group) * p.fo + feat);
      static_cast<OutT*>(p.y)[static_cast<size_t>(row0 + r) * p.fo + feat] = from_float<OutT>(v);
    }
    __syncthreads();
  }
}

template <class Operand, class OutT>
int launch(FewArgs p, cudaStream_t st) {
  // as many warps as keep the memory busy: the depth is split where the features of the groups are too few, into parts of four
  // steps at least.  Eight warps to a block, fewer where blocks would not be found on every SM.
  const int used = std::min(p.groups, p.rows);
  const long long warps = static_cast<long long>(ceil_div(p.fo, Operand::kFeatures)) * used;
  int splits = 1;
  while (splits < kMaxWarps && 2 * warps * splits <= kNumSMs * kMaxWarps && p.k_bytes / splits > 4 * Operand::kStepBytes) splits *= 2;
  p.feature_warps = std::max(1, 8 / splits);
  while (p.feature_warps > 1 && warps / p.feature_warps < kNumSMs) p.feature_warps /= 2;
  p.splits = splits;
  p.split_bytes = (ceil_div(p.k_bytes, splits) + 127) / 128 * 128;
  const dim3 grid(ceil_div(p.fo, p.feature_warps * Operand::kFeatures), p.groups + (p.rows - 1) / Operand::kRows);
  const int block_warps = p.feature_warps * splits, smem = block_warps * Operand::kRows * Operand::kFeatures * 4;
  static thread_local int configured_device = -1;
  int dev = 0;
  SPTIR_CUDA_OK(cudaGetDevice(&dev));
  if (configured_device != dev) {
    SPTIR_CUDA_OK(cudaFuncSetAttribute(few_rows_kernel<Operand, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kMaxWarps * Operand::kRows * Operand::kFeatures * 4));
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

template <class T>
int launch_type(const FewArgs& p, int y_type, bool along_k, cudaStream_t st) {
  const bool eight = p.rows <= 4ll * std::min(p.groups, p.rows);
  return with_type(y_type, [&](auto o) {
    using O = decltype(o);
    return eight ? launch_layout<T, 1, O>(p, along_k, st) : launch_layout<T, 2, O>(p, along_k, st);
  });
}

}  // namespace

int few_rows(const FewArgs& p, int type, int y_type, bool along_k, cudaStream_t st) {
  if (type < 0) return launch_type<int8_t>(p, y_type, along_k, st);
  if (type == SPARSETIR_F16) return launch_type<__half>(p, y_type, along_k, st);
  return launch_type<__nv_bfloat16>(p, y_type, along_k, st);
}

}  // namespace sptir
