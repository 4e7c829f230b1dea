// Products of 8-bit floating point (e4m3) grouped by expert, with a scale for each 128 of a row of x and for each 128 x 128 of W, and the gated
// block of such operands, on the tensor cores.
//
// A tile is 128 rows of a group x 256 rows of W (256 features, or 128 of a gated block), one to a block of threads, the rows of x as the
// left operand.  A stage of the ring is 128 of K, what shares scales, so that its sums stand by themselves in one of two accumulators, which change by
// turns; eight warps add them, scaled, to 128 sums in each lane's registers while the tensor core fills the other.  A lane's sums are
// of one row and, but for a gated block's other projection, of one block of W: they share one scale, and nothing but TMEM is read between
// one step and the next.
//
// What bounds it is the way there and back: from the issue of a step's MMAs (512 clocks) to their sums in registers, to take them (350 clocks) and
// until the issuing thread knows, with two accumulators on the way.  Of the 2,100 clocks of that round trip some 570 are not accounted for.
// Us, 65,536 rows in 64 equal groups, 2048 -> 2048, by pairs of blocks on
// 256 rows: with the features as the left operand and the rows' scales out of shared memory 512 to 566, rows as the left operand 367, with
// the loads of TMEM in flight across the steps 328, with waits that ask again and again 310 to 320.  This kernel, without another block to wait for,
// takes 331, and 562 for 8192^3 where the pairs took 513; it wastes less on ragged groups and reads weights for few rows as well as tiles of
// their own did (us, calls in a row of two sets of inputs, pairs / this: 8,192
// rows to eight of 64 ragged groups with their quantisation 391 / 382, 4,096 to four of 32 120 / 107, gated 230 / 192; 4,096 rows in 64 groups, 2048 ->
// 2048 71 / 60, 6,400 rows 1024 -> 1024 28 / 19, 500 rows 2048 -> 2048 56 / 56: 268 MB of weights).  The gated form spills 76 bytes of a thread's
// registers.
// 8-bit integers, which are scaled at the end alone, take 228 where this takes 331.
#define SPARSETIR_GROUPED_KERNEL_ONLY
#include "grouped.cu"

namespace sptir {
namespace {

constexpr int kXBytes = 16 * 1024;                // of a stage: 128 rows of x
constexpr int kF8Bytes = kXBytes + 32 * 1024;     // and 256 of W
constexpr int kF8Stages = 4;
constexpr int kF8Threads = (kFirstEpilogue + 8) * 32;
constexpr int kF8Smem = kF8Stages * kF8Bytes + 8 * kStagedBytes + 1024;
// Registers of a thread: one of the epilogue holds 128 sums, the others need few.  What the block was launched with is shared out again:
// 128 * 40 + 256 * 232 = 384 * 168.
constexpr int kF8Others = 40, kF8Epilogue = 232;

// An epilogue warp's share of a tile: 32 rows, 128 columns; gated: 64 features of the gate and the same 64 of the other projection, 16 by 16.
template <int OUT, class OutT>
struct RowWarp {
  static constexpr bool kTwo = OUT == kGated;
  const GatedArgs& p;
  const Tile t;
  const int feat0;        // of the result, of the warp's first column
  const int columns;      // that the tensor core fills for the warp, 128 at most, may be <= 0
  const int row0, rows;   // of the warp's lanes: the first, and how many live, may be <= 0 or > 32
  unsigned char* const staged;
  const int lane;
  float sum[128];

  // of_tile: columns of the tile
  __device__ __forceinline__ RowWarp(const GatedArgs& args, const Tile& tile, int of_tile, int half, int first_row, unsigned char* mem, int l)
      : p(args), t(tile), feat0(tile.feat0 + half * (kTwo ? 64 : 128)), columns(min(of_tile - half * 128, 128)), row0(tile.col0 + first_row),
        rows(tile.n - first_row), staged(mem), lane(l) {}

  // false: a wait ran out
  __device__ __forceinline__ bool add(uint32_t taddr, int buffer, uint64_t* full, uint64_t* empty, int acc) {
    const int blocks = (p.k + SPARSETIR_F8_BLOCK - 1) / SPARSETIR_F8_BLOCK;
    const int of_w = ((kTwo ? 2 : 1) * p.features + SPARSETIR_F8_BLOCK - 1) / SPARSETIR_F8_BLOCK;
    auto scales = [&](int f) { return p.w_scale + (static_cast<size_t>(t.group) * of_w + f / SPARSETIR_F8_BLOCK) * blocks + t.step0; };
    const int f = min(feat0, p.features - 1), up = p.features + f;
    const float* const ws = scales(f);
    const float* const wu = scales(up);
    const float* const wv = scales(min(up + 63, 2 * p.features - 1));
    const int change = ((up / SPARSETIR_F8_BLOCK) + 1) * SPARSETIR_F8_BLOCK - up;  // gated: features from here on have the scales of wv
    const float* xs = p.x_scale + static_cast<size_t>(t.step0) * p.rows + row0 + lane;
    struct Step { float x, w, u, v; };
    auto fetch = [&](int k) {
      Step s{0.f, 0.f, 0.f, 0.f};
      if (k >= t.steps) return s;
      if (lane < rows) s.x = ld_global(xs);
      xs += p.rows;
      s.w = ld_global(ws + k);
      if constexpr (kTwo) {
        s.u = ld_global(wu + k);
        s.v = ld_global(wv + k);
      }
      return s;
    };
    Step a = fetch(0), b = fetch(1);
#pragma unroll
    for (int i = 0; i < 128; ++i) sum[i] = 0.f;
    const bool dead = columns <= 0 || rows <= 0;
    auto wait = [&](int n) { return __all_sync(0xffffffffu, tc05::mbar_spin(full + (n & 1), (n >> 1) & 1)) != 0; };
    // 32 columns; those of a gated block: 16 of the gate, 16 of the other projection
    auto add32 = [&](int j, const uint32_t (&r)[32], float s, float u, float v, auto mixed) {
      const int left = change - 16 * j;  // features with the scales of u
      const float by = !kTwo ? s : left > 0 ? u : v;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float f = i < 16 ? s : mixed.value && kTwo ? (i - 16 < left ? u : v) : by;
        sum[32 * j + i] = fmaf(__uint_as_float(r[i]), f, sum[32 * j + i]);
      }
    };
    if (!dead && columns == 128 && !(kTwo && change < 64 && change % 16 != 0)) {
      // All of it: the loads of the next 32 columns, across the steps, while these are added.  Whether the next step's sums are complete is
      // asked ahead, since the answer takes 0.1 us.
      if (!wait(acc)) return false;
      tc05::fence_after_sync();
      uint32_t r[2][32];
      tc05::tmem_ask32(taddr + (acc & 1) * buffer, r[0]);
      for (int k = 0; k < t.steps; ++k, ++acc) {
        const float s = a.x * a.w, u = a.x * a.u, v = a.x * a.v;
        a = b;
        b = fetch(k + 2);
        const uint32_t from = taddr + (acc & 1) * buffer, next = taddr + ((acc + 1) & 1) * buffer;
        const bool more = k + 1 < t.steps;
        bool over = true;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          tc05::tmem_ld_wait(r[j & 1]);
          if (j < 3) {
            tc05::tmem_ask32(from + 32 * (j + 1), r[(j + 1) & 1]);
          } else {
            taken(empty + (acc & 1));
            if (more) {
              if (!__all_sync(0xffffffffu, over) && !wait(acc + 1)) return false;
              tc05::fence_after_sync();
              tc05::tmem_ask32(next, r[0]);
            }
          }
          if (j == 2 && more) over = tc05::mbar_over(full + ((acc + 1) & 1), ((acc + 1) >> 1) & 1);
          add32(j, r[j & 1], s, u, v, std::false_type{});
        }
      }
      return true;
    }
    for (int k = 0; k < t.steps; ++k, ++acc) {
      const float s = a.x * a.w, u = a.x * a.u, v = a.x * a.v;
      a = b;
      b = fetch(k + 2);
      if (!wait(acc)) return false;
      tc05::fence_after_sync();
      if (dead) {
        taken(empty + (acc & 1));
        continue;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (32 * j >= columns) break;
        uint32_t r[32];
        tc05::tmem_ld32(taddr + (acc & 1) * buffer + 32 * j, r);
        if (32 * (j + 1) >= columns) taken(empty + (acc & 1));
        add32(j, r, s, u, v, std::true_type{});
      }
    }
    return true;
  }
  __device__ __forceinline__ void taken(uint64_t* empty) const {  // the sums of the step are in registers: the accumulator may be written again
    tc05::fence_before_sync();
    __syncwarp();
    if (lane == 0) tc05::mbar_arrive(empty);
  }

  // A lane's 64 bytes, of its row, to rows of the result: pieces of 16 bytes through shared memory, so that four lanes have a row's.  O: elements,
  // `to` where row 0's first piece goes, `live` elements of a row.
  template <class O>
  __device__ __forceinline__ void leave(const uint4 (&v)[4], O* to, size_t pitch, int live) const {
    constexpr int N = 16 / sizeof(O);
    using Place = Warp<__half>;
    __syncwarp();  // the last ones have left
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(staged + Place::place64(lane, q)) = v[q];
    __syncwarp();
    const int r = lane >> 2, q = lane & 3;
    const bool wide = pitch % N == 0 && (reinterpret_cast<uintptr_t>(to) & 15u) == 0 && N * q + N <= live;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 w = *reinterpret_cast<const uint4*>(staged + Place::place64(r + 8 * i, q));
      if (r + 8 * i >= rows) continue;
      O* at = to + (r + 8 * i) * pitch + N * q;
      if (wide) {
        *reinterpret_cast<uint4*>(at) = w;
      } else {
        const O* e = reinterpret_cast<const O*>(&w);
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (N * q + n < live) at[n] = e[n];
      }
    }
  }
  __device__ __forceinline__ void emit() const {
    if (columns <= 0 || rows <= 0) return;
    if (p.splits > 1) {
      const size_t pitch = kTwo ? 2 * static_cast<size_t>(p.features) : p.features;
      float* const to = static_cast<float*>(p.parts) + t.split * p.part + static_cast<size_t>(row0) * pitch;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int f = feat0 + (kTwo ? 16 * (j >> 1) : 16 * j);
        if (f < p.features) floats(j, to + f + (kTwo && (j & 1) != 0 ? p.features : 0), pitch, p.features - f);
      }
      return;
    }
    OutT* const to = static_cast<OutT*>(p.out) + static_cast<size_t>(row0) * p.features;
    if constexpr (sizeof(OutT) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (feat0 + 16 * j < p.features) floats(j, to + feat0 + 16 * j, p.features, p.features - feat0 - 16 * j);
    } else {
#pragma unroll
      for (int j = 0; j < (kTwo ? 2 : 4); ++j) {  // 32 features at a time
        const int f = feat0 + 32 * j;
        if (f >= p.features) break;
        uint4 v[4];
        uint32_t* const w = reinterpret_cast<uint32_t*>(v);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if constexpr (kTwo) {
            const int at = 64 * j + 32 * (i >> 3) + 2 * (i & 7);
            const Two g(sum[at], sum[at + 1]), u(sum[at + 16], sum[at + 17]);
            const Two a = p.gate.gelu ? Gate::act<true>(g, u) : Gate::act<false>(g, u);
            w[i] = pack2<OutT>(a.lo(), a.hi());
          } else {
            w[i] = pack2<OutT>(sum[32 * j + 2 * i], sum[32 * j + 2 * i + 1]);
          }
        }
        leave(v, to + f, p.features, p.features - f);
      }
    }
  }
  // Columns 16 j to 16 j + 15 as they are
  __device__ __forceinline__ void floats(int j, float* to, size_t pitch, int live) const {
    uint4 v[4];
    uint32_t* const w = reinterpret_cast<uint32_t*>(v);
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(sum[16 * j + i]);
    leave(v, to, pitch, live);
  }
  __device__ __forceinline__ void zeros() {
#pragma unroll
    for (int i = 0; i < 128; ++i) sum[i] = 0.f;
    emit();
  }
};

// Both forms take GatedArgs: of these sizes the larger one is the faster to launch (FewGatedArgs; a call 4.9 us on the host, with Args 5.2).
template <int OUT, class OutT>
__global__ void __launch_bounds__(kF8Threads, 1)
f8_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x64, const __grid_constant__ CUtensorMap tm_x16,
          const __grid_constant__ GatedArgs p) {
  constexpr int kN = 128, kDepth = 128, kFeatures = OUT == kGated ? 128 : 256;  // rows and features of a tile
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kF8Stages];
  __shared__ __align__(8) uint64_t bar_empty[kF8Stages];  // the tensor core has read the stage
  __shared__ __align__(8) uint64_t bar_acc_full[2];
  __shared__ __align__(8) uint64_t bar_acc_empty[2];
  __shared__ __align__(8) uint64_t bar_drain;
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* const stages = smem_raw + (((tc05::smem_u32(smem_raw) + 1023u) & ~1023u) - tc05::smem_u32(smem_raw));

  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kF8Stages; ++s) {
        tc05::mbar_init(&bar_full[s], 1);
        tc05::mbar_init(&bar_empty[s], 1);
      }
      for (int b = 0; b < 2; ++b) {
        tc05::mbar_init(&bar_acc_full[b], 1);
        tc05::mbar_init(&bar_acc_empty[b], 8);
      }
      tc05::mbar_init(&bar_drain, 1);
      tc05::fence_mbar_init();
      tc05::prefetch_tensormap(&tm_w);
      tc05::prefetch_tensormap(&tm_x64);
    }
    __syncwarp();
    tc05::tmem_alloc(&s_tmem, 512);
  }
  chain_wait();
  tc05::fence_before_sync();
  __syncthreads();
  chain_trigger();
  tc05::fence_after_sync();
  const uint32_t tmem = s_tmem;
  bool ok = true;
  int armed = 0;

  // as in grouped_kernel
  int stage = 0;
  uint32_t phase = 0;
  auto advance = [&](int steps) {
    const int q = stage + steps;
    phase ^= static_cast<uint32_t>(q / kF8Stages) & 1u;
    stage = q % kF8Stages;
  };
  Walker<false, kN, kDepth, kFeatures> walk(p);
  Tile tile;
  int unit = -1;
  auto next = [&]() {  // a role's next tile
    unit = unit < 0 ? static_cast<int>(blockIdx.x) : unit + static_cast<int>(gridDim.x);
    return unit < p.max_tiles && walk.at(unit, &tile);
  };
  // Columns of a tile: rows of W, 32 at a time
  auto columns_of = [&](const Tile& t) { return min(256, ((OUT == kGated ? 2 : 1) * (p.features - t.feat0) + 31) & ~31); };

  if (warp >= kFirstEpilogue) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kF8Epilogue));
    const int half = (warp - kFirstEpilogue) / 4, first_row = (warp & 3) * 32;
    unsigned char* const staged = stages + kF8Stages * kF8Bytes + (warp - kFirstEpilogue) * kStagedBytes;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(first_row) << 16) + 128 * half;
    int acc = 0;
    while (ok && next()) {
      RowWarp<OUT, OutT> w(p, tile, columns_of(tile), half, first_row, staged, lane);
      if (tile.steps == 0) {  // nothing of the depth is left for this unit
        w.zeros();
        continue;
      }
      ok = w.add(taddr, 256, bar_acc_full, bar_acc_empty, acc);
      acc += tile.steps;
      if (ok) w.emit();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kF8Others));
    if (warp == 0) {
      // ---- loads
      while (ok && next()) {
        const int units = (tile.n + 15) / 16;  // rows of x, 16 at a time
        if (tc05::elect_one()) {
          int s = stage;
          uint32_t ph = phase;
          for (int k = tile.step0; k < tile.step0 + tile.steps; ++k) {
            if (!tc05::mbar_wait(&bar_empty[s], ph ^ 1u)) { ok = false; break; }
            unsigned char* const st = stages + s * kF8Bytes;
            tc05::mbar_arrive_expect_tx(&bar_full[s], kF8Bytes - kXBytes + units * 2048);
            if constexpr (OUT == kGated) {  // 16 rows of the gate, 16 of the other projection, and so on
#pragma unroll
              for (int q = 0; q < 8; ++q)
                tc05::tma_load_4d(st + kXBytes + q * 4096, &tm_w, k * kDepth, tile.feat0 + 16 * q, 0, tile.group, &bar_full[s]);
            } else {
              tc05::tma_load_3d(st + kXBytes, &tm_w, k * kDepth, tile.feat0, tile.group, &bar_full[s]);
            }
            int u = 0;
            for (; u + 4 <= units; u += 4) tc05::tma_load_2d(st + u * 2048, &tm_x64, k * kDepth, tile.col0 + u * 16, &bar_full[s]);
            for (; u < units; ++u) tc05::tma_load_2d(st + u * 2048, &tm_x16, k * kDepth, tile.col0 + u * 16, &bar_full[s]);
            ++armed;
            if (++s == kF8Stages) { s = 0; ph ^= 1u; }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        advance(tile.steps);
      }
      // The tensor core's last arrivals have come before the block ends.
      for (int i = 0; i < kF8Stages && ok; ++i) {
        ok = __all_sync(0xffffffffu, tc05::mbar_wait(&bar_empty[stage], phase ^ 1u));
        advance(1);
      }
    } else if (warp == 1) {
      // ---- MMAs: M = 128 rows of x (those that are not there are whatever a stage held before, and nobody's), N = rows of W
      int acc = 0;
      const uint32_t base = tc05::smem_u32(stages);
      const uint64_t dx0 = tc05::smem_desc_swizzled(base, 0, 1024, tc05::kSwizzle128B);
      const uint64_t dw0 = tc05::smem_desc_swizzled(base + kXBytes, 0, 1024, tc05::kSwizzle128B);
      while (ok && next()) {
        if (tile.steps == 0) continue;
        if (tc05::elect_one()) {
          const uint32_t idesc = p.idesc | static_cast<uint32_t>(columns_of(tile) >> 3) << 17;
          int s = stage;
          uint32_t ph = phase;
          for (int k = tile.step0; k < tile.step0 + tile.steps; ++k) {
            // every step has sums of its own; its operands are there long before the accumulator is free
            const int n = acc + k - tile.step0, b = n & 1;
            if (!tc05::mbar_spin(&bar_full[s], ph) || !tc05::mbar_spin(&bar_acc_empty[b], ((n >> 1) & 1) ^ 1)) { ok = false; break; }
            tc05::fence_after_sync();
            const uint64_t dx = tc05::desc_advance(dx0, s * kF8Bytes), dw = tc05::desc_advance(dw0, s * kF8Bytes);
            const int left = tile.depth - k * kDepth;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i * 32 < left) tc05::mma_f8(tmem + b * 256, tc05::desc_advance(dx, i * 32), tc05::desc_advance(dw, i * 32), idesc, i > 0 ? 1u : 0u);
            tc05::mma_commit(&bar_acc_full[b]);
            tc05::mma_commit(&bar_empty[s]);
            if (++s == kF8Stages) { s = 0; ph ^= 1u; }
          }
          if (!ok) {  // gave up: what has been issued is over before the block's memory is released
            tc05::mma_commit(&bar_drain);
            tc05::mbar_wait(&bar_drain, 0);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        acc += tile.steps;
        advance(tile.steps);
      }
    }
  }

  const bool all_ok = !__syncthreads_or(!ok);
  if (!all_ok) {
    if (tid == 0) atomicAdd(&g_grouped_timeouts, 1u);
    // gave up: the loads that have been issued land (bounded) before the block's memory is released
    for (int it = max(0, armed - kF8Stages); it < armed; ++it) tc05::mbar_wait(&bar_full[it % kF8Stages], (it / kF8Stages) & 1);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  __syncwarp();
  tc05::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc05::tmem_dealloc(tmem, 512);
}

template <int OUT, class OutT>
int launch_f8(const CUtensorMap& w, const CUtensorMap& x64, const CUtensorMap& x16, const GatedArgs& p, cudaStream_t st) {
  static thread_local int configured_device = -1;
  const auto kernel = f8_kernel<OUT, OutT>;
  int dev = 0;
  SPTIR_CUDA_OK(cudaGetDevice(&dev));
  if (configured_device != dev) {
    SPTIR_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kF8Smem));
    // a share of more registers than the block has would be waited for for good
    cudaFuncAttributes attr;
    SPTIR_CUDA_OK(cudaFuncGetAttributes(&attr, kernel));
    if (attr.numRegs * kF8Threads < 128 * kF8Others + (kF8Threads - 128) * kF8Epilogue)
      return fail("f8_kernel was built with %d registers to a thread", attr.numRegs);
    configured_device = dev;
  }
  launch_chained(kernel, std::min(p.max_tiles, kNumSMs), kF8Threads, kF8Smem, st, w, x64, x16, p);
  SPTIR_LAUNCH_OK("f8_kernel");
  return join_parts<false, OUT, OutT>(p, st);
}

int product_f8(const char* fn, const void* x, const float* x_scale, const void* w, const float* w_scale, void* y, int y_type,
               const int32_t* indptr, int rows, int groups, int fi, int fo, bool gated, const Gate& gate, int device_id, cudaStream_t st) {
  GatedArgs p{};
  p.out = y;
  p.gate = gate;
  p.indptr = indptr;
  p.x_scale = x_scale;
  p.w_scale = w_scale;
  p.rows = rows;
  p.groups = groups;
  p.k = fi;
  p.features = fo;
  p.idesc = tc05::instr_desc(tc05::kFmtE4M3, kM, 0, 0, 0);
  const int each = gated ? 2 * fo : fo;  // rows of one W
  if (plan_f8(fn, &p, each) != 0) return -1;
  Operand ox{x, rows, fi, 1}, ow{w, static_cast<long long>(groups) * each, fi, 1};
  // us, weights out of HBM, the kernel for few rows / this one: 1 row, 4096 -> 8192 10.3 / 14.2; 16 rows 12.5 / 15.1; 8 groups of 8 rows, 2048 -> 2048
  // 12.2 / 14.0 (of 10 and more rows this one: 14.1), gated, 1024 -> 2 x 2048 12.9 / 15.0; 32 groups, 1024 -> 1024, of 4 rows 10.8 / 11.4, of 8 12.7 / 11.7
  const bool few = fi <= kFewF8Depth && few_rows_pay(rows, groups, fi, each, true);
  const size_t bytes = ox.copy_bytes() + ow.copy_bytes() + (few ? 0 : part_bytes(p));
  CallScratch cs;
  if (bytes > 0 && take_scratch(device_id, st, bytes, 0, &cs) != 0) return -1;
  char* scratch = cs.scratch;
  if (place_operand(&ox, &scratch, st) != 0 || place_operand(&ow, &scratch, st) != 0) return -1;
  if (few) {
    const FewGatedArgs f{{ox.data, ow.data, y, x_scale, w_scale, indptr, ox.pitch, ow.pitch, rows, groups, fi, fo, fi, 0, 0, 0}, nullptr, gate};
    const int done = few_rows_f8(f, y_type, gated, st);
    return done != 0 ? done : return_scratch(cs, st);
  }
  p.parts = scratch;
  CUtensorMap tm_w, tm_x64, tm_x16;
  if (map_operands(&tm_w, &tm_x64, &tm_x16, CU_TENSOR_MAP_DATA_TYPE_UINT8, ow, ox, fo, groups, true, gated, 2 * kM) != 0) return -1;
  const int rc = with_type(y_type, [&](auto o) {
    using O = decltype(o);
    if constexpr (sizeof(O) == 2)
      if (gated) return launch_f8<kGated, O>(tm_w, tm_x64, tm_x16, p, st);
    return launch_f8<kPlain, O>(tm_w, tm_x64, tm_x16, p, st);
  });
  return rc != 0 ? rc : return_scratch(cs, st);
}

}  // namespace

int f8_timeouts(unsigned int* count) {
  SPTIR_CUDA_OK(cudaMemcpyFromSymbol(count, g_grouped_timeouts, sizeof(unsigned int)));
  return 0;
}

}  // namespace sptir

using namespace sptir;

extern "C" int sparsetir_grouped_mm_f8_raw(const void* x, const float* x_scale, const void* w, const float* w_scale, void* y, int y_type,
                                           const int32_t* indptr, int rows, int num_groups, int feat_in, int feat_out, int device_id,
                                           void* stream) {
  const char* fn = "sparsetir_grouped_mm_f8";
  if (check_block(fn, indptr, rows, num_groups, feat_in, feat_out, false, 0, 0) != 0) return -1;
  if (y_type < SPARSETIR_F32 || y_type > SPARSETIR_BF16) return fail("%s: unknown element type %d", fn, y_type);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !x_scale || !w || !w_scale || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return product_f8(fn, x, x_scale, w, w_scale, y, y_type, indptr, rows, num_groups, feat_in, feat_out, false, Gate(), device_id, st);
}

extern "C" int sparsetir_grouped_mm_gated_f8_raw(const void* x, const float* x_scale, const void* w, const float* w_scale, void* y,
                                                 int y_type, const int32_t* indptr, int rows, int num_groups, int feat_in, int width,
                                                 int flags, int device_id, void* stream) {
  const char* fn = "sparsetir_grouped_mm_gated_f8";
  if (check_block(fn, indptr, rows, num_groups, feat_in, width, true, flags, SPARSETIR_GATED_GELU) != 0) return -1;
  if (y_type != SPARSETIR_F16 && y_type != SPARSETIR_BF16) return fail("%s: y is f16 or bf16", fn);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !x_scale || !w || !w_scale || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return product_f8(fn, x, x_scale, w, w_scale, y, y_type, indptr, rows, num_groups, feat_in, width, true,
                    Gate((flags & SPARSETIR_GATED_GELU) != 0), device_id, st);
}
