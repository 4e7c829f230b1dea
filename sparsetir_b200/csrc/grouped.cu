// Products grouped by expert, ragged sizes, on the tensor cores:
//   grouped_mm         y[s, :] = x[s, :] * W[g]                       s in [indptr[g], indptr[g + 1])
//   grouped_mm_i8      the same in 8-bit integers, scaled per row and per output feature
//   grouped_mm_grad_w  dW[g, a, b] = sum over the rows s of group g of pa[s, a] * pb[s, b]
//
// All three are one kernel, and so are the products of grouped_gated.cu, which includes this file; grouped_f8.cu, which does too, has a kernel of its own
// and takes the walk over the tiles and what the hosts share.  A
// pair of blocks (cta_group::2) holds 256 of what is contiguous in the result (output
// features; b) as the rows of the tensor core's left operand, and up to 256 of what is not (rows of the group; a) as the columns:
// the result comes out of TMEM with neighbouring lanes at neighbouring addresses, and a ragged group costs its rows rounded
// up to 32, whatever the group's neighbours are.  Rows of the neighbours that a load brings along become columns that nobody
// stores; in the gradient, where rows are the depth, they are cleared in shared memory.  How many rows a group has is read from
// indptr on the device.
//
// A ring of six stages of 32 KB is fed by TMA, MMAs of 256 x 256 x 16 (x 32) go to one of two accumulators while eight warps
// take the other one out; a pair's units are those of its number, of its number plus the pairs, and so on.
// With all operands in L2 a step of K (64 deep, 512 clocks of the tensor core) takes 0.28 us of loads, 117 GB/s into each SM:
// loads and MMAs are even, and beyond about 1.2 PFLOP/s the power limit lowers the clock.  65,536 rows in 64 ragged groups, 2048 ->
// 2048, bf16: 0.45-0.53 ms, 1.04-1.2 PFLOP/s, by the clock (8192^3 in one group: 0.71-0.83 ms; a library product 0.75).  The
// gradient of 64 weights of 2048 x 1024 over 32,768 rows, 8 steps to a tile, 0.16-0.17 ms: its 470 MB alone are 72 us.
// Tried and taken back: equal column tiles instead of 256 and a remainder (more, smaller loads: 45 -> 54 us on 6,001 rows); a
// prefetch of the next tiles' operands to L2 (44 -> 60); the whole tiles of all groups first (no change); one arrival
// of the loading thread at the other block's barrier per step (935 us where now 500).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gate.cuh"
#include "grouped.h"
#include "launch.cuh"
#include "lowp.cuh"
#include "tc05.cuh"
#include "tmap.h"
#include "vec.cuh"

namespace sptir {
namespace {

constexpr int kM = 128;               // features per block
constexpr int kABytes = 16 * 1024;    // left operand of a stage: 128 rows of 128 bytes
constexpr int kAtom = 8 * 1024;       // 64 rows of 128 bytes
constexpr int kFirstEpilogue = 4;     // warp 0 loads, 1 issues, 2 clears the tails of groups (grad_w), from 4 on the epilogue
constexpr int kStagedBytes = 32 * 64; // 32 columns of 32 features on their way, per epilogue warp
constexpr int kBand = 8;              // column tiles of a group that are walked side by side

// What becomes of the sums: the result, a gradient of weights (rows of a group are the depth), or, in grouped_gated.cuh, a gated block
// (two rows of W to a feature) and the gradient of one, with rows at 16-byte addresses or at any.
enum Out { kPlain, kWeights, kGated, kGatedGrad, kGatedGradAny };

// Columns of a tile, and what follows from them.  128 leave room for two pairs of blocks on two SMs: for many groups of few rows,
// where the loads of one pair hide the other's beginning and end (us, 256 / 128 columns: 64 groups of 16 rows, 512 -> 512
// 13.6 / 7.6; 500 rows in 64 groups, 2048 -> 2048 91.4 / 90.3; 8 groups of 500 rows 39 / 41).
template <int N, int OUT = kPlain> struct Shape {
  static constexpr int kBytes = kABytes + N / 2 * 128;  // of a stage
  static constexpr int kStages = N == 256 ? 6 : OUT >= kGatedGrad ? 3 : 4;  // what shared memory holds
  static constexpr int kBlocks = N == 256 ? 1 : 2;      // per SM
  static constexpr int kTmemCols = 2 * N;               // two accumulators
  static constexpr int kEpilogue = N == 256 ? 8 : 4;    // warps
  static constexpr int kThreads = (kFirstEpilogue + kEpilogue) * 32;
  static constexpr int kStaged = OUT >= kGatedGrad ? 2 * kStagedBytes : OUT == kGated ? kStagedBytes + kStagedBytes / 2 : kStagedBytes;
  static constexpr int kSmem = kStages * kBytes + kEpilogue * kStaged + 1024;
};

__device__ unsigned int g_grouped_timeouts = 0;

// Quotients by numbers that the host knows, of dividends below 2^31: a product and a shift (a division is tens of
// instructions, and every role makes several per tile).
struct Divisor {
  uint32_t by = 1, mul = 1u << 31;
  int shift = 31;
  Divisor() = default;
  explicit Divisor(uint32_t d) : by(d), shift(31) {
    while ((1ull << (shift - 31)) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << shift) + d - 1) / d);
  }
  __device__ __forceinline__ int quotient(int n) const {
    return static_cast<int>((static_cast<unsigned long long>(static_cast<uint32_t>(n)) * mul) >> shift);
  }
};

struct Args {
  void* out;
  const int32_t* indptr;
  const float* x_scale;
  const float* w_scale;
  int rows, groups;
  int k;          // depth of the product; grad_w: unused
  int features;   // contiguous in the result; gated: of act, half the rows of W
  int columns;    // grad_w: rows of each dW
  int mt, nt;     // tiles of 256 rows of W (256 features); grad_w: column tiles
  Divisor per_split, per_group, per_band;  // splits; grad_w: mt * nt; kBand * mt
  int max_tiles;  // no valid indptr has more; times splits
  int splits;     // units that share the depth of a tile, each with sums of its own in `parts`
  void* parts;    // [splits][rows of the result][features; gated: both halves], 32 bits each
  long long part; // elements of one split's
  uint32_t idesc; // without N
  int a_mn;       // the left operand is contiguous along the features
  int wide;       // rows of the result start at 16-byte addresses, and so do those of GatedArgs
};
static_assert(sizeof(Args) == 136, "what a launch was measured with (FewGatedArgs)");
// Of a gated block and its gradient.
struct GatedArgs : Args {
  const void* hidden_in;  // gradient: the block's projections
  void* hidden;   // the projections, or null; gradient: theirs.  `out` is act, in the gradient it may be null
  Gate gate;
};
template <int OUT> using ArgsOf = std::conditional_t<(OUT >= kGated), GatedArgs, Args>;

// First and past the last row of group g, inside the array whatever the pointers say.
__device__ __forceinline__ void group_rows(const Args& p, int g, int* first, int* last) {
  if (p.indptr == nullptr) { *first = 0; *last = p.rows; return; }
  *first = min(max(ld_global(p.indptr + g), 0), p.rows);
  *last = max(min(ld_global(p.indptr + g + 1), p.rows), *first);
}

struct Tile {
  int group, feat0;
  int col0, n, n_mma;      // columns: first, how many there are, rounded up to 32
  int row0, depth;         // depth: of K; grad_w: the rows of the group, from row0 on
  int split, step0, steps; // the unit's share of the depth
};

// The tile of a unit.  All lanes of a warp call at() together, with units that rise; lane l holds the prefix of tile counts of group base + l.
// Sums stop at 2^30: wild pointers give tiles inside the arrays, and no more than max_tiles of them.
template <bool GRAD, int kN, int kDepth, int kFeatures = 2 * kM>
struct Walker {
  const Args& p;
  int base = -32;
  unsigned before = 0, upto = 0;  // tiles ahead of the group of lane 0, and up to the group of this lane
  unsigned all = 0;               // up to the last of the 32
  int first = 0, last = 0;
  __device__ __forceinline__ explicit Walker(const Args& a) : p(a) {}
  __device__ __forceinline__ bool at(int unit, Tile* out) {
    const int t = p.per_split.quotient(unit);
    out->split = unit - t * p.splits;
    if constexpr (GRAD) {
      const int g = p.per_group.quotient(t), r = t - g * static_cast<int>(p.per_group.by);
      int f, l;
      group_rows(p, g, &f, &l);
      place(r, p.nt, out);
      out->group = g;
      out->col0 *= kN;
      out->n = min(kN, p.columns - out->col0);
      out->row0 = f;
      out->depth = l - f;
    } else {
      const int lane = threadIdx.x & 31;
      while (static_cast<unsigned>(t) >= all) {
        base += 32;
        if (base >= p.groups) return false;
        before = all;
        unsigned mine = 0;
        first = last = 0;
        if (base + lane < p.groups) {
          group_rows(p, base + lane, &first, &last);
          mine = static_cast<unsigned>(min(static_cast<long long>((last - first + kN - 1) / kN) * p.mt, 1ll << 30));
        }
        upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned up = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto = min(upto + up, 1u << 30);
        }
        upto = min(upto + before, 1u << 30);
        all = __shfl_sync(0xffffffffu, upto, 31);
      }
      const int src = __ffs(__ballot_sync(0xffffffffu, upto > static_cast<unsigned>(t))) - 1;
      const unsigned prev = __shfl_sync(0xffffffffu, upto, max(src - 1, 0));
      const int f = __shfl_sync(0xffffffffu, first, src), l = __shfl_sync(0xffffffffu, last, src);
      place(t - static_cast<int>(src == 0 ? before : prev), (l - f + kN - 1) / kN, out);
      out->group = base + src;
      out->col0 = f + out->col0 * kN;
      out->n = min(kN, l - out->col0);
      out->row0 = 0;
      out->depth = p.k;
    }
    out->n_mma = (out->n + 31) & ~31;
    const int steps = (out->depth + kDepth - 1) / kDepth, share = p.per_split.quotient(steps + p.splits - 1);
    out->step0 = min(out->split * share, steps);
    out->steps = min(share, steps - out->step0);
    return true;
  }
  // Tile r of a group with `cols` column tiles: bands of kBand column tiles, in a band one column tile after the other.
  // col0 is left in tiles.
  __device__ __forceinline__ void place(int r, int cols, Tile* out) const {
    // ceil(2^32 / width): exact for quotients of less than 2^29
    constexpr uint32_t kInverse[kBand + 1] = {0u, 0u, 0x80000000u, 0x55555556u, 0x40000000u, 0x33333334u, 0x2aaaaaabu, 0x24924925u, 0x20000000u};
    const int band = p.per_band.quotient(r), in = r - band * static_cast<int>(p.per_band.by);
    const int width = min(kBand, cols - band * kBand);
    uint32_t inverse = 0u;
#pragma unroll
    for (int w = 2; w <= kBand; ++w) inverse = width == w ? kInverse[w] : inverse;
    const int f = width == 1 ? in : static_cast<int>(__umulhi(static_cast<uint32_t>(in), inverse));
    out->feat0 = f * kFeatures;
    out->col0 = band * kBand + in - f * width;
  }
};

__device__ __forceinline__ float sum_of(uint32_t bits, bool i8) {
  return i8 ? static_cast<float>(static_cast<int>(bits)) : __uint_as_float(bits);
}
template <class OutT> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t&>(v);
}

// Columns first .. n - 1, 32 of every STEP, of 32 features from TMEM to rows of the result, 16-bit elements at 16-byte
// addresses.  The fragments of 8 columns and 32 features are transposed on their way to shared memory (rows of 32 features,
// pieces of 16 bytes exchanged so that neither side collides) and leave as 16 bytes to a lane.  With a 2-byte store per lane and column the epilogue took
// longer than the products of shallow tiles (us, then / with this: gradient of 64 weights of 2048 x 1024 287 / 175).
template <bool I8, int STEP, class OutT, class Take>
__device__ __forceinline__ void store_halves(OutT* to, int pitch, int feats, int first, int n, uint32_t taddr, unsigned char* staged,
                                             const float* xs, const float* ws, int lane, Take&& take) {
  float scale[4] = {};  // of features lane / 4 + 8 q
  if constexpr (I8) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (lane / 4 + 8 * q < feats) scale[q] = ld_global(ws + lane / 4 + 8 * q);
  }
  const uint32_t put = tc05::smem_u32(staged);
  const int get_row = lane >> 2, get_piece = lane & 3;
  const unsigned char* get = staged + get_row * 64 + ((get_piece ^ ((get_row >> 1) & 3)) << 4);  // rows 8 apart alike
  OutT* out = to + static_cast<size_t>(get_row) * pitch + get_piece * 8;
  const bool live = get_piece * 8 < feats;
  if (first >= n) return;
  uint32_t a[16], b[16];
  tc05::tmem_ld16x32(taddr + first, a);
  tc05::tmem_ld16x32(taddr + (16u << 16) + first, b);
  for (int c0 = first; c0 < n; c0 += STEP) {
    float x[8];
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + 8 * (i >> 1) + 2 * (lane & 3) + (i & 1);
        x[i] = c < n ? ld_global(xs + c) : 0.f;
      }
    }
    tc05::tmem_ld_wait();
    take(c0);
    __syncwarp();  // the reads of the last 32 columns are over
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // columns 8 i .. 8 i + 7
      uint32_t v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t* f = q < 2 ? a : b;
        float lo = sum_of(f[4 * i + 2 * (q & 1)], I8), hi = sum_of(f[4 * i + 2 * (q & 1) + 1], I8);
        if constexpr (I8) {
          lo *= x[2 * i] * scale[q];
          hi *= x[2 * i + 1] * scale[q];
        }
        v[q] = pack2<OutT>(lo, hi);
      }
      const int r = 8 * i + (lane & 7), q = lane >> 3;  // row and piece that this lane addresses
      asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(put + r * 64 + ((q ^ ((r >> 1) & 3)) << 4)),
                   "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                   : "memory");
    }
    if (c0 + STEP < n) {  // the next columns while these leave
      tc05::tmem_ld16x32(taddr + c0 + STEP, a);
      tc05::tmem_ld16x32(taddr + (16u << 16) + c0 + STEP, b);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(get + 8 * i * 64);
      if (live && c0 + 8 * i + get_row < n) *reinterpret_cast<uint4*>(out + static_cast<size_t>(c0 + 8 * i) * pitch) = v;
    }
  }
}

// Zeros to the same places.
template <int STEP, class OutT>
__device__ __forceinline__ void store_zeros(OutT* to, int pitch, int feats, int first, int n, bool wide, int lane) {
  for (int c0 = first; c0 < n; c0 += STEP) {
    if (sizeof(OutT) == 2 && wide) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + 8 * i + (lane >> 2), f = (lane & 3) * 8;
        if (c < n && f < feats) *reinterpret_cast<uint4*>(to + static_cast<size_t>(c) * pitch + f) = make_uint4(0u, 0u, 0u, 0u);
      }
    } else if (lane < feats) {
#pragma unroll 8
      for (int c = c0; c < min(c0 + 32, n); ++c) to[static_cast<size_t>(c) * pitch + lane] = OutT{};
    }
  }
}

// The same as store_halves for 32-bit elements and for rows at any address: lane = feature, a store per column.
template <bool I8, int STEP, class OutT, class Take>
__device__ __forceinline__ void store_lanes(OutT* to, int pitch, int feats, int first, int n, uint32_t taddr, const float* xs, const float* ws,
                                            int lane, Take&& take) {
  const bool live = lane < feats;
  float scale = 0.f;
  if constexpr (I8) {
    if (live) scale = ld_global(ws + lane);
  }
  for (int c0 = first; c0 < n; c0 += STEP) {
    OutT* out = to + static_cast<size_t>(c0) * pitch + lane;
    float x = 0.f;
    if constexpr (I8) {
      if (c0 + lane < n) x = ld_global(xs + c0 + lane);
    }
    uint32_t r[32];
    tc05::tmem_ld32(taddr + c0, r);
    take(c0);
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      float v = sum_of(r[c], I8);
      if constexpr (I8) v *= __shfl_sync(0xffffffffu, x, c) * scale;
      if (live && c0 + c < n) *out = from_float<OutT>(v);
      out += pitch;
    }
  }
}

}  // namespace
}  // namespace sptir

#include "grouped_gated.cuh"

namespace sptir {
namespace {

template <bool I8, int OUT, class OutT, int kN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Shape<kN>::kThreads, Shape<kN>::kBlocks)
grouped_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b64,
               const __grid_constant__ CUtensorMap tm_b16, const __grid_constant__ ArgsOf<OUT> p) {
  constexpr int kDepth = I8 ? 128 : 64;  // of K per stage
  constexpr int kInstr = I8 ? 32 : 16;   // of K per instruction
  using S = Shape<kN, OUT>;
  constexpr bool GRAD = OUT == kWeights;
  constexpr int kStages = S::kStages, kStageBytes = S::kBytes, kTmemCols = S::kTmemCols;
  constexpr int kEpilogue = S::kEpilogue;
  constexpr int kBlockFeatures = OUT == kGated ? kM / 2 : kM;  // of the result, per block
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kStages];   // rank 0: both blocks' operands are there
  __shared__ __align__(8) uint64_t bar_empty[kStages];  // the tensor core has read the stage
  __shared__ __align__(8) uint64_t bar_tail[kStages];   // the last rows of a group are there, to be cleared past its end
  __shared__ __align__(8) uint64_t bar_acc_full[2];
  __shared__ __align__(8) uint64_t bar_acc_empty[2];    // rank 0: both blocks have taken the result
  __shared__ __align__(8) uint64_t bar_drain;
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = tc05::pair::rank();
  const uint32_t base = (tc05::smem_u32(smem_raw) + 1023u) & ~1023u;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kStages; ++s) {
        tc05::mbar_init(&bar_full[s], 2);
        tc05::mbar_init(&bar_empty[s], 1);
        tc05::mbar_init(&bar_tail[s], 1);
      }
      for (int b = 0; b < 2; ++b) {
        tc05::mbar_init(&bar_acc_full[b], 1);
        tc05::mbar_init(&bar_acc_empty[b], 2 * kEpilogue);
      }
      tc05::mbar_init(&bar_drain, 1);
      tc05::fence_mbar_init();
      tc05::prefetch_tensormap(&tm_a);
      tc05::prefetch_tensormap(&tm_b64);
    }
    __syncwarp();
    tc05::pair::tmem_alloc(&s_tmem, kTmemCols);
  }
  chain_wait();
  tc05::fence_before_sync();
  __syncthreads();
  tc05::pair::sync();  // the other block's barriers are there
  chain_trigger();
  tc05::fence_after_sync();
  const uint32_t tmem = s_tmem;
  bool ok = true;
  int armed = 0;

  // Stage and phase of the ring move by whole tiles in all lanes of a role's warp; its elected thread walks them step by step.
  int stage = 0;
  uint32_t phase = 0;
  auto advance = [&](int steps) {
    const int q = stage + steps;
    phase ^= static_cast<uint32_t>(q / kStages) & 1u;
    stage = q % kStages;
  };
  Walker<GRAD, kN, kDepth, 2 * kBlockFeatures> walk(p);
  Tile tile;
  // Every role of both blocks finds them by itself.  Units taken over from pairs that do not run yet (cluster launch control), handed to
  // the roles through a ring of entries in both blocks' shared memory, were faster by up to 15 %, but about one launch in a
  // million had a role of the other block read an entry from before: taken back.
  int unit = -1;
  auto next = [&]() {  // a role's next tile
    unit = unit < 0 ? pair : unit + pairs;
    return unit < p.max_tiles && walk.at(unit, &tile);
  };

  if (warp == 0) {
    // ---- loads.  Each block fetches its 128 features and its half of the columns, and tells rank 0's barrier.
    while (ok && next()) {
      const int half = tile.n_mma / 2, units = half / 16;
      const int feat = tile.feat0 + static_cast<int>(rank) * kBlockFeatures, col = tile.col0 + static_cast<int>(rank) * half;
      if (tc05::elect_one()) {
        const uint32_t bytes = kABytes + (GRAD ? (half > 64 ? 2 : 1) * kAtom : units * 2048);
        int s = stage;
        uint32_t ph = phase;
        for (int k = tile.step0; k < tile.step0 + tile.steps; ++k) {
          if (!tc05::mbar_wait(&bar_empty[s], ph ^ 1u)) { ok = false; break; }
          const uint32_t st = base + s * kStageBytes;
          uint32_t bar;
          if (GRAD && (k + 1) * kDepth > tile.depth) {
            bar = tc05::smem_u32(&bar_tail[s]);
            tc05::mbar_arrive_expect_tx(&bar_tail[s], bytes);
          } else {
            bar = tc05::pair::at_first(&bar_full[s]);
            if (rank == 0) {  // for both blocks: an arrival from the other one at every step took 1 us each
              tc05::mbar_arrive_expect_tx(&bar_full[s], 2 * bytes);
              tc05::mbar_arrive(&bar_full[s]);
            }
          }
          if constexpr (GRAD) {
            const int row = tile.row0 + k * kDepth;
            tc05::pair::tma_load_2d(st, &tm_a, feat, row, bar);
            tc05::pair::tma_load_2d(st + kAtom, &tm_a, feat + 64, row, bar);
            tc05::pair::tma_load_2d(st + kABytes, &tm_b64, col, row, bar);
            if (half > 64) tc05::pair::tma_load_2d(st + kABytes + kAtom, &tm_b64, col + 64, row, bar);
          } else {
            if constexpr (OUT == kGated) {  // 16 rows of the gate, 16 of the other projection, and so on
#pragma unroll
              for (int q = 0; q < 4; ++q) tc05::pair::tma_load_4d(st + q * 4096, &tm_a, k * kDepth, feat + 16 * q, 0, tile.group, bar);
            } else if (p.a_mn) {
              tc05::pair::tma_load_3d(st, &tm_a, feat, k * kDepth, tile.group, bar);
              tc05::pair::tma_load_3d(st + kAtom, &tm_a, feat + 64, k * kDepth, tile.group, bar);
            } else {
              tc05::pair::tma_load_3d(st, &tm_a, k * kDepth, feat, tile.group, bar);
            }
            int u = 0;
            for (; u + 4 <= units; u += 4) tc05::pair::tma_load_2d(st + kABytes + u * 2048, &tm_b64, k * kDepth, col + u * 16, bar);
            for (; u < units; ++u) tc05::pair::tma_load_2d(st + kABytes + u * 2048, &tm_b16, k * kDepth, col + u * 16, bar);
          }
          ++armed;
          if (++s == kStages) { s = 0; ph ^= 1u; }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      advance(tile.steps);
    }
    // The last arrivals at this block's barriers come from the other block too: they have come before the block ends.
    for (int i = 0; i < kStages && ok; ++i) {
      ok = __all_sync(0xffffffffu, tc05::mbar_wait(&bar_empty[stage], phase ^ 1u));
      advance(1);
    }
  } else if (warp == 1) {
    // ---- MMAs of both blocks, from rank 0: M = 256 features, N = the tile's columns
    int acc = 0;
    const bool a_mn = GRAD || p.a_mn != 0;
    const uint32_t a_step = a_mn ? 2048u : 32u, b_step = GRAD ? 2048u : 32u;
    const uint64_t da0 = tc05::smem_desc_swizzled(base, a_mn ? kAtom : 0, 1024, tc05::kSwizzle128B);
    const uint64_t db0 = tc05::smem_desc_swizzled(base + kABytes, GRAD ? kAtom : 0, 1024, tc05::kSwizzle128B);
    while (rank == 0 && ok && next()) {
      if (tile.steps == 0) continue;
      if (tc05::elect_one()) {
        const int buf = acc & 1;
        const uint32_t idesc = p.idesc | static_cast<uint32_t>(tile.n_mma >> 3) << 17;
        const uint32_t d = tmem + buf * kN;
        int s = stage;
        uint32_t ph = phase;
        ok = tc05::pair::mbar_wait(&bar_acc_empty[buf], ((acc >> 1) & 1) ^ 1);
        tc05::fence_after_sync();
        for (int k = tile.step0; k < tile.step0 + tile.steps && ok; ++k) {
          const bool cleared = GRAD && (k + 1) * kDepth > tile.depth;  // by threads of both blocks
          if (!(cleared ? tc05::pair::mbar_wait(&bar_full[s], ph) : tc05::mbar_wait(&bar_full[s], ph))) { ok = false; break; }
          tc05::fence_after_sync();
          const uint64_t da = tc05::desc_advance(da0, s * kStageBytes), db = tc05::desc_advance(db0, s * kStageBytes);
          const int left = tile.depth - k * kDepth;
#pragma unroll
          for (int i = 0; i < kDepth / kInstr; ++i)
            if (i * kInstr < left)
              tc05::pair::mma<I8>(d, tc05::desc_advance(da, i * a_step), tc05::desc_advance(db, i * b_step), idesc,
                                  (k > tile.step0 || i > 0) ? 1u : 0u);
          tc05::pair::mma_commit(&bar_empty[s]);
          if (++s == kStages) { s = 0; ph ^= 1u; }
        }
        tc05::pair::mma_commit(&bar_acc_full[buf]);
        if (!ok) {  // gave up: what has been issued is over before the block's memory is released
          tc05::pair::mma_commit(&bar_drain);
          tc05::mbar_wait(&bar_drain, 0);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      ++acc;
      advance(tile.steps);
    }
  } else if (GRAD && warp == 2) {
    // ---- The last step of a group holds rows of its neighbours: zeros in their place, in both operands (0 times what is
    // not a number would not be zero), up to where the instructions read.
    uint32_t tail_phase = 0;
    while (ok && next()) {
      const int rem = tile.depth % kDepth;
      if (rem != 0 && tile.steps > 0 && (tile.step0 + tile.steps) * kDepth > tile.depth) {
        const int s = (stage + tile.steps - 1) % kStages;
        ok = __all_sync(0xffffffffu, tc05::mbar_wait(&bar_tail[s], (tail_phase >> s) & 1u));
        tail_phase ^= 1u << s;
        const int clear = (((rem + kInstr - 1) / kInstr) * kInstr - rem) * 8;  // pieces of 16 bytes in each atom
        unsigned char* at = smem_raw + (base - tc05::smem_u32(smem_raw)) + s * kStageBytes + rem * 128;
        for (int i = lane; i < kStageBytes / kAtom * clear; i += 32) {
          const int atom = i / clear;
          *reinterpret_cast<uint4*>(at + atom * kAtom + (i - atom * clear) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        tc05::fence_async_smem();
        __syncwarp();
        if (lane == 0) tc05::pair::arrive_release(tc05::pair::at_first(&bar_full[s]));
      }
      advance(tile.steps);
    }
  } else if (warp >= kFirstEpilogue) {
    // ---- epilogue: a warp takes the 32 features of its lanes of TMEM, columns 32 at a time; two warps share them
    int acc = 0;
    const int mine = (warp - kFirstEpilogue) / 4 * 32;  // first columns of the warp
    constexpr int kStep = kEpilogue / 4 * 32;
    unsigned char* const staged = smem_raw + (base - tc05::smem_u32(smem_raw)) + kStages * kStageBytes + (warp - kFirstEpilogue) * S::kStaged;
    while (ok && next()) {
      const int feat0 = tile.feat0 + static_cast<int>(rank) * kBlockFeatures + (warp & 3) * (kBlockFeatures / 4);
      size_t row = static_cast<size_t>(tile.col0);
      if constexpr (GRAD) row += static_cast<size_t>(tile.group) * p.columns;
      if constexpr (OUT >= kGated) {
        const Warp<OutT> w(p, tile, feat0, mine, kStep, staged, lane);
        const uint32_t taddr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        if (tile.steps == 0) {  // nothing of the depth is left for this unit
          w.template zeros<OUT>();
        } else {
          const int buf = acc & 1;
          ok = w.template out_of_tmem<OUT>(taddr + buf * kN, &bar_acc_full[buf], &bar_acc_empty[buf], (acc >> 1) & 1);
          ++acc;
        }
        continue;
      }
      const size_t at = row * p.features + feat0;  // column 0, feature 0 of the warp's
      OutT* const to = static_cast<OutT*>(p.out) + at;
      uint32_t* const part = p.splits > 1 ? static_cast<uint32_t*>(p.parts) + tile.split * p.part + at : nullptr;
      const int feats = p.features - feat0;  // live ones of the warp's, may be <= 0 or > 32
      if (tile.steps == 0) {  // a group without rows, or nothing of the depth left for this unit
        if (part != nullptr) {
          store_zeros<kStep>(part, p.features, feats, mine, tile.n, false, lane);
        } else {
          store_zeros<kStep>(to, p.features, feats, mine, tile.n, p.wide != 0, lane);
        }
        continue;
      }
      const int buf = acc & 1;
      ok = __all_sync(0xffffffffu, tc05::mbar_wait(&bar_acc_full[buf], (acc >> 1) & 1));
      if (!ok) break;
      tc05::fence_after_sync();
      const uint32_t taddr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + buf * kN;
      const uint32_t taken = tc05::pair::at_first(&bar_acc_empty[buf]);
      auto take = [&](int c0) {  // the warp's last columns are in registers: the accumulator may be written again
        if (c0 + kStep < tile.n) return;
        tc05::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc05::pair::arrive(taken);
      };
      if (mine >= tile.n) take(tile.n);
      const float* const xs = I8 ? p.x_scale + tile.col0 : nullptr;
      const float* const ws = I8 ? p.w_scale + static_cast<size_t>(tile.group) * p.features + feat0 : nullptr;
      bool done = false;
      if (part != nullptr) {
        store_lanes<false, kStep>(reinterpret_cast<float*>(part), p.features, feats, mine, tile.n, taddr, xs, ws, lane, take);
        done = true;
      }
      if constexpr (sizeof(OutT) == 2) {
        if (!done && p.wide) {
          store_halves<I8, kStep>(to, p.features, feats, mine, tile.n, taddr, staged, xs, ws, lane, take);
          done = true;
        }
      }
      if (!done) store_lanes<I8, kStep>(to, p.features, feats, mine, tile.n, taddr, xs, ws, lane, take);
      ++acc;
    }
  }

  const bool all_ok = !__syncthreads_or(!ok);
  if (!all_ok) {
    if (tid == 0) atomicAdd(&g_grouped_timeouts, 1u);
    // gave up: the loads that have been issued land (bounded) before the blocks' memory is released
    if (rank == 0)
      for (int it = max(0, armed - kStages); it < armed; ++it) tc05::mbar_wait(&bar_full[it % kStages], (it / kStages) & 1);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  __syncwarp();
  tc05::fence_before_sync();
  tc05::pair::sync();
  if (warp == 0) tc05::pair::tmem_dealloc(tmem, kTmemCols);
}

// ---- the sums of the units that share a tile, added in their order: thread = an element of the result
template <bool I8, bool GRAD, class OutT>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args p) {
  chain_wait();
  const int lane = threadIdx.x & 31;
  const long long row = blockIdx.y + static_cast<long long>(blockIdx.z) * gridDim.y;
  const int feat = blockIdx.x * 256 + threadIdx.x;
  int group = 0;
  if constexpr (!GRAD) {  // rows of no group are not written; 8-bit integers: the group's scales
    if (row >= p.rows) return;
    if (p.indptr != nullptr) {
      if (row < ld_global(p.indptr) || row >= ld_global(p.indptr + p.groups)) return;
      if constexpr (I8) group = group_of_row(p.indptr, p.groups, row, lane);
    }
  } else if (row >= static_cast<long long>(p.groups) * p.columns) {
    return;
  }
  if (feat >= p.features) return;
  const size_t at = static_cast<size_t>(row) * p.features + feat;
  const uint32_t* from = static_cast<const uint32_t*>(p.parts) + at;
  float v;
  if constexpr (I8) {
    int sum = 0;
#pragma unroll 8
    for (int s = 0; s < p.splits; ++s) sum += static_cast<int>(ld_global(from + s * p.part));
    v = static_cast<float>(sum) * (ld_global(p.x_scale + row) * ld_global(p.w_scale + static_cast<size_t>(group) * p.features + feat));
  } else {
    v = 0.f;
#pragma unroll 8
    for (int s = 0; s < p.splits; ++s) v += __uint_as_float(ld_global(from + s * p.part));
  }
  static_cast<OutT*>(p.out)[at] = from_float<OutT>(v);
}

// ---- rows at aligned addresses: TMA wants pitches that are multiples of 16 bytes.  A copy reads and writes the operand once more, which
// the large products can bear and the small ones feel (us, the same without a copy behind it: 4,593 rows in 16 groups,
// 3641 -> 3576 296, 3640 -> 3576 168; 16 rows in 8 groups, 1782 -> 1111 19, 1784 -> 1112 5.5).  Cutting 16 bytes out of two aligned
// loads in the kernel for few rows instead gained where weights are small (8 groups, 1001 -> 999 11.9 -> 8.5) and lost where
// they are not (64 rows, 2047 -> 2047 38 -> 62): taken back.

// A thread has 16 bytes of a row, in units of U bytes, the largest that rows and operand are multiples of (a gated block in 8 bits, 396
// rows in 16 groups, 1832 -> 1224: 91 us with units of a byte, 70 with units of 8).
template <int U>
__global__ void __launch_bounds__(256) pad_rows_kernel(const Piece<U>* src, uint4* dst, long long rows, int cols, int pieces) {
  constexpr int N = 16 / U;
  chain_wait();
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long row = at / pieces;
  const int c0 = static_cast<int>(at - row * pieces) * N;
  if (row >= rows) return;
  const Piece<U>* from = src + row * cols + c0;
  Piece<16> v = make_uint4(0u, 0u, 0u, 0u);
  Piece<U>* e = reinterpret_cast<Piece<U>*>(&v);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (c0 + i < cols) e[i] = from[i];
  dst[at] = v;
}

// A row-major operand of elements of `size` bytes as TMA can read it: where it is, or a padded copy.
struct Operand {
  const void* data;
  long long rows;
  int cols, size;
  size_t pitch = 0;  // bytes of a row
  bool fits() const { return aligned16(data) && static_cast<size_t>(cols) * size % 16 == 0; }
  size_t padded() const { return (static_cast<size_t>(cols) * size + 15) / 16 * 16; }
  size_t copy_bytes() const { return fits() ? 0 : (padded() * rows + 255) / 256 * 256; }
};
inline int place_operand(Operand* o, char** scratch, cudaStream_t st) {
  o->pitch = o->padded();
  if (o->fits() || o->rows == 0) return 0;
  const int pieces = static_cast<int>(o->pitch / 16);
  const long long blocks = (o->rows * pieces + 255) / 256;
  if (blocks > INT32_MAX) return fail("operand too large to be copied to aligned rows");
  uint4* to = reinterpret_cast<uint4*>(*scratch);
  const size_t row_bytes = static_cast<size_t>(o->cols) * o->size;
  auto run = [&](auto unit) {
    constexpr int U = unit.value;
    launch_chained(pad_rows_kernel<U>, static_cast<unsigned>(blocks), 256, 0, st, static_cast<const Piece<U>*>(o->data), to, o->rows,
                   static_cast<int>(row_bytes / U), pieces);
  };
  const size_t both = row_bytes | reinterpret_cast<uintptr_t>(o->data);
  if (both % 8 == 0) run(std::integral_constant<int, 8>{});
  else if (both % 4 == 0) run(std::integral_constant<int, 4>{});
  else if (both % 2 == 0) run(std::integral_constant<int, 2>{});
  else run(std::integral_constant<int, 1>{});
  SPTIR_LAUNCH_OK("pad_rows_kernel");
  *scratch += o->copy_bytes();
  o->data = to;
  return 0;
}

// Behind a product whose depth units share
template <bool I8, int OUT, class OutT>
int join_parts(const ArgsOf<OUT>& p, cudaStream_t st) {
  if (p.splits > 1) {
    const long long rows = p.part / (OUT == kGated ? 2ll * p.features : p.features);
    const unsigned y = static_cast<unsigned>(std::min<long long>(rows, 32768));
    const dim3 grid(ceil_div(p.features, 256), y, ceil_div(rows, y));
    if constexpr (OUT >= kGated) {
      launch_chained(join_gated_kernel<OUT, OutT>, grid, 256, 0, st, p);
    } else {
      launch_chained(join_kernel<I8, OUT == kWeights, OutT>, grid, 256, 0, st, p);
    }
    SPTIR_LAUNCH_OK("join_kernel");
  }
  return 0;
}

template <bool I8, int OUT, class OutT, int N>
int launch(const CUtensorMap& tm_a, const CUtensorMap& tm_b64, const CUtensorMap& tm_b16, const ArgsOf<OUT>& p, cudaStream_t st) {
  using S = Shape<N, OUT>;
  static thread_local int configured_device = -1;
  constexpr int smem = S::kSmem;
  const auto kernel = grouped_kernel<I8, OUT, OutT, N>;
  int dev = 0;
  SPTIR_CUDA_OK(cudaGetDevice(&dev));
  if (configured_device != dev) {
    SPTIR_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    SPTIR_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    configured_device = dev;
  }
  launch_chained(kernel, 2 * std::min(p.max_tiles, kNumSMs / 2 * S::kBlocks), S::kThreads, smem, st, tm_a, tm_b64, tm_b16, p);
  SPTIR_LAUNCH_OK("grouped_kernel");
  return join_parts<I8, OUT, OutT>(p, st);
}

inline int check_pointers(const char* fn, const int32_t* indptr, int rows, int groups, cudaStream_t st) {
  if (!indptr || !validate_enabled()) return 0;
  if (validate_indptr(fn, "indptr", indptr, groups, -1, st) != 0) return -1;
  return validate_range(fn, "indptr", indptr, groups + 1ll, rows + 1ll, st);
}
// Sets the tiles of p, and how many units share the depth of a tile, from what the host knows: `wide` rows of the left operand, `bound(n)`
// column tiles of n at most, about `some(n)` of them, `depth` steps each, and `rows` rows of the result.  Returns the columns of a tile, or -1.
// Units share a depth where the tiles are half as many as the pairs or fewer, into parts of four steps at least, and where that
// spares the twelve steps that the second launch costs (us, one unit / several: 100 rows, 4096 -> 4096 23 / 14; gradient of one
// 504 x 1000 weight over 60,000 rows 263 / 67; 300 rows, 4096 -> 4096, two units, 23 / 24).
template <class Bound, class Some>
int set_tiles(const char* fn, Args* p, int wide, bool few_columns, Bound&& bound, Some&& some, int depth, long long rows) {
  p->mt = ceil_div(wide, 2 * kM);
  const long long tiles = some(256) * p->mt;
  const int columns = few_columns && tiles > kNumSMs / 2 ? 128 : 256;
  p->splits = 1;
  if (columns == 256) {
    const int most = static_cast<int>(std::min<long long>(kNumSMs / 2 / std::max<long long>(tiles, 1), depth / 4));
    if (most > 1 && depth - depth / most >= 12) p->splits = most;
  }
  const long long units = bound(columns) * p->mt;
  if (units > (1 << 29) / p->splits) return fail("%s: too many tiles for 32-bit indices", fn);
  p->max_tiles = static_cast<int>(units) * p->splits;
  p->per_split = Divisor(p->splits);
  p->per_band = Divisor(kBand * p->mt);
  p->part = rows * wide;
  return columns;
}
// For rows, groups and k of p, `wide` rows of every W, steps of `depth` of K.
inline int plan_product(const char* fn, Args* p, int wide, int depth) {
  const long long rows = p->rows, used = std::min(p->groups, p->rows);
  return set_tiles(fn, p, wide, rows <= 128 * used, [&](int n) { return rows / n + used; },
                   [&](int n) { return used * ((rows + used * n - 1) / (used * n)); }, ceil_div(p->k, depth), rows);
}
// The same for f8_kernel (grouped_f8.cu): tiles of 128 rows x 256 rows of W, one to a block, by the same rule for a shared depth.
inline int plan_f8(const char* fn, Args* p, int wide) {
  const long long rows = p->rows, used = std::min(p->groups, p->rows);
  p->mt = ceil_div(wide, 2 * kM);
  const long long tiles = used * ((rows + used * 128 - 1) / (used * 128)) * p->mt, units = (rows / 128 + used) * p->mt;
  const int depth = ceil_div(p->k, 128);
  const int most = static_cast<int>(std::min<long long>(kNumSMs / std::max<long long>(tiles, 1), depth / 4));
  p->splits = most > 1 && depth - depth / most >= 12 ? most : 1;
  if (units > (1 << 29) / p->splits) return fail("%s: too many tiles for 32-bit indices", fn);
  p->max_tiles = static_cast<int>(units) * p->splits;
  p->per_split = Divisor(p->splits);
  p->per_band = Divisor(kBand * p->mt);
  p->part = rows * wide;
  return 0;
}
inline size_t part_bytes(const Args& p) { return p.splits > 1 ? p.part * p.splits * sizeof(float) : 0; }

inline CUtensorMapDataType map_type(int type) {
  return type == SPARSETIR_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
         : type == SPARSETIR_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
}
inline uint32_t map_format(int type) { return type == SPARSETIR_F16 ? tc05::kFmtF16 : tc05::kFmtBF16; }

// What the gated products and those of 8-bit floating point check; `half`: feat_out is the width of a gated block, half of W's rows
[[maybe_unused]] inline int check_block(const char* fn, const int32_t* indptr, int rows, int groups, int fi, int fo, bool half, int flags, int known) {
  if (rows < 0 || groups < 0) return fail("%s: negative size", fn);
  if (fi < 1 || fo < 1) return fail("%s: feat_in and %s must be positive", fn, half ? "width" : "feat_out");
  if (std::max(std::max(rows, groups), std::max(fi, fo)) > kLargestSize || (half && fo > kLargestSize / 2) ||
      (groups > 0 && static_cast<long long>(fi) * fo * (half ? 2 : 1) > INT64_MAX / groups))
    return fail("%s: too large for 32-bit indices", fn);
  if ((flags & ~known) != 0) return fail("%s: unknown flags %d", fn, flags);
  if (!indptr && groups > 1) return fail("%s: indptr may be null with num_groups 1 only", fn);
  return 0;
}
// Maps of a product's operands, in boxes of `depth` of K: W (`each` rows to a group) along K or along the features, or a gated block's along K,
// 16 rows of the gate and 16 of the other projection, `each` rows further on, to a box.
inline int map_operands(CUtensorMap* w, CUtensorMap* x64, CUtensorMap* x16, CUtensorMapDataType dt, const Operand& ow, const Operand& ox,
                        int each, int groups, bool along_k, bool gated, cuuint32_t box_rows = kM) {
  const cuuint32_t depth = 128 / ow.size;
  // the weights of the next step come with this one's (us, 128 / 256 bytes: 500 rows, 64 groups, 2048 -> 2048 90.8 / 84.8)
  const CUtensorMapL2promotion fetch = CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
  const cuuint64_t cols = ow.cols, n = each, g = groups;
  const cuuint64_t dims[3] = {cols, n, g}, strides[2] = {ow.pitch, ow.pitch * n};
  const cuuint32_t box[3] = {along_k ? depth : 64, along_k ? box_rows : depth, 1};
  const cuuint64_t two_dims[4] = {cols, n, 2, g}, two_strides[3] = {ow.pitch, ow.pitch * n, ow.pitch * n * 2};
  const cuuint32_t two_box[4] = {depth, 16, 2, 1};
  if (make_tmap(w, dt, ow.data, gated ? 4 : 3, gated ? two_dims : dims, gated ? two_strides : strides, gated ? two_box : box,
                CU_TENSOR_MAP_SWIZZLE_128B, fetch) != 0 ||
      make_tmap_2d(x64, dt, ox.data, ox.cols, ox.rows, ox.pitch, depth, 64, CU_TENSOR_MAP_SWIZZLE_128B) != 0 ||
      make_tmap_2d(x16, dt, ox.data, ox.cols, ox.rows, ox.pitch, depth, 16, CU_TENSOR_MAP_SWIZZLE_128B) != 0)
    return -1;
  return 0;
}
// f(T{}) for a type of 16 bits
template <class F>
int with_half(int type, F&& f) {
  if (type == SPARSETIR_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

inline bool wide_rows(const void* out, int type, int features) {
  return type != SPARSETIR_F32 && aligned16(out) && features % 8 == 0;
}

// Whether the kernel for groups of a few rows takes a product, from what the host knows (us, that kernel / this one, 16-bit elements
// unless said otherwise; rows, groups, features): W contiguous along the depth 2, 1, 4096 -> 4096 7.9 / 13.4; 16, 1, 4096 -> 4096
// 9.0 / 14.0; 16, 8, 1024 -> 1024 3.8 / 8.8; 64, 8, 2048 -> 2048 15.5 / 15.8; 8-bit integers 1, 1, 4096 -> 8192 8.2 / 14; but 128, 8,
// 2048 -> 2048 20 / 16 and 500, 64, 2048 -> 2048 114 / 90, which have tiles enough; along the features 16, 8, 512 -> 512 3.2 / 6.5,
// 1, 1, 4096 -> 4096 8.0 / 11.9, 16, 8, 1784 -> 1112 7.9 / 12.6, but 48, 8, 1024 -> 4096 17.4 / 14.2.  The bound on the rows
// is for batches that meet in one group, whose weights it reads again for every 8 or 16 rows (256 rows in one of 64 groups,
// 2048 -> 1024 28 / 15; 8-bit integers 17 / 10; 512 -> 512 6.9 / 7.6); it holds bytes of the depth in 32 bits.
inline bool few_rows_pay(int rows, int groups, int fi, int fo, bool along_k) {
  const long long used = std::min(groups, rows);
  const long long tiles = used * ceil_div(fo, 2 * kM);
  if (rows > 256 || rows > (tiles < kNumSMs / 4 ? 16 : 8) * used || groups > 65000 || fi > (1 << 29)) return false;
  return along_k ? tiles <= 256 : used * fi <= (24 << 20) / fo;
}

}  // namespace
}  // namespace sptir

#ifndef SPARSETIR_GROUPED_KERNEL_ONLY  // by the files that have entry points of their own

namespace sptir {
namespace {

// The kernel for results of `type`, with tiles of `columns` columns.
template <bool I8, int OUT>
int launch_type(int columns, int type, const CUtensorMap& tm_a, const CUtensorMap& tm_b64, const CUtensorMap& tm_b16, const Args& p,
                cudaStream_t st) {
  return with_type(type, [&](auto o) {
    using O = decltype(o);
    if constexpr (OUT != kWeights)
      if (columns == 128) return launch<I8, OUT, O, 128>(tm_a, tm_b64, tm_b16, p, st);
    return launch<I8, OUT, O, 256>(tm_a, tm_b64, tm_b16, p, st);
  });
}

int check_groups(const char* fn, const int32_t* indptr, int rows, int groups, int fi, int fo, int flags) {
  if (rows < 0 || groups < 0) return fail("%s: negative size", fn);
  if (fi < 1 || fo < 1) return fail("%s: feat_in and feat_out must be positive", fn);
  if (std::max(std::max(rows, groups), std::max(fi, fo)) > kLargestSize ||
      (groups > 0 && static_cast<long long>(fi) * fo > INT64_MAX / groups))
    return fail("%s: too large for 32-bit indices", fn);
  if ((flags & ~SPARSETIR_GROUPED_W_OUT_IN) != 0) return fail("%s: unknown flags %d", fn, flags);
  if (!indptr && groups > 1) return fail("%s: indptr may be null with num_groups 1 only", fn);
  return 0;
}
// For rows, groups, features and columns of p.
int plan_grad(const char* fn, Args* p) {
  auto tiles = [&](int n) { return static_cast<long long>(p->groups) * ceil_div(p->columns, n); };
  const int columns = set_tiles(fn, p, p->features, false, tiles, tiles, ceil_div(ceil_div(p->rows, p->groups), 64),
                                static_cast<long long>(p->groups) * p->columns);
  if (columns < 0) return -1;
  p->nt = ceil_div(p->columns, columns);
  p->per_group = Divisor(p->mt * p->nt);
  return columns;
}
// y = x * W: `type` of the elements of x and W, -1 for 8-bit integers
int product(const char* fn, const void* x, const void* w, int type, void* y, int y_type, const float* xs, const float* ws,
            const int32_t* indptr, int rows, int groups, int fi, int fo, bool out_in, int device_id, cudaStream_t st) {
  const bool i8 = type < 0;
  const int size = i8 ? 1 : 2, depth = 128 / size;
  Args p{};
  p.out = y;
  p.indptr = indptr;
  p.x_scale = xs;
  p.w_scale = ws;
  p.rows = rows;
  p.groups = groups;
  p.k = fi;
  p.features = fo;
  p.a_mn = out_in ? 0 : 1;
  p.wide = wide_rows(y, y_type, fo);
  p.idesc = i8 ? tc05::instr_desc_i8(2 * kM, 0) : tc05::instr_desc(map_format(type), 2 * kM, 0, p.a_mn, 0);
  const int columns = plan_product(fn, &p, fo, depth);
  if (columns < 0) return -1;
  const bool few = few_rows_pay(rows, groups, fi, fo, out_in);
  Operand ox{x, rows, fi, size}, ow{w, static_cast<long long>(groups) * (out_in ? fo : fi), out_in ? fi : fo, size};
  const size_t bytes = ox.copy_bytes() + ow.copy_bytes() + (few ? 0 : part_bytes(p));
  CallScratch cs;
  if (bytes > 0 && take_scratch(device_id, st, bytes, 0, &cs) != 0) return -1;
  char* scratch = cs.scratch;
  if (place_operand(&ox, &scratch, st) != 0 || place_operand(&ow, &scratch, st) != 0) return -1;
  if (few) {
    FewArgs f{ox.data, ow.data, y, xs, ws, indptr, ox.pitch, ow.pitch, rows, groups, fi, fo, fi * size, 0, 0, 0};
    const int done = few_rows(f, type, y_type, out_in, st);
    return done != 0 ? done : return_scratch(cs, st);
  }
  p.parts = scratch;
  CUtensorMap tm_w, tm_x64, tm_x16;
  if (map_operands(&tm_w, &tm_x64, &tm_x16, map_type(type), ow, ox, out_in ? fo : fi, groups, out_in, false) != 0) return -1;
  const int rc = i8 ? launch_type<true, kPlain>(columns, y_type, tm_w, tm_x64, tm_x16, p, st)
                    : launch_type<false, kPlain>(columns, y_type, tm_w, tm_x64, tm_x16, p, st);
  return rc != 0 ? rc : return_scratch(cs, st);
}

}  // namespace

int grouped_timeouts(unsigned int* count) {
  SPTIR_CUDA_OK(cudaMemcpyFromSymbol(count, g_grouped_timeouts, sizeof(unsigned int)));
  return 0;
}

}  // namespace sptir

using namespace sptir;

extern "C" int sparsetir_grouped_mm_raw(const void* x, const void* w, int type, void* y, int y_type, const int32_t* indptr,
                                        int rows, int num_groups, int feat_in, int feat_out, int flags, int device_id,
                                        void* stream) {
  const char* fn = "sparsetir_grouped_mm";
  if (check_groups(fn, indptr, rows, num_groups, feat_in, feat_out, flags) != 0) return -1;
  if (type != SPARSETIR_F16 && type != SPARSETIR_BF16) return fail("%s: x and w are f16 or bf16", fn);
  if (y_type != type && y_type != SPARSETIR_F32) return fail("%s: y has the type of x, or f32", fn);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !w || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return product(fn, x, w, type, y, y_type, nullptr, nullptr, indptr, rows, num_groups, feat_in, feat_out,
                 (flags & SPARSETIR_GROUPED_W_OUT_IN) != 0, device_id, st);
}

extern "C" int sparsetir_grouped_mm_i8_raw(const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale, void* y,
                                           int y_type, const int32_t* indptr, int rows, int num_groups, int feat_in, int feat_out,
                                           int device_id, void* stream) {
  const char* fn = "sparsetir_grouped_mm_i8";
  if (check_groups(fn, indptr, rows, num_groups, feat_in, feat_out, 0) != 0) return -1;
  if (feat_in >= 131072) return fail("%s: feat_in = %d: sums of more than 131071 products may not fit 32 bits", fn, feat_in);
  if (y_type < SPARSETIR_F32 || y_type > SPARSETIR_BF16) return fail("%s: unknown element type %d", fn, y_type);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !x_scale || !w || !w_scale || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return product(fn, x, w, /*type=*/-1, y, y_type, x_scale, w_scale, indptr, rows, num_groups, feat_in, feat_out, /*out_in=*/true,
                 device_id, st);
}

extern "C" int sparsetir_grouped_mm_grad_w_raw(const void* x, const void* dy, int type, void* dw, int dw_type,
                                               const int32_t* indptr, int rows, int num_groups, int feat_in, int feat_out,
                                               int flags, int device_id, void* stream) {
  const char* fn = "sparsetir_grouped_mm_grad_w";
  if (check_groups(fn, indptr, rows, num_groups, feat_in, feat_out, flags) != 0) return -1;
  if (type != SPARSETIR_F16 && type != SPARSETIR_BF16) return fail("%s: x and dy are f16 or bf16", fn);
  if (dw_type != type && dw_type != SPARSETIR_F32) return fail("%s: dw has the type of x, or f32", fn);
  if (num_groups == 0) return 0;
  if (!dw || (rows > 0 && (!x || !dy))) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    const size_t bytes = static_cast<size_t>(num_groups) * feat_in * feat_out * (dw_type == SPARSETIR_F32 ? 4 : 2);
    SPTIR_CUDA_OK(cudaMemsetAsync(dw, 0, bytes, st));
    return 0;
  }
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  const bool out_in = (flags & SPARSETIR_GROUPED_W_OUT_IN) != 0;
  Args p{};
  p.out = dw;
  p.indptr = indptr;
  p.rows = rows;
  p.groups = num_groups;
  p.features = out_in ? feat_in : feat_out;
  p.columns = out_in ? feat_out : feat_in;
  p.wide = wide_rows(dw, dw_type, p.features);
  p.idesc = tc05::instr_desc(map_format(type), 2 * kM, 0, 1, 1);
  const int columns = plan_grad(fn, &p);
  if (columns < 0) return -1;
  Operand oa{out_in ? x : dy, rows, p.features, 2}, ob{out_in ? dy : x, rows, p.columns, 2};
  const size_t bytes = oa.copy_bytes() + ob.copy_bytes() + part_bytes(p);
  CallScratch cs;
  if (bytes > 0 && take_scratch(device_id, st, bytes, 0, &cs) != 0) return -1;
  char* scratch = cs.scratch;
  if (place_operand(&oa, &scratch, st) != 0 || place_operand(&ob, &scratch, st) != 0) return -1;
  p.parts = scratch;
  CUtensorMap tm_a, tm_b;
  const CUtensorMapDataType dt = map_type(type);
  if (make_tmap_2d(&tm_a, dt, oa.data, oa.cols, rows, oa.pitch, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B) != 0 ||
      make_tmap_2d(&tm_b, dt, ob.data, ob.cols, rows, ob.pitch, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B) != 0)
    return -1;
  const int rc = launch_type<false, kWeights>(columns, dw_type, tm_a, tm_b, tm_b, p, st);
  return rc != 0 ? rc : return_scratch(cs, st);
}

extern "C" int sparsetir_grouped_mm_workspace(int rows, int num_groups, int feat_in, int feat_out, int element_bytes, int flags,
                                              size_t* scratch_bytes) {
  const char* fn = "sparsetir_grouped_mm_workspace";
  const int32_t some = 0;  // pointers are not looked at
  if (check_block(fn, &some, rows, num_groups, feat_in, feat_out, false, flags, SPARSETIR_GROUPED_W_OUT_IN | SPARSETIR_GATED_GELU) != 0) return -1;
  if ((element_bytes != 1 && element_bytes != 2) || !scratch_bytes) return fail("%s: bad argument", fn);
  *scratch_bytes = 0;
  if (rows == 0 || num_groups == 0) return 0;
  const bool out_in = element_bytes == 1 || (flags & SPARSETIR_GROUPED_W_OUT_IN) != 0;
  // copies of both operands, whatever their addresses, and the sums of units that share a tile
  auto copy = [&](long long n, int cols) -> size_t { return (Operand{nullptr, n, cols, element_bytes}.padded() * n + 255) / 256 * 256; };
  Args p{};
  p.rows = rows;
  p.groups = num_groups;
  p.k = feat_in;
  p.features = feat_out;
  if (plan_product(fn, &p, feat_out, 128 / element_bytes) < 0) return -1;
  size_t parts = part_bytes(p);
  if (element_bytes == 1) {  // of 8-bit integers, or of floating point
    if (plan_f8(fn, &p, feat_out) != 0) return -1;
    parts = std::max(parts, part_bytes(p));
  }
  // W along the depth, or, where the flags do not say so, the larger of the two: a gated product has it so without a flag
  const size_t along_k = copy(static_cast<long long>(num_groups) * feat_out, feat_in);
  const size_t product = (out_in ? along_k : std::max(along_k, copy(static_cast<long long>(num_groups) * feat_in, feat_out))) + parts;
  p.features = out_in ? feat_in : feat_out;
  p.columns = out_in ? feat_out : feat_in;
  if (plan_grad(fn, &p) < 0) return -1;
  *scratch_bytes = copy(rows, feat_in) + std::max(product, element_bytes == 1 ? 0 : copy(rows, feat_out) + part_bytes(p));
  return 0;
}
#endif
