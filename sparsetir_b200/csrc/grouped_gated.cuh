// Epilogues of grouped_kernel (grouped.cu, which includes this): a gated block, the gradient of one, and sums with a scale for each
// 128 of K.  All take the sums as fragments (tmem_ld16x32): 16 lanes of TMEM, 32 columns, v[4 i + 2 h + c] = lane 8 h + l / 4 of the 16, column
// 8 i + 2 (l % 4) + c, for lane l of the warp.
//   Gated: of the 32 rows of W that a warp's lanes of TMEM stand for, the first 16 are the gate's and the last 16 the other projection's of
//   the same features: the two fragments that a thread loads belong together, and nothing is exchanged.
#ifndef SPARSETIR_B200_GROUPED_GATED_CUH_
#define SPARSETIR_B200_GROUPED_GATED_CUH_

#include <type_traits>

namespace sptir {
namespace {

// Registers of a thread in the kernel with scaled sums: a thread of the epilogue holds 128 sums, the others need few.  What a block
// was launched with is shared out again: (kN = 256) 128 * 40 + 256 * 232 = 384 * 168, (128) 128 * 40 + 128 * 216 = 256 * 128.
template <int N> struct F8Registers {
  static constexpr int kOthers = 40;
  static constexpr int kEpilogue = N == 256 ? 232 : 216;
};

// The scales of 8-bit floating point on their way to an epilogue warp whose columns are rows of x: every lane copies its four columns' and those of
// W's rows, four steps of K ahead, into places that it alone reads, and multiplies them for all lanes when their step comes.
template <int OUT>
struct Scales {
  static constexpr int kW = OUT == kGated ? 3 : 1;  // of W: gated: the gate's, and two of the other projection's, whose rows may lie in two blocks
  static constexpr int kSlots = 4, kSlot = 128 + 32 * kW;  // floats
  static constexpr int kBytes = kSlots * kSlot * 4;
  static constexpr int kArray = 132;  // scales of 128 columns times one of W's; arrays start in different banks
  static constexpr int kProducts = 2 * kW * kArray * 4;  // bytes of two steps'
  const float* xs;
  const float* ws[kW];
  uint32_t mine;  // the lane's first place
  int live, steps, rows, asked;
  int array;      // that holds the scales of the lane's row of W

  __device__ __forceinline__ void begin(const Args& p, const Tile& t, int feat0, int first, int columns, float* slots, int lane) {
    live = min(t.n - first, columns);
    steps = t.steps;
    rows = p.rows;
    asked = 0;
    mine = tc05::smem_u32(slots + lane);
    const int blocks = (p.k + SPARSETIR_F8_BLOCK - 1) / SPARSETIR_F8_BLOCK;
    const int of_w = ((OUT == kGated ? 2 : 1) * p.features + SPARSETIR_F8_BLOCK - 1) / SPARSETIR_F8_BLOCK;
    auto block = [&](int f) { return min(f, p.features - 1) / SPARSETIR_F8_BLOCK; };
    auto of = [&](int b) { return p.w_scale + (static_cast<size_t>(t.group) * of_w + b) * blocks + t.step0; };
    ws[0] = of(block(feat0));
    array = 0;
    if constexpr (OUT == kGated) {
      auto up = [&](int f) { return (p.features + min(f, p.features - 1)) / SPARSETIR_F8_BLOCK; };
      ws[1] = of(up(feat0));
      ws[2] = of(up(feat0 + 15));
      if (lane >= 16) array = up(feat0 + lane - 16) == up(feat0) ? 1 : 2;
    }
    xs = p.x_scale + static_cast<size_t>(t.step0) * p.rows + t.col0 + first + lane;
#pragma unroll
    for (int i = 0; i < kSlots - 1; ++i) ask(lane);
  }
  __device__ __forceinline__ static void copy4(uint32_t to, const float* from, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(in ? 4 : 0) : "memory");
  }
  // The next step's; past the last none
  __device__ __forceinline__ void ask(int lane) {
    if (asked < steps) {
      const uint32_t to = mine + (asked & (kSlots - 1)) * kSlot * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) copy4(to + 128 * j, lane + 32 * j < live ? xs + 32 * j : ws[0], lane + 32 * j < live);
#pragma unroll
      for (int i = 0; i < kW; ++i) copy4(to + 512 + 128 * i, ws[i] + asked, true);
      xs += rows;
    }
    ++asked;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Step k's products of scales into the arrays of `to`
  __device__ __forceinline__ void multiply(int k, float* slots, float* to, int lane) {
    ask(lane);
    asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 1) : "memory");
    const float* from = slots + lane + (k & (kSlots - 1)) * kSlot;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = from[32 * j];
#pragma unroll
      for (int i = 0; i < kW; ++i) to[i * kArray + 32 * j + lane] = x * from[128 + 32 * i];
    }
  }
};

// An epilogue warp's share of a tile: features feat0 and so on, columns first, first + step and so on up to last, 32 at a time.
template <class OutT>
struct Warp {
  const Args& p;
  const Tile& t;
  const int feat0, first, step, last;
  unsigned char* const staged;
  const int lane;
  const int feats;  // live ones from feat0 on, may be <= 0

  __device__ __forceinline__ Warp(const Args& args, const Tile& tile, int feat, int column, int stride, int columns, unsigned char* mem, int l)
      : p(args), t(tile), feat0(feat), first(column), step(stride), last(min(tile.n, column + columns)), staged(mem), lane(l), feats(args.features - feat) {}

  // Row of column c of the tile
  __device__ __forceinline__ size_t row(int c) const { return static_cast<size_t>(t.col0) + c; }

  // ---- one element to a store, whatever the alignment; eight lanes have neighbouring features
  template <class O>
  __device__ __forceinline__ void direct(O* to, size_t pitch, int live, const float* v, int c0) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int f = 8 * ((i >> 1) & 1) + lane / 4, c = 8 * (i >> 2) + 2 * (lane & 3) + (i & 1);
      if (f < live && c0 + c < t.n) to[c * pitch + f] = from_float<O>(v[i]);
    }
  }
  // Sums of a unit that shares the depth: both fragments' rows of the left operand
  template <int OUT>
  __device__ __forceinline__ void to_parts(const float* a, const float* b, int c0) const {
    const size_t pitch = OUT == kGated ? 2 * static_cast<size_t>(p.features) : p.features;
    float* to = static_cast<float*>(p.parts) + t.split * p.part + row(c0) * pitch + feat0;
    direct(to, pitch, feats, a, c0);
    if constexpr (OUT == kGated) direct(to + p.features, pitch, feats, b, c0);
    else direct(to + 16, pitch, feats - 16, b, c0);
  }
  template <int OUT>
  __device__ __forceinline__ void zeros() const {
    const float none[16] = {};
    for (int c0 = first; c0 < last; c0 += step) to_parts<OUT>(none, none, c0);
  }

  // ---- 16-bit elements at 16-byte addresses, through shared memory: 32 rows (columns of the tile) of 64 bytes, pieces of 16 bytes exchanged
  // so that neither side collides.  v[q]: features 8 q + l / 4, columns 8 i + 2 (l % 4) and the next
  __device__ __forceinline__ static uint32_t place64(int r, int q) { return static_cast<uint32_t>(r * 64 + ((q ^ ((r >> 1) & 3)) << 4)); }
  __device__ __forceinline__ void put64(int at, int i, uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3) const {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                     tc05::smem_u32(staged) + at + place64(8 * i + (lane & 7), lane >> 3)),
                 "r"(v0), "r"(v1), "r"(v2), "r"(v3)
                 : "memory");
  }
  __device__ __forceinline__ void get64(int at, int i, uint32_t (&v)[4]) const {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(tc05::smem_u32(staged) + at + place64(8 * i + (lane & 7), lane >> 3))
                 : "memory");
  }
  // A lane has the piece lane % 4 of the rows lane / 4, 8 further and so on: to `to`, where its piece of row lane / 4 goes
  __device__ __forceinline__ void leave64(int at, OutT* to, size_t pitch, bool live, int c0) const {
    const unsigned char* from = staged + at + place64(lane >> 2, lane & 3);  // rows 8 apart alike
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(from + 8 * i * 64);
      if (live && c0 + 8 * i + (lane >> 2) < t.n) *reinterpret_cast<uint4*>(to + 8 * i * pitch) = v;
    }
  }
  // The same for 16 features: rows of 32 bytes
  __device__ __forceinline__ static uint32_t place32(int r, int q) { return static_cast<uint32_t>(r * 32 + ((q ^ ((r >> 2) & 1)) << 4)); }
  __device__ __forceinline__ void put32(int at, int i, uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3) const {  // of columns 8 i.., 8 i + 8..
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                     tc05::smem_u32(staged) + at + place32(8 * (i + (lane >> 4)) + (lane & 7), (lane >> 3) & 1)),
                 "r"(v0), "r"(v1), "r"(v2), "r"(v3)
                 : "memory");
  }
  __device__ __forceinline__ void leave32(int at, OutT* to, size_t pitch, bool live, int c0) const {
    const unsigned char* from = staged + at + place32(lane >> 1, lane & 1);  // rows 16 apart alike
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(from + 16 * i * 32);
      if (live && c0 + 16 * i + (lane >> 1) < t.n) *reinterpret_cast<uint4*>(to + 16 * i * pitch) = v;
    }
  }

  // ---- what becomes of 32 columns' sums; next(): they are not needed any more
  template <class Next>
  __device__ __forceinline__ void plain(const float* a, const float* b, int c0, Next&& next) const {
    OutT* to = static_cast<OutT*>(p.out) + row(c0) * p.features + feat0;
    if constexpr (sizeof(OutT) == 2) {
      if (p.wide) {
        __syncwarp();  // the reads of the last 32 columns are over
#pragma unroll
        for (int i = 0; i < 4; ++i)
          put64(0, i, pack2<OutT>(a[4 * i], a[4 * i + 1]), pack2<OutT>(a[4 * i + 2], a[4 * i + 3]), pack2<OutT>(b[4 * i], b[4 * i + 1]),
                pack2<OutT>(b[4 * i + 2], b[4 * i + 3]));
        next();
        __syncwarp();
        leave64(0, to + static_cast<size_t>(lane >> 2) * p.features + 8 * (lane & 3), p.features, 8 * (lane & 3) < feats, c0);
        return;
      }
    }
    direct(to, p.features, feats, a, c0);
    direct(to + 16, p.features, feats - 16, b, c0);
    next();
  }
  template <class Next>
  __device__ __forceinline__ void gated(const float* g, const float* u, int c0, Next&& next) const {
    const size_t width = p.features;
    OutT* const to = static_cast<OutT*>(p.out) + row(c0) * width + feat0;
    OutT* const kept = static_cast<OutT*>(p.hidden) + row(c0) * 2 * width + feat0;
    if (p.wide) {
      uint32_t act[8];
      auto activate = [&](auto gelu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const Two a = Gate::act<gelu.value>(Two(g[2 * i], g[2 * i + 1]), Two(u[2 * i], u[2 * i + 1]));
          act[i] = pack2<OutT>(a.lo(), a.hi());
        }
      };
      if (p.gate.gelu) activate(std::true_type{});
      else activate(std::false_type{});
      __syncwarp();  // the reads of the last 32 columns are over
      put32(kStagedBytes, 0, act[0], act[1], act[2], act[3]);
      put32(kStagedBytes, 2, act[4], act[5], act[6], act[7]);
      if (p.hidden != nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          put64(0, i, pack2<OutT>(g[4 * i], g[4 * i + 1]), pack2<OutT>(g[4 * i + 2], g[4 * i + 3]), pack2<OutT>(u[4 * i], u[4 * i + 1]),
                pack2<OutT>(u[4 * i + 2], u[4 * i + 3]));
      }
      next();
      __syncwarp();
      leave32(kStagedBytes, to + static_cast<size_t>(lane >> 1) * width + 8 * (lane & 1), width, 8 * (lane & 1) < feats, c0);
      if (p.hidden != nullptr)  // pieces 0 and 1 are the gate's
        leave64(0, kept + static_cast<size_t>(lane >> 2) * 2 * width + ((lane & 2) != 0 ? width : 0) + 8 * (lane & 1), 2 * width,
                8 * (lane & 1) < feats, c0);
      return;
    }
    float act[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) act[i] = p.gate.act(g[i], u[i]);
    direct(to, width, feats, act, c0);
    if (p.hidden != nullptr) {
      direct(kept, 2 * width, feats, g, c0);
      direct(kept + width, 2 * width, feats, u, c0);
    }
    next();
  }

  // The projections of 32 features and columns, for the gradient: asked for ahead, put where put64 puts them.
  struct Ahead { uint4 g[4], u[4]; };
  __device__ __forceinline__ void ask(int c0, Ahead& h) const {
    const size_t width = p.features;
    const OutT* from = static_cast<const OutT*>(p.hidden_in) + row(c0 + (lane >> 2)) * 2 * width + feat0 + 8 * (lane & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (8 * (lane & 3) < feats && c0 + 8 * i + (lane >> 2) < t.n) {
        h.g[i] = ld_global(reinterpret_cast<const uint4*>(from + 8 * i * 2 * width));
        h.u[i] = ld_global(reinterpret_cast<const uint4*>(from + 8 * i * 2 * width + width));
      } else {
        h.g[i] = h.u[i] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
  __device__ __forceinline__ static Two halves_of(uint32_t v) {
    if constexpr (std::is_same<OutT, __half>::value) {
      const float2 f = __half22float2(reinterpret_cast<const __half2&>(v));
      return Two(f.x, f.y);
    } else {
      return Two(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
  }
  template <class Next>
  __device__ __forceinline__ void gated_grad(const float* da, const float* db, int c0, Ahead& ahead, Next&& next) const {
    const size_t width = p.features;
    OutT* const dg = static_cast<OutT*>(p.hidden) + row(c0) * 2 * width + feat0;
    if (p.wide) {
      __syncwarp();  // the reads of the last 32 columns are over
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = static_cast<int>(place64(8 * i + (lane >> 2), lane & 3));
        *reinterpret_cast<uint4*>(staged + at) = ahead.g[i];
        *reinterpret_cast<uint4*>(staged + kStagedBytes + at) = ahead.u[i];
      }
      if (c0 + step < t.n) ask(c0 + step, ahead);
      __syncwarp();
      uint32_t act[16];
      auto differentiate = [&](auto gelu) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t g[4], u[4], og[4], ou[4];
          get64(0, i, g);
          get64(kStagedBytes, i, u);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float* d = (q < 2 ? da : db) + 4 * i + 2 * (q & 1);
            Two xg, xu, xa;
            Gate::grad<gelu.value>(halves_of(g[q]), halves_of(u[q]), Two(d[0], d[1]), &xg, &xu, &xa);
            og[q] = pack2<OutT>(xg.lo(), xg.hi());
            ou[q] = pack2<OutT>(xu.lo(), xu.hi());
            act[4 * i + q] = pack2<OutT>(xa.lo(), xa.hi());
          }
          __syncwarp();
          put64(0, i, og[0], og[1], og[2], og[3]);  // in the place of what was read
          put64(kStagedBytes, i, ou[0], ou[1], ou[2], ou[3]);
        }
      };
      if (p.gate.gelu) differentiate(std::true_type{});
      else differentiate(std::false_type{});
      next();
      __syncwarp();
      OutT* const to = dg + static_cast<size_t>(lane >> 2) * 2 * width + 8 * (lane & 3);
      const bool live = 8 * (lane & 3) < feats;
      leave64(0, to, 2 * width, live, c0);
      leave64(kStagedBytes, to + width, 2 * width, live, c0);
      if (p.out != nullptr) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) put64(0, i, act[4 * i], act[4 * i + 1], act[4 * i + 2], act[4 * i + 3]);
        __syncwarp();
        leave64(0, static_cast<OutT*>(p.out) + row(c0 + (lane >> 2)) * width + feat0 + 8 * (lane & 3), width, live, c0);
      }
      return;
    }
    const OutT* const h = static_cast<const OutT*>(p.hidden_in) + row(c0) * 2 * width + feat0;
    OutT* const act = static_cast<OutT*>(p.out) + row(c0) * width + feat0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int f = 16 * (i >> 4) + 8 * ((i >> 1) & 1) + lane / 4, c = 8 * ((i >> 2) & 3) + 2 * (lane & 3) + (i & 1);
      if (f >= feats || c0 + c >= t.n) continue;
      const size_t at = c * 2 * width + f;
      float xg, xu, xa;
      p.gate.grad(to_float(ld_global(h + at)), to_float(ld_global(h + at + width)), i < 16 ? da[i & 15] : db[i & 15], &xg, &xu, &xa);
      dg[at] = from_float<OutT>(xg);
      dg[at + width] = from_float<OutT>(xu);
      if (p.out != nullptr) act[c * width + f] = from_float<OutT>(xa);
    }
    next();
  }

  // ---- sums that are complete in TMEM; take(): the warp's last columns are in registers, the accumulator may be written again
  template <int OUT, class Take>
  __device__ __forceinline__ void emit(uint32_t taddr, Ahead& ahead, Take&& take) const {
    if (first >= last) {
      take();
      return;
    }
    uint32_t a[16], b[16];
    tc05::tmem_ld16x32(taddr + first, a);
    tc05::tmem_ld16x32(taddr + (16u << 16) + first, b);
    for (int c0 = first; c0 < last; c0 += step) {
      tc05::tmem_ld_wait(a);
      tc05::tmem_ld_wait(b);
      if (c0 + step >= last) take();
      float va[16], vb[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        va[i] = __uint_as_float(a[i]);
        vb[i] = __uint_as_float(b[i]);
      }
      auto next = [&]() {  // the next columns while these leave
        if (c0 + step >= last) return;
        tc05::tmem_ld16x32(taddr + c0 + step, a);
        tc05::tmem_ld16x32(taddr + (16u << 16) + c0 + step, b);
      };
      if (p.splits > 1) {
        to_parts<OUT>(va, vb, c0);
        next();
      } else if constexpr (OUT == kGated) {
        gated(va, vb, c0, next);
      } else if constexpr (OUT == kGatedGrad) {
        gated_grad(va, vb, c0, ahead, next);
      } else {
        plain(va, vb, c0, next);
      }
    }
  }
  __device__ __forceinline__ void taken(uint64_t* empty) const {
    tc05::fence_before_sync();
    __syncwarp();
    if (lane == 0) tc05::pair::arrive(tc05::pair::at_first(empty));
  }
  // false: the wait ran out
  template <int OUT>
  __device__ __forceinline__ bool out_of_tmem(uint32_t taddr, uint64_t* full, uint64_t* empty, uint32_t parity) const {
    Ahead ahead;
    if (OUT == kGatedGrad && p.wide != 0 && p.splits == 1 && first < last) ask(first, ahead);
    if (!__all_sync(0xffffffffu, tc05::mbar_wait(full, parity))) return false;
    tc05::fence_after_sync();
    emit<OUT>(taddr, ahead, [&] { taken(empty); });
    return true;
  }

  // ---- a tile of 8-bit floating point: the sums of every 128 of K come by themselves, from accumulators that change by turns, and are
  // scaled and added in registers: lane = row of W, 128 columns.  At the end the sums go where the last came from, to leave like others.
  // false: a wait ran out
  template <int OUT>
  __device__ __forceinline__ bool add_scaled(uint32_t taddr, int buffer, uint64_t* full, uint64_t* empty, int acc, Scales<OUT>& scales,
                                             float* slots) const {
    float sum[128];
#pragma unroll
    for (int i = 0; i < 128; ++i) sum[i] = 0.f;
    const int live = last - first;  // columns, may be <= 0
    __syncwarp();  // the last tile has left shared memory
    for (int k = 0; k < t.steps; ++k, ++acc) {
      float* const products = reinterpret_cast<float*>(staged) + (k & 1) * (Scales<OUT>::kW * Scales<OUT>::kArray);
      scales.multiply(k, slots, products, lane);
      __syncwarp();
      const float* const s = products + scales.array * Scales<OUT>::kArray;
      const int buf = acc & 1;
      if (!__all_sync(0xffffffffu, tc05::mbar_wait(full + buf, (acc >> 1) & 1))) return false;
      tc05::fence_after_sync();
      const uint32_t from = taddr + buf * buffer + first;
      const bool ends = k + 1 == t.steps;
      if (live <= 0) {
        if (!ends) taken(empty + buf);
        continue;
      }
      uint32_t r[2][16];
      tc05::tmem_ld16(from, r[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (16 * j >= live) break;
        tc05::tmem_ld_wait(r[j & 1]);
        if (j < 7 && 16 * (j + 1) < live) tc05::tmem_ld16(from + 16 * (j + 1), r[(j + 1) & 1]);
        else if (!ends) taken(empty + buf);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 sc = *reinterpret_cast<const float4*>(s + 16 * j + i);
          const uint32_t* v = r[j & 1] + i;
          float* to = sum + 16 * j + i;
          to[0] = fmaf(__uint_as_float(v[0]), sc.x, to[0]);
          to[1] = fmaf(__uint_as_float(v[1]), sc.y, to[1]);
          to[2] = fmaf(__uint_as_float(v[2]), sc.z, to[2]);
          to[3] = fmaf(__uint_as_float(v[3]), sc.w, to[3]);
        }
      }
      if (!ends) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (32 * j >= live) break;
        uint32_t out[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) out[i] = __float_as_uint(sum[32 * j + i]);
        tc05::tmem_st32(from + 32 * j, out);
      }
      tc05::tmem_st_wait();
      __syncwarp();  // the scales are read
    }
    return true;
  }
};

// ---- 8-bit floating point, tiles of 256 rows: the rows of x are those of the tensor core's left operand, 256 features (gated: 128 and 128, 16 by
// 16) its columns.  A lane's 128 sums are of one row and, but for a gated block's other projection, of one block of W: they share one scale, and
// nothing but TMEM is read between one step of K and the next.  Us, 65,536 rows in 64 equal groups, 2048 -> 2048: with the features as the left
// operand and the rows' scales out of shared memory 512 to 566, this way 367, with the loads of TMEM in flight across the steps 328, with waits that
// ask again and again 310 (the same product of 8-bit integers, scaled at the end alone, 228).  What is left is the way there and back: from the issue of
// a step's MMAs (512 clocks) to their sums in registers 1,160 clocks, 350 to take them and 200 until the issuing thread knows, with two accumulators
// on the way.  The same in two halves of 128 columns with barriers of their own was slower (345), and TMEM has no room for a third of 256.
template <int OUT, class OutT>
struct RowWarp {
  static constexpr bool kTwo = OUT == kGated;
  const Args& p;
  const Tile t;
  const int feat0;        // of the result, of the warp's first column
  const int columns;      // that the tensor core fills for the warp, 128 at most, may be <= 0
  const int row0, rows;   // of the warp's lanes: the first, and how many live, may be <= 0 or > 32
  unsigned char* const staged;
  const int lane;
  float sum[128];

  __device__ __forceinline__ RowWarp(const Args& args, const Tile& tile, int n_mma, int half, int first_row, unsigned char* mem, int l)
      : p(args), t(tile), feat0(tile.feat0 + half * (kTwo ? 64 : 128)), columns(min(n_mma - half * 128, 128)), row0(tile.col0 + first_row),
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
    if (lane == 0) tc05::pair::arrive(tc05::pair::at_first(empty));
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

// The sums of the units that share a tile, added in their order, and what becomes of them: thread = a feature of a row
template <int OUT, class T>
__global__ void __launch_bounds__(256) join_gated_kernel(const __grid_constant__ Args p) {
  chain_wait();
  const long long row = blockIdx.y + static_cast<long long>(blockIdx.z) * gridDim.y;
  const int feat = blockIdx.x * 256 + threadIdx.x;
  if (row >= p.rows || feat >= p.features) return;
  if (p.indptr != nullptr && (row < ld_global(p.indptr) || row >= ld_global(p.indptr + p.groups))) return;  // of no group
  const size_t width = p.features;
  const float* from = static_cast<const float*>(p.parts) + static_cast<size_t>(row) * (OUT == kGated ? 2 : 1) * width + feat;
  float a = 0.f, b = 0.f;
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) {
    a += ld_global(from + s * p.part);
    if constexpr (OUT == kGated) b += ld_global(from + s * p.part + width);
  }
  const size_t at = static_cast<size_t>(row) * width + feat, two = static_cast<size_t>(row) * 2 * width + feat;
  T* const hidden = static_cast<T*>(p.hidden);
  T* const out = static_cast<T*>(p.out);
  if constexpr (OUT == kGated) {
    out[at] = from_float<T>(p.gate.act(a, b));
    if (hidden != nullptr) {
      hidden[two] = from_float<T>(a);
      hidden[two + width] = from_float<T>(b);
    }
  } else {
    const T* const h = static_cast<const T*>(p.hidden_in);
    float xg, xu, xa;
    p.gate.grad(to_float(ld_global(h + two)), to_float(ld_global(h + two + width)), a, &xg, &xu, &xa);
    hidden[two] = from_float<T>(xg);
    hidden[two + width] = from_float<T>(xu);
    if (out != nullptr) out[at] = from_float<T>(xa);
  }
}

}  // namespace
}  // namespace sptir
#endif  // SPARSETIR_B200_GROUPED_GATED_CUH_
