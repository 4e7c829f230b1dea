// Epilogues of grouped_kernel (grouped.cu, which includes this): a gated block and the gradient of one.  Both take the sums as fragments (tmem_ld16x32): 16 lanes of TMEM, 32 columns, v[4 i + 2 h + c] = lane 8 h + l / 4 of the 16, column
// 8 i + 2 (l % 4) + c, for lane l of the warp.
//   Gated: of the 32 rows of W that a warp's lanes of TMEM stand for, the first 16 are the gate's and the last 16 the other projection's of
//   the same features: the two fragments that a thread loads belong together, and nothing is exchanged.
#ifndef SPARSETIR_B200_GROUPED_GATED_CUH_
#define SPARSETIR_B200_GROUPED_GATED_CUH_

#include <type_traits>

namespace sptir {
namespace {

// An epilogue warp's share of a tile: features feat0 and so on, columns first, first + step and so on 32 at a time.
template <class OutT>
struct Warp {
  const GatedArgs& p;
  const Tile& t;
  const int feat0, first, step;
  unsigned char* const staged;
  const int lane;
  const int feats;  // live ones from feat0 on, may be <= 0

  __device__ __forceinline__ Warp(const GatedArgs& args, const Tile& tile, int feat, int column, int stride, unsigned char* mem, int l)
      : p(args), t(tile), feat0(feat), first(column), step(stride), staged(mem), lane(l), feats(args.features - feat) {}

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
    for (int c0 = first; c0 < t.n; c0 += step) to_parts<OUT>(none, none, c0);
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
  }
  template <class Next>
  __device__ __forceinline__ void gated_grad_any(const float* da, const float* db, int c0, Next&& next) const {
    const size_t width = p.features;
    OutT* const dg = static_cast<OutT*>(p.hidden) + row(c0) * 2 * width + feat0;
    // At any address: the sums through shared memory, lane = feature, eight columns' projections on their way at a time (14,774 rows in 8
    // groups, 1024 -> 826: 138 us, one element after the other out of the fragments 243).  An instantiation of its own: its registers cost
    // the form for aligned rows 10% (65,536 rows in 64 groups, 2048 -> 1024: 291 us, with both in one kernel 316).
    float* const sums = reinterpret_cast<float*>(staged);
    auto place = [](int c, int f) { return c * 32 + (f ^ ((c & 14) << 1)); };  // lanes of a column, and of a fragment, in different banks
    __syncwarp();  // the reads of the last 32 columns are over
#pragma unroll
    for (int i = 0; i < 32; ++i)
      sums[place(8 * ((i >> 2) & 3) + 2 * (lane & 3) + (i & 1), 16 * (i >> 4) + 8 * ((i >> 1) & 1) + lane / 4)] = i < 16 ? da[i & 15] : db[i & 15];
    next();
    __syncwarp();
    const OutT* const h = static_cast<const OutT*>(p.hidden_in) + row(c0) * 2 * width + feat0 + lane;
    OutT* const act = static_cast<OutT*>(p.out) + row(c0) * width + feat0 + lane;
    const int n = min(32, t.n - c0);
    for (int c = 0; lane < feats && c < n; c += 8) {
      OutT hg[8], hu[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        hg[q] = hu[q] = OutT{};
        if (c + q < n) {
          hg[q] = ld_global(h + (c + q) * 2 * width);
          hu[q] = ld_global(h + (c + q) * 2 * width + width);
        }
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (c + q >= n) break;
        float xg, xu, xa;
        p.gate.grad(to_float(hg[q]), to_float(hu[q]), sums[place(c + q, lane)], &xg, &xu, &xa);
        OutT* const to = dg + (c + q) * 2 * width + lane;
        to[0] = from_float<OutT>(xg);
        to[width] = from_float<OutT>(xu);
        if (p.out != nullptr) act[(c + q) * width] = from_float<OutT>(xa);
      }
    }
    __syncwarp();
  }

  // ---- sums that are complete in TMEM; take(): the warp's last columns are in registers, the accumulator may be written again
  template <int OUT, class Take>
  __device__ __forceinline__ void emit(uint32_t taddr, Ahead& ahead, Take&& take) const {
    if (first >= t.n) {
      take();
      return;
    }
    uint32_t a[16], b[16];
    tc05::tmem_ld16x32(taddr + first, a);
    tc05::tmem_ld16x32(taddr + (16u << 16) + first, b);
    for (int c0 = first; c0 < t.n; c0 += step) {
      tc05::tmem_ld_wait(a);
      tc05::tmem_ld_wait(b);
      if (c0 + step >= t.n) take();
      float va[16], vb[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        va[i] = __uint_as_float(a[i]);
        vb[i] = __uint_as_float(b[i]);
      }
      auto next = [&]() {  // the next columns while these leave
        if (c0 + step >= t.n) return;
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
        gated_grad_any(va, vb, c0, next);
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
    if (OUT == kGatedGrad && p.splits == 1 && first < t.n) ask(first, ahead);
    if (!__all_sync(0xffffffffu, tc05::mbar_wait(full, parity))) return false;
    tc05::fence_after_sync();
    emit<OUT>(taddr, ahead, [&] { taken(empty); });
    return true;
  }
};

// The sums of the units that share a tile, added in their order, and what becomes of them: thread = a feature of a row
template <int OUT, class T>
__global__ void __launch_bounds__(256) join_gated_kernel(const __grid_constant__ GatedArgs p) {
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
