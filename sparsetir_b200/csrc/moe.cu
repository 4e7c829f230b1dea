// Router of a mixture of experts, and the exchange of rows between the order of the tokens and that of the experts.
// The products between the two are in grouped.cu.
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "launch.cuh"
#include "lowp.cuh"

namespace sptir {
namespace {

constexpr int kWarps = 8;
constexpr unsigned kFull = 0xffffffffu;

// ---- router ---------------------------------------------------------------------------------------------------------

// Floats in an order of unsigned integers: larger float, larger key.  0 for what masks an expert (-inf, NaN); both
// zeros have one key, so that the lower index wins between them as between other equal logits.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((b >> 31) != 0u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) != 0u ? 0x80000000u : 0xffffffffu));
}
// exp(v - top) for a logit of a token whose largest is top; 0 for a masked one (-inf), 1 for the largest even if it is +inf
__device__ __forceinline__ float over_top(float v, float top) {
  const float e = expf(v - top);
  return v == top ? 1.f : v > -INFINITY ? e : 0.f;
}

// Reductions over the L lanes of a token.
template <int L>
__device__ __forceinline__ uint32_t most_of(uint32_t v) {
  if constexpr (L == 32) {
    return __reduce_max_sync(kFull, v);
  } else {
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) v = max(v, __shfl_xor_sync(kFull, v, o));
    return v;
  }
}
template <int L>
__device__ __forceinline__ int least_of(int v) {
  if constexpr (L == 32) {
    return __reduce_min_sync(kFull, v);
  } else {
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) v = min(v, __shfl_xor_sync(kFull, v, o));
    return v;
  }
}
template <int L>
__device__ __forceinline__ float sum_of(float v) {
#pragma unroll
  for (int o = L / 2; o >= 1; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// A token's logits, R to each of L lanes: lane l has those of the experts l, l + L, ...; -inf for what masks an expert.
// Returns the largest of the token, NaN if all are masked.
template <class T, int L, int R>
__device__ __forceinline__ float load_logits(const T* row, int num_experts, int l, bool live, float (&v)[R]) {
  constexpr int G = R < 8 ? R : 8;  // in flight
#pragma unroll
  for (int r0 = 0; r0 < R; r0 += G) {
    T raw[G];
#pragma unroll
    for (int r = 0; r < G; ++r)
      if (live && l + L * (r0 + r) < num_experts) raw[r] = ld_global(row + l + L * (r0 + r));
#pragma unroll
    for (int r = 0; r < G; ++r) {
      const float x = live && l + L * (r0 + r) < num_experts ? to_float(raw[r]) : -INFINITY;
      v[r0 + r] = x > -INFINITY ? x : -INFINITY;
    }
  }
  float most = v[0];
#pragma unroll
  for (int r = 1; r < R; ++r) most = fmaxf(most, v[r]);
  return key_value(most_of<L>(order_key(most)));
}

// The router is two launches, or one where a single block has all tokens.  Each block of the first chooses for its share of
// the tokens, L lanes to a token, and counts the pairs of every expert; each block of the second sums the counts of all
// shares (they are few: 148 at most) and places its share's pairs.  Nothing depends on the order in which blocks run.
constexpr int kRouteThreads = 1024, kRouteWarps = kRouteThreads / 32;
constexpr int kRouteAlone = 32;   // tokens that a single block takes
constexpr int kRouteTokens = 32;   // of a share at least; more where there would be over 148 shares

struct PlaceShared {
  int next[SPARSETIR_MOE_MAX_EXPERTS];  // where the share's next pair of every expert goes
  uint4 count[SPARSETIR_MOE_MAX_EXPERTS][kRouteWarps / 16];  // a byte for every warp
  int sums[kRouteWarps];
};

// next[e] += the sum of total[0 .. e-1], one expert to a thread; the sum of all is returned.
__device__ __forceinline__ int add_bases(PlaceShared& s, int total) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int upto = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += up;
  }
  if (lane == 31) s.sums[warp] = upto;
  __syncthreads();
  const int sum = s.sums[lane];
  const int before = __reduce_add_sync(kFull, lane < warp ? sum : 0);
  s.next[tid] += before + upto - total;
  return __reduce_add_sync(kFull, sum);
}
// Sum of the first n bytes of 32
__device__ __forceinline__ int sum_bytes(const uint4 (&c)[kRouteWarps / 16], int n) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(c);
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kRouteWarps / 4; ++i) {
    const int left = min(max(n - 4 * i, 0), 4);
    const uint32_t ones = left == 4 ? 0x01010101u : 0x01010101u & ((1u << (8 * left)) - 1u);
    sum = __dp4a(w[i], ones, static_cast<uint32_t>(sum));
  }
  return sum;
}

// Pairs [first, last) in order: the place of each is next of its expert plus the pairs of that expert ahead of it, in its
// warp by a match, in the warps ahead by their counts.
__device__ __forceinline__ void place_pairs(PlaceShared& s, const int32_t* experts, int32_t* slots, int first, int last,
                                            int num_experts) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int p0 = first; p0 < last; p0 += kRouteThreads) {
    const int p = p0 + tid;
    const int e = p < last ? ld_global(experts + p) : -1;
    if (tid < num_experts) s.count[tid][0] = s.count[tid][1] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    const unsigned same = __match_any_sync(kFull, e);
    const int ahead = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && ahead == 0) reinterpret_cast<unsigned char*>(s.count[e])[warp] = static_cast<unsigned char>(__popc(same));
    __syncthreads();
    if (p < last) slots[p] = e >= 0 ? s.next[e] + ahead + sum_bytes(s.count[e], warp) : -1;
    __syncthreads();
    if (p0 + kRouteThreads < last) {
      if (tid < num_experts) s.next[tid] += sum_bytes(s.count[tid], kRouteWarps);
      __syncthreads();
    }
  }
}

// p[i] = exp(z[i] - max z) / sum; the top_k <= L largest are found one after the other, each by a maximum over the keys of the
// token's lanes and the lowest index that has it.  What it costs is instructions, a hundred to a choice of the four tokens of a
// warp, and one token's chain of them where there are few: the 8.4 MB of 16,384 tokens of 128 logits would be 1.3 us, this
// launch and the next take 17.0 (8 choices), those of 65,536 tokens of 64 logits 25.7 (6), of 24 tokens 4.4 in one.
// The schedulers issue in 58 % of the cycles.  Maxima over a warp by shuffles took as long as those of the hardware.
template <class T, int L, int R>
__global__ void __launch_bounds__(kRouteThreads)
choose_kernel(const T* logits, float* gates, int32_t* experts, int32_t* slots, int32_t* indptr, int32_t* counts, int tokens,
              int share, int num_experts, int top_k, int renormalize) {
  __shared__ PlaceShared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int l = lane % L, first_lane = lane - l;
  s.next[tid] = 0;
  chain_wait();
  __syncthreads();
  const int t0 = blockIdx.x * share, t1 = t0 + min(share, tokens - t0);
  for (int tw = t0 + warp * (32 / L); tw < t1; tw += kRouteWarps * (32 / L)) {
    const int t = tw + lane / L;
    const bool live = t < t1;
    uint32_t key[R];
    float top, sum = 0.f;
    {
      float v[R];
      top = load_logits<T, L, R>(logits + static_cast<size_t>(t) * num_experts, num_experts, l, live, v);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        sum += over_top(v[r], top);
        key[r] = order_key(v[r]);
      }
    }
    sum = sum_of<L>(sum);
    int expert = -1;     // of choice l
    uint32_t chosen = 0u;
    for (int j = 0; j < top_k; ++j) {
      uint32_t best = 0u;  // the lane's largest that is left, and its first place
      int at = 0;
#pragma unroll
      for (int r = R - 1; r >= 0; --r) {
        at = key[r] >= best ? r : at;
        best = max(best, key[r]);
      }
      const uint32_t found = most_of<L>(best);
      if (!__any_sync(kFull, found != 0u)) break;
      const unsigned have = (__ballot_sync(kFull, best == found) >> first_lane) & (L == 32 ? kFull : (1u << (L & 31)) - 1u);
      // several lanes: the lowest expert, whose row of L comes first, and then its lane
      int src = __ffs(have) - 1;
      if (__any_sync(kFull, (have & (have - 1u)) != 0u)) src = least_of<L>(best == found ? at * L + l : 0x7fffffff) % L;
      const int row = __shfl_sync(kFull, at, first_lane + src);
      const int gone = l == src ? row : -1;
#pragma unroll
      for (int r = 0; r < R; ++r) key[r] = gone == r ? 0u : key[r];
      if (l == j && found != 0u) {
        expert = row * L + src;
        chosen = found;
      }
    }
    const float value = chosen != 0u ? over_top(key_value(chosen), top) : 0.f;
    if (renormalize) sum = sum_of<L>(value);
    if (live && l < top_k) {
      const size_t p = static_cast<size_t>(t) * top_k + l;
      experts[p] = expert;
      gates[p] = expert < 0 ? 0.f : value / sum;
      if (expert >= 0) atomicAdd(&s.next[expert], 1);
    }
  }
  __syncthreads();
  const int mine = s.next[tid];
  if (counts != nullptr) {
    if (tid < num_experts) counts[static_cast<size_t>(blockIdx.x) * num_experts + tid] = mine;
    return;
  }
  s.next[tid] = 0;
  const int all = add_bases(s, mine);
  __syncthreads();
  if (tid < num_experts) indptr[tid] = s.next[tid];
  if (tid == 0) indptr[num_experts] = all;
  place_pairs(s, experts, slots, 0, tokens * top_k, num_experts);
}

// The places of a share's pairs.  Three round trips (counts, choices, places) and two scans with their barriers, not bytes, are what it
// takes: 16,384 tokens of 8 choices would be 0.2 us, it is 6 behind choose_kernel.
__global__ void __launch_bounds__(kRouteThreads)
place_kernel(const int32_t* experts, int32_t* slots, int32_t* indptr, const int32_t* counts, int tokens, int share, int num_experts,
             int top_k) {
  __shared__ PlaceShared s;
  __shared__ int total[SPARSETIR_MOE_MAX_EXPERTS];
  const int tid = threadIdx.x;
  s.next[tid] = 0;
  total[tid] = 0;
  chain_wait();
  __syncthreads();
  // of every expert: the pairs of the shares ahead, and of all; several threads share an expert's column of counts
  const int shares = gridDim.x, block = blockIdx.x;
  const int rows = kRouteThreads / num_experts, row = tid / num_experts, e = tid - row * num_experts;
  if (row < rows) {
    int before = 0, all = 0;
#pragma unroll 8
    for (int i = row; i < shares; i += rows) {
      const int b = i + block < shares ? i + block : i + block - shares;  // no two blocks at the same place at a time
      const int c = ld_global(counts + static_cast<size_t>(b) * num_experts + e);
      all += c;
      before += b < block ? c : 0;
    }
    atomicAdd(&s.next[e], before);
    atomicAdd(&total[e], all);
  }
  __syncthreads();
  const int all = add_bases(s, total[tid]);
  __syncthreads();
  if (block == 0) {
    if (tid < num_experts) indptr[tid] = s.next[tid];
    if (tid == 0) indptr[num_experts] = all;
  }
  const int t0 = block * share, t1 = t0 + min(share, tokens - t0);
  place_pairs(s, experts, slots, t0 * top_k, t1 * top_k, num_experts);
}

// dz[i] = g_i dg_i [i chosen] - p_i sum g dg with the probabilities made again from the logits, or, renormalised, g_i (dg_i - sum
// g dg) [i chosen] without them.  What the chosen experts have is put into a row in shared memory: found by comparing every logit's
// place with every choice 16,384 tokens of 128 logits with 8 choices took 7.4 us, this way 4.7 (their 17 MB would be 2.6).
template <class T, int L, int R>
__global__ void __launch_bounds__(kWarps * 32)
route_grad_kernel(const T* logits, const float* gates, const int32_t* experts, const float* d_gates, T* d_logits, int tokens,
                  int num_experts, int top_k, int renormalize) {
  chain_wait();
  const int lane = threadIdx.x & 31, l = lane % L;
  const int t = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * (32 / L) + lane / L;
  const bool live = t < tokens;
  int expert = -1;
  float gate = 0.f, dg = 0.f;
  if (live && l < top_k) {
    const size_t p = static_cast<size_t>(t) * top_k + l;
    expert = ld_global(experts + p);
    gate = ld_global(gates + p);
    dg = ld_global(d_gates + p);
  }
  float v[R];
  const float top = load_logits<T, L, R>(logits + static_cast<size_t>(t) * num_experts, num_experts, l, live, v);
  if (expert < 0 || expert >= num_experts) gate = dg = 0.f;
  const float mean = sum_of<L>(gate * dg);
  // what the chosen experts have besides, in a row of the token's own
  extern __shared__ float rows[];
  float* const row = rows + static_cast<size_t>(threadIdx.x / L) * num_experts;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (l + L * r < num_experts) row[l + L * r] = 0.f;
  __syncwarp();
  if (gate != 0.f) row[expert] = gate * (renormalize ? dg - mean : dg);
  __syncwarp();
  float scale = 0.f;  // of the probabilities
  if (!renormalize) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      v[r] = over_top(v[r], top);
      sum += v[r];
    }
    sum = sum_of<L>(sum);
    scale = sum > 0.f ? -mean / sum : 0.f;
  }
  if (!live) return;
  T* out = d_logits + static_cast<size_t>(t) * num_experts;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = l + L * r;
    if (e < num_experts) out[e] = from_float<T>(renormalize ? row[e] : fmaf(scale, v[r], row[e]));
  }
}

// f(L, R) as integral constants, L * R >= num_experts.  8 lanes to a token, for up to `most` experts, where the SMs have warps
// enough all the same (us, 32 lanes / 8: router of 16,384 tokens, 128 experts, 8 choices 20.4 / 17.5, 65,536 tokens, 64, 6 36.8 /
// 27.0, 8,192, 128, 8 14.0 / 13.9, 2,000, 128, 8 8.8 / 9.8; the gradient of the first 7.4 / 7.8, of the second 16.4 / 11.6).
template <class F>
int with_lanes(int tokens, int num_experts, int top_k, int most, F&& f) {
  using std::integral_constant;
  if (tokens >= 8192 && num_experts <= most && top_k <= 8) {
    if (num_experts <= 32) return f(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    if (num_experts <= 64) return f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    return f(integral_constant<int, 8>{}, integral_constant<int, 16>{});
  }
  if (num_experts <= 32) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  if (num_experts <= 64) return f(integral_constant<int, 32>{}, integral_constant<int, 2>{});
  if (num_experts <= 128) return f(integral_constant<int, 32>{}, integral_constant<int, 4>{});
  if (num_experts <= 256) return f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
  if (num_experts <= 512) return f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  return f(integral_constant<int, 32>{}, integral_constant<int, 32>{});
}

// ---- rows -----------------------------------------------------------------------------------------------------------

constexpr int kHold = 4;  // pieces of a row that a lane has in flight

// Slot of pair t * top_k + lane, -1 where there is none
__device__ __forceinline__ int pair_slot(const int32_t* slots, int t, int top_k, int rows, int lane) {
  int s = -1;
  if (lane < top_k) s = ld_global(slots + static_cast<size_t>(t) * top_k + lane);
  return static_cast<unsigned>(s) < static_cast<unsigned>(rows) ? s : -1;
}

// A warp copies up to kHold * 32 pieces of a token's row to its slots: the row is read once.  HBM bounds it: 302 MB (8,192 rows of 2048
// to 65,536 pairs, 16 bits) in 49.4 us, 6.1 TB/s.
template <int B>
__global__ void __launch_bounds__(kWarps * 32)
dispatch_kernel(const Piece<B>* x, const int32_t* slots, Piece<B>* z, int tokens, int rows, int pieces, int chunks, int top_k) {
  chain_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(item / chunks), c = static_cast<int>(item - static_cast<long long>(t) * chunks);
  if (t >= tokens) return;
  const int slot = pair_slot(slots, t, top_k, rows, lane);
  const int first = c * (kHold * 32) + lane;
  Piece<B> v[kHold];
#pragma unroll
  for (int i = 0; i < kHold; ++i)
    if (first + 32 * i < pieces) v[i] = ld_global(x + static_cast<size_t>(t) * pieces + first + 32 * i);
  for (int j = 0; j < top_k; ++j) {
    const int s = __shfl_sync(kFull, slot, j);
    if (s < 0) continue;
    Piece<B>* to = z + static_cast<size_t>(s) * pieces + first;
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (first + 32 * i < pieces) to[32 * i] = v[i];
  }
}

// A warp sums up to 64 pieces of a token's rows, four rows requested together, in 32 bits and in the order of the choices.  HBM
// bounds the large ones (8,192 x 8 rows of 2048 in 16 bits, 302 MB in 49.8 us, 6.06 TB/s); those of a decoding step are the chain
// slots -> rows and a launch (24 tokens: 2.5 us in a graph).
template <class T, class OutT, int B>
__global__ void __launch_bounds__(kWarps * 32)
combine_kernel(const Piece<B>* z, const int32_t* slots, const float* gates, OutT* y, int tokens, int rows, int pieces,
               int chunks, int top_k) {
  constexpr int N = B / sizeof(T), U = 2, J = 4;
  chain_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(item / chunks), c = static_cast<int>(item - static_cast<long long>(t) * chunks);
  if (t >= tokens) return;
  const int slot = pair_slot(slots, t, top_k, rows, lane);
  float gate = 1.f;
  if (gates != nullptr && lane < top_k) gate = ld_global(gates + static_cast<size_t>(t) * top_k + lane);
  const int first = c * (U * 32) + lane;
  float acc[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int n = 0; n < N; ++n) acc[u][n] = 0.f;
  for (int j0 = 0; j0 < top_k; j0 += J) {
    Piece<B> v[J][U];
    int s[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      s[j] = j0 + j < top_k ? __shfl_sync(kFull, slot, (j0 + j) & 31) : -1;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s[j] >= 0 && first + 32 * u < pieces) v[j][u] = ld_global(z + static_cast<size_t>(s[j]) * pieces + first + 32 * u);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float w = __shfl_sync(kFull, gate, (j0 + j) & 31);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s[j] >= 0 && first + 32 * u < pieces) {
          float f[N];
          unpack<T, B>(v[j][u], f);
#pragma unroll
          for (int n = 0; n < N; ++n) acc[u][n] = fmaf(w, f[n], acc[u][n]);
        }
      }
    }
  }
  constexpr int OB = N * static_cast<int>(sizeof(OutT)) > 16 ? 16 : N * static_cast<int>(sizeof(OutT));
  constexpr int ON = OB / sizeof(OutT);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (first + 32 * u >= pieces) continue;
    OutT* to = y + (static_cast<size_t>(t) * pieces + first + 32 * u) * N;
#pragma unroll
    for (int q = 0; q < N / ON; ++q) {
      float part[ON];
#pragma unroll
      for (int n = 0; n < ON; ++n) part[n] = acc[u][q * ON + n];
      *reinterpret_cast<Piece<OB>*>(to + q * ON) = pack<OutT, OB>(part);
    }
  }
}

constexpr int kRowThreads = 128;  // a block per token
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kRowHold = 2;       // pieces of a row that a thread of it has in flight

// Block per token: dy in registers, kRowHold pieces to a thread at a time, the rows of z one after the other, each read once for its
// scalar product while its gradient leaves.  HBM bounds it: 6,007 tokens with four rows of 2040 in 16 bits, 221 MB in 38.1 us,
// 5.8 TB/s (48.5 with one piece to a thread and no row ahead).
template <class T, int B>
__global__ void __launch_bounds__(kRowThreads)
combine_grad_kernel(const Piece<B>* dy, const Piece<B>* z, const int32_t* slots, const float* gates, Piece<B>* dz, float* d_gates,
                    int rows, int pieces, int top_k) {
  constexpr int N = B / sizeof(T);
  __shared__ float part[SPARSETIR_MOE_MAX_TOP_K][kRowWarps];
  chain_wait();
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = pair_slot(slots, t, top_k, rows, lane);
  float gate = 0.f;
  if (lane < top_k) {
    gate = ld_global(gates + static_cast<size_t>(t) * top_k + lane);
    part[lane][warp] = 0.f;
  }
  __syncwarp();
  for (int base = 0; base < pieces; base += kRowHold * kRowThreads) {
    const int first = base + tid;
    Piece<B> d[kRowHold];
#pragma unroll
    for (int i = 0; i < kRowHold; ++i)
      if (first + i * kRowThreads < pieces) d[i] = ld_global(dy + static_cast<size_t>(t) * pieces + first + i * kRowThreads);
    // the pieces of the next row are asked for before this one's are used
    auto ask = [&](int j, Piece<B> (&v)[kRowHold]) {
      const int s = j < top_k ? __shfl_sync(kFull, slot, j) : -1;
      if (s < 0) return s;
#pragma unroll
      for (int i = 0; i < kRowHold; ++i)
        if (first + i * kRowThreads < pieces) v[i] = ld_global(z + static_cast<size_t>(s) * pieces + first + i * kRowThreads);
      return s;
    };
    auto use = [&](int j, int s, const Piece<B> (&v)[kRowHold]) {
      if (s < 0) return;
      const float w = __shfl_sync(kFull, gate, j);
      Piece<B>* to = dz + static_cast<size_t>(s) * pieces + first;
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < kRowHold; ++i) {
        if (first + i * kRowThreads < pieces) {
          float a[N], b[N], o[N];
          unpack<T, B>(d[i], a);
          unpack<T, B>(v[i], b);
#pragma unroll
          for (int n = 0; n < N; ++n) {
            dot = fmaf(a[n], b[n], dot);
            o[n] = w * a[n];
          }
          to[i * kRowThreads] = pack<T, B>(o);
        }
      }
      dot = sum_of<32>(dot);
      if (lane == 0) part[j][warp] += dot;
    };
    Piece<B> u[kRowHold], v[kRowHold];
    int su = ask(0, u);
    for (int j = 0; j < top_k; j += 2) {
      const int sv = ask(j + 1, v);
      use(j, su, u);
      su = ask(j + 2, u);
      if (j + 1 < top_k) use(j + 1, sv, v);
    }
  }
  __syncthreads();
  if (tid < top_k) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) sum += part[tid][w];
    d_gates[static_cast<size_t>(t) * top_k + tid] = slot >= 0 ? sum : 0.f;
  }
}

// Block per token: the largest magnitude, as the bits of a float without its sign (so that an infinity or a NaN is
// larger than all numbers and stays), then the quotients.  Rows of up to kRowHold pieces to a thread are read once.
// 4,096 rows of 2048 in 16 bits to four slots each, 50 MB: 11.7 us, issue 68 %, so the conversions bound it as much as HBM.
template <class T, int B>
__global__ void __launch_bounds__(kRowThreads)
dispatch_i8_kernel(const Piece<B>* x, const int32_t* slots, Piece<B / sizeof(T)>* q, float* scale, int rows, int pieces,
                   int top_k) {
  constexpr int N = B / sizeof(T);
  __shared__ uint32_t most[kRowWarps];
  chain_wait();
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = slots != nullptr ? pair_slot(slots, t, top_k, rows, lane) : (lane == 0 ? t : -1);
  const Piece<B>* xr = x + static_cast<size_t>(t) * pieces;
  Piece<B> v[kRowHold];
  uint32_t bits = 0u;
  for (int base = 0; base < pieces; base += kRowHold * kRowThreads) {
#pragma unroll
    for (int i = 0; i < kRowHold; ++i)
      if (base + tid + i * kRowThreads < pieces) v[i] = ld_global(xr + base + tid + i * kRowThreads);
#pragma unroll
    for (int i = 0; i < kRowHold; ++i) {
      if (base + tid + i * kRowThreads < pieces) {
        float f[N];
        unpack<T, B>(v[i], f);
#pragma unroll
        for (int n = 0; n < N; ++n) bits = max(bits, __float_as_uint(f[n]) & 0x7fffffffu);
      }
    }
  }
  bits = __reduce_max_sync(kFull, bits);
  if (lane == 0) most[warp] = bits;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) bits = max(bits, most[w]);
  const float a = __uint_as_float(bits);
  const bool zeros = !(a >= 0x1p-119f && a < INFINITY);
  const float inv = zeros ? 0.f : 127.f / a;
  if (tid < top_k && slot >= 0) scale[slot] = a < 0x1p-119f ? 0.f : a / 127.f;
  for (int base = 0; base < pieces; base += kRowHold * kRowThreads) {
    if (pieces > kRowHold * kRowThreads) {  // otherwise they are here still
#pragma unroll
      for (int i = 0; i < kRowHold; ++i)
        if (base + tid + i * kRowThreads < pieces) v[i] = ld_global(xr + base + tid + i * kRowThreads);
    }
#pragma unroll
    for (int i = 0; i < kRowHold; ++i) {
      const int at = base + tid + i * kRowThreads;
      Piece<N> o;
      if (at < pieces) {
        float f[N];
        unpack<T, B>(v[i], f);
        int8_t* b = reinterpret_cast<int8_t*>(&o);
#pragma unroll
        for (int n = 0; n < N; ++n) b[n] = zeros ? 0 : static_cast<int8_t>(__float2int_rn(f[n] * inv));
      }
      for (int j = 0; j < top_k; ++j) {
        const int s = __shfl_sync(kFull, slot, j);
        if (s >= 0 && at < pieces) q[static_cast<size_t>(s) * pieces + at] = o;
      }
    }
  }
}

// Four numbers to e4m3, to nearest, ties to even.
__device__ __forceinline__ uint32_t pack_f8(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return __byte_perm(lo, hi, 0x5410);
}
__device__ __forceinline__ float2 unpack_f8(uint32_t two) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3)));
}
// Of lo and hi, neighbours or the same, the nearer one to 0.875 x / unit, or their middle, which is rounded to the even one: by the sign of
// 0.875 x - middle * unit.  Each product and what its rounding leaves are exact, so are their differences, a few bits beside each other, and
// that of the products themselves, which are next to each other.  `by`: a power of two that keeps what is left above the smallest numbers.
__device__ __forceinline__ float nearer(float x, float unit, float lo, float hi, float by) {
  const float middle = 0.5f * (lo + hi), y = x * by, u = unit * by, a = __fmul_rn(0.875f, y), b = __fmul_rn(middle, u);
  const float d = (a - b) + (fmaf(0.875f, y, -a) - fmaf(middle, u, -b));
  return d == 0.f ? middle : d > 0.f ? fmaxf(lo, hi) : fminf(lo, hi);
}
// 448 x / a to the nearest e4m3, ties to even, for |x| <= a: the quotient of 0.875 x by unit = a / 512.  below and above are 0.875 / unit moved by
// four units of its last place: where x times both has one place between the numbers of 8 bits, so has the quotient, and four divisions are spared.
// For elements of 16 bits 0.875 x is exact, and so is the place of the rounded quotient, ties among them; for 32 bits it is not.
template <class T>
__device__ __forceinline__ uint32_t quotients_f8(const float* x, float unit, float below, float above) {
  const uint32_t q = pack_f8(x[0] * below, x[1] * below, x[2] * below, x[3] * below);
  const uint32_t r = pack_f8(x[0] * above, x[1] * above, x[2] * above, x[3] * above);
  if (q == r) return q;
  if constexpr (sizeof(T) == 4) {
    const float by = unit < 1.f ? 0x1p20f : 0x1p-20f;
    const float2 q01 = unpack_f8(q & 0xffffu), q23 = unpack_f8(q >> 16), r01 = unpack_f8(r & 0xffffu), r23 = unpack_f8(r >> 16);
    return pack_f8(nearer(x[0], unit, q01.x, r01.x, by), nearer(x[1], unit, q01.y, r01.y, by), nearer(x[2], unit, q23.x, r23.x, by),
                   nearer(x[3], unit, q23.y, r23.y, by));
  }
  return pack_f8(0.875f * x[0] / unit, 0.875f * x[1] / unit, 0.875f * x[2] / unit, 0.875f * x[3] / unit);
}
// The largest magnitude of pieces, in the order of unsigned integers (so that an infinity or a NaN is larger than all numbers), and as the bits of
// a float: of 16-bit elements two at a time.
template <class T>
struct Largest {
  uint32_t bits = 0u;
  template <int B>
  __device__ __forceinline__ void take(const Piece<B>& v) {
    if constexpr (sizeof(T) == 2 && B == 2) {
      bits = max(bits, static_cast<uint32_t>(v) & 0x7fffu);
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
      for (int i = 0; i < B / 4; ++i) bits = sizeof(T) == 2 ? __vmaxs2(bits, w[i] & 0x7fff7fffu) : max(bits, w[i] & 0x7fffffffu);
    }
  }
  template <int L>
  __device__ __forceinline__ float over_lanes() const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(most_of<L>(bits));
    const uint16_t most = static_cast<uint16_t>(most_of<L>(max(bits & 0xffffu, bits >> 16)));
    return to_float(reinterpret_cast<const T&>(most));
  }
};

// Rows to 8-bit floating point with a scale for each block of 128 features: L lanes have a block, P pieces each that lie side by side, and a
// warp kHold times as many blocks as it has room for.  (Us, 8,192 rows of 2048 in bfloat16 to eight slots each, 172 MB: 36.0 with a
// division to an element and 8 bytes to a store, now 29.2; one slot each, 16,384 rows of 4096, 201 MB: 71 and 47, in float16 38, in 32 bits, 336 MB, 53.)
template <class T, int B, bool WIDE>
struct F8Lanes {
  static constexpr int N = B / sizeof(T);  // elements of a piece
  static constexpr int kPieces = SPARSETIR_F8_BLOCK / N > 32 ? SPARSETIR_F8_BLOCK / N / 32 : WIDE ? 16 / N : 1;
  static constexpr int kLanes = SPARSETIR_F8_BLOCK / N / kPieces;
  static constexpr int kBlocks = 32 / kLanes;  // of 128 features that a warp has side by side
  static constexpr int kHold = kPieces < 4 ? 4 / kPieces : 1;
  static constexpr int kOut = WIDE ? kPieces * N : N;  // bytes of a store
};
template <class T, int B, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32)
dispatch_f8_kernel(const Piece<B>* x, const int32_t* slots, uint8_t* q, float* scale, int tokens, int rows, int pieces, int blocks,
                   int chunks, int top_k) {
  using Lanes = F8Lanes<T, B, WIDE>;
  constexpr int N = Lanes::N, L = Lanes::kLanes, P = Lanes::kPieces, H = Lanes::kHold, OUT = Lanes::kOut;
  chain_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(item / chunks), c = static_cast<int>(item - static_cast<long long>(t) * chunks);
  if (t >= tokens) return;
  const int slot = slots != nullptr ? pair_slot(slots, t, top_k, rows, lane) : (lane == 0 ? t : -1);
  const int block0 = c * (H * Lanes::kBlocks) + lane / L;  // and every kBlocks further
  const int first = (block0 * L + lane % L) * P;
  Piece<B> v[H][P];
  constexpr int E = P * N;  // elements of a lane in a block, a multiple of four
  __align__(16) uint32_t o[H][E / 4];
  float s_of[H];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int at = first + h * (Lanes::kBlocks * L * P) + i;
      v[h][i] = Piece<B>{};
      if (at < pieces) v[h][i] = ld_global(x + static_cast<size_t>(t) * pieces + at);
    }
#pragma unroll
  for (int h = 0; h < H; ++h) {
    Largest<T> largest;
#pragma unroll
    for (int i = 0; i < P; ++i) largest.template take<B>(v[h][i]);
    const float a = largest.template over_lanes<L>();
    const bool zeros = !(a >= 0x1p-110f && a < INFINITY);
    const float unit = zeros ? 1.f : a * 0x1p-9f, times = __fdividef(0.875f, unit);  // two units off at most
    s_of[h] = a < 0x1p-110f ? 0.f : a / 448.f;
    float f[E];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float part[N];
      unpack<T, B>(v[h][i], part);
#pragma unroll
      for (int n = 0; n < N; ++n) f[i * N + n] = part[n];
    }
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const uint32_t q4 = quotients_f8<T>(f + e, unit, times * (1.f - 0x1p-21f), times * (1.f + 0x1p-21f));
      o[h][e / 4] = zeros ? 0u : q4;
    }
  }
  for (int j = 0; j < top_k; ++j) {
    const int s = __shfl_sync(kFull, slot, j);
    if (s < 0) continue;
    uint8_t* const to = q + static_cast<size_t>(s) * pieces * N;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int block = block0 + h * Lanes::kBlocks;
      if (lane % L == 0 && block < blocks) scale[static_cast<size_t>(block) * rows + s] = s_of[h];
#pragma unroll
      for (int i = 0; i < E / OUT; ++i) {
        const int at = first * N + h * (Lanes::kBlocks * L * E) + i * OUT;  // rows are whole stores
        Piece<OUT> out;
        if constexpr (OUT >= 4) {
          out = *reinterpret_cast<const Piece<OUT>*>(&o[h][i * OUT / 4]);
        } else {
          out = static_cast<Piece<OUT>>(o[h][i * OUT / 4] >> (8 * (i * OUT % 4)));
        }
        if (at < pieces * N) *reinterpret_cast<Piece<OUT>*>(to + at) = out;
      }
    }
  }
}

// Widest piece, in bytes, that divides rows of `row_bytes` and fits the pointers.
int piece_bytes(size_t row_bytes, uintptr_t pointers) {
  for (int b : {16, 8, 4})
    if (row_bytes % b == 0 && pointers % b == 0) return b;
  return 2;
}
uintptr_t bits_of(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// f(integral constant B) for pieces of b bytes of elements of `size` bytes
template <int SIZE, class F>
int with_piece(int b, F&& f) {
  if (b == 16) return f(std::integral_constant<int, 16>{});
  if (b == 8) return f(std::integral_constant<int, 8>{});
  if (b == 4) return f(std::integral_constant<int, 4>{});
  if constexpr (SIZE == 2) return f(std::integral_constant<int, 2>{});
  return fail("misaligned f32 operand");
}

int check_rows(const char* fn, int type, int tokens, int rows, int feat, int top_k) {
  if (type < SPARSETIR_F32 || type > SPARSETIR_BF16) return fail("%s: unknown element type %d", fn, type);
  if (tokens < 0 || rows < 0 || feat < 0) return fail("%s: negative size", fn);
  if (std::max(tokens, std::max(rows, feat)) > kLargestSize) return fail("%s: too large for 32-bit indices", fn);
  if (top_k < 1 || top_k > SPARSETIR_MOE_MAX_TOP_K)
    return fail("%s: top_k = %d is not in [1, %d]", fn, top_k, SPARSETIR_MOE_MAX_TOP_K);
  return 0;
}
int check_slots(const char* fn, const int32_t* slots, int tokens, int rows, int top_k, cudaStream_t st) {
  if (!validate_enabled()) return 0;
  return validate_range(fn, "slots", slots, static_cast<long long>(tokens) * top_k, rows, st, /*lowest=*/-1);
}
size_t element(int type) { return type == SPARSETIR_F32 ? 4 : 2; }

int check_route(const char* fn, int type, int tokens, int num_experts, int top_k, int flags) {
  if (check_rows(fn, type, tokens, 0, 0, top_k) != 0) return -1;
  if (num_experts < top_k || num_experts > SPARSETIR_MOE_MAX_EXPERTS)
    return fail("%s: num_experts = %d is not in [top_k, %d]", fn, num_experts, SPARSETIR_MOE_MAX_EXPERTS);
  if ((flags & ~SPARSETIR_MOE_RENORMALIZE) != 0) return fail("%s: unknown flags %d", fn, flags);
  if (static_cast<long long>(tokens) * top_k > INT32_MAX - 2 * kRouteThreads) return fail("%s: too many pairs for 32-bit indices", fn);
  return 0;
}

int route_share(int tokens) { return tokens <= kRouteAlone ? kRouteAlone : std::max(kRouteTokens, ceil_div(tokens, kNumSMs)); }
size_t route_counts(int shares, int num_experts) { return static_cast<size_t>(shares) * num_experts * sizeof(int32_t); }

}  // namespace
}  // namespace sptir

using namespace sptir;

extern "C" int sparsetir_moe_route_raw(const void* logits, int logits_type, float* gates, int32_t* experts, int32_t* slots,
                                       int32_t* indptr, int tokens, int num_experts, int top_k, int flags, int device_id,
                                       void* stream) {
  const char* fn = "sparsetir_moe_route";
  if (check_route(fn, logits_type, tokens, num_experts, top_k, flags) != 0) return -1;
  if (!indptr || (tokens > 0 && (!logits || !gates || !experts || !slots))) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int share = route_share(tokens), shares = std::max(1, ceil_div(tokens, share));
  CallScratch cs;
  if (shares > 1 && take_scratch(device_id, st, route_counts(shares, num_experts), 0, &cs) != 0) return -1;
  int32_t* counts = reinterpret_cast<int32_t*>(cs.scratch);
  const int rc = with_type(logits_type, [&](auto t) {
    using T = decltype(t);
    return with_lanes(tokens, num_experts, top_k, 128, [&](auto l, auto r) {
      launch_chained(choose_kernel<T, l.value, r.value>, shares, kRouteThreads, 0, st, static_cast<const T*>(logits), gates, experts, slots,
                     indptr, counts, tokens, share, num_experts, top_k, flags & SPARSETIR_MOE_RENORMALIZE);
      SPTIR_LAUNCH_OK("choose_kernel");
      return 0;
    });
  });
  if (rc != 0 || shares == 1) return rc;
  launch_chained(place_kernel, shares, kRouteThreads, 0, st, experts, slots, indptr, counts, tokens, share, num_experts, top_k);
  SPTIR_LAUNCH_OK("place_kernel");
  return return_scratch(cs, st);
}

extern "C" int sparsetir_moe_route_workspace(int tokens, int num_experts, size_t* scratch_bytes) {
  if (tokens < 0 || num_experts < 1 || num_experts > SPARSETIR_MOE_MAX_EXPERTS || !scratch_bytes)
    return fail("sparsetir_moe_route_workspace: bad argument");
  const int shares = ceil_div(tokens, route_share(tokens));
  *scratch_bytes = shares > 1 ? route_counts(shares, num_experts) : 0;
  return 0;
}

extern "C" int sparsetir_moe_route_grad_raw(const void* logits, int logits_type, const float* gates, const int32_t* experts,
                                            const float* d_gates, void* d_logits, int tokens, int num_experts, int top_k,
                                            int flags, int device_id, void* stream) {
  const char* fn = "sparsetir_moe_route_grad";
  if (check_route(fn, logits_type, tokens, num_experts, top_k, flags) != 0) return -1;
  if (tokens == 0) return 0;
  if (!logits || !gates || !experts || !d_gates || !d_logits) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (validate_enabled() && validate_range(fn, "experts", experts, static_cast<long long>(tokens) * top_k, num_experts, st,
                                           /*lowest=*/-1) != 0)
    return -1;
  return with_type(logits_type, [&](auto t) {
    using T = decltype(t);
    return with_lanes(tokens, num_experts, top_k, 64, [&](auto l, auto r) {
      launch_chained(route_grad_kernel<T, l.value, r.value>, ceil_div(tokens, kWarps * 32 / l.value), kWarps * 32,
                     kWarps * (32 / l.value) * num_experts * sizeof(float), st, static_cast<const T*>(logits),
                     gates, experts, d_gates, static_cast<T*>(d_logits), tokens, num_experts, top_k,
                     flags & SPARSETIR_MOE_RENORMALIZE);
      SPTIR_LAUNCH_OK("route_grad_kernel");
      return 0;
    });
  });
}

extern "C" int sparsetir_moe_dispatch_raw(const void* x, const int32_t* slots, void* z, int type, int tokens, int rows, int feat,
                                          int top_k, int device_id, void* stream) {
  const char* fn = "sparsetir_moe_dispatch";
  if (check_rows(fn, type, tokens, rows, feat, top_k) != 0) return -1;
  if (tokens == 0 || rows == 0 || feat == 0) return 0;
  if (!x || !slots || !z) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_slots(fn, slots, tokens, rows, top_k, st) != 0) return -1;
  const size_t row_bytes = element(type) * feat;
  const int b = piece_bytes(row_bytes, bits_of(x) | bits_of(z));
  return with_piece<2>(b, [&](auto bytes) {
    using P = Piece<bytes.value>;
    const int pieces = static_cast<int>(row_bytes / bytes.value), chunks = ceil_div(pieces, kHold * 32);
    const long long blocks = (static_cast<long long>(tokens) * chunks + kWarps - 1) / kWarps;
    if (blocks > INT32_MAX) return fail("%s: too large for one launch", fn);
    launch_chained(dispatch_kernel<bytes.value>, static_cast<unsigned>(blocks), kWarps * 32, 0, st, static_cast<const P*>(x), slots,
                   static_cast<P*>(z), tokens, rows, pieces, chunks, top_k);
    SPTIR_LAUNCH_OK("dispatch_kernel");
    return 0;
  });
}

extern "C" int sparsetir_moe_dispatch_i8_raw(const void* x, int type, const int32_t* slots, int8_t* q, float* scale, int tokens,
                                             int rows, int feat, int top_k, int device_id, void* stream) {
  const char* fn = "sparsetir_moe_dispatch_i8";
  if (check_rows(fn, type, tokens, rows, feat, top_k) != 0) return -1;
  if (tokens == 0) return 0;
  if (!slots && (top_k != 1 || rows != tokens)) return fail("%s: slots may be null with top_k 1 and a row per token only", fn);
  if (rows == 0 || feat == 0) return 0;
  if (!x || !q || !scale) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (slots && check_slots(fn, slots, tokens, rows, top_k, st) != 0) return -1;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    // a piece of N elements leaves as N bytes
    int b = piece_bytes(sizeof(T) * feat, bits_of(x));
    while (b > static_cast<int>(sizeof(T)) && bits_of(q) % (b / sizeof(T)) != 0) b /= 2;
    return with_piece<sizeof(T)>(b, [&](auto bytes) {
      constexpr int B = bytes.value;
      using Q = Piece<B / sizeof(T)>;
      launch_chained(dispatch_i8_kernel<T, B>, tokens, kRowThreads, 0, st, static_cast<const Piece<B>*>(x), slots,
                     reinterpret_cast<Q*>(q), scale, rows, static_cast<int>(sizeof(T) * feat / B), top_k);
      SPTIR_LAUNCH_OK("dispatch_i8_kernel");
      return 0;
    });
  });
}

extern "C" int sparsetir_moe_dispatch_f8_raw(const void* x, int type, const int32_t* slots, void* q, float* scale, int tokens,
                                             int rows, int feat, int top_k, int device_id, void* stream) {
  const char* fn = "sparsetir_moe_dispatch_f8";
  if (check_rows(fn, type, tokens, rows, feat, top_k) != 0) return -1;
  if (tokens == 0) return 0;
  if (!slots && (top_k != 1 || rows != tokens)) return fail("%s: slots may be null with top_k 1 and a row per token only", fn);
  if (rows == 0 || feat == 0) return 0;
  if (!x || !q || !scale) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (slots && check_slots(fn, slots, tokens, rows, top_k, st) != 0) return -1;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    // a piece of N elements leaves as N bytes, or two (four) as 16
    int b = piece_bytes(sizeof(T) * feat, bits_of(x));
    while (b > static_cast<int>(sizeof(T)) && bits_of(q) % (b / sizeof(T)) != 0) b /= 2;
    auto run = [&](auto bytes, auto wide) {
      constexpr int B = bytes.value;
      using Lanes = F8Lanes<T, B, wide.value>;
      const int scales = ceil_div(feat, SPARSETIR_F8_BLOCK), chunks = ceil_div(scales, Lanes::kBlocks * Lanes::kHold);
      const long long blocks = (static_cast<long long>(tokens) * chunks + kWarps - 1) / kWarps;
      if (blocks > INT32_MAX) return fail("%s: too large for one launch", fn);
      launch_chained(dispatch_f8_kernel<T, B, wide.value>, static_cast<unsigned>(blocks), kWarps * 32, 0, st,
                     static_cast<const Piece<B>*>(x), slots, static_cast<uint8_t*>(q), scale, tokens, rows,
                     static_cast<int>(sizeof(T) * feat / B), scales, chunks, top_k);
      SPTIR_LAUNCH_OK("dispatch_f8_kernel");
      return 0;
    };
    if (b == 16 && feat % 16 == 0 && bits_of(q) % 16 == 0) return run(std::integral_constant<int, 16>{}, std::true_type{});
    return with_piece<sizeof(T)>(b, [&](auto bytes) { return run(bytes, std::false_type{}); });
  });
}

extern "C" int sparsetir_moe_combine_raw(const void* z, int z_type, const int32_t* slots, const float* gates, void* y, int y_type,
                                         int tokens, int rows, int feat, int top_k, int device_id, void* stream) {
  const char* fn = "sparsetir_moe_combine";
  if (check_rows(fn, z_type, tokens, rows, feat, top_k) != 0) return -1;
  if (y_type != z_type && y_type != SPARSETIR_F32) return fail("%s: y has the type of z, or f32", fn);
  if (tokens == 0 || feat == 0) return 0;
  if ((!z && rows > 0) || !slots || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_slots(fn, slots, tokens, rows, top_k, st) != 0) return -1;
  return with_type(z_type, [&](auto t) {
    using T = decltype(t);
    // a piece of N elements leaves in stores of up to 16 bytes
    int b = piece_bytes(sizeof(T) * feat, bits_of(z));
    while (b > static_cast<int>(sizeof(T)) && bits_of(y) % std::min<size_t>(16, b / sizeof(T) * element(y_type)) != 0) b /= 2;
    return with_piece<sizeof(T)>(b, [&](auto bytes) {
      constexpr int B = bytes.value;
      const int pieces = static_cast<int>(sizeof(T) * feat / B), chunks = ceil_div(pieces, 64);
      const long long blocks = (static_cast<long long>(tokens) * chunks + kWarps - 1) / kWarps;
      if (blocks > INT32_MAX) return fail("%s: too large for one launch", fn);
      const dim3 grid(static_cast<unsigned>(blocks));
      if (y_type == z_type)
        launch_chained(combine_kernel<T, T, B>, grid, kWarps * 32, 0, st, static_cast<const Piece<B>*>(z), slots, gates,
                       static_cast<T*>(y), tokens, rows, pieces, chunks, top_k);
      else
        launch_chained(combine_kernel<T, float, B>, grid, kWarps * 32, 0, st, static_cast<const Piece<B>*>(z), slots, gates,
                       static_cast<float*>(y), tokens, rows, pieces, chunks, top_k);
      SPTIR_LAUNCH_OK("combine_kernel");
      return 0;
    });
  });
}

extern "C" int sparsetir_moe_combine_grad_raw(const void* dy, const void* z, int type, const int32_t* slots, const float* gates,
                                              void* dz, float* d_gates, int tokens, int rows, int feat, int top_k, int device_id,
                                              void* stream) {
  const char* fn = "sparsetir_moe_combine_grad";
  if (check_rows(fn, type, tokens, rows, feat, top_k) != 0) return -1;
  if (tokens == 0) return 0;
  if (!slots || !gates || !d_gates || (feat > 0 && (!dy || (rows > 0 && (!z || !dz))))) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_slots(fn, slots, tokens, rows, top_k, st) != 0) return -1;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    const int b = piece_bytes(sizeof(T) * feat, bits_of(dy) | bits_of(z) | bits_of(dz));
    return with_piece<sizeof(T)>(b, [&](auto bytes) {
      constexpr int B = bytes.value;
      launch_chained(combine_grad_kernel<T, B>, tokens, kRowThreads, 0, st, static_cast<const Piece<B>*>(dy),
                     static_cast<const Piece<B>*>(z), slots, gates, static_cast<Piece<B>*>(dz), d_gates, rows,
                     static_cast<int>(sizeof(T) * feat / B), top_k);
      SPTIR_LAUNCH_OK("combine_grad_kernel");
      return 0;
    });
  });
}
