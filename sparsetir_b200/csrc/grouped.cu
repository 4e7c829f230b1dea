// Products grouped by expert, ragged sizes, on the tensor cores:
//   grouped_mm         y[s, :] = x[s, :] * W[g]                       s in [indptr[g], indptr[g + 1])
//   grouped_mm_i8      the same in 8-bit integers, scaled per row and per output feature
//   grouped_mm_grad_w  dW[g, a, b] = sum over the rows s of group g of pa[s, a] * pb[s, b]
//
// All three are one kernel.  A pair of blocks (cta_group::2) holds 256 of what is contiguous in the result (output
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

#include "grouped_tile.cuh"

namespace sptir {
namespace {

// The kernel for results of `type`, with tiles of `columns` columns.
template <int ELEM, int OUT>
int launch_type(int columns, int type, const CUtensorMap& tm_a, const CUtensorMap& tm_b64, const CUtensorMap& tm_b16, const Args& p,
                cudaStream_t st) {
  return with_type(type, [&](auto o) {
    using O = decltype(o);
    if constexpr (OUT != kWeights)
      if (columns == 128) return launch<ELEM, OUT, O, 128>(tm_a, tm_b64, tm_b16, p, st);
    return launch<ELEM, OUT, O, 256>(tm_a, tm_b64, tm_b16, p, st);
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
    FewArgs f{ox.data, ow.data, y, xs, ws, indptr, ox.pitch, ow.pitch, rows, groups, fi, fo, fi * size, 0, 0, 0, nullptr, Gate()};
    const int done = few_rows(f, type, y_type, out_in, st);
    return done != 0 ? done : return_scratch(cs, st);
  }
  p.parts = scratch;
  CUtensorMap tm_w, tm_x64, tm_x16;
  if (map_operands(&tm_w, &tm_x64, &tm_x16, map_type(type), ow, ox, out_in ? fo : fi, groups, out_in, false) != 0) return -1;
  const int rc = i8 ? launch_type<kInt8, kPlain>(columns, y_type, tm_w, tm_x64, tm_x16, p, st)
                    : launch_type<kHalf, kPlain>(columns, y_type, tm_w, tm_x64, tm_x16, p, st);
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
  const int rc = launch_type<kHalf, kWeights>(columns, dw_type, tm_a, tm_b, tm_b, p, st);
  return rc != 0 ? rc : return_scratch(cs, st);
}

extern "C" int sparsetir_grouped_mm_workspace(int rows, int num_groups, int feat_in, int feat_out, int element_bytes, int flags,
                                              size_t* scratch_bytes) {
  const char* fn = "sparsetir_grouped_mm_workspace";
  const int32_t some = 0;  // pointers are not looked at
  if (check_groups(fn, &some, rows, num_groups, feat_in, feat_out, flags) != 0) return -1;
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
  const size_t product = copy(static_cast<long long>(num_groups) * (out_in ? feat_out : feat_in), out_in ? feat_in : feat_out) + part_bytes(p);
  p.features = out_in ? feat_in : feat_out;
  p.columns = out_in ? feat_out : feat_in;
  if (plan_grad(fn, &p) < 0) return -1;
  *scratch_bytes = copy(rows, feat_in) + std::max(product, element_bytes == 1 ? 0 : copy(rows, feat_out) + part_bytes(p));
  return 0;
}
