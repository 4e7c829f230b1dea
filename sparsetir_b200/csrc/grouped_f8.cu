// Products of 8-bit floating point (e4m3) grouped by expert, with a scale for each 128 of a row of x and for each 128 x 128 of W, and the gated
// block of such operands, on the tensor cores (grouped.cu; the epilogue is in grouped_gated.cuh).
// A step of the ring is 128 of K: its sums are complete in one of two accumulators, which change by turns, and the epilogue's warps add them, scaled, to
// sums in their registers while the tensor core fills the other.  Tiles of 256 rows have the rows of x as the left operand (one scale to a lane);
// those of 128 rows, for groups of few rows, the features, as the other products have (us, tiles of 128 / 256 rows: 500 rows in 64
// groups, 2048 -> 2048 56 / 76, 4,096 rows 71 / 81, 6,400 rows 1024 -> 1024 28 / 32).
// Power: 8192^3 505 us, 2.18 PFLOP/s of values of one sign.
#define SPARSETIR_GROUPED_KERNEL_ONLY
#include "grouped.cu"

namespace sptir {
namespace {

int product_f8(const char* fn, const void* x, const float* x_scale, const void* w, const float* w_scale, void* y, int y_type,
               const int32_t* indptr, int rows, int groups, int fi, int fo, bool gated, const Gate& gate, int device_id, cudaStream_t st) {
  Args p{};
  p.out = y;
  p.gate = gate;
  p.indptr = indptr;
  p.x_scale = x_scale;
  p.w_scale = w_scale;
  p.rows = rows;
  p.groups = groups;
  p.k = fi;
  p.features = fo;
  p.wide = wide_rows(y, y_type, fo);
  p.idesc = tc05::instr_desc(tc05::kFmtE4M3, 2 * kM, 0, 0, 0);
  const int each = gated ? 2 * fo : fo;  // rows of one W
  const int columns = plan_product(fn, &p, each, 128);
  if (columns < 0) return -1;
  Operand ox{x, rows, fi, 1}, ow{w, static_cast<long long>(groups) * each, fi, 1};
  // us, the kernel for few rows / this one: 1 row, 4096 -> 8192 7.6 / 16.7; 16 rows 10.8 / 17.4; 48 rows, 8 groups, 1024 -> 4096 8.5 / 16.7; 64 rows,
  // 8 groups, 2048 -> 2048 10.3 / 14.3, gated 17.3 / 29.3
  const bool few = fi <= kFewF8Depth && few_rows_pay(rows, groups, fi, each, true);
  const size_t bytes = ox.copy_bytes() + ow.copy_bytes() + (few ? 0 : part_bytes(p));
  CallScratch cs;
  if (bytes > 0 && take_scratch(device_id, st, bytes, 0, &cs) != 0) return -1;
  char* scratch = cs.scratch;
  if (place_operand(&ox, &scratch, st) != 0 || place_operand(&ow, &scratch, st) != 0) return -1;
  if (few) {
    const FewArgs f{ox.data, ow.data, y, x_scale, w_scale, indptr, ox.pitch, ow.pitch, rows, groups, fi, fo, fi, 0, 0, 0, nullptr, gate};
    const int done = few_rows_f8(f, y_type, gated, st);
    return done != 0 ? done : return_scratch(cs, st);
  }
  p.parts = scratch;
  CUtensorMap tm_w, tm_x64, tm_x16;
  if (map_operands(&tm_w, &tm_x64, &tm_x16, CU_TENSOR_MAP_DATA_TYPE_UINT8, ow, ox, fo, groups, true, gated) != 0) return -1;
  int rc;
  if (gated)
    rc = with_half(y_type, [&](auto t) {
      using T = decltype(t);
      if (columns == 128) return launch<kFloat8, kGated, T, 128>(tm_w, tm_x64, tm_x16, p, st);
      return launch<kFloat8, kGated, T, 256>(tm_w, tm_x64, tm_x16, p, st);
    });
  else
    rc = with_type(y_type, [&](auto t) {
      using T = decltype(t);
      if (columns == 128) return launch<kFloat8, kPlain, T, 128>(tm_w, tm_x64, tm_x16, p, st);
      return launch<kFloat8, kPlain, T, 256>(tm_w, tm_x64, tm_x16, p, st);
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
