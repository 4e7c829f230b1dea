// The gated block of an expert in one product, and its gradient through the product that follows it, on the tensor cores
// (grouped.cu; the epilogues are in grouped_gated.cuh):
//   grouped_mm_gated       h = x W[g]^T of 2 * width features, act = f(h[:, :width]) * h[:, width:]  (gate.cuh)
//   grouped_mm_gated_grad  d = dy W[g], and from d and h the gradient to h
// A gated tile is 128 features of act, 256 rows of W: in every 32 of them 16 of the gate and the same 16 of the other projection, which TMA brings
// side by side (a box of 16 x 2 rows), so that both meet in one thread of the epilogue.  The gradient's epilogue has the projections of the next 32
// rows on their way while it works, and puts their gradients where they lay in shared memory.
// 65,536 rows, 64 groups, 2048 -> 2 x 1024, bf16: 434 us with both projections kept (even groups; 1.27 PFLOP/s, the plain product of that size
// 404 to 460), 462 to 564 with ragged ones (calls in a row, runs of seconds); the gradient 285 and 317 to 362: without its loads and stores of the projections 226, its 1.2 GB alone are 184.
#define SPARSETIR_GROUPED_KERNEL_ONLY
#include "grouped.cu"

namespace sptir {
namespace {

template <int OUT>
int launch_half(int columns, int type, const CUtensorMap& w, const CUtensorMap& x64, const CUtensorMap& x16, const GatedArgs& p, cudaStream_t st) {
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    if (columns == 128) return launch<false, OUT, T, 128>(w, x64, x16, p, st);
    return launch<false, OUT, T, 256>(w, x64, x16, p, st);
  });
}

}  // namespace

int gated_timeouts(unsigned int* count) {
  SPTIR_CUDA_OK(cudaMemcpyFromSymbol(count, g_grouped_timeouts, sizeof(unsigned int)));
  return 0;
}

}  // namespace sptir

using namespace sptir;

extern "C" int sparsetir_grouped_mm_gated_raw(const void* x, const void* w, void* y, void* hidden, int type, const int32_t* indptr,
                                              int rows, int num_groups, int feat_in, int width, int flags, int device_id,
                                              void* stream) {
  const char* fn = "sparsetir_grouped_mm_gated";
  if (check_block(fn, indptr, rows, num_groups, feat_in, width, true, flags, SPARSETIR_GATED_GELU) != 0) return -1;
  if (type != SPARSETIR_F16 && type != SPARSETIR_BF16) return fail("%s: x, w, y and hidden are f16 or bf16", fn);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !w || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  GatedArgs p{};
  p.out = y;
  p.hidden = hidden;
  p.gate = Gate((flags & SPARSETIR_GATED_GELU) != 0);
  p.indptr = indptr;
  p.rows = rows;
  p.groups = num_groups;
  p.k = feat_in;
  p.features = width;
  p.wide = wide_rows(y, type, width) && aligned16(hidden);
  p.idesc = tc05::instr_desc(map_format(type), 2 * kM, 0, 0, 0);
  const int columns = plan_product(fn, &p, 2 * width, 64);
  if (columns < 0) return -1;
  // us, weights out of HBM, the kernel for few rows / this one: 8 groups of 3 and 8 rows, 1024 -> 2 x 2048 13.8 / 14.8, 14.6 / 14.9; one group of 1 and
  // 16 rows, 4096 -> 2 x 4096 13.2 / 17.9, 14.2 / 18.4
  const bool few = few_rows_pay(rows, num_groups, feat_in, 2 * width, true);
  Operand ox{x, rows, feat_in, 2}, ow{w, static_cast<long long>(num_groups) * 2 * width, feat_in, 2};
  const size_t bytes = ox.copy_bytes() + ow.copy_bytes() + (few ? 0 : part_bytes(p));
  CallScratch cs;
  if (bytes > 0 && take_scratch(device_id, st, bytes, 0, &cs) != 0) return -1;
  char* scratch = cs.scratch;
  if (place_operand(&ox, &scratch, st) != 0 || place_operand(&ow, &scratch, st) != 0) return -1;
  if (few) {
    const FewGatedArgs f{{ox.data, ow.data, y, nullptr, nullptr, indptr, ox.pitch, ow.pitch, rows, num_groups, feat_in, width, feat_in * 2, 0, 0, 0},
                         hidden, p.gate};
    const int done = few_rows_gated(f, type, st);
    return done != 0 ? done : return_scratch(cs, st);
  }
  p.parts = scratch;
  CUtensorMap tm_w, tm_x64, tm_x16;
  if (map_operands(&tm_w, &tm_x64, &tm_x16, map_type(type), ow, ox, width, num_groups, true, true) != 0) return -1;
  const int rc = launch_half<kGated>(columns, type, tm_w, tm_x64, tm_x16, p, st);
  return rc != 0 ? rc : return_scratch(cs, st);
}

extern "C" int sparsetir_grouped_mm_gated_grad_raw(const void* dy, const void* w, const void* hidden, void* d_hidden, void* act,
                                                   int type, const int32_t* indptr, int rows, int num_groups, int feat, int width,
                                                   int flags, int device_id, void* stream) {
  const char* fn = "sparsetir_grouped_mm_gated_grad";
  if (check_block(fn, indptr, rows, num_groups, feat, width, true, flags, SPARSETIR_GATED_GELU | SPARSETIR_GROUPED_W_OUT_IN) != 0) return -1;
  if (type != SPARSETIR_F16 && type != SPARSETIR_BF16) return fail("%s: all tensors are f16 or bf16", fn);
  if (rows == 0 || num_groups == 0) return 0;
  if (!dy || !w || !hidden || !d_hidden) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  const bool out_in = (flags & SPARSETIR_GROUPED_W_OUT_IN) != 0;
  GatedArgs p{};
  p.out = act;
  p.hidden_in = hidden;
  p.hidden = d_hidden;
  p.gate = Gate((flags & SPARSETIR_GATED_GELU) != 0);
  p.indptr = indptr;
  p.rows = rows;
  p.groups = num_groups;
  p.k = feat;
  p.features = width;
  p.a_mn = out_in ? 0 : 1;
  p.wide = wide_rows(d_hidden, type, width) && aligned16(hidden) && aligned16(act);
  p.idesc = tc05::instr_desc(map_format(type), 2 * kM, 0, p.a_mn, 0);
  const int columns = plan_product(fn, &p, width, 64);
  if (columns < 0) return -1;
  Operand ox{dy, rows, feat, 2}, ow{w, static_cast<long long>(num_groups) * (out_in ? width : feat), out_in ? feat : width, 2};
  const size_t bytes = ox.copy_bytes() + ow.copy_bytes() + part_bytes(p);
  CallScratch cs;
  if (bytes > 0 && take_scratch(device_id, st, bytes, 0, &cs) != 0) return -1;
  char* scratch = cs.scratch;
  if (place_operand(&ox, &scratch, st) != 0 || place_operand(&ow, &scratch, st) != 0) return -1;
  p.parts = scratch;
  CUtensorMap tm_w, tm_x64, tm_x16;
  if (map_operands(&tm_w, &tm_x64, &tm_x16, map_type(type), ow, ox, out_in ? width : feat, num_groups, out_in, false) != 0) return -1;
  const int rc = p.wide ? launch_half<kGatedGrad>(columns, type, tm_w, tm_x64, tm_x16, p, st)
                        : launch_half<kGatedGradAny>(columns, type, tm_w, tm_x64, tm_x16, p, st);
  return rc != 0 ? rc : return_scratch(cs, st);
}
