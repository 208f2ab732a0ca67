// mr_mxmm.cu — entry points of the MXFP4 x MXFP4 products (mr_mxmm.cuh).
#include "mr_mxmm.cuh"

#include <algorithm>

#include "mr_host.h"

namespace mr {
namespace {

constexpr int kMmSmem = 227 * 1024;

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000,
                                                           cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeFn>(p)
                                                                : nullptr;
  }();
  return fn;
}

// Rows of `bytes` bytes, boxes of box_rows x 128 bytes, 128-byte swizzle.
// Bytes past a row's end and rows past the last read as zero.
bool encode_codes(CUtensorMap* map, const void* base, int64_t rows, int64_t bytes, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)bytes};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t step[2] = {1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides,
                   box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

mr_status check_operand(mr_ctx* ctx, const mr_mxfp4_desc* d, bool empty_ok, const char* name) {
  if (!d) return fail(ctx, MR_ERR_INVALID_ARGUMENT, std::string(name) + " is NULL");
  if (empty_ok && d->out_features == 0) return MR_OK;
  char why[256] = "";
  if (mr_status st = mr_mxfp4_validate(d, why, sizeof why))
    return fail(ctx, st, std::string(name) + ": " + why);
  if (addr(d->packed) % 16)
    return fail(ctx, MR_ERR_UNSUPPORTED, std::string(name) + ": packed must be 16-byte aligned");
  const int64_t rows = std::max<int64_t>(d->experts, 1) * d->out_features;
  if (rows > INT32_MAX - 256 || d->in_features > INT32_MAX / 2)
    return fail(ctx, MR_ERR_UNSUPPORTED, std::string(name) + ": more than 2^31 rows or columns");
  return MR_OK;
}

// rows: of the result. plan == NULL: one matrix.
mr_status product(mr_ctx* ctx, const mr_mxfp4_desc* a, const mr_mxfp4_desc* w,
                  const mr_sorted* plan, bool by_token, int64_t rows, mr_dtype out_dtype,
                  void* out, void* stream) {
  if (a->in_features != w->in_features)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                "a has " + std::to_string(a->in_features) + " features, weights expect " +
                    std::to_string(w->in_features));
  if (out_dtype != MR_DTYPE_BF16 && out_dtype != MR_DTYPE_F32)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "out must be bf16 or f32");
  if (rows == 0) return MR_OK;
  if (!out) return fail(ctx, MR_ERR_INVALID_ARGUMENT, "out must be non-NULL");
  if (addr(out) % (out_dtype == MR_DTYPE_F32 ? 4 : 2))
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "out must be aligned to its type");
  if (!encoder()) return fail(ctx, MR_ERR_UNSUPPORTED, "the driver has no tensor maps");

  MmParams p{};
  p.w_scales = w->scales;
  p.a_scales = a->scales;
  p.offsets = plan ? plan->offsets : nullptr;
  p.order = by_token ? plan->order : nullptr;
  p.out = out;
  p.error = ctx->d_error;
  p.rows = rows;
  p.arows = a->out_features;
  p.out_features = w->out_features;
  p.E = plan ? w->experts : 1;
  const uint64_t k = plan ? plan->top_k : 1;
  while ((1ull << p.k_shift) < k) ++p.k_shift;
  p.k_mul = (uint32_t)(((1ull << (31 + p.k_shift)) + k - 1) / k);
  p.groups = (int)(w->in_features / 32);
  p.nstages = (int)((w->in_features + kMmK - 1) / kMmK);
  p.out_f32 = out_dtype == MR_DTYPE_F32;
  const bool wide =
      p.groups % 16 == 0 && addr(w->scales) % 16 == 0 && addr(a->scales) % 16 == 0;
  // Tile width: three times an expert's mean rows, so that few experts need a
  // second tile, which would load their weights again; narrow tiles leave room
  // for a deeper ring. Against twice the mean, 256 experts of 1024 x 3584 and
  // 8 slots a token: 512 tokens 84 -> 82 us and 1024 84 -> 86 with even experts,
  // 91 -> 83 and 100 -> 90 where the most popular has ten times the mean; four
  // times is as good as three. Tiles are at most one per expert with rows and
  // the full ones.
  const int64_t mean = plan ? (rows + p.E - 1) / p.E : rows;
  const int64_t want = plan ? std::min(rows, 3 * mean) : rows;
  const int sms = ctx->sm_count;
  auto tiles_of = [&](int ntile, int cg) {
    return (std::min<int64_t>(p.E, rows) + (rows - 1) / ntile) *
           ((w->out_features + kMmRows * cg - 1) / (kMmRows * cg));
  };
  p.ntile = want <= 16 ? 16 : want <= 32 ? 32 : want <= 64 ? 64 : want <= 128 ? 128 : kMmMaxN;
  const int cg = p.ntile > 64 ? 2 : 1;
  const int64_t tiles = tiles_of(p.ntile, cg);
  if (tiles > INT32_MAX)
    return fail(ctx, MR_ERR_UNSUPPORTED, "the product has more than 2^31 tiles");
  p.ksplit = 1;
  // CTAs share a tile where there are few, the rows are long and the tile is
  // narrow (1 and 16 rows x 2048 x 7168 in L2: 8.3 -> 6.5 us and 8.1 -> 6.8; with 32
  // rows, or rows of 2048, the exchange costs what the shorter loop saves).
  while (p.ntile == 16 && p.ksplit < kMmSplit && 2 * p.ksplit * tiles <= sms && p.nstages >= 8)
    p.ksplit *= 2;
  p.mtiles = (int)((w->out_features + kMmRows * cg - 1) / (kMmRows * cg));
  p.box = p.order ? 1 : p.ntile > 32 ? p.ntile / 2 : p.ntile;
  const int fixed = mm_fixed_bytes(p.E, p.ntile, p.ksplit);
  p.nst = std::min((512 - 2 * p.ntile) / mm_sf_cols(p.ntile),
                   (kMmSmem - fixed) / mm_stage_bytes(p.ntile, cg));
  const int used = fixed + p.nst * mm_stage_bytes(p.ntile, cg);
  const int part = p.ksplit > 1 ? p.ntile * kMmRows * 4 : 0;
  p.part_at = (used - 1024 - part) & ~15;  // the last bytes; the first 1024 are for alignment
  const int smem = used;

  MmMaps maps;
  const int64_t bytes = w->in_features / 2;
  if (!encode_codes(&maps.w, w->packed, (int64_t)p.E * w->out_features, bytes, kMmRows) ||
      !encode_codes(&maps.a, a->packed, a->out_features, bytes, p.box))
    return fail(ctx, MR_ERR_UNSUPPORTED, "cannot describe the operands as tensor maps");
  const int unit = cg * p.ksplit;  // CTAs that work together
  const int grid = (int)std::min<int64_t>(sms / unit, tiles) * unit;
  const int threads = kMmThreads + (p.order ? 32 * kMmGatherWarps : 0);
  auto* kernel = cg == 1 ? (wide ? mxmm_kernel<true, 1> : mxmm_kernel<false, 1>)
                         : (wide ? mxmm_kernel<true, 2> : mxmm_kernel<false, 2>);
  const DeviceScope on(ctx);
  cudaError_t e = on.err;
  if (e == cudaSuccess)
    e = attrs_once(ctx, kAttrProduct << (2 * (cg - 1) + wide), [&] {
      return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMmSmem);
    });
  if (e == cudaSuccess) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unit;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kernel, p, maps);
  }
  return cuda_check(ctx, e, "MXFP4 product");
}

}  // namespace
}  // namespace mr

using namespace mr;

extern "C" {

mr_status mr_mxfp4_scaled_mm(mr_ctx* ctx, const mr_mxfp4_desc* a, const mr_mxfp4_desc* w,
                             mr_dtype out_dtype, void* out, void* stream) {
  if (!ctx) return MR_ERR_INVALID_ARGUMENT;
  return guarded([&]() -> mr_status {
    mr_status st = check_operand(ctx, a, true, "a");
    if (!st) st = check_operand(ctx, w, false, "w");
    if (st) return st;
    if (a->experts != 0 || w->experts != 0)
      return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                  "mxfp4 scaled mm needs single matrices; use the grouped form for a stack");
    if (a->out_features > INT32_MAX - 256)
      return fail(ctx, MR_ERR_UNSUPPORTED, "more than 2^31 rows");
    return product(ctx, a, w, nullptr, false, a->out_features, out_dtype, out, stream);
  });
}

mr_status mr_mxfp4_grouped_mm(mr_ctx* ctx, const mr_mxfp4_desc* a, const mr_mxfp4_desc* w,
                              const mr_sorted* plan, int by_token, mr_dtype out_dtype, void* out,
                              void* stream) {
  if (!ctx) return MR_ERR_INVALID_ARGUMENT;
  return guarded([&]() -> mr_status {
    mr_status st = check_plan(ctx, plan);
    if (!st) st = check_operand(ctx, a, plan->tokens == 0, "a");
    if (!st) st = check_operand(ctx, w, false, "w");
    if (st) return st;
    if (a->experts != 0 || w->experts == 0)
      return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                  "mxfp4 grouped mm needs a single matrix of activations and an expert stack");
    if (w->experts != plan->experts)
      return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                  "the stack has " + std::to_string(w->experts) + " experts, the tokens are " +
                      "sorted into " + std::to_string(plan->experts));
    if (w->experts > kMaxExperts)
      return fail(ctx, MR_ERR_UNSUPPORTED, "expert stacks larger than 1024 are not built here");
    const int64_t rows = plan->tokens * plan->top_k;
    if (a->out_features != (by_token ? plan->tokens : rows))
      return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                  "a must hold the " + std::string(by_token ? "tokens'" : "sorted") + " rows, " +
                      std::to_string(by_token ? plan->tokens : rows) + ", and has " +
                      std::to_string(a->out_features));
    if (rows > INT32_MAX - 256) return fail(ctx, MR_ERR_UNSUPPORTED, "more than 2^31 rows");
    return product(ctx, a, w, plan, by_token != 0, rows, out_dtype, out, stream);
  });
}

}  // extern "C"
