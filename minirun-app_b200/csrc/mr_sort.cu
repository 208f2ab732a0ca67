// mr_sort.cu — the (token, slot) pairs of a router's choice sorted by expert,
// the tokens' rows copied into that order, and the weighted way back, with
// the gradients of both copies.
//
// With P = T*k pairs, pair p = t*k + j, a plan is
//   offsets[e] = #{p : id(p) < e}, order[offsets[e] + r] = the r-th pair of e,
//   inverse[order[r]] = r
// (stable: pairs of one expert keep their order; no atomics, so the same
// input always gives the same plan). A slot without an expert (id -1) has
// inverse -1; the rows past offsets[E] have order -1.
//   dispatch:          xs[r]   = x[order[r] / k]
//   its gradient:      dx[t]   = sum_j dxs[inverse[t, j]]
//   combine:           out[t]  = base[t] + sum_j w[t, j] * ys[inverse[t, j]]
//   its gradient:      dys[r]  = w(order[r]) * dout[order[r] / k]
//                      dw[t,j] = <dout[t], ys[inverse[t, j]]>
// Sums run in fp32 in slot order and are rounded once, to the rows' type.
#include "mr_host.h"

#include <cooperative_groups.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace mr {
namespace {

// ------------------------------------------------------------------ sort

struct SortParams {
  const int32_t* ids;
  int64_t P;
  int E;
  int64_t chunk;  // pairs per warp, a multiple of 32
  int32_t* order;
  int32_t* inverse;
  int32_t* offsets;
  unsigned* error;
};

constexpr int kSortThreads = 1024;
constexpr int kSortCluster = 8;
constexpr int64_t kSortOneCta = 4096;  // pairs one CTA sorts alone
constexpr int kSortAhead = 4;          // ids in flight per lane

// A counting sort in one launch. Every warp owns a run of consecutive pairs
// and a histogram in shared memory: pass 1 counts (lanes of one expert find
// each other with match.any, so a count is one plain add), prefixes over
// warps, CTAs (distributed shared memory of the cluster) and experts turn
// the histograms into first rows, pass 2 hands out the rows. The grid is one
// cluster (or one CTA); blockDim.x >= E.
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const SortParams p) {
  extern __shared__ int hist[];  // [warps][E], then [E] CTA totals, [E] first rows, [32]
  pdl_wait_and_release();
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int E = p.E;
  const unsigned rank = cluster.block_rank(), ctas = cluster.num_blocks();
  int* total = hist + warps * E;
  int* first = total + E;
  int* wsum = first + E;
  int* mine = hist + warp * E;
  for (int i = tid; i < warps * E; i += blockDim.x) hist[i] = 0;
  __syncthreads();

  const int64_t begin = ((int64_t)rank * warps + warp) * p.chunk;
  const int64_t end = min(begin + p.chunk, p.P);
  bool bad = false;
  for (int64_t b = begin; b < end; b += 32 * kSortAhead) {
    int id[kSortAhead];
#pragma unroll
    for (int a = 0; a < kSortAhead; ++a) {
      const int64_t i = b + 32 * a + lane;
      id[a] = i < end ? __ldg(p.ids + i) : -1;
    }
#pragma unroll
    for (int a = 0; a < kSortAhead; ++a) {
      const bool ok = (unsigned)id[a] < (unsigned)E;
      bad |= !ok && id[a] != -1;
      const unsigned same = __match_any_sync(0xffffffffu, ok ? id[a] : -1);
      if (ok && lane == __ffs(same) - 1) mine[id[a]] += __popc(same);
      __syncwarp();
    }
  }
  if (bad) atomicOr(p.error, MR_DEVERR_BAD_EXPERT_ID);
  __syncthreads();
  // thread e: its expert's counts over the warps, then over the CTAs
  if (tid < E) {
    int run = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = hist[w * E + tid];
      hist[w * E + tid] = run;
      run += c;
    }
    total[tid] = run;
  }
  cluster.sync();
  int before = 0, all = 0;
  if (tid < E) {
    for (unsigned c = 0; c < ctas; ++c) {
      const int n = *cluster.map_shared_rank(total + tid, c);
      if (c < rank) before += n;
      all += n;
    }
  }
  // exclusive scan over the experts
  int incl = all;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += n;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int s = lane < warps ? wsum[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += n;
    }
    wsum[lane] = s;
  }
  __syncthreads();
  const int start = incl - all + (warp ? wsum[warp - 1] : 0);
  const int kept = wsum[warps - 1];
  if (tid < E) {
    first[tid] = start + before;
    if (rank == 0) p.offsets[tid] = start;
  }
  if (rank == 0 && tid == 0) p.offsets[E] = kept;
  __syncthreads();
  for (int64_t b = begin; b < end; b += 32 * kSortAhead) {
    int id[kSortAhead];
#pragma unroll
    for (int a = 0; a < kSortAhead; ++a) {
      const int64_t i = b + 32 * a + lane;
      id[a] = i < end ? __ldg(p.ids + i) : -1;
    }
#pragma unroll
    for (int a = 0; a < kSortAhead; ++a) {
      const int64_t i = b + 32 * a + lane;
      const bool ok = (unsigned)id[a] < (unsigned)E;
      const unsigned same = __match_any_sync(0xffffffffu, ok ? id[a] : -1);
      int row = -1;
      if (ok) row = first[id[a]] + mine[id[a]] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (ok && lane == __ffs(same) - 1) mine[id[a]] += __popc(same);
      __syncwarp();
      if (ok) p.order[row] = (int)i;
      if (i < end) p.inverse[i] = row;
    }
  }
  for (int64_t r = kept + (int64_t)rank * blockDim.x + tid; r < p.P;
       r += (int64_t)ctas * blockDim.x)
    p.order[r] = -1;
  cluster.sync();  // no CTA leaves while another may read its totals
}

// ------------------------------------------------------------- row copies

template <int B>
struct VecOf;
template <>
struct VecOf<16> {
  using T = uint4;
};
template <>
struct VecOf<8> {
  using T = uint2;
};
template <>
struct VecOf<4> {
  using T = uint32_t;
};
template <>
struct VecOf<2> {
  using T = uint16_t;
};

// VB bytes of rows of a type as fp32, and back with one rounding.
template <int DT, int VB>
struct Elems {
  static constexpr int kN = VB / (DT == MR_DTYPE_F32 ? 4 : 2);
  using V = typename VecOf<VB>::T;
  static MR_DEVICE void load(const V& v, float (&f)[kN]) {
    if constexpr (DT == MR_DTYPE_F32) {
      memcpy(f, &v, VB);
    } else {
      uint16_t h[kN];
      memcpy(h, &v, VB);
#pragma unroll
      for (int i = 0; i < kN; ++i)
        f[i] = DT == MR_DTYPE_BF16 ? bf16_bits_to_f32(h[i]) : __half2float(__ushort_as_half(h[i]));
    }
  }
  static MR_DEVICE V store(const float (&f)[kN]) {
    V v;
    if constexpr (DT == MR_DTYPE_F32) {
      memcpy(&v, f, VB);
    } else {
      uint16_t h[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i)
        h[i] = DT == MR_DTYPE_BF16 ? f32_to_bf16_bits(f[i])
                                   : __half_as_ushort(__float2half_rn(f[i]));
      memcpy(&v, h, VB);
    }
    return v;
  }
};

// Rows of `nvec` vectors; a CTA is 256 / group tokens of `group` threads, and
// blockIdx.y one of gridDim.y equal parts of a row.
struct RowParams {
  const char* src;      // token rows (dispatch) or sorted rows (combine)
  int64_t src_stride;   // bytes
  char* dst;            // contiguous
  const char* base;     // combine: contiguous token rows to add, or NULL
  const float* weights; // [T, k], or NULL for ones
  const int32_t* inverse;
  const int32_t* offsets;
  int64_t T, P;
  int k, E;
  int nvec, group, part;  // part: vectors per blockIdx.y
};
constexpr int kRowThreads = 256;

template <typename V>
MR_DEVICE void zero_dropped_rows(char* dst, int64_t P, int64_t kept, int nvec) {
  // rows past offsets[E]: slots without an expert
  const int64_t cta = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  for (int64_t r = max(kept, (int64_t)0) + cta; r < P; r += (int64_t)gridDim.x * gridDim.y)
    for (int v = threadIdx.x; v < nvec; v += blockDim.x)
      reinterpret_cast<V*>(dst)[r * nvec + v] = V{};
}

// xs[inverse[t, j]] = x[t] for every slot: each token row is read once and
// written k times (a copy of P rows reads it k times). Bound by the writes.
template <int VB>
__global__ void __launch_bounds__(kRowThreads) dispatch_kernel(const RowParams p) {
  using V = typename VecOf<VB>::T;
  pdl_wait_and_release();
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / p.group) + threadIdx.x / p.group;
  const int lane = threadIdx.x % p.group;
  const int v1 = min(p.nvec, (int)(blockIdx.y + 1) * p.part);
  if (t < p.T) {
    const V* src = reinterpret_cast<const V*>(p.src + t * p.src_stride);
    V* dst = reinterpret_cast<V*>(p.dst);
    for (int v = blockIdx.y * p.part + lane; v < v1; v += p.group) {
      const V x = __ldg(src + v);
#pragma unroll 8
      for (int j = 0; j < p.k; ++j) {
        const int r = __ldg(p.inverse + t * p.k + j);
        if ((unsigned)r < (unsigned)p.P) dst[(int64_t)r * p.nvec + v] = x;
      }
    }
  }
  zero_dropped_rows<V>(p.dst, p.P, __ldg(p.offsets + p.E), p.nvec);
}

// out[t] = base[t] + sum_j w[t, j] * ys[inverse[t, j]], eight slots' loads in
// flight, added in slot order. Bound by the reads of ys.
template <int DT, int VB>
__global__ void __launch_bounds__(kRowThreads) combine_rows_kernel(const RowParams p) {
  using EL = Elems<DT, VB>;
  using V = typename EL::V;
  constexpr int kN = EL::kN, kAhead = 8;
  pdl_wait_and_release();
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / p.group) + threadIdx.x / p.group;
  const int lane = threadIdx.x % p.group;
  const int v1 = min(p.nvec, (int)(blockIdx.y + 1) * p.part);
  if (t >= p.T) return;
  for (int v = blockIdx.y * p.part + lane; v < v1; v += p.group) {
    float acc[kN];
    if (p.base) {
      EL::load(__ldg(reinterpret_cast<const V*>(p.base) + t * p.nvec + v), acc);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) acc[i] = 0.f;
    }
    for (int j0 = 0; j0 < p.k; j0 += kAhead) {
      V y[kAhead];
      float w[kAhead];
      bool on[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int r = j0 + a < p.k ? __ldg(p.inverse + t * p.k + j0 + a) : -1;
        on[a] = (unsigned)r < (unsigned)p.P;
        if (on[a]) {
          y[a] = __ldg(reinterpret_cast<const V*>(p.src + (int64_t)r * p.src_stride) + v);
          w[a] = p.weights ? __ldg(p.weights + t * p.k + j0 + a) : 1.f;
        }
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (!on[a]) continue;
        float f[kN];
        EL::load(y[a], f);
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[i] = fmaf(w[a], f[i], acc[i]);
      }
    }
    reinterpret_cast<V*>(p.dst)[t * p.nvec + v] = EL::store(acc);
  }
}

struct CombineBwdParams {
  const char* dout;
  int64_t dout_stride;  // bytes
  const char* ys;
  int64_t ys_stride;
  const float* weights;
  const int32_t* inverse;
  const int32_t* offsets;
  char* dys;   // contiguous
  float* dw;   // [T, k]
  int64_t T, P;
  int k, E;
  int nvec;
};

// One CTA per (token, kJ slots): dout[t] and the slots' ys rows pass once;
// dys rows are written from the same registers, and dw is a sum over the CTA
// (lanes by shuffles, warps through shared memory: always the same order).
// Bound by the traffic of ys and dys.
template <int DT, int VB, int kJ>
__global__ void __launch_bounds__(kRowThreads) combine_bwd_kernel(const CombineBwdParams p) {
  using EL = Elems<DT, VB>;
  using V = typename EL::V;
  constexpr int kN = EL::kN, kWarps = kRowThreads / 32;
  __shared__ float part[kWarps][kJ];
  pdl_wait_and_release();
  const int64_t t = blockIdx.x;
  const int j0 = blockIdx.y * kJ;
  int row[kJ];
  float w[kJ], dot[kJ];
#pragma unroll
  for (int a = 0; a < kJ; ++a) {
    const bool in = j0 + a < p.k;
    const int r = in ? __ldg(p.inverse + t * p.k + j0 + a) : -1;
    row[a] = (unsigned)r < (unsigned)p.P ? r : -1;
    w[a] = in ? __ldg(p.weights + t * p.k + j0 + a) : 0.f;
    dot[a] = 0.f;
  }
  const V* g = reinterpret_cast<const V*>(p.dout + t * p.dout_stride);
  for (int v = threadIdx.x; v < p.nvec; v += blockDim.x) {
    V y[kJ];
    const V gv = __ldg(g + v);
#pragma unroll
    for (int a = 0; a < kJ; ++a)
      if (row[a] >= 0)
        y[a] = __ldg(reinterpret_cast<const V*>(p.ys + (int64_t)row[a] * p.ys_stride) + v);
    float gf[kN];
    EL::load(gv, gf);
#pragma unroll
    for (int a = 0; a < kJ; ++a) {
      if (row[a] < 0) continue;
      float f[kN], d[kN];
      EL::load(y[a], f);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        dot[a] = fmaf(gf[i], f[i], dot[a]);
        d[i] = w[a] * gf[i];
      }
      reinterpret_cast<V*>(p.dys)[(int64_t)row[a] * p.nvec + v] = EL::store(d);
    }
  }
#pragma unroll
  for (int a = 0; a < kJ; ++a)
#pragma unroll
    for (int d = 16; d; d >>= 1) dot[a] += __shfl_xor_sync(0xffffffffu, dot[a], d);
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int a = 0; a < kJ; ++a) part[threadIdx.x >> 5][a] = dot[a];
  __syncthreads();
  if (threadIdx.x < kJ && j0 + (int)threadIdx.x < p.k) {
    float s = 0.f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += part[i][threadIdx.x];
    p.dw[t * p.k + j0 + threadIdx.x] = s;
  }
  zero_dropped_rows<V>(p.dys, p.P, __ldg(p.offsets + p.E), p.nvec);
}

// ---------------------------------------------------------------- host

int elem_bytes(mr_dtype d) { return d == MR_DTYPE_F32 ? 4 : 2; }

// Widest vector that divides every address, stride and row.
int vec_bytes(std::initializer_list<uint64_t> all) {
  uint64_t m = 16;
  for (uint64_t a : all) m |= a;
  return (m & 15) == 0 ? 16 : (m & 7) == 0 ? 8 : (m & 3) == 0 ? 4 : 2;
}

}  // namespace

mr_status check_plan(mr_ctx* ctx, const mr_sorted* s) {
  if (!s) return fail(ctx, MR_ERR_INVALID_ARGUMENT, "sorted tokens are NULL");
  if (s->tokens < 0 || s->top_k <= 0 || s->experts <= 0)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                "sorted tokens need tokens >= 0, top_k > 0 and experts > 0 (tokens " +
                    std::to_string(s->tokens) + ", top_k " + std::to_string(s->top_k) +
                    ", experts " + std::to_string(s->experts) + ")");
  if (s->top_k > 1024)
    return fail(ctx, MR_ERR_UNSUPPORTED, "more than 1024 slots a token are not built here");
  if (s->tokens > INT32_MAX / s->top_k)
    return fail(ctx, MR_ERR_UNSUPPORTED, "more than 2^31 - 1 (token, slot) pairs");
  if (!s->offsets || (s->tokens > 0 && (!s->order || !s->inverse)))
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "order, inverse and offsets must be non-NULL");
  return MR_OK;
}

namespace {

mr_status check_rows(mr_ctx* ctx, const mr_sorted* s, mr_dtype dt, int64_t hidden,
                     std::initializer_list<const void*> bufs,
                     std::initializer_list<int64_t> strides) {
  if (mr_status st = check_plan(ctx, s)) return st;
  if (dt != MR_DTYPE_BF16 && dt != MR_DTYPE_F16 && dt != MR_DTYPE_F32)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "rows must be bf16, f16 or f32");
  if (hidden <= 0 || hidden > INT32_MAX / 4)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "hidden must be in 1..2^29");
  for (int64_t n : strides)
    if (n < hidden)
      return fail(ctx, MR_ERR_INVALID_ARGUMENT, "row stride is smaller than the row");
  if (s->tokens > 0)
    for (const void* b : bufs) {
      if (!b) return fail(ctx, MR_ERR_INVALID_ARGUMENT, "row buffers must be non-NULL");
      if (addr(b) % elem_bytes(dt))
        return fail(ctx, MR_ERR_INVALID_ARGUMENT, "row buffers must be aligned to their type");
    }
  return MR_OK;
}

// Threads a token and parts a row is cut into: rows of few vectors share a
// CTA; a batch too small to fill the GPU spreads each row over several CTAs.
void row_shape(const mr_ctx* ctx, RowParams& p, dim3& grid) {
  int g = 8;
  while (g < kRowThreads && g < p.nvec) g *= 2;
  p.group = g;
  const int64_t ctas = (p.T + kRowThreads / g - 1) / (kRowThreads / g);
  int64_t parts = std::min<int64_t>((p.nvec + g - 1) / g, (2 * ctx->sm_count + ctas - 1) / ctas);
  p.part = (int)(((p.nvec + parts - 1) / parts + g - 1) / g * g);
  grid = dim3((unsigned)ctas, (unsigned)((p.nvec + p.part - 1) / p.part));
}

template <int DT>
cudaError_t launch_combine(const RowParams& p, int vb, dim3 grid, cudaStream_t s) {
  switch (vb) {
    case 16: return launch_pdl(combine_rows_kernel<DT, 16>, grid, kRowThreads, 0, s, p);
    case 8: return launch_pdl(combine_rows_kernel<DT, 8>, grid, kRowThreads, 0, s, p);
    case 4: return launch_pdl(combine_rows_kernel<DT, 4>, grid, kRowThreads, 0, s, p);
    default:
      if constexpr (DT != MR_DTYPE_F32)
        return launch_pdl(combine_rows_kernel<DT, 2>, grid, kRowThreads, 0, s, p);
      return cudaErrorMisalignedAddress;  // f32 buffers are 4-byte aligned
  }
}

mr_status combine_rows(mr_ctx* ctx, const void* ys, mr_dtype dt, int64_t stride, int64_t hidden,
                       const float* weights, const void* base, const mr_sorted* s, void* out,
                       void* stream, const char* what) {
  const int es = elem_bytes(dt);
  RowParams p{};
  p.src = static_cast<const char*>(ys);
  p.src_stride = stride * es;
  p.dst = static_cast<char*>(out);
  p.base = static_cast<const char*>(base);
  p.weights = weights;
  p.inverse = s->inverse;
  p.offsets = s->offsets;
  p.T = s->tokens;
  p.k = s->top_k;
  p.P = p.T * p.k;
  p.E = s->experts;
  const int vb = vec_bytes({addr(ys), addr(out), addr(base), (uint64_t)p.src_stride,
                            (uint64_t)(hidden * es)});
  p.nvec = (int)(hidden * es / vb);
  dim3 grid;
  row_shape(ctx, p, grid);
  cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = set_device(ctx);
  if (e == cudaSuccess)
    e = dt == MR_DTYPE_BF16  ? launch_combine<MR_DTYPE_BF16>(p, vb, grid, cs)
        : dt == MR_DTYPE_F16 ? launch_combine<MR_DTYPE_F16>(p, vb, grid, cs)
                             : launch_combine<MR_DTYPE_F32>(p, vb, grid, cs);
  return cuda_check(ctx, e, what);
}

template <int DT, int VB>
cudaError_t launch_bwd(const CombineBwdParams& p, int jn, int threads, cudaStream_t s) {
  const dim3 grid((unsigned)p.T, (unsigned)((p.k + jn - 1) / jn));
  switch (jn) {
    case 8: return launch_pdl(combine_bwd_kernel<DT, VB, 8>, grid, threads, 0, s, p);
    case 4: return launch_pdl(combine_bwd_kernel<DT, VB, 4>, grid, threads, 0, s, p);
    case 2: return launch_pdl(combine_bwd_kernel<DT, VB, 2>, grid, threads, 0, s, p);
    default: return launch_pdl(combine_bwd_kernel<DT, VB, 1>, grid, threads, 0, s, p);
  }
}
template <int DT>
cudaError_t launch_bwd_vec(const CombineBwdParams& p, int vb, int jn, int threads,
                           cudaStream_t s) {
  switch (vb) {
    case 16: return launch_bwd<DT, 16>(p, jn, threads, s);
    case 8: return launch_bwd<DT, 8>(p, jn, threads, s);
    case 4: return launch_bwd<DT, 4>(p, jn, threads, s);
    default:
      if constexpr (DT != MR_DTYPE_F32) return launch_bwd<DT, 2>(p, jn, threads, s);
      return cudaErrorMisalignedAddress;
  }
}

}  // namespace
}  // namespace mr

using namespace mr;

extern "C" {

mr_status mr_moe_sort(mr_ctx* ctx, const int32_t* ids, int64_t tokens, int32_t top_k,
                      int32_t experts, int32_t* order, int32_t* inverse, int32_t* offsets,
                      void* stream) {
  if (!ctx) return MR_ERR_INVALID_ARGUMENT;
  return guarded([&]() -> mr_status {
    const mr_sorted s{order, inverse, offsets, tokens, top_k, experts};
    if (mr_status st = check_plan(ctx, &s)) return st;
    if (tokens > 0 && !ids) return fail(ctx, MR_ERR_INVALID_ARGUMENT, "ids must be non-NULL");
    if (experts > kMaxExperts)
      return fail(ctx, MR_ERR_UNSUPPORTED, "expert counts above 1024 are not built here");
    SortParams p{ids, tokens * top_k, experts, 0, order, inverse, offsets, ctx->d_error};
    const int ctas = p.P <= kSortOneCta ? 1 : kSortCluster;
    const int64_t want = std::max<int64_t>((p.P + 31) / 32, (experts + 31) / 32);
    const int warps = ctas > 1 ? kSortThreads / 32
                               : (int)std::min<int64_t>(kSortThreads / 32, std::max<int64_t>(want, 1));
    const int64_t per = (p.P + (int64_t)ctas * warps - 1) / ((int64_t)ctas * warps);
    p.chunk = (per + 31) / 32 * 32;
    const size_t smem = sizeof(int) * ((size_t)warps * experts + 2 * experts + 32);
    cudaError_t e = set_device(ctx);
    if (e == cudaSuccess && smem > 48 * 1024)
      e = cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) {
      cudaLaunchAttribute attr[2];
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[0].val.programmaticStreamSerializationAllowed = 1;
      attr[1].id = cudaLaunchAttributeClusterDimension;
      attr[1].val.clusterDim.x = ctas;
      attr[1].val.clusterDim.y = 1;
      attr[1].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(ctas);
      cfg.blockDim = dim3(warps * 32);
      cfg.dynamicSmemBytes = smem;
      cfg.stream = reinterpret_cast<cudaStream_t>(stream);
      cfg.attrs = attr;
      cfg.numAttrs = 2;
      e = cudaLaunchKernelEx(&cfg, sort_kernel, p);
    }
    return cuda_check(ctx, e, "sort by expert");
  });
}

mr_status mr_moe_dispatch(mr_ctx* ctx, const void* x, mr_dtype dtype, int64_t x_stride,
                          int64_t hidden, const mr_sorted* plan, void* xs, void* stream) {
  if (!ctx) return MR_ERR_INVALID_ARGUMENT;
  return guarded([&]() -> mr_status {
    if (mr_status st = check_rows(ctx, plan, dtype, hidden, {x, xs}, {x_stride})) return st;
    if (plan->tokens == 0) return MR_OK;
    const int es = elem_bytes(dtype);
    RowParams p{};
    p.src = static_cast<const char*>(x);
    p.src_stride = x_stride * es;
    p.dst = static_cast<char*>(xs);
    p.inverse = plan->inverse;
    p.offsets = plan->offsets;
    p.T = plan->tokens;
    p.k = plan->top_k;
    p.P = p.T * p.k;
    p.E = plan->experts;
    const int vb =
        vec_bytes({addr(x), addr(xs), (uint64_t)p.src_stride, (uint64_t)(hidden * es)});
    p.nvec = (int)(hidden * es / vb);
    dim3 grid;
    row_shape(ctx, p, grid);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = set_device(ctx);
    if (e == cudaSuccess)
      e = vb == 16  ? launch_pdl(dispatch_kernel<16>, grid, kRowThreads, 0, s, p)
          : vb == 8 ? launch_pdl(dispatch_kernel<8>, grid, kRowThreads, 0, s, p)
          : vb == 4 ? launch_pdl(dispatch_kernel<4>, grid, kRowThreads, 0, s, p)
                    : launch_pdl(dispatch_kernel<2>, grid, kRowThreads, 0, s, p);
    return cuda_check(ctx, e, "dispatch");
  });
}

mr_status mr_moe_dispatch_backward(mr_ctx* ctx, const void* dxs, mr_dtype dtype,
                                   int64_t dxs_stride, int64_t hidden, const mr_sorted* plan,
                                   void* dx, void* stream) {
  if (!ctx) return MR_ERR_INVALID_ARGUMENT;
  return guarded([&]() -> mr_status {
    if (mr_status st = check_rows(ctx, plan, dtype, hidden, {dxs, dx}, {dxs_stride})) return st;
    if (plan->tokens == 0) return MR_OK;
    return combine_rows(ctx, dxs, dtype, dxs_stride, hidden, nullptr, nullptr, plan, dx, stream,
                        "dispatch backward");
  });
}

mr_status mr_moe_combine(mr_ctx* ctx, const void* ys, mr_dtype dtype, int64_t ys_stride,
                         int64_t hidden, const float* weights, const void* base,
                         const mr_sorted* plan, void* out, void* stream) {
  if (!ctx) return MR_ERR_INVALID_ARGUMENT;
  return guarded([&]() -> mr_status {
    if (mr_status st = check_rows(ctx, plan, dtype, hidden, {ys, out}, {ys_stride})) return st;
    if (plan->tokens == 0) return MR_OK;
    if (!weights) return fail(ctx, MR_ERR_INVALID_ARGUMENT, "weights must be non-NULL");
    if (addr(base) % elem_bytes(dtype))
      return fail(ctx, MR_ERR_INVALID_ARGUMENT, "row buffers must be aligned to their type");
    return combine_rows(ctx, ys, dtype, ys_stride, hidden, weights, base, plan, out, stream,
                        "combine");
  });
}

mr_status mr_moe_combine_backward(mr_ctx* ctx, const void* dout, int64_t dout_stride,
                                  const void* ys, int64_t ys_stride, mr_dtype dtype,
                                  int64_t hidden, const float* weights, const mr_sorted* plan,
                                  void* dys, float* dweights, void* stream) {
  if (!ctx) return MR_ERR_INVALID_ARGUMENT;
  return guarded([&]() -> mr_status {
    if (mr_status st = check_rows(ctx, plan, dtype, hidden, {dout, ys, dys},
                                  {dout_stride, ys_stride}))
      return st;
    if (plan->tokens == 0) return MR_OK;
    if (!weights || !dweights)
      return fail(ctx, MR_ERR_INVALID_ARGUMENT, "weights and dweights must be non-NULL");
    const int es = elem_bytes(dtype);
    CombineBwdParams p{};
    p.dout = static_cast<const char*>(dout);
    p.dout_stride = dout_stride * es;
    p.ys = static_cast<const char*>(ys);
    p.ys_stride = ys_stride * es;
    p.weights = weights;
    p.inverse = plan->inverse;
    p.offsets = plan->offsets;
    p.dys = static_cast<char*>(dys);
    p.dw = dweights;
    p.T = plan->tokens;
    p.k = plan->top_k;
    p.P = p.T * p.k;
    p.E = plan->experts;
    const int vb = vec_bytes({addr(dout), addr(ys), addr(dys), (uint64_t)p.dout_stride,
                              (uint64_t)p.ys_stride, (uint64_t)(hidden * es)});
    p.nvec = (int)(hidden * es / vb);
    const int threads = std::min(kRowThreads, (p.nvec + 31) / 32 * 32);
    int jn = 1;  // slots per CTA: all of them once the tokens alone fill the GPU
    while (jn < 8 && jn < p.k && p.T * ((p.k + 2 * jn - 1) / (2 * jn)) >= 4 * ctx->sm_count)
      jn *= 2;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = set_device(ctx);
    if (e == cudaSuccess)
      e = dtype == MR_DTYPE_BF16  ? launch_bwd_vec<MR_DTYPE_BF16>(p, vb, jn, threads, s)
          : dtype == MR_DTYPE_F16 ? launch_bwd_vec<MR_DTYPE_F16>(p, vb, jn, threads, s)
                                  : launch_bwd_vec<MR_DTYPE_F32>(p, vb, jn, threads, s);
    return cuda_check(ctx, e, "combine backward");
  });
}

}  // extern "C"
