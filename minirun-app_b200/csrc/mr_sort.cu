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
  int bits;       // 2^bits > E
  int32_t* order;
  int32_t* inverse;
  int32_t* offsets;
  unsigned* error;
};

constexpr int kSortThreads = 1024;
constexpr int kSortCluster = 16;  // CTAs of a large sort's cluster
constexpr int64_t kSortOneCta = 4096;  // pairs one CTA sorts alone
constexpr int kSortSmem = 4 * (kSortThreads / 32 * kMaxExperts + 2 * kMaxExperts + 32);
constexpr int kSortBatch = 4;          // groups of 32 pairs a warp has in registers
constexpr int kSortColumn = 8;         // histogram entries loaded together

// The lanes of the warp with this lane's key (< 2^bits). Ballots: match.any
// took 50 cycles of the SM a time, most of the kernel's at 32768 pairs.
MR_DEVICE unsigned lanes_with(unsigned key, int bits) {
  unsigned same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = key >> b & 1;
    const unsigned v = __ballot_sync(0xffffffffu, one);
    same &= one ? v : ~v;
  }
  return same;
}

// A counting sort in one launch. Every warp owns a run of consecutive pairs
// and a histogram in shared memory: pass 1 counts (lanes of one expert find
// each other by ballots, so a count is one plain add), prefixes over
// warps, CTAs (distributed shared memory of the cluster) and experts turn
// the histograms into first rows, pass 2 hands out the rows. The grid is one
// cluster (or one CTA); blockDim.x >= E. Latency-bound: ids, then the
// cluster barrier, then the scattered rows. 256 experts: 32 pairs 2 us, 32768
// 7.6 us (one CTA 13.7), 65536 9 us (22). More than 4096 pairs need a GPU (or a
// part of one) that places 16 CTAs of one cluster; where it cannot, the launch
// fails and the call says so.
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const SortParams p) {
  extern __shared__ int hist[];  // [warps][E], then [E] CTA totals, [E] first rows, [32]
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int E = p.E;
  const unsigned rank = cluster.block_rank(), ctas = cluster.num_blocks();
  int* total = hist + warps * E;
  int* first = total + E;
  int* wsum = first + E;
  int* mine = hist + warp * E;
  for (int i = lane; i < E; i += 32) mine[i] = 0;
  __syncwarp();
  pdl_wait_and_release();

  const int64_t begin = ((int64_t)rank * warps + warp) * p.chunk;
  const int64_t end = min(begin + p.chunk, p.P);
  bool bad = false;
  int id[kSortBatch];
  unsigned same[kSortBatch];
  auto load = [&](int64_t b) {
#pragma unroll
    for (int a = 0; a < kSortBatch; ++a) {
      const int64_t i = b + 32 * a + lane;
      id[a] = i < end ? __ldg(p.ids + i) : -1;
    }
  };
  for (int64_t b = begin; b < end; b += 32 * kSortBatch) {
    load(b);
#pragma unroll
    for (int a = 0; a < kSortBatch; ++a) {
      if (b + 32 * a >= end) break;
      const bool ok = (unsigned)id[a] < (unsigned)E;
      bad |= !ok && id[a] != -1;
      same[a] = lanes_with(ok ? id[a] : E, p.bits);
      if (ok && lane == __ffs(same[a]) - 1) mine[id[a]] += __popc(same[a]);
      __syncwarp();
    }
  }
  if (bad) atomicOr(p.error, MR_DEVERR_BAD_EXPERT_ID);
  __syncthreads();
  // thread e: its expert's counts over the warps, then over the CTAs
  if (tid < E) {
    int run = 0;
    for (int w0 = 0; w0 < warps; w0 += kSortColumn) {
      int c[kSortColumn];
#pragma unroll
      for (int i = 0; i < kSortColumn; ++i) c[i] = w0 + i < warps ? hist[(w0 + i) * E + tid] : 0;
#pragma unroll
      for (int i = 0; i < kSortColumn; ++i) {
        if (w0 + i < warps) hist[(w0 + i) * E + tid] = run;
        run += c[i];
      }
    }
    total[tid] = run;
  }
  int before = 0, all = 0;
  if (ctas == 1) {
    if (tid < E) all = total[tid];
  } else {
    cluster.sync();
    if (tid < E) {
      int n[kSortCluster];
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c)
        n[c] = c < (int)ctas ? *cluster.map_shared_rank(total + tid, c) : 0;
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c) {
        if (c < (int)rank) before += n[c];
        all += n[c];
      }
    }
    // no CTA leaves (below) before the others have read its totals; not the
    // .aligned forms: a warp's lanes may have parted above
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
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
  int ws = lane < warps ? wsum[lane] : 0;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, ws, d);
    if (lane >= d) ws += n;
  }
  const int kept = __shfl_sync(0xffffffffu, ws, 31);
  const int lower = __shfl_sync(0xffffffffu, ws, max(warp - 1, 0));
  const int start = incl - all + (warp ? lower : 0);
  if (tid < E) {
    first[tid] = start + before;
    if (rank == 0) p.offsets[tid] = start;
  }
  if (rank == 0 && tid == 0) p.offsets[E] = kept;
  __syncthreads();
  const bool in_registers = p.chunk <= 32 * kSortBatch;
  for (int64_t b = begin; b < end; b += 32 * kSortBatch) {
    if (!in_registers) load(b);
#pragma unroll
    for (int a = 0; a < kSortBatch; ++a) {
      if (b + 32 * a >= end) break;
      const int64_t i = b + 32 * a + lane;
      const bool ok = (unsigned)id[a] < (unsigned)E;
      if (!in_registers) same[a] = lanes_with(ok ? id[a] : E, p.bits);
      int row = -1;
      if (ok) row = first[id[a]] + mine[id[a]] + __popc(same[a] & ((1u << lane) - 1u));
      __syncwarp();
      if (ok && lane == __ffs(same[a]) - 1) mine[id[a]] += __popc(same[a]);
      __syncwarp();
      if (ok) p.order[row] = (int)i;
      if (i < end) p.inverse[i] = row;
    }
  }
  for (int64_t r = kept + (int64_t)rank * blockDim.x + tid; r < p.P;
       r += (int64_t)ctas * blockDim.x)
    p.order[r] = -1;
  if (ctas > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
}

// ------------------------------------------------------------- row copies
//
// VB: rows are worked on in vectors of 16, 8 or 4 bytes, the widest that
// divides every address, stride and width. Rows of 16-bit elements at odd
// places have no such vector (VB = 0): they go in 16-byte pieces of the row
// that is written, so that the stores are whole vectors but for a row's first
// and last, and what is read comes from the one or two aligned vectors around
// it (30000 x 2 rows of 131 f16: 20 us, 32 us element by element; at 8 bytes
// the vectors are faster, 6.9 against 9.8 us for 1021 x 6 rows of 1030 fp32).
template <int VB>
struct VecOf {
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

// Elements of a vector as fp32, and back with one rounding.
template <int DT, int VB>
struct Elems {
  static constexpr int kSize = DT == MR_DTYPE_F32 ? 4 : 2;
  static constexpr int kBytes = VB ? VB : 16;
  static constexpr int kN = kBytes / kSize;
  using V = typename VecOf<VB>::T;
  static MR_DEVICE void load(const V& v, float (&f)[kN]) {
    if constexpr (DT == MR_DTYPE_F32) {
      memcpy(f, &v, kBytes);
    } else {
      uint16_t h[kN];
      memcpy(h, &v, kBytes);
#pragma unroll
      for (int i = 0; i < kN; ++i)
        f[i] = DT == MR_DTYPE_BF16 ? bf16_bits_to_f32(h[i]) : __half2float(__ushort_as_half(h[i]));
    }
  }
  static MR_DEVICE V store(const float (&f)[kN]) {
    V v;
    if constexpr (DT == MR_DTYPE_F32) {
      memcpy(&v, f, kBytes);
    } else {
      uint16_t h[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i)
        h[i] = DT == MR_DTYPE_BF16 ? f32_to_bf16_bits(f[i])
                                   : __half_as_ushort(__float2half_rn(f[i]));
      memcpy(&v, h, kBytes);
    }
    return v;
  }
};

// What may be read of a tensor of rows.
struct Span {
  const char* lo;
  const char* hi;
};
MR_DEVICE Span span_of(const char* base, int64_t rows, int64_t stride, int64_t bytes) {
  return Span{base, base + (rows - 1) * stride + bytes};
}

// 16 bytes at a 16-bit element; those outside the span are zero.
MR_DEVICE uint4 load_any(const char* at, const Span& s) {
  const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(at) & 15u;
  const char* base = at - off;
  uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (base >= s.lo && base + 32 <= s.hi) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(base));
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(base) + 1);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = (off & 8) ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = (off & 4) ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (off & 2));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const char* e = at + 2 * i;
      if (e >= s.lo && e + 2 <= s.hi)
        w[i >> 1] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(e)) << (16 * (i & 1));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Vector v of a row; VB = 0: the 16 bytes from `at` (see first_of).
template <int VB>
MR_DEVICE typename VecOf<VB>::T load_vec(const char* row, int v, int64_t at, const Span& s) {
  if constexpr (VB != 0)
    return __ldg(reinterpret_cast<const typename VecOf<VB>::T*>(row) + v);
  else
    return load_any(row + at, s);
}
// VB = 0: piece v's first byte relative to the row's that is written; negative
// in the first piece of a row that does not start on a boundary.
template <int VB>
MR_DEVICE int64_t first_of(const char* row, int v) {
  return VB ? 0 : 16 * (int64_t)v - (int64_t)(reinterpret_cast<uintptr_t>(row) & 15u);
}
template <int VB>
MR_DEVICE void store_vec(char* row, int v, int64_t at, int64_t bytes,
                         const typename VecOf<VB>::T& x) {
  if constexpr (VB != 0) {
    reinterpret_cast<typename VecOf<VB>::T*>(row)[v] = x;
  } else if (at >= 0 && at + 16 <= bytes) {
    *reinterpret_cast<uint4*>(row + at) = x;
  } else {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t e = at + 2 * i;
      if (e >= 0 && e < bytes)
        *reinterpret_cast<uint16_t*>(row + e) = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// A CTA is kRowThreads / group tokens of `group` threads; blockIdx.y is one of
// gridDim.y equal parts of a row (combine backward: of the slots).
struct RowParams {
  const char* src;      // token rows (dispatch) or sorted rows
  int64_t src_stride;   // bytes
  const char* dout;     // combine backward: token rows
  int64_t dout_stride;
  char* dst;            // contiguous
  const char* base;     // combine: contiguous token rows to add, or NULL
  const float* weights; // [T, k], or NULL for ones
  float* dw;            // combine backward: [T, k]
  const int32_t* inverse;
  const int32_t* offsets;
  int64_t T, P;
  int64_t bytes;        // of a row
  int k, E;
  int nvec, part;         // vectors of a row at most, of a part
  int group, log_group;   // threads of a token, a power of two
};
constexpr int kRowThreads = 256;
constexpr int kRowSlots = 8;  // slots whose loads are in flight together

// rows past offsets[E]: slots without an expert
template <int VB>
MR_DEVICE void zero_dropped_rows(const RowParams& p) {
  const int64_t kept = max((int64_t)__ldg(p.offsets + p.E), (int64_t)0);
  const int64_t cta = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  for (int64_t r = kept + cta; r < p.P; r += (int64_t)gridDim.x * gridDim.y) {
    char* row = p.dst + r * p.bytes;
    for (int v = threadIdx.x; v < p.nvec; v += blockDim.x)
      store_vec<VB>(row, v, first_of<VB>(row, v), p.bytes, typename VecOf<VB>::T{});
  }
}

// xs[inverse[t, j]] = x[t] for every slot: each token row is read once and
// written k times (a copy of P rows reads it k times). Bound by the writes: 91
// us at 4096 x 8 rows of 7168 bf16, 0.88 of the copy rate.
template <int VB>
__global__ void __launch_bounds__(kRowThreads) dispatch_kernel(const RowParams p) {
  using V = typename VecOf<VB>::T;
  pdl_wait_and_release();
  const int64_t t = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> p.log_group;
  const int lane = threadIdx.x & (p.group - 1);
  const int v1 = min(p.nvec, (int)(blockIdx.y + 1) * p.part);
  if (t < p.T) {
    const char* src = p.src + t * p.src_stride;
    const Span span = span_of(p.src, p.T, p.src_stride, p.bytes);
    for (int v = blockIdx.y * p.part + lane; v < v1; v += p.group) {
      V x;
      if constexpr (VB != 0) x = load_vec<VB>(src, v, 0, span);
#pragma unroll 8
      for (int j = 0; j < p.k; ++j) {
        const int r = __ldg(p.inverse + t * p.k + j);
        if ((unsigned)r >= (unsigned)p.P) continue;
        char* dst = p.dst + (int64_t)r * p.bytes;
        const int64_t at = first_of<VB>(dst, v);
        if constexpr (VB == 0) {
          if (at >= p.bytes) continue;
          x = load_vec<VB>(src, v, at, span);
        }
        store_vec<VB>(dst, v, at, p.bytes, x);
      }
    }
  }
  zero_dropped_rows<VB>(p);
}

// out[t] = base[t] + sum_j w[t, j] * ys[inverse[t, j]], the loads of eight
// slots in flight, added in slot order. Bound by the reads of ys: 86 us at
// 4096 x 8 rows of 7168 bf16, 0.94 of the copy rate. (With the rows' numbers
// loaded inside the loop over a row the kernel took twice as long.)
template <int DT, int VB>
__global__ void __launch_bounds__(kRowThreads) combine_rows_kernel(const RowParams p) {
  using EL = Elems<DT, VB>;
  using V = typename EL::V;
  constexpr int kN = EL::kN;
  pdl_wait_and_release();
  const int64_t t = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> p.log_group;
  const int lane = threadIdx.x & (p.group - 1);
  const int v1 = min(p.nvec, (int)(blockIdx.y + 1) * p.part);
  if (t >= p.T) return;
  const Span span = span_of(p.src, p.P, p.src_stride, p.bytes);
  const Span bspan = span_of(p.base, p.T, p.bytes, p.bytes);
  char* out = p.dst + t * p.bytes;
  const char* src[kRowSlots];
  float w[kRowSlots];
  unsigned on = 0;  // which of these slots have an expert
  auto slots = [&](int j0) {
    on = 0;
#pragma unroll
    for (int a = 0; a < kRowSlots; ++a) {
      const int r = j0 + a < p.k ? __ldg(p.inverse + t * p.k + j0 + a) : -1;
      const bool has = (unsigned)r < (unsigned)p.P;
      on |= (unsigned)has << a;
      src[a] = p.src + (has ? r : 0) * p.src_stride;
      w[a] = has && p.weights ? __ldg(p.weights + t * p.k + j0 + a) : 1.f;
    }
  };
  slots(0);
  for (int v = blockIdx.y * p.part + lane; v < v1; v += p.group) {
    const int64_t at = first_of<VB>(out, v);
    if (VB == 0 && at >= p.bytes) break;
    float acc[kN];
    if (p.base) {
      EL::load(load_vec<VB>(p.base + t * p.bytes, v, at, bspan), acc);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) acc[i] = 0.f;
    }
    for (int j0 = 0; j0 < p.k; j0 += kRowSlots) {
      if (p.k > kRowSlots) slots(j0);
      V y[kRowSlots];
#pragma unroll
      for (int a = 0; a < kRowSlots; ++a)
        if (on >> a & 1) y[a] = load_vec<VB>(src[a], v, at, span);
#pragma unroll
      for (int a = 0; a < kRowSlots; ++a) {
        if (!(on >> a & 1)) continue;
        float f[kN];
        EL::load(y[a], f);
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[i] = fmaf(w[a], f[i], acc[i]);
      }
    }
    store_vec<VB>(out, v, at, p.bytes, EL::store(acc));
  }
}

// A group of threads per (token, kJ slots): dout[t] and the slots' ys rows
// pass once; dys rows are written from the same registers, and dw is a sum
// over the group (lanes by shuffles, warps through shared memory: always the
// same order). Bound by the traffic of ys and dys: 161 us at 4096 x 8 rows of
// 7168 bf16, 0.94 of the copy rate.
template <int DT, int VB, int kJ>
__global__ void __launch_bounds__(kRowThreads) combine_bwd_kernel(const RowParams p) {
  using EL = Elems<DT, VB>;
  using V = typename EL::V;
  constexpr int ES = EL::kSize, kN = EL::kN, kWarps = kRowThreads / 32;
  __shared__ float part[kWarps][kJ];
  pdl_wait_and_release();
  const int64_t t = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> p.log_group;
  const int lane = threadIdx.x & (p.group - 1);
  const bool here = t < p.T;
  const int j0 = blockIdx.y * kJ;
  int row[kJ];
  float w[kJ], dot[kJ];
#pragma unroll
  for (int a = 0; a < kJ; ++a) {
    const bool in = here && j0 + a < p.k;
    const int r = in ? __ldg(p.inverse + t * p.k + j0 + a) : -1;
    row[a] = (unsigned)r < (unsigned)p.P ? r : -1;
    w[a] = in ? __ldg(p.weights + t * p.k + j0 + a) : 0.f;
    dot[a] = 0.f;
  }
  const char* g = p.dout + t * p.dout_stride;
  const Span gspan = span_of(p.dout, p.T, p.dout_stride, p.bytes);
  const Span span = span_of(p.src, p.P, p.src_stride, p.bytes);
  for (int v = here ? lane : p.nvec; v < p.nvec; v += p.group) {
    V y[kJ], gv;
    if constexpr (VB != 0) {
      gv = load_vec<VB>(g, v, 0, gspan);
#pragma unroll
      for (int a = 0; a < kJ; ++a)
        if (row[a] >= 0) y[a] = load_vec<VB>(p.src + (int64_t)row[a] * p.src_stride, v, 0, span);
    }
    float gf[kN];
    if constexpr (VB != 0) EL::load(gv, gf);
#pragma unroll
    for (int a = 0; a < kJ; ++a) {
      if (row[a] < 0) continue;
      char* dst = p.dst + (int64_t)row[a] * p.bytes;
      const int64_t at = first_of<VB>(dst, v);
      if constexpr (VB == 0) {
        if (at >= p.bytes) continue;
        y[a] = load_any(p.src + (int64_t)row[a] * p.src_stride + at, span);
        EL::load(load_any(g + at, gspan), gf);
      }
      float f[kN], d[kN];
      EL::load(y[a], f);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        if (VB != 0 || (at + ES * i >= 0 && at + ES * i < p.bytes))
          dot[a] = fmaf(gf[i], f[i], dot[a]);
        d[i] = w[a] * gf[i];
      }
      store_vec<VB>(dst, v, at, p.bytes, EL::store(d));
    }
  }
#pragma unroll
  for (int a = 0; a < kJ; ++a)
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, dot[a], d);
      if (d < p.group) dot[a] += o;
    }
  if (p.group > 32) {
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int a = 0; a < kJ; ++a) part[threadIdx.x >> 5][a] = dot[a];
    __syncthreads();
  }
  // thread a of the group (of 8 at least) has slot a
  if (lane < kJ && here && j0 + lane < p.k) {
    float s = dot[0];
#pragma unroll
    for (int a = 1; a < kJ; ++a) s = lane == a ? dot[a] : s;
    for (int i = 1; i < p.group / 32; ++i) s += part[(threadIdx.x >> 5) + i][lane];
    p.dw[t * p.k + j0 + lane] = s;
  }
  zero_dropped_rows<VB>(p);
}

// ---------------------------------------------------------------- host

int elem_bytes(mr_dtype d) { return d == MR_DTYPE_F32 ? 4 : 2; }

// Widest vector that divides every address, stride and row; 0: none of 4 bytes.
int vec_bytes(std::initializer_list<uint64_t> all) {
  uint64_t m = 16;
  for (uint64_t a : all) m |= a;
  return (m & 15) == 0 ? 16 : (m & 7) == 0 ? 8 : (m & 3) == 0 ? 4 : 0;
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
  if ((addr(s->order) | addr(s->inverse) | addr(s->offsets)) % 4)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                "order, inverse and offsets must be aligned to their type");
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

RowParams row_params(const mr_sorted* s, int64_t bytes, int vb) {
  RowParams p{};
  p.inverse = s->inverse;
  p.offsets = s->offsets;
  p.T = s->tokens;
  p.k = s->top_k;
  p.P = p.T * p.k;
  p.E = s->experts;
  p.bytes = bytes;
  p.nvec = (int)(vb ? bytes / vb : (bytes + 15) / 16 + 1);
  p.group = 8;  // rows of few vectors share a CTA
  p.log_group = 3;
  while (p.group < kRowThreads && p.group < p.nvec) {
    p.group *= 2;
    ++p.log_group;
  }
  p.part = p.nvec;
  return p;
}

// A batch too small to fill the GPU spreads each row over several CTAs.
dim3 row_grid(const mr_ctx* ctx, RowParams& p) {
  const int g = p.group;
  const int64_t ctas = (p.T + kRowThreads / g - 1) / (kRowThreads / g);
  const int64_t parts =
      std::min<int64_t>((p.nvec + g - 1) / g, (2 * ctx->sm_count + ctas - 1) / ctas);
  p.part = (int)(((p.nvec + parts - 1) / parts + g - 1) / g * g);
  return dim3((unsigned)ctas, (unsigned)((p.nvec + p.part - 1) / p.part));
}

template <int DT>
cudaError_t launch_combine(const RowParams& p, int vb, dim3 grid, cudaStream_t s) {
  switch (vb) {
    case 16: return launch_pdl(combine_rows_kernel<DT, 16>, grid, kRowThreads, 0, s, p);
    case 8: return launch_pdl(combine_rows_kernel<DT, 8>, grid, kRowThreads, 0, s, p);
    case 4: return launch_pdl(combine_rows_kernel<DT, 4>, grid, kRowThreads, 0, s, p);
    default:
      if constexpr (DT != MR_DTYPE_F32)
        return launch_pdl(combine_rows_kernel<DT, 0>, grid, kRowThreads, 0, s, p);
      return cudaErrorMisalignedAddress;  // f32 buffers are 4-byte aligned
  }
}

mr_status combine_rows(mr_ctx* ctx, const void* ys, mr_dtype dt, int64_t stride, int64_t hidden,
                       const float* weights, const void* base, const mr_sorted* s, void* out,
                       void* stream, const char* what) {
  const int es = elem_bytes(dt);
  const int vb = vec_bytes(
      {addr(ys), addr(out), addr(base), (uint64_t)(stride * es), (uint64_t)(hidden * es)});
  RowParams p = row_params(s, hidden * es, vb);
  p.src = static_cast<const char*>(ys);
  p.src_stride = stride * es;
  p.dst = static_cast<char*>(out);
  p.base = static_cast<const char*>(base);
  p.weights = weights;
  const dim3 grid = row_grid(ctx, p);
  cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  const DeviceScope on(ctx);
  cudaError_t e = on.err;
  if (e == cudaSuccess)
    e = dt == MR_DTYPE_BF16  ? launch_combine<MR_DTYPE_BF16>(p, vb, grid, cs)
        : dt == MR_DTYPE_F16 ? launch_combine<MR_DTYPE_F16>(p, vb, grid, cs)
                             : launch_combine<MR_DTYPE_F32>(p, vb, grid, cs);
  return cuda_check(ctx, e, what);
}

template <int DT, int VB>
cudaError_t launch_bwd(const RowParams& p, int jn, cudaStream_t s) {
  const int per = kRowThreads / p.group;
  const dim3 grid((unsigned)((p.T + per - 1) / per), (unsigned)((p.k + jn - 1) / jn));
  switch (jn) {
    case 8: return launch_pdl(combine_bwd_kernel<DT, VB, 8>, grid, kRowThreads, 0, s, p);
    case 4: return launch_pdl(combine_bwd_kernel<DT, VB, 4>, grid, kRowThreads, 0, s, p);
    case 2: return launch_pdl(combine_bwd_kernel<DT, VB, 2>, grid, kRowThreads, 0, s, p);
    default: return launch_pdl(combine_bwd_kernel<DT, VB, 1>, grid, kRowThreads, 0, s, p);
  }
}
template <int DT>
cudaError_t launch_bwd_of(const RowParams& p, int vb, int jn, cudaStream_t s) {
  switch (vb) {
    case 16: return launch_bwd<DT, 16>(p, jn, s);
    case 8: return launch_bwd<DT, 8>(p, jn, s);
    case 4: return launch_bwd<DT, 4>(p, jn, s);
    default:
      if constexpr (DT != MR_DTYPE_F32) return launch_bwd<DT, 0>(p, jn, s);
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
    if (addr(ids) % 4)
      return fail(ctx, MR_ERR_INVALID_ARGUMENT, "ids must be aligned to their type");
    if (experts > kMaxExperts)
      return fail(ctx, MR_ERR_UNSUPPORTED, "expert counts above 1024 are not built here");
    SortParams p{ids, tokens * top_k, experts, 0, 0, order, inverse, offsets, ctx->d_error};
    while ((1 << p.bits) <= experts) ++p.bits;
    const int ctas = p.P <= kSortOneCta ? 1 : kSortCluster;
    const int64_t want = std::max<int64_t>((p.P + 31) / 32, (experts + 31) / 32);
    const int warps = ctas > 1 ? kSortThreads / 32
                               : (int)std::min<int64_t>(kSortThreads / 32, std::max<int64_t>(want, 1));
    const int64_t per = (p.P + (int64_t)ctas * warps - 1) / ((int64_t)ctas * warps);
    p.chunk = (per + 31) / 32 * 32;
    const size_t smem = sizeof(int) * ((size_t)warps * experts + 2 * experts + 32);
    const DeviceScope on(ctx);
    cudaError_t e = on.err;
    if (e == cudaSuccess)
      e = attrs_once(ctx, kAttrSort, [] {
        const cudaError_t a = cudaFuncSetAttribute(
            sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem);
        return a != cudaSuccess ? a
                                : cudaFuncSetAttribute(
                                      sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      });
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
    const int vb =
        vec_bytes({addr(x), addr(xs), (uint64_t)(x_stride * es), (uint64_t)(hidden * es)});
    RowParams p = row_params(plan, hidden * es, vb);
    p.src = static_cast<const char*>(x);
    p.src_stride = x_stride * es;
    p.dst = static_cast<char*>(xs);
    const dim3 grid = row_grid(ctx, p);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const DeviceScope on(ctx);
    cudaError_t e = on.err;
    if (e == cudaSuccess)
      e = vb == 16  ? launch_pdl(dispatch_kernel<16>, grid, kRowThreads, 0, s, p)
          : vb == 8 ? launch_pdl(dispatch_kernel<8>, grid, kRowThreads, 0, s, p)
          : vb == 4 ? launch_pdl(dispatch_kernel<4>, grid, kRowThreads, 0, s, p)
                    : launch_pdl(dispatch_kernel<0>, grid, kRowThreads, 0, s, p);
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
    if (addr(weights) % 4)
      return fail(ctx, MR_ERR_INVALID_ARGUMENT, "weights must be aligned to their type");
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
    if ((addr(weights) | addr(dweights)) % 4)
      return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                  "weights and dweights must be aligned to their type");
    const int es = elem_bytes(dtype);
    const int vb = vec_bytes({addr(dout), addr(ys), addr(dys), (uint64_t)(dout_stride * es),
                              (uint64_t)(ys_stride * es), (uint64_t)(hidden * es)});
    RowParams p = row_params(plan, hidden * es, vb);
    p.dout = static_cast<const char*>(dout);
    p.dout_stride = dout_stride * es;
    p.src = static_cast<const char*>(ys);
    p.src_stride = ys_stride * es;
    p.weights = weights;
    p.dst = static_cast<char*>(dys);
    p.dw = dweights;
    int jn = 1;  // slots a group: all of them once the tokens alone fill the GPU
    while (jn < 8 && jn < p.k &&
           p.T * p.group / kRowThreads * ((p.k + 2 * jn - 1) / (2 * jn)) >= 4 * ctx->sm_count)
      jn *= 2;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const DeviceScope on(ctx);
    cudaError_t e = on.err;
    if (e == cudaSuccess)
      e = dtype == MR_DTYPE_BF16  ? launch_bwd_of<MR_DTYPE_BF16>(p, vb, jn, s)
          : dtype == MR_DTYPE_F16 ? launch_bwd_of<MR_DTYPE_F16>(p, vb, jn, s)
                                  : launch_bwd_of<MR_DTYPE_F32>(p, vb, jn, s);
    return cuda_check(ctx, e, "combine backward");
  });
}

}  // extern "C"
