// mr_mxmm.cuh — MXFP4 x MXFP4 products on the 5th-generation tensor cores'
// block-scaled 4-bit form, one matrix or an expert stack over sorted rows.
//
//   out[r, o] = sum_b 2^(ea[r, b] + ew[o, b] - 254) * sum_{i in b} a[r, i] * w[o, i]
//
// over blocks b of 32 elements; tcgen05.mma kind::mxf4 multiplies e2m1 codes
// and both e8m0 scales exactly and sums in fp32. A tile is 128 weight rows
// a CTA (the M side, one TMEM lane each) by up to `ntile` activation rows
// (the N side, one TMEM column each): weight matrices are whole multiples of
// 128 rows while an expert's rows are any number, and N steps by 16.
//
// CG = 1: one CTA a tile. CG = 2: a cluster of two CTAs a tile of 256 weight
// rows; each loads its own 128 rows and half of the activations, and the
// leader's MMAs (cta_group::2) read both halves: per stage of 176 rows a CTA
// takes 54 KB of codes from L2 instead of 76. At 64 bytes a cycle from L2 to an
// SM a stage of n rows is 512 + 2n cycles of loads (512 + 4n without the pair)
// against 4n of MMAs.
//
// Measured, out bf16: 4096 x 16384 x 7168 200 to 209 us (4.6 to 4.8 PFLOP/s; 230
// in a loop of two seconds, at 1.2 GHz under the power cap); 64 tokens x 8 of 256
// experts of 2048 x 7168 252 us (the weights at 6.9 TB/s). 2048 tokens x 8 of 32
// experts 118 us sorted and 134 by token, tiles of 148 rows: a stage takes 0.70
// and 0.80 us, 1110 and 1470 cycles at the clocks of a loop of two seconds, where
// the loads need 808 and the MMAs 592. Neither is the bound (1024 tokens: tensor
// pipe active 41 % of the time, L2 38 %); most likely the three or four slots of
// the ring do not cover the loads' latency, 1200-1900 cycles.
// One token x 8 of 256 14.3 us (floor 9.5): the first copy starts 2.8 us after
// the kernel does (the table 1.3, the rest the fetch of each role's code), the
// last tile's result leaves 1.1 us after its codes are there, and between the
// two HBM runs at 0.99. One row x 2048 x 7168 7.4 us, 6.5 with the weights in
// L2. (Tried for the start, each within 1 % or slower: the first weights'
// copies right behind the table, 10.2 -> 11.1 us at 64 experts of 1024 x 4096;
// the table's code run once on nothing before the wait for the kernels ahead;
// one tile lookup that every role calls.)
//
// Where there are few narrow tiles (CG = 1), a cluster of `ksplit` CTAs shares each:
// every CTA multiplies its part of the row's stages and leaves the partial
// result in its shared memory, and each then sums a share of the columns over
// the cluster, always in the order of the parts.
//
// Persistent CTAs (or pairs) loop over tiles (expert's row tile x weight
// rows, the weight rows fastest, so that CTAs working side by side share
// activations). Per stage of 512 elements (256 bytes of codes a row, as two
// pieces of the 128 that the swizzle spans):
//   - warp 0: TMA loads of the codes (128-byte swizzle) into the ring;
//   - warps 12-15, by_token: the activations' codes instead, by TMA gathers of
//     four rows (58 cycles each to issue: more than one warp can in a stage);
//   - warps 2 and 3: the exponents of weights / activations, 16 a row, from
//     global to shared memory;
//   - warps 8-11: the exponents from there into tensor memory, each warp its
//     lane quadrant (the tensor core reads the exponents of 32 rows a column,
//     in every quadrant). No proxy fence is on this way: one in the loading
//     warps waited for the loads of the next exponents too (1000 cycles a
//     stage), and copies by the tensor core (tcgen05.cp) cost the MMA warp
//     more issue time than the MMAs;
//   - warp 1: one MMA per 64 elements. Its lane, like those that issue TMA,
//     is chosen by elect.sync: from a branch on the lane's number each such
//     instruction cost 90-110 cycles (its operands live in uniform
//     registers), so 30-40; the other lanes leave;
//   - warps 4-7: a finished tile's accumulator to global memory while the
//     next tile's MMAs run (two accumulators).
// Every ring slot has exponents' columns of its own in TMEM, so they are only
// overwritten once the MMAs that read them are complete.
// Tensor-memory loads, stores and (de)allocation are warp-aligned: each is
// preceded by __syncwarp wherever the lanes may have parted (waits, stores of
// a row's last weight rows).
// Every wait is bounded: on expiry the kernel flags MR_DEVERR_TIMEOUT and
// runs to its end on garbage, drains its copies and MMAs, frees its TMEM. No
// CTA of a cluster leaves before every thread of the others is done with its
// memory (leave_cluster), also where one of them gave up a wait early.
#pragma once

#include <cooperative_groups.h>

#include "mr_gemv_umma.cuh"

namespace mr {

constexpr int kMmRows = 128;     // weight rows of a CTA (MMA M = 128 CG)
constexpr int kMmK = 512;        // elements of a stage: with 256 the waits of one, 50-200
                                 // cycles each, took longer than its MMAs
constexpr int kMmMaxN = 176;     // activation rows of a tile: two accumulators and three
                                 // slots of exponents fit the 512 TMEM columns
// Widest tile of a form, and its rows in groups of 32. (Code is fetched once a
// kernel: a form without the other's unrolled rows starts 1-2 us earlier.)
MR_DEVICE __host__ constexpr int mm_max_n(int cg) { return cg == 1 ? 64 : kMmMaxN; }
MR_DEVICE __host__ constexpr int mm_max_b(int cg) { return (mm_max_n(cg) + 31) / 32; }
constexpr int kMmThreads = 384;  // plus the gather warps
constexpr int kMmGatherWarps = 4;  // sixteen warps in all: more would leave 96 registers each
constexpr int kMmAPiece = kMmRows * 128;
constexpr int kMmSplit = 4;  // CTAs that share a tile's stages, at most
constexpr int kMmRaw = 3;  // slots of the exponents' ring in shared memory

// The MMAs' N, and a tile's width, step by 16.
MR_DEVICE __host__ constexpr int mm_round(int n) { return (n + 15) & ~15; }
// TMEM columns of a word (four exponents a row) of B, and of a stage.
MR_DEVICE __host__ constexpr int mm_sf_word(int ntile) { return 4 * ((ntile + 127) / 128); }
MR_DEVICE __host__ constexpr int mm_sf_cols(int ntile) { return 16 + 4 * mm_sf_word(ntile); }
// Rows of exponents of one slot in shared memory.
MR_DEVICE __host__ constexpr int mm_raw_rows(int ntile) { return kMmRows + (ntile + 31) / 32 * 32; }

struct MmParams {
  const uint8_t* w_scales;  // [E, out, in / 32]
  const uint8_t* a_scales;  // [arows, in / 32]
  const int32_t* offsets;   // [E + 1], or NULL: one matrix over all rows
  const int32_t* order;     // by_token: the pair at each sorted row, else NULL
  void* out;                // [rows, out]
  unsigned* error;
  int64_t rows, arows, out_features;
  int E;
  uint32_t k_mul, k_shift;  // pair / top_k, see mm_act_row
  int groups;           // in / 32
  int nstages, mtiles;
  int ntile, box, nst;  // tile width, rows of an activation box, ring stages
  int ksplit;           // CTAs that share a tile's stages
  int part_at;          // where the partial result lies in shared memory
  int out_f32;
};
struct MmMaps {
  CUtensorMap w, a;
};

// Shared memory: ring of codes, ring of exponents, barriers, group table.
inline int mm_stage_bytes(int ntile, int cg) { return 2 * (kMmAPiece + ntile / cg * 128); }
inline int mm_fixed_bytes(int E, int ntile, int ksplit) {
  return 1024 + kMmRaw * mm_raw_rows(ntile) * 16 + 768 + 2 * (E + 1) * 4 +
         (ksplit > 1 ? ntile * kMmRows * 4 : 0);
}

// ------------------------------------------------------------ instructions

// True in one lane of a converged warp.
MR_DEVICE bool elect_one() {
  uint32_t on;
  asm volatile("{ .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p; }"
               : "=r"(on));
  return on != 0;
}
MR_DEVICE uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
template <int CG>
MR_DEVICE void mm_tmem_alloc(uint32_t* dst) {
  if constexpr (CG == 1) {
    tmem_alloc(dst, 512);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(dst))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
MR_DEVICE void mm_tmem_dealloc() {
  if constexpr (CG == 1)
    tmem_dealloc(0, 512);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(0u) : "memory");
}
// Arrive on `bar` (of both CTAs of a pair) when this thread's MMAs are done.
template <int CG>
MR_DEVICE void mm_commit(uint64_t* bar) {
  if constexpr (CG == 1)
    tc_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// D[128 CG x N] (+)= A . B^T with scales; both operands by shared descriptors.
template <int CG>
MR_DEVICE void tc_mma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                           uint32_t sfa, uint32_t sfb, uint32_t acc) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], "
        "[%5], p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], "
        "[%5], p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
}
// kind::mxf4, e2m1 x e2m1, e8m0 scales, M = 128 CG; `half`: which two of a
// word's four exponents (both operands).
template <int CG>
MR_DEVICE uint32_t umma_idesc_mxf4(int n, uint32_t half) {
  return (half << 5)                   // B exponents: id 0 or 2 at bits 4-5
         | (1u << 7) | (1u << 10)      // A, B: e2m1
         | ((uint32_t)(n >> 3) << 17)  // N / 8
         | (1u << 23)                  // exponents: e8m0
         | ((uint32_t)CG << 27)        // M / 128
         | (half << 30);               // A exponents: id at bits 29-30
}
// Sixteen consecutive TMEM columns of this thread's lane.
MR_DEVICE void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
MR_DEVICE uint32_t word_of(const uint4& x, int w) {
  return w == 0 ? x.x : w == 1 ? x.y : w == 2 ? x.z : x.w;
}
// A look at a barrier that never blocks, to be made ahead of the wait.
MR_DEVICE bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Four rows (y) of 128 bytes at column x.
MR_DEVICE void tma_gather4(void* dst, const CUtensorMap* map, int x, const int4& y,
                           uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w),
      "r"(smem_u32(bar))
      : "memory");
}
// Arrive on the barrier at this place in the CTA of rank `to`. Relaxed: what
// it tells of is complete by itself (tensor memory after tcgen05.wait, copies
// after their barrier, MMAs after their commit) and no plain store is handed
// over; a release at cluster scope took 500-2000 cycles.
template <int CG>
MR_DEVICE void mm_arrive(uint64_t* bar, uint32_t to, uint32_t rank) {
  if (CG == 1 || to == rank) {
    mbar_arrive(bar);
  } else {
    asm volatile(
        "{ .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, %1;\n"
        "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [r]; }" ::"r"(smem_u32(bar)),
        "r"(to)
        : "memory");
  }
}
// Partial sums: made visible to the cluster, and read from another CTA.
MR_DEVICE void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
MR_DEVICE uint32_t at_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
MR_DEVICE float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// Arrive (relaxed: after fence_cluster) on this barrier of every CTA.
MR_DEVICE void arrive_all(uint64_t* bar, int ctas) {
  for (int c = 0; c < ctas; ++c)
    asm volatile(
        "{ .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, %1;\n"
        "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [r]; }" ::"r"(smem_u32(bar)),
        "r"(c)
        : "memory");
}

// The last thing a thread of a cluster of CTAs does: what it did to another
// CTA's memory is done, and it waits for all threads of the cluster that have
// not ended to say the same. (The CTAs' own barriers cannot serve for this: a
// CTA whose wait expired leaves its further waits early.) At least one lane of
// every warp has to come here, and the lanes that do together (__syncwarp in
// the roles of whole warps): with whole warps gone for good the barrier did not
// complete. It has no limit of its own: every wait before it is bounded, so all
// come here. It costs a pair of CTAs 0.3 to 0.6 us of a call (77 x 2048 x
// 7168), a split tile's CTAs nothing.
MR_DEVICE void leave_cluster() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// wait_bounded as one look at the barrier and a call where that is not
// enough: sixteen warps run different code, and its size costs each of them.
// One lane of a warp waits alone only where the others have left; elsewhere
// all lanes wait together. (Lanes parked at a warp barrier made every branch
// of the running one slow: 185-280 cycles for a wait that is already over,
// against 53.)
__device__ __noinline__ void wait_called(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                         unsigned* error) {
  wait_bounded(bar, parity, abort_flag, error);
}
MR_DEVICE void wait_mbar(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                         unsigned* error, bool seen) {
  if (__builtin_expect(!seen, 0)) wait_called(bar, parity, abort_flag, error);
}
MR_DEVICE void wait_mbar(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                         unsigned* error) {
  if (__builtin_expect(!mbar_try_wait(bar, parity), 0)) wait_called(bar, parity, abort_flag, error);
}

MR_DEVICE void put(float* p, float v) { *p = v; }
MR_DEVICE void put(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }
// One result of each of 16 rows (`left` of which exist), `pitch` apart. The
// whole chunk has no branch between its stores: with one for each row the
// epilogue took 36 cycles a row, longer than the MMAs of a narrow matrix.
template <typename T>
MR_DEVICE void store16(T* p, int64_t pitch, int left, const float (&v)[16]) {
  if (left >= 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) put(p + i * pitch, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left) put(p + i * pitch, v[i]);
  }
}

// ------------------------------------------------------------------- tiles

// An expert's n rows in tiles of equal width: as few as ntile allows, none
// empty.
MR_DEVICE int mm_width(int n, int ntile) {
  if (n <= ntile) return max(mm_round(n), 16);
  const uint32_t c = (uint32_t)(n + ntile - 1) / (uint32_t)ntile;
  return mm_round((int)((uint32_t)(n + c - 1) / c));
}
MR_DEVICE int mm_tiles(int n, int ntile) {
  if (n <= ntile) return n > 0;
  const uint32_t w = mm_width(n, ntile);
  return (int)((uint32_t)(n + w - 1) / w);
}

// Gathers of four rows that a CTA's half of a tile of n rows takes. The rest of
// the half keeps what shared memory holds: those columns' results are not
// kept. (Gathered as repeats of the last row, which 128 CTAs then read at
// once, they made a single token's product 2 us slower; rows outside the
// tensor, which read as zeros, a prefill 6 % slower.)
MR_DEVICE int mm_quads(int n, int half, int rank) {
  return (min(max(n - rank * half, 0), half) + 3) / 4;
}

// Walks the CTA's (or pair's) tiles in order: item -> expert, rows, and the
// CTA's weight rows.
template <int CG>
struct MmWalk {
  const int* goff;   // [E + 1] first row of each expert
  const int* gtile;  // [E + 1] first row tile of each expert
  int E, mtiles, ntile;
  int m_in;          // the CTA's first row in a tile
  int e;             // the first tile's expert, then the last one's
  int row0, n, m0;
  MR_DEVICE void at(int item) {
    const int t = (int)((uint32_t)item / (uint32_t)mtiles);
    m0 = (item - t * mtiles) * (kMmRows * CG) + m_in;
    if (gtile[e + 1] <= t) {
      int hi = E;  // gtile[e] <= t < gtile[hi]
      while (hi - e > 1) {
        const int mid = (e + hi) >> 1;
        if (gtile[mid] <= t)
          e = mid;
        else
          hi = mid;
      }
    }
    const int all = goff[e + 1] - goff[e];
    const int w = mm_width(all, ntile);
    const int first = (t - gtile[e]) * w;
    row0 = goff[e] + first;
    n = min(w, all - first);
  }
};

// ------------------------------------------------------------ exponents

// The row of `a` that sorted row r takes its activations from.
MR_DEVICE int64_t mm_act_row(const MmParams& p, int64_t r) {
  if (p.order) {
    // pair / top_k for pair < 2^31: k_mul = ceil(2^(31 + k_shift) / top_k) with
    // 2^k_shift >= top_k
    const int pair = max(__ldg(p.order + r), 0);
    r = (int64_t)(((uint64_t)(uint32_t)pair * p.k_mul) >> (31 + p.k_shift));
  }
  return min(r, p.arows - 1);
}

// 16 bytes at an aligned address, of which only [lo, hi) may be read.
MR_DEVICE uint4 mm_ldg16(const uint8_t* at, const uint8_t* lo, const uint8_t* hi) {
  if (at >= lo && at + 16 <= hi) return __ldg(reinterpret_cast<const uint4*>(at));
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 16; ++i)
    if (at + i >= lo && at + i < hi) w[i >> 2] |= (uint32_t)__ldg(at + i) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One warp's exponents: rows lane + 32 i (i < NB) of a tile's weights or
// activations, 16 a row (a stage's). WIDE: every row is made of
// aligned 16-byte pieces. Otherwise a row starts at any byte and 16 exponents
// lie in one or two aligned pieces, shifted together when they are used.
template <int NB, bool WIDE>
struct MmScaleRegs {
  uint4 a[NB], b[WIDE ? 1 : NB];
  uint32_t off[WIDE ? 1 : NB];  // first byte in the pieces
  int left;                     // exponents from here to the row's end

  MR_DEVICE void load(const uint8_t* const (&src)[NB], int q, int groups, const uint8_t* lo,
                      const uint8_t* hi) {
    left = groups - 16 * q;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (!src[i]) continue;
      const uint8_t* at = src[i] + 16 * q;
      if constexpr (WIDE) {
        a[i] = __ldg(reinterpret_cast<const uint4*>(at));
      } else {
        off[i] = (uint32_t)reinterpret_cast<uintptr_t>(at) & 15;
        at -= off[i];
        a[i] = mm_ldg16(at, lo, hi);
        if (off[i] && at + 16 < hi) b[i] = mm_ldg16(at + 16, lo, hi);
      }
    }
  }
  // row i's exponents; those past the row's end become 127: their codes are
  // zero, but another row's NaN must not come in
  MR_DEVICE uint4 get(int i) const {
    if constexpr (WIDE) return a[i];
    uint32_t w[8] = {a[i].x, a[i].y, a[i].z, a[i].w, b[i].x, b[i].y, b[i].z, b[i].w};
    const uint32_t o = off[i];
    if (o) {
#pragma unroll
      for (int k = 0; k < 6; ++k) w[k] = (o & 8) ? w[k + 2] : w[k];
#pragma unroll
      for (int k = 0; k < 5; ++k) w[k] = (o & 4) ? w[k + 1] : w[k];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 8 * (o & 3));
    }
    if (left < 16) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = left - 4 * k;  // bytes of this word in the row
        const uint32_t keep = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        w[k] = (w[k] & keep) | (0x7F7F7F7Fu & ~keep);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Exponents from global to shared memory, loaded one to four stages (also of
// the next tile) ahead of their use: the loads' latency stays out of the
// pipeline. A slot holds 16 bytes a row. Every lane of the warp.
template <int NB, bool WIDE, bool IS_A, int CG>
MR_DEVICE void mm_load_scales(const MmParams& p, const MmWalk<CG>& walk, int lane, int first,
                              int stride, int n_items, int st0, int st1, uint4* raw,
                              uint64_t* rfull, uint64_t* rempty, volatile int* flags) {
  const int slot_rows = mm_raw_rows(p.ntile);
  const uint8_t* lo = IS_A ? p.w_scales : p.a_scales;
  const uint8_t* hi = lo + (IS_A ? (int64_t)p.E * p.out_features : p.arows) * p.groups;
  MmWalk<CG> it = walk;
  const uint8_t* src[NB];
  auto open = [&](int item) {
    if (item >= n_items) return;
    it.at(item);
    const int have = IS_A ? kMmRows : it.n;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      src[i] = nullptr;
      if (32 * i >= have) continue;
      // rows past the tile's end repeat its last: their results are not kept
      const int r = min(lane + 32 * i, have - 1);
      const int64_t row =
          IS_A ? (int64_t)it.e * p.out_features + min((int64_t)it.m0 + r, p.out_features - 1)
               : mm_act_row(p, (int64_t)it.row0 + r);
      src[i] = lo + row * p.groups;
    }
  };
  // Narrow tiles are few stages of HBM's latency long: four ahead against two is
  // 15.3 -> 14.7 us for a token's 8 experts of 2048 x 7168. Wide ones load from
  // L2 and lose 1 % by it. Registers of two unaligned stages would spill.
  constexpr int kAhead = !WIDE ? 1 : CG == 1 ? 4 : 2;
  MmScaleRegs<NB, WIDE> v[kAhead];
#pragma unroll
  for (int b = 0; b < kAhead; ++b)
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      v[b].a[i] = make_uint4(0, 0, 0, 0);
      if constexpr (!WIDE) {
        v[b].b[i] = make_uint4(0, 0, 0, 0);
        v[b].off[i] = 0;
      }
    }
  int litem = first, lq = st0;  // the stage to load next
  open(litem);
  auto load = [&](MmScaleRegs<NB, WIDE>& r) {
    if (litem >= n_items) return;
    r.load(src, lq, p.groups, lo, hi);
    if (++lq == st1) {
      lq = st0;
      litem += stride;
      open(litem);
    }
  };
#pragma unroll
  for (int b = 0; b < kAhead; ++b) load(v[b]);
  uint32_t slot = 0, phase = 0;
  int item = first, q = st0;  // the stage to hand on next
  while (item < n_items) {
#pragma unroll
    for (int b = 0; b < kAhead; ++b) {
      if (item >= n_items) break;
      wait_mbar(rempty + slot, phase ^ 1u, flags, p.error);
      uint4* dst = raw + slot * slot_rows + (IS_A ? 0 : kMmRows) + lane;
#pragma unroll
      for (int i = 0; i < NB; ++i)
        if (IS_A || 32 * i < p.ntile) dst[32 * i] = v[b].get(i);
      __syncwarp();
      if (lane == 0) mbar_arrive(rfull + slot);
      if (++slot == kMmRaw) {
        slot = 0;
        phase ^= 1u;
      }
      load(v[b]);
      if (++q == st1) {
        q = st0;
        item += stride;
      }
    }
  }
}

template <bool WIDE, int CG>
__global__ void __launch_bounds__(kMmThreads + 32 * kMmGatherWarps, 1)
    mxmm_kernel(const MmParams p, const __grid_constant__ MmMaps maps) {
  extern __shared__ char smem_raw[];
  char* smem =
      reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int b_piece = p.ntile / CG * 128;
  const int nst = p.nst;
  char* bring = smem + nst * 2 * kMmAPiece;
  uint4* raw = reinterpret_cast<uint4*>(bring + nst * 2 * b_piece);  // [kMmRaw][raw rows]
  uint64_t* lfull = reinterpret_cast<uint64_t*>(raw + kMmRaw * mm_raw_rows(p.ntile));  // [nst]
  uint64_t* full = lfull + nst;       // [nst] a stage's operands there, of both CTAs
  uint64_t* empty = full + nst;       // [nst]
  uint64_t* rfull = empty + nst;      // [kMmRaw] exponents in shared memory
  uint64_t* rempty = rfull + kMmRaw;  // [kMmRaw] and read from there
  uint64_t* dfull = rempty + kMmRaw;  // [2]
  uint64_t* dempty = dfull + 2;       // [2]
  uint64_t* drain = dempty + 2;       // every MMA complete
  uint64_t* done = drain + 1;         // every other access of TMEM too
  uint64_t* pfull = done + 1;         // every CTA's partial result is there (ksplit > 1)
  uint64_t* pempty = pfull + 1;       // this CTA's has been read by all
  uint32_t* tslot = reinterpret_cast<uint32_t*>(pempty + 1);
  volatile int* flags = reinterpret_cast<volatile int*>(tslot + 1);
  int* scan = reinterpret_cast<int*>(tslot + 2);  // [18] warp sums, [31] first tile's expert
  int* goff = scan + 32;
  int* gtile = goff + p.E + 1;
  // [ntile][128] this CTA's partial result, 16-byte aligned: after the ring
  float* part = reinterpret_cast<float*>(smem + p.part_at);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = CG == 1 ? 0 : cluster_rank();
  const int ks = CG == 1 ? p.ksplit : 1;
  const int kpart = ks > 1 ? (int)cluster_rank() : 0;
  const int st0 = p.nstages * kpart / ks, st1 = p.nstages * (kpart + 1) / ks;
  const int first = blockIdx.x / (CG * ks), stride = gridDim.x / (CG * ks);
  // the leader's copies complete on `full` itself, the other CTA's on a
  // barrier of its own, whose arrival is passed on
  uint64_t* cfull = rank == 0 ? full : lfull;
  if (tid == 0) {
    for (int s = 0; s < nst; ++s) {
      mbar_init(lfull + s, 1);
      mbar_init(full + s, 5 * CG);  // a CTA's copies and four warps' exponents
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < kMmRaw; ++s) {
      mbar_init(rfull + s, 2);
      mbar_init(rempty + s, 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(dfull + b, 1);
      mbar_init(dempty + b, 4 * CG);
    }
    mbar_init(drain, 1);
    mbar_init(done, rank == 0 ? 8 : 9);
    mbar_init(pfull, 4 * ks);
    mbar_init(pempty, 4 * ks);
    flags[0] = 0;
    fence_mbar_init();
  }
  if (warp == 4) mm_tmem_alloc<CG>(tslot);
  pdl_wait_and_release();
  // The group table. The threads have an expert each (of which there may be
  // several rounds); the one with this CTA's first tile says so.
  if (tid == 0) {
    goff[p.E] = 0;
    gtile[p.E] = 0;
    scan[31] = 0;
  }
  const int tile0 = (int)((uint32_t)first / (uint32_t)p.mtiles);
  for (int base = 0; base < p.E; base += kMmThreads) {
    const int e = base + tid;
    int a = 0, b = (int)p.rows, cnt = 0;
    if (e < p.E && tid < kMmThreads) {
      if (p.offsets) {
        a = min(max(__ldg(p.offsets + e), 0), (int)p.rows);
        b = min(max(__ldg(p.offsets + e + 1), a), (int)p.rows);
      }
      goff[e] = a;
      cnt = mm_tiles(b - a, p.ntile);
    }
    int run = 0;
    if (p.E > 1) {
      int incl = cnt;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += n;
      }
      if (lane == 31) scan[warp] = incl;
      __syncthreads();
      // warps before this one, and the rounds before (at the end of the table)
      int w = lane < warp ? scan[lane] : 0;
#pragma unroll
      for (int d = 16; d; d >>= 1) w += __shfl_xor_sync(0xffffffffu, w, d);
      run = gtile[p.E] + w + incl - cnt;
      __syncthreads();
    }
    if (e < p.E && tid < kMmThreads) {
      gtile[e] = run;
      if (cnt > 0 && tile0 >= run && tile0 < run + cnt) scan[31] = e;
      if (e + 1 == p.E || tid + 1 == kMmThreads) {
        goff[p.E] = b;
        gtile[p.E] = run + cnt;
      }
    }
    if (base + kMmThreads < p.E) __syncthreads();
  }
  tc_fence_before();
  if (CG * ks == 1)
    __syncthreads();
  else
    cooperative_groups::this_cluster().sync();  // the other CTAs' barriers are there too
  tc_fence_after();
  constexpr uint32_t tbase = 0;  // all 512 columns are this CTA's: they start at 0
  const int n_items = gtile[p.E] * p.mtiles;
  MmWalk<CG> it{goff, gtile, p.E, p.mtiles, p.ntile, (int)rank * kMmRows, scan[31], 0, 0, 0};

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (!elect_one()) return;
    uint32_t slot = 0, phase = 0, issued = 0;
    for (int item = first; item < n_items; item += stride) {
      it.at(item);
      const int y0 = it.e * (int)p.out_features + it.m0;
      const int half = mm_round(it.n) / CG;  // activation rows of this CTA
      const int ya = it.row0 + (int)rank * half;
      const int boxes = (half + p.box - 1) / p.box;
      const int got = p.order ? 4 * mm_quads(it.n, half, (int)rank) : boxes * p.box;
      const uint32_t bytes = kMmAPiece + got * 128;  // of a piece
      for (int st = st0; st < st1; ++st, ++issued) {
        const int pieces = min(2, (p.groups - st * 16 + 7) / 8);
        wait_mbar(empty + slot, phase ^ 1u, flags, p.error);
        mbar_arrive_expect_tx(cfull + slot, pieces * bytes);
        for (int k = 0; k < pieces; ++k) {
          const int x = st * 256 + k * 128;
          tma_load_2d(smem + (2 * slot + k) * kMmAPiece, &maps.w, x, y0, cfull + slot);
          if (!p.order)
            for (int b = 0; b < boxes; ++b)
              tma_load_2d(bring + (2 * slot + k) * b_piece + b * p.box * 128, &maps.a, x,
                          ya + b * p.box, cfull + slot);
        }
        if (++slot == (uint32_t)nst) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
    if (flags[0]) {
      // after an abort, let the copies in flight land before exiting
      for (uint32_t j = (issued > (uint32_t)nst ? issued - nst : 0); j < issued; ++j)
        for (uint32_t i = 0; i < kSpinLimit; ++i)
          if (mbar_try_wait(cfull + (j % nst), (j / nst) & 1u)) break;
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (!elect_one()) return;
    if (rank != 0) {
      // this CTA's copies have landed: tell the leader
      uint32_t slot = 0, phase = 0;
      for (int item = first; item < n_items; item += stride)
        for (int st = st0; st < st1; ++st) {
          wait_mbar(lfull + slot, phase, flags, p.error);
          mm_arrive<CG>(full + slot, 0, rank);
          if (++slot == (uint32_t)nst) {
            slot = 0;
            phase ^= 1u;
          }
        }
      mbar_arrive(done);
      leave_cluster();
      return;
    }
    const int sfc = mm_sf_cols(p.ntile), sfw = mm_sf_word(p.ntile);
    const uint64_t ad0 = umma_desc_sw128(smem_u32(smem)), bd0 = umma_desc_sw128(smem_u32(bring));
    uint32_t slot = 0, phase = 0, t = 0;
    for (int item = first; item < n_items; item += stride, ++t) {
      it.at(item);
      const uint32_t db = t & 1u;
      const int nn = mm_round(it.n);
      const uint32_t id0 = umma_idesc_mxf4<CG>(nn, 0), id1 = umma_idesc_mxf4<CG>(nn, 1);
      wait_mbar(dempty + db, ((t >> 1) & 1u) ^ 1u, flags, p.error);
      const uint32_t d_t = db * p.ntile;
      for (int st = st0; st < st1; ++st) {
        const uint32_t sfa = 2 * p.ntile + slot * sfc, sfb = sfa + 16;
        const uint64_t ad = ad0 + slot * (2 * kMmAPiece >> 4), bd = bd0 + slot * (2 * b_piece >> 4);
        wait_mbar(full + slot, phase, flags, p.error);
        tc_fence_after();
        // a row's last stage may hold fewer than eight steps of 64
        const int steps = min(8, (p.groups - st * 16 + 1) / 2);
        auto mma = [&](int kk) {
          tc_mma_mxf4<CG>(d_t, ad + ((kk >> 2) * (kMmAPiece >> 4) + (kk & 3) * 2),
                          bd + ((kk >> 2) * (b_piece >> 4) + (kk & 3) * 2), (kk & 1) ? id1 : id0,
                          sfa + 4 * (kk >> 1), sfb + sfw * (kk >> 1), (st > st0 || kk > 0) ? 1u : 0u);
        };
        if (steps == 8) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) mma(kk);
        } else {
          for (int kk = 0; kk < steps; ++kk) mma(kk);
        }
        mm_commit<CG>(empty + slot);
        if (++slot == (uint32_t)nst) {
          slot = 0;
          phase ^= 1u;
        }
      }
      mm_commit<CG>(dfull + db);
    }
    mm_commit<CG>(drain);
    wait_mbar(drain, 0, flags, p.error);
  } else if (warp < 4) {
    // ------------------------------------------- exponents to shared memory
    if (warp == 2)
      mm_load_scales<4, WIDE, true>(p, it, lane, first, stride, n_items, st0, st1, raw, rfull,
                                    rempty, flags);
    else
      mm_load_scales<mm_max_b(CG), WIDE, false>(p, it, lane, first, stride, n_items, st0, st1,
                                                       raw, rfull, rempty, flags);
    __syncwarp();
  } else if (warp >= 8 && warp < 12) {
    // -------------------------------------------- exponents to tensor memory
    const uint32_t lane_t = tbase + ((uint32_t)((warp & 3) * 32) << 16) + 2 * p.ntile;
    constexpr int kB = mm_max_b(CG);
    const int sfc = mm_sf_cols(p.ntile), sfw = mm_sf_word(p.ntile);
    const int slot_rows = mm_raw_rows(p.ntile);
    uint32_t slot = 0, phase = 0, rslot = 0, rphase = 0;
    for (int item = first; item < n_items; item += stride)
      for (int st = st0; st < st1; ++st) {
        wait_mbar(rfull + rslot, rphase, flags, p.error);
        const bool free = mbar_test(empty + slot, phase ^ 1u);
        const uint4* src = raw + rslot * slot_rows + lane;
        uint4 a[4], b[kB];  // rows lane + 32 i
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = src[32 * i];
#pragma unroll
        for (int i = 0; i < kB; ++i)
          b[i] = 32 * i < p.ntile ? src[kMmRows + 32 * i] : make_uint4(0, 0, 0, 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(rempty + rslot);
        if (++rslot == kMmRaw) {
          rslot = 0;
          rphase ^= 1u;
        }
        wait_mbar(empty + slot, phase ^ 1u, flags, p.error, free);
        __syncwarp();  // lanes may leave a wait one by one
        tc_fence_after();
        // columns 4 w + i (B: sfw w + i): word w of rows lane + 32 i
        const uint32_t t = lane_t + slot * sfc;
        uint32_t x[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = word_of(a[k & 3], k >> 2);
        tmem_st16(t, x);
        if (CG == 2 && p.ntile > 128) {
          uint32_t y[32];
#pragma unroll
          for (int k = 0; k < 32; ++k)
            y[k] = (k & 7) < kB ? word_of(b[(k & 7) < kB ? k & 7 : 0], k >> 3) : 0u;
          tmem_st32(t + 16, y);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) x[k] = (k & 3) < kB ? word_of(b[(k & 3) < kB ? k & 3 : 0], k >> 2) : 0u;
          tmem_st16(t + 16, x);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mm_arrive<CG>(full + slot, 0, rank);
        if (++slot == (uint32_t)nst) {
          slot = 0;
          phase ^= 1u;
        }
      }
    if (lane == 0) mbar_arrive(done);
    __syncwarp();
  } else if (warp >= 12) {
    // -------------------------------------------------------------- gathers
    if (!elect_one()) return;
    constexpr int kMine = (mm_max_n(CG) / CG / 4 + kMmGatherWarps - 1) / kMmGatherWarps;
    const int w = warp - 12;
    uint32_t slot = 0, phase = 0;
    for (int item = first; item < n_items; item += stride) {
      it.at(item);
      const int half = mm_round(it.n) / CG, nq = mm_quads(it.n, half, (int)rank);
      int4 rows[kMine];  // every kMmGatherWarps-th gather is this warp's
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (w + i * kMmGatherWarps >= nq) break;
        const int r0 = it.row0 + (int)rank * half + 4 * (w + i * kMmGatherWarps);
        const int r1 = it.row0 + it.n - 1;  // a last gather of fewer than four repeats one
        rows[i] =
            make_int4((int)mm_act_row(p, min(r0, r1)), (int)mm_act_row(p, min(r0 + 1, r1)),
                      (int)mm_act_row(p, min(r0 + 2, r1)), (int)mm_act_row(p, min(r0 + 3, r1)));
      }
      for (int st = st0; st < st1; ++st) {
        const int pieces = min(2, (p.groups - st * 16 + 7) / 8);
        wait_mbar(empty + slot, phase ^ 1u, flags, p.error);
        for (int k = 0; k < pieces; ++k) {
          char* dst = bring + (2 * slot + k) * b_piece;
#pragma unroll
          for (int i = 0; i < kMine; ++i) {
            const int q = w + i * kMmGatherWarps;
            if (q < nq)
              tma_gather4(dst + q * 512, &maps.a, st * 256 + k * 128, rows[i], cfull + slot);
          }
        }
        if (++slot == (uint32_t)nst) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
  } else {
    // ------------------------------------------------------------- epilogue
    const int q = warp & 3;
    uint32_t t = 0;
    for (int item = first; item < n_items; item += stride, ++t) {
      it.at(item);
      const uint32_t db = t & 1u;
      wait_mbar(dfull + db, (t >> 1) & 1u, flags, p.error);
      __syncwarp();
      tc_fence_after();
      const int64_t o = it.m0 + q * 32 + lane;
      const uint32_t d_t = tbase + db * p.ntile + ((uint32_t)(q * 32) << 16);
      if (ks > 1) {
        const int row = q * 32 + lane;
        wait_mbar(pempty, (t & 1u) ^ 1u, flags, p.error);
        for (int c = 0; c < it.n; c += 16) {
          float v[16];
          __syncwarp();
          tmem_ld16(d_t + c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) part[(c + i) * kMmRows + row] = v[i];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(dempty + db);
          fence_cluster();
          arrive_all(pfull, ks);
        }
        __syncwarp();
        wait_mbar(pfull, t & 1u, flags, p.error);
        fence_cluster();
        // this CTA's share of the columns, four at a time: all parts' loads first
        const int share = (it.n + ks - 1) / ks, c1 = min(it.n, (kpart + 1) * share);
        uint32_t from[kMmSplit];
#pragma unroll
        for (int k = 0; k < kMmSplit; ++k)
          from[k] = at_rank(smem_u32(part + row), k < ks ? k : 0);
        for (int c = kpart * share; c < c1; c += 4) {
          float x[4][kMmSplit];
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < kMmSplit; ++k)
              x[j][k] = k < ks && c + j < c1 ? ld_cluster(from[k] + (c + j) * kMmRows * 4) : 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float sum = x[j][0];
#pragma unroll
            for (int k = 1; k < kMmSplit; ++k) sum += x[j][k];
            if (c + j >= c1 || o >= p.out_features) continue;
            const int64_t to = ((int64_t)it.row0 + c + j) * p.out_features + o;
            if (p.out_f32)
              put(reinterpret_cast<float*>(p.out) + to, sum);
            else
              put(reinterpret_cast<uint16_t*>(p.out) + to, sum);
          }
        }
        __syncwarp();
        if (lane == 0) {
          fence_cluster();
          arrive_all(pempty, ks);
        }
        __syncwarp();
        continue;
      }
      for (int c = 0; c < it.n; c += 16) {
        float v[16];
        __syncwarp();  // lanes without a weight row skip the stores below
        tmem_ld16(d_t + c, v);
        if (o < p.out_features) {
          const int64_t at = ((int64_t)it.row0 + c) * p.out_features + o;
          if (p.out_f32)
            store16(reinterpret_cast<float*>(p.out) + at, p.out_features, it.n - c, v);
          else
            store16(reinterpret_cast<uint16_t*>(p.out) + at, p.out_features, it.n - c, v);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mm_arrive<CG>(dempty + db, 0, rank);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(done);
    if (warp == 4) {
      wait_mbar(done, 0, flags, p.error);
      wait_mbar(drain, 0, flags, p.error);
      if (CG == 2 && t > 0) {
        // the last arrivals at the ring's barriers, which nobody else waits for:
        // use j of the ring is slot j % nst, phase j / nst
        const uint32_t last = t * (uint32_t)p.nstages - 1, a = last / nst, r = last - a * nst;
        for (int s = 0; s < nst && (uint32_t)s <= last; ++s)
          wait_mbar(empty + s, ((uint32_t)s <= r ? a : a - 1) & 1u, flags, p.error);
      }
      __syncwarp();
      tc_fence_after();
      mm_tmem_dealloc<CG>();
    }
    // rows without a pair
    const int64_t z0 = (int64_t)goff[p.E] * p.out_features, z1 = p.rows * p.out_features;
    for (int64_t i = z0 + (int64_t)blockIdx.x * 128 + (tid - 128); i < z1;
         i += (int64_t)gridDim.x * 128) {
      if (p.out_f32)
        reinterpret_cast<float*>(p.out)[i] = 0.f;
      else
        reinterpret_cast<uint16_t*>(p.out)[i] = 0;
    }
    __syncwarp();
  }
  if (CG * ks > 1) leave_cluster();
}

}  // namespace mr
