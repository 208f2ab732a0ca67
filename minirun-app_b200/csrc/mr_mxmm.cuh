// mr_mxmm.cuh — MXFP4 x MXFP4 products on the 5th-generation tensor cores'
// block-scaled 4-bit form, one matrix or an expert stack over sorted rows.
//
//   out[r, o] = sum_b 2^(ea[r, b] + ew[o, b] - 254) * sum_{i in b} a[r, i] * w[o, i]
//
// over blocks b of 32 elements; tcgen05.mma kind::mxf4 multiplies e2m1 codes
// and both e8m0 scales exactly and sums in fp32. A tile is 128 weight rows
// (the M side, one TMEM lane each) by up to `ntile` activation rows (the N
// side, one TMEM column each): weight matrices are whole multiples of 128
// rows while an expert's rows are any number, and N steps by 16.
//
// One CTA per SM loops over tiles (expert's row tile x 128 weight rows, the
// weight rows fastest, so that CTAs working side by side share activations).
// Per stage of 256 elements (128 bytes of codes a row):
//   - warp 0: TMA loads of both operands' codes (128-byte swizzle) into the
//     ring;
//   - warps 12-15, by_token: the activations' codes instead, by TMA gathers of
//     four rows (48 a stage are more than one warp issues in a stage's time);
//   - warps 2 and 3: the exponents of weights / activations, 16 a row (two
//     stages) at a time, from global to shared memory;
//   - warps 8-11: the exponents from there into tensor memory, each warp its
//     lane quadrant (the tensor core reads the exponents of 32 rows a column,
//     in every quadrant). No proxy fence is on this way: one in the loading
//     warps waited for the loads of the next exponents too (1000 cycles a
//     stage), and copies by the tensor core (tcgen05.cp) cost the MMA warp
//     more issue time than the MMAs;
//   - warp 1: one MMA per 64 elements. Its lane, like those that issue TMA,
//     is chosen by elect.sync: from a branch on the lane's number each such
//     instruction cost 90-110 cycles (its operands live in uniform
//     registers), so 40; the other lanes leave;
//   - warps 4-7: a finished tile's accumulator to global memory while the
//     next tile's MMAs run (two accumulators).
// Every ring slot has exponents' columns of its own in TMEM, so they are only
// overwritten once the MMAs that read them are complete.
// Every wait is bounded: on expiry the kernel flags MR_DEVERR_TIMEOUT and
// runs to its end on garbage, drains its copies and MMAs, frees its TMEM.
#pragma once

#include "mr_gemv_umma.cuh"

namespace mr {

constexpr int kMmRows = 128;    // weight rows of a tile (MMA M)
constexpr int kMmK = 256;       // elements of a stage
constexpr int kMmMaxN = 192;      // activation rows of a tile: two accumulators and five
                                // slots of exponents fit the 512 TMEM columns
constexpr int kMmThreads = 384;   // plus the gather warps
constexpr int kMmGatherWarps = 4;
constexpr int kMmGathers = kMmMaxN / 4 / kMmGatherWarps;  // a warp's in a stage, at most
constexpr int kMmABytes = kMmRows * 128;
constexpr int kMmRaw = 3;  // slots of the exponents' ring in shared memory, two stages each
// TMEM columns of one stage's exponents: 4 a word of A, 4 a word and 128 rows of B.
MR_DEVICE __host__ constexpr int mm_sf_cols(int ntile) { return 8 + 8 * ((ntile + 127) / 128); }

struct MmParams {
  const uint8_t* w_scales;  // [E, out, in / 32]
  const uint8_t* a_scales;  // [arows, in / 32]
  const int32_t* offsets;   // [E + 1], or NULL: one matrix over all rows
  const int32_t* order;     // by_token: the pair at each sorted row, else NULL
  void* out;                // [rows, out]
  unsigned* error;
  int64_t rows, arows, out_features;
  int E, top_k;
  int groups;               // in / 32
  int nstages, mtiles;
  int ntile, box, nst;      // tile width, rows of an activation box, ring stages
  int out_f32;
};
struct MmMaps {
  CUtensorMap w, a;
};

// Shared memory: ring of codes, ring of exponents, barriers, group table.
MR_DEVICE __host__ constexpr int mm_raw_bytes(int ntile) { return (kMmRows + ntile) * 16; }
inline int mm_stage_bytes(int ntile) { return kMmABytes + ntile * 128; }
inline int mm_fixed_bytes(int E, int ntile) {
  return 1024 + kMmRaw * mm_raw_bytes(ntile) + 512 + 2 * (E + 1) * 4;
}

// True in one lane of a converged warp.
MR_DEVICE bool elect_one() {
  uint32_t on;
  asm volatile("{ .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p; }" : "=r"(on));
  return on != 0;
}
// D[128 x N] (+)= A . B^T with scales; both operands by shared descriptors.
MR_DEVICE void tc_mma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                           uint32_t sfa, uint32_t sfb, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], "
      "[%5], p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
      : "memory");
}
// wait_bounded with its first look at the barrier outside the loop. One lane
// of a warp waits so only where the others have left; elsewhere all lanes
// wait together. (Lanes parked at a warp barrier made every branch of the
// running one slow: 185-280 cycles for a wait that is already over, here 53.)
MR_DEVICE void wait_mbar(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                         unsigned* error) {
  if (!mbar_try_wait(bar, parity)) wait_bounded(bar, parity, abort_flag, error);
}
// Four consecutive TMEM columns of this thread's lane.
MR_DEVICE void tmem_st4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
// kind::mxf4, e2m1 x e2m1, e8m0 scales, M = 128; `half`: which two of a
// word's four exponents (both operands).
MR_DEVICE uint32_t umma_idesc_mxf4(int n, uint32_t half) {
  return (half << 5)                   // B exponents: id 0 or 2 at bits 4-5
         | (1u << 7) | (1u << 10)      // A, B: e2m1
         | ((uint32_t)(n >> 3) << 17)  // N / 8
         | (1u << 23)                  // exponents: e8m0
         | (1u << 27)                  // M / 128
         | (half << 30);               // A exponents: id at bits 29-30
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

// An expert's n rows in tiles of equal width, a multiple of 16: as few as
// ntile allows, none empty.
MR_DEVICE int mm_width(int n, int ntile) {
  const int c = (n + ntile - 1) / ntile;
  return c > 0 ? ((n + c - 1) / c + 15) & ~15 : 16;
}
MR_DEVICE int mm_tiles(int n, int ntile) {
  const int w = mm_width(n, ntile);
  return (n + w - 1) / w;
}

// Walks the CTA's tiles in order: item -> expert, rows and weight rows.
struct MmWalk {
  const int* goff;    // [E + 1] first row of each expert
  const int* gtile;   // [E + 1] first row tile of each expert
  int mtiles, ntile;
  int e = 0, row0 = 0, n = 0, m0 = 0;
  MR_DEVICE void at(int item) {
    const int t = item / mtiles;
    m0 = (item - t * mtiles) * kMmRows;
    while (gtile[e + 1] <= t) ++e;
    const int all = goff[e + 1] - goff[e];
    const int w = mm_width(all, ntile);
    const int first = (t - gtile[e]) * w;
    row0 = goff[e] + first;
    n = min(w, all - first);
  }
};

// The token row that sorted row r takes its activations from.
MR_DEVICE int64_t mm_act_row(const MmParams& p, int64_t r) {
  if (p.order) {
    const int pair = __ldg(p.order + r);
    r = pair < 0 ? 0 : pair / p.top_k;
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
// activations, 16 a row (two stages) at a time. WIDE: every row is made of
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

// Exponents from global to shared memory, loaded one or two pairs of stages
// (also of the next tile) ahead of their use: the loads' latency stays out of the
// pipeline. A slot holds 16 bytes a row. Every lane of the warp.
template <int NB, bool WIDE, bool IS_A>
MR_DEVICE void mm_load_scales(const MmParams& p, const MmWalk& walk, int lane, int n_items,
                              uint4* raw, uint64_t* rfull, uint64_t* rempty,
                              volatile int* flags) {
  const int npairs = (p.nstages + 1) / 2;
  const int slot_rows = kMmRows + p.ntile;
  const uint8_t* lo = IS_A ? p.w_scales : p.a_scales;
  const uint8_t* hi = lo + (IS_A ? (int64_t)p.E * p.out_features : p.arows) * p.groups;
  MmWalk it = walk;
  const uint8_t* src[NB];
  auto open = [&](int item) {
    if (item >= n_items) return;
    it.at(item);
    const int have = IS_A ? kMmRows : it.n;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      // rows past the tile's end repeat its last: their results are not kept
      const int r = min(lane + 32 * i, have - 1);
      const int64_t row =
          IS_A ? (int64_t)it.e * p.out_features + min((int64_t)it.m0 + r, p.out_features - 1)
               : mm_act_row(p, (int64_t)it.row0 + r);
      src[i] = 32 * i < have ? lo + row * p.groups : nullptr;
    }
  };
  constexpr int kAhead = WIDE ? 2 : 1;  // registers of two unaligned pairs would spill
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
  int litem = blockIdx.x, lq = 0;  // the pair to load next
  open(litem);
  auto load = [&](MmScaleRegs<NB, WIDE>& r) {
    if (litem >= n_items) return;
    r.load(src, lq, p.groups, lo, hi);
    if (++lq == npairs) {
      lq = 0;
      litem += gridDim.x;
      open(litem);
    }
  };
#pragma unroll
  for (int b = 0; b < kAhead; ++b) load(v[b]);
  uint32_t slot = 0, phase = 0;
  int item = blockIdx.x, q = 0;  // the pair to hand on next
  while (item < n_items) {
#pragma unroll
    for (int b = 0; b < kAhead; ++b) {
      if (item >= n_items) break;
      wait_mbar(rempty + slot, phase ^ 1u, flags, p.error);
      uint4* dst = raw + slot * slot_rows + (IS_A ? 0 : kMmRows) + lane;
#pragma unroll
      for (int i = 0; i < NB; ++i)
        if (IS_A || 32 * i + lane < p.ntile) dst[32 * i] = v[b].get(i);
      __syncwarp();
      if (lane == 0) mbar_arrive(rfull + slot);
      if (++slot == kMmRaw) {
        slot = 0;
        phase ^= 1u;
      }
      load(v[b]);
      if (++q == npairs) {
        q = 0;
        item += gridDim.x;
      }
    }
  }
}

template <bool WIDE>
__global__ void __launch_bounds__(kMmThreads + 32 * kMmGatherWarps, 1)
    mxmm_kernel(const MmParams p, const __grid_constant__ MmMaps maps) {
  extern __shared__ char smem_raw[];
  char* smem =
      reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int b_bytes = p.ntile * 128;
  const int nst = p.nst;
  char* bring = smem + nst * kMmABytes;
  uint4* raw = reinterpret_cast<uint4*>(bring + nst * b_bytes);  // [kMmRaw][128 + ntile]
  uint64_t* full = reinterpret_cast<uint64_t*>(raw + kMmRaw * (kMmRows + p.ntile));  // [nst]
  uint64_t* empty = full + nst;       // [nst]
  uint64_t* rfull = empty + nst;      // [kMmRaw] exponents in shared memory
  uint64_t* rempty = rfull + kMmRaw;  // [kMmRaw] and read from there
  uint64_t* dfull = rempty + kMmRaw;  // [2]
  uint64_t* dempty = dfull + 2;       // [2]
  uint64_t* drain = dempty + 2;       // every MMA complete
  uint64_t* done = drain + 1;         // every other access of TMEM too
  uint32_t* tslot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* flags = reinterpret_cast<volatile int*>(tslot + 1);
  int* scan = reinterpret_cast<int*>(tslot + 2);  // [16] warp sums
  int* goff = scan + 16;
  int* gtile = goff + p.E + 1;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int s = 0; s < nst; ++s) {
      mbar_init(full + s, 5);  // the copies' bytes, four warps' exponents
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < kMmRaw; ++s) {
      mbar_init(rfull + s, 2);
      mbar_init(rempty + s, 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(dfull + b, 1);
      mbar_init(dempty + b, 4);
    }
    mbar_init(drain, 1);
    mbar_init(done, 8);
    flags[0] = 0;
    fence_mbar_init();
  }
  if (warp == 4) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  pdl_wait_and_release();
  // the group table: thread i has experts 4i .. 4i+3 (E <= 1024: the first 256 threads)
  {
    int cnt[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = 4 * tid + i;
      cnt[i] = 0;
      if (e < p.E) {
        int a = 0, b = (int)p.rows;
        if (p.offsets) {
          a = min(max(__ldg(p.offsets + e), 0), (int)p.rows);
          b = min(max(__ldg(p.offsets + e + 1), a), (int)p.rows);
        }
        goff[e] = a;
        if (e + 1 == p.E) goff[p.E] = b;
        cnt[i] = mm_tiles(b - a, p.ntile);
      }
      sum += cnt[i];
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += n;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int run = incl - sum;
    for (int w = 0; w < warp; ++w) run += scan[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = 4 * tid + i;
      if (e < p.E) {
        gtile[e] = run;
        run += cnt[i];
        if (e + 1 == p.E) gtile[p.E] = run;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tbase = 0;  // all 512 columns are this CTA's: they start at 0
  const int n_items = gtile[p.E] * p.mtiles;
  MmWalk it{goff, gtile, p.mtiles, p.ntile};

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (!elect_one()) return;
    uint32_t slot = 0, phase = 0, issued = 0;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
      it.at(item);
      const int y0 = it.e * (int)p.out_features + it.m0;
      const int boxes = (it.n + p.box - 1) / p.box;
      const uint32_t bytes =
          kMmABytes + (p.order ? (it.n + 15) / 16 * 16 : boxes * p.box) * 128;
      for (int st = 0; st < p.nstages; ++st, ++issued) {
        wait_mbar(empty + slot, phase ^ 1u, flags, p.error);
        mbar_arrive_expect_tx(full + slot, bytes);
        tma_load_2d(smem + slot * kMmABytes, &maps.w, st * 128, y0, full + slot);
        if (!p.order)
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(bring + slot * b_bytes + b * p.box * 128, &maps.a, st * 128,
                        it.row0 + b * p.box, full + slot);
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
          if (mbar_try_wait(full + (j % nst), (j / nst) & 1u)) break;
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (!elect_one()) return;
    const int sfc = mm_sf_cols(p.ntile), sfw = sfc / 2 - 4;
    const uint32_t a0 = smem_u32(smem), b0 = smem_u32(bring);
    uint32_t slot = 0, phase = 0, t = 0;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x, ++t) {
      it.at(item);
      const uint32_t db = t & 1u;
      const int nn = (it.n + 15) & ~15;
      wait_mbar(dempty + db, ((t >> 1) & 1u) ^ 1u, flags, p.error);
      const uint32_t d_t = db * p.ntile;
      for (int st = 0; st < p.nstages; ++st) {
        const uint32_t sfa = 2 * p.ntile + slot * sfc, sfb = sfa + 8;
        const uint32_t at = a0 + slot * kMmABytes, bt = b0 + slot * b_bytes;
        wait_mbar(full + slot, phase, flags, p.error);
        tc_fence_after();
        // a row's last stage may hold fewer than four steps of 64
        const int steps = min(4, (p.groups - st * 8 + 1) / 2);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          if (kk < steps)
            tc_mma_mxf4(d_t, umma_desc_sw128(at + kk * 32), umma_desc_sw128(bt + kk * 32),
                        umma_idesc_mxf4(nn, kk & 1), sfa + 4 * (kk >> 1), sfb + sfw * (kk >> 1),
                        (st | kk) ? 1u : 0u);
        tc_commit(empty + slot);
        if (++slot == (uint32_t)nst) {
          slot = 0;
          phase ^= 1u;
        }
      }
      tc_commit(dfull + db);
    }
    tc_commit(drain);
    wait_mbar(drain, 0, flags, p.error);
  } else if (warp < 4) {
    // ------------------------------------------- exponents to shared memory
    if (warp == 2)
      mm_load_scales<4, WIDE, true>(p, it, lane, n_items, raw, rfull, rempty, flags);
    else
      mm_load_scales<kMmMaxN / 32, WIDE, false>(p, it, lane, n_items, raw, rfull, rempty, flags);
  } else if (warp >= 8 && warp < 12) {
    // -------------------------------------------- exponents to tensor memory
    const uint32_t lane_t = tbase + ((uint32_t)((warp & 3) * 32) << 16) + 2 * p.ntile;
    const int sfc = mm_sf_cols(p.ntile), slot_rows = kMmRows + p.ntile;
    uint32_t slot = 0, phase = 0, rslot = 0, rphase = 0;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
      for (int st = 0; st < p.nstages; st += 2) {
        wait_mbar(rfull + rslot, rphase, flags, p.error);
        const uint4* src = raw + rslot * slot_rows + lane;
        uint4 a[4], b[8];  // rows lane + 32 i
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = src[32 * i];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          b[i] = 32 * i + lane < p.ntile ? src[kMmRows + 32 * i] : make_uint4(0, 0, 0, 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(rempty + rslot);
        if (++rslot == kMmRaw) {
          rslot = 0;
          rphase ^= 1u;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (st + h >= p.nstages) break;
          wait_mbar(empty + slot, phase ^ 1u, flags, p.error);
          tc_fence_after();
          const uint32_t t = lane_t + slot * sfc;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            // word 2 h + w of each row
            auto word = [&](const uint4& v) {
              return h == 0 ? (w == 0 ? v.x : v.y) : (w == 0 ? v.z : v.w);
            };
            tmem_st4(t + 4 * w, word(a[0]), word(a[1]), word(a[2]), word(a[3]));
            const uint32_t tb = t + 8 + w * (sfc / 2 - 4);
            tmem_st4(tb, word(b[0]), word(b[1]), word(b[2]), word(b[3]));
            if (p.ntile > 128) tmem_st4(tb + 4, word(b[4]), word(b[5]), word(b[6]), word(b[7]));
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(full + slot);
          if (++slot == (uint32_t)nst) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
    }
    if (lane == 0) mbar_arrive(done);
  } else if (warp >= 12) {
    // -------------------------------------------------------------- gathers
    if (!elect_one()) return;
    const int w = warp - 12;
    uint32_t slot = 0, phase = 0;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
      it.at(item);
      const int nq = (it.n + 15) / 16 * 4;
      int4 rows[kMmGathers];  // every kMmGatherWarps-th gather is this warp's
#pragma unroll
      for (int i = 0; i < kMmGathers; ++i) {
        const int r0 = it.row0 + 4 * (w + i * kMmGatherWarps), r1 = it.row0 + it.n - 1;
        // rows past the tile's end repeat its last
        rows[i] = make_int4((int)mm_act_row(p, min(r0, r1)), (int)mm_act_row(p, min(r0 + 1, r1)),
                            (int)mm_act_row(p, min(r0 + 2, r1)), (int)mm_act_row(p, min(r0 + 3, r1)));
      }
      for (int st = 0; st < p.nstages; ++st) {
        wait_mbar(empty + slot, phase ^ 1u, flags, p.error);
        char* dst = bring + slot * b_bytes;
#pragma unroll
        for (int i = 0; i < kMmGathers; ++i) {
          const int q = w + i * kMmGatherWarps;
          if (q < nq) tma_gather4(dst + q * 512, &maps.a, st * 128, rows[i], full + slot);
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
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
      it.at(item);
      const uint32_t db = t & 1u;
      wait_mbar(dfull + db, (t >> 1) & 1u, flags, p.error);
      tc_fence_after();
      const int64_t o = it.m0 + q * 32 + lane;
      const uint32_t d_t = tbase + db * p.ntile + ((uint32_t)(q * 32) << 16);
      for (int c = 0; c < it.n; c += 16) {
        float v[16];
        tmem_ld16(d_t + c, v);
        if (o < p.out_features) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (c + i >= it.n) break;
            const int64_t at = ((int64_t)it.row0 + c + i) * p.out_features + o;
            if (p.out_f32)
              reinterpret_cast<float*>(p.out)[at] = v[i];
            else
              reinterpret_cast<uint16_t*>(p.out)[at] = f32_to_bf16_bits(v[i]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dempty + db);
      ++t;
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(done);
    if (warp == 4) {
      wait_mbar(done, 0, flags, p.error);
      wait_mbar(drain, 0, flags, p.error);
      tc_fence_after();
      tmem_dealloc(tbase, 512);
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
  }
}

}  // namespace mr
