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
//     ring; by_token rows through one-row gathers of four;
//   - warps 2 and 3: the stage's 8 exponents a row of weights / activations
//     from global memory into the layout the tensor core wants them copied
//     from (per 128 rows and 4 exponents 512 bytes: row r at (r % 32) * 16 +
//     (r / 32) * 4);
//   - warp 1, one lane: tcgen05.cp of the exponents to TMEM, then one MMA per
//     64 elements;
//   - warps 4-7: a finished tile's accumulator to global memory while the
//     next tile's MMAs run (two accumulators).
// Exponents in TMEM are double-buffered: the copy for a stage is issued once
// the MMAs of two stages ago, the last to read that buffer, are complete.
// Every wait is bounded: on expiry the kernel flags MR_DEVERR_TIMEOUT and
// runs to its end on garbage, drains its copies and MMAs, frees its TMEM.
#pragma once

#include "mr_gemv_umma.cuh"

namespace mr {

constexpr int kMmRows = 128;    // weight rows of a tile (MMA M)
constexpr int kMmK = 256;       // elements of a stage
constexpr int kMmMaxN = 224;    // activation rows of a tile: two accumulators and the
                                // exponents' buffers fill the 512 TMEM columns
constexpr int kMmThreads = 256;
constexpr int kMmABytes = kMmRows * 128;
constexpr int kMmSfCols = 24;   // TMEM columns of one stage's exponents: 8 of A, 16 of B
constexpr int kMmSfCol0 = 2 * kMmMaxN;
static_assert(kMmSfCol0 + 2 * kMmSfCols <= 512, "TMEM holds 512 columns");

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
  int wide_scales;          // rows of exponents are whole, aligned 16-byte pieces
};
struct MmMaps {
  CUtensorMap w, a;
};

// Shared memory: ring of codes, ring of exponents, barriers, group table.
MR_DEVICE __host__ constexpr int mm_sf_bytes(int ntile) {
  return 1024 + 1024 * ((ntile + 127) / 128);
}
inline int mm_stage_bytes(int ntile) { return kMmABytes + ntile * 128 + mm_sf_bytes(ntile); }
inline int mm_fixed_bytes(int E) { return 1024 + 512 + 2 * (E + 1) * 4; }

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
// 512 bytes (32 rows of 16) to 4 TMEM columns of all four lane quadrants.
MR_DEVICE void tc_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}
// Unswizzled K-major descriptor: 8-row groups of 128 contiguous bytes.
MR_DEVICE uint64_t umma_desc_plain(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 16) |
         ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
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
MR_DEVICE void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Four rows (y0..y3) of 128 bytes at column x.
MR_DEVICE void tma_gather4(void* dst, const CUtensorMap* map, int x, int4 y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w),
      "r"(smem_u32(bar))
      : "memory");
}

// Tiles of an expert with n rows: as few as ntile allows, of equal width (a
// multiple of 16).
MR_DEVICE int mm_tiles(int n, int ntile) { return (n + ntile - 1) / ntile; }

// Walks the CTA's tiles: item -> expert, rows and weight rows.
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
    const int c = gtile[e + 1] - gtile[e];
    const int w = ((all + c - 1) / c + 15) & ~15;
    const int first = (t - gtile[e]) * w;
    row0 = goff[e] + first;
    n = min(w, all - first);  // may be <= 0: rounding up can leave the last tile empty
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

// One stage's 8 exponents of a row; 127 past the row's end.
MR_DEVICE uint2 mm_load_scales(const uint8_t* row, int g0, int groups) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t e = g0 + i < groups ? (uint32_t)__ldg(row + g0 + i) : 127u;
    w[i >> 2] |= e << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

__global__ void __launch_bounds__(kMmThreads, 1)
    mxmm_kernel(const MmParams p, const __grid_constant__ MmMaps maps) {
  extern __shared__ char smem_raw[];
  char* smem =
      reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int b_bytes = p.ntile * 128, sf_bytes = mm_sf_bytes(p.ntile);
  const int nst = p.nst;
  char* bring = smem + nst * kMmABytes;
  char* sring = bring + nst * b_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sring + nst * sf_bytes);  // [nst]
  uint64_t* empty = full + nst;  // [nst]
  uint64_t* dfull = empty + nst;  // [2]
  uint64_t* dempty = dfull + 2;   // [2]
  uint64_t* drain = dempty + 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* flags = reinterpret_cast<volatile int*>(tslot + 1);
  int* scan = reinterpret_cast<int*>(tslot + 2);  // [8] warp sums
  int* goff = scan + 8;
  int* gtile = goff + p.E + 1;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int s = 0; s < nst; ++s) {
      mbar_init(full + s, 3);  // producer, two exponent warps
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(dfull + b, 1);
      mbar_init(dempty + b, 4);
    }
    mbar_init(drain, 1);
    flags[0] = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  pdl_wait_and_release();
  // the group table: thread i has experts 4i .. 4i+3 (E <= 1024)
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
  const uint32_t tbase = *tslot;
  const int n_items = gtile[p.E] * p.mtiles;
  MmWalk it{goff, gtile, p.mtiles, p.ntile};

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    uint32_t slot = 0, phase = 0, issued = 0;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
      it.at(item);
      if (it.n <= 0) continue;
      const int y0 = it.e * (int)p.out_features + it.m0;
      const int boxes = (it.n + p.box - 1) / p.box;
      int4 rows[2];
      if (p.order) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          int y[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            y[q] = (int)mm_act_row(p, it.row0 + min(4 * (lane + 32 * i) + q, it.n - 1));
          rows[i] = make_int4(y[0], y[1], y[2], y[3]);
        }
      }
      const int quads = (it.n + 15) / 16 * 4;  // gathers of four rows: N of the MMA
      for (int st = 0; st < p.nstages; ++st) {
        char* A = smem + slot * kMmABytes;
        char* B = bring + slot * b_bytes;
        if (lane == 0) {
          wait_bounded(empty + slot, phase ^ 1u, flags, p.error);
          mbar_arrive_expect_tx(full + slot,
                                kMmABytes + (p.order ? quads * 512 : boxes * p.box * 128));
          tma_load_2d(A, &maps.w, st * 128, y0, full + slot);
        }
        __syncwarp();
        if (p.order) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (lane + 32 * i < quads)
              tma_gather4(B + (lane + 32 * i) * 512, &maps.a, st * 128, rows[i], full + slot);
        } else if (lane < boxes) {
          tma_load_2d(B + lane * p.box * 128, &maps.a, st * 128, it.row0 + lane * p.box,
                      full + slot);
        }
        ++issued;
        if (++slot == (uint32_t)nst) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
    if (lane == 0 && flags[0]) {
      // after an abort, let the copies in flight land before exiting
      for (uint32_t j = (issued > (uint32_t)nst ? issued - nst : 0); j < issued; ++j)
        for (uint32_t i = 0; i < kSpinLimit; ++i)
          if (mbar_try_wait(full + (j % nst), (j / nst) & 1u)) break;
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0) {
      uint32_t slot = 0, phase = 0, j = 0, t = 0;
      for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        it.at(item);
        if (it.n <= 0) continue;
        const uint32_t db = t & 1u;
        const int nn = (it.n + 15) & ~15;
        const int nblk = (nn + 127) / 128, sblk = (p.ntile + 127) / 128;
        wait_bounded(dempty + db, ((t >> 1) & 1u) ^ 1u, flags, p.error);
        const uint32_t d_t = tbase + db * kMmMaxN;
        for (int st = 0; st < p.nstages; ++st, ++j) {
          wait_bounded(full + slot, phase, flags, p.error);
          if (j >= 2)  // the exponents' buffer: free once stage j - 2 is done
            wait_bounded(empty + (j - 2) % nst, ((j - 2) / nst) & 1u, flags, p.error);
          tc_fence_after();
          const uint32_t sfa = tbase + kMmSfCol0 + (j & 1u) * kMmSfCols, sfb = sfa + 8;
          const uint32_t sf = smem_u32(sring + slot * sf_bytes);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            tc_cp_scales(sfa + 4 * w, umma_desc_plain(sf + 512 * w));
            for (int b = 0; b < nblk; ++b)
              tc_cp_scales(sfb + 8 * w + 4 * b,
                           umma_desc_plain(sf + 1024 + 512 * (w * sblk + b)));
          }
          const uint32_t at = smem_u32(smem + slot * kMmABytes);
          const uint32_t bt = smem_u32(bring + slot * b_bytes);
          // a row's last stage may hold fewer than four steps of 64
          const int steps = min(4, (p.groups - st * 8 + 1) / 2);
          for (int kk = 0; kk < steps; ++kk)
            tc_mma_mxf4(d_t, umma_desc_sw128(at + kk * 32), umma_desc_sw128(bt + kk * 32),
                        umma_idesc_mxf4(nn, kk & 1), sfa + 4 * (kk >> 1), sfb + 8 * (kk >> 1),
                        (st | kk) ? 1u : 0u);
          tc_commit(empty + slot);
          if (++slot == (uint32_t)nst) {
            slot = 0;
            phase ^= 1u;
          }
        }
        tc_commit(dfull + db);
        ++t;
      }
      tc_commit(drain);
      wait_bounded(drain, 0, flags, p.error);
    }
  } else if (warp < 4) {
    // ----------------------------------------------------- exponents to smem
    const bool is_a = warp == 2;
    const int nrow = is_a ? 4 : 8;  // rows of a lane: lane + 32 i
    const int sblk = (p.ntile + 127) / 128;
    uint32_t slot = 0, phase = 0;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
      it.at(item);
      if (it.n <= 0) continue;
      const uint8_t* src[8];
      const int have = is_a ? kMmRows : it.n;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= nrow || 32 * i >= have) {
          src[i] = nullptr;
          continue;
        }
        // rows past the tile's end repeat its last: their results are not kept
        const int r = min(lane + 32 * i, have - 1);
        src[i] = is_a ? p.w_scales + ((int64_t)it.e * p.out_features +
                                      min((int64_t)it.m0 + r, p.out_features - 1)) * p.groups
                      : p.a_scales + mm_act_row(p, (int64_t)it.row0 + r) * p.groups;
      }
      uint4 pair[8];  // two stages' exponents of each row
      for (int st = 0; st < p.nstages; ++st) {
        uint2 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = make_uint2(0, 0);
          if (!src[i]) continue;
          if (p.wide_scales) {
            if ((st & 1) == 0) pair[i] = __ldg(reinterpret_cast<const uint4*>(src[i] + st * 8));
            v[i] = (st & 1) ? make_uint2(pair[i].z, pair[i].w) : make_uint2(pair[i].x, pair[i].y);
          } else {
            v[i] = mm_load_scales(src[i], st * 8, p.groups);
          }
        }
        if (lane == 0) wait_bounded(empty + slot, phase ^ 1u, flags, p.error);
        __syncwarp();
        uint4* dst = reinterpret_cast<uint4*>(sring + slot * sf_bytes + (is_a ? 0 : 1024));
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (b && (is_a || 128 >= have)) break;
          const int nb = is_a ? 1 : sblk;
          dst[(0 * nb + b) * 32 + lane] =
              make_uint4(v[4 * b].x, v[4 * b + 1].x, v[4 * b + 2].x, v[4 * b + 3].x);
          dst[(1 * nb + b) * 32 + lane] =
              make_uint4(v[4 * b].y, v[4 * b + 1].y, v[4 * b + 2].y, v[4 * b + 3].y);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full + slot);
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
      if (it.n <= 0) continue;
      const uint32_t db = t & 1u;
      if (lane == 0) wait_bounded(dfull + db, (t >> 1) & 1u, flags, p.error);
      __syncwarp();
      (void)mbar_try_wait(dfull + db, (t >> 1) & 1u);
      tc_fence_after();
      const int64_t o = it.m0 + q * 32 + lane;
      const uint32_t d_t = tbase + db * kMmMaxN + ((uint32_t)(q * 32) << 16);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tbase, 512);
}

}  // namespace mr
