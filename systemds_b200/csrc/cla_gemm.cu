// Products of dense operands in 8 and 16 bits with their epilogues (GemmCall of cla_dense.cuh), on the 5th-generation tensor cores: operands by
// TMA into 128-byte-swizzled shared memory, sums in tensor memory (FP32, or 32-bit integers for 8-bit operands), epilogues from there.
//  * k_gemm_pair: two CTAs share a 256 x 256 tile. For large results.
//  * k_gemm_few: tiles of 128 columns of the result and 16 to 128 of its rows, whose depth the CTAs share evenly; k_gemm_join adds up the
//    parts of tiles that several CTAs share. For few rows.
//  * k_gemm_rows: 8-bit products of many rows with few columns, which quantises the rows on the way.
// All are launched with at most one CTA an SM, which takes all of the SM's shared and tensor memory and loops: no CTA waits for tensor memory.
#include <cuda.h>
#include <algorithm>
#include <atomic>
#include "cla_dense.cuh"

namespace cla {

static __device__ int32_t denseErr;

// ---- PTX ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t gm_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool gm_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done)
               : "r"(bar), "r"(parity)
               : "memory");
  return done != 0;
}
// Gives up after 16.6 s (a try that finds nothing lasts 3.95 us): a mistake ends as an error and not as a hung GPU. The longest wait of a launch without one is
// that for a tile's sums, 0.17 us for 64 terms: 2.9 s for 2^30, the most rows that a gradient of the weights sums over.
__device__ __forceinline__ bool gm_wait(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < (1 << 22); i++)
    if (gm_try(bar, parity)) return true;
  return false;
}
__device__ __forceinline__ uint32_t gm_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
// The warp's number, of which the compiler knows that all lanes have it: what depends on it alone then stays in the warp's own registers, where the
// copies and products take their operands (a loop of one lane spent 600 clocks a stage on bringing them there; this one 300)
__device__ __forceinline__ int gm_warp() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }
// A wait of the whole warp
__device__ __forceinline__ bool gm_wait_all(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, gm_wait(bar, parity)); }
__device__ __forceinline__ uint32_t gm_peer(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// (the warps whole before and after: what follows may need all lanes together)
__device__ __forceinline__ void gm_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ bool gm_elect() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void gm_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void gm_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A box at element (x, y); PAIR: the barrier may be the other CTA's
template <bool PAIR>
__device__ __forceinline__ void gm_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
template <bool PAIR, bool I8>
__device__ __forceinline__ void gm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
#define GM_MMA(GROUP, KIND)                                                                                                             \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}" ::"r"(d), \
               "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)                                                                            \
               : "memory")
  if (PAIR) {
    if (I8) GM_MMA("2", "i8");
    else GM_MMA("2", "f16");
  } else {
    if (I8) GM_MMA("1", "i8");
    else GM_MMA("1", "f16");
  }
#undef GM_MMA
}
// The barrier gets an arrival when the products issued so far are done; PAIR: both CTAs' barriers
template <bool PAIR>
__device__ __forceinline__ void gm_commit(uint32_t bar) {
  if (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 16 columns of a warp's 32 lanes; gm_loaded() before the registers are read
__device__ __forceinline__ void gm_tmem16(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void gm_tmem8(uint32_t addr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(addr)
               : "memory");
}
template <int N>
__device__ __forceinline__ void gm_loaded(uint32_t (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+r"(v[i]));
}

// The end of a copying warp: every stage that it filled `issued` times in turn has been read (its own copies, and the products from it, are over). After a
// wait that ran out, the copies alone, where this CTA's barriers tell of them.
__device__ __forceinline__ void gm_drain(bool& ok, bool own, uint32_t fullAt, uint32_t emptyAt, int issued, int stages) {
  for (int i = 0; i < stages && i < issued; i++) {
    const uint32_t last = (uint32_t)((issued - i + stages - 1) / stages - 1) & 1u;
    if (ok) ok = gm_wait_all(emptyAt + i * 8, last);
    else if (own) gm_wait_all(fullAt + i * 8, last);
  }
}

// ---- operands in shared memory ----------------------------------------------------------------------------------------
// A stage is 128 bytes deep: 64 values of 16 bits, 128 of 8. Rows of 128 bytes, swizzled over 1024-byte groups of eight.
// Depth contiguous (K-major): a row per index, groups of eight indexes 1024 bytes apart; the next 32 bytes of depth lie 32 bytes on.
// Index contiguous (16-bit types): a row per depth step, 64 indexes wide, 64 rows to a box of 8 KB; the next 16 steps lie 2 KB on.
constexpr uint32_t GM_OPERAND = 128 * 128;  // bytes of 128 indexes
__device__ __forceinline__ uint64_t gm_desc(uint32_t addr, bool mn) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(mn ? 8192 >> 4 : 1) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
__host__ __device__ constexpr uint32_t gm_step(bool mn) { return mn ? 2048 >> 4 : 32 >> 4; }

struct alignas(64) GemmArgs {
  CUtensorMap a[2], b[2];
  GemmCall c;
  int depth;             // values of a stage
  int kBlocks;           // stages of a segment
  int tilesM, tilesN;    // PAIR: tilesN of both products
  int wide;              // k_gemm_pair: columns of a tile (GATE: of each product)
  int stages;            // of the ring
  int nc;                // k_gemm_few: rows of a tile,
  int ctas, whole;       // CTAs, and whether each has whole tiles
  uint32_t idesc;
};

// ---- epilogues ----------------------------------------------------------------------------------------------------------
template <class O> __device__ __forceinline__ O gm_cast(float v) { return from_f32<O>(v); }

// Whether all of some of a CTA's warps say so
__device__ __forceinline__ bool gm_group_all(int id, int threads, bool ok) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.and.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r)
               : "r"(id), "r"(threads), "r"((uint32_t)ok)
               : "memory");
  return r != 0;
}
// The warps that hold the same 32 rows of a tile (a lane each), G of them, write `width` columns of these rows. f(j, o): columns j .. j + CH - 1 of
// the lane's row, all lanes together. The warps take LINE / G bytes of a row in turn into the shared memory of the group; from there whole rows
// of up to LINE bytes go out, 32 / G rows a warp: in pieces of 16 bytes where rows start on 16-byte boundaries (vec), else a word a
// lane. (Long pieces count where rows do not start on sectors: each piece then writes parts of two sectors.) The pieces of shared
// memory are swizzled over the rows.
template <class O, int CH, int G, class F>
__device__ __forceinline__ void gm_rows(O* out, int64_t ld, int rows, int64_t cols, int width, bool vec, uint32_t buf, int part, int id, F&& f) {
  constexpr int LINE = 256, PIECES = CH * (int)sizeof(O) / 16;
  const int lane = threadIdx.x & 31, mine = min(LINE / G / (int)sizeof(O), width / G), all = mine * G;  // columns of a warp, of the group
  const auto place = [&](int r, int piece) { return buf + r * LINE + (piece ^ (r & 7)) * 16; };
#pragma unroll 1
  for (int c0 = 0; c0 < width; c0 += all) {
#pragma unroll 1
    for (int j = part * mine; j < (part + 1) * mine; j += CH) {
      alignas(16) O o[CH];
      f(c0 + j, o);
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const uint4 x = *(const uint4*)(o + i * (CH / PIECES));
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(lane, j * (int)sizeof(O) / 16 + i)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
      }
    }
    gm_group_sync(id, G * 32);
    const int there = (int)max((int64_t)0, min((int64_t)all, cols - c0)) * (int)sizeof(O);  // bytes of a row
    const int end = min(rows, (part + 1) * (32 / G));
    if (vec) {
      const int per = all * (int)sizeof(O) / 16, down = 32 / per;  // pieces of a row, rows at a time (all powers of two)
      const int piece = lane & (per - 1), left = there - piece * 16;
#pragma unroll 2
      for (int r = part * (32 / G) + lane / per; r < end; r += down) {
        uint4 x;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(place(r, piece)) : "memory");
        char* p = (char*)(out + r * ld + c0) + piece * 16;
        if (left >= 16) {
          *(uint4*)p = x;
        } else {
#pragma unroll
          for (int i = 0; i < 16 / (int)sizeof(O); i++)
            if ((i + 1) * (int)sizeof(O) <= left) ((O*)p)[i] = ((const O*)&x)[i];
        }
      }
    } else {
      const auto word = [&](int r, int w) {
        uint32_t v;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(place(r, w >> 2) + (w & 3) * 4) : "memory");
        return v;
      };
      char* row = (char*)(out + part * (32 / G) * ld + c0);
      if (there == LINE) {  // two words a lane
#pragma unroll 4
        for (int r = part * (32 / G); r < end; r++, row += ld * (int)sizeof(O)) {
          const uint32_t v = word(r, lane), u = word(r, lane + 32);
          if (sizeof(O) >= 4 || ((uintptr_t)row & 2) == 0) {
            ((uint32_t*)row)[lane] = v;
            ((uint32_t*)row)[lane + 32] = u;
          } else {  // the row starts in the middle of a word: the words are the upper half of one and the lower half of the next
            const uint32_t mid = __shfl_sync(0xffffffffu, u, 0);
            uint32_t nv = __shfl_down_sync(0xffffffffu, v, 1), nu = __shfl_down_sync(0xffffffffu, u, 1);
            if (lane == 31) nv = mid;
            uint32_t* q = (uint32_t*)(row + 2);
            q[lane] = __byte_perm(v, nv, 0x5432);
            if (lane < 31) q[lane + 32] = __byte_perm(u, nu, 0x5432);
            else *(uint16_t*)(q + 63) = (uint16_t)(u >> 16);
            if (lane == 0) *(uint16_t*)row = (uint16_t)v;
          }
        }
      } else {
        for (int r = part * (32 / G); r < end; r++, row += ld * (int)sizeof(O)) {
          if (sizeof(O) >= 4 || ((uintptr_t)row & 2) == 0) {
            for (int w = lane; 4 * w < there; w += 32) {
              if (4 * w + 4 <= there) *(uint32_t*)(row + 4 * w) = word(r, w);
              else *(uint16_t*)(row + 4 * w) = (uint16_t)word(r, w);
            }
          } else {
            if (lane == 0 && there > 0) *(uint16_t*)row = (uint16_t)word(r, 0);
            for (int w = lane; 4 * w + 2 < there; w += 32) {
              const uint32_t v = word(r, w);
              if (4 * w + 6 <= there) *(uint32_t*)(row + 4 * w + 2) = __byte_perm(v, word(r, w + 1), 0x5432);
              else *(uint16_t*)(row + 4 * w + 2) = (uint16_t)(v >> 16);
            }
          }
        }
      }
    }
    gm_group_sync(id, G * 32);
  }
}
// (sums as doubles: below the 32 bits that a number of 2^52 leaves, shifted to be positive; a conversion takes four times as long)
template <class O, class W>
__device__ __forceinline__ O gm_scaled(int32_t sum, W sa, W sb) {
  if constexpr (sizeof(O) == 8) return (__hiloint2double(0x43300000, sum ^ (int32_t)0x80000000) - (0x1p52 + 0x1p31)) * (double)sa * (double)sb;
  else return gm_cast<O>((float)sum * sa * sb);
}

// ---- large results --------------------------------------------------------------------------------------------------------
// Tile 256 x 256 per pair of CTAs (GATE: 256 x 128 of both products; narrower for few columns): each CTA holds the sums of its 128 rows and
// brings 128 rows and 128 columns of the operands, 32 KB a stage. One warp copies, one multiplies (the first CTA's, for both), eight or sixteen (gp_out) take the
// sums out of one half of tensor memory while the other fills. A launch's pairs take tiles in turn, along the rows within groups of GP_GROUP row tiles, so that what
// runs at once shares operands in L2.
constexpr int GP_STAGES = 10, GP_RING = 6 * 2 * GM_OPERAND, GP_GROUP = 8;

// Warps that take the sums out. GATE: 16, for the activation and the dropout of a tile keep eight busy for twice as long as its products take at a
// depth of 2048 (18 against 9 us: few instructions of a warp at a time are independent). 8 bits: 16 as well, for the conversions (8192 x 256 x 4097 to
// BF16 56 to 60 us, by eight 65; FP32 61 and 69). The others: eight (64 x 1024 x 4096: 11.3 us, by 16 12.6).
__host__ __device__ constexpr int gp_out(int kind) { return kind == GK_GATE || kind == GK_Q8 ? 16 : 8; }

__device__ __forceinline__ void gp_tile(const GemmArgs& A, int t, int& tm, int& tn) {
  const int per = GP_GROUP * A.tilesN, g = t / per, first = g * GP_GROUP, n = min(GP_GROUP, A.tilesM - first), r = t - g * per;
  tm = first + r % n;
  tn = r / n;
}

template <int KIND, class O>
__global__ void __launch_bounds__(128 + gp_out(KIND) * 32, 1) __cluster_dims__(2) k_gemm_pair(const __grid_constant__ GemmArgs A) {
  constexpr bool I8 = KIND == GK_Q8;
  constexpr int OUT = gp_out(KIND), G = OUT / 4;  // warps that write results, and of each 32 rows of a tile
  extern __shared__ __align__(1024) unsigned char gmsm[];
  __shared__ __align__(8) uint64_t full[GP_STAGES], empty[GP_STAGES], sumFull[2], sumRead[2], sumEmpty[2];
  __shared__ uint32_t tmemAt;
  const GemmCall& c = A.c;
  const int lane = threadIdx.x & 31, warp = gm_warp();
  const uint32_t rank = gm_rank(), smem = (gm_smem(gmsm) + 1023u) & ~1023u;
  const int pairs = gridDim.x / 2, pair = blockIdx.x / 2, tiles = A.tilesM * A.tilesN;
  const int segments = KIND == GK_SUM ? 2 : 1, nk = A.kBlocks * segments;
  const bool aMn = !I8 && c.a[0].mn, bMn = !I8 && c.b[0].mn;
  const int mine = KIND == GK_GATE ? A.wide : A.wide / 2, stages = A.stages;  // columns that a CTA brings
  const uint32_t stage = GM_OPERAND + mine * 128;
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(gm_smem(&tmemAt)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < GP_STAGES; i++) {
      gm_init(gm_smem(full + i), 1);
      gm_init(gm_smem(empty + i), 1);
    }
    for (int i = 0; i < 2; i++) {
      gm_init(gm_smem(sumFull + i), 1);
      gm_init(gm_smem(sumRead + i), OUT);
      gm_init(gm_smem(sumEmpty + i), 2);  // both CTAs
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  gm_cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmemAt;
  bool ok = true;
  const uint32_t fullAt = gm_smem(full), emptyAt = gm_smem(empty);
  if (c.after != AFTER_NONE) {
    gm_after_previous();
    gm_let_next();  // (not before: an AFTER_NONE kernel relies on the ones before this one)
  }
  if (warp == 0) {
    const uint32_t barAt = gm_peer(fullAt, 0);  // the first CTA's
    int s = 0, issued = 0;
    uint32_t ph = 1;
    for (int t = pair; t < tiles && ok; t += pairs) {
      int tm, tn;
      gp_tile(A, t, tm, tn);
      const int m0 = tm * 256 + rank * 128;
      const int halfN = A.tilesN / 2, which = KIND == GK_GATE ? (int)rank : KIND == GK_PAIR && tn >= halfN;
      const int n0 = KIND == GK_GATE ? tn * A.wide : (KIND == GK_PAIR && tn >= halfN ? tn - halfN : tn) * A.wide + rank * mine;
      for (int seg = 0; seg < segments && ok; seg++) {
        const CUtensorMap *ma = A.a + seg, *mb = A.b + (KIND == GK_SUM ? seg : which);
        for (int k0 = 0; k0 < A.kBlocks * A.depth; k0 += A.depth) {
          ok = gm_wait_all(emptyAt + s * 8, ph);
          if (!ok) break;
          const uint32_t bar = barAt + s * 8, da = smem + s * stage, db = da + GM_OPERAND;
          if (gm_elect()) {
            if (rank == 0) gm_expect(fullAt + s * 8, 2 * stage);
            if (aMn) {
              gm_load<true>(da, ma, m0, k0, bar);
              gm_load<true>(da + 8192, ma, m0 + 64, k0, bar);
            } else {
              gm_load<true>(da, ma, k0, m0, bar);
            }
            if (bMn) {
              gm_load<true>(db, mb, n0, k0, bar);
              if (mine > 64) gm_load<true>(db + 8192, mb, n0 + 64, k0, bar);
            } else {
              gm_load<true>(db, mb, k0, n0, bar);
            }
          }
          __syncwarp();
          issued++;
          if (++s == stages) s = 0, ph ^= 1;
        }
      }
    }
    gm_drain(ok, rank == 0, fullAt, emptyAt, issued, stages);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint64_t a0 = gm_desc(smem, aMn), b0 = gm_desc(smem + GM_OPERAND, bMn);
      const uint32_t da = gm_step(aMn), db = gm_step(bMn);
      int s = 0, n = 0;
      uint32_t ph = 0;
      for (int t = pair; t < tiles && ok; t += pairs, n++) {
        const int buf = n & 1;
        ok = gm_wait_all(gm_smem(sumEmpty + buf), ((n >> 1) & 1) ^ 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int kb = 0; kb < nk; kb++) {
          ok = gm_wait_all(fullAt + s * 8, ph);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t a = a0 + (uint32_t)s * (stage >> 4), b = b0 + (uint32_t)s * (stage >> 4);
          if (gm_elect()) {
#pragma unroll
            for (int i = 0; i < 4; i++) gm_mma<true, I8>(tmem + buf * 256, a + i * da, b + i * db, A.idesc, kb > 0 || i > 0);
            gm_commit<true>(emptyAt + s * 8);
            if (kb == nk - 1) gm_commit<true>(gm_smem(sumFull + buf));
          }
          __syncwarp();
          if (++s == stages) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == 3) {
    // Tells the first CTA that this one's sums have been read. Not a matter for the warps that read them: an arrival at another CTA waits for all that a
    // warp has written, which for their results took 2000 clocks a tile.
    int n = 0;
    for (int t = pair; t + 2 * pairs < tiles; t += pairs, n++) {  // (somebody waits for it: no arrival on its way when the CTAs end)
      const int buf = n & 1;
      ok = gm_wait_all(gm_smem(sumRead + buf), (n >> 1) & 1);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(gm_peer(gm_smem(sumEmpty + buf), 0)) : "memory");
      __syncwarp();
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, part = (warp - 4) >> 2;  // of the rows, of the columns
    int n = 0;
    for (int t = pair; t < tiles; t += pairs, n++) {
      const int buf = n & 1;
      ok = gm_group_all(1 + quarter, G * 32, gm_wait(gm_smem(sumFull + buf), (n >> 1) & 1));  // (together: they wait for one another below)
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      int tm, tn;
      gp_tile(A, t, tm, tn);
      const int64_t m0 = (int64_t)tm * 256 + rank * 128 + quarter * 32, m = m0 + lane;
      const int rows = (int)max((int64_t)0, min((int64_t)32, c.M - m0));
      const uint32_t at = tmem + buf * 256 + ((uint32_t)quarter << 21), room = smem + GP_RING + quarter * 8192;
      auto aligned = [&](int o) { return ((uintptr_t)c.out[o] | (uintptr_t)(c.ldo[o] * sizeof(O))) % 16 == 0; };
      if constexpr (KIND == GK_GATE) {
        const int64_t n0 = (int64_t)tn * A.wide;
        gm_rows<O, 8, G>((O*)c.out[0] + m0 * c.ldo[0] + n0, c.ldo[0], rows, c.N - n0, A.wide, aligned(0), room, part, 1 + quarter, [&](int j, O(&o)[8]) {
          uint32_t v[16];
          gm_tmem8(at + j, v);
          gm_tmem8(at + A.wide + j, v + 8);
          uint4 words[2];  // (while the sums come)
          if (c.drop.on) {
#pragma unroll
            for (int q = 0; q < 2; q++) words[q] = drop_words(c.drop, (uint32_t)m, (uint32_t)((n0 + j) / 4 + q));
          }
          gm_loaded(v);
          float h[8];
          with_act(c.act, [&](auto act) {
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = act_value(decltype(act)::value, __uint_as_float(v[i])) * __uint_as_float(v[8 + i]);
          });
          if (c.drop.on) {
#pragma unroll
            for (int q = 0; q < 8; q += 4) {
#pragma unroll
              for (int i = 0; i < 4; i++) h[q + i] = word_of(words[q / 4], i) >= c.drop.cut ? h[q + i] * c.drop.scale : 0.f;
            }
          }
#pragma unroll
          for (int i = 0; i < 8; i += 2) *(uint32_t*)(o + i) = to_word<O>(h[i], h[i + 1]);
        });
        if (c.out[1])
          for (int p = 0; p < 2; p++)
            gm_rows<O, 8, G>((O*)c.out[1 + p] + m0 * c.ldo[1 + p] + n0, c.ldo[1 + p], rows, c.N - n0, A.wide, aligned(1 + p), room, part, 1 + quarter,
                             [&](int j, O(&o)[8]) {
                               uint32_t v[8];
                               gm_tmem8(at + p * A.wide + j, v);
                               gm_loaded(v);
#pragma unroll
                               for (int i = 0; i < 8; i += 2) *(uint32_t*)(o + i) = to_word<O>(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                             });
      } else {
        const int halfN = A.tilesN / 2, which = KIND == GK_PAIR && tn >= halfN;
        const int64_t n0 = (int64_t)(which ? tn - halfN : tn) * A.wide;
        const float sa = I8 && m < c.M ? c.aScale[m] : 0.f;
        constexpr int CH = OUT == 16 ? 8 : 16;
        gm_rows<O, CH, G>((O*)c.out[which] + m0 * c.ldo[which] + n0, c.ldo[which], rows, c.N - n0, A.wide, aligned(which), room, part, 1 + quarter,
                          [&](int j, O(&o)[CH]) {
                            uint32_t v[CH];
                            if constexpr (CH == 8) gm_tmem8(at + j, v);
                            else gm_tmem16(at + j, v);
                            gm_loaded(v);
#pragma unroll
                            for (int i = 0; i < CH; i++) {
                              if constexpr (I8) o[i] = gm_scaled<O>((int32_t)v[i], sa, n0 + j + i < c.N ? __ldg(c.bScale + n0 + j + i) : 0.f);
                              else if constexpr (sizeof(O) == 2) {
                                if (i % 2 == 0) *(uint32_t*)(o + i) = to_word<O>(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                              } else o[i] = gm_cast<O>(__uint_as_float(v[i]));
                            }
                          });
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(gm_smem(sumRead + buf)) : "memory");
    }
  }
  if (c.after == AFTER_NONE) gm_after_previous();
  if (!ok) atomicExch(&denseErr, 201);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  gm_cluster_sync();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---- few rows -------------------------------------------------------------------------------------------------------------
// Tiles of 128 columns of the result (the lanes of tensor memory) by nc rows, so that little of the tensor cores' width is spent on rows that are
// not there; GATE: both weights' tiles in a stage, two sums. The stages of all tiles, one tile after the other, are dealt to the CTAs in even
// ranges (or in whole tiles, where that takes no longer). A CTA writes the results of the tiles that are its own alone; of a tile that it shares its
// sums go to the workspace, in its first room where its range starts in the tile, in its second where it ends there, and k_gemm_join
// adds them up in the order of the depth.
// The operand of the rows may come from the kernel before (quantised activations), whose end is waited for only where they are
// needed: the weights are on their way by then.
constexpr int GF_T = 256, GF_STAGES = 16, GF_RING = 220 * 1024;

// The first stage of CTA i's range; `whole`: of tiles. (of n stages in tiles of nk)
__host__ __device__ inline int gf_start(int i, int ctas, int n, int nk, bool whole) {
  return whole ? (int)((int64_t)(n / nk) * i / ctas) * nk : (int)((int64_t)n * i / ctas);
}

template <int KIND, class O>
__device__ __forceinline__ void gm_finish(const GemmCall& c, int which, int64_t m, int64_t n, uint32_t v0, uint32_t v1, float sa, float sb) {
  if constexpr (KIND == GK_Q8) {
    ((O*)c.out[0])[m * c.ldo[0] + n] = gm_scaled<O>((int32_t)v0, sa, sb);
  } else if constexpr (KIND == GK_GATE) {
    const float g = __uint_as_float(v0), u = __uint_as_float(v1);
    float h = act_value(c.act, g) * u;
    if (c.drop.on) h = word_of(drop_words(c.drop, (uint32_t)m, (uint32_t)(n / 4)), (int)(n & 3)) >= c.drop.cut ? h * c.drop.scale : 0.f;
    ((O*)c.out[0])[m * c.ldo[0] + n] = gm_cast<O>(h);
    if (c.out[1]) {
      ((O*)c.out[1])[m * c.ldo[1] + n] = gm_cast<O>(g);
      ((O*)c.out[2])[m * c.ldo[2] + n] = gm_cast<O>(u);
    }
  } else {
    ((O*)c.out[which])[m * c.ldo[which] + n] = gm_cast<O>(__uint_as_float(v0));
  }
}

// Tile t: its product (PAIR), first column and first row. Tiles of the same columns lie next to each other: their CTAs share the weights in L2.
template <int KIND>
__device__ __forceinline__ void gf_tile(const GemmArgs& A, int t, int& which, int& n0, int64_t& m0) {
  const int tn = t / A.tilesM;
  m0 = (int64_t)(t - tn * A.tilesM) * A.nc;
  which = KIND == GK_PAIR && tn >= A.tilesN / 2;
  n0 = (which ? tn - A.tilesN / 2 : tn) * 128;
}

// The scales of rows that the product quantises itself: behind the parts of the sums
__host__ __device__ inline int64_t gf_parts_bytes(int ctas, int np, int nc) { return (int64_t)ctas * 2 * np * nc * 128 * 4; }
__device__ __forceinline__ float* gf_scales(const GemmArgs& A) { return (float*)((char*)A.c.parts + gf_parts_bytes(A.ctas, 1, A.nc)); }

// X: the type of rows that the kernel quantises itself (void: they come in 8 bits), at most 16. The warps that write the results first find
// the rows' scales, every CTA for itself, and bring a stage's share of the rows where else the copying warp does: no kernel before, no
// copy of the rows in memory. One row of 4096 values: 1 us until the first stage, next to 4 us and a launch of the quantisation's own.
template <int KIND, class O, class X>
__global__ void __launch_bounds__(GF_T, 1) k_gemm_few(const __grid_constant__ GemmArgs A) {
  constexpr bool I8 = KIND == GK_Q8, OWN = !std::is_void_v<X>;
  constexpr int NP = KIND == GK_GATE ? 2 : 1;
  __shared__ float ownScale[16];
  __shared__ unsigned long long ownMost[16];
  extern __shared__ __align__(1024) unsigned char gmsm[];
  __shared__ __align__(8) uint64_t full[GF_STAGES], empty[GF_STAGES], sumFull[2], sumEmpty[2];
  __shared__ uint32_t tmemAt;
  const GemmCall& c = A.c;
  const int lane = threadIdx.x & 31, warp = gm_warp();
  const uint32_t smem = (gm_smem(gmsm) + 1023u) & ~1023u;
  const int nk = max(1, A.kBlocks * (KIND == GK_SUM ? 2 : 1));  // (a depth of zero: one stage that nothing is added from)
  const bool none = A.kBlocks == 0;
  const int n = A.tilesM * A.tilesN * nk, b0 = gf_start(blockIdx.x, gridDim.x, n, nk, A.whole), b1 = gf_start(blockIdx.x + 1, gridDim.x, n, nk, A.whole);
  const bool cMn = !I8 && c.a[0].mn, lMn = !I8 && c.b[0].mn;  // the result's rows and columns
  const uint32_t stage = NP * GM_OPERAND + A.nc * 128;
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(gm_smem(&tmemAt)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (OWN && threadIdx.x >= 128 && threadIdx.x < 144) ownMost[threadIdx.x - 128] = 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < A.stages; i++) {
      gm_init(gm_smem(full + i), OWN ? 2 : 1);  // the copies, and the warp that quantises
      gm_init(gm_smem(empty + i), 1);
    }
    for (int i = 0; i < 2; i++) {
      gm_init(gm_smem(sumFull + i), 1);
      gm_init(gm_smem(sumEmpty + i), 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmemAt;
  bool ok = true;
  const uint32_t fullAt = gm_smem(full), emptyAt = gm_smem(empty);
  if (warp == 0) {
    if (!none) {
      // the place of a stage in the tiles, kept from one to the next
      struct Place {
        int t, kb, which, n0;
        int64_t m0;
      };
      auto place = [&](int b) {
        Place p;
        p.t = b / nk;
        p.kb = b - p.t * nk;
        gf_tile<KIND>(A, p.t, p.which, p.n0, p.m0);
        return p;
      };
      auto next = [&](Place& p) {
        if (++p.kb == nk) {
          p.kb = 0;
          gf_tile<KIND>(A, ++p.t, p.which, p.n0, p.m0);
        }
      };
      // one lane's
      auto columns = [&](const Place& q, int s) {
        const int seg = KIND == GK_SUM && q.kb >= A.kBlocks, k0 = (q.kb - seg * A.kBlocks) * A.depth;
        const uint32_t bar = fullAt + s * 8, dl = smem + s * stage;
        gm_expect(bar, OWN ? NP * GM_OPERAND : stage);
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const CUtensorMap* ml = A.b + (KIND == GK_GATE ? p : KIND == GK_SUM ? seg : q.which);
          if (lMn) {
            gm_load<false>(dl + p * GM_OPERAND, ml, q.n0, k0, bar);
            gm_load<false>(dl + p * GM_OPERAND + 8192, ml, q.n0 + 64, k0, bar);
          } else {
            gm_load<false>(dl + p * GM_OPERAND, ml, k0, q.n0, bar);
          }
        }
      };
      auto rows = [&](const Place& q, int s) {
        const int seg = KIND == GK_SUM && q.kb >= A.kBlocks, k0 = (q.kb - seg * A.kBlocks) * A.depth;
        const uint32_t bar = fullAt + s * 8, dc = smem + s * stage + NP * GM_OPERAND;
        if (cMn) {
          gm_load<false>(dc, A.a + seg, (int)q.m0, k0, bar);
          if (A.nc > 64) gm_load<false>(dc + 8192, A.a + seg, (int)q.m0 + 64, k0, bar);
        } else {
          gm_load<false>(dc, A.a + seg, k0, (int)q.m0, bar);
        }
      };
      const int ahead = c.after == AFTER_A ? min(A.stages, b1 - b0) : 0;  // stages whose weights do not wait for the kernel before
      Place q = place(b0);
      for (int i = 0; i < ahead; i++) {
        if (gm_elect()) columns(q, i);
        __syncwarp();
        next(q);
      }
      if (c.after != AFTER_NONE) gm_after_previous();
      q = place(b0);
      int s = 0, issued = 0;
      uint32_t ph = 1;
      for (int b = b0; b < b1; b++) {
        const bool fresh = issued >= ahead;
        if (fresh) ok = gm_wait_all(emptyAt + s * 8, ph);
        if (!ok) break;
        if (gm_elect()) {
          if (fresh) columns(q, s);
          if (!OWN) rows(q, s);
        }
        __syncwarp();
        next(q);
        issued++;
        if (++s == A.stages) s = 0, ph ^= 1;
      }
      gm_drain(ok, true, fullAt, emptyAt, issued, A.stages);
    }
  } else if (warp == 1) {
    if (!none) {
      const uint64_t d0 = gm_desc(smem + NP * GM_OPERAND, cMn), l0 = gm_desc(smem, lMn);
      const uint32_t dd = gm_step(cMn), dl = gm_step(lMn);
      int s = 0, buf = 0;
      uint32_t ph = 0, phSum = 1;
      for (int b = b0; b < b1 && ok;) {
        const int first = b, end = min(b1, (b / nk + 1) * nk);  // of this tile's part of the range
        ok = gm_wait_all(gm_smem(sumEmpty + buf), phSum);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (; b < end; b++) {
          ok = gm_wait_all(fullAt + s * 8, ph);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t d = d0 + (uint32_t)s * (stage >> 4), l = l0 + (uint32_t)s * (stage >> 4);
          if (gm_elect()) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
              for (int p = 0; p < NP; p++)
                gm_mma<false, I8>(tmem + buf * 256 + p * A.nc, l + (p * GM_OPERAND >> 4) + i * dl, d + i * dd, A.idesc, b > first || i > 0);
            gm_commit<false>(emptyAt + s * 8);
            if (b == end - 1) gm_commit<false>(gm_smem(sumFull + buf));
          }
          __syncwarp();
          if (++s == A.stages) s = 0, ph ^= 1;
        }
        buf ^= 1;
        if (buf == 0) phSum ^= 1;
      }
    }
  } else if (warp >= 4) {
    if (c.after != AFTER_NONE) gm_after_previous();
    gm_let_next();  // (not before, see k_gemm_pair)
    const int quarter = warp - 4;
    int buf = 0, s = 0, turn = quarter;  // (the warps quantise stages in turn)
    uint32_t ph = 0, phStage = 1;
    using V = std::conditional_t<OWN, X, float>;
    using W = typename WideOf<V>::type;
    constexpr int P = DN_V<V>;
    if constexpr (OWN) {
      for (int r = 0; r < c.M; r++) {
        const V* p = (const V*)c.a[0].p + r * c.a[0].ld;
        decltype(magnitude(W())) most = 0;
#pragma unroll 4
        for (int k = (threadIdx.x - 128) * P; k < c.K; k += 128 * P) {
          alignas(16) V v[P];
          load_vec(p + k, (int)min((int64_t)P, c.K - k), false, v);
#pragma unroll
          for (int i = 0; i < P; i++) most = max(most, magnitude(widen(v[i])));
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
        if (lane == 0) atomicMax(ownMost + r, (unsigned long long)most);
      }
      gm_group_sync(1, 128);
      if (const int r = threadIdx.x - 128; r < c.M) {
        ownScale[r] = q8_scale((decltype(magnitude(W())))ownMost[r]);
        if (!A.whole && blockIdx.x == 0) gf_scales(A)[r] = ownScale[r];
      }
      gm_group_sync(1, 128);
    }
    for (int b = b0; b < b1;) {
      const int t = b / nk, end = min(b1, (t + 1) * nk);
      const bool mine = b == t * nk && end == (t + 1) * nk, head = b == b0;
      int which, n0;
      int64_t m0;
      gf_tile<KIND>(A, t, which, n0, m0);
      if constexpr (OWN) {
        for (int kb = b - t * nk; b < end; b++, kb++) {
          if (turn == 0) {
            ok = gm_wait_all(emptyAt + s * 8, phStage);
            if (!ok) break;
            for (int row = 0; row < c.M; row++) {  // four values a lane
              const int k0 = kb * 128 + lane * 4;
              const V* x = (const V*)c.a[0].p + row * c.a[0].ld + k0;
              const Q8Row<W> q8(ownScale[row]);
              W v[4];
              uint32_t o[4];
              bool near = !q8.quick;
#pragma unroll
              for (int j = 0; j < 4; j++) v[j] = k0 + j < c.K ? widen(x[j]) : (W)0;
#pragma unroll
              for (int j = 0; j < 4; j++) o[j] = q8.product(v[j], near);
              if (near) {
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = q8_quotient(v[j], q8.scale, q8.some);
              }
              const uint32_t w = __byte_perm(__byte_perm(o[0], o[1], 0x0040), __byte_perm(o[2], o[3], 0x0040), 0x5410);
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(smem + s * stage + NP * GM_OPERAND + row * 128 + (((lane >> 2) ^ (row & 7)) * 16) + (lane & 3) * 4),
                           "r"(w)
                           : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(fullAt + s * 8) : "memory");
          }
          turn = (turn + 3) & 3;
          if (++s == A.stages) s = 0, phStage ^= 1;
        }
        if (!ok) break;
      }
      if (!none) {
        ok = gm_wait(gm_smem(sumFull + buf), ph);
        if (!__all_sync(0xffffffffu, ok)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      const int rows = (int)min((int64_t)A.nc, c.M - m0);
      const int64_t col = n0 + quarter * 32 + lane;  // the lane's column of the result
      const float sb = I8 && col < c.N ? c.bScale[col] : 0.f;
      const uint32_t at = tmem + buf * 256 + ((uint32_t)quarter << 21);
      uint32_t* room = (uint32_t*)c.parts + ((int64_t)blockIdx.x * 2 + (head ? 0 : 1)) * NP * A.nc * 128 + quarter * 32 + lane;
#pragma unroll 1
      for (int r = 0; r < rows; r += 16) {
        uint32_t v[NP * 16];
#pragma unroll
        for (int p = 0; p < NP; p++) gm_tmem16(at + p * A.nc + r, v + 16 * p);
        gm_loaded(v);
        if (none) {
#pragma unroll
          for (int i = 0; i < NP * 16; i++) v[i] = 0;
        }
        if (col < c.N) {
#pragma unroll
          for (int i = 0; i < 16; i++) {
            if (r + i >= rows) break;
            if (mine) {
              gm_finish<KIND, O>(c, which, m0 + r + i, col, v[i], v[16 * (NP - 1) + i], OWN ? ownScale[r + i] : I8 ? c.aScale[m0 + r + i] : 0.f, sb);
            } else {
#pragma unroll
              for (int p = 0; p < NP; p++) room[(p * A.nc + r + i) * 128] = v[16 * p + i];
            }
          }
        }
        __syncwarp();
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0 && !none) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(gm_smem(sumEmpty + buf)) : "memory");
      buf ^= 1;
      if (buf == 0) ph ^= 1;
      b = end;
    }
  }
  if (c.after == AFTER_NONE) gm_after_previous();
  if (!ok) atomicExch(&denseErr, 202);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Tiles that several CTAs share: their sums, added up in the order of the depth, and the epilogue. A CTA per tile and row, a thread per column.
template <int KIND, class O>
__global__ void __launch_bounds__(128) k_gemm_join(const __grid_constant__ GemmArgs A) {
  constexpr bool I8 = KIND == GK_Q8;
  constexpr int NP = KIND == GK_GATE ? 2 : 1;
  const GemmCall& c = A.c;
  const int nk = A.kBlocks * (KIND == GK_SUM ? 2 : 1);
  const int t = blockIdx.x, n = A.tilesM * A.tilesN * nk;
  int which, n0;
  int64_t m0;
  gf_tile<KIND>(A, t, which, n0, m0);
  // the CTAs that hold the tile's first and last stage: start(i) <= stage < start(i + 1)
  auto holder = [&](int b) { return (int)(((int64_t)(b + 1) * A.ctas - 1) / n); };
  const int first = holder(t * nk), last = holder(t * nk + nk - 1);
  gm_after_previous();
  if (first == last) return;
  const int64_t col = n0 + threadIdx.x;
  if (col >= c.N) return;
  const float sb = I8 ? c.bScale[col] : 0.f;
  const float* aScale = c.quantize ? gf_scales(A) : c.aScale;
  // the first CTA's range starts in this tile or before it, the others' in it
  const int64_t room = (int64_t)NP * A.nc * 128;
  const int64_t head = (int64_t)first * 2 + (gf_start(first, A.ctas, n, nk, false) < t * nk);
  for (int r = blockIdx.y; r < A.nc && m0 + r < c.M; r += gridDim.y) {
    const uint32_t* at = (const uint32_t*)c.parts + r * 128 + threadIdx.x;
    uint32_t u = at[head * room];
    float f[2];
#pragma unroll
    for (int p = 0; p < NP; p++) f[p] = __uint_as_float(at[head * room + p * A.nc * 128]);
#pragma unroll 8
    for (int q = first + 1; q <= last; q++) {
      if (I8) u += at[q * 2 * room];
      else
#pragma unroll
        for (int p = 0; p < NP; p++) f[p] += __uint_as_float(at[q * 2 * room + p * A.nc * 128]);
    }
    gm_finish<KIND, O>(c, which, m0 + r, col, I8 ? u : __float_as_uint(f[0]), __float_as_uint(f[NP - 1]), I8 ? aScale[m0 + r] : 0.f, sb);
  }
}

// ---- few columns ----------------------------------------------------------------------------------------------------------
// Products of rows that are quantised on the way, for so few columns that a CTA holds all of the weights: the rows come from memory once and in
// nothing but their own type, with no copy of them in 8 bits. A CTA takes an even range of the rows, its sixteen warps one row after another each: a
// warp brings its next rows to its own places of shared memory, by copies of the 16-byte pieces that hold a row (it may start anywhere; copying them for all
// warps, one lane was busy for 200 clocks a row and took longest), finds the scale, and puts the 8-bit values where the products read them, 128 rows a
// tile. Then come the tile's products, which take a twentieth of the time, and all warps write the results while the next rows are on their way.
// Bound: memory next to the instructions of the quantisation (100,003 rows of 501 values, 64 columns: FP64 85 us, 5.3 TB/s; FP32 57 us, BF16 66 us, where
// the issue slots are 55 % busy).
constexpr int GR_WARPS = 16, GR_T = GR_WARPS * 32, GR_SLOTS = 128, GR_ROOM = 223 * 1024;
// Blocks of a row's depth up to which a warp takes two rows at once
constexpr int gr_pairs(int bytes) { return bytes == 8 ? 2 : 4; }
struct RowsPlan {
  int kb, wide, slot, slots;  // blocks of the depth; columns with those that are not there; bytes of a row in the ring, rows
  bool fits = false;
};
static RowsPlan rows_plan(int64_t N, int64_t K, int type) {
  RowsPlan p;
  if (N > 256 || K <= 0 || K > 2048) return p;
  p.kb = (int)(K + 127) / 128;
  p.wide = 32;
  while (p.wide < N) p.wide *= 2;
  p.slot = (int)round_up(K * type_bytes(type), 16) + 16;
  const int left = GR_ROOM - 1024 - std::max(p.kb * (int)GM_OPERAND, 4 * 8192) - p.kb * p.wide * 128;
  p.slots = left > 0 ? std::min(GR_SLOTS, left / p.slot / GR_WARPS * GR_WARPS) : 0;
  // one place a warp is enough where a row takes long to come: 100,003 x 640 FP64, 64 columns 119 us, by two kernels 174, FP32 x 700 99 and 117; 16 bits x 1000,
  // 16 columns 130 and 117
  const int least = type_bytes(type) > 2 && p.kb > gr_pairs(type_bytes(type)) ? 1 : 2;
  p.fits = p.slots == GR_SLOTS || (p.slots >= least * GR_WARPS && p.slots * p.slot >= 24 << 10);
  return p;
}

__device__ __forceinline__ uint32_t gr_most(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ unsigned long long gr_most(unsigned long long v) {
  const uint32_t hi = (uint32_t)(v >> 32), most = __reduce_max_sync(0xffffffffu, hi);
  return (unsigned long long)most << 32 | __reduce_max_sync(0xffffffffu, hi == most ? (uint32_t)v : 0u);
}

// ROWS: how many rows a warp takes at once (of a row alone one operation waits for another most of the time: 100,003 FP64 rows of 100 values, 64
// columns: 49 us, one at a time 55; longer ones of FP64 leave the memory less to do meanwhile). KEPT: blocks of a row that stay in registers, all of
// them or none (the row is then read a second time).
template <class X, int ROWS, int KEPT>
__global__ void __launch_bounds__(GR_T, 1) k_gemm_rows(const __grid_constant__ GemmArgs A) {
  using W = typename WideOf<X>::type;
  extern __shared__ __align__(1024) unsigned char gmsm[];
  __shared__ __align__(8) uint64_t full[GR_SLOTS], bFull, sumFull;
  __shared__ float scale[128];
  __shared__ W columns[256];  // the columns' scales
  __shared__ uint32_t tmemAt;
  const GemmCall& c = A.c;
  const int lane = threadIdx.x & 31, warp = gm_warp(), kbs = A.kBlocks, wide = A.wide, slots = A.stages, slot = A.nc;
  const uint32_t smem = (gm_smem(gmsm) + 1023u) & ~1023u, atB = smem + max(kbs * (int)GM_OPERAND, 4 * 8192), ring = atB + kbs * wide * 128;
  const int64_t r0 = c.M * blockIdx.x / gridDim.x;
  const int rows = (int)(c.M * (blockIdx.x + 1) / gridDim.x - r0);
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(gm_smem(&tmemAt)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < slots; i++) gm_init(gm_smem(full + i), 1);
    gm_init(gm_smem(&bFull), 1);
    gm_init(gm_smem(&sumFull), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmemAt, fullAt = gm_smem(full);
  bool ok = true;
  const auto row = [&](int i) { return (const X*)c.a[0].p + (r0 + i) * c.a[0].ld; };
  const auto bring = [&](int i, int s) {  // (all lanes)
    if (i < rows && gm_elect()) {
      const uintptr_t first = (uintptr_t)row(i), from = first & ~(uintptr_t)15;
      const uint32_t bytes = (uint32_t)(((first + c.K * sizeof(X) + 15) & ~(uintptr_t)15) - from);
      gm_expect(fullAt + s * 8, bytes);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ring + s * slot), "l"(from), "r"(bytes),
                   "r"(fullAt + s * 8)
                   : "memory");
    }
    __syncwarp();
  };
  for (int i = warp; i < slots; i += GR_WARPS) bring(i, i);
  if (warp == 0) {
    if (gm_elect()) {
      gm_expect(gm_smem(&bFull), kbs * wide * 128);
      for (int kb = 0; kb < kbs; kb++) gm_load<false>(atB + kb * wide * 128, A.b, kb * 128, 0, gm_smem(&bFull));
    }
    __syncwarp();
  }
  if (threadIdx.x < wide) columns[threadIdx.x] = threadIdx.x < c.N ? (W)c.bScale[threadIdx.x] : (W)0;
  const unsigned char* ringAt = gmsm + (ring - gm_smem(gmsm));
  int at = warp, place = warp;  // the warp's row, and where it is
  uint32_t turn = 0;
  const int left = (int)c.K - lane;
  // The warp's next R rows, side by side
  const auto take = [&](auto count, int t0) {
    constexpr int R = decltype(count)::value;
    const X* x[R];
    int from[R];
    uint32_t to[R], swizzle[R];
    decltype(magnitude(W())) most[R];
    const uint32_t half = lane >> 4;
    int p = place;
    uint32_t parity = turn;
#pragma unroll
    for (int q = 0; q < R; q++) {
      if (!gm_wait_all(fullAt + p * 8, parity)) return false;
      const int i = at + q * GR_WARPS, r = i - t0;
      x[q] = (const X*)(ringAt + p * slot + ((uintptr_t)row(i) & 15)) + lane;
      from[q] = p;
      to[q] = smem + r * 128 + (lane & 15), swizzle[q] = r & 7;
      most[q] = 0;
      p += GR_WARPS;
      if (p >= slots) p = warp, parity ^= 1;
    }
    const auto load = [&](int q, int kb, W(&v)[4]) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        v[j] = kb * 128 + j * 32 < left ? widen(x[q][kb * 128 + j * 32]) : (W)0;
        most[q] = max(most[q], magnitude(v[j]));
      }
    };
    const auto store = [&](int q, const Q8Row<W>& q8, int kb, const W(&v)[4]) {
      uint32_t o[4];
      bool near = !q8.quick;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = q8.product(v[j], near);
      if (near) q8_quotients<X>(q8, v, o);
#pragma unroll
      for (int j = 0; j < 4; j++)
        asm volatile("st.shared.u8 [%0], %1;" ::"r"(to[q] + kb * GM_OPERAND + ((2 * j + half) ^ swizzle[q]) * 16), "r"(o[j]) : "memory");
    };
    W v[R][KEPT ? KEPT : 1][4];
    if constexpr (KEPT > 0) {
#pragma unroll
      for (int kb = 0; kb < KEPT; kb++)
#pragma unroll
        for (int q = 0; q < R; q++)
          if (kb < kbs) load(q, kb, v[q][kb]);
    } else {
#pragma unroll 2
      for (int kb = 0; kb < kbs; kb++) load(0, kb, v[0][0]);
    }
#pragma unroll
    for (int q = 0; q < R; q++) most[q] = gr_most(most[q]);  // (of values that all lanes have read)
    if constexpr (KEPT > 0)
#pragma unroll
      for (int q = 0; q < R; q++) bring(at + q * GR_WARPS + slots, from[q]);
    float sc[R];
#pragma unroll
    for (int q = 0; q < R; q++) sc[q] = q8_scale(most[q]);
#pragma unroll
    for (int q = 0; q < R; q++) {
      if (lane == 0) scale[at + q * GR_WARPS - t0] = sc[q];
      const Q8Row<W> q8(sc[q]);
      if constexpr (KEPT > 0) {
#pragma unroll
        for (int kb = 0; kb < KEPT; kb++)
          if (kb < kbs) store(q, q8, kb, v[q][kb]);
      } else {
#pragma unroll 2
        for (int kb = 0; kb < kbs; kb++) {
          load(0, kb, v[0][0]);
          store(0, q8, kb, v[0][0]);
        }
        __syncwarp();
        bring(at + slots, from[0]);
      }
    }
    at += R * GR_WARPS, place = p, turn = parity;
    return true;
  };
  {
    const int quarter = warp & 3;
    const uint64_t da = gm_desc(smem, false), db = gm_desc(atB, false);
    uint32_t ph = 0;
    for (int t0 = 0; t0 < rows; t0 += 128, ph ^= 1) {
      const int n = min(128, rows - t0);
      while (ok && at < t0 + n) {
        if (ROWS == 2 && at + GR_WARPS < t0 + n) ok = take(std::integral_constant<int, ROWS>(), t0);
        else ok = take(std::integral_constant<int, 1>(), t0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      ok = gm_group_all(1, GR_T, ok);
      if (!ok) break;
      if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        ok = gm_wait_all(gm_smem(&bFull), 0);
        if (ok && gm_elect()) {
          for (int kb = 0; kb < kbs; kb++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              gm_mma<false, true>(tmem, da + (kb * GM_OPERAND >> 4) + i * gm_step(false), db + (kb * wide * 128 >> 4) + i * gm_step(false), A.idesc, kb > 0 || i > 0);
          gm_commit<false>(gm_smem(&sumFull));
        }
        __syncwarp();
      }
      ok = gm_wait_all(gm_smem(&sumFull), ph) && ok;
      ok = gm_group_all(1, GR_T, ok);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int64_t m0 = r0 + t0 + quarter * 32;
      const W sa = scale[quarter * 32 + lane];
      const bool aligned = ((uintptr_t)c.out[0] | (uintptr_t)(c.ldo[0] * sizeof(X))) % 16 == 0;
      gm_rows<X, 8, GR_WARPS / 4>((X*)c.out[0] + m0 * c.ldo[0], c.ldo[0], max(0, min(32, n - quarter * 32)), c.N, wide, aligned, smem + quarter * 8192, warp >> 2,
                                  2 + quarter, [&](int j, X(&o)[8]) {
                                    uint32_t v[8];
                                    gm_tmem8(tmem + ((uint32_t)quarter << 21) + j, v);
                                    gm_loaded(v);
#pragma unroll
                                    for (int i = 0; i < 8; i++) o[i] = gm_scaled<X>((int32_t)v[i], sa, columns[j + i]);
                                  });
      gm_group_sync(1, GR_T);  // (the results passed through the tile's place)
    }
  }
  if (!ok) {  // the copies that are on their way
    for (int i = at; i < min(rows, at + slots); i += GR_WARPS) gm_wait_all(fullAt + i % slots * 8, i / slots & 1);
    gm_wait_all(gm_smem(&bFull), 0);
  }
  if (!ok) atomicExch(&denseErr, 203);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
int64_t dense_status(int device) {
  (void)device;
  int32_t e = 0, zero = 0;
  CLA_CUDA(cudaDeviceSynchronize());  // (the copy itself waits for no stream that was made not to)
  CLA_CUDA(cudaMemcpyFromSymbol(&e, denseErr, sizeof(e)));
  if (!e) return CLA_OK;
  CLA_CUDA(cudaMemcpyToSymbol(denseErr, &zero, sizeof(zero)));
  return fail(CLA_ERR_DEVICE_CHECK, "a dense product's self-check tripped (code " + std::to_string(e) + ")");
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
  static EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? (EncodeTiled)p
               : nullptr;
  }();
  return f;
}
// An operand of `count` indexes and depth k, in boxes of `box` indexes (index contiguous: always 64) and a stage's depth
static int64_t operand_map(CUtensorMap& map, const GemmOperand& o, int type, int64_t count, int64_t k, int box) {
  EncodeTiled enc = encode_tiled();
  if (!enc) return fail(CLA_ERR_CUDA, "dense product: the driver has no tensor maps");
  const int bytes = type_bytes(type);
  const cuuint64_t dims[2] = {(cuuint64_t)(o.mn ? count : k), (cuuint64_t)(o.mn ? k : count)}, stride[1] = {(cuuint64_t)(o.ld * bytes)};
  const cuuint32_t boxes[2] = {o.mn ? 64u : 128u / bytes, o.mn ? 64u : (cuuint32_t)box}, ones[2] = {1, 1};
  const CUtensorMapDataType t =
      type == CLA_T_I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == CLA_T_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = enc(&map, t, 2, (void*)o.p, dims, stride, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? CLA_OK : fail(CLA_ERR_CUDA, "dense product: tensor map refused (" + std::to_string((int)r) + ")");
}

// All of an SM's shared memory for a CTA, as it takes all of its tensor memory: CTAs that wait for tensor memory while others wait for
// them could hold up one another. room: how much it is, where the caller wants to know (threads that meet write the same)
template <class K>
static int64_t all_smem(OncePerDevice& once, std::atomic<int>* room, int device, K kernel) {
  return once(device, [&]() -> int64_t {
    cudaFuncAttributes a;
    CLA_CUDA(cudaFuncGetAttributes(&a, kernel));
    const int most = 227 * 1024 - (int)a.sharedSizeBytes;  // of a CTA; 1 KB more is kept for it
    CLA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    if (room) room->store(most, std::memory_order_relaxed);
    return CLA_OK;
  });
}

// Which kernel and tile: the one that an estimate in microseconds makes the fastest. For 148 SMs: the workspace does not depend on the device.
struct GemmPlan {
  bool large = false;
  int wide = 0;                      // k_gemm_pair
  int nc = 0, ctas = 0, stages = 1;  // k_gemm_few
  bool whole = true;
  double us = 1e30;
};
constexpr int GM_SMS = 148;
static int gemm_blocks(const GemmCall& c) {  // stages of a segment
  const int depth = 128 / type_bytes(c.type);
  return (int)((c.K + depth - 1) / depth);
}
bool gemm_quantizes(int64_t M, int64_t K, int type) { return M <= 16 && K > 0 && M * K * type_bytes(type) <= 32 << 10; }

// (16 rows and fewer: k_gemm_few, with the columns over all SMs. FP32, 300 values a row, 128 columns: 1000 rows in 10.7 us a call and 7.7 us of the
// device's, quantised by a kernel of their own 15.4 and 6.6; 6000 rows 9.5 and 9.6 us of the device's; FP64, 200 values, 256 columns: 1000 rows 12.4 and
// 6.6 us, 6000 rows 14.5 and 15.9. 100,003 FP64 rows of 501 values, 64 columns: 85 and 130 us.)
bool gemm_scores(int64_t M, int64_t N, int64_t K, int type) { return M > 16 && (N <= 128 || M >= 4096) && rows_plan(N, K, type).fits; }

static GemmPlan find_plan(const GemmCall& c) {
  GemmPlan best;
  const int nk = gemm_blocks(c) * (c.kind == GK_SUM ? 2 : 1);
  const int np = c.kind == GK_GATE ? 2 : 1, products = c.kind == GK_PAIR ? 2 : 1;
  const auto ceil_div = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  // The terms were measured over 1 to 2048 rows, 1000 to 16384 columns, depths of 500 to 5504, weights not in L2 (both sides of every
  // choice; the choice was the fastest or within a tenth of it in nine of ten). What the operands take from memory at 6.2 GB a ms:
  const double memory = (double)type_bytes(c.type) * c.K * (c.kind == GK_SUM ? 2 : 1) * (c.M + c.N * (c.kind == GK_Q8 ? 1 : 2)) / 6.2e6;
  // k_gemm_pair: a stage takes 0.17 us (waits and issue) or its products' time, 4 clocks a column that a CTA brings, at 1.85 GHz; a tile's results
  // leave in 12 ns a column while the next tile's come
  // (32 rows and fewer leave its copies of them nearly empty, which take up to twice the time: not for deep products of so few)
  for (int wide = 256 / np; wide >= 64 && nk > 0 && (c.M > 32 || nk <= 8) && !c.quantize; wide /= 2) {
    const int mine = np == 2 ? wide : wide / 2;
    if (c.b[0].mn && mine < 64) break;
    const int64_t tiles = ceil_div(c.M, 256) * ceil_div(c.N, wide) * products, turns = ceil_div(tiles, GM_SMS / 2);
    const double out = wide * np * 0.012, chain = nk * std::max(0.17, 4 * mine / 1850.0) + 0.5;
    const double t = 7.0 + std::max(memory, turns * std::max(chain, out)) + out;
    if (t < best.us) best.large = true, best.wide = wide, best.us = t;
  }
  // k_gemm_few: a stage takes 0.24 us (two products 0.32), more with more rows; all SMs' stages together come at 10 GB a ms. A row of results
  // leaves in 50 ns a product, of sums to be joined in 10, and joining costs a second kernel that moves the sums at 4 GB a ms
  // (two products: never the faster one for more than 32 rows)
  for (int nc = 16; nc <= 128; nc *= 2) {
    const int least = c.a[0].mn ? 64 : 16;
    if (nc < least || (best.large && c.M > 32 && c.kind != GK_Q8 && c.kind != GK_SUM)) continue;
    if (nc > least && nc / 2 >= c.M) break;
    const int stage = np * (int)GM_OPERAND + nc * 128;
    const int64_t tiles = ceil_div(c.M, nc) * ceil_div(c.N, 128) * products, n = tiles * std::max(1, nk);
    if (n > INT32_MAX / 2) continue;  // (counted in 32 bits)
    const double step = (np == 2 ? 0.32 : 0.24) + nc * np * 0.0012;
    for (int whole = 1; whole >= (c.split && nk > 0 ? 0 : 1); whole--) {
      const int64_t ctas = whole ? std::min<int64_t>(tiles, GM_SMS) : std::min<int64_t>(GM_SMS, tiles * ceil_div(nk, 4));
      const double out = 0.2 + std::min<int64_t>(nc, c.M) * np * (whole ? 0.05 : 0.01);
      const double chain = whole ? ceil_div(tiles, ctas) * std::max(nk * step, out) : ceil_div(n, ctas) * step;
      const double join = 4.0 + (double)tiles * std::min<int64_t>(nc, c.M) * np * 512 * 2.5 / 4.0e6;
      const double t = 5.5 + std::max({memory, chain, (double)n * stage / 10.0e6}) + out + (whole ? 0.0 : join);
      if (t >= best.us) continue;
      best.large = false, best.nc = nc, best.ctas = (int)ctas, best.whole = whole, best.us = t;
      best.stages = (int)std::min<int64_t>(GF_STAGES, GF_RING / stage);
    }
  }
  return best;
}
// A call asks for its plan three times, and programs ask for the same sizes again: the last few are kept, by all that they depend on
static GemmPlan gemm_plan(const GemmCall& c) {
  struct Kept {
    int64_t M = -1, N, K;
    int how;
    GemmPlan plan;
  };
  static thread_local Kept kept[16];
  const int how = (int)c.kind * 64 + (c.type == CLA_T_I8) * 32 + c.split * 16 + c.quantize * 8 + c.a[0].mn * 4 + c.b[0].mn * 2;
  Kept& k = kept[(uint64_t)(c.M * 31 + c.N * 7 + c.K * 3 + how) % 16];
  if (k.M != c.M || k.N != c.N || k.K != c.K || k.how != how) k = {c.M, c.N, c.K, how, find_plan(c)};
  return k.plan;
}
int64_t gemm_workspace(const GemmCall& c) {
  if (c.M == 0 || c.N == 0 || c.scores) return 0;
  const GemmPlan p = gemm_plan(c);
  return p.large || p.whole ? 0 : gf_parts_bytes(p.ctas, c.kind == GK_GATE ? 2 : 1, p.nc) + 64;
}

template <int KIND, class O>
static int64_t launch_kind(GemmArgs& A, cudaStream_t s) {
  const GemmCall& c = A.c;
  A.depth = 128 / type_bytes(c.type);
  A.kBlocks = gemm_blocks(c);
  const GemmPlan p = gemm_plan(c);
  // both operands' types, where their index is contiguous, sums in 32 bits
  const uint32_t type = c.type == CLA_T_BF16 || c.type == CLA_T_I8 ? 1u : 0u;
  const uint32_t base = (KIND == GK_Q8 ? 2u : 1u) << 4 | type << 7 | type << 10;
  if (A.kBlocks > 0)
    for (int i = 0; i < 2; i++) {
      const int boxB = !p.large ? 128 : KIND == GK_GATE ? p.wide : p.wide / 2;
      if ((i == 0 || KIND == GK_SUM) && !c.quantize)
        if (const int64_t rc = operand_map(A.a[i], c.a[i], c.type, c.M, c.K, p.large ? 128 : p.nc); rc < 0) return rc;
      if (i == 0 || KIND != GK_Q8)
        if (const int64_t rc = operand_map(A.b[i], c.b[i], c.type, c.N, c.K, boxB); rc < 0) return rc;
    }
  const int np = KIND == GK_GATE ? 2 : 1, products = KIND == GK_PAIR ? 2 : 1;
  static OncePerDevice oncePair, onceFew;
  static std::atomic<int> roomPair;
  if (p.large) {
    A.wide = p.wide;
    A.stages = std::min(GP_STAGES, GP_RING / ((int)GM_OPERAND + (KIND == GK_GATE ? p.wide : p.wide / 2) * 128));
    A.tilesM = (int)((c.M + 255) / 256);
    A.tilesN = (int)((c.N + p.wide - 1) / p.wide) * products;
    A.idesc = base | (uint32_t)c.a[0].mn << 15 | (uint32_t)c.b[0].mn << 16 | (uint32_t)(p.wide * np >> 3) << 17 | (256u >> 4) << 24;
    if (const int64_t e = all_smem(oncePair, &roomPair, c.device, k_gemm_pair<KIND, O>); e < 0) return e;
    static_assert(GP_RING + 1024 + 8 * 4096 <= 226 * 1024, "the ring and the warps' rooms fit");
    const unsigned ctas = 2 * (unsigned)std::min<int64_t>((int64_t)A.tilesM * A.tilesN, GM_SMS / 2);
    EarlyLaunch pair(ctas, 128 + gp_out(KIND) * 32, roomPair.load(std::memory_order_relaxed), s, c.after != AFTER_CALL);
    CLA_CUDA(cudaLaunchKernelEx(&pair.cfg, k_gemm_pair<KIND, O>, A));
    return CLA_OK;
  }
  A.nc = p.nc;
  A.stages = p.stages;
  A.ctas = p.ctas;
  A.whole = p.whole;
  A.tilesM = (int)((c.M + A.nc - 1) / A.nc);
  A.tilesN = (int)((c.N + 127) / 128) * products;
  A.idesc = base | (uint32_t)c.b[0].mn << 15 | (uint32_t)c.a[0].mn << 16 | (uint32_t)(A.nc >> 3) << 17 | (128u >> 4) << 24;
  static_assert(GF_RING + 1024 <= 226 * 1024, "the ring fits");
  const auto few = [&](auto kernel, OncePerDevice& once) -> int64_t {
    if (const int64_t e = all_smem(once, nullptr, c.device, kernel); e < 0) return e;
    // (all but 5 KB: CTAs of k_gemm_join may wait next to it, none with tensor memory)
    EarlyLaunch l(p.ctas, GF_T, GF_RING + 1024, s, c.after != AFTER_CALL);
    CLA_CUDA(cudaLaunchKernelEx(&l.cfg, kernel, A));
    return CLA_OK;
  };
  int64_t rc;
  if constexpr (KIND == GK_Q8) {
    static OncePerDevice onceOwn;
    rc = c.quantize ? few(k_gemm_few<KIND, O, O>, onceOwn) : few(k_gemm_few<KIND, O, void>, onceFew);
  } else {
    rc = few(k_gemm_few<KIND, O, void>, onceFew);
  }
  if (rc < 0) return rc;
  if (!p.whole) {
    static OncePerDevice onceJoin;
    if (const int64_t e = onceJoin(c.device, [] { return like_products(k_gemm_join<KIND, O>); }); e < 0) return e;
    EarlyLaunch join(dim3((unsigned)A.tilesM * A.tilesN, (unsigned)std::min<int64_t>(c.M, A.nc)), 128, 0, s, true);
    CLA_CUDA(cudaLaunchKernelEx(&join.cfg, k_gemm_join<KIND, O>, A));
  }
  return CLA_OK;
}

template <class X>
static int64_t launch_rows(GemmArgs& A, cudaStream_t s) {
  const GemmCall& c = A.c;
  const RowsPlan p = rows_plan(c.N, c.K, c.outType);
  A.kBlocks = p.kb, A.wide = p.wide, A.nc = p.slot, A.stages = p.slots;
  A.idesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(p.wide >> 3) << 17 | (128u >> 4) << 24;
  if (const int64_t rc = operand_map(A.b[0], c.b[0], CLA_T_I8, c.N, c.K, p.wide); rc < 0) return rc;
  const auto go = [&](auto kernel, OncePerDevice& once) -> int64_t {
    if (const int64_t e = all_smem(once, nullptr, c.device, kernel); e < 0) return e;
    EarlyLaunch l((unsigned)std::min<int64_t>(GM_SMS, (c.M + GR_WARPS - 1) / GR_WARPS), GR_T, GR_ROOM, s, false);
    CLA_CUDA(cudaLaunchKernelEx(&l.cfg, kernel, A));
    return CLA_OK;
  };
  static OncePerDevice once[3];
  if (p.kb <= 2) return go(k_gemm_rows<X, 2, 2>, once[0]);
  if (p.kb <= 4) return go(k_gemm_rows<X, gr_pairs(sizeof(X)) == 4 ? 2 : 1, 4>, once[1]);
  return go(k_gemm_rows<X, 1, 0>, once[2]);
}

int64_t launch_gemm(const GemmCall& c, cudaStream_t s) {
  if (c.M == 0 || c.N == 0) return CLA_OK;
  GemmArgs A = {};
  A.c = c;
  if (c.scores) {
    if (c.outType == CLA_T_F64) return launch_rows<double>(A, s);
    if (c.outType == CLA_T_F32) return launch_rows<float>(A, s);
    if (c.outType == CLA_T_BF16) return launch_rows<__nv_bfloat16>(A, s);
    return launch_rows<__half>(A, s);
  }
  if (c.kind == GK_Q8) {
    if (c.outType == CLA_T_F64) return launch_kind<GK_Q8, double>(A, s);
    if (c.outType == CLA_T_F32) return launch_kind<GK_Q8, float>(A, s);
    if (c.outType == CLA_T_BF16) return launch_kind<GK_Q8, __nv_bfloat16>(A, s);
    return launch_kind<GK_Q8, __half>(A, s);
  }
  const bool bf = c.type == CLA_T_BF16;
  if (c.kind == GK_GATE) return bf ? launch_kind<GK_GATE, __nv_bfloat16>(A, s) : launch_kind<GK_GATE, __half>(A, s);
  if (c.kind == GK_SUM) return bf ? launch_kind<GK_SUM, __nv_bfloat16>(A, s) : launch_kind<GK_SUM, __half>(A, s);
  return bf ? launch_kind<GK_PAIR, __nv_bfloat16>(A, s) : launch_kind<GK_PAIR, __half>(A, s);
}

}  // namespace cla
