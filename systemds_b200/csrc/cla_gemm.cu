// Products of dense operands in 8 and 16 bits with their epilogues (GemmCall of cla_dense.cuh), on the 5th-generation tensor cores: operands by
// TMA into 128-byte-swizzled shared memory, sums in tensor memory (FP32, or 32-bit integers for 8-bit operands), epilogues from there.
//  * k_gemm_pair: two CTAs share a 256 x 256 tile. For large results.
//  * k_gemm_few: one CTA per 128 columns of the result and 16 to 128 of its rows, the depth split over a cluster. For few rows.
#include <cuda.h>
#include <algorithm>
#include "cla_dense.cuh"

namespace cla {

static __device__ int32_t denseErr;

// ---- PTX ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t gm_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t gm_now() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool gm_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done)
               : "r"(bar), "r"(parity)
               : "memory");
  return done != 0;
}
// Gives up after GM_LIMIT ns: far longer than any launch, so that a mistake ends as an error and not as a hung GPU
constexpr uint64_t GM_LIMIT = 8000000000ull;
__device__ __noinline__ bool gm_wait_long(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = gm_now();
  do {
    for (int i = 0; i < 64; i++)
      if (gm_try(bar, parity)) return true;
  } while (gm_now() - t0 < GM_LIMIT);
  return false;
}
__device__ __forceinline__ bool gm_wait(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < 32; i++)
    if (gm_try(bar, parity)) return true;
  return gm_wait_long(bar, parity);
}
__device__ __forceinline__ uint32_t gm_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t gm_peer(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void gm_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
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
template <int N>
__device__ __forceinline__ void gm_loaded(uint32_t (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+r"(v[i]));
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
  int nc, stages;        // k_gemm_few: rows of a tile, stages of the ring
  uint32_t idesc;
};

// ---- epilogues ----------------------------------------------------------------------------------------------------------
template <class O> __device__ __forceinline__ O gm_cast(float v) { return from_f32<O>(v); }

// 32 rows (a lane each) of `width` columns to memory. f(j, o): columns j .. j + 15 of the lane's row, all lanes together. vec: the rows' pieces
// start on 16-byte boundaries, and a lane writes its own; else they go through the warp's 4 KB of shared memory, 128 bytes of every row at
// a time, and are written row by row, a word or its two halves a lane.
template <class O, class F>
__device__ __forceinline__ void gm_rows(O* out, int64_t ld, int rows, int64_t cols, int width, bool vec, uint32_t buf, F&& f) {
  const int lane = threadIdx.x & 31;
  if (vec) {
    O* p = out + lane * ld;
#pragma unroll 1
    for (int j = 0; j < width; j += 16) {
      alignas(16) O o[16];
      f(j, o);
      const int valid = lane < rows ? (int)min((int64_t)16, cols - j) : 0;
      if (valid == 16) {
#pragma unroll
        for (int i = 0; i < 16; i += 16 / (int)sizeof(O)) *(uint4*)(p + j + i) = *(const uint4*)(o + i);
      } else {
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (i < valid) p[j + i] = o[i];
      }
      __syncwarp();
    }
    return;
  }
  constexpr int PIECE = 128 / (int)sizeof(O), WORDS = 16 * (int)sizeof(O) / 4;
#pragma unroll 1
  for (int c0 = 0; c0 < width; c0 += PIECE) {
#pragma unroll 1
    for (int j = 0; j < min(PIECE, width - c0); j += 16) {
      alignas(16) O o[16];
      f(c0 + j, o);
      const int w0 = j * (int)sizeof(O) / 4;
#pragma unroll
      for (int i = 0; i < WORDS; i++)
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(buf + (lane * 32 + ((w0 + i) ^ lane)) * 4), "r"(((const uint32_t*)o)[i]) : "memory");
    }
    __syncwarp();
    // the elements of word `lane`
    const int64_t left = min((int64_t)min(PIECE, width - c0), cols - c0) * (int)sizeof(O) - 4 * lane;
    for (int r = 0; r < rows; r++) {
      uint32_t v;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(buf + (r * 32 + (lane ^ r)) * 4) : "memory");
      char* p = (char*)(out + r * ld + c0) + 4 * lane;
      if (sizeof(O) >= 4 || ((uintptr_t)p & 3) == 0) {
        if (left >= 4) *(uint32_t*)p = v;
        else if (left > 0) *(uint16_t*)p = (uint16_t)v;
      } else {
        if (left > 0) *(uint16_t*)p = (uint16_t)v;
        if (left > 2) *(uint16_t*)(p + 2) = (uint16_t)(v >> 16);
      }
    }
    __syncwarp();
  }
}
template <int KIND, class O>
__device__ __forceinline__ O gm_scaled(const GemmCall& c, int32_t sum, float sa, float sb) {
  if constexpr (sizeof(O) == 8) return (double)sum * sa * sb;
  else return gm_cast<O>((float)sum * sa * sb);
}

// ---- large results --------------------------------------------------------------------------------------------------------
// Tile 256 x 256 per pair of CTAs (GATE: 256 x 128 of both products; narrower for few columns): each CTA holds the sums of its 128 rows and
// brings 128 rows and 128 columns of the operands, 32 KB a stage. One warp copies, one multiplies (the first CTA's, for both), eight take the sums out of one half of
// tensor memory while the other fills. A launch's pairs take tiles in turn, along the rows within groups of GP_GROUP row tiles, so that what
// runs at once shares operands in L2.
constexpr int GP_T = 384, GP_STAGES = 6, GP_STAGE = 2 * GM_OPERAND, GP_GROUP = 8;

__device__ __forceinline__ void gp_tile(const GemmArgs& A, int t, int& tm, int& tn) {
  const int per = GP_GROUP * A.tilesN, g = t / per, first = g * GP_GROUP, n = min(GP_GROUP, A.tilesM - first), r = t - g * per;
  tm = first + r % n;
  tn = r / n;
}

template <int KIND, class O>
__global__ void __launch_bounds__(GP_T, 1) __cluster_dims__(2) k_gemm_pair(const __grid_constant__ GemmArgs A) {
  constexpr bool I8 = KIND == GK_Q8;
  extern __shared__ __align__(1024) unsigned char gmsm[];
  __shared__ __align__(8) uint64_t full[GP_STAGES], empty[GP_STAGES], sumFull[2], sumEmpty[2];
  __shared__ uint32_t tmemAt;
  const GemmCall& c = A.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = gm_rank(), smem = (gm_smem(gmsm) + 1023u) & ~1023u;
  const int pairs = gridDim.x / 2, pair = blockIdx.x / 2, tiles = A.tilesM * A.tilesN;
  const int segments = KIND == GK_SUM ? 2 : 1, nk = A.kBlocks * segments;
  const bool aMn = !I8 && c.a[0].mn, bMn = !I8 && c.b[0].mn;
  const int mine = KIND == GK_GATE ? A.wide : A.wide / 2;  // columns that a CTA brings
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
      gm_init(gm_smem(sumEmpty + i), 16);  // the eight warps of both CTAs
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
  if (warp == 0) {
    if (gm_elect()) {
      int s = 0;
      uint32_t ph = 1;
      int64_t issued = 0;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int tm, tn;
        gp_tile(A, t, tm, tn);
        const int m0 = tm * 256 + rank * 128;
        const int halfN = A.tilesN / 2, which = KIND == GK_GATE ? (int)rank : KIND == GK_PAIR && tn >= halfN;
        const int n0 = KIND == GK_GATE ? tn * A.wide : (KIND == GK_PAIR && tn >= halfN ? tn - halfN : tn) * A.wide + rank * mine;
        for (int kb = 0; kb < nk; kb++) {
          ok = gm_wait(gm_smem(empty + s), ph);
          if (!ok) break;
          const int seg = KIND == GK_SUM && kb >= A.kBlocks, k0 = (kb - seg * A.kBlocks) * A.depth;
          const uint32_t bar = gm_peer(gm_smem(full + s), 0), da = smem + s * GP_STAGE, db = da + GM_OPERAND;
          if (rank == 0) gm_expect(gm_smem(full + s), 2 * (GM_OPERAND + mine * 128));
          const CUtensorMap *ma = A.a + seg, *mb = A.b + (KIND == GK_SUM ? seg : which);
          if (aMn) {
            gm_load<true>(da, ma, m0, k0, bar);
            gm_load<true>(da + 8192, ma, m0 + 64, k0, bar);
          } else {
            gm_load<true>(da, ma, k0, m0, bar);
          }
          if (bMn) {
            for (int i = 0; i < mine; i += 64) gm_load<true>(db + i * 128, mb, n0 + i, k0, bar);
          } else {
            gm_load<true>(db, mb, k0, n0, bar);
          }
          issued++;
          if (++s == GP_STAGES) s = 0, ph ^= 1;
        }
      }
      // what is still on its way, here and to the other CTA's barriers
      for (int i = 0; i < GP_STAGES; i++) {
        const int64_t n = (issued - i + GP_STAGES - 1) / GP_STAGES;  // times stage i was filled
        if (n <= 0) break;
        if (!ok && rank == 0) gm_wait(gm_smem(full + i), (uint32_t)(n - 1) & 1u);
        if (ok && !gm_wait(gm_smem(empty + i), (uint32_t)(n - 1) & 1u)) ok = false;
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && gm_elect()) {
      int s = 0;
      uint32_t ph = 0;
      int n = 0;
      for (int t = pair; t < tiles && ok; t += pairs, n++) {
        const int buf = n & 1;
        ok = gm_wait(gm_smem(sumEmpty + buf), ((n >> 1) & 1) ^ 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int kb = 0; kb < nk; kb++) {
          ok = gm_wait(gm_smem(full + s), ph);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          uint64_t a = gm_desc(smem + s * GP_STAGE, aMn), b = gm_desc(smem + s * GP_STAGE + GM_OPERAND, bMn);
#pragma unroll
          for (int i = 0; i < 4; i++, a += gm_step(aMn), b += gm_step(bMn)) gm_mma<true, I8>(tmem + buf * 256, a, b, A.idesc, kb > 0 || i > 0);
          gm_commit<true>(gm_smem(empty + s));
          if (++s == GP_STAGES) s = 0, ph ^= 1;
        }
        if (ok) gm_commit<true>(gm_smem(sumFull + buf));
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    int n = 0;
    for (int t = pair; t < tiles; t += pairs, n++) {
      const int buf = n & 1;
      ok = gm_wait(gm_smem(sumFull + buf), (n >> 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      int tm, tn;
      gp_tile(A, t, tm, tn);
      const int64_t m0 = (int64_t)tm * 256 + rank * 128 + quarter * 32, m = m0 + lane;
      const int rows = (int)max((int64_t)0, min((int64_t)32, c.M - m0)), width = A.wide / 2;
      const uint32_t at = tmem + buf * 256 + half * width + ((uint32_t)quarter << 21), room = smem + GP_STAGES * GP_STAGE + (warp - 4) * 4096;
      auto aligned = [&](int o) { return ((uintptr_t)c.out[o] | (uintptr_t)(c.ldo[o] * sizeof(O))) % 16 == 0; };
      if constexpr (KIND == GK_GATE) {
        const int64_t n0 = (int64_t)tn * A.wide + half * width;
        gm_rows((O*)c.out[0] + m0 * c.ldo[0] + n0, c.ldo[0], rows, c.N - n0, width, aligned(0), room, [&](int j, O(&o)[16]) {
          uint32_t v[32];
          gm_tmem16(at + j, v);
          gm_tmem16(at + A.wide + j, v + 16);
          gm_loaded(v);
          float h[16];
          with_act(c.act, [&](auto act) {
#pragma unroll
            for (int i = 0; i < 16; i++) h[i] = act_value(decltype(act)::value, __uint_as_float(v[i])) * __uint_as_float(v[16 + i]);
          });
          if (c.drop.on) {
#pragma unroll
            for (int q = 0; q < 16; q += 4) {
              const uint4 w = drop_words(c.drop, (uint32_t)m, (uint32_t)((n0 + j + q) / 4));
#pragma unroll
              for (int i = 0; i < 4; i++) h[q + i] = word_of(w, i) >= c.drop.cut ? h[q + i] * c.drop.scale : 0.f;
            }
          }
#pragma unroll
          for (int i = 0; i < 16; i++) o[i] = gm_cast<O>(h[i]);
        });
        if (c.out[1])
          for (int p = 0; p < 2; p++)
            gm_rows((O*)c.out[1 + p] + m0 * c.ldo[1 + p] + n0, c.ldo[1 + p], rows, c.N - n0, width, aligned(1 + p), room, [&](int j, O(&o)[16]) {
              uint32_t v[16];
              gm_tmem16(at + p * A.wide + j, v);
              gm_loaded(v);
#pragma unroll
              for (int i = 0; i < 16; i++) o[i] = gm_cast<O>(__uint_as_float(v[i]));
            });
      } else {
        const int halfN = A.tilesN / 2, which = KIND == GK_PAIR && tn >= halfN;
        const int64_t n0 = (int64_t)(which ? tn - halfN : tn) * A.wide + half * width;
        const float sa = I8 && m < c.M ? c.aScale[m] : 0.f;
        gm_rows((O*)c.out[which] + m0 * c.ldo[which] + n0, c.ldo[which], rows, c.N - n0, width, aligned(which), room, [&](int j, O(&o)[16]) {
          uint32_t v[16];
          gm_tmem16(at + j, v);
          gm_loaded(v);
#pragma unroll
          for (int i = 0; i < 16; i++) {
            if constexpr (I8) o[i] = gm_scaled<KIND, O>(c, (int32_t)v[i], sa, n0 + j + i < c.N ? __ldg(c.bScale + n0 + j + i) : 0.f);
            else o[i] = gm_cast<O>(__uint_as_float(v[i]));
          }
        });
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(gm_peer(gm_smem(sumEmpty + buf), 0)) : "memory");
    }
  }
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
// A CTA per 128 columns of the result (the lanes of tensor memory) and nc rows, so that little of the tensor cores' width is spent on
// rows that are not there; the depth is split over the CTAs of a cluster, whose partial sums meet in shared memory, each CTA adding up its
// share of the rows in the order of the ranks. GATE: both weights' tiles in a stage, two sums.
constexpr int GF_T = 192;

template <int KIND, class O>
__global__ void __launch_bounds__(GF_T, 1) k_gemm_few(const __grid_constant__ GemmArgs A) {
  constexpr bool I8 = KIND == GK_Q8;
  constexpr int NP = KIND == GK_GATE ? 2 : 1;
  constexpr int MOST = 16;
  extern __shared__ __align__(1024) unsigned char gmsm[];
  __shared__ __align__(8) uint64_t full[MOST], empty[MOST], sumFull;
  __shared__ uint32_t tmemAt;
  const GemmCall& c = A.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = gm_rank(), smem = (gm_smem(gmsm) + 1023u) & ~1023u;
  uint32_t split;
  asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(split));
  const int tile = blockIdx.x / split, tn = tile % A.tilesN, tm = tile / A.tilesN;
  const int halfN = A.tilesN / 2, which = KIND == GK_PAIR && tn >= halfN;
  const int n0 = (which ? tn - halfN : tn) * 128, m0 = tm * A.nc;
  const int nk = A.kBlocks * (KIND == GK_SUM ? 2 : 1);
  const int kb0 = (int)((int64_t)nk * rank / split), kb1 = (int)((int64_t)nk * (rank + 1) / split);
  const bool cMn = !I8 && c.a[0].mn, lMn = !I8 && c.b[0].mn;  // the result's rows and columns
  const uint32_t stage = NP * GM_OPERAND + A.nc * 128, cols = max(32, NP * A.nc);
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(gm_smem(&tmemAt)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < A.stages; i++) {
      gm_init(gm_smem(full + i), 1);
      gm_init(gm_smem(empty + i), 1);
    }
    gm_init(gm_smem(&sumFull), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmemAt;
  bool ok = true;
  if (warp == 4) {
    if (gm_elect()) {
      int s = 0, issued = 0;
      uint32_t ph = 1;
      for (int kb = kb0; kb < kb1; kb++) {
        ok = gm_wait(gm_smem(empty + s), ph);
        if (!ok) break;
        const int seg = KIND == GK_SUM && kb >= A.kBlocks, k0 = (kb - seg * A.kBlocks) * A.depth;
        const uint32_t bar = gm_smem(full + s), dl = smem + s * stage, dc = dl + NP * GM_OPERAND;
        gm_expect(bar, stage);
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const CUtensorMap* ml = A.b + (KIND == GK_GATE ? p : KIND == GK_SUM ? seg : which);
          if (lMn) {
            gm_load<false>(dl + p * GM_OPERAND, ml, n0, k0, bar);
            gm_load<false>(dl + p * GM_OPERAND + 8192, ml, n0 + 64, k0, bar);
          } else {
            gm_load<false>(dl + p * GM_OPERAND, ml, k0, n0, bar);
          }
        }
        if (cMn) {
          for (int i = 0; i < A.nc; i += 64) gm_load<false>(dc + i * 128, A.a + seg, m0 + i, k0, bar);
        } else {
          gm_load<false>(dc, A.a + seg, k0, m0, bar);
        }
        issued++;
        if (++s == A.stages) s = 0, ph ^= 1;
      }
      for (int i = 0; i < min(issued, A.stages); i++) {
        const int n = (issued - i + A.stages - 1) / A.stages;
        if (!ok) gm_wait(gm_smem(full + i), (uint32_t)(n - 1) & 1u);
        else if (!gm_wait(gm_smem(empty + i), (uint32_t)(n - 1) & 1u)) ok = false;
      }
    }
  } else if (warp == 5) {
    if (gm_elect()) {
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; kb++) {
        ok = gm_wait(gm_smem(full + s), ph);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t dl = smem + s * stage;
        uint64_t b = gm_desc(dl + NP * GM_OPERAND, cMn);
        uint64_t l[NP];
#pragma unroll
        for (int p = 0; p < NP; p++) l[p] = gm_desc(dl + p * GM_OPERAND, lMn);
#pragma unroll
        for (int i = 0; i < 4; i++, b += gm_step(cMn))
#pragma unroll
          for (int p = 0; p < NP; p++) {
            gm_mma<false, I8>(tmem + p * A.nc, l[p], b, A.idesc, kb > kb0 || i > 0);
            l[p] += gm_step(lMn);
          }
        gm_commit<false>(gm_smem(empty + s));
        if (++s == A.stages) s = 0, ph ^= 1;
      }
      if (ok) gm_commit<false>(gm_smem(&sumFull));
    }
  } else {
    ok = gm_wait(gm_smem(&sumFull), 0);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  __syncwarp();
  // The sums of lane n0 + 32 warp + lane (a column of the result), rows m0 .. m0 + nc
  const int rows = (int)min((int64_t)A.nc, c.M - m0);
  const int64_t n = n0 + warp * 32 + lane;
  const float sb = I8 && warp < 4 && n < c.N ? c.bScale[n] : 0.f;
  auto put = [&](int r, const uint32_t (&v)[NP]) {
    const int64_t m = m0 + r;
    if (n >= c.N) return;
    if constexpr (I8) {
      ((O*)c.out[0])[m * c.ldo[0] + n] = gm_scaled<KIND, O>(c, (int32_t)v[0], c.aScale[m], sb);
    } else if constexpr (KIND == GK_GATE) {
      const float g = __uint_as_float(v[0]), u = __uint_as_float(v[1]);
      float h = act_value(c.act, g) * u;
      if (c.drop.on) h = word_of(drop_words(c.drop, (uint32_t)m, (uint32_t)(n / 4)), (int)(n & 3)) >= c.drop.cut ? h * c.drop.scale : 0.f;
      ((O*)c.out[0])[m * c.ldo[0] + n] = gm_cast<O>(h);
      if (c.out[1]) {
        ((O*)c.out[1])[m * c.ldo[1] + n] = gm_cast<O>(g);
        ((O*)c.out[2])[m * c.ldo[2] + n] = gm_cast<O>(u);
      }
    } else {
      ((O*)c.out[which])[m * c.ldo[which] + n] = gm_cast<O>(__uint_as_float(v[0]));
    }
  };
  const uint32_t at = tmem + ((uint32_t)(warp & 3) << 21);
  if (warp < 4) {
    for (int r = 0; r < rows; r += 16) {
      uint32_t v[NP * 16];
#pragma unroll
      for (int p = 0; p < NP; p++) gm_tmem16(at + p * A.nc + r, v + 16 * p);
      gm_loaded(v);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        if (r + i >= rows) break;
        uint32_t w[NP];
#pragma unroll
        for (int p = 0; p < NP; p++) w[p] = kb1 > kb0 ? v[16 * p + i] : 0u;
        if (split == 1) put(r + i, w);
        else
#pragma unroll
          for (int p = 0; p < NP; p++) asm volatile("st.shared.b32 [%0], %1;" ::"r"(smem + ((p * A.nc + r + i) * 128 + threadIdx.x) * 4), "r"(w[p]) : "memory");
      }
      __syncwarp();
    }
  }
  if (split > 1) {
    gm_cluster_sync();
    if (warp < 4) {
      for (int r = rank; r < rows; r += split) {
        uint32_t w[NP];
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const uint32_t mine = smem + ((p * A.nc + r) * 128 + threadIdx.x) * 4;
          float f = 0.f;
          uint32_t sum = 0;
          for (uint32_t q = 0; q < split; q++) {
            uint32_t x;
            asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(x) : "r"(gm_peer(mine, q)) : "memory");
            if (I8) sum += x;
            else f += __uint_as_float(x);
          }
          w[p] = I8 ? sum : __float_as_uint(f);
        }
        put(r, w);
      }
    }
  }
  if (!ok) atomicExch(&denseErr, 202);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (split > 1) gm_cluster_sync();  // (the others may still read this one's sums)
  if (warp == 5) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
int64_t dense_status(int device) {
  (void)device;
  int32_t e = 0, zero = 0;
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

// Shared memory of a CTA in proportion to its columns of tensor memory, so that an SM never holds CTAs of more columns than it has: CTAs that
// wait for columns while their cluster waits for them could otherwise hold up one another, of any launches.
constexpr int GM_SM_SMEM = 228 * 1024, GM_CTA_SMEM = 1024;  // an SM's, and what it keeps for each CTA
template <class K>
static int64_t smem_for(OncePerDevice& once, int* room, int device, int cols, K kernel, int& least) {
  const int64_t rc = once(device, [&]() -> int64_t {
    cudaFuncAttributes a;
    CLA_CUDA(cudaFuncGetAttributes(&a, kernel));
    const int most = GM_SM_SMEM - GM_CTA_SMEM - (int)a.sharedSizeBytes;
    CLA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    *room = most;
    return CLA_OK;
  });
  least = GM_SM_SMEM / 512 * cols - (GM_SM_SMEM - *room);
  return rc;
}

// Which kernel and tile: the one that a count of clocks makes the fastest.
struct GemmPlan {
  bool large = false;
  int wide = 0;                      // k_gemm_pair
  int nc = 0, split = 1, stages = 1; // k_gemm_few
  double clocks = 1e30;
};
static GemmPlan gemm_plan(const GemmCall& c, int nk, int sms) {
  GemmPlan best;
  const int np = c.kind == GK_GATE ? 2 : 1, products = c.kind == GK_PAIR ? 2 : 1;
  const auto ceil_div = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const double L2 = 40;  // bytes a clock that an SM gets
  for (int wide = 256 / np; wide >= 64 && nk > 0; wide /= 2) {
    const int mine = np == 2 ? wide : wide / 2;
    if (c.b[0].mn && mine < 64) break;
    const int64_t tiles = ceil_div(c.M, 256) * ceil_div(c.N, wide) * products, turns = ceil_div(tiles, sms / 2);
    const double step = std::max(2.0 * mine * 2, (GM_OPERAND + mine * 128) / L2 / 1.5), t = 5000 + turns * (nk * step + 600);
    if (t < best.clocks) best.large = true, best.wide = wide, best.clocks = t;
  }
  for (int nc = 16; nc <= 128; nc *= 2) {
    const int least = c.a[0].mn ? 64 : 16;
    if (nc < least) continue;
    if (nc > least && nc / 2 >= c.M) break;
    const int stage = np * (int)GM_OPERAND + nc * 128;
    const int64_t tiles = ceil_div(c.M, nc) * ceil_div(c.N, 128) * products;
    for (int split = 1; split <= 8 && split <= std::max(1, nk); split++) {
      const int perSm = 2 * stage <= 111 * 1024 && (split == 1 || np * nc * 512 <= 111 * 1024) ? 2 : 1;
      const int64_t ctas = tiles * split, slots = (int64_t)sms * perSm, turns = ceil_div(ctas, slots);
      const double together = std::min<double>(perSm, (double)ceil_div(ctas, sms));
      const double step = together * std::max(2.0 * nc * np, stage / L2), t = 4000 + (split > 1 ? 1500 + nc * np * 4 : 0) + turns * (ceil_div(nk, split) * step + 2000 + nc * 20);
      if (t < best.clocks) {
        best.large = false, best.nc = nc, best.split = split, best.clocks = t;
        best.stages = (int)std::max<int64_t>(1, std::min<int64_t>({16, (ctas > sms && perSm == 2 ? 111 : 220) * 1024 / stage, ceil_div(nk, split)}));
      }
    }
  }
  return best;
}

template <int KIND, class O>
static int64_t launch_kind(GemmArgs& A, cudaStream_t s) {
  const GemmCall& c = A.c;
  const int bytes = type_bytes(c.type), segs = KIND == GK_SUM ? 2 : 1;
  int sms = 148;
  CLA_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c.device));
  A.depth = 128 / bytes;
  A.kBlocks = (int)((c.K + A.depth - 1) / A.depth);
  const int nk = A.kBlocks * segs;
  const GemmPlan p = gemm_plan(c, nk, sms);
  // both operands' types, where their index is contiguous, sums in 32 bits
  const uint32_t type = c.type == CLA_T_BF16 || c.type == CLA_T_I8 ? 1u : 0u;
  const uint32_t base = (KIND == GK_Q8 ? 2u : 1u) << 4 | type << 7 | type << 10;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = s;
  if (nk > 0)
    for (int i = 0; i < 2; i++) {
      const int boxB = !p.large ? 128 : KIND == GK_GATE ? p.wide : p.wide / 2;
      if (i == 0 || KIND == GK_SUM)
        if (const int64_t rc = operand_map(A.a[i], c.a[i], c.type, c.M, c.K, p.large ? 128 : p.nc); rc < 0) return rc;
      if (i == 0 || KIND != GK_Q8)
        if (const int64_t rc = operand_map(A.b[i], c.b[i], c.type, c.N, c.K, boxB); rc < 0) return rc;
    }
  const int np = KIND == GK_GATE ? 2 : 1, products = KIND == GK_PAIR ? 2 : 1;
  static OncePerDevice oncePair, onceFew;
  static int roomPair, roomFew;
  int smem;
  if (p.large) {
    A.wide = p.wide;
    A.tilesM = (int)((c.M + 255) / 256);
    A.tilesN = (int)((c.N + p.wide - 1) / p.wide) * products;
    A.idesc = base | (uint32_t)c.a[0].mn << 15 | (uint32_t)c.b[0].mn << 16 | (uint32_t)(p.wide * np >> 3) << 17 | (256u >> 4) << 24;
    if (const int64_t e = smem_for(oncePair, &roomPair, c.device, 512, k_gemm_pair<KIND, O>, smem); e < 0) return e;
    static_assert(GP_STAGES * GP_STAGE + 1024 + 8 * 4096 <= GM_SM_SMEM - GM_CTA_SMEM - 1024, "the ring and the warps' rooms fit");
    cfg.gridDim = 2 * (unsigned)std::min<int64_t>((int64_t)A.tilesM * A.tilesN, sms / 2);
    cfg.blockDim = GP_T;
    cfg.dynamicSmemBytes = smem;
    CLA_CUDA(cudaLaunchKernelEx(&cfg, k_gemm_pair<KIND, O>, A));
    return CLA_OK;
  }
  A.nc = p.nc;
  A.stages = p.stages;
  A.tilesM = (int)((c.M + A.nc - 1) / A.nc);
  A.tilesN = (int)((c.N + 127) / 128) * products;
  A.idesc = base | (uint32_t)c.b[0].mn << 15 | (uint32_t)c.a[0].mn << 16 | (uint32_t)(A.nc >> 3) << 17 | (128u >> 4) << 24;
  if (const int64_t e = smem_for(onceFew, &roomFew, c.device, std::max(32, np * A.nc), k_gemm_few<KIND, O>, smem); e < 0) return e;
  smem = std::max(smem, std::max(A.stages * (np * (int)GM_OPERAND + A.nc * 128), p.split > 1 ? np * A.nc * 512 : 0) + 1024);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)p.split, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cfg.gridDim = (unsigned)((int64_t)A.tilesM * A.tilesN * p.split);
  cfg.blockDim = GF_T;
  cfg.dynamicSmemBytes = smem;
  CLA_CUDA(cudaLaunchKernelEx(&cfg, k_gemm_few<KIND, O>, A));
  return CLA_OK;
}

int64_t launch_gemm(const GemmCall& c, cudaStream_t s) {
  if (c.M == 0 || c.N == 0) return CLA_OK;
  GemmArgs A = {};
  A.c = c;
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
