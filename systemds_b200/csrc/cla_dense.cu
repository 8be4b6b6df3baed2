// Dense operators beside the compressed products (cla_*_dev of include/systemds_cla.h): dropout, quantisation to 8 bits, products in 8 bits,
// the gated feed-forward block with its gradients. Their products are in cla_gemm.cu; here are the entry points and the kernels that
// go once over a matrix, all bound by memory.
#include "cla_dense.cuh"
#include <algorithm>
#include <cmath>
#include <initializer_list>

namespace cla {

std::shared_ptr<Matrix> lookup(cla_handle h);

constexpr int DN_T = 256;

template <class T>
__device__ __forceinline__ void store_vec(T* p, int n, bool vec, const T (&v)[DN_V<T>]) {
  if (vec && n >= DN_V<T>) {
    *(uint4*)p = *(const uint4*)v;
  } else {
#pragma unroll
    for (int i = 0; i < DN_V<T>; i++)
      if (i < n) p[i] = v[i];
  }
}
inline bool rows_aligned(const void* p, int64_t ld, int64_t rows, int bytes, int to = 16) {
  return ((uintptr_t)p % to) == 0 && (rows <= 1 || (ld * bytes) % to == 0);
}

// Which pieces of a matrix a thread takes: 2^log adjacent threads along a row, the others of the block down the rows, U rows at a time so
// that U loads are on their way before the first is used. columns(c): what a thread keeps for piece c of its rows; f(kept, r, step, n): rows
// r, r + step, .. (n of them).
struct Walk {
  int log;         // threads along a row
  int64_t rows;
  int per;         // pieces of a row
};
__device__ __forceinline__ int64_t walk_first(const Walk& w) { return (int64_t)blockIdx.y * (DN_T >> w.log) + (threadIdx.x >> w.log); }
__device__ __forceinline__ int64_t walk_step(const Walk& w) { return (int64_t)gridDim.y * (DN_T >> w.log); }
template <int U, class C, class F>
__device__ __forceinline__ void walk(const Walk& w, C&& columns, F&& f) {
  const int tx = threadIdx.x & ((1 << w.log) - 1);
  const int64_t step = walk_step(w);
  for (int c = blockIdx.x * (1 << w.log) + tx; c < w.per; c += gridDim.x << w.log) {
    auto kept = columns(c);
    for (int64_t r = walk_first(w); r < w.rows; r += U * step)
      f(kept, r, step, (int)min((int64_t)U, (w.rows - r + step - 1) / step));
  }
}
template <int N> struct DropPieces {  // of 4 N columns
  DropColumns c[N];
};
template <int N>
__device__ __forceinline__ DropPieces<N> drop_pieces(const DropDev& d, int64_t c) {
  if constexpr (N == 1) return {{DropColumns(d, (uint32_t)(c / 4))}};
  else return {{DropColumns(d, (uint32_t)(c / 4)), DropColumns(d, (uint32_t)(c / 4) + 1)}};
}

// V values of a row, on their way until they are used. VEC: from a 16-byte boundary; else 16-bit values come as the words that hold them, which are put
// in place when they are used (before, whoever asked for them waited: the gradients of 4069 x 8315 gates took 131 us, and 78 so).
// (not through the read-only path: dropout's result may go where its operand is)
template <class T, bool VEC, int V, bool SHIFTED = !VEC && sizeof(T) == 2>
struct Words {
  alignas(16) T v[V];
  __device__ __forceinline__ void load(const T* p, int left) {
    if constexpr (sizeof(T) == 8 && !VEC) {
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = i < left ? p[i] : T(0);
    } else {
#pragma unroll
      for (int h = 0; h < V; h += DN_V<T>) load_vec(p + h, left - h, VEC, (T(&)[DN_V<T>])v[h]);
    }
  }
  __device__ __forceinline__ void place(const T*, T (&to)[V]) const {
#pragma unroll
    for (int i = 0; i < V; i++) to[i] = v[i];
  }
};
template <class T, bool VEC, int V>
struct Words<T, VEC, V, true> {
  uint32_t w[V / 2 + 1];
  __device__ __forceinline__ void load(const T* p, int left) {
    const uint32_t off = (uint32_t)(uintptr_t)p & 2, end = off + 2 * min(left, V);
    const uint32_t* from = (const uint32_t*)((uintptr_t)p & ~(uintptr_t)3);
#pragma unroll
    for (int k = 0; k <= V / 2; k++) w[k] = 4 * k < end ? from[k] : 0u;
  }
  __device__ __forceinline__ void place(const T* p, T (&to)[V]) const {
#pragma unroll
    for (int k = 0; k < V / 2; k++) ((uint32_t*)to)[k] = __funnelshift_r(w[k], w[k + 1], ((uint32_t)(uintptr_t)p & 2) * 8);
  }
};
// The same for a warp's results, V a lane, side by side in a row that starts anywhere: through the warp's place in shared memory (32 lanes' values
// and a word), so that a store's words lie together. lanes: how many of the warp are there, the first ones; count: values.
template <class T, int V>
__device__ __forceinline__ void store_across(T* to, int64_t count, const T (&v)[V], uint32_t* place, int lanes) {
  constexpr int N = V * (int)sizeof(T) / 4;
  const uint32_t lane = threadIdx.x & 31, mask = lanes == 32 ? 0xffffffffu : (1u << lanes) - 1;
  const int off = (int)((uintptr_t)to & 2), end = off + (int)count * (int)sizeof(T);
  char* base = (char*)to - off;
#pragma unroll
  for (int i = 0; i < N; i += 4) *(uint4*)(place + 4 + lane * N + i) = ((const uint4*)v)[i / 4];
  __syncwarp(mask);
  const auto word = [&](int k) { return off ? __funnelshift_r(place[3 + k], place[4 + k], 16) : place[4 + k]; };
  const auto put = [&](int k) {
    if ((k > 0 || off == 0) && 4 * k + 4 <= end) *(uint32_t*)(base + 4 * k) = word(k);
    else if (k == 0 && off) *(uint16_t*)(base + 2) = (uint16_t)(word(0) >> 16);
    else *(uint16_t*)(base + 4 * k) = (uint16_t)word(k);
  };
  if (count == 32 * V) {
    put(lane);
#pragma unroll
    for (int i = 1; i < N; i++) *(uint32_t*)(base + 4 * (lane + 32 * i)) = word(lane + 32 * i);
    if (off && lane == 0) *(uint16_t*)(base + 128 * N) = (uint16_t)word(32 * N);
  } else {
    for (int k = lane; 4 * k < end; k += lanes) put(k);
  }
  __syncwarp(mask);
}

// ---- dropout --------------------------------------------------------------------------------------------------------
// Pieces of 16 bytes (F64: 32, the four columns of a counter). Bound: the words (sixteen 64-bit products and as many three-way logic
// operations for four columns) next to memory.
template <class T, bool VEC>
__global__ void __launch_bounds__(DN_T, VEC ? 5 : 4) k_dropout(const T* x, int64_t ldx, int64_t cols, T* y, int64_t ldy, const __grid_constant__ DropDev d,
                                                               const __grid_constant__ Walk w) {
  constexpr int P = DN_V<T>, V = P < 4 ? 4 : P, N = V / 4;
  __shared__ __align__(16) uint32_t places[VEC ? 1 : DN_T / 32][VEC ? 1 : 32 * V * sizeof(T) / 4 + 4 + 4];
  struct Kept {
    const T* x;
    T* y;
    int64_t stepX, stepY;
    int left;
    DropPieces<N> drop;
    Words<T, VEC, V> next;  // the next row's values: on their way while a row's are worked on
  };
  const int64_t r0 = walk_first(w), step = walk_step(w);
  walk<1>(
      w,
      [&](int piece) {
        const int64_t c = (int64_t)piece * V;
        Kept k{x + r0 * ldx + c, y + r0 * ldy + c, step * ldx, step * ldy, (int)min((int64_t)V, cols - c), drop_pieces<N>(d, c), {}};
        if (r0 < w.rows) k.next.load(k.x, k.left);
        return k;
      },
      [&](Kept& k, int64_t r, int64_t, int) {
        const Words<T, VEC, V> here = k.next;
        const T* from = k.x;
        k.x += k.stepX;
        if (r + step < w.rows) k.next.load(k.x, k.left);
        alignas(16) T v[V];
        here.place(from, v);
        if (d.on) {
#pragma unroll
          for (int q = 0; q < V; q += 4) {
            const uint4 words = k.drop.c[q / 4].words(d, (uint32_t)r);
            if constexpr (sizeof(T) == 2) {
#pragma unroll
              for (int j = 0; j < 4; j += 2) {
                uint32_t& w = *(uint32_t*)(v + q + j);
                float a, b;
                from_word<T>(w, a, b);
                a *= d.scale, b *= d.scale;
                w = to_word<T>(word_of(words, j) >= d.cut ? a : 0.f, word_of(words, j + 1) >= d.cut ? b : 0.f);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 4; j++) {
                if constexpr (sizeof(T) == 8) v[q + j] = word_of(words, j) >= d.cut ? v[q + j] * d.scale64 : 0.0;
                else v[q + j] = word_of(words, j) >= d.cut ? v[q + j] * d.scale : 0.f;
              }
            }
          }
        }
        if constexpr (VEC) {
#pragma unroll
          for (int h = 0; h < V; h += P) store_vec(k.y + h, k.left - h, true, (const T(&)[P])v[h]);
        } else if (sizeof(T) != 4 && w.log >= 5) {  // (a warp is in one row; FP32 values are words already: 252 us for 16384 x 8191, through shared memory 304)
          const int lane = threadIdx.x & 31;
          const int64_t there = cols - (k.y - y - r * ldy) + (int64_t)lane * V;  // from the warp's first value on
          store_across<T, V>(k.y - lane * V, min((int64_t)32 * V, there), v, places[threadIdx.x / 32], (int)min((int64_t)32, (there + V - 1) / V));
        } else {
#pragma unroll
          for (int h = 0; h < V; h += P) store_vec(k.y + h, k.left - h, false, (const T(&)[P])v[h]);
        }
        k.y += k.stepY;
      });
}

// ---- quantisation -----------------------------------------------------------------------------------------------------
// G threads per row, which they keep in registers: its largest magnitude, then its quotients. One pass over x; rows longer than G * C pieces are
// read a second time. VEC: rows start on 16-byte boundaries, a piece is 16 bytes; else the threads take single values in turn. Bound: memory.
template <class T, int G, int C, bool VEC>
__global__ void __launch_bounds__(DN_T, 3) k_quantize_rows(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols, int8_t* __restrict__ q,
                                                        int64_t ldq, float* __restrict__ scale) {
  using W = typename WideOf<T>::type;
  using Bits = decltype(magnitude(W()));
  constexpr int V = DN_V<T>, ROUND = G * V * C;
  __shared__ Bits part[DN_T / 32];
  const int lane = threadIdx.x % G, warp = threadIdx.x / 32;
  const int64_t r = (int64_t)blockIdx.x * (DN_T / G) + threadIdx.x / G;
  if (G < DN_T && r >= rows) return;  // (with all of its group)
  gm_let_next();  // (the product's weights may come meanwhile)
  const T* p = x + r * ldx + (VEC ? lane * V : lane);
  int8_t* to = q + r * ldq + (VEC ? lane * V : lane);
  alignas(16) T v[C][V];
  // value i of piece k of a round is at k * G * V + (VEC ? i : i * G) from p; how many from p on are there: left
  auto load = [&](int first) {
    const int left = cols - first - (VEC ? lane * V : lane);
#pragma unroll
    for (int k = 0; k < C; k++) {
      if (VEC && left >= k * G * V + V) {
        *(uint4*)v[k] = *(const uint4*)(p + first + k * G * V);
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
          const int at = k * G * V + (VEC ? i : i * G);
          v[k][i] = at < left ? p[first + at] : from_f32<T>(0.f);
        }
      }
    }
  };
  Bits most = 0;
  uint32_t most2 = 0;  // of 16-bit values two at a time: their bits have their order too
  for (int first = 0; first < cols; first += ROUND) {
    load(first);
#pragma unroll
    for (int j = 0; j < C; j++) {
      if (sizeof(T) < 8 && first + j * G * V >= cols) break;
#pragma unroll
      for (int i = 0; i < V; i += sizeof(T) == 2 ? 2 : 1) {
        if constexpr (sizeof(T) == 2) most2 = __vmaxu2(most2, *(const uint32_t*)&v[j][i] & 0x7fff7fffu);
        else most = max(most, magnitude(widen(v[j][i])));
      }
    }
  }
  if constexpr (sizeof(T) == 2) {
    const uint16_t larger = (uint16_t)max(most2 & 0xffffu, most2 >> 16);
    most = magnitude(widen(*(const T*)&larger));
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
  if (G > 32) {
    const int group = threadIdx.x / G;
    if (threadIdx.x % 32 == 0) part[warp] = most;
    gm_group_sync(1 + group, G);
    most = part[group * (G / 32)];
#pragma unroll
    for (int i = 1; i < G / 32; i++) most = max(most, part[group * (G / 32) + i]);
  }
  const float s = q8_scale(most);
  const Q8Row<W> q8(s);
  if (lane == 0) scale[r] = s;
  for (int first = 0; first < cols; first += ROUND) {
    if (cols > ROUND) load(first);
    const int left = cols - first - (VEC ? lane * V : lane);
    // how many pieces are asked about together: FP64 values hardly ever come near, FP32 ones in one of a hundred pieces of a warp
    constexpr int ASK = sizeof(T) == 8 ? C : 1;
#pragma unroll
    for (int j0 = 0; j0 < C; j0 += ASK) {
      if (first + j0 * G * V >= cols) break;
      alignas(16) uint8_t o[ASK][V];
      bool near = !q8.quick;
#pragma unroll
      for (int j = 0; j < ASK; j++)
#pragma unroll
        for (int i = 0; i < V; i++) o[j][i] = (uint8_t)q8.product(widen(v[j0 + j][i]), near);
      if (near) {  // (calls, which are not made before it is known whether they are wanted)
#pragma unroll
        for (int j = 0; j < ASK; j++) {
          W x[V];
#pragma unroll
          for (int i = 0; i < V; i++) x[i] = widen(v[j0 + j][i]);
          q8_quotients<T>(q8, x, o[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < ASK; j++) {
        const int at = (j0 + j) * G * V;
        int8_t* t = to + first + at;
        if (VEC && left >= at + V) {
          if constexpr (V == 8) *(uint2*)t = *(const uint2*)o[j];
          else if constexpr (V == 4) *(uint32_t*)t = *(const uint32_t*)o[j];
          else *(uint16_t*)t = *(const uint16_t*)o[j];
        } else {
#pragma unroll
          for (int i = 0; i < V; i++)
            if (at + (VEC ? i : i * G) < left) t[VEC ? i : i * G] = (int8_t)o[j][i];
        }
      }
    }
  }
}

// 32 columns per CTA, 32 threads down each: the columns' largest magnitudes, then their quotients, turned in shared memory.
template <class T>
__global__ void __launch_bounds__(1024) k_quantize_cols(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t cols, int8_t* __restrict__ q,
                                                        int64_t ldq, float* __restrict__ scale) {
  using W = typename WideOf<T>::type;
  using Bits = decltype(magnitude(W()));
  __shared__ Bits part[32][33];
  __shared__ float sc[32];
  __shared__ int8_t tile[32][132];
  const int tx = threadIdx.x, ty = threadIdx.y;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;
  Bits most = 0;
  if (c < cols)
    for (int64_t r = ty; r < rows; r += 32) most = max(most, magnitude(widen(x[r * ldx + c])));
  part[ty][tx] = most;
  __syncthreads();
  if (ty == 0) {
    for (int i = 1; i < 32; i++) most = max(most, part[i][tx]);
    sc[tx] = q8_scale(most);
    if (c < cols) scale[c] = sc[tx];
  }
  __syncthreads();
  const Q8Row<W> q8(sc[tx]);
  for (int64_t r0 = 0; r0 < rows; r0 += 128) {
#pragma unroll
    for (int i = 0; i < 128; i += 32) {
      const int64_t r = r0 + i + ty;
      tile[tx][i + ty] = c < cols && r < rows ? (int8_t)q8_quotient(widen(x[r * ldx + c]), q8.scale, q8.some) : 0;
    }
    __syncthreads();
    const int64_t oc = (int64_t)blockIdx.x * 32 + ty;
    if (oc < cols)
#pragma unroll
      for (int i = 0; i < 128; i += 32)
        if (r0 + i + tx < rows) q[oc * ldq + r0 + i + tx] = tile[ty][i + tx];
    __syncthreads();
  }
}

// ---- the gated block's elementwise gradients ----------------------------------------------------------------------------
// dG and dU in FP32, rounded to the type once: the products that follow take operands of 16 bits, and FP32 ones would pass through the tensor
// cores in three parts, three times the work. It costs the gradients 1.4 times the error of FP32 operands (relative, 64 bits compared: BF16 0.0023
// against 0.0017, FP16 0.00029 against 0.00021).
// (the next row's values are on their way while a row's are worked on)
template <class T, bool VEC>
__global__ void __launch_bounds__(DN_T, 3) k_gate_grad(const T* __restrict__ dh, int64_t lddh, const T* __restrict__ g, int64_t ldg,
                                                       const T* __restrict__ u, int64_t ldu, int64_t cols, T* __restrict__ dg, T* __restrict__ du,
                                                       int64_t ldo, const __grid_constant__ DropDev d, int act, const __grid_constant__ Walk w) {
  constexpr int V = DN_V<T>, N = V / 4;
  const int64_t r0 = walk_first(w), step = walk_step(w);
  struct Values {
    Words<T, VEC, V> h, g, u;
  };
  struct Kept {
    int64_t c;
    int left;
    DropPieces<N> drop;
    Values next;
  };
  gm_let_next();
  auto load = [&](int64_t r, int64_t c, int left, Values& v) {
    v.h.load(dh + r * lddh + c, left);
    v.g.load(g + r * ldg + c, left);
    v.u.load(u + r * ldu + c, left);
  };
  with_act(act, [&](auto name) {
    walk<1>(
        w,
        [&](int piece) {
          const int64_t c = (int64_t)piece * V;
          Kept k{c, (int)min((int64_t)V, cols - c), drop_pieces<N>(d, c), {}};
          if (r0 < w.rows) load(r0, c, k.left, k.next);
          return k;
        },
        [&](Kept& k, int64_t r, int64_t, int) {
          Values v = k.next;
          if (r + step < w.rows) load(r + step, k.c, k.left, k.next);
          alignas(16) T inH[V], inG[V], inU[V], toG[V], toU[V];
          v.h.place(dh + r * lddh, inH);
          v.g.place(g + r * ldg, inG);
          v.u.place(u + r * ldu, inU);
#pragma unroll
          for (int q = 0; q < V; q += 4) {
            uint4 words;
            if (d.on) words = k.drop.c[q / 4].words(d, (uint32_t)r);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              float h[2], gate[2], up[2];
              from_word<T>(*(const uint32_t*)(inH + q + j), h[0], h[1]);
              from_word<T>(*(const uint32_t*)(inG + q + j), gate[0], gate[1]);
              from_word<T>(*(const uint32_t*)(inU + q + j), up[0], up[1]);
#pragma unroll
              for (int i = 0; i < 2; i++) {
                float a;
                if (d.on) h[i] = word_of(words, j + i) >= d.cut ? h[i] * d.scale : 0.f;
                const float slope = act_slope(decltype(name)::value, gate[i], a);
                gate[i] = h[i] * up[i] * slope;
                up[i] = h[i] * a;
              }
              *(uint32_t*)(toG + q + j) = to_word<T>(gate[0], gate[1]);
              *(uint32_t*)(toU + q + j) = to_word<T>(up[0], up[1]);
            }
          }
          store_vec(dg + r * ldo + k.c, k.left, true, toG);
          store_vec(du + r * ldo + k.c, k.left, true, toU);
        });
  });
  gm_after_previous();  // (the copies next to this: who waits for this kernel has waited for both)
}

// ---- copies -----------------------------------------------------------------------------------------------------------
// Rows to rows that start on lines of 128 bytes, as the products read them; up to three matrices a launch. In bytes: the elements' size is of no matter.
struct Copies {
  const void* from[3];
  void* to[3];
  int64_t ldFrom[3], ldTo[3];
  int64_t bytes[3];  // of a row
  Walk walk[3];
  int ctas[4];   // the first CTA of each, down the rows
};
__global__ void __launch_bounds__(DN_T) k_repitch(const __grid_constant__ Copies c) {
  gm_let_next();
  const int k = (int)blockIdx.y >= c.ctas[2] ? 2 : (int)blockIdx.y >= c.ctas[1] ? 1 : 0;
  const Walk& w = c.walk[k];
  const uint8_t* x = (const uint8_t*)c.from[k];
  uint8_t* y = (uint8_t*)c.to[k];
  const int tx = threadIdx.x & ((1 << w.log) - 1), down = DN_T >> w.log, ctas = c.ctas[k + 1] - c.ctas[k];
  const int64_t step = (int64_t)ctas * down, ldx = c.ldFrom[k], ldy = c.ldTo[k];
  for (int piece = blockIdx.x * (1 << w.log) + tx; piece < w.per; piece += gridDim.x << w.log) {
    const int64_t at = (int64_t)piece * 16;
    const int left = (int)min((int64_t)16, c.bytes[k] - at);
    for (int64_t r = (int64_t)(blockIdx.y - c.ctas[k]) * down + (threadIdx.x >> w.log); r < w.rows; r += 2 * step) {
      alignas(16) uint8_t v[2][16];
      const bool two = r + step < w.rows;
      load_vec(x + r * ldx + at, left, false, v[0]);
      if (two) load_vec(x + (r + step) * ldx + at, left, false, v[1]);
      store_vec(y + r * ldy + at, left, true, v[0]);
      if (two) store_vec(y + (r + step) * ldy + at, left, true, v[1]);
    }
  }
}
template <class T, int U>
__global__ void __launch_bounds__(DN_T) k_narrow(const double* __restrict__ x, int64_t cols, T* __restrict__ y, int64_t ldy,
                                                 const __grid_constant__ Walk w) {
  walk<U>(
      w, [](int piece) { return piece; },
      [&](int c, int64_t r, int64_t step, int n) {
        double v[U];
#pragma unroll
        for (int k = 0; k < U; k++)
          if (k < n) v[k] = x[(r + k * step) * cols + c];
#pragma unroll
        for (int k = 0; k < U; k++)
          if (k < n) y[(r + k * step) * ldy + c] = from_f64<T>(v[k]);
      });
}

// ---- host side --------------------------------------------------------------------------------------------------------
namespace {

// The call's device is current while it lives, then the caller's again
struct OnDevice {
  int before = -1;
  int64_t rc = CLA_OK;
  explicit OnDevice(int device) {
    int now = -1;
    cudaError_t e = cudaGetDevice(&now);
    if (e == cudaSuccess && now != device) {
      e = cudaSetDevice(device);
      if (e == cudaSuccess) before = now;
    }
    if (e == cudaSuccess) return;
    rc = fail(CLA_ERR_CUDA, std::string("device of a dense call: ") + cudaGetErrorString(e));
    cudaGetLastError();  // (or the next launch would be taken for the one that failed)
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// The grid of a walk over rows of `per` pieces, `at` rows at a time: eight CTAs an SM, or fewer
dim3 walk_grid(Walk& w, int64_t rows, int64_t per, int at) {
  w.rows = rows;
  w.per = (int)per;
  w.log = 0;
  while (w.log < 8 && (1 << w.log) < per) w.log++;
  const int64_t x = (per + (1 << w.log) - 1) >> w.log, down = DN_T >> w.log;
  const int64_t most = std::max<int64_t>(1, 148 * 8 / x), need = (rows + down * at - 1) / (down * at);
  return dim3((unsigned)std::min<int64_t>(x, 148 * 8), (unsigned)std::max<int64_t>(1, std::min(most, need)));
}

int64_t check_matrix(const char* what, const void* p, int64_t rows, int64_t cols, int64_t ld, int bytes) {
  if (rows < 0 || cols < 0) return fail(CLA_ERR_SHAPE, std::string(what) + ": negative size");
  if (rows > 1 << 30 || cols > 1 << 30) return fail(CLA_ERR_UNSUPPORTED, std::string(what) + ": more than 2^30 rows or columns");
  if (rows == 0 || cols == 0) return CLA_OK;
  if (!p) return fail(CLA_ERR_BAD_ARG, std::string(what) + ": null buffer");
  if (ld < cols) return fail(CLA_ERR_SHAPE, std::string(what) + ": rows overlap (ld below the row's length)");
  if (ld > (int64_t)1 << 38) return fail(CLA_ERR_UNSUPPORTED, std::string(what) + ": rows too far apart");
  if ((uintptr_t)p % bytes) return fail(CLA_ERR_BAD_ARG, std::string(what) + ": address not a multiple of the element size");
  return CLA_OK;
}
#define DN_CHECK(...)                                     \
  do {                                                    \
    if (const int64_t rc_ = (__VA_ARGS__); rc_ < 0) return rc_; \
  } while (0)

// A matrix as the bytes that a call reads or writes of it; ld in bytes
struct Area {
  const void* p;
  int64_t rows, bytes, ld;
};
Area area(const void* p, int64_t rows, int64_t cols, int64_t ld, int bytes) { return {p, p ? rows : 0, cols * bytes, ld * bytes}; }
Area area(const void* p, int64_t bytes) { return {p, p ? 1 : 0, bytes, bytes}; }
// Whether two of them share a byte. Matrices side by side in the rows of a larger one do not, though their addresses are mixed.
bool share(Area a, Area b) {
  using Wide = __int128;  // (rows times strides pass 64 bits before anybody has such memory)
  if (a.rows <= 0 || b.rows <= 0 || a.bytes <= 0 || b.bytes <= 0) return false;
  const Wide d = (Wide)(uintptr_t)a.p - (Wide)(uintptr_t)b.p;
  if (d >= (Wide)(b.rows - 1) * b.ld + b.bytes || -d >= (Wide)(a.rows - 1) * a.ld + a.bytes) return false;
  const auto floor_div = [](Wide n, Wide by) { return n / by - (n % by < 0); };
  // rows of a stride s: the first of b's rows -most .. most from a's that ends behind its start
  const auto meets = [&](Wide off, int64_t s, int64_t least, int64_t most) {
    const Wide k = std::max<Wide>(floor_div(-a.bytes - off, s) + 1, least);
    return k <= most && off + k * s < b.bytes;
  };
  if (a.rows == 1) a.ld = b.ld;
  if (b.rows == 1) b.ld = a.ld;
  if (a.rows == 1 && b.rows == 1) return true;
  if (a.ld == b.ld) return meets(d, a.ld, -(b.rows - 1), a.rows - 1);
  if (a.rows < b.rows) return share(b, a);
  for (int64_t j = 0; j < b.rows; j++)  // (a's rows against row j of b)
    if (meets(d - (Wide)j * b.ld, a.ld, 0, a.rows - 1)) return true;
  return false;
}
// Outputs that share a byte with an input or with one another: CTAs would read what others have written already
int64_t check_apart(const char* what, std::initializer_list<Area> outs, std::initializer_list<Area> ins) {
  for (const Area* o = outs.begin(); o != outs.end(); o++) {
    for (const Area& i : ins)
      if (share(*o, i)) return fail(CLA_ERR_BAD_ARG, std::string(what) + ": a result or the workspace overlaps an operand");
    for (const Area* q = outs.begin(); q != o; q++)
      if (share(*o, *q)) return fail(CLA_ERR_BAD_ARG, std::string(what) + ": results or the workspace overlap one another");
  }
  return CLA_OK;
}

int64_t drop_device(const cla_drop& d, int64_t rows, DropDev& o) {
  if (!(d.p >= 0.0 && d.p < 1.0)) return fail(CLA_ERR_BAD_ARG, "dropout: p must be at least 0 and below 1");
  if (d.row0 < 0 || d.row0 > ((int64_t)1 << 32) - rows) return fail(CLA_ERR_BAD_ARG, "dropout: rows beyond 2^32");
  o.on = d.p > 0.0;
  o.cut = (uint32_t)std::floor(d.p * 4294967296.0);
  o.row0 = (uint32_t)d.row0;
  for (uint32_t i = 0; i < 10; i++) {
    o.key[2 * i] = (uint32_t)d.seed + i * 0x9E3779B9u;
    o.key[2 * i + 1] = (uint32_t)(d.seed >> 32) + i * 0xBB67AE85u;
  }
  o.step[0] = (uint32_t)d.step, o.step[1] = (uint32_t)(d.step >> 32);
  o.scale64 = 1.0 / (1.0 - d.p);
  o.scale = (float)o.scale64;
  return CLA_OK;
}
bool is_float_type(int t) { return t == CLA_T_F64 || t == CLA_T_F32 || t == CLA_T_BF16 || t == CLA_T_F16; }

// Calls f with a pointer of the type: f(T())
template <class F> void with_type(int type, F&& f) {
  if (type == CLA_T_F64) f(double());
  else if (type == CLA_T_F32) f(float());
  else if (type == CLA_T_BF16) f(__nv_bfloat16());
  else f(__half());
}

int64_t quantize(int type, const void* x, int64_t ldx, int64_t rows, int64_t cols, bool byCols, int8_t* q, int64_t ldq, float* scale,
                 int device, cudaStream_t s) {
  if ((byCols ? cols : rows) == 0) return CLA_OK;
  int64_t rc = CLA_OK;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    if (byCols) {
      k_quantize_cols<T><<<(unsigned)((cols + 31) / 32), dim3(32, 32), 0, s>>>((const T*)x, ldx, rows, cols, q, ldq, scale);
      return;
    }
    constexpr int V = DN_V<T>, C = sizeof(T) == 8 ? 8 : 4;
    const bool vec = rows_aligned(x, ldx, rows, sizeof(T)) && rows_aligned(q, ldq, rows, 1, V);
    // the fewest threads that hold the row: a warp (no barrier), two, half a CTA, a CTA (50,000 rows of 520 FP64 values: by two warps 69 us, by four 128,
    // most of them idle). More where rows are too few for that to matter: a CTA where there is not one for every SM, 16 values of 16 bits a thread
    // while there are not two for every SM (they are divided more often: 500 x 2000 by two warps 6.8 us, by a CTA 4.0)
    int group = 32;
    while (group < DN_T && (cols > group * C * V || rows < 148 || (sizeof(T) == 2 && cols > group * 16 && rows * group < 148 * 2 * DN_T))) group *= 2;
    auto go = [&](auto kernel, OncePerDevice& once) {
      rc = once(device, [&] { return like_products(kernel); });
      const int down = DN_T / group;
      if (rc >= 0) kernel<<<(unsigned)((rows + down - 1) / down), DN_T, 0, s>>>((const T*)x, ldx, rows, (int)cols, q, ldq, scale);
    };
    static OncePerDevice once[8];
    if (group == 32) vec ? go(k_quantize_rows<T, 32, C, true>, once[0]) : go(k_quantize_rows<T, 32, C, false>, once[1]);
    else if (group == 64) vec ? go(k_quantize_rows<T, 64, C, true>, once[6]) : go(k_quantize_rows<T, 64, C, false>, once[7]);
    else if (group == 128) vec ? go(k_quantize_rows<T, 128, C, true>, once[2]) : go(k_quantize_rows<T, 128, C, false>, once[3]);
    else vec ? go(k_quantize_rows<T, DN_T, C, true>, once[4]) : go(k_quantize_rows<T, DN_T, C, false>, once[5]);
  });
  if (rc < 0) return rc;
  CLA_CUDA(cudaGetLastError());
  return CLA_OK;
}

// Hands out parts of the caller's workspace; with a null base it only counts
struct Work {
  char* p;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* r = p ? p + used : nullptr;
    used += round_up(bytes, 256);
    return r;
  }
};
// Rows of copies and intermediate results: on lines of 128 bytes, which is what the products read of a row at a time (4095 x 2048 x 5461, weights with
// rows on 16-byte boundaries only: 188 us; on lines: 182 us)
constexpr int PITCH = 128;
// Operands as the products read them: themselves, or copies in the workspace where their rows do not start on 16-byte boundaries. The copies are made in
// one launch, by run().
struct Aligned {
  Copies c = {};
  int n = 0;
  Work& w;
  explicit Aligned(Work& work) : w(work) {}
  void operator()(GemmOperand& o, int64_t i, int64_t k, int type) {
    const int bytes = type_bytes(type);
    const int64_t rows = o.mn ? k : i, cols = o.mn ? i : k;
    if (rows <= 1 && (uintptr_t)o.p % 16 == 0) o.ld = round_up(o.ld, 16 / bytes);  // (no second row)
    if (rows_aligned(o.p, o.ld, 2, bytes)) return;
    const int64_t ld = round_up(cols, PITCH / bytes);
    void* to = w.take(rows * ld * bytes);
    if (rows && cols) {
      c.from[n] = o.p, c.to[n] = to;
      c.ldFrom[n] = o.ld * bytes, c.ldTo[n] = ld * bytes;
      c.bytes[n] = cols * bytes;
      c.walk[n].rows = rows;
      n++;
    }
    o.p = to;
    o.ld = ld;
  }
  int64_t run(int device, cudaStream_t s) {
    if (n == 0) return CLA_OK;
    static OncePerDevice once;
    DN_CHECK(once(device, [] { return like_products(k_repitch); }));
    unsigned x = 1;
    for (int k = 0; k < n; k++) {
      const dim3 g = walk_grid(c.walk[k], c.walk[k].rows, (c.bytes[k] + 15) / 16, 2);
      x = std::max(x, g.x);
      c.ctas[k + 1] = c.ctas[k] + (int)g.y;
    }
    const unsigned y = (unsigned)c.ctas[n];
    for (int k = n + 1; k < 4; k++) c.ctas[k] = (int)y;
    k_repitch<<<dim3(x, y), DN_T, 0, s>>>(c);
    CLA_CUDA(cudaGetLastError());
    return CLA_OK;
  }
};
int64_t product(GemmCall& g, Work& w, bool run, cudaStream_t s) {
  if (const int64_t n = gemm_workspace(g)) g.parts = w.take(n);
  return run ? launch_gemm(g, s) : CLA_OK;
}

int64_t check_q8(const cla_q8* c) {
  if (!c) return fail(CLA_ERR_BAD_ARG, "8-bit product: null arguments");
  if (c->aType != CLA_T_I8 && !is_float_type(c->aType)) return fail(CLA_ERR_UNSUPPORTED, "8-bit product: type of a");
  if (!is_float_type(c->outType)) return fail(CLA_ERR_UNSUPPORTED, "8-bit product: type of the result");
  if (c->K > 131071) return fail(CLA_ERR_UNSUPPORTED, "8-bit product: more than 131071 terms may leave 32 bits");
  DN_CHECK(check_matrix("8-bit product, a", c->a, c->M, c->K, c->lda, type_bytes(c->aType)));
  DN_CHECK(check_matrix("8-bit product, b", c->b, c->N, c->K, c->ldb, 1));
  DN_CHECK(check_matrix("8-bit product, result", c->out, c->M, c->N, c->ldo, type_bytes(c->outType)));
  if (c->M && c->N && ((c->aType == CLA_T_I8 && !c->aScale) || !c->bScale)) return fail(CLA_ERR_BAD_ARG, "8-bit product: null scales");
  return CLA_OK;
}
int64_t q8_run(const cla_q8& c, bool run, Work& w, cudaStream_t s, bool split = true) {
  GemmCall g;
  g.kind = GK_Q8;
  g.type = CLA_T_I8;
  g.outType = c.outType;
  g.M = c.M, g.N = c.N, g.K = c.K;
  g.a[0] = {c.a, c.lda, false};
  g.b[0] = {c.b, c.ldb, false};
  g.out[0] = c.out, g.ldo[0] = c.ldo;
  g.aScale = c.aScale, g.bScale = c.bScale;
  g.device = c.device;
  g.split = split;
  if (c.M == 0 || c.N == 0) return CLA_OK;
  Aligned aligned(w);
  aligned(g.b[0], c.N, c.K, CLA_T_I8);
  if (c.aType == CLA_T_I8) aligned(g.a[0], c.M, c.K, CLA_T_I8);
  if (run) DN_CHECK(aligned.run(c.device, s));
  if (aligned.n) g.after = AFTER_ALL;
  if (split && c.aType == c.outType && gemm_quantizes(c.M, c.K, c.aType)) {
    g.quantize = true;
  } else if (c.aType == c.outType && gemm_scores(c.M, c.N, c.K, c.aType)) {
    g.scores = true;
  } else if (c.aType != CLA_T_I8) {
    const int64_t ld = round_up(c.K, PITCH);
    int8_t* q = (int8_t*)w.take(c.M * ld);
    float* sc = (float*)w.take(c.M * 4);
    if (run) DN_CHECK(quantize(c.aType, c.a, c.lda, c.M, c.K, false, q, ld, sc, c.device, s));
    g.a[0] = {q, ld, false};
    g.aScale = sc;
    g.after = AFTER_A;  // (the last kernel before the product)
  }
  return product(g, w, run, s);
}

int64_t check_gated(const cla_gated* c, bool backward, DropDev& d) {
  if (!c) return fail(CLA_ERR_BAD_ARG, "gated block: null arguments");
  if (c->type != CLA_T_BF16 && c->type != CLA_T_F16) return fail(CLA_ERR_UNSUPPORTED, "gated block: types BF16 and F16");
  if (c->act < CLA_ACT_SILU || c->act > CLA_ACT_SIGMOID) return fail(CLA_ERR_UNSUPPORTED, "gated block: unknown activation");
  if (c->wTrans != 0 && c->wTrans != 1) return fail(CLA_ERR_BAD_ARG, "gated block: wTrans is 0 or 1");
  const int64_t wr = c->wTrans ? c->F : c->D, wc = c->wTrans ? c->D : c->F;
  DN_CHECK(check_matrix("gated block, x", c->x, c->M, c->D, c->ldx, 2));
  DN_CHECK(check_matrix("gated block, wg", c->wg, wr, wc, c->ldwg, 2));
  DN_CHECK(check_matrix("gated block, wu", c->wu, wr, wc, c->ldwu, 2));
  DN_CHECK(drop_device(c->drop, c->M, d));
  if (!backward) {
    DN_CHECK(check_matrix("gated block, h", c->h, c->M, c->F, c->ldh, 2));
    if (!c->g != !c->u) return fail(CLA_ERR_BAD_ARG, "gated block: g and u go together");
    if (!c->g) return CLA_OK;
  } else {
    DN_CHECK(check_matrix("gated block, dh", c->dh, c->M, c->F, c->lddh, 2));
    if (!c->dwg != !c->dwu) return fail(CLA_ERR_BAD_ARG, "gated block: dwg and dwu go together");
    if (c->dx) DN_CHECK(check_matrix("gated block, dx", c->dx, c->M, c->D, c->lddx, 2));
    if (c->dwg) {
      DN_CHECK(check_matrix("gated block, dwg", c->dwg, c->D, c->F, c->lddwg, 2));
      DN_CHECK(check_matrix("gated block, dwu", c->dwu, c->D, c->F, c->lddwu, 2));
    }
  }
  DN_CHECK(check_matrix("gated block, g", c->g, c->M, c->F, c->ldg, 2));
  return check_matrix("gated block, u", c->u, c->M, c->F, c->ldu, 2);
}
GemmCall gated_call(const cla_gated& c, GemmKind kind, int64_t M, int64_t N, int64_t K) {
  GemmCall g;
  g.kind = kind;
  g.type = g.outType = c.type;
  g.M = M, g.N = N, g.K = K;
  g.act = c.act;
  g.device = c.device;
  return g;
}
int64_t gated_fwd(const cla_gated& c, const DropDev& d, bool run, Work& w, cudaStream_t s) {
  if (c.M == 0 || c.F == 0) return CLA_OK;
  GemmCall g = gated_call(c, GK_GATE, c.M, c.F, c.D);
  g.a[0] = {c.x, c.ldx, false};
  g.b[0] = {c.wg, c.ldwg, !c.wTrans};
  g.b[1] = {c.wu, c.ldwu, !c.wTrans};
  Aligned aligned(w);
  aligned(g.a[0], c.M, c.D, c.type);
  for (int i = 0; i < 2; i++) aligned(g.b[i], c.F, c.D, c.type);
  if (run) DN_CHECK(aligned.run(c.device, s));
  if (aligned.n) g.after = AFTER_ALL;
  g.out[0] = c.h, g.out[1] = c.g, g.out[2] = c.u;
  g.ldo[0] = c.ldh, g.ldo[1] = c.ldg, g.ldo[2] = c.ldu;
  g.drop = d;
  return product(g, w, run, s);
}
int64_t gated_bwd(const cla_gated& c, const DropDev& d, bool run, Work& w, cudaStream_t s) {
  const int64_t ld = round_up(c.F, PITCH / 2);
  void* dg = w.take(c.M * ld * 2);
  void* du = w.take(c.M * ld * 2);
  const bool wantX = c.dx && c.M && c.D, wantW = c.dwg && c.D && c.F;
  GemmCall x = gated_call(c, GK_SUM, c.M, c.D, c.F), wt = gated_call(c, GK_PAIR, c.D, c.F, c.M);
  x.a[0] = {dg, ld, false};
  x.a[1] = {du, ld, false};
  x.b[0] = {c.wg, c.ldwg, (bool)c.wTrans};
  x.b[1] = {c.wu, c.ldwu, (bool)c.wTrans};
  x.out[0] = c.dx, x.ldo[0] = c.lddx;
  wt.a[0] = {c.x, c.ldx, true};
  wt.b[0] = {dg, ld, true};
  wt.b[1] = {du, ld, true};
  wt.out[0] = c.dwg, wt.out[1] = c.dwu;
  wt.ldo[0] = c.lddwg, wt.ldo[1] = c.lddwu;
  Aligned aligned(w);
  if (wantX)
    for (int i = 0; i < 2; i++) aligned(x.b[i], c.D, c.F, c.type);
  if (wantW) aligned(wt.a[0], c.D, c.M, c.type);
  if (run) DN_CHECK(aligned.run(c.device, s));
  const bool grads = c.M && c.F;
  if (run && grads) {
    const bool vec = rows_aligned(c.dh, c.lddh, c.M, 2) && rows_aligned(c.g, c.ldg, c.M, 2) && rows_aligned(c.u, c.ldu, c.M, 2);
    Walk k;
    const dim3 grid = walk_grid(k, c.M, (c.F + 7) / 8, 1);
    auto go = [&](auto t, auto kernel, OncePerDevice& once) -> int64_t {
      using T = decltype(t);
      DN_CHECK(once(c.device, [&] { return like_products(kernel); }));
      EarlyLaunch l(grid, DN_T, 0, s, aligned.n > 0);  // (next to the copies)
      CLA_CUDA(cudaLaunchKernelEx(&l.cfg, kernel, (const T*)c.dh, c.lddh, (const T*)c.g, c.ldg, (const T*)c.u, c.ldu, c.F, (T*)dg, (T*)du, ld,
                                  d, (int)c.act, k));
      return CLA_OK;
    };
    static OncePerDevice once[4];
    using B = __nv_bfloat16;
    if (c.type == CLA_T_BF16) DN_CHECK(vec ? go(B(), k_gate_grad<B, true>, once[0]) : go(B(), k_gate_grad<B, false>, once[1]));
    else DN_CHECK(vec ? go(__half(), k_gate_grad<__half, true>, once[2]) : go(__half(), k_gate_grad<__half, false>, once[3]));
  }
  x.after = wt.after = grads || aligned.n ? AFTER_ALL : AFTER_CALL;
  if (wantX && c.F) wt.after = AFTER_NONE;
  if (wantX) DN_CHECK(product(x, w, run, s));
  if (wantW) DN_CHECK(product(wt, w, run, s));
  return CLA_OK;
}
int64_t check_work(const Work& need, const void* work, int64_t bytes) {
  if (need.used == 0) return CLA_OK;
  if (!work || bytes < need.used) return fail(CLA_ERR_BAD_ARG, "workspace smaller than " + std::to_string(need.used) + " bytes");
  if ((uintptr_t)work % 256) return fail(CLA_ERR_BAD_ARG, "workspace not 256-byte aligned");
  return CLA_OK;
}

int64_t check_q8_apart(const cla_q8& c, int64_t used) {
  const bool i8 = c.aType == CLA_T_I8;
  return check_apart("8-bit product", {area(c.out, c.M, c.N, c.ldo, type_bytes(c.outType)), area(c.work, used)},
                     {area(c.a, c.M, c.K, c.lda, type_bytes(c.aType)), area(c.b, c.N, c.K, c.ldb, 1), area(i8 ? c.aScale : nullptr, c.M * 4),
                      area(c.bScale, c.N * 4)});
}
int64_t check_gated_apart(const cla_gated& c, bool backward, int64_t used) {
  const int64_t wr = c.wTrans ? c.F : c.D, wc = c.wTrans ? c.D : c.F;
  const Area x = area(c.x, c.M, c.D, c.ldx, 2), wg = area(c.wg, wr, wc, c.ldwg, 2), wu = area(c.wu, wr, wc, c.ldwu, 2), work = area(c.work, used);
  const Area g = area(c.g, c.M, c.F, c.ldg, 2), u = area(c.u, c.M, c.F, c.ldu, 2);
  if (!backward) return check_apart("gated block", {area(c.h, c.M, c.F, c.ldh, 2), g, u, work}, {x, wg, wu});
  return check_apart("gated block",
                     {area(c.dx, c.M, c.D, c.lddx, 2), area(c.dwg, c.D, c.F, c.lddwg, 2), area(c.dwu, c.D, c.F, c.lddwu, 2), work},
                     {x, wg, wu, g, u, area(c.dh, c.M, c.F, c.lddh, 2)});
}

// ---- rows of a compressed block ---------------------------------------------------------------------------------------
constexpr int64_t ROWS_CHUNK = 64ll << 20;  // bytes of FP64 rows at a time that the workspace functions ask for: half the L2
// Rows [row0, row0 + rows) through an FP64 buffer of `cap` rows: use(first row, rows, their cells). Decompression starts where the skip
// indexes have entries, so a chunk may begin with rows that were not asked for.
template <class F>
int64_t for_rows(Matrix* m, int64_t row0, int64_t rows, double* X, int64_t cap, cudaStream_t s, F&& use) {
  for (int64_t r = row0; r < row0 + rows;) {
    const int64_t from = r / SKIP_ROWS * SKIP_ROWS, to = std::min(row0 + rows, from + cap);
    DN_CHECK(launch_decompress_range(m, (int)from, (int)to, X, s));
    DN_CHECK(use(r, to - r, X + (r - from) * m->nCols));
    r = to;
  }
  return CLA_OK;
}
int64_t chunk_rows(const Matrix* m, int64_t rows) {
  const int64_t cols = std::max(m->nCols, 1), most = std::max<int64_t>(1, ROWS_CHUNK / 8 / cols / SKIP_ROWS);
  return std::min(most, rows / SKIP_ROWS + 2) * SKIP_ROWS;
}
// What the 8-bit product of a chunk of so many rows needs: their cells, q and scales
int64_t q8_chunk_bytes(const Matrix* m, int64_t rows) {
  return round_up(rows * round_up(m->nCols, PITCH), 256) + round_up(rows * 4, 256) + round_up(rows * m->nCols * 8, 256);
}

}  // namespace
}  // namespace cla

using namespace cla;

#define DN_MATRIX(h)                                                       \
  std::shared_ptr<Matrix> mp = lookup(h);                                  \
  if (!mp) return fail(CLA_ERR_BAD_HANDLE, "unknown or destroyed handle"); \
  Matrix* m = mp.get();                                                    \
  std::lock_guard<std::mutex> lk(m->mu);                                   \
  if (!m->finalized) return fail(CLA_ERR_STATE, "cla_finalize has not been called on this handle")

extern "C" {

int64_t cla_dropout_dev(int32_t type, const void* x, int64_t ldx, int64_t rows, int64_t cols, void* y, int64_t ldy, const cla_drop* drop,
                        int32_t device, void* stream) {
  if (!is_float_type(type)) return fail(CLA_ERR_UNSUPPORTED, "dropout: unknown type");
  if (!drop) return fail(CLA_ERR_BAD_ARG, "dropout: null arguments");
  DN_CHECK(check_matrix("dropout, x", x, rows, cols, ldx, type_bytes(type)));
  DN_CHECK(check_matrix("dropout, y", y, rows, cols, ldy, type_bytes(type)));
  DropDev d;
  DN_CHECK(drop_device(*drop, rows, d));
  if (x != y || (rows > 1 && ldx != ldy))  // (onto its own input: every thread reads an element before it writes it)
    DN_CHECK(check_apart("dropout", {area(y, rows, cols, ldy, type_bytes(type))}, {area(x, rows, cols, ldx, type_bytes(type))}));
  OnDevice on(device);
  if (on.rc < 0) return on.rc;
  if (rows == 0 || cols == 0) return CLA_OK;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr int V = std::max(4, DN_V<T>);
    const bool vec = rows_aligned(x, ldx, rows, sizeof(T)) && rows_aligned(y, ldy, rows, sizeof(T));
    Walk w;
    const dim3 grid = walk_grid(w, rows, (cols + V - 1) / V, 1);
    (vec ? k_dropout<T, true> : k_dropout<T, false>)<<<grid, DN_T, 0, (cudaStream_t)stream>>>((const T*)x, ldx, cols, (T*)y, ldy, d, w);
  });
  CLA_CUDA(cudaGetLastError());
  return CLA_OK;
}

int64_t cla_q8_quantize_dev(int32_t type, const void* x, int64_t ldx, int64_t rows, int64_t cols, int32_t byCols, int8_t* q, int64_t ldq,
                            float* scale, int32_t device, void* stream) {
  if (!is_float_type(type)) return fail(CLA_ERR_UNSUPPORTED, "quantize: unknown type");
  if (byCols != 0 && byCols != 1) return fail(CLA_ERR_BAD_ARG, "quantize: byCols is 0 or 1");
  DN_CHECK(check_matrix("quantize, x", x, rows, cols, ldx, type_bytes(type)));
  DN_CHECK(check_matrix("quantize, q", q, byCols ? cols : rows, byCols ? rows : cols, ldq, 1));
  if ((byCols ? cols : rows) && !scale) return fail(CLA_ERR_BAD_ARG, "quantize: null scales");
  DN_CHECK(check_apart("quantize", {area(q, byCols ? cols : rows, byCols ? rows : cols, ldq, 1), area(scale, (byCols ? cols : rows) * 4)},
                       {area(x, rows, cols, ldx, type_bytes(type))}));
  OnDevice on(device);
  if (on.rc < 0) return on.rc;
  return quantize(type, x, ldx, rows, cols, byCols, q, ldq, scale, device, (cudaStream_t)stream);
}

int64_t cla_q8_workspace(const cla_q8* c) {
  DN_CHECK(check_q8(c));
  Work w{nullptr};
  DN_CHECK(q8_run(*c, false, w, nullptr));
  return w.used;
}
int64_t cla_q8_mm_dev(const cla_q8* c, void* stream) {
  DN_CHECK(check_q8(c));
  Work need{nullptr}, w{(char*)c->work};
  DN_CHECK(q8_run(*c, false, need, nullptr));
  DN_CHECK(check_work(need, c->work, c->workBytes));
  DN_CHECK(check_q8_apart(*c, need.used));
  OnDevice on(c->device);
  if (on.rc < 0) return on.rc;
  return q8_run(*c, true, w, (cudaStream_t)stream);
}

int64_t cla_gated_workspace(const cla_gated* c, int32_t backward) {
  DropDev d;
  DN_CHECK(check_gated(c, backward != 0, d));
  Work w{nullptr};
  DN_CHECK(backward ? gated_bwd(*c, d, false, w, nullptr) : gated_fwd(*c, d, false, w, nullptr));
  return w.used;
}
static int64_t gated_dev(const cla_gated* c, bool backward, void* stream) {
  DropDev d;
  DN_CHECK(check_gated(c, backward, d));
  Work need{nullptr}, w{(char*)c->work};
  DN_CHECK(backward ? gated_bwd(*c, d, false, need, nullptr) : gated_fwd(*c, d, false, need, nullptr));
  DN_CHECK(check_work(need, c->work, c->workBytes));
  DN_CHECK(check_gated_apart(*c, backward, need.used));
  OnDevice on(c->device);
  if (on.rc < 0) return on.rc;
  return backward ? gated_bwd(*c, d, true, w, (cudaStream_t)stream) : gated_fwd(*c, d, true, w, (cudaStream_t)stream);
}
int64_t cla_gated_fwd_dev(const cla_gated* c, void* stream) { return gated_dev(c, false, stream); }
int64_t cla_gated_bwd_dev(const cla_gated* c, void* stream) { return gated_dev(c, true, stream); }

int64_t cla_rows_workspace(cla_handle h, int64_t rows, int32_t type) {
  DN_MATRIX(h);
  if (!is_float_type(type)) return fail(CLA_ERR_UNSUPPORTED, "rows of a block: unknown type");
  if (rows < 0) return fail(CLA_ERR_SHAPE, "rows of a block: negative size");
  return round_up(chunk_rows(m, rows) * m->nCols * 8, 256);
}
int64_t cla_decompress_rows_dev(cla_handle h, int64_t row0, int64_t rows, int32_t type, void* out, int64_t ldo, void* work, int64_t workBytes,
                                void* stream) {
  DN_MATRIX(h);
  if (!is_float_type(type)) return fail(CLA_ERR_UNSUPPORTED, "rows of a block: unknown type");
  if (row0 < 0 || rows < 0 || rows > m->nRows || row0 > m->nRows - rows) return fail(CLA_ERR_SHAPE, "rows of a block: outside the matrix");
  DN_CHECK(check_matrix("rows of a block, result", out, rows, m->nCols, ldo, type_bytes(type)));
  if (rows == 0 || m->nCols == 0) return CLA_OK;
  const int64_t cap = workBytes / 8 / m->nCols / SKIP_ROWS * SKIP_ROWS;
  if (!work || cap < SKIP_ROWS) return fail(CLA_ERR_BAD_ARG, "rows of a block: workspace below 1024 rows of FP64");
  if ((uintptr_t)work % 256) return fail(CLA_ERR_BAD_ARG, "workspace not 256-byte aligned");
  DN_CHECK(check_apart("rows of a block", {area(out, rows, m->nCols, ldo, type_bytes(type)), area(work, std::min(cap, round_up(rows, SKIP_ROWS) + SKIP_ROWS) * m->nCols * 8)}, {}));
  OnDevice on(m->device);
  if (on.rc < 0) return on.rc;
  cudaStream_t s = (cudaStream_t)stream;
  m->stats.calls_decompress++;
  DN_CHECK(order_begin(m, s));
  const int64_t rc = for_rows(m, row0, rows, (double*)work, cap, s, [&](int64_t r, int64_t n, const double* X) -> int64_t {
    with_type(type, [&](auto t) {
      using T = decltype(t);
      Walk w;
      const dim3 grid = walk_grid(w, n, m->nCols, 4);
      k_narrow<T, 4><<<grid, DN_T, 0, s>>>(X, m->nCols, (T*)out + (r - row0) * ldo, ldo, w);
    });
    m->stats.kernel_launches++;
    CLA_CUDA(cudaGetLastError());
    return CLA_OK;
  });
  const int64_t rc2 = order_end(m, s);
  return rc < 0 ? rc : rc2;
}

int64_t cla_q8_rmm_workspace(cla_handle h, int64_t N) {
  DN_MATRIX(h);
  if (N < 0) return fail(CLA_ERR_SHAPE, "8-bit right product: negative size");
  if (N > 1 << 30) return fail(CLA_ERR_UNSUPPORTED, "8-bit right product: more than 2^30 columns");
  return q8_chunk_bytes(m, chunk_rows(m, m->nRows)) + round_up(N * round_up(m->nCols, PITCH), 256);
}
int64_t cla_q8_rmm_dev(cla_handle h, const int8_t* b, int64_t ldb, const float* bScale, int64_t N, int32_t outType, void* out, int64_t ldo,
                       void* work, int64_t workBytes, void* stream) {
  DN_MATRIX(h);
  cla_q8 c = {};
  c.M = m->nRows, c.N = N, c.K = m->nCols;
  c.a = work, c.lda = m->nCols, c.aType = CLA_T_F64;  // (each chunk's cells)
  c.b = b, c.ldb = ldb, c.bScale = bScale;
  c.out = out, c.ldo = ldo, c.outType = outType;
  c.device = m->device;
  DN_CHECK(check_q8(&c));
  if (c.M == 0 || c.N == 0) return CLA_OK;
  Work w{(char*)work};
  GemmOperand bo{b, ldb, false};
  if ((uintptr_t)work % 256) return fail(CLA_ERR_BAD_ARG, "workspace not 256-byte aligned");
  const int64_t room = workBytes - round_up(N * round_up(m->nCols, PITCH), 256);
  int64_t cap = room / std::max<int64_t>(1, q8_chunk_bytes(m, SKIP_ROWS)) * SKIP_ROWS;
  if (!work || cap < SKIP_ROWS) return fail(CLA_ERR_BAD_ARG, "8-bit right product: workspace below 1024 rows");
  cap = std::min(cap, round_up(c.M, SKIP_ROWS));
  cla_q8 apart = c;
  apart.a = nullptr, apart.work = work;
  DN_CHECK(check_q8_apart(apart, q8_chunk_bytes(m, cap) + round_up(N * round_up(m->nCols, PITCH), 256)));
  OnDevice on(m->device);
  if (on.rc < 0) return on.rc;
  cudaStream_t s = (cudaStream_t)stream;
  m->stats.calls_rmm++;
  DN_CHECK(order_begin(m, s));
  Aligned aligned(w);
  aligned(bo, N, c.K, CLA_T_I8);
  int64_t rc = aligned.run(c.device, s);
  c.b = (const int8_t*)bo.p, c.ldb = bo.ld;
  double* X = (double*)w.take(cap * m->nCols * 8);
  if (rc >= 0)
    rc = for_rows(m, 0, c.M, X, cap, s, [&](int64_t r, int64_t n, const double* cells) -> int64_t {
      cla_q8 part = c;
      part.M = n;
      part.a = cells;
      part.out = (char*)out + r * ldo * type_bytes(outType);
      Work q = w;
      return q8_run(part, true, q, s, false);  // (rows enough without: its workspace goes by the rows alone)
    });
  const int64_t rc2 = order_end(m, s);
  return rc < 0 ? rc : rc2;
}

int64_t cla_dense_status(int32_t device) {
  OnDevice on(device);
  if (on.rc < 0) return on.rc;
  return dense_status(device);
}

}  // extern "C"
