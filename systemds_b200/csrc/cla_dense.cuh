// What the dense operators share: element types, the activation and its slope, the dropout words, and the product behind them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "cla_common.cuh"

namespace cla {

inline int type_bytes(int type) {
  return type == CLA_T_F64 ? 8 : type == CLA_T_F32 ? 4 : type == CLA_T_I8 ? 1 : 2;
}
// Kernels that run just before or after a product, with the split of an SM's memory that the product has: no SM is emptied to change it
template <class K>
int64_t like_products(K kernel) {
  CLA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  return CLA_OK;
}
inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

template <class T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
// (one rounding to the nearest, of a value held in 32 or 64 bits)
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <class T> __device__ __forceinline__ T from_f64(double v) { return (T)v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f64(double v) { return __double2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f64(double v) { return __double2half(v); }

// 16 bytes of a row of T: one vector where every row starts on a 16-byte boundary (vec), else out of the two vectors that hold them (each has some of
// the wanted bytes, so neither reaches beyond what can be read), and at a row's end element by element.
template <class T> constexpr int DN_V = 16 / (int)sizeof(T);
__device__ __forceinline__ uint4 load_across(const void* p) {
  const uint4* a = (const uint4*)((uintptr_t)p & ~(uintptr_t)15);
  const uint4 lo = a[0], hi = a[1];
  const uint32_t words = ((uint32_t)(uintptr_t)p >> 2) & 3, bits = ((uint32_t)(uintptr_t)p & 3) * 8;
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 7; i++) w[i] = words & 1 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 5; i++) w[i] = words & 2 ? w[i + 2] : w[i];
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}
template <class T>
__device__ __forceinline__ void load_vec(const T* p, int n, bool vec, T (&v)[DN_V<T>]) {
  if (n >= DN_V<T>) {
    *(uint4*)v = vec || ((uintptr_t)p & 15) == 0 ? *(const uint4*)p : load_across(p);
  } else {
#pragma unroll
    for (int i = 0; i < DN_V<T>; i++) v[i] = i < n ? p[i] : from_f32<T>(0.f);
  }
}

// Two 16-bit values of a word, and back. (The lower bfloat16 by a byte permutation: the compiler's choice is a product, of which the words
// of dropout leave the pipe few.)
template <class T> __device__ __forceinline__ void from_word(uint32_t w, float& a, float& b) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(*(const __half2*)&w);
    a = f.x, b = f.y;
  } else {
    a = __uint_as_float(__byte_perm(w, 0, 0x1044));
    b = __uint_as_float(w & 0xffff0000u);
  }
}
template <class T> __device__ __forceinline__ uint32_t to_word(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
  }
}

// ---- dropout --------------------------------------------------------------------------------------------------------
struct DropDev {
  uint32_t cut = 0;  // kept where word >= cut
  uint32_t row0 = 0;
  uint32_t key[20] = {}, step[2] = {};  // the rounds' keys, the same for every counter
  float scale = 1.f;
  double scale64 = 1.0;
  int on = 0;
};
// The four words of columns 4 c .. 4 c + 3 of a row: Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011)
__device__ __forceinline__ uint4 drop_words(const DropDev& d, uint32_t row, uint32_t c) {
  uint32_t x0 = c, x1 = d.row0 + row, x2 = d.step[0], x3 = d.step[1];
#pragma unroll
  for (int i = 0; i < 10; i++) {
    const uint64_t a = (uint64_t)0xD2511F53u * x0, b = (uint64_t)0xCD9E8D57u * x2;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ d.key[2 * i];
    x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ d.key[2 * i + 1];
    x3 = (uint32_t)a;
  }
  return make_uint4(x0, x1, x2, x3);
}
// The same for many rows of four columns. Of the twenty products four depend on the columns alone: those of the first round, and one each
// of the second and third (a counter's words reach one another a round apart).
struct DropColumns {
  uint32_t first, second, third, hi, lo;  // what the rounds' words are xored with, and the third round's known product
  __device__ __forceinline__ DropColumns(const DropDev& d, uint32_t c) {
    const uint64_t a1 = (uint64_t)0xD2511F53u * c, b1 = (uint64_t)0xCD9E8D57u * d.step[0];
    const uint64_t b2 = (uint64_t)0xCD9E8D57u * ((uint32_t)(a1 >> 32) ^ d.step[1] ^ d.key[1]);
    const uint64_t a3 = (uint64_t)0xD2511F53u * ((uint32_t)(b2 >> 32) ^ (uint32_t)b1 ^ d.key[2]);
    first = (uint32_t)(b1 >> 32) ^ d.key[0];
    second = (uint32_t)a1 ^ d.key[3];
    third = (uint32_t)b2 ^ d.key[4];
    hi = (uint32_t)(a3 >> 32) ^ d.key[5];
    lo = (uint32_t)a3;
  }
  __device__ __forceinline__ uint4 words(const DropDev& d, uint32_t row) const {
    const uint64_t a2 = (uint64_t)0xD2511F53u * (first ^ (d.row0 + row)), b3 = (uint64_t)0xCD9E8D57u * ((uint32_t)(a2 >> 32) ^ second);
    uint32_t x0 = (uint32_t)(b3 >> 32) ^ third, x1 = (uint32_t)b3, x2 = hi ^ (uint32_t)a2, x3 = lo;
#pragma unroll
    for (int i = 3; i < 10; i++) {
      const uint64_t a = (uint64_t)0xD2511F53u * x0, b = (uint64_t)0xCD9E8D57u * x2;
      x0 = (uint32_t)(b >> 32) ^ x1 ^ d.key[2 * i];
      x1 = (uint32_t)b;
      x2 = (uint32_t)(a >> 32) ^ x3 ^ d.key[2 * i + 1];
      x3 = (uint32_t)a;
    }
    return make_uint4(x0, x1, x2, x3);
  }
};
__device__ __forceinline__ uint32_t word_of(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }

// ---- quantisation ---------------------------------------------------------------------------------------------------
template <class T> struct WideOf { using type = float; };
template <> struct WideOf<double> { using type = double; };
template <class T> __device__ __forceinline__ typename WideOf<T>::type widen(T v) { return to_f32(v); }
template <> __device__ __forceinline__ double widen(double v) { return v; }

// Magnitudes as whole numbers, which have the values' order with infinity and then NaN as the largest
__device__ __forceinline__ unsigned long long magnitude(double v) { return (unsigned long long)__double_as_longlong(v) & 0x7fffffffffffffffull; }
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float q8_scale(unsigned long long most) { return (float)(__longlong_as_double((long long)most) / 127.0); }
__device__ __forceinline__ float q8_scale(uint32_t most) { return __uint_as_float(most) / 127.f; }
// The nearest whole number of x / scale, as the low byte of the result. The product with the reciprocal is off by roundings of a value
// below 128: unless it comes that near to a half, where the quotient itself decides, both have the same nearest whole number. So the product
// is taken first, rounded by adding 1.5 times the power of two whose unit is 1, and whether some value came near is asked once
// for many of them: the quotients are then taken for all.
template <class W> struct Q8Row {
  W scale, inv;
  bool some, quick;  // a scale to divide by; whose reciprocal is finite
  __device__ __forceinline__ explicit Q8Row(float s)
      : scale((W)s), inv((W)1 / (W)s), some(s > 0.f && s < INFINITY), quick(s >= 0x1p-126f && s < INFINITY) {}
  __device__ __forceinline__ uint32_t product(W x, bool& near) const {
    constexpr W MAGIC = sizeof(W) == 8 ? (W)0x1.8p52 : (W)0x1.8p23;
    constexpr W FAR = (W)0.5 - (sizeof(W) == 8 ? (W)0x1p-43 : (W)0x1p-15);  // above 127 times two roundings of 2^-53, 2^-24 (of the reciprocal, of the quotient) and the last one
    const W r = fma(x, inv, MAGIC);
    near |= !(fabs(fma(x, inv, MAGIC - r)) <= FAR);
    if constexpr (sizeof(W) == 8) return (uint32_t)__double2loint(r);
    else return __float_as_uint(r);
  }
};
template <class W> __device__ __noinline__ uint32_t q8_quotient(W x, W scale, bool some) {
  return some ? (uint32_t)(int)fmin((W)127, fmax((W)-127, rint(x / scale))) : 0u;
}

// The quotients of values of which some product came near. Of 16-bit values one in 200 does (quotients of two of 256 numbers, times 127): then only those
// are divided that a lane of the warp asks for (16384 x 4096 BF16 values: 53 us, all of a piece divided 70).
template <class T, int N, class O>
__device__ __forceinline__ void q8_quotients(const Q8Row<typename WideOf<T>::type>& q8, const typename WideOf<T>::type (&v)[N], O (&o)[N]) {
#pragma unroll
  for (int j = 0; j < N; j++) {
    bool near = !q8.quick;
    if (sizeof(T) == 2) q8.product(v[j], near);
    if (sizeof(T) > 2 || near) o[j] = (O)q8_quotient(v[j], q8.scale, q8.some);
  }
}

// ---- the activation, in FP32 ------------------------------------------------------------------------------------------
// No tail is what is left of a 1: sigmoid(g) is a quotient of 1 or e = exp(-|g|), whose denominator is between 1 and 2, and the normal distribution's
// share below -|g| is exp(-g^2 / 2) times a smooth function. So the tails keep their relative error, in units of 2^-23 (the fast exponential of x:
// 2 + 1.2 |x|, the fast quotient 2, the roundings of an argument x: |x|): SiLU and sigmoid 6 + 1.2 |g|, GELU 10 + 1.2 g^2, its tanh form 6 + 3.2 |y|
// for sigmoid(y). Slopes two to three times that, of their terms' magnitudes. A rounding to 16 bits of 2^-8 or 2^-11 follows.
__device__ __forceinline__ float sigmoid_of(float g) {
  const float e = __expf(-fabsf(g));
  return __fdividef(g < 0.f ? e : 1.f, 1.f + e);
}
// (1 + tanh(y)) / 2 is sigmoid(2 y)
__device__ __forceinline__ float gelu_arg(float g) { return 1.5957691216057308f * (g + 0.044715f * g * g * g); }
// The normal distribution's share below g, (1 + erf(g / sqrt 2)) / 2, and exp(-g^2 / 2). Below -a it is exp(-a^2 / 2) t R(t) with t = 1 / (1 + 0.28 a): R is a
// polynomial fitted for the least relative error over all a >= 0 (1.7e-7; in FP32 4.4 units of 2^-23). One exponential serves value and
// slope (forward of 4095 x 2048 x 5461 with dropout, saved: 190 us with erfcf, 179 so).
struct Normal {
  float share, e;
};
__device__ __forceinline__ Normal normal_of(float g) {
  const float e = __expf(-0.5f * g * g), t = __fdividef(1.f, fmaf(0.28f, fabsf(g), 1.f));
  float r = 0.0247199624f;
  r = fmaf(r, t, -0.0935930849f);
  r = fmaf(r, t, 0.0924280604f);
  r = fmaf(r, t, -0.00644913645f);
  r = fmaf(r, t, 0.0727749934f);
  r = fmaf(r, t, 0.0836307955f);
  r = fmaf(r, t, 0.103084664f);
  r = fmaf(r, t, 0.111699803f);
  r = fmaf(r, t, 0.111703858f);
  const float tail = e * (t * r);
  return {g < 0.f ? tail : 1.f - tail, e};
}
__device__ __forceinline__ float act_value(int act, float g) {
  switch (act) {
    case CLA_ACT_SILU: return g * sigmoid_of(g);
    case CLA_ACT_SIGMOID: return sigmoid_of(g);
    case CLA_ACT_RELU: return g < 0.f ? 0.f : g;
    case CLA_ACT_GELU: return g * normal_of(g).share;
    default: return g * sigmoid_of(gelu_arg(g));
  }
}
__device__ __forceinline__ float act_slope(int act, float g, float& value) {
  switch (act) {
    case CLA_ACT_SILU: {
      const float s = sigmoid_of(g);
      value = g * s;
      return s * (1.f + g * (1.f - s));  // (where 1 - s cancels it is next to the 1: off by |g| / 2 units, and 0 from g = 17 on)
    }
    case CLA_ACT_SIGMOID: {
      const float e = __expf(-fabsf(g)), q = __fdividef(1.f, 1.f + e);
      value = g < 0.f ? e * q : q;
      return e * q * q;  // (of g and -g: the same)
    }
    case CLA_ACT_RELU: value = g < 0.f ? 0.f : g; return g > 0.f ? 1.f : 0.f;
    case CLA_ACT_GELU: {
      const Normal v = normal_of(g);
      value = g * v.share;
      return v.share + g * v.e * 0.39894228040143268f;
    }
    default: {
      const float s = sigmoid_of(gelu_arg(g));
      value = g * s;
      return s + g * s * (1.f - s) * 1.5957691216057308f * (1.f + 0.134145f * fminf(g * g, 1e4f));  // (beyond, 1 - s or s is 0, and the square may be infinite)
    }
  }
}
template <class F> __device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case CLA_ACT_SILU: f(std::integral_constant<int, CLA_ACT_SILU>()); break;
    case CLA_ACT_GELU: f(std::integral_constant<int, CLA_ACT_GELU>()); break;
    case CLA_ACT_GELU_TANH: f(std::integral_constant<int, CLA_ACT_GELU_TANH>()); break;
    case CLA_ACT_RELU: f(std::integral_constant<int, CLA_ACT_RELU>()); break;
    default: f(std::integral_constant<int, CLA_ACT_SIGMOID>()); break;
  }
}

// ---- products (cla_gemm.cu) -------------------------------------------------------------------------------------------
struct GemmOperand {
  const void* p = nullptr;
  int64_t ld = 0;   // elements
  bool mn = false;  // element (i, k) at p[k * ld + i]; else at p[i * ld + k]
};
enum GemmKind {
  GK_Q8,    // out0 = aScale bScale a0 b0, 8-bit integers
  GK_GATE,  // out0 = dropout(act(a0 b0) * (a0 b1)); out1, out2 = the two products, where not null
  GK_SUM,   // out0 = a0 b0 + a1 b1
  GK_PAIR   // out0 = a0 b0, out1 = a0 b1
};
struct GemmCall {
  GemmKind kind;
  int type, outType;    // of the operands (I8, BF16 or F16), of the results
  int64_t M, N, K;      // results [M x N], sums over K
  GemmOperand a[2], b[2];  // a: the rows' side; addresses 16-byte aligned, ld * element size a multiple of 16
  void* out[3] = {};
  int64_t ldo[3] = {};
  const float *aScale = nullptr, *bScale = nullptr;
  int act = 0;
  DropDev drop;
  int device = 0;
  bool split = true;      // whether the depth may be split (gemm_workspace() is 0 if not)
  void* parts = nullptr;  // gemm_workspace() bytes, 256-byte aligned
  int after = 0;          // AFTER_*
  bool quantize = false;  // Q8: a holds rows of outType, which the product quantises itself (gemm_quantizes())
  bool scores = false;    // the same, for few columns (gemm_scores()); the rows of a need no alignment
};
// What a kernel has to do with the one that the same call has launched just before it (which itself came after all that the stream held). The kernel may
// then start while that one still runs, and waits for its end where it says; the one before lets it by gm_let_next().
enum After {
  AFTER_CALL,  // there is none: an ordinary launch
  AFTER_ALL,   // it writes operands: before they are read
  AFTER_A,     // it writes a and aScale alone: the weights are read before
  AFTER_NONE   // the two read and write nothing that the other writes: at the end, so that who waits for this one has waited for both. The one
               // before has let this one by only after its own wait, so that what came before both is over when this one starts
};
// A barrier of some of a CTA's warps
__device__ __forceinline__ void gm_group_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void gm_after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void gm_let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// A launch configuration with the kernel before still running, or not (After)
struct EarlyLaunch {
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = {};
  EarlyLaunch(dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool early) {
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = early ? 1 : 0;
  }
  EarlyLaunch(const EarlyLaunch&) = delete;
};
// Whether a product quantises so many rows itself, of the type that the results have
bool gemm_quantizes(int64_t M, int64_t K, int type);
bool gemm_scores(int64_t M, int64_t N, int64_t K, int type);  // so many rows for so few columns
int64_t gemm_workspace(const GemmCall& c);  // goes by the sizes, the types and which index is contiguous
int64_t launch_gemm(const GemmCall& c, cudaStream_t s);
int64_t dense_status(int device);  // the self-check word of the product kernels, cleared

}  // namespace cla
