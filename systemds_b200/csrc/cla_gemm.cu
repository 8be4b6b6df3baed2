// Products of dense operands in 8 and 16 bits with their epilogues: see cla_dense.cuh.
#include "cla_dense.cuh"

namespace cla {

// The plain kernel: a CTA per 64 x 64 results, operands through shared memory 16 deep, a thread per 4 x 4 results, sums in FP32 (8-bit
// operands: 32-bit integers). Bound: the FMA pipe.
constexpr int GS_T = 64, GS_K = 16;
template <class T> struct SumOf { using type = float; };
template <> struct SumOf<int8_t> { using type = int32_t; };

template <class T>
__global__ void __launch_bounds__(256) k_gemm_simple(const __grid_constant__ GemmCall c) {
  using S = typename SumOf<T>::type;
  __shared__ S sa[GS_K][GS_T + 4], sb[2][GS_K][GS_T + 4];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int64_t m0 = (int64_t)blockIdx.y * GS_T, n0 = (int64_t)blockIdx.x * GS_T;
  const int which = blockIdx.z;  // PAIR: the product
  const bool two = c.kind == GK_GATE;
  S acc[2][4][4] = {};
  for (int seg = 0; seg < (c.kind == GK_SUM ? 2 : 1); seg++)
    for (int64_t k0 = 0; k0 < c.K; k0 += GS_K) {
      for (int e = tid; e < GS_T * GS_K; e += 256) {
        auto load = [&](const GemmOperand& o, int64_t i0, int64_t rows, S (*dst)[GS_T + 4]) {
          const int i = o.mn ? e % GS_T : e / GS_K, k = o.mn ? e / GS_T : e % GS_K;
          S v = 0;
          if (i0 + i < rows && k0 + k < c.K) {
            const T* p = (const T*)o.p;
            v = (S)to_f32(p[o.mn ? (k0 + k) * o.ld + i0 + i : (i0 + i) * o.ld + k0 + k]);
          }
          dst[k][i] = v;
        };
        load(c.a[seg], m0, c.M, sa);
        load(c.b[c.kind == GK_PAIR ? which : seg], n0, c.N, sb[0]);
        if (two) load(c.b[1], n0, c.N, sb[1]);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < GS_K; k++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            acc[0][i][j] += sa[k][ty * 4 + i] * sb[0][k][tx * 4 + j];
            if (two) acc[1][i][j] += sa[k][ty * 4 + i] * sb[1][k][tx * 4 + j];
          }
      __syncthreads();
    }
  for (int i = 0; i < 4; i++) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= c.M) break;
    uint4 w;
    if (c.drop.on) w = drop_words(c.drop, (uint32_t)m, (uint32_t)((n0 + tx * 4) / 4));
    for (int j = 0; j < 4; j++) {
      const int64_t n = n0 + tx * 4 + j;
      if (n >= c.N) break;
      auto put = [&](int o, int outType, double d, float f) {
        const int64_t at = m * c.ldo[o] + n;
        if (outType == CLA_T_F64) ((double*)c.out[o])[at] = d;
        else if (outType == CLA_T_F32) ((float*)c.out[o])[at] = f;
        else if (outType == CLA_T_BF16) ((__nv_bfloat16*)c.out[o])[at] = from_f32<__nv_bfloat16>(f);
        else ((__half*)c.out[o])[at] = from_f32<__half>(f);
      };
      if (c.kind == GK_Q8) {
        if (c.outType == CLA_T_F64) put(0, c.outType, (double)acc[0][i][j] * c.aScale[m] * c.bScale[n], 0.f);
        else put(0, c.outType, 0.0, (float)acc[0][i][j] * c.aScale[m] * c.bScale[n]);
      } else if (c.kind == GK_GATE) {
        const float g = (float)acc[0][i][j], u = (float)acc[1][i][j];
        float h = act_value(c.act, g) * u;
        if (c.drop.on) h = word_of(w, j) >= c.drop.cut ? h * c.drop.scale : 0.f;
        put(0, c.outType, 0.0, h);
        if (c.out[1]) {
          put(1, c.outType, 0.0, g);
          put(2, c.outType, 0.0, u);
        }
      } else {
        put(c.kind == GK_PAIR ? which : 0, c.outType, 0.0, (float)acc[0][i][j]);
      }
    }
  }
}

static __device__ int32_t denseErr;

int64_t dense_status(int device) {
  (void)device;
  int32_t e = 0, zero = 0;
  CLA_CUDA(cudaMemcpyFromSymbol(&e, denseErr, sizeof(e)));
  if (!e) return CLA_OK;
  CLA_CUDA(cudaMemcpyToSymbol(denseErr, &zero, sizeof(zero)));
  return fail(CLA_ERR_DEVICE_CHECK, "a dense product's self-check tripped (code " + std::to_string(e) + ")");
}

int64_t launch_gemm(const GemmCall& c, cudaStream_t s) {
  if (c.M == 0 || c.N == 0) return CLA_OK;
  const dim3 grid((unsigned)((c.N + GS_T - 1) / GS_T), (unsigned)((c.M + GS_T - 1) / GS_T), c.kind == GK_PAIR ? 2 : 1);
  if (c.type == CLA_T_I8) k_gemm_simple<int8_t><<<grid, 256, 0, s>>>(c);
  else if (c.type == CLA_T_BF16) k_gemm_simple<__nv_bfloat16><<<grid, 256, 0, s>>>(c);
  else k_gemm_simple<__half><<<grid, 256, 0, s>>>(c);
  CLA_CUDA(cudaGetLastError());
  return CLA_OK;
}

}  // namespace cla
