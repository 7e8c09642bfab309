// Matrix product of int8 rows with int8 weights, a scale per row and per output channel:
//   y[m, n] = (sum_k a[m, k] w[n, k]) * a_scales[m] * w_scales[n] (+ bias[n])      int32 sums, exact up to K = 131056
// rounded once to fp16, bf16 or fp32.  SiLU: w holds gate rows, then as many up rows; out[m, n] = silu(gate) * up of the fp32 values.
//
// Tiles of 64 x 64 from shared memory, four products per dp4a.
#include "../../include/b200_vllm.h"
#include "common.cuh"

namespace b200 {
namespace gemm8 {

constexpr int kMaxK = 131056;        // 2^31 / 128^2 = 131072 products of the largest size overflow; the multiple of 16 below

enum Out { kF16 = 0, kBF16 = 1, kF32 = 2 };

struct Args {
  const int8_t* a;
  const float* a_scales;
  const int8_t* w;
  const float* w_scales;
  const void* bias;
  void* c;
  int M, N, K;
};

template <int OUT>
__device__ __forceinline__ float load_elem(const void* p, size_t i) {
  if constexpr (OUT == kF32) return static_cast<const float*>(p)[i];
  else return bits16_to_f32<OUT == kBF16>(static_cast<const uint16_t*>(p)[i]);
}
template <int OUT>
__device__ __forceinline__ void store_elem(void* p, size_t i, float v) {
  if constexpr (OUT == kF32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = f32_to_bits16<OUT == kBF16>(v);
}
__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + expf(-g)) * u; }

template <int OUT, bool SILU>
__global__ void __launch_bounds__(256) simple_kernel(const Args g) {
  __shared__ int sa[64][17], sw[SILU ? 2 : 1][64][17];
  pdl_trigger();
  pdl_wait();
  const int n_out = SILU ? g.N / 2 : g.N, m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15, kw = g.K / 4;
  int acc[SILU ? 2 : 1][4][4] = {};
  for (int k0 = 0; k0 < kw; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i >> 4, k = i & 15;
      const bool in = k0 + k < kw;
      sa[r][k] = in && m0 + r < g.M ? reinterpret_cast<const int*>(g.a)[static_cast<size_t>(m0 + r) * kw + k0 + k] : 0;
#pragma unroll
      for (int h = 0; h < (SILU ? 2 : 1); ++h)
        sw[h][r][k] = in && n0 + r < n_out ? reinterpret_cast<const int*>(g.w)[static_cast<size_t>(h * n_out + n0 + r) * kw + k0 + k] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int h = 0; h < (SILU ? 2 : 1); ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[h][i][j] = __dp4a(sa[ty + 16 * i][k], sw[h][tx + 16 * j][k], acc[h][i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= g.M || n >= n_out) continue;
      float v[SILU ? 2 : 1];
#pragma unroll
      for (int h = 0; h < (SILU ? 2 : 1); ++h) {
        v[h] = static_cast<float>(acc[h][i][j]) * g.a_scales[m] * g.w_scales[h * n_out + n];
        if (g.bias) v[h] += load_elem<OUT>(g.bias, h * n_out + n);
      }
      store_elem<OUT>(g.c, static_cast<size_t>(m) * n_out + n, SILU ? silu_mul(v[0], v[SILU ? 1 : 0]) : v[0]);
    }
}

template <int OUT>
static void gemm(const Args& g, int epilogue, int64_t stream) {
  const bool silu = epilogue == B200_EPI_SILU_MUL;
  B200_CHECK_ARG(g.a && g.a_scales && g.w && g.w_scales && g.c && g.N > 0 && g.K > 0, "gemm_i8: bad arguments");
  B200_CHECK_ARG(g.K % 16 == 0 && g.K <= kMaxK, "gemm_i8: k must be a multiple of 16 and at most 131056");
  B200_CHECK_ARG(((reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.w)) & 15) == 0,
                 "gemm_i8: rows and weights must be 16-byte aligned");
  B200_CHECK_ARG(epilogue == B200_EPI_NONE || (silu && g.N % 2 == 0), "gemm_i8: unknown epilogue, or an odd number of gate and up rows");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int n_out = silu ? g.N / 2 : g.N;
  const dim3 grid((n_out + 63) / 64, (g.M + 63) / 64);
  if (silu) launch_pdl(simple_kernel<OUT, true>, grid, dim3(256), 0, st, g);
  else launch_pdl(simple_kernel<OUT, false>, grid, dim3(256), 0, st, g);
  B200_CUDA_LAUNCH_CHECK();
}

}  // namespace gemm8
}  // namespace b200

#define B200_GEMM_I8(SUFFIX, OUT)                                                                                              \
  extern "C" void b200_gemm_i8_##SUFFIX(const void* a, const float* a_scales, const void* w, const float* w_scales,            \
                                        const void* bias, void* c, int32_t m, int32_t n, int32_t k, int32_t epilogue,          \
                                        int64_t stream) {                                                                      \
    using namespace b200;                                                                                                      \
    if (m <= 0) return;                                                                                                        \
    gemm8::gemm<gemm8::OUT>({static_cast<const int8_t*>(a), a_scales, static_cast<const int8_t*>(w), w_scales, bias, c, m, n, k}, \
                            epilogue, stream);                                                                                 \
  }
B200_GEMM_I8(f16, kF16)
B200_GEMM_I8(bf16, kBF16)
B200_GEMM_I8(f32, kF32)
