// Rows of 16-bit activations to 8-bit integers with a scale per row: plain, behind an RMS norm, and behind the residual's
// addition and an RMS norm (what the int8 products of int8_gemm.cu read; the 16-bit forms are rmsnorm_kernel of glue.cu).
//
//   t = x (plain) or x * w (norm);   A = max|t|;   scale = A / 127 (norm: A / (127 rms));   q = round(127 t / A)
//
// The norm's 1 / rms multiplies numerator and maximum alike, so it appears in the scale alone and one pass over the row gives
// the sum of squares and the maximum together.  t is exact in fp32 (two 16-bit factors).  The quotient is rounded to the nearest
// integer, ties to even, EXACTLY: fp32 decides unless it lies within 3e-5 of a border (its error is below 127 * 2^-23), then
// 254 |t| is compared with (2 floor + 1) A in fp64, where both are exact.  So codes do not depend on how threads share a row.
// A row of zeros has scale 0 and codes 0.  A row with a NaN or an infinity has scale NaN and codes 0: all that is computed from
// it is NaN.  Maxima are taken over the bits, where every NaN is larger than infinity.
#include "../../include/b200_vllm.h"
#include "common.cuh"

namespace b200 {
namespace rows8 {

struct Args {
  int8_t* out;
  float* scales;
  uint16_t* residual;
  const uint16_t* x;
  const uint16_t* w;
  int rows, width;
  float eps;
};

// How a row's codes follow from its maximum.
struct Coder {
  float mul, up, top;
  __device__ __forceinline__ explicit Coder(float top_) : top(top_) {
    up = top < 1e-30f ? 18446744073709551616.f : 1.f;        // 2^64: 127 / A would overflow (exact, as is t * up)
    mul = top > 0.f ? 127.f / (top * up) : 0.f;
  }
  // the code in the low byte
  __device__ __forceinline__ uint32_t operator()(float t) const {
    constexpr float kMagic = 12582912.f;                       // 1.5 * 2^23: a sum with it is rounded to an integer
    const float u = t * up;
    float m = fmaf(u, mul, kMagic);
    const float k = m - kMagic;
    const float d = fabsf(fmaf(u, mul, -k));
    if (d > 0.49997f) {
      const float f = floorf(fabsf(u * mul));
      const double lhs = 254.0 * fabs(static_cast<double>(t)), rhs = (2.0 * static_cast<double>(f) + 1.0) * static_cast<double>(top);
      const bool odd = static_cast<int>(f) & 1;
      const float r = lhs > rhs || (lhs == rhs && odd) ? f + 1.f : f;
      m = copysignf(r, t) + kMagic;
    }
    return __float_as_uint(m);
  }
};

__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Eight elements of a row from index i on.  VEC: 16-byte accesses (width a multiple of 8, all aligned).
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* p, int i, int width) {
  if constexpr (VEC) {
    return *reinterpret_cast<const uint4*>(p + i);
  } else {
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = i + 2 * j < width ? p[i + 2 * j] : 0u, hi = i + 2 * j + 1 < width ? p[i + 2 * j + 1] : 0u;
      h[j] = lo | hi << 16;
    }
    return make_uint4(h[0], h[1], h[2], h[3]);
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* p, int i, int width, const uint4& v) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(p + i) = v;
  } else {
    const uint32_t h[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < width) p[i + j] = static_cast<uint16_t>(h[j >> 1] >> (16 * (j & 1)));
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(int8_t* p, int i, int width, uint32_t lo, uint32_t hi) {
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(p + i) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < width) p[i + j] = static_cast<int8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
}

// The values t of eight elements; the sum of squares and the bits of the maximum so far take them in.
template <bool BF, bool NORM>
__device__ __forceinline__ void take8(const uint4& a, const uint4& w, float (&t)[8], float& ss, uint32_t& top) {
  const uint32_t ah[4] = {a.x, a.y, a.z, a.w}, wh[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float2 f = unpack16x2<BF>(ah[j]);
    if constexpr (NORM) {
      const float2 g = unpack16x2<BF>(wh[j]);
      ss = fmaf(f.x, f.x, ss);
      ss = fmaf(f.y, f.y, ss);
      f.x *= g.x;
      f.y *= g.y;
    }
    t[2 * j] = f.x;
    t[2 * j + 1] = f.y;
    top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
  }
}
template <bool BF>
__device__ __forceinline__ uint4 add8(uint4 a, const uint4& r) {
  a.x = add16x2<BF>(a.x, r.x);
  a.y = add16x2<BF>(a.y, r.y);
  a.z = add16x2<BF>(a.z, r.z);
  a.w = add16x2<BF>(a.w, r.w);
  return a;
}

// A block per row, NC pieces of eight elements per thread (0: as many as it takes, read twice).
template <bool BF, bool NORM, bool ADD, bool VEC, int NC>
__global__ void rows_i8_kernel(const Args a) {
  pdl_trigger();
  pdl_wait();
  __shared__ float red_ss[32];
  __shared__ uint32_t red_top[32];
  const size_t at = static_cast<size_t>(blockIdx.x) * a.width;
  const uint16_t* x = a.x + at;
  uint16_t* res = ADD ? a.residual + at : nullptr;
  int8_t* out = a.out + at;
  const int step = blockDim.x * 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float ss = 0.f;
  uint32_t top = 0;

  auto fetch = [&](int i, float (&t)[8]) {
    uint4 v = load8<VEC>(x, i, a.width);
    if constexpr (ADD) {
      v = add8<BF>(v, load8<VEC>(res, i, a.width));
      store8<VEC>(res, i, a.width, v);
    }
    take8<BF, NORM>(v, NORM ? load8<VEC>(a.w, i, a.width) : make_uint4(0, 0, 0, 0), t, ss, top);
  };
  float t[NC ? NC : 1][8];
  if constexpr (NC) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = threadIdx.x * 8 + c * step;
      if (i < a.width) fetch(i, t[c]);
    }
  } else {
    for (int i = threadIdx.x * 8; i < a.width; i += step) fetch(i, t[0]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (NORM) ss = warp_sum(ss);
  if (lane == 0) {
    red_top[warp] = top;
    red_ss[warp] = ss;
  }
  __syncthreads();
  const int warps = blockDim.x >> 5;
  ss = 0.f;
  for (int i = 0; i < warps; ++i) {
    top = max(top, red_top[i]);
    if constexpr (NORM) ss += red_ss[i];
  }
  const bool finite = top < 0x7f800000u;
  const float A = __uint_as_float(top);
  if (threadIdx.x == 0) {
    float s = A;
    if constexpr (NORM) s *= rsqrtf(ss / static_cast<float>(a.width) + a.eps);
    a.scales[blockIdx.x] = finite ? s / 127.f : __uint_as_float(0x7fc00000u);
  }
  const Coder code(finite ? A : 0.f);
  auto put = [&](int i, const float (&v)[8]) {
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = finite ? code(v[j]) : 0u;
    store8<VEC>(out, i, a.width, low_bytes(q[0], q[1], q[2], q[3]), low_bytes(q[4], q[5], q[6], q[7]));
  };
  if constexpr (NC) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = threadIdx.x * 8 + c * step;
      if (i < a.width) put(i, t[c]);
    }
  } else {
    for (int i = threadIdx.x * 8; i < a.width; i += step) {
      const uint4 v = ADD ? load8<VEC>(res, i, a.width) : load8<VEC>(x, i, a.width);
      take8<BF, NORM>(v, NORM ? load8<VEC>(a.w, i, a.width) : make_uint4(0, 0, 0, 0), t[0], ss, top);
      put(i, t[0]);
    }
  }
}

template <bool BF, bool NORM, bool ADD, bool VEC>
static void launch(const Args& a, cudaStream_t st) {
  const int pieces = (a.width + 7) / 8;
  const auto go = [&](auto kern, int nc) {
    const int threads = nc ? ((pieces + nc - 1) / nc + 31) / 32 * 32 : 1024;
    launch_pdl(kern, dim3(a.rows), dim3(threads), 0, st, a);
    B200_CUDA_LAUNCH_CHECK();
  };
  if (pieces <= 256) go(rows_i8_kernel<BF, NORM, ADD, VEC, 1>, 1);
  else if (pieces <= 1024) go(rows_i8_kernel<BF, NORM, ADD, VEC, 2>, 2);
  else if (pieces <= 4096) go(rows_i8_kernel<BF, NORM, ADD, VEC, 4>, 4);
  else go(rows_i8_kernel<BF, NORM, ADD, VEC, 0>, 0);
}

template <bool BF, bool NORM, bool ADD>
static void rows_i8(void* out, float* scales, void* residual, const void* x, const void* w, int rows, int width, float eps,
                    int64_t stream) {
  const Args a{static_cast<int8_t*>(out), scales, static_cast<uint16_t*>(residual), static_cast<const uint16_t*>(x),
               static_cast<const uint16_t*>(w), rows, width, eps};
  const uintptr_t wide = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(w);
  const bool vec = width % 8 == 0 && (wide & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (vec) launch<BF, NORM, ADD, true>(a, st);
  else launch<BF, NORM, ADD, false>(a, st);
}

}  // namespace rows8
}  // namespace b200

#define B200_ROWS_I8(SUFFIX, BF)                                                                                               \
  extern "C" void b200_rmsnorm_i8_##SUFFIX(void* out, float* scales, const void* x, const void* weight, int32_t num_tokens,    \
                                           int32_t hidden, float eps, int64_t stream) {                                        \
    using namespace b200;                                                                                                      \
    if (num_tokens <= 0) return;                                                                                               \
    B200_CHECK_ARG(out && scales && x && weight && hidden > 0, "rmsnorm_i8: bad arguments");                                   \
    rows8::rows_i8<BF, true, false>(out, scales, nullptr, x, weight, num_tokens, hidden, eps, stream);                         \
  }                                                                                                                            \
  extern "C" void b200_add_rmsnorm_i8_##SUFFIX(void* out, float* scales, void* residual, const void* x, const void* weight,    \
                                               int32_t num_tokens, int32_t hidden, float eps, int64_t stream) {                \
    using namespace b200;                                                                                                      \
    if (num_tokens <= 0) return;                                                                                               \
    B200_CHECK_ARG(out && scales && residual && x && weight && hidden > 0, "add_rmsnorm_i8: bad arguments");                   \
    rows8::rows_i8<BF, true, true>(out, scales, residual, x, weight, num_tokens, hidden, eps, stream);                         \
  }                                                                                                                            \
  extern "C" void b200_quant_rows_i8_##SUFFIX(void* out, float* scales, const void* x, int32_t rows, int32_t width,            \
                                              int64_t stream) {                                                                \
    using namespace b200;                                                                                                      \
    if (rows <= 0) return;                                                                                                     \
    B200_CHECK_ARG(out && scales && x && width > 0, "quant_rows_i8: bad arguments");                                           \
    rows8::rows_i8<BF, false, false>(out, scales, nullptr, x, nullptr, rows, width, 0.f, stream);                              \
  }
B200_ROWS_I8(f16, false)
B200_ROWS_I8(bf16, true)
