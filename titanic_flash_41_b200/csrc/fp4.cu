// Rows quantised to MXFP4 (packed e2m1, one UE8M0 scale per 32 inputs) and back; their product is gemm_fp4.cu.
//
//   s = 2^ceil(log2(amax / 6)), at least 2^-127 and at most 2^120 (a stored scale byte is 0 .. 247)      v = e2m1(x / s)
//
// A power of two divides exactly, so every rounding is the formula's, ties to even included.  A block that holds a NaN or an
// infinity gets the scale byte 255 (NaN) and goes on as NaN through the product.
// Layout: values [rows][Kp / 2] (even element in the low nibble), Kp = K rounded up to 256 (two 128-input units), zeros behind
// K; scales in the units of the block-scaled GEMMs, 128 bytes for 32 rows x 128 inputs, byte (row % 32) * 4 + (k / 32) % 4, ordered
// [k / 128][row / 32].
//
// Bound by HBM: a thread takes one block, 64 (or 128) contiguous bytes of a row in, 16 bytes and a scale out.
#include "fp4.cuh"

namespace {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__global__ void __launch_bounds__(128) fp4_quant_kernel(const T* __restrict__ x, long ldx, uint8_t* __restrict__ q,
                                                        uint8_t* __restrict__ sf, int units, int rows, int K, int blocks, int vec) {
  tf_pdl_sync();
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long)rows * blocks) return;
  const int r = (int)(i / blocks), b = (int)(i - (long)r * blocks);
  const T* src = x + (long)r * ldx + b * 32;
  const int n = min(K - b * 32, 32);
  float v[32];
  if (vec && n == 32) {
    constexpr int V = 16 / sizeof(T);
    T raw[32];
#pragma unroll
    for (int j = 0; j < 32 / V; ++j) *reinterpret_cast<uint4*>(raw + j * V) = *reinterpret_cast<const uint4*>(src + j * V);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = to_f<T>(raw[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = j < n ? to_f<T>(src[j]) : 0.f;
  }
  uint32_t top = 0;                                      // of the magnitudes' bits: NaN and infinity are above all numbers
#pragma unroll
  for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  int code;
  if (top >= 0x7f800000u) {
    code = 255;
  } else {
    // amax = f 2^(e - 127), 1 <= f < 2: amax <= 6 * 2^n from n = e - 129 on where f <= 1.5, else from e - 128
    // (a subnormal amax is below 2^-126 <= 6 * 2^-127)
    code = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0);
    code = min(max(code, 0), 247);
  }
  const float down = __uint_as_float((uint32_t)(254 - code) << 23);        // 2^(127 - code); the block of 255 is not read
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  if (code != 255) {
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j >> 2] |= fp4::f2_to_e2m1x2(v[2 * j] * down, v[2 * j + 1] * down) << 8 * (j & 3);
  }
  *reinterpret_cast<uint4*>(q + ((long)r * blocks + b) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  sf[((long)(b >> 2) * units + (r >> 5)) * 128 + (r & 31) * 4 + (b & 3)] = (uint8_t)code;
}

template <typename T>
__global__ void __launch_bounds__(128) fp4_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sf, int units,
                                                          T* __restrict__ y, long ldy, int rows, int K, int blocks, int vec) {
  tf_pdl_sync();
  const int kb = (K + 31) / 32;
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long)rows * kb) return;
  const int r = (int)(i / kb), b = (int)(i - (long)r * kb);
  const uint4 raw = *reinterpret_cast<const uint4*>(q + ((long)r * blocks + b) * 16);
  const float s = ue8m0_to_float(sf[((long)(b >> 2) * units + (r >> 5)) * 128 + (r & 31) * 4 + (b & 3)]);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  T* dst = y + (long)r * ldy + b * 32;
  const int n = min(K - b * 32, 32);
  T o[32];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h[4];
    fp4::e2m1x8_to_h2x4(w[j], h);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[e]));
      o[8 * j + 2 * e] = (T)(f.x * s);
      o[8 * j + 2 * e + 1] = (T)(f.y * s);
    }
  }
  if (vec && n == 32) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 32 / V; ++j) *reinterpret_cast<uint4*>(dst + j * V) = *reinterpret_cast<const uint4*>(o + j * V);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < n) dst[j] = o[j];
  }
}

template <typename T>
int quant(const void* x, long ldx, void* q, void* sf, int units, int rows, int K, cudaStream_t st) {
  const int blocks = (K + 255) / 256 * 8;
  const int vec = !(reinterpret_cast<uintptr_t>(x) & 15) && ldx * sizeof(T) % 16 == 0;
  const long n = (long)rows * blocks;
  if ((n + 127) / 128 > 0x7fffffffl) return -1;
  tf_launch(fp4_quant_kernel<T>, dim3((unsigned)((n + 127) / 128)), dim3(128), 0, st, (const T*)x, ldx, (uint8_t*)q, (uint8_t*)sf, units,
            rows, K, blocks, vec);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
template <typename T>
int dequant(const void* q, const void* sf, int units, void* y, long ldy, int rows, int K, cudaStream_t st) {
  const int blocks = (K + 255) / 256 * 8;
  const int vec = !(reinterpret_cast<uintptr_t>(y) & 15) && ldy * sizeof(T) % 16 == 0;
  const long n = (long)rows * ((K + 31) / 32);
  if ((n + 127) / 128 > 0x7fffffffl) return -1;
  tf_launch(fp4_dequant_kernel<T>, dim3((unsigned)((n + 127) / 128)), dim3(128), 0, st, (const uint8_t*)q, (const uint8_t*)sf, units, (T*)y,
            ldy, rows, K, blocks, vec);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace

// x [rows, K] (kind 0 f32, 1 f16, 2 bf16; row pitch ldx elements) -> q [rows, Kp / 2], sf [Kp / 128][units][128]
TF_API int tf_fp4_quant_rows(const void* x, int kind, long ldx, void* q, void* sf, int units, int rows, int K, cudaStream_t st) {
  if (!x || !q || !sf || rows < 1 || K < 1 || ldx < 0 || units * 32l < rows || (reinterpret_cast<uintptr_t>(q) & 15)) return -1;
  if (kind == 0) return quant<float>(x, ldx, q, sf, units, rows, K, st);
  if (kind == 1) return quant<__half>(x, ldx, q, sf, units, rows, K, st);
  if (kind == 2) return quant<__nv_bfloat16>(x, ldx, q, sf, units, rows, K, st);
  return -1;
}

// the numbers that they stand for, y [rows, K] (kind as above; exact in bf16 and f32, in f16 within its range)
TF_API int tf_fp4_dequant_rows(const void* q, const void* sf, int units, void* y, int kind, long ldy, int rows, int K, cudaStream_t st) {
  if (!y || !q || !sf || rows < 1 || K < 1 || ldy < K || units * 32l < rows || (reinterpret_cast<uintptr_t>(q) & 15)) return -1;
  if (kind == 0) return dequant<float>(q, sf, units, y, ldy, rows, K, st);
  if (kind == 1) return dequant<__half>(q, sf, units, y, ldy, rows, K, st);
  if (kind == 2) return dequant<__nv_bfloat16>(q, sf, units, y, ldy, rows, K, st);
  return -1;
}
