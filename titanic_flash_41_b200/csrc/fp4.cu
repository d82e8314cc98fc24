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
// Bound by HBM: K * size bytes of a row in, K * 17 / 32 out.  16,384 x 4,096 bf16: 37 us there, 31 - 33 back (0.7 and 0.8 - 0.85 of the copy
// rate; 27 with the packed rows still in L2).
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

// A block's scale byte from the bits of its largest magnitude.  amax = f 2^(e - 127), 1 <= f < 2: amax <= 6 * 2^n from n = e - 129 on
// where f <= 1.5, else from e - 128 (a subnormal amax is below 2^-126 <= 6 * 2^-127).  NaN and infinity are above all numbers.
__device__ __forceinline__ int scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  return min(max((int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0), 0), 247);
}
// 2^(127 - code), the reciprocal of the scale (0 for a block of NaN: its values are not read)
__device__ __forceinline__ float down_of(int code) { return code == 255 ? 0.f : __uint_as_float((uint32_t)(254 - code) << 23); }

// One thread a block.  VEC: rows on 16-byte boundaries and K a multiple of 32.  The wide strides of the loads (64 bytes a lane) are
// served by L1: with four lanes a block, whole lines a load and four loads in flight, the shuffles cost more (16,384 x 4,096 bf16: 59 us
// against 36).
template <typename T, bool VEC>
__global__ void __launch_bounds__(128) fp4_quant_kernel(const T* __restrict__ x, long ldx, uint8_t* __restrict__ q, uint8_t* __restrict__ sf,
                                                        int units, int rows, int K, int blocks) {
  tf_pdl_sync();
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long)rows * blocks) return;
  const int r = i >> 31 ? (int)(i / blocks) : (int)((uint32_t)i / (uint32_t)blocks), b = (int)(i - (long)r * blocks), n = K - b * 32;
  const T* src = x + (long)r * ldx + b * 32;
  float v[32];
  if (VEC) {
    constexpr int V = 16 / sizeof(T);
    T raw[32];
#pragma unroll
    for (int j = 0; j < 32 / V; ++j)
      *reinterpret_cast<uint4*>(raw + j * V) = n > 0 ? __ldg(reinterpret_cast<const uint4*>(src + j * V)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = to_f<T>(raw[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = j < n ? to_f<T>(src[j]) : 0.f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  const int code = scale_byte(top);
  const float down = down_of(code);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float* u = v + 8 * j;
    const float lo[4] = {u[0] * down, u[2] * down, u[4] * down, u[6] * down}, hi[4] = {u[1] * down, u[3] * down, u[5] * down, u[7] * down};
    w[j] = code == 255 ? 0u : fp4::e2m1x8(lo, hi);
  }
  *reinterpret_cast<uint4*>(q + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  sf[((long)(b >> 2) * units + (r >> 5)) * 128 + (r & 31) * 4 + (b & 3)] = (uint8_t)code;
}

template <typename T>
struct Eight {                             // 8 values of a row as they lie in memory
  uint4 w[sizeof(T) / 2];
};
// Back: a lane 8 values, a warp 256 of a row, kAhead such pieces in flight (VEC: rows of y on 16-byte boundaries and K a multiple of
// 8).  16,384 x 4,096 to bf16: 43 us with a thread a block, 31 so.
constexpr int kAhead = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp4_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sf, int units,
                                                          T* __restrict__ y, long ldy, int rows, int K, int pieces) {
  tf_pdl_sync();
  const int lane = threadIdx.x & 31;
  const long items = (long)rows * pieces, first = ((long)blockIdx.x * 8 + (threadIdx.x >> 5)) * kAhead;
  uint32_t w[kAhead], s[kAhead];
  int row[kAhead], piece[kAhead];
  int r = first >> 31 ? (int)(first / pieces) : (int)((uint32_t)first / (uint32_t)pieces), c0 = (int)(first - (long)r * pieces);
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    row[i] = first + i < items ? r : -1;
    piece[i] = c0;
    if (++c0 == pieces) {
      c0 = 0;
      ++r;
    }
    if (row[i] < 0) continue;
    w[i] = __ldg(reinterpret_cast<const uint32_t*>(q) + (first + i) * 32 + lane);
    s[i] = __ldg(reinterpret_cast<const uint32_t*>(sf + ((long)(2 * piece[i] + (lane >> 4)) * units + (row[i] >> 5)) * 128 + (row[i] & 31) * 4));
  }
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    if (row[i] < 0) break;
    const int c = piece[i] * 256 + lane * 8;
    if (c >= K) continue;
    const float f = ue8m0_to_float((uint8_t)(s[i] >> 8 * (lane >> 2 & 3)));
    uint32_t h[4];
    fp4::e2m1x8_to_h2x4(w[i], h);
    Eight<T> o;
    T* t = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 g = __half22float2(*reinterpret_cast<__half2*>(&h[e]));
      t[2 * e] = (T)(g.x * f);
      t[2 * e + 1] = (T)(g.y * f);
    }
    T* dst = y + row[i] * ldy + c;
    if (VEC) {
#pragma unroll
      for (int e = 0; e < (int)sizeof(T) / 2; ++e) reinterpret_cast<uint4*>(dst)[e] = o.w[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < K) dst[e] = t[e];
    }
  }
}

template <typename T>
int quant(const void* x, long ldx, void* q, void* sf, int units, int rows, int K, cudaStream_t st) {
  const int blocks = (K + 255) / 256 * 8;
  const bool vec = !(reinterpret_cast<uintptr_t>(x) & 15) && ldx * sizeof(T) % 16 == 0 && K % 32 == 0;
  const long n = ((long)rows * blocks + 127) / 128;
  if (n > 0x7fffffffl) return -1;
  auto kernel = vec ? fp4_quant_kernel<T, true> : fp4_quant_kernel<T, false>;
  tf_launch(kernel, dim3((unsigned)n), dim3(128), 0, st, (const T*)x, ldx, (uint8_t*)q, (uint8_t*)sf, units, rows, K, blocks);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
template <typename T>
int dequant(const void* q, const void* sf, int units, void* y, long ldy, int rows, int K, cudaStream_t st) {
  const int pieces = (K + 255) / 256;
  const bool vec = !(reinterpret_cast<uintptr_t>(y) & 15) && ldy * sizeof(T) % 16 == 0 && K % 8 == 0;
  const long n = ((long)rows * pieces + 8 * kAhead - 1) / (8 * kAhead);
  if (n > 0x7fffffffl) return -1;
  auto kernel = vec ? fp4_dequant_kernel<T, true> : fp4_dequant_kernel<T, false>;
  tf_launch(kernel, dim3((unsigned)n), dim3(256), 0, st, (const uint8_t*)q, (const uint8_t*)sf, units, (T*)y, ldy, rows, K, pieces);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace

// x [rows, K] (kind 0 f32, 1 f16, 2 bf16; row pitch ldx elements) -> q [rows, Kp / 2], sf [Kp / 128][units][128]
TF_API int tf_fp4_quant_rows(const void* x, int kind, long ldx, void* q, void* sf, int units, int rows, int K, cudaStream_t st) {
  if (!x || !q || !sf || rows < 1 || K < 1 || ldx < 0 || units * 32l < rows || ((reinterpret_cast<uintptr_t>(q) & 15) | (reinterpret_cast<uintptr_t>(sf) & 3))) return -1;
  if (kind == 0) return quant<float>(x, ldx, q, sf, units, rows, K, st);
  if (kind == 1) return quant<__half>(x, ldx, q, sf, units, rows, K, st);
  if (kind == 2) return quant<__nv_bfloat16>(x, ldx, q, sf, units, rows, K, st);
  return -1;
}

// the numbers that they stand for, y [rows, K] (kind as above; exact in bf16 and f32, in f16 within its range)
TF_API int tf_fp4_dequant_rows(const void* q, const void* sf, int units, void* y, int kind, long ldy, int rows, int K, cudaStream_t st) {
  if (!y || !q || !sf || rows < 1 || K < 1 || ldy < K || units * 32l < rows || ((reinterpret_cast<uintptr_t>(q) & 15) | (reinterpret_cast<uintptr_t>(sf) & 3))) return -1;
  if (kind == 0) return dequant<float>(q, sf, units, y, ldy, rows, K, st);
  if (kind == 1) return dequant<__half>(q, sf, units, y, ldy, rows, K, st);
  if (kind == 2) return dequant<__nv_bfloat16>(q, sf, units, y, ldy, rows, K, st);
  return -1;
}
