// Division of small numbers by one that is known at run time.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define TF_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TF_HOST_DEVICE inline
#endif

// i -> (i / n, i % n) for i >= 0, n >= 1, i + n < 2^31, by a multiplication.  m = ceil(2^32 / n) is less than 1 above 2^32 / n, so i m / 2^32 is less than
// i / 2^32 < 1/2 above i / n: its floor is the quotient or one more, and a remainder below zero tells.
struct Divide {
  int n;
  uint32_t m;
  TF_HOST_DEVICE explicit Divide(int n_) : n(n_), m(n_ > 1 ? 0xffffffffu / (uint32_t)n_ + 1u : 0u) {}
  TF_HOST_DEVICE int operator()(int i, int* rest) const {
    int k = n > 1 ? high((uint32_t)i) : i, r = i - k * n;
    if (r < 0) {
      --k;
      r += n;
    }
    *rest = r;
    return k;
  }
  // The same without looking at the remainder: exact for n <= 8192 and i < 33 n, behind that the quotient may be one too large (the append of 16,384 rows
  // takes 125 us so, 127 with the remainder)
  TF_HOST_DEVICE int small(int i, int* rest) const {
    const int k = n > 1 ? high((uint32_t)i) : i;
    *rest = i - k * n;
    return k;
  }
  TF_HOST_DEVICE int high(uint32_t i) const {
#ifdef __CUDA_ARCH__
    return (int)__umulhi(i, m);            // (written as below the append spills more registers)
#else
    return (int)((uint64_t)i * m >> 32);
#endif
  }
};
