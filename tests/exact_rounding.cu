// Compares dense.cuh's reciprocals and roots with the library's, bit for bit, over every float
// that they take.  Prints how many differ: reciprocals, roots.
//
// A warp in which one value is outside a method's range takes the library for all of its values, so
// each sweep is run twice: as it is, and with those values replaced by a neighbour in range.
#include <cstdio>

#include "dense.cuh"

using namespace eps_b200::dense;

template <bool ROOTS, bool REPLACE>
__global__ void compare(unsigned first, unsigned last, unsigned long long* differing) {
  const unsigned stride = gridDim.x * blockDim.x * 8;
  unsigned long long n = 0;
  for (unsigned long long base = first; base <= last; base += stride) {
    float x[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned long long at = base + (blockIdx.x * blockDim.x + threadIdx.x) * 8ull + i;
      unsigned u = at <= last ? (unsigned)at : last;
      if (REPLACE && !ROOTS && (u & 0x7FFFFF) == 0x7FFFFF) --u;
      x[i] = __uint_as_float(u);
      y[i] = x[i];
    }
    if (ROOTS) roots(x, y);
    else reciprocals<8>(y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float want = ROOTS ? __fsqrt_rn(x[i]) : __fdiv_rn(1.f, x[i]);
      n += __float_as_uint(y[i]) != __float_as_uint(want) && !(y[i] != y[i] && want != want);
    }
  }
  if (n) atomicAdd(differing, n);
}

template <bool ROOTS, bool REPLACE>
static unsigned long long differing(unsigned first, unsigned last) {
  unsigned long long *d, n = ~0ull;
  if (cudaMalloc(&d, sizeof n) != cudaSuccess || cudaMemset(d, 0, sizeof n) != cudaSuccess) return n;
  compare<ROOTS, REPLACE><<<148 * 4, 256>>>(first, last, d);
  if (cudaMemcpy(&n, d, sizeof n, cudaMemcpyDeviceToHost) != cudaSuccess) n = ~0ull;
  cudaFree(d);
  return n;
}

int main() {
  const unsigned one = 0x3F800000u, top = 0x71800000u, nan = 0x7FC00000u, low = 0x0F800000u, infinity = 0x7F800000u;
  const unsigned long long r = differing<false, false>(one, nan) + differing<false, true>(one, top);
  const unsigned long long s = differing<true, false>(0, nan) + differing<true, true>(low, infinity - 1);
  std::printf("%llu %llu\n", r, s);
  return r || s;
}
