// Every float that root_of is used for, against sqrtf; built and run by test_gpu_root.py.
#include "root.cuh"

__global__ void check_kernel(unsigned long long *count) {
  const unsigned long long step = (unsigned long long)gridDim.x * blockDim.x;
  unsigned long long plain = 0, wrong = 0;
  for (unsigned long long i = blockIdx.x * (unsigned long long)blockDim.x + threadIdx.x; i <= 0xFFFFFFFFull; i += step) {
    const unsigned bits = unsigned(i);
    if (!arb::root_is_plain(bits, bits)) continue;
    const float v = __uint_as_float(bits);
    const unsigned other = bits == 0x7E800000u ? bits : bits + 1;  // the pair's second float
    const float w = __uint_as_float(other);
    const float2 r = arb::root_of(make_float2(v, w));
    ++plain;
    wrong += __float_as_uint(r.x) != __float_as_uint(sqrtf(v)) || __float_as_uint(r.y) != __float_as_uint(sqrtf(w)) ||
             __float_as_uint(r.x) != __float_as_uint(float(sqrt(double(v))));
  }
  atomicAdd(&count[0], plain);
  atomicAdd(&count[1], wrong);
}

// count[0]: floats looked at, count[1]: of them different; returns a cudaError_t
extern "C" int check_roots(unsigned long long *count) {
  unsigned long long *d = nullptr;
  cudaError_t e = cudaMalloc(&d, 16);
  if (e == cudaSuccess) e = cudaMemset(d, 0, 16);
  if (e == cudaSuccess) {
    check_kernel<<<148 * 8, 256>>>(d);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpy(count, d, 16, cudaMemcpyDeviceToHost);
  cudaFree(d);
  return int(e);
}
