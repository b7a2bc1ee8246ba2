// Matrix-vector products of expert rows with 4-bit weights and group scales:
//   y[r, n] = sum over groups G of scale[e, n, G] * sum over k in G of (q[e, n, k] - 8) * x[r, k]
// for the rows r of expert e's segments.  Products and sums are fp32, rounded once to x's type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vb/launch.h"

namespace vb {
namespace {

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// One warp per output element; a row that no segment covers is zero.
template <typename T, typename S>
__global__ void __launch_bounds__(256) int4_product_kernel(Int4Args a) {
  const int lane = threadIdx.x & 31;
  const long long n = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (n >= a.n) return;
  for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    int found = -1;
    for (int s = lane; s < a.segments; s += 32) {
      const int first = a.starts[s];
      if (r >= first && r < (long long)first + a.counts[s]) found = s;
    }
    found = __reduce_max_sync(0xffffffffu, found);
    float sum = 0.f;
    if (found >= 0) {
      const long long row = (found % a.experts) * a.n + n;
      const unsigned char* q = a.packed + row * (a.inner / 2);
      const S* scale = static_cast<const S*>(a.scales) + row * (a.inner / a.group);
      const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
      for (long long i = lane; i < a.inner / 2; i += 32) {
        const float s = to_f(scale[2 * i / a.group]);
        const int lo = (q[i] & 15) - 8, hi = (q[i] >> 4) - 8;
        sum += s * (lo * to_f(x[2 * i]) + hi * to_f(x[2 * i + 1]));
      }
    }
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) static_cast<T*>(a.out)[r * a.out_stride + n] = from_f<T>(sum);
  }
}

}  // namespace

cudaError_t launch_int4_product(const Int4Args& a, cudaStream_t stream) {
  if (a.rows == 0 || a.n == 0) return cudaSuccess;
  const dim3 grid((unsigned)((a.n + 7) / 8), (unsigned)(a.rows < 65535 ? a.rows : 65535));
  if (a.dtype == DT_BF16) {
    if (a.scales_fp32) int4_product_kernel<__nv_bfloat16, float><<<grid, 256, 0, stream>>>(a);
    else int4_product_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  } else {
    if (a.scales_fp32) int4_product_kernel<__half, float><<<grid, 256, 0, stream>>>(a);
    else int4_product_kernel<__half, __half><<<grid, 256, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace vb
