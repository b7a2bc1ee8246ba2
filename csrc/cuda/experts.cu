// Mixture-of-experts operators on both sides of an AllToAll of tokens: the router's choice, the stable sort of
// assignments by expert, the copy of tokens to their experts' rows and the weighted sum back, with gradients.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vb/launch.h"

namespace vb {
namespace {

constexpr unsigned kFull = 0xffffffffu;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(kFull, v, off);
  return v;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, off));
  return v;
}

// ---- router -------------------------------------------------------------------------------------------

// Unsigned keys in the order of the floats; 0 for what is never chosen (NaN, -inf).  -0 counts as +0.
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned u = __float_as_uint(v + 0.0f);
  if (!(v > -INFINITY)) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One warp per token, NV logits per lane (expert lane + 32 * i).  k rounds take the largest remaining key, ties
// to the lowest expert: one warp maximum of the keys, one warp minimum of the experts that hold it.
template <typename T, int NV>
__global__ void __launch_bounds__(256) route_kernel(RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const long long t = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.logits_stride;
  float v[NV];
  unsigned key[NV];
  float m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    v[i] = e < a.experts ? to_f(row[e]) : -INFINITY;
    key[i] = order_key(v[i]);
    nan |= v[i] != v[i];
    m = fmaxf(m, v[i]);
  }
  m = warp_max(m);
  nan = __any_sync(kFull, nan);
  float sum = 0.f;
  if (!a.renormalize) {
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += expf(v[i] - m);
    sum = warp_sum(sum);
  }
  int my_id = -1;            // lane j keeps choice j
  float my_v = -INFINITY;
  for (int j = 0; j < a.k; ++j) {
    unsigned best = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(kFull, best);
    if (best == 0) break;
    unsigned at = 0xffffffffu;
#pragma unroll
    for (int i = NV - 1; i >= 0; --i)
      if (key[i] == best) at = lane + 32 * i;
    at = __reduce_min_sync(kFull, at);
    float value = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at == (unsigned)(lane + 32 * i)) { key[i] = 0; value = v[i]; }
    value = __shfl_sync(kFull, value, at & 31);
    if (lane == j) { my_id = (int)at; my_v = value; }
  }
  float w = my_id >= 0 ? expf(my_v - m) : 0.f;
  if (a.renormalize) sum = warp_sum(w);
  if (my_id >= 0) w = nan ? __int_as_float(0x7fffffff) : w / sum;
  if (lane < a.k) {
    a.ids[t * a.k + lane] = my_id;
    a.weights[t * a.k + lane] = w;
  }
}

// dl = w (g - <g, w>) on the chosen logits (softmax over the chosen), or p (g [chosen] - <g, w>) on all.
template <typename T, int NV>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const long long t = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  int id = -1;
  float w = 0.f, g = 0.f;
  if (lane < a.k) {
    id = a.ids[t * a.k + lane];
    w = a.weights[t * a.k + lane];
    g = a.grad_weights[t * a.k + lane];
  }
  if (id < 0) { w = 0.f; g = 0.f; }
  const float inner = warp_sum(w * g);
  float acc[NV], p[NV];
  T* out = static_cast<T*>(a.grad_logits) + t * a.experts;
  if (!a.renormalize) {
    const T* row = static_cast<const T*>(a.logits) + t * a.logits_stride;
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 32 * i;
      p[i] = e < a.experts ? to_f(row[e]) : -INFINITY;
      m = fmaxf(m, p[i]);
    }
    m = warp_max(m);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      p[i] = m > -INFINITY ? expf(p[i] - m) : 0.f;
      sum += p[i];
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      p[i] = sum == 0.f ? 0.f : p[i] / sum;
      acc[i] = -inner;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) { p[i] = 1.f; acc[i] = 0.f; }
    g = w * (g - inner);
  }
  for (int j = 0; j < a.k; ++j) {
    const int e = __shfl_sync(kFull, id, j);
    const float add = __shfl_sync(kFull, g, j);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e == lane + 32 * i) acc[i] += add;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    if (e < a.experts) out[e] = from_f<T>(p[i] * acc[i]);
  }
}

template <typename T, bool BACKWARD>
void route_launch(const RouteArgs& a, cudaStream_t stream) {
  const unsigned grid = (unsigned)((a.tokens + 7) / 8);
#define VB_ROUTE(NV)                                                        \
  if (a.experts <= 32 * NV) {                                               \
    if (BACKWARD) route_backward_kernel<T, NV><<<grid, 256, 0, stream>>>(a); \
    else route_kernel<T, NV><<<grid, 256, 0, stream>>>(a);                  \
    return;                                                                 \
  }
  VB_ROUTE(1) VB_ROUTE(2) VB_ROUTE(4) VB_ROUTE(8) VB_ROUTE(16) VB_ROUTE(32)
#undef VB_ROUTE
}

template <bool BACKWARD>
cudaError_t route_any(const RouteArgs& a, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  if (a.dtype == DT_F32) route_launch<float, BACKWARD>(a, stream);
  else if (a.dtype == DT_BF16) route_launch<__nv_bfloat16, BACKWARD>(a, stream);
  else route_launch<__half, BACKWARD>(a, stream);
  return cudaGetLastError();
}

// ---- stable sort by expert ------------------------------------------------------------------------------
//
// Each warp owns a contiguous run of assignments.  Pass 1 counts each warp's assignments per expert (the lanes
// that hold one expert elect a leader with match_any, so no count depends on the order of atomics), a scan over
// the warps and the experts turns the counts into each warp's first place per expert, pass 2 hands the places
// out in the order of the assignments.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;

template <typename I>
__device__ __forceinline__ int expert_of(const SortArgs& a, long long i, long long hi) {
  if (i >= hi) return -1;
  const I e = static_cast<const I*>(a.ids)[i];
  return e >= 0 && e < a.experts ? (int)e : -1;
}

template <typename I>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(SortArgs a) {
  extern __shared__ int sm[];
  const int E = a.experts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* hist = sm;                       // [kSortWarps][E]
  int* first = sm + kSortWarps * E;     // [E] first row of each expert
  int* total = first + E;               // [E]
  for (int i = tid; i < kSortWarps * E; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  const long long per = ((a.assignments + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
  const long long lo = warp * per, hi = min(a.assignments, lo + per);
  int* mine = hist + warp * E;
  for (long long base = lo; base < hi; base += 32) {
    const long long i = base + lane;
    const int e = expert_of<I>(a, i, hi);
    const unsigned peers = __match_any_sync(kFull, e);
    if (e >= 0 && lane == __ffs(peers) - 1) mine[e] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  for (int e = tid; e < E; e += kSortThreads) {
    int run = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = hist[w * E + e];
      hist[w * E + e] = run;
      run += c;
    }
    total[e] = run;
  }
  __syncthreads();
  if (warp == 0) {                      // exclusive scan over the experts
    int carry = 0;
    for (int base = 0; base < E; base += 32) {
      const int e = base + lane;
      const int c = e < E ? total[e] : 0;
      int x = c;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(kFull, x, off);
        if (lane >= off) x += y;
      }
      if (e < E) first[e] = carry + x - c;
      carry += __shfl_sync(kFull, x, 31);
    }
  }
  __syncthreads();
  for (int e = tid; e < E; e += kSortThreads) {
    a.starts[e] = a.capacity ? (int)(e * a.capacity) : first[e];
    a.counts[e] = a.capacity && total[e] > a.capacity ? (int)a.capacity : total[e];
  }
  // rows without an assignment
  if (a.capacity) {
    for (long long r = tid; r < a.rows; r += kSortThreads)
      if (r % a.capacity >= total[r / a.capacity]) a.source[r] = -1;
  } else {
    for (long long r = (long long)first[E - 1] + total[E - 1] + tid; r < a.rows; r += kSortThreads) a.source[r] = -1;
  }
  for (long long base = lo; base < hi; base += 32) {
    const long long i = base + lane;
    const int e = expert_of<I>(a, i, hi);
    const unsigned peers = __match_any_sync(kFull, e);
    int place = 0;
    if (e >= 0) place = mine[e] + __popc(peers & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(peers) - 1) mine[e] += __popc(peers);
    __syncwarp();
    if (i < hi) {
      int row = -1;
      if (e >= 0 && !(a.capacity && place >= a.capacity))
        row = a.capacity ? (int)(e * a.capacity + place) : first[e] + place;
      a.slot[i] = row;
      if (row >= 0) a.source[row] = (int)i;
    }
  }
}

// ---- rows -----------------------------------------------------------------------------------------------

// One CTA per token: the token is copied to each of its rows; the rest of the grid clears rows without a token.
template <typename V>
__global__ void __launch_bounds__(256) dispatch_kernel(ExchangeRowsArgs a, long long units) {
  const V* in = static_cast<const V*>(a.in);
  V* out = static_cast<V*>(a.out);
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x)
    for (long long c = threadIdx.x; c < units; c += blockDim.x) {
      const V v = in[t * a.in_stride + c];
      for (int j = 0; j < a.k; ++j) {
        const int r = a.slot[t * a.k + j];
        if (r >= 0 && r < a.rows) out[r * a.out_stride + c] = v;
      }
    }
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x)
    if (a.source[r] < 0)
      for (long long c = threadIdx.x; c < units; c += blockDim.x) out[r * a.out_stride + c] = V{};
}

// One CTA per token: its rows are summed in fp32, in the order of the choices.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(ExchangeRowsArgs a) {
  const T* in = static_cast<const T*>(a.in);
  T* out = static_cast<T*>(a.out);
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x)
    for (long long c = threadIdx.x; c < a.hidden; c += blockDim.x) {
      float acc = 0.f;
      for (int j = 0; j < a.k; ++j) {
        const int r = a.slot[t * a.k + j];
        if (r < 0 || r >= a.rows) continue;
        acc = fmaf(a.weights ? a.weights[t * a.k + j] : 1.f, to_f(in[r * a.in_stride + c]), acc);
      }
      out[t * a.out_stride + c] = from_f<T>(acc);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) combine_backward_kernel(ExchangeRowsArgs a) {
  __shared__ float part[8];
  const T* grad = static_cast<const T*>(a.in);
  const T* rows = static_cast<const T*>(a.saved);
  T* out = static_cast<T*>(a.out);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x)
    for (int j = 0; j < a.k; ++j) {
      const int r = a.slot[t * a.k + j];
      const bool kept = r >= 0 && r < a.rows;
      float dot = 0.f;
      if (kept) {
        const float w = a.weights[t * a.k + j];
        for (long long c = threadIdx.x; c < a.hidden; c += blockDim.x) {
          const float g = to_f(grad[t * a.in_stride + c]);
          dot = fmaf(g, to_f(rows[r * a.saved_stride + c]), dot);
          out[r * a.out_stride + c] = from_f<T>(w * g);
        }
      }
      dot = warp_sum(dot);
      if (lane == 0) part[warp] = dot;
      __syncthreads();
      if (threadIdx.x == 0) {
        float sum = 0.f;
        for (int w = 0; w < 8; ++w) sum += part[w];
        a.grad_weights[t * a.k + j] = sum;
      }
      __syncthreads();
    }
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x)
    if (a.source[r] < 0)
      for (long long c = threadIdx.x; c < a.hidden; c += blockDim.x) out[r * a.out_stride + c] = from_f<T>(0.f);
}

unsigned row_grid(const ExchangeRowsArgs& a, bool rows) {
  const long long n = rows && a.rows > a.tokens ? a.rows : a.tokens;
  return (unsigned)(n < 1 ? 1 : n > 148 * 64 ? 148 * 64 : n);
}

int elem_size(int dtype) { return dtype == DT_F32 ? 4 : 2; }

}  // namespace

cudaError_t launch_route(const RouteArgs& a, cudaStream_t stream) { return route_any<false>(a, stream); }
cudaError_t launch_route_backward(const RouteArgs& a, cudaStream_t stream) { return route_any<true>(a, stream); }

cudaError_t launch_sort(const SortArgs& a, cudaStream_t stream) {
  const size_t bytes = sizeof(int) * ((size_t)kSortWarps + 2) * a.experts;
  auto kernel = a.ids64 ? sort_kernel<long long> : sort_kernel<int>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return e;
  kernel<<<1, kSortThreads, bytes, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_dispatch(const ExchangeRowsArgs& a, cudaStream_t stream) {
  if (a.hidden == 0 || (a.rows == 0)) return cudaSuccess;
  if (elem_size(a.dtype) == 4) dispatch_kernel<unsigned><<<row_grid(a, true), 256, 0, stream>>>(a, a.hidden);
  else dispatch_kernel<unsigned short><<<row_grid(a, true), 256, 0, stream>>>(a, a.hidden);
  return cudaGetLastError();
}

cudaError_t launch_combine(const ExchangeRowsArgs& a, cudaStream_t stream) {
  if (a.hidden == 0 || a.tokens == 0) return cudaSuccess;
  const unsigned grid = row_grid(a, false);
  if (a.dtype == DT_F32) combine_kernel<float><<<grid, 256, 0, stream>>>(a);
  else if (a.dtype == DT_BF16) combine_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else combine_kernel<__half><<<grid, 256, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_combine_backward(const ExchangeRowsArgs& a, cudaStream_t stream) {
  if (a.tokens == 0 && a.rows == 0) return cudaSuccess;
  const unsigned grid = row_grid(a, true);
  if (a.dtype == DT_F32) combine_backward_kernel<float><<<grid, 256, 0, stream>>>(a);
  else if (a.dtype == DT_BF16) combine_backward_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else combine_backward_kernel<__half><<<grid, 256, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace vb
