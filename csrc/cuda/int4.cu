// Matrix-vector products of expert rows with 4-bit weights and group scales:
//   y[r, n] = sum over groups G of scale[e, n, G] * sum over k in G of (q[e, n, k] - 8) * x[r, k]
// for the rows r of expert e's segments.
//
// The weights are read once and are what bounds a few rows, so a weight may cost little more than one
// instruction.  Eight 4-bit values of a word become four registers of two 16-bit numbers each (mask, or in an
// exponent, subtract: exact in bf16 and fp16), which are fragments of a 16 x 16 matrix-unit product with up to
// 8 rows of x as the other side; its sums are fp32.  One group's sum is scaled in fp32 and added to the total,
// so a scale is never rounded into a weight.
//
// A lane holds weight rows g and g + 8 (g = lane / 4) and, of every group, the group / 4 values from
// (lane % 4) * group / 4 on; x is staged in shared memory in that order, so a fragment is one conflict-free
// 16-byte load.  A CTA of 8 warps covers 128 weight rows; a cluster of 1 to 8 CTAs splits the inner size and
// joins its fp32 sums through distributed shared memory in the order of the CTAs.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cstdint>
#include <type_traits>

#include "vb/launch.h"

namespace vb {
namespace {

constexpr int kThreads = 256;
constexpr int kTileN = 128;           // weight rows of a CTA, 16 per warp
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

__device__ __forceinline__ unsigned bits(__nv_bfloat162 v) { return *reinterpret_cast<unsigned*>(&v); }
__device__ __forceinline__ unsigned bits(__half2 v) { return *reinterpret_cast<unsigned*>(&v); }

// q - 8 of the 4-bit values at bits [0, 4) and [16, 20): 128 + q in bf16 and 1024 + q in fp16 have q in their
// lowest mantissa bits, and the difference is exact
template <typename T> __device__ __forceinline__ unsigned two_values(unsigned w);
template <> __device__ __forceinline__ unsigned two_values<__nv_bfloat16>(unsigned w) {
  const unsigned u = (w & 0x000f000fu) | 0x43004300u;
  return bits(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(136.f)));
}
template <> __device__ __forceinline__ unsigned two_values<__half>(unsigned w) {
  const unsigned u = (w & 0x000f000fu) | 0x64006400u;
  return bits(__hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(1032.f)));
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                    unsigned b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// VEC words (8 values each) of one lane's part of a group, read once
template <int VEC>
__device__ __forceinline__ void load_words(unsigned (&w)[VEC], const unsigned char* p) {
  if constexpr (VEC == 4)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  else if constexpr (VEC == 2)
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  else
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
}

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float remote_f(unsigned addr, unsigned rank) {
  unsigned there;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}

struct Geometry {
  long long slice;     // inner values of one CTA of the cluster, a multiple of the chunk's group
  int chunk;           // inner values staged at a time
  int aligned;         // rows of x can be read 16 bytes at a time
  unsigned n_tiles, items;
};

// rows [first, first + count) of segment s inside the matrix
__device__ __forceinline__ void segment(const Int4Args& a, int s, long long& first, long long& count) {
  const long long lo = a.starts[s], hi = lo + a.counts[s];
  first = lo < 0 ? 0 : lo;
  count = (hi > a.rows ? a.rows : hi) - first;
  if (count < 0) count = 0;
}

template <typename T, typename S, int VEC, int NT>
__global__ void __launch_bounds__(kThreads) int4_product_kernel(Int4Args a, Geometry geo) {
  constexpr int GROUP = 32 * VEC;
  constexpr int TOK = 8 * NT;               // rows of x of one item
  constexpr int DEPTH = 16 / VEC;           // groups in flight per warp: 4 KB
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int pick[3];                   // segment, first row, rows of this CTA's item
  __shared__ int scan[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned rank = cluster_rank(), ranks = cluster_size();
  const int item = (int)(blockIdx.x / ranks / geo.n_tiles);
  const long long n0 = (long long)(blockIdx.x / ranks % geo.n_tiles) * kTileN;

  // which segment and rows: the items count the segments' tiles of TOK rows
  {
    const int per = (a.segments + kThreads - 1) / kThreads, s0 = tid * per;
    int mine = 0;
    for (int s = s0; s < s0 + per && s < a.segments; ++s) {
      long long first, count;
      segment(a, s, first, count);
      mine += (int)((count + TOK - 1) / TOK);
    }
    int x = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(kFull, x, off);
      if (lane >= off) x += y;
    }
    if (lane == 31) scan[warp] = x;
    if (tid == 0) pick[0] = -1;
    __syncthreads();
    int before = x - mine;
    for (int w = 0; w < warp; ++w) before += scan[w];
    if (item >= before && item < before + mine)
      for (int s = s0; s < s0 + per && s < a.segments; ++s) {
        long long first, count;
        segment(a, s, first, count);
        const int tiles = (int)((count + TOK - 1) / TOK);
        if (item >= before && item < before + tiles) {
          const long long at = (long long)(item - before) * TOK;
          pick[0] = s;
          pick[1] = (int)(first + at);
          pick[2] = (int)(count - at < TOK ? count - at : TOK);
        }
        before += tiles;
      }
    __syncthreads();
  }

  if (pick[0] >= 0) {                       // the same for every CTA of the cluster
    const int expert = pick[0] % a.experts, row0 = pick[1], tokens = pick[2];
    const int g = lane >> 2, tq = lane & 3;
    const long long groups = a.inner / GROUP;
    const long long k_lo = rank * geo.slice, k_hi = min(a.inner, k_lo + geo.slice);
    const long long n_a = n0 + warp * 16 + g, n_b = n_a + 8;
    const long long base = (long long)expert * a.n;
    // rows past the last are clamped to it and not written
    const unsigned char* qa = a.packed + (base + min(n_a, a.n - 1)) * (a.inner / 2) + tq * (4 * VEC);
    const unsigned char* qb = a.packed + (base + min(n_b, a.n - 1)) * (a.inner / 2) + tq * (4 * VEC);
    const T* x = static_cast<const T*>(a.x);
    uint4* xs = reinterpret_cast<uint4*>(smem);                       // [chunk / 32 units][TOK][4]
    S* sc = reinterpret_cast<S*>(smem + (size_t)geo.chunk * TOK * 2); // [chunk / GROUP][kTileN]
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;

    for (long long c0 = k_lo; c0 < k_hi; c0 += geo.chunk) {
      const int len = (int)min((long long)geo.chunk, k_hi - c0);      // a multiple of GROUP
      const int units = len / GROUP;
      const unsigned char* wa = qa + c0 / 2;
      const unsigned char* wb = qb + c0 / 2;
      unsigned ra[DEPTH][VEC], rb[DEPTH][VEC];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d)
        if (d < units) {
          load_words<VEC>(ra[d], wa + d * (GROUP / 2));
          load_words<VEC>(rb[d], wb + d * (GROUP / 2));
        }
      // stage x: 16-byte units of 8 inner values in the order 0 4 1 5 2 6 3 7
      for (int i = tid; i < len / 8 * TOK; i += kThreads) {
        const int token = i / (len / 8), k8 = i % (len / 8);
        T v[8];
        if (token < tokens) {
          const T* p = x + (row0 + token) * a.x_stride + c0 + 8 * k8;
          if (geo.aligned) {
            *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[e];
          }
        } else {
          *reinterpret_cast<uint4*>(v) = make_uint4(0, 0, 0, 0);
        }
        T o[8] = {v[0], v[4], v[1], v[5], v[2], v[6], v[3], v[7]};
        const int grp = k8 / (4 * VEC), in = k8 % (4 * VEC);          // in = tq * VEC + word
        xs[((grp * VEC + in % VEC) * TOK + token) * 4 + in / VEC] = *reinterpret_cast<uint4*>(o);
      }
      for (int i = tid; i < units * kTileN; i += kThreads) {
        const int row = i / units, u = i % units;
        const long long n = min(n0 + row, a.n - 1);
        sc[u * kTileN + row] = static_cast<const S*>(a.scales)[(base + n) * groups + c0 / GROUP + u];
      }
      __syncthreads();
      for (int u0 = 0; u0 < units; u0 += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
          const int u = u0 + d;
          if (u < units) {
            float part[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) part[t][i] = 0.f;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              unsigned va[4], vb[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                va[i] = two_values<T>(ra[d][v] >> (4 * i));
                vb[i] = two_values<T>(rb[d][v] >> (4 * i));
              }
#pragma unroll
              for (int t = 0; t < NT; ++t)
                if (8 * t < tokens) {
                  const uint4 b = xs[((u * VEC + v) * TOK + 8 * t + g) * 4 + tq];
                  mma<T>(part[t], va[0], vb[0], va[1], vb[1], b.x, b.y);
                  mma<T>(part[t], va[2], vb[2], va[3], vb[3], b.z, b.w);
                }
            }
            if (u + DEPTH < units) {
              load_words<VEC>(ra[d], wa + (u + DEPTH) * (GROUP / 2));
              load_words<VEC>(rb[d], wb + (u + DEPTH) * (GROUP / 2));
            }
            const float sa = to_f(sc[u * kTileN + warp * 16 + g]), sb = to_f(sc[u * kTileN + warp * 16 + g + 8]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              acc[t][0] = fmaf(sa, part[t][0], acc[t][0]);
              acc[t][1] = fmaf(sa, part[t][1], acc[t][1]);
              acc[t][2] = fmaf(sb, part[t][2], acc[t][2]);
              acc[t][3] = fmaf(sb, part[t][3], acc[t][3]);
            }
          }
        }
      }
      __syncthreads();
    }

    // join the cluster's sums: sums[token][row], CTA `rank` finishes every ranks-th part of the outputs
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int token = 8 * t + 2 * tq, row = warp * 16 + g;
      sums[token * kTileN + row] = acc[t][0];
      sums[(token + 1) * kTileN + row] = acc[t][1];
      sums[token * kTileN + row + 8] = acc[t][2];
      sums[(token + 1) * kTileN + row + 8] = acc[t][3];
    }
    if (ranks > 1) cluster_sync(); else __syncthreads();
    const unsigned sums_at = (unsigned)__cvta_generic_to_shared(sums);
    T* out = static_cast<T*>(a.out);
    for (int i = rank * kThreads + tid; i < tokens * kTileN; i += ranks * kThreads) {
      const int token = i / kTileN, row = i % kTileN;
      float v = 0.f;
      for (unsigned r = 0; r < ranks; ++r) v += remote_f(sums_at + 4u * i, r);
      if (n0 + row < a.n) out[(row0 + token) * a.out_stride + n0 + row] = from_f<T>(v);
    }
    if (ranks > 1) cluster_sync();          // the sums stay until every CTA has read them
  }

  // rows that no segment covers are zero; row r belongs to item r mod the items
  if (rank == 0)
    for (long long r = item + (long long)warp * geo.items; r < a.rows; r += 8ll * geo.items) {
      bool covered = false;
      for (int s = lane; s < a.segments; s += 32) {
        const long long lo = a.starts[s];
        covered |= r >= lo && r < lo + a.counts[s];
      }
      if (!__any_sync(kFull, covered))
        for (int c = lane; c < kTileN && n0 + c < a.n; c += 32) static_cast<T*>(a.out)[r * a.out_stride + n0 + c] = from_f<T>(0.f);
    }
}

template <typename T, typename S, int VEC, int NT>
cudaError_t launch(const Int4Args& a, cudaStream_t stream) {
  constexpr int TOK = 8 * NT, GROUP = 32 * VEC;
  // tiles: every segment's last may be partial
  const long long items = (a.rows + TOK - 1) / TOK + (a.segments < a.rows ? a.segments : a.rows) - 1;
  const long long n_tiles = (a.n + kTileN - 1) / kTileN;
  // split the inner size until the GPU is full, as long as a CTA keeps 256 values
  int ranks = 1;
  while (ranks < 8 && n_tiles * items * ranks < 148 * 4 && a.inner / (2 * ranks) >= 256) ranks *= 2;
  Geometry geo{};
  const long long groups = a.inner / GROUP;
  geo.slice = (groups + ranks - 1) / ranks * GROUP;
  const long long most = 2048 / NT;
  geo.chunk = (int)(geo.slice < most ? geo.slice : most);
  geo.n_tiles = (unsigned)n_tiles;
  geo.items = (unsigned)items;
  geo.aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride % 8 == 0;
  size_t bytes = (size_t)geo.chunk * TOK * 2 + (size_t)geo.chunk / GROUP * kTileN * sizeof(S);
  const size_t sums = sizeof(float) * TOK * kTileN;
  if (bytes < sums) bytes = sums;
  auto kernel = int4_product_kernel<T, S, VEC, NT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t config{};
  if (n_tiles * items * ranks > INT_MAX) return cudaErrorInvalidConfiguration;
  config.gridDim = dim3((unsigned)(n_tiles * items * ranks));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, a, geo);
}

template <typename T, typename S, int VEC>
cudaError_t launch_tokens(const Int4Args& a, cudaStream_t stream) {
  return a.rows <= 8 ? launch<T, S, VEC, 1>(a, stream) : launch<T, S, VEC, 4>(a, stream);
}

template <typename T, typename S>
cudaError_t launch_group(const Int4Args& a, cudaStream_t stream) {
  if (a.group == 128) return launch_tokens<T, S, 4>(a, stream);
  if (a.group == 64) return launch_tokens<T, S, 2>(a, stream);
  return launch_tokens<T, S, 1>(a, stream);
}

}  // namespace

cudaError_t launch_int4_product(const Int4Args& a, cudaStream_t stream) {
  if (a.rows == 0 || a.n == 0) return cudaSuccess;
  if (a.dtype == DT_BF16)
    return a.scales_fp32 ? launch_group<__nv_bfloat16, float>(a, stream) : launch_group<__nv_bfloat16, __nv_bfloat16>(a, stream);
  return a.scales_fp32 ? launch_group<__half, float>(a, stream) : launch_group<__half, __half>(a, stream);
}

}  // namespace vb
