// Mixture-of-experts operators on both sides of an AllToAll of tokens: the router's choice, the stable sort of
// assignments by expert, the copy of tokens to their experts' rows and the weighted sum back, with gradients.
//
// Times compare forms on one set of inputs, launched again and again: inputs below 126 MB are then in the L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>

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

__device__ __forceinline__ float key_value(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// One warp per token, NV logits per lane (expert lane + 32 * i).  The k-th largest of the lanes' largest keys bounds
// the k-th largest key from below, so only the few keys from it on (k to about 2 k of them) are candidates; they are
// dealt to the lanes, and k rounds take the largest, ties to the lowest expert, in a few instructions each.  More
// than 32 candidates (many equal logits, a k near the experts) take the rounds over all keys, and so do 33 to 64
// experts, whose few keys do not pay for the detour (16384 tokens x 64, k = 2: 4.9 us, with candidates 5.8).  What
// this costs is instructions, not bytes: 16384 tokens x 256 experts, k = 8, fp32, take 12.6 us, with the rounds over
// all keys 17.5, and the bytes alone 2.7.
template <typename T, int NV>
__global__ void __launch_bounds__(256) route_kernel(RouteArgs a) {
  __shared__ unsigned cand_key[8][32];
  __shared__ unsigned cand_expert[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = blockIdx.x * 8ll + warp;
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.logits_stride;
  float v[NV];
  unsigned key[NV], best = 0;
  float m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    v[i] = e < a.experts ? to_f(row[e]) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    key[i] = order_key(v[i]);
    best = max(best, key[i]);
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
  unsigned my_key = 0, my_expert = 0;    // one candidate per lane
  int found = 32;                        // candidates
  if (NV == 1) {
    my_key = key[0];
    my_expert = lane;
  } else if (NV == 2) {
    found = 33;
  } else {
    unsigned bound = 1, rest = best;     // 0 is never chosen
    for (int j = 0; j < a.k; ++j) {
      const unsigned top = __reduce_max_sync(kFull, rest);
      if (top == 0) { bound = 1; break; }
      bound = top;
      if (__ffs(__ballot_sync(kFull, rest == top)) - 1 == lane) rest = 0;
    }
    found = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool in = key[i] >= bound;
      const unsigned votes = __ballot_sync(kFull, in);
      const int at = found + __popc(votes & ((1u << lane) - 1));
      if (in && at < 32) {
        cand_key[warp][at] = key[i];
        cand_expert[warp][at] = lane + 32 * i;
      }
      found += __popc(votes);
    }
    __syncwarp();
    if (found <= 32 && lane < found) {
      my_key = cand_key[warp][lane];
      my_expert = cand_expert[warp][lane];
    }
  }
  int my_id = -1;                        // lane j keeps choice j
  unsigned my_choice = 0;
  if (found <= 32) {
    for (int j = 0; j < a.k; ++j) {
      const unsigned top = __reduce_max_sync(kFull, my_key);
      if (top == 0) break;
      const unsigned at = __reduce_min_sync(kFull, my_key == top ? my_expert : 0xffffffffu);
      if (lane == j) { my_id = (int)at; my_choice = top; }
      if (my_key == top && my_expert == at) my_key = 0;
    }
  } else {
    for (int j = 0; j < a.k; ++j) {
      best = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(kFull, best);
      if (best == 0) break;
      unsigned at = 0xffffffffu;
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
        if (key[i] == best) at = lane + 32 * i;
      at = __reduce_min_sync(kFull, at);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (at == (unsigned)(lane + 32 * i)) key[i] = 0;
      if (lane == j) { my_id = (int)at; my_choice = best; }
    }
  }
  float w = my_id >= 0 ? expf(key_value(my_choice) - m) : 0.f;
  if (a.renormalize) sum = warp_sum(w);
  if (my_id >= 0) w = nan ? __int_as_float(0x7fffffff) : w / sum;
  if (lane < a.k) {
    a.ids[t * a.k + lane] = my_id;
    a.weights[t * a.k + lane] = w;
  }
}

// dl = w (g - <g, w>) on the chosen logits (softmax over the chosen), or p (g [chosen] - <g, w>) on all.  The chosen
// experts' parts go through shared memory to the lanes that hold them.
template <typename T, int NV>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteArgs a) {
  __shared__ float chosen[8][32 * NV];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = blockIdx.x * 8ll + warp;
  if (t >= a.tokens) return;
  int id = -1;
  float w = 0.f, g = 0.f;
  if (lane < a.k) {
    id = a.ids[t * a.k + lane];
    if (id >= 0 && id < a.experts) {
      w = a.weights[t * a.k + lane];
      g = a.grad_weights[t * a.k + lane];
    } else {
      id = -1;
    }
  }
  float p[NV], scale = 1.f;
  if (!a.renormalize) {
    const T* row = static_cast<const T*>(a.logits) + t * a.logits_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 32 * i;
      p[i] = e < a.experts ? to_f(row[e]) : -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) chosen[warp][lane + 32 * i] = 0.f;
  const float inner = warp_sum(w * g);
  if (a.renormalize) g = w * (g - inner);
  // an expert that ids hold twice (no choice of route does) gets the sum in the order of the choices
  const unsigned peers = __match_any_sync(kFull, id);
  float add = g;
  if (__any_sync(kFull, id >= 0 && (peers & (peers - 1)))) {
    add = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const float other = __shfl_sync(kFull, g, j);
      if (peers >> j & 1) add += other;
    }
  }
  __syncwarp();
  if (id >= 0) chosen[warp][id] = add;
  __syncwarp();
  T* out = static_cast<T*>(a.grad_logits) + t * a.experts;
  if (!a.renormalize) {
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, p[i]);
    m = warp_max(m);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      p[i] = m > -INFINITY ? expf(p[i] - m) : 0.f;
      sum += p[i];
    }
    sum = warp_sum(sum);
    scale = sum == 0.f ? 0.f : 1.f / sum;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    const float part = chosen[warp][e];
    if (e < a.experts) out[e] = from_f<T>(a.renormalize ? part : p[i] * scale * (part - inner));
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
// One cluster of 1 to 16 CTAs; every warp owns a contiguous run of assignments.  Pass 1 counts each warp's
// assignments per expert (the lanes that hold one expert find each other by a vote per bit of the expert's number
// and elect a leader, so no count depends on the order of atomics) and leaves each assignment's place among them in
// its slot.  Scans over the warps, over the CTAs (through distributed shared memory) and over the experts turn the
// counts into first rows, which pass 2 adds.  One launch and no workspace: what it costs is the latency of these
// steps and the votes of at most 512 warps, not its few bytes.
constexpr int kSortWarps = 32;         // most warps of a CTA
constexpr int kSortCtas = 16;          // most CTAs of the cluster
constexpr int kSortRun = 32;           // assignments of a warp before another warp or CTA is added (16384
                                       // assignments take 11.0 us with runs of 128, 7.8 with 32)

// The lanes that hold the same expert: a vote per bit.  (match_any does this in one instruction, but sorting 131072
// assignments to 128 experts took 23.5 us with it and takes 17.9 with the votes.)
__device__ __forceinline__ unsigned same_expert(int e, int bits) {
  unsigned peers = kFull;
#pragma unroll 1
  for (int b = 0; b < bits; ++b) {
    const unsigned votes = __ballot_sync(kFull, e >> b & 1);
    peers &= e >> b & 1 ? votes : ~votes;
  }
  return peers;
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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ int remote_int(const int* p, unsigned rank) {
  unsigned there;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(there) : "memory");
  return v;
}

template <typename I>
__device__ __forceinline__ int expert_of(const SortArgs& a, long long i, long long hi) {
  if (i >= hi) return -1;
  const I e = static_cast<const I*>(a.ids)[i];
  return e >= 0 && e < a.experts ? (int)e : -1;
}

__device__ __forceinline__ int inclusive_scan(int x, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(kFull, x, off);
    if (lane >= off) x += y;
  }
  return x;
}

template <typename I>
__global__ void __launch_bounds__(kSortWarps * 32) sort_kernel(SortArgs a) {
  extern __shared__ int sm[];
  constexpr int AHEAD = 4;              // loads of a lane in flight
  const int E = a.experts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int threads = blockDim.x, warps = threads >> 5, pitch = E | 1;   // an odd pitch: a column meets all banks
  const int rank = (int)cluster_rank(), ctas = (int)cluster_size();
  const int bits = 33 - __clz(E);       // -1, no expert, has every bit set: one bit more than an expert's number
  int* hist = sm;                       // [warps][pitch] counts, then first places
  int* total = sm + warps * pitch;      // [E] of this CTA, read by the others
  int* before = total + E;              // [E] assignments of earlier CTAs
  int* all = before + E;                // [E] of the cluster
  int* first = all + E;                 // [E] first row
  for (int i = tid; i < warps * pitch; i += threads) hist[i] = 0;
  __syncthreads();
  const long long workers = (long long)ctas * warps;
  const long long per = ((a.assignments + workers - 1) / workers + 31) / 32 * 32;
  const long long lo = (rank * warps + warp) * per, hi = min(a.assignments, lo + per);
  int* mine = hist + warp * pitch;
  for (long long base = lo; base < hi; base += 32 * AHEAD) {
    int e[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) e[j] = expert_of<I>(a, base + 32 * j + lane, hi);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (base + 32 * j >= hi) break;
      const unsigned peers = same_expert(e[j], bits);
      int place = 0;
      if (e[j] >= 0) place = mine[e[j]] + __popc(peers & ((1u << lane) - 1));
      __syncwarp();
      if (e[j] >= 0 && lane == __ffs(peers) - 1) mine[e[j]] += __popc(peers);
      __syncwarp();
      if (base + 32 * j + lane < hi) a.slot[base + 32 * j + lane] = place;
    }
  }
  __syncthreads();
  for (int e = warp; e < E; e += warps) {
    const int c = lane < warps ? hist[lane * pitch + e] : 0;
    const int x = inclusive_scan(c, lane);
    if (lane < warps) hist[lane * pitch + e] = x - c;
    if (lane == 31) total[e] = x;
  }
  if (ctas > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
  // one thread per expert: the launch has at least as many
  int sum = 0, earlier = 0;
  if (tid < E) {
    if (ctas == 1) sum = total[tid];
    else
      for (int r = 0; r < ctas; ++r) {
        const int c = remote_int(total + tid, r);
        if (r < rank) earlier += c;
        sum += c;
      }
  }
  if (ctas > 1) cluster_arrive();       // this CTA has read the others' totals
  const int upto = inclusive_scan(sum, lane);
  __shared__ int warp_sum_of[kSortWarps];
  if (lane == 31) warp_sum_of[warp] = upto;
  __syncthreads();
  int start = upto - sum;
  for (int w = 0; w < warp; ++w) start += warp_sum_of[w];
  if (tid < E) {
    all[tid] = sum;
    first[tid] = start;
    // pass 2 adds one number: the first row of this CTA's assignments, or their first place under a capacity
    before[tid] = a.capacity ? earlier : start + earlier;
  }
  __syncthreads();
  if (rank == 0)
    for (int e = tid; e < E; e += threads) {
      a.starts[e] = a.capacity ? (int)(e * a.capacity) : first[e];
      a.counts[e] = a.capacity && all[e] > a.capacity ? (int)a.capacity : all[e];
    }
  // rows without an assignment
  if (a.capacity) {
    for (int e = rank * warps + warp; e < E; e += (int)workers)
      for (long long p = all[e] + lane; p < a.capacity; p += 32) a.source[e * a.capacity + p] = -1;
  } else {
    for (long long r = (long long)first[E - 1] + all[E - 1] + rank * threads + tid; r < a.rows; r += (long long)ctas * threads)
      a.source[r] = -1;
  }
  for (long long base = lo; base < hi; base += 32 * AHEAD) {
    int e[AHEAD], place[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const long long i = base + 32 * j + lane;
      e[j] = expert_of<I>(a, i, hi);
      place[j] = i < hi ? a.slot[i] : 0;
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const long long i = base + 32 * j + lane;
      if (i >= hi) continue;
      int row = -1;
      if (e[j] >= 0) {
        place[j] += mine[e[j]] + before[e[j]];
        row = a.capacity == 0 ? place[j] : place[j] < a.capacity ? (int)(e[j] * a.capacity + place[j]) : -1;
      }
      a.slot[i] = row;
      if (row >= 0) a.source[row] = (int)i;
    }
  }
  if (ctas > 1) cluster_wait();         // the totals stay until every CTA has read them
}

// ---- rows -----------------------------------------------------------------------------------------------
//
// All three kernels are bound by the bytes they move.  A warp moves a piece of 2 or 4 vectors a lane of one token
// to or from the token's rows: the token's side is read or written once however many rows it has, and the piece's
// vectors are all in flight together.  Vectors are the widest (16, 8 bytes or one element) that every address,
// stride and row length allows; blockIdx.y is the piece, so no index is divided.  The grid's first
// blocks clear the rows that have no token.
//
// A piece is 1 KB of 16-byte vectors.  Longer pieces, or rows requested ahead, cost registers and with them the
// warps that hide the latency: combining 8192 tokens x 8 rows x 2048 bf16 takes 53.7 us with 2 vectors a lane, 62.2
// with 4 and 70.3 with 2 and a row ahead; dispatching 256 x 8 x 4096 takes 4.7 us with 2 and 6.0 with 4.  Shorter
// vectors take 4 a lane (fp32 rows of 1030: dispatch 22.0 us, with 2 23.2).
//
// Rows that together exceed half of the L2 are read and written as streams (evicted first), as they will not be
// found there again: 8192 x 8 x 2048 bf16 dispatch 50.9 -> 46.9 us, combine 53.7 -> 46.8, its gradient 109 -> 105 us.
// Smaller ones stay for the kernel that follows.
template <int BYTES> constexpr int kPieces = BYTES == 16 ? 2 : 4;
constexpr int kRowWarps = 8;
constexpr long long kStreamBytes = 64ll << 20;

template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = unsigned; };
template <> struct Word<2> { using type = unsigned short; };

template <bool STREAM, typename V>
__device__ __forceinline__ V load_row(const V* p) {
  using W = typename Word<sizeof(V)>::type;
  const W w = STREAM ? __ldcs(reinterpret_cast<const W*>(p)) : *reinterpret_cast<const W*>(p);
  return *reinterpret_cast<const V*>(&w);
}

template <bool STREAM, typename V>
__device__ __forceinline__ void store_row(V* p, const V& v) {
  using W = typename Word<sizeof(V)>::type;
  const W w = *reinterpret_cast<const W*>(&v);
  if (STREAM) __stcs(reinterpret_cast<W*>(p), w);
  else *reinterpret_cast<W*>(p) = w;
}

__device__ __forceinline__ uint4 zero_vec(uint4) { return make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ uint2 zero_vec(uint2) { return make_uint2(0, 0); }
__device__ __forceinline__ unsigned zero_vec(unsigned) { return 0; }
__device__ __forceinline__ unsigned short zero_vec(unsigned short) { return 0; }

// Rows of `source` without an assignment, 32 a warp: the warps of the first `blocks` blocks take every row in turn, as
// the empty rows of an expert lie together and 32 of them at one warp would outlast the copies (30720 rows of 1030
// fp32, 9000 of them empty: 31 us, so 27).
__device__ __forceinline__ unsigned empty_rows(const ExchangeRowsArgs& a, unsigned blocks, long long& first, long long& step) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  first = (long long)blockIdx.x * warps + (threadIdx.x >> 5);
  step = (long long)blocks * warps;
  const long long r = first + lane * step;
  return __ballot_sync(kFull, r < a.rows && a.source[r] < 0);
}

template <typename V>
__device__ __forceinline__ void clear_rows(const ExchangeRowsArgs& a, V* out, long long stride, unsigned blocks, long long units) {
  constexpr int P = kPieces<sizeof(V)>;
  const long long c0 = (long long)blockIdx.y * (32 * P) + (threadIdx.x & 31);
  long long first, step;
  for (unsigned empty = empty_rows(a, blocks, first, step); empty; empty &= empty - 1) {
    V* to = out + (first + (__ffs(empty) - 1) * step) * stride + c0;
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (c0 + 32 * i < units) to[32 * i] = zero_vec(V{});
  }
}

// V-sized vectors; strides and lengths are in vectors
template <typename V, bool STREAM>
__global__ void __launch_bounds__(kRowWarps * 32) dispatch_kernel(ExchangeRowsArgs a, long long units, unsigned clear_blocks) {
  const V* in = static_cast<const V*>(a.in);
  V* out = static_cast<V*>(a.out);
  if (blockIdx.x < clear_blocks) { clear_rows(a, out, a.out_stride, clear_blocks, units); return; }
  const int lane = threadIdx.x & 31;
  const long long t = (long long)(blockIdx.x - clear_blocks) * kRowWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const int mine = lane < a.k ? a.slot[t * a.k + lane] : -1;
  constexpr int P = kPieces<sizeof(V)>;
  const long long c0 = (long long)blockIdx.y * (32 * P) + lane;
  V v[P];
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (c0 + 32 * i < units) v[i] = in[t * a.in_stride + c0 + 32 * i];
  for (int j = 0; j < a.k; ++j) {
    const int r = __shfl_sync(kFull, mine, j);
    if (r < 0 || r >= a.rows) continue;
    V* to = out + r * a.out_stride + c0;
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (c0 + 32 * i < units) store_row<STREAM>(to + 32 * i, v[i]);
  }
}

template <typename T, int N> struct __align__(sizeof(T) * N) Vec { T v[N]; };

// A token's rows are summed in fp32, in the order of the choices (weights nullptr: 1).
template <typename T, int N, bool STREAM>
__global__ void __launch_bounds__(kRowWarps * 32) combine_kernel(ExchangeRowsArgs a, long long units) {
  using V = Vec<T, N>;
  constexpr int P = kPieces<sizeof(V)>;
  const int lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  int mine = -1;
  float weight = 1.f;
  if (lane < a.k) {
    mine = a.slot[t * a.k + lane];
    if (a.weights) weight = a.weights[t * a.k + lane];
    if (mine >= a.rows) mine = -1;
  }
  const long long c0 = (long long)blockIdx.y * (32 * P) + lane;
  const V* in = static_cast<const V*>(a.in) + c0;
  float acc[P][N];
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int n = 0; n < N; ++n) acc[i][n] = 0.f;
  for (unsigned left = __ballot_sync(kFull, mine >= 0); left; left &= left - 1) {
    const int j = __ffs(left) - 1;
    const V* from = in + __shfl_sync(kFull, mine, j) * a.in_stride;
    const float w = __shfl_sync(kFull, weight, j);
    V v[P];
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (c0 + 32 * i < units) v[i] = load_row<STREAM>(from + 32 * i);
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n) acc[i][n] = fmaf(w, to_f(v[i].v[n]), acc[i][n]);
  }
  V* out = static_cast<V*>(a.out) + t * a.out_stride + c0;
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (c0 + 32 * i < units) {
      V o;
#pragma unroll
      for (int n = 0; n < N; ++n) o.v[n] = from_f<T>(acc[i][n]);
      out[32 * i] = o;
    }
}

// One CTA per token, its warps share the pieces: a piece of the gradient is read once and multiplied with and into
// each of the token's rows.  The products of the pieces are added in a fixed order.  Many rows are held to 64
// registers a thread for their warps' sake (8192 x 8 x 2048 bf16: 106 -> 98.5 us), few are faster without (256 x 8 x
// 4096: 6.0 us, held 6.8).  Many are those that are streamed; where between the two sizes the forms meet was not measured.
template <typename T, int N, bool STREAM>
__global__ void __launch_bounds__(kRowWarps * 32, STREAM ? 4 : 1) combine_backward_kernel(ExchangeRowsArgs a, long long units, unsigned clear_blocks) {
  using V = Vec<T, N>;
  constexpr int P = kPieces<sizeof(V)>;
  __shared__ float part[kRowWarps][kMaxChoices];
  V* out = static_cast<V*>(a.out);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (blockIdx.x < clear_blocks) {      // every piece of the rows
    V zero;
#pragma unroll
    for (int n = 0; n < N; ++n) zero.v[n] = from_f<T>(0.f);
    long long first, step;
    for (unsigned empty = empty_rows(a, clear_blocks, first, step); empty; empty &= empty - 1) {
      V* to = out + (first + (__ffs(empty) - 1) * step) * a.out_stride;
      for (long long c = lane; c < units; c += 32) to[c] = zero;
    }
    return;
  }
  const long long t = blockIdx.x - clear_blocks;
  int mine = -1;
  float weight = 0.f, dots = 0.f;       // lane j: choice j
  if (lane < a.k) {
    mine = a.slot[t * a.k + lane];
    weight = a.weights[t * a.k + lane];
    if (mine >= a.rows) mine = -1;
  }
  const unsigned kept = __ballot_sync(kFull, mine >= 0);
  for (long long c0 = (long long)warp * (32 * P) + lane; c0 - lane < units; c0 += (long long)warps * (32 * P)) {
    const V* from = static_cast<const V*>(a.in) + t * a.in_stride + c0;
    const V* rows = static_cast<const V*>(a.saved) + c0;
    V g[P];
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (c0 + 32 * i < units) g[i] = from[32 * i];
    for (unsigned left = kept; left; left &= left - 1) {
      const int j = __ffs(left) - 1;
      const long long r = __shfl_sync(kFull, mine, j);
      const float w = __shfl_sync(kFull, weight, j);
      V v[P];
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (c0 + 32 * i < units) v[i] = load_row<STREAM>(rows + r * a.saved_stride + 32 * i);
      V* to = out + r * a.out_stride + c0;
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (c0 + 32 * i < units) {
          V o;
#pragma unroll
          for (int n = 0; n < N; ++n) {
            const float x = to_f(g[i].v[n]);
            dot = fmaf(x, to_f(v[i].v[n]), dot);
            o.v[n] = from_f<T>(w * x);
          }
          store_row<STREAM>(to + 32 * i, o);
        }
      dot = warp_sum(dot);
      if (lane == j) dots += dot;
    }
  }
  part[warp][lane] = dots;
  __syncthreads();
  if (threadIdx.x < a.k) {
    float sum = 0.f;
    for (int w = 0; w < warps; ++w) sum += part[w][threadIdx.x];
    a.grad_weights[t * a.k + threadIdx.x] = sum;
  }
}

int elem_size(int dtype) { return dtype == DT_F32 ? 4 : 2; }

}  // namespace

cudaError_t launch_route(const RouteArgs& a, cudaStream_t stream) { return route_any<false>(a, stream); }
cudaError_t launch_route_backward(const RouteArgs& a, cudaStream_t stream) { return route_any<true>(a, stream); }

cudaError_t launch_sort(const SortArgs& a, cudaStream_t stream) {
  // warps first, then CTAs, each with a run of at least kSortRun assignments; a warp scans at most 8 experts where
  // the warps allow it
  const long long workers = (a.assignments + kSortRun - 1) / kSortRun;
  const long long scanners = (a.experts + 7) / 8, both = workers > scanners ? workers : scanners;
  const int warps = both > kSortWarps ? kSortWarps : (int)both;
  int ctas = 1;
  while (ctas < kSortCtas && (long long)ctas * kSortWarps < workers) ctas *= 2;
  const size_t bytes = sizeof(int) * ((size_t)warps * (a.experts | 1) + 4 * (size_t)a.experts);
  auto kernel = a.ids64 ? sort_kernel<long long> : sort_kernel<int>;
  // the attributes are set once per device and index type, for the most experts
  static std::atomic<unsigned long long> allowed[2];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device >= 64 || !(allowed[a.ids64 ? 1 : 0].load() >> device & 1))) {
    const size_t most = sizeof(int) * ((size_t)kSortWarps * (kMaxExperts | 1) + 4 * kMaxExperts);
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && device < 64) allowed[a.ids64 ? 1 : 0].fetch_or(1ull << device);
  }
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(warps * 32);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, a);
}

namespace {

// The widest vector (16, 8 bytes or one element) of every matrix of the call, in bytes.
int vector_bytes(const ExchangeRowsArgs& a) {
  const int es = elem_size(a.dtype);
  const unsigned long long bits = reinterpret_cast<uintptr_t>(a.in) | reinterpret_cast<uintptr_t>(a.out) |
                                  reinterpret_cast<uintptr_t>(a.saved) | (unsigned long long)(a.hidden * es) |
                                  (unsigned long long)(a.in_stride * es) | (unsigned long long)(a.out_stride * es) |
                                  (unsigned long long)(a.saved_stride * es);
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : es;
}

bool streams(const ExchangeRowsArgs& a) { return a.rows * a.hidden * elem_size(a.dtype) > kStreamBytes; }

// strides and lengths in vectors of `per` elements; the number of pieces of a row
long long in_vectors(ExchangeRowsArgs& a, int per, int pieces) {
  a.hidden /= per;
  a.in_stride /= per;
  a.out_stride /= per;
  a.saved_stride /= per;
  return (a.hidden + 32 * pieces - 1) / (32 * pieces);
}

template <typename V>
cudaError_t dispatch_as(ExchangeRowsArgs a, cudaStream_t stream) {
  const bool streamed = streams(a);
  const long long pieces = in_vectors(a, (int)sizeof(V) / elem_size(a.dtype), kPieces<sizeof(V)>);
  const unsigned token_blocks = (unsigned)((a.tokens + kRowWarps - 1) / kRowWarps);
  const unsigned clear_blocks = (unsigned)((a.rows + 32 * kRowWarps - 1) / (32 * kRowWarps));
  if (pieces > 65535) return cudaErrorInvalidConfiguration;
  auto kernel = streamed ? dispatch_kernel<V, true> : dispatch_kernel<V, false>;
  kernel<<<dim3(token_blocks + clear_blocks, (unsigned)pieces), kRowWarps * 32, 0, stream>>>(a, a.hidden, clear_blocks);
  return cudaGetLastError();
}

template <typename T, int N>
cudaError_t combine_as(ExchangeRowsArgs a, cudaStream_t stream) {
  const bool streamed = streams(a);
  const long long pieces = in_vectors(a, N, kPieces<sizeof(T) * N>);
  if (pieces > 65535) return cudaErrorInvalidConfiguration;
  const unsigned blocks = (unsigned)((a.tokens + kRowWarps - 1) / kRowWarps);
  auto kernel = streamed ? combine_kernel<T, N, true> : combine_kernel<T, N, false>;
  kernel<<<dim3(blocks, (unsigned)pieces), kRowWarps * 32, 0, stream>>>(a, a.hidden);
  return cudaGetLastError();
}

template <typename T, int N>
cudaError_t combine_backward_as(ExchangeRowsArgs a, cudaStream_t stream) {
  const bool streamed = streams(a);
  const long long pieces = in_vectors(a, N, kPieces<sizeof(T) * N>);
  const int warps = pieces < 1 ? 1 : pieces > kRowWarps ? kRowWarps : (int)pieces;
  const unsigned clear_blocks = (unsigned)((a.rows + 32 * warps - 1) / (32 * warps));
  if (a.tokens + clear_blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  auto kernel = streamed ? combine_backward_kernel<T, N, true> : combine_backward_kernel<T, N, false>;
  kernel<<<(unsigned)a.tokens + clear_blocks, warps * 32, 0, stream>>>(a, a.hidden, clear_blocks);
  return cudaGetLastError();
}

template <typename T, bool BACKWARD>
cudaError_t combine_any(const ExchangeRowsArgs& a, cudaStream_t stream) {
  constexpr int es = (int)sizeof(T);
  const int bytes = vector_bytes(a);
  if (bytes == 16) return BACKWARD ? combine_backward_as<T, 16 / es>(a, stream) : combine_as<T, 16 / es>(a, stream);
  if (bytes == 8) return BACKWARD ? combine_backward_as<T, 8 / es>(a, stream) : combine_as<T, 8 / es>(a, stream);
  return BACKWARD ? combine_backward_as<T, 1>(a, stream) : combine_as<T, 1>(a, stream);
}

}  // namespace

cudaError_t launch_dispatch(const ExchangeRowsArgs& a, cudaStream_t stream) {
  if (a.hidden == 0 || a.rows == 0) return cudaSuccess;
  const int bytes = vector_bytes(a);
  if (bytes == 16) return dispatch_as<uint4>(a, stream);
  if (bytes == 8) return dispatch_as<uint2>(a, stream);
  return bytes == 4 ? dispatch_as<unsigned>(a, stream) : dispatch_as<unsigned short>(a, stream);
}

cudaError_t launch_combine(const ExchangeRowsArgs& a, cudaStream_t stream) {
  if (a.hidden == 0 || a.tokens == 0) return cudaSuccess;
  if (a.dtype == DT_F32) return combine_any<float, false>(a, stream);
  if (a.dtype == DT_BF16) return combine_any<__nv_bfloat16, false>(a, stream);
  return combine_any<__half, false>(a, stream);
}

cudaError_t launch_combine_backward(const ExchangeRowsArgs& a, cudaStream_t stream) {
  if (a.tokens == 0 && a.rows == 0) return cudaSuccess;
  if (a.dtype == DT_F32) return combine_any<float, true>(a, stream);
  if (a.dtype == DT_BF16) return combine_any<__nv_bfloat16, true>(a, stream);
  return combine_any<__half, true>(a, stream);
}

}  // namespace vb
