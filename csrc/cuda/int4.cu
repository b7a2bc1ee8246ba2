// Matrix-vector products of expert rows with 4-bit weights and group scales:
//   y[r, n] = sum over groups G of scale[e, n, G] * sum over k in G of (q[e, n, k] - 8) * x[r, k]
// for the rows r of expert e's segments.
//
// The weights are read once and are what bounds a few rows, so a weight may cost little more than one
// instruction.  Eight 4-bit values of a word become four registers of two 16-bit numbers each, in nine instructions,
// which are fragments of a 16 x 16 matrix-unit product with up to 8 rows of x as the other side; its sums are fp32.
// One group's sum is scaled in fp32 and added to the total, so a scale is never rounded into a weight.
//
// A CTA of 8 warps covers 128 weight rows, 16 a warp, and two CTAs share an SM.  Every warp streams its rows through
// its own ring of two 4 KB tiles (16 rows of 256 bytes, 512 inner values) that TMA fills, so no warp waits for
// another and the bytes in flight (128 KB of an SM) cost no registers.  A lane holds, of two weight rows and of every
// group, the group / 4 values from (lane % 4) * group / 4 on; x is staged in shared memory in that order, so its
// fragment is one conflict-free 16-byte load.  A cluster of 1 to 8 CTAs splits the inner size where the CTAs would
// not fill the GPU and joins its fp32 sums through distributed shared memory in the order of the CTAs.
//
// Times are of launches in a graph on inputs that are not in the L2, unless they say otherwise.  One row for each of 8
// experts 4096 x 4096 (69 MB): 20.5 us, 3.4 TB/s.  With these inputs in the L2 it takes 18.0, without its arithmetic 15
// and without its loads 14, so what is left is that the two overlap only in part: the arithmetic keeps its integer pipe
// 60 % busy, and 16 warps of an SM are what its registers and ring allow.  Measured as calls and not kept, where this
// form took 20.2 to 20.6: three CTAs of fewer registers (24.5), a barrier per 2 KB box (22.8), and one CTA per SM
// walking equal runs of strips (26.8).  From about 16 rows an expert on the matrix unit bounds it: 1024 rows of 8
// experts 1024 x 2048 take 30.1 us, 143 TFLOP/s.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "vb/launch.h"

namespace vb {
namespace {

constexpr int kThreads = 256;
constexpr int kTileN = 128;           // weight rows of a CTA, 16 per warp
constexpr int kItem = 32;             // rows of x of an item
constexpr int kBoxK = 256;            // inner values of a TMA box: 128 bytes, the span of the swizzle
constexpr int kBoxes = 2;             // boxes of a tile
constexpr int kTileK = kBoxes * kBoxK;
constexpr int kStages = 2;            // tiles in flight of a warp
constexpr unsigned kBoxBytes = 16 * 128;
constexpr int kSms = 148;             // of a B200
constexpr int kPool = 44 * 1024;      // shared memory for a stage of x and scales
constexpr unsigned kTileBytes = kBoxes * kBoxBytes;
constexpr unsigned kFull = 0xffffffffu;
constexpr unsigned kWaitNs = 1000000000u;   // of a tile, and of what is in flight once a tile did not come; a limit from the
                                            // arguments costs a register (ragged fp16 rows in the L2 16.7 -> 17.3 us)

// set when a copy did not arrive in time: the outputs it was for are NaN
__device__ int late_copies = 0;

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// q - 8 of the 4-bit values at bits [0, 4) (HIGH 0) or [4, 8) (HIGH 1) of both halves of w, in two instructions.
// fp16: 1024 + q (or 1024 + 16 q) has q in its mantissa, and one fma takes the 1024 off (the published way to read small
// integers as floats: Kim, Henry, Fahim, Awadalla, Who Says Elephants Can't Run, 2022).  bf16 has too few mantissa bits
// for the upper four, but below 2^-125 its numbers are evenly spaced, so the masked bits are already q 2^-133 or
// 16 q 2^-133; one fma makes them (q - 8) 2^-6, and the total is multiplied by 64 once at the end.  All exact.
template <typename T, int HIGH>
__device__ __forceinline__ unsigned two_values(unsigned w) {
  constexpr unsigned mask = HIGH ? 0x00f000f0u : 0x000f000fu;
  unsigned r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    r = w & mask;
    asm("fma.rn.bf16x2 %0, %0, %1, %2;" : "+r"(r) : "r"(HIGH ? 0x7d007d00u : 0x7f007f00u), "r"(0xbe00be00u));
  } else {
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(0x64006400u));   // (w & mask) | 1024
    if (HIGH) asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(r) : "r"(0x2c002c00u), "r"(0xd480d480u));
    else asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64086408u));
  }
  return r;
}
template <typename T> constexpr float kUnscale = std::is_same<T, __nv_bfloat16>::value ? 64.f : 1.f;

// d = A B + (first ? 0 : d), the fragments i and i + 1
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], const unsigned (&b)[4], int i, unsigned b0,
                                    unsigned b1, bool first) {
  const float c0 = first ? 0.f : d[0], c1 = first ? 0.f : d[1], c2 = first ? 0.f : d[2], c3 = first ? 0.f : d[3];
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[i]), "r"(b[i]), "r"(a[i + 1]), "r"(b[i + 1]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[i]), "r"(b[i]), "r"(a[i + 1]), "r"(b[i + 1]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// VEC words (8 values each) of one lane's part of a group
template <int VEC>
__device__ __forceinline__ void load_words(unsigned (&w)[VEC], const unsigned char* at) {
  if constexpr (VEC == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (VEC == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const unsigned*>(at);
  }
}

__device__ __forceinline__ void barrier_init(unsigned bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
}

// one tile of 16 weight rows x 256 bytes into shared memory; the barrier counts its bytes (what lies past the end
// of a row arrives as zeros and counts too)
__device__ __forceinline__ void load_tile(const CUtensorMap* map, unsigned to, unsigned bar, int x, int y) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(kTileBytes) : "memory");
#pragma unroll
  for (int i = 0; i < kBoxes; ++i)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(to + i * kBoxBytes), "l"(map), "r"(x + i * (kBoxK / 2)), "r"(y), "r"(bar) : "memory");
}

// the lower half of the GPU's nanosecond timer: differences are right up to 4 seconds
__device__ __forceinline__ unsigned globaltimer_lo() {
  unsigned t;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
  return t;
}

// whether the barrier's phase is over, asked for up to about a microsecond (a hint to the hardware, not a bound)
__device__ __forceinline__ bool try_tile(unsigned bar, unsigned phase) {
  unsigned done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(phase), "r"(1000u) : "memory");
  return done;
}

// Waits until the barrier's phase is over; false after a second without it.
__device__ __forceinline__ bool wait_tile(unsigned bar, unsigned phase) {
  if (try_tile(bar, phase)) return true;
  const unsigned t0 = globaltimer_lo();
  do {
    if (try_tile(bar, phase)) return true;
  } while (globaltimer_lo() - t0 < kWaitNs);
  return false;
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

// scales of PAIR groups of one weight row
template <int PAIR>
__device__ __forceinline__ void load_scales(float (&f)[PAIR], const float* s) {
#pragma unroll
  for (int p = 0; p < PAIR; ++p) f[p] = s[p];
}
template <int PAIR, typename S>
__device__ __forceinline__ void load_scales(float (&f)[PAIR], const S* s) {
  if constexpr (PAIR == 2) {                // at an even place: one word
    const unsigned w = *reinterpret_cast<const unsigned*>(s);
    const unsigned short lo = (unsigned short)w, hi = (unsigned short)(w >> 16);
    f[0] = to_f(*reinterpret_cast<const S*>(&lo));
    f[1] = to_f(*reinterpret_cast<const S*>(&hi));
  } else {
    f[0] = to_f(s[0]);
  }
}

// PAIR groups of 16 weight rows times COLS x 8 rows of x, scaled and added to acc; the groups' products alternate, so
// that a product seldom waits for the one before it.  `x` is the lane's first unit, the next word's is `step` units
// further (32 * COLS, or with one column 4 times its rows rounded to a power of two); `scale` points to the lane's
// first weight row, the second is `second` further.  A lane whose row of x does not exist computes with what lies
// there: columns of a product do not mix, and that column is not written.
template <typename T, typename S, int VEC, int COLS, int PAIR>
__device__ __forceinline__ void group_product(float (&acc)[COLS][4], const unsigned char* tile, unsigned at, int u0,
                                              const uint4* x, int step, const S* scale, int second) {
  unsigned ra[PAIR][VEC], rb[PAIR][VEC];
  float part[PAIR][COLS][4];
#pragma unroll
  for (int p = 0; p < PAIR; ++p) {
    // within a box the groups differ in the chunk bits, which the swizzle leaves to an exclusive or
    const int u = u0 + p, in_box = kBoxK / (32 * VEC);
    const unsigned char* from = tile + (at ^ (16 * VEC * (u % in_box))) + u / in_box * kBoxBytes;
    load_words<VEC>(ra[p], from);
    load_words<VEC>(rb[p], from + 1024);
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v)
#pragma unroll
    for (int p = 0; p < PAIR; ++p) {
      const unsigned wa = ra[p][v], wb = rb[p][v];
      const unsigned va[4] = {two_values<T, 0>(wa), two_values<T, 1>(wa), two_values<T, 0>(wa >> 8), two_values<T, 1>(wa >> 8)};
      const unsigned vb[4] = {two_values<T, 0>(wb), two_values<T, 1>(wb), two_values<T, 0>(wb >> 8), two_values<T, 1>(wb >> 8)};
#pragma unroll
      for (int t = 0; t < COLS; ++t) {
        const uint4 b = x[(p * VEC + v) * (COLS == 1 ? step : 32 * COLS) + t * 32];
        mma<T>(part[p][t], va, vb, 0, b.x, b.y, v == 0);
        mma<T>(part[p][t], va, vb, 2, b.z, b.w, false);
      }
    }
  float first[PAIR], other[PAIR];
  load_scales<PAIR>(first, scale);
  load_scales<PAIR>(other, scale + second);
#pragma unroll
  for (int p = 0; p < PAIR; ++p) {
    const float sa = first[p], sb = other[p];
#pragma unroll
    for (int t = 0; t < COLS; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(i < 2 ? sa : sb, part[p][t][i], acc[t][i]);
  }
}

// items of more than 8 rows of a segment; its length rounded up may pass 31 bits
__device__ __forceinline__ int longer_items(int rows) { return (int)(((unsigned)rows + kItem - 9) / kItem); }

struct Geometry {
  long long slice;     // inner values of one CTA of the cluster, whole tiles
  int aligned;         // rows of x can be read 16 bytes at a time
  unsigned n_tiles, items;
};

// rows of a unit of x with one column: a power of two
__device__ __forceinline__ int staged_rows(int rows) { return rows > 4 ? 8 : rows > 2 ? 4 : rows; }

struct Item {
  int expert, row0, rows;    // rows of x: row0 ... row0 + rows - 1, at most 32
  long long n0;              // the CTA's first weight row
  int k_lo, k_hi;            // its inner values
};

// One CTA's part of an item of at most 8 * COLS rows of x: its sums over its inner values, [row of x][weight row],
// left in shared memory.
template <typename T, typename S, int VEC, int COLS>
__device__ __forceinline__ void item_sums(const CUtensorMap* map, const Int4Args& a, const Geometry& geo, const Item& it,
                                          unsigned char* smem, unsigned bars) {
  constexpr int GROUP = 32 * VEC, UNITS = kTileK / GROUP;               // groups of a tile
  constexpr int PAIR = COLS <= 2 ? 2 : 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
  const int groups = (int)(a.inner / GROUP), units = (it.k_hi - it.k_lo) / GROUP, tiles = (units + UNITS - 1) / UNITS;
  const long long base = (long long)it.expert * a.n;
  // the warp's ring; a warp whose rows are all past the last has nothing to do
  const unsigned char* ring = smem + warp * (kStages * kTileBytes);
  const unsigned to = (unsigned)__cvta_generic_to_shared(ring), bar = bars + warp * (kStages * 8);
  const bool busy = it.n0 + warp * 16 < a.n;
  const int y = (int)(base + it.n0) + warp * 16;
  if (busy && lane == 0)
    for (int i = 0; i < kStages && i < tiles; ++i)
      load_tile(map, to + i * kTileBytes, bar + 8 * i, it.k_lo / 2 + i * (kTileK / 2), y);
  // rows are dealt to the lanes so that the lanes of one shared-memory phase meet different banks of the
  // 128-byte swizzle (16-byte chunk c of row r is at c ^ (r % 8))
  const int row = VEC == 4 ? (g & 1) * 4 + (g >> 1) : VEC == 2 ? (g & 3) * 2 + (g >> 2) : g;
  const unsigned lane_at = row * 128 + (((tq * VEC / 4) ^ row) << 4) + (tq * VEC % 4) * 4;
  const T* x = static_cast<const T*>(a.x) + it.row0 * a.x_stride + it.k_lo;
  const S* scales = static_cast<const S*>(a.scales) + it.k_lo / GROUP;
  unsigned char* staged = smem + (kThreads / 32) * kStages * kTileBytes;
  // a stage takes as many tiles as the pool holds, equal numbers in all stages; fewer rows of x leave room for more
  const int unit = COLS == 1 ? staged_rows(it.rows) : 8 * COLS, step = 4 * unit;
  const int fits = kPool / (kTileK * 2 * unit + kTileN * (UNITS * (int)sizeof(S) + 8)), stages = (tiles + fits - 1) / fits;
  const int chunk = (tiles + stages - 1) / max(stages, 1) * UNITS;      // groups
  const int pitch = sizeof(S) == 4 ? chunk | 1 : 2 * ((chunk + 1) / 2 | 1);   // an odd number of words: no bank conflicts
  uint4* xs = reinterpret_cast<uint4*>(staged);                         // [groups * VEC][unit][4]
  S* sc = reinterpret_cast<S*>(staged + chunk * GROUP * 2 * unit);      // [kTileN][pitch]
  float acc[COLS][4];
#pragma unroll
  for (int t = 0; t < COLS; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
  int slot = 0;
  unsigned phase = 0;
  int late = busy && a.give_up ? 0 : -1;    // the tile that did not come

  for (int c0 = 0; c0 < units; c0 += chunk) {
    const int here = min(chunk, units - c0), eighths = here * (GROUP / 8);
    if (c0) __syncthreads();                // the stage before has been read
    // a warp stages the scales of its own rows, along the groups (of two rows at once where those are few), and its
    // share of x: 16-byte units of 8 inner values in the order 0 4 1 5 2 6 3 7, four loads in flight
    {
      const bool narrow = here <= 16;
      const int su = narrow ? lane & 15 : lane, sr = narrow ? lane >> 4 : 0, rows_at_once = narrow ? 2 : 1;
      S sv[8];
      auto ask = [&](int r0, int u) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (u < here)
            sv[i] = scales[(base + min(it.n0 + warp * 16 + r0 + i * rows_at_once + sr, a.n - 1)) * groups + c0 + u];
      };
      ask(0, su);                           // on its way while x is staged
      // a row's units go to 8 / unit warps (one where there are 8 rows or more)
      const int at_once = COLS == 1 ? unit : 8, parts = 8 / at_once;
      const int k8_first = (warp / at_once) * 32 + lane, k8_step = 32 * parts;
      const T* p = x + (long long)c0 * GROUP;
      int token = warp % at_once, k8 = k8_first;
      while (token < it.rows) {
        uint4 v[4];
        int at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          at[i] = -1;
          if (token < it.rows && k8 < eighths) {
            const T* from = p + token * a.x_stride + 8 * k8;
            if (geo.aligned) {
              v[i] = *reinterpret_cast<const uint4*>(from);
            } else {
              __align__(16) T e[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) e[j] = from[j];
              v[i] = *reinterpret_cast<uint4*>(e);
            }
            const int grp = k8 / (4 * VEC), in = k8 % (4 * VEC);        // in = (lane % 4) * VEC + word
            at[i] = ((grp * VEC + in % VEC) * unit + token) * 4 + in / VEC;
          }
          k8 += k8_step;
          if (k8 - lane >= eighths) { k8 = k8_first; token += at_once; }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (at[i] >= 0)
            xs[at[i]] = make_uint4(__byte_perm(v[i].x, v[i].z, 0x5410), __byte_perm(v[i].x, v[i].z, 0x7632),
                                   __byte_perm(v[i].y, v[i].w, 0x5410), __byte_perm(v[i].y, v[i].w, 0x7632));
      }
      for (int r0 = 0, u = su;;) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (u < here) sc[(warp * 16 + r0 + i * rows_at_once + sr) * pitch + u] = sv[i];
        u += 32;
        if (u - su >= here) { u = su; r0 += 8 * rows_at_once; }
        if (r0 == 16) break;
        ask(r0, u);
      }
    }
    __syncthreads();
    const uint4* xw = xs + g * 4 + tq;
    const S* sw = sc + (warp * 16 + row) * pitch;
    if (busy)
      for (int u0 = 0; u0 < here; u0 += UNITS) {
        if (late < 0 && !__all_sync(kFull, wait_tile(bar + 8 * slot, phase))) late = (c0 + u0) / UNITS;
        const unsigned char* tile = ring + slot * kTileBytes;
        if (u0 + UNITS <= here) {
          // unrolled with one column only: with more the registers spill (1024 rows of 8 experts 34.9 us, so 30.1)
#pragma unroll (COLS == 1 ? UNITS : 1)
          for (int u = 0; u < UNITS; u += PAIR)
            group_product<T, S, VEC, COLS, PAIR>(acc, tile, lane_at, u, xw + u * VEC * step, step, sw + u, 8 * pitch);
        } else {
          for (int u = 0; u0 + u < here; ++u)
            group_product<T, S, VEC, COLS, 1>(acc, tile, lane_at, u, xw + u * VEC * step, step, sw + u, 8 * pitch);
        }
        xw += UNITS * VEC * step;
        sw += UNITS;
        __syncwarp();                       // the tile has been read by every lane
        const int coming = (c0 + u0) / UNITS + kStages;
        if (lane == 0 && coming < tiles && late < 0)
          load_tile(map, to + slot * kTileBytes, bar + 8 * slot, it.k_lo / 2 + coming * (kTileK / 2), y);
        if (++slot == kStages) { slot = 0; phase ^= 1; }
      }
  }
  float unscale = kUnscale<T>;
  if (late >= 0) {                          // NaN; what is in flight lands before its memory is given back
    if (lane == 0) atomicExch(&late_copies, 1);
    for (int i = late; i < tiles && i < late + kStages; ++i) wait_tile(bar + 8 * (i % kStages), i / kStages & 1);
    unscale = __int_as_float(0x7fffffff);
  }
  __syncthreads();
  float* sums = reinterpret_cast<float*>(staged);
#pragma unroll
  for (int t = 0; t < COLS; ++t) {
    float* at = sums + (8 * t + 2 * tq) * kTileN + warp * 16 + row;
    at[0] = acc[t][0] * unscale;
    at[kTileN] = acc[t][1] * unscale;
    at[8] = acc[t][2] * unscale;
    at[kTileN + 8] = acc[t][3] * unscale;
  }
}

// MOST: the most columns of 8 rows of x an item of this call can have.
template <typename T, typename S, int VEC, int MOST>
__global__ void __launch_bounds__(kThreads, 2) int4_product_kernel(const __grid_constant__ CUtensorMap map, Int4Args a,
                                                                Geometry geo) {
  extern __shared__ unsigned char dynamic[];
  // the swizzle's pattern repeats every 1024 bytes of the address
  unsigned char* smem = dynamic + (-(unsigned)__cvta_generic_to_shared(dynamic) & 1023u);
  __shared__ __align__(8) unsigned long long bars[kThreads / 32][kStages];
  __shared__ int pick[3];                   // segment, first row, rows of this CTA's item
  __shared__ int3 scan[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned rank = cluster_rank(), ranks = cluster_size();
  const int item = (int)(blockIdx.x / ranks / geo.n_tiles);
  const long long n0 = (long long)(blockIdx.x / ranks % geo.n_tiles) * kTileN;

  // which segment and rows: the items are the segments' tiles of kItem rows, those of more than 8 rows first, so that
  // the longer ones do not start last
  int covered = 0;                          // rows that some segment covers
  {
    constexpr int PER = 1024 / kThreads;    // at most 1024 segments, PER consecutive ones a thread
    int first[PER], count[PER], rows = 0;
    int2 mine = make_int2(0, 0);            // longer and shorter items
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = tid * PER + i;
      first[i] = s < a.segments ? a.starts[s] : 0;
      count[i] = s < a.segments ? a.counts[s] : 0;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {         // kept inside the matrix
      const long long lo = first[i], hi = min(lo + count[i], a.rows);
      first[i] = max(first[i], 0);
      count[i] = (int)max(hi - first[i], 0ll);
      mine.x += longer_items(count[i]);
      mine.y += (unsigned)(count[i] - 1) % kItem < 8 && count[i];
      rows += count[i];
    }
    int2 x = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(kFull, x.x, off), z = __shfl_up_sync(kFull, x.y, off);
      if (lane >= off) x.x += y, x.y += z;
    }
    rows = __reduce_add_sync(kFull, rows);
    if (lane == 31) scan[warp] = make_int3(x.x, x.y, rows);
    if (tid == 0) pick[0] = -1;
    if (tid < kThreads / 32 * kStages) barrier_init((unsigned)__cvta_generic_to_shared(&bars[0][0] + tid));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    int before = x.x - mine.x, before_short = x.y - mine.y;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const int3 got = scan[w];
      before_short += got.x + (w < warp ? got.y : 0);                   // all the longer ones come first
      if (w < warp) before += got.x;
      covered += got.z;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int longer = longer_items(count[i]), shorter = (unsigned)(count[i] - 1) % kItem < 8 && count[i];
      int at = -1;
      if (item >= before && item < before + longer) at = (item - before) * kItem;
      if (shorter && item == before_short) at = longer * kItem;
      if (at >= 0) {
        pick[0] = tid * PER + i;
        pick[1] = first[i] + at;
        pick[2] = min(count[i] - at, kItem);
      }
      before += longer;
      before_short += shorter;
    }
    __syncthreads();
  }

  if (pick[0] >= 0) {                       // the same for every CTA of the cluster
    Item it;
    it.expert = pick[0] % a.experts;
    it.row0 = pick[1];
    it.rows = pick[2];
    it.n0 = n0;
    it.k_lo = (int)min(a.inner, rank * geo.slice);
    it.k_hi = (int)min(a.inner, it.k_lo + geo.slice);
    const unsigned bar = (unsigned)__cvta_generic_to_shared(&bars[0][0]);
    const int columns = MOST == 1 ? 1 : (it.rows + 7) / 8;
    if (columns == 1) item_sums<T, S, VEC, 1>(&map, a, geo, it, smem, bar);
    else if constexpr (MOST > 1) {
      if (columns == 2) item_sums<T, S, VEC, 2>(&map, a, geo, it, smem, bar);
      else if (columns == 3) item_sums<T, S, VEC, 3>(&map, a, geo, it, smem, bar);
      else item_sums<T, S, VEC, 4>(&map, a, geo, it, smem, bar);
    }
    // join the cluster's sums: CTA `rank` finishes every ranks-th part of the outputs
    float* sums = reinterpret_cast<float*>(smem + (kThreads / 32) * kStages * kTileBytes);
    if (ranks > 1) cluster_sync(); else __syncthreads();
    const unsigned sums_at = (unsigned)__cvta_generic_to_shared(sums);
    T* out = static_cast<T*>(a.out);
    for (int i = rank * kThreads + tid; i < it.rows * kTileN; i += ranks * kThreads) {
      const int token = i / kTileN, n = i % kTileN;
      float v = 0.f;
      for (unsigned r = 0; r < ranks; ++r) v += remote_f(sums_at + 4u * i, r);
      if (n0 + n < a.n) out[(it.row0 + token) * a.out_stride + n0 + n] = from_f<T>(v);
    }
    if (ranks > 1) cluster_sync();          // the sums stay until every CTA has read them
  }

  // rows that no segment covers are zero; row r belongs to item r mod the items
  if (rank == 0 && covered < a.rows)
    for (long long r = item + (long long)warp * geo.items; r < a.rows; r += 8ll * geo.items) {
      bool inside = false;
      for (int s = lane; s < a.segments; s += 32) {
        const long long lo = a.starts[s];
        inside |= r >= lo && r < lo + a.counts[s];
      }
      if (!__any_sync(kFull, inside))
        for (int c = lane; c < kTileN && n0 + c < a.n; c += 32) static_cast<T*>(a.out)[r * a.out_stride + n0 + c] = from_f<T>(0.f);
    }
}

template <typename T, typename S, int VEC, int MOST>
cudaError_t launch(const Int4Args& a, cudaStream_t stream) {
  // items: every segment's last may be partial
  const long long items = (a.rows + kItem - 1) / kItem + (a.segments < a.rows ? a.segments : a.rows) - 1;
  const long long n_tiles = (a.n + kTileN - 1) / kTileN;
  // split the inner size until the GPU is full, as long as a CTA keeps a tile
  int ranks = 1;
  while (ranks < 8 && n_tiles * items * ranks * 2 <= kSms * 2 && a.inner / (2 * ranks) >= kTileK) ranks *= 2;
  Geometry geo{};
  const long long tiles = (a.inner + kTileK - 1) / kTileK;
  geo.slice = (tiles + ranks - 1) / ranks * kTileK;
  geo.n_tiles = (unsigned)n_tiles;
  geo.items = (unsigned)items;
  geo.aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride % 8 == 0;
  size_t bytes = kPool;
  bytes += kThreads / 32 * kStages * kTileBytes + 1024;
  CUtensorMap map;
  const cuuint64_t size[2] = {(cuuint64_t)(a.inner / 2), (cuuint64_t)a.experts * a.n}, pitch[1] = {(cuuint64_t)(a.inner / 2)};
  const cuuint32_t box[2] = {128, 16}, step[2] = {1, 1};
  if (cuTensorMapEncodeTiled(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<unsigned char*>(a.packed), size, pitch, box,
                             step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  auto kernel = int4_product_kernel<T, S, VEC, MOST>;
  // the shared-memory limit is raised once per device and instance
  static std::atomic<unsigned long long> allowed{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device >= 64 || !(allowed.load() >> device & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && device < 64) allowed.fetch_or(1ull << device);
  }
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
  return cudaLaunchKernelEx(&config, kernel, map, a, geo);
}

// Up to 8 rows have one column: an instance without the others' registers (one token of 8 experts 20.5 us, not 21.3).
// The host knows only the rows of the call, so more rows take the other instance however few each expert has.
template <typename T, typename S, int VEC>
cudaError_t launch_columns(const Int4Args& a, cudaStream_t stream) {
  return a.rows <= 8 ? launch<T, S, VEC, 1>(a, stream) : launch<T, S, VEC, 4>(a, stream);
}

template <typename T, typename S>
cudaError_t launch_group(const Int4Args& a, cudaStream_t stream) {
  if (a.group == 128) return launch_columns<T, S, 4>(a, stream);
  if (a.group == 64) return launch_columns<T, S, 2>(a, stream);
  return launch_columns<T, S, 1>(a, stream);
}

}  // namespace

// The device is waited for: a copy on the legacy default stream alone does not wait for non-blocking streams.
cudaError_t int4_late_copies(int* flag) {
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(flag, late_copies, sizeof(int));
  const int none = 0;
  if (e == cudaSuccess && *flag) e = cudaMemcpyToSymbol(late_copies, &none, sizeof(int));
  return e;
}

cudaError_t launch_int4_product(const Int4Args& a, cudaStream_t stream) {
  if (a.rows == 0 || a.n == 0) return cudaSuccess;
  if (a.dtype == DT_BF16)
    return a.scales_fp32 ? launch_group<__nv_bfloat16, float>(a, stream) : launch_group<__nv_bfloat16, __nv_bfloat16>(a, stream);
  return a.scales_fp32 ? launch_group<__half, float>(a, stream) : launch_group<__half, __half>(a, stream);
}

}  // namespace vb
