// The next token of every row from its logits and a given uniform number:
// gptoss_decode_sample in include/gptoss_decode_b200.h.
//
// The kept set is a prefix of the order (logit descending, id ascending), so it is one
// threshold: all logits above a value and the first few ids among those equal to it.  Nothing
// is sorted.  Weights are integers (multiples of 2^-44), so every sum is exact whatever its
// order, and a draw is the same for any split of the row.
//
// A cluster of up to 8 CTAs holds a row in its shared memory: the logits are read from HBM
// once, and what follows runs on chip:
//   1. load, maximum (joined over the cluster)
//   2. a top-k of up to kList / 2: the top_k-th largest of the threads' maxima bounds it from
//      below; the logits from there on go to a list that every CTA sorts for itself, and top-p
//      is then found in that list too.  Otherwise: counts (top-k) or counts and weights (top-p)
//      of kBins bins of equal width below the maximum, summed over the cluster, and the bin in
//      which the limit falls; its logits go to the list.  A bin with more than kList of them is
//      cut into kBins parts first, and where a part still has more (equal logits, or what lies
//      beyond the last bin) it is searched by the digits of their bits
//   3. running sums in the order of the ids: threads own consecutive ids, block and cluster
//      prefix; the warp of the thread in whose run the drawn value falls walks that run again
// What bounds it: for large batches the chain of a CTA's steps - load 4 us, maximum 2, weights 5
// (some fifty instructions a logit, 11 of them fp64), sums 2, pick 1 - of which two CTAs per SM
// overlap (512 rows of 201088 by temperature 251 us, 1.6 TB/s, issue 55 %); with top-p without
// top-k the weights once more and the shared atomics of the bins, 13 us (96 rows of 50257: 59
// us); for a few rows the cluster barriers between the steps, 1.3 us each (one row of 201088
// with all limits 16 us in a graph, 64 rows of mixed settings 89).  64 rows of 201088 by top-k
// alone: 46 us for the first 50, 63 for 512, the most that the sorted list takes, 64 for 513, 96
// for 20000.
//
// A weight is within half a unit of 2^-44 of the likeliest token's (what is lighter has fewer
// bits); fp32's 2^-24 would not do: with 200000 kept tokens a draw lies within 2^-24 of some
// running sum every few rows, and would then pick the wrong one.
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "decode_ops.h"
#include "engine.h"
#include "umma_2sm.cuh"

namespace gptoss {

typedef unsigned long long u64;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleMaxSplit = 8;     // CTAs of a row
constexpr int kSampleMaxVocab = 1 << 18;
constexpr int kSamplePart = 25600;     // logits of a CTA that leave room for two CTAs on an SM
constexpr int kBins = 512;
constexpr int kList = 1024;
constexpr unsigned kAll = 0xffffffffu;        // no limit among equal logits; no id
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // sample_key(-infinity)
constexpr u64 kOne = 1ull << 44;              // weight of the likeliest token

// Order-preserving bits of a logit (never NaN or -0 here).
__device__ __forceinline__ uint32_t sample_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// NaN counts as -infinity, -0 as +0
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY) + 0.0f; }
__device__ __forceinline__ float logit_at(const float *p) { return *p; }
__device__ __forceinline__ float logit_at(const bf16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float logit_at(const __half *p) { return __half2float(*p); }

struct SampleShared {
  double table[16];                // 2^(44 - j / 16)
  union {
    u64 mass[kBins];               // cluster reads: weight of a bin in this CTA's part of the row
    uint32_t merged[kList];        // the cluster's lists together, largest first
  };
  unsigned count[kBins];           // cluster reads: logits of a bin
  uint32_t list[kList];            // cluster reads: keys that the CTA contributes to a list
  u64 warp_sum[2][kSampleWarps];
  float warp_max[kSampleWarps];
  uint32_t best;                   // cluster reads: key of the CTA's largest logit
  unsigned first;                  // cluster reads: lowest id of the largest logit
  u64 sum;                         // cluster reads: the CTA's weight
  unsigned listed[3];              // cluster reads: lengths of the CTA's lists
  unsigned equal;                  // cluster reads: logits equal to the edge in the CTA
  // results of a search, the same in all CTAs
  uint32_t edge;
  unsigned need, take, equals, size, before;
  u64 above;
  int bin;
};

__device__ __forceinline__ uint32_t peer_addr(const void *p, int cta) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(cta));
  return remote;
}
__device__ __forceinline__ u64 peer_u64(const u64 *p, int cta) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_addr(p, cta)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned peer_u32(const unsigned *p, int cta) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_addr(p, cta)) : "memory");
  return v;
}

// Weights: 2^(44 - y), y = (max - x) / (T ln 2), rounded to an integer.  16 y = k + r with an
// integer k: 2^(44 - k/16) from a table and an exponent, 2^(-r/16) by its Taylor polynomial of
// degree 6 (|r| <= 1/2: below 1e-15 relative).  All in fp64; the two additions of a power of
// two round to integers and leave them in the low bits, which spares the slow conversions.
// (Per SM and cycle: 64 fp64 operations, 16 conversions of fp32 to fp64, and 15.6 lookups in a
// table of 16 doubles, which lie in different banks; of 128 only 6.9.)
struct Weigher {
  double max, scale;      // scale = 16 / (T ln 2)
  float floor;            // 46 T ln 2 below the maximum: weighs 0, and so does what lies below
  const double *table;
  // N weights plus kBias each (the bits of 2^52, which the rounding leaves in place).  N at a
  // time: a weight is a chain of a dozen dependent fp64 operations of about 50 cycles each.
  static constexpr u64 kBias = 0x4330000000000000ull;
  template <int N>
  __device__ __forceinline__ void biased(const float (&x)[N], u64 (&w)[N]) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
    constexpr double c1 = -0.69314718055994530942 / 16, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4,
                     c5 = c4 * c1 / 5, c6 = c5 * c1 / 6;
    double p[N], r[N];
    int k[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      const double d = max - static_cast<double>(fmaxf(x[i], floor));
      const double shifted = fma(d, scale, kRound);
      k[i] = __double2loint(shifted);
      r[i] = fma(d, scale, kRound - shifted);
    }
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = fma(r[i], c6, c5);
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = fma(p[i], r[i], c4);
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = fma(p[i], r[i], c3);
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = fma(p[i], r[i], c2);
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = fma(p[i], r[i], c1);
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = fma(p[i], r[i], 1.0);
#pragma unroll
    for (int i = 0; i < N; i++) {
      // times 2^(44 - k / 16) (the whole part, at most 47, by the exponent), rounded to an integer
      const double at = table[k[i] & 15];
      const double power = __hiloint2double(__double2hiint(at) - ((k[i] & ~15) << 16), __double2loint(at));
      w[i] = static_cast<u64>(__double_as_longlong(fma(p[i], power, 4503599627370496.0)));  // 2^52
    }
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    const float in[1] = {x};
    u64 w[1];
    biased(in, w);
    return w[0] - kBias;
  }
};

// Sum over the block of v; every thread gets the exclusive prefix in *before.  Two scans in a row
// use different scratch, so that one barrier each is enough.
__device__ u64 block_scan(u64 v, u64 *before, u64 *scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 inc = v;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, inc, i);
    if (lane >= i) inc += o;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  const u64 mine = scratch[lane & (kSampleWarps - 1)];
  u64 sums = mine;
#pragma unroll
  for (int i = 1; i < kSampleWarps; i <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, sums, i);
    if (lane >= i) sums += o;
  }
  *before = __shfl_sync(0xffffffffu, sums - mine, warp) + inc - v;
  return __shfl_sync(0xffffffffu, sums, kSampleWarps - 1);
}

// split: CTAs of a row
template <typename T, int split>
__global__ void __launch_bounds__(kSampleThreads)
sample_kernel(const gptoss_sample_args_t a, int per) {
  extern __shared__ __align__(16) float slice_mem[];
  __shared__ SampleShared s;
  const int tid = threadIdx.x, lane = tid & 31;
  const int rank = split > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int row = blockIdx.x / split;
  int turn = 0;
  auto scan = [&](u64 v, u64 *before) { return block_scan(v, before, s.warp_sum[turn ^= 1]); };
  auto sync = [&]() {
    if (split > 1)
      cluster_barrier_all();
    else
      __syncthreads();
  };
  if (a.pos && a.pos[row] < 0) {  // the whole cluster alike
    if (rank == 0 && tid == 0) a.next[row] = -1;
    return;
  }
  const int id0 = min(a.vocab, rank * per), n = min(a.vocab, id0 + per) - id0;
  const T *x = static_cast<const T *>(a.logits) + row * a.stride + id0;
  // the row's settings, on their way while the logits are
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  const int top_k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f;
  const float min_p = a.min_p ? a.min_p[row] : 0.0f;
  const float u0 = a.u[row];
  // ------------------------------------------------------------------ 1. load, maximum
  // 16-byte loads from the first 16-byte boundary on; the slice starts so far into its buffer
  // that those end up on 16-byte boundaries there too
  constexpr int kVec = 16 / sizeof(T);
  const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T)));
  float *slice = slice_mem + ((kVec - head) & 3);
  float best = -INFINITY;  // of the logits that this thread loads
  if (tid < head) best = slice[tid] = clean(logit_at(x + tid));
  const int vecs = (n - head) / kVec;
  const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
#pragma unroll 4
  for (int v = tid; v < vecs; v += kSampleThreads) {
    const uint4 raw = __ldcs(xv + v);
    const T *e = reinterpret_cast<const T *>(&raw);
    float f[kVec];
#pragma unroll
    for (int j = 0; j < kVec; j++) f[j] = clean(logit_at(e + j));
    const int i = head + v * kVec;
#pragma unroll
    for (int j = 0; j < kVec; j += 4)
      *reinterpret_cast<float4 *>(slice + i + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
#pragma unroll
    for (int j = 0; j < kVec; j++) best = fmaxf(best, f[j]);
  }
  for (int i = head + vecs * kVec + tid; i < n; i += kSampleThreads) {
    slice[i] = clean(logit_at(x + i));
    best = fmaxf(best, slice[i]);
  }
  {
    float all = best;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, i));
    if (lane == 0) s.warp_max[tid >> 5] = all;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kSampleWarps; w++) all = fmaxf(all, s.warp_max[w]);
      s.best = sample_key(all);
      s.first = kAll;
    }
  }
  if (tid < 16) s.table[tid] = exp2(44 - tid / 16.0);
  if (tid < 3) s.listed[tid] = 0;
  for (int i = tid; i < kBins; i += kSampleThreads) s.mass[i] = s.count[i] = 0;
  const double t = fmin(static_cast<double>(temp), 1e36);
  const double reach = 46 * 0.69314718055994530942 * t;
  const double scale = 16 * 1.44269504088896340736 / t;
  sync();
  uint32_t key = 0;
#pragma unroll
  for (int c = 0; c < split; c++) key = max(key, split > 1 ? peer_u32(&s.best, c) : s.best);
  if (!(temp > 0.0f) || key == kKeyNegInf) {
    // greedy: the lowest id of the largest logit (-infinity everywhere: the first id)
    const float want = key_value(key);
    unsigned mine = kAll;
    for (int i = tid; i < n && mine == kAll; i += kSampleThreads)
      if (slice[i] == want) mine = id0 + i;
    mine = __reduce_min_sync(0xffffffffu, mine);
    if (lane == 0 && mine != kAll) atomicMin(&s.first, mine);
    sync();
    if (rank == 0 && tid == 0) {
      unsigned id = kAll;
#pragma unroll
      for (int c = 0; c < split; c++) id = min(id, split > 1 ? peer_u32(&s.first, c) : s.first);
      a.next[row] = static_cast<int>(id);
    }
    if (split > 1) cluster_barrier_all();  // nobody leaves while its shared memory is read
    return;
  }
  float top = key_value(key);
  // Weights need a finite maximum, room below it, and fp32 steps there that are small against
  // the temperature.  +infinity: those logits become 0, the others -infinity.  A maximum near
  // the lowest value (a row of masks), or far larger than the temperature: logits relative to it.
  auto floor_of = [&](float from) { return nextafterf(static_cast<float>(from - reach), -INFINITY); };
  if (top == INFINITY || top - reach < -3.4e38 ||
      (static_cast<double>(top) - floor_of(top)) * scale > 46.9 * 16) {
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
      const float v = slice[i];
      slice[i] = top == INFINITY ? (v == INFINITY ? 0.0f : -INFINITY) : v - top;
    }
    best = best == -INFINITY ? best : (top == INFINITY ? (best == INFINITY ? 0.0f : -INFINITY) : best - top);
    top = 0.0f;
    __syncthreads();
  }
  Weigher weigher;
  weigher.max = static_cast<double>(top);
  weigher.scale = scale;
  weigher.floor = floor_of(top);
  weigher.table = s.table;
  const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.0f;
  // kept: keys above `edge`, and the first `need` ids of those equal to it
  uint32_t edge = 0;
  unsigned need = kAll;

  if (by_count || by_mass) {
    // ---------------------------------------------------------------- 2. thresholds
    // bins of T / 16 below the maximum (of 1 / 16 above temperature 1, where the logits' own
    // spread is what matters), the last one open; float arithmetic is monotonic, so bins
    // respect the order.  -infinity takes no part.
    const float to_bin = 16.0f * fmaxf(1.0f, static_cast<float>(1.0 / t));
    auto place = [&](float v) {  // in bins
      return v == top ? 0.0f : fminf((top - v) * to_bin, static_cast<float>(kBins - 1));
    };
    auto bin_of = [&](float v) { return static_cast<int>(place(v)); };
    // 64-bit sums in shared memory as two 32-bit ones with a carry (6.3 a cycle and SM; the
    // 64-bit atomic manages 1.1)
    auto add_mass = [&](int b, u64 w) {
      if (w == 0) return;
      unsigned *word = reinterpret_cast<unsigned *>(&s.mass[b]);
      const unsigned lo = static_cast<unsigned>(w);
      const unsigned carry = atomicAdd(word, lo) + lo < lo;
      const unsigned hi = static_cast<unsigned>(w >> 32) + carry;
      if (hi) atomicAdd(word + 1, hi);
    };
    // the row's count and weight of digit or bin b
    auto gather = [&](int b, bool weights, unsigned *c, u64 *w) {
      unsigned cs[split];
      u64 ws[split];
#pragma unroll
      for (int k = 0; k < split; k++) {
        cs[k] = split > 1 ? peer_u32(&s.count[b], k) : s.count[b];
        ws[k] = 0;
        if (weights) ws[k] = split > 1 ? peer_u64(&s.mass[b], k) : s.mass[b];
      }
      *c = 0;
      *w = 0;
#pragma unroll
      for (int k = 0; k < split; k++) {
        *c += cs[k];
        *w += ws[k];
      }
    };
    static_assert(kBins == kSampleThreads, "a thread per bin in the scans");
    unsigned my_count;
    u64 my_mass, count_before, mass_before, all_count, all_mass;
    // Logits outside [low, high] are in none of the bins lo .. hi (bounds one bin wider).
    auto bounds = [&](int lo, int hi, float floor_value, float *low, float *high) {
      *low = fmaxf(floor_value, hi < kBins - 1 ? top - static_cast<float>(hi + 2) / to_bin * 1.0001f : -FLT_MAX);
      *high = lo > 0 ? top - static_cast<float>(lo - 1) / to_bin * 0.9999f : INFINITY;
      *low = fmaxf(*low, -FLT_MAX);
    };
    // Counts (and weights) of the bins, of the logits from `least` on; with bin >= 0 of that
    // bin's logits alone, in kBins parts of it.
    auto histogram = [&](bool weights, float least, int bin) {
      float low = fmaxf(least, -FLT_MAX), high = INFINITY;
      if (bin >= 0) bounds(bin, bin, least, &low, &high);
      for (int i0 = tid; i0 < n; i0 += 4 * kSampleThreads) {
        float v[4];
        bool in[4];
        u64 w[4] = {0, 0, 0, 0};
        bool some = false;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int i = i0 + j * kSampleThreads;
          v[j] = i < n ? slice[i] : -INFINITY;
          in[j] = v[j] >= low && v[j] <= high;
          some |= in[j];
        }
        if (!some) continue;
        if (weights) {
          weigher.biased(v, w);
#pragma unroll
          for (int j = 0; j < 4; j++) w[j] -= Weigher::kBias;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (!in[j]) continue;
          const float p = place(v[j]);
          int b = static_cast<int>(p);
          if (bin >= 0) {
            if (b != bin) continue;
            b = static_cast<int>((p - static_cast<float>(bin)) * kBins);
          }
          atomicAdd(&s.count[b], 1u);
          add_mass(b, w[j]);
        }
      }
      sync();
      gather(tid, weights, &my_count, &my_mass);
      all_count = scan(my_count, &count_before);
      all_mass = scan(my_mass, &mass_before);
    };
    // The arrays are cleared for another histogram once everyone has read them.
    auto clear = [&]() {
      sync();
      s.mass[tid] = s.count[tid] = 0;
      __syncthreads();
    };

    // How many of the `equal` logits of weight w have less than `limit` in front of them, with
    // `front` in front of the first.
    auto take_of = [&](u64 front, u64 w, unsigned equal, double limit) {
      if (w == 0) return equal;
      const double q = (limit - static_cast<double>(front)) / static_cast<double>(w);
      unsigned take = q < 1.0 ? 1u : static_cast<unsigned>(fmin(q, 262144.0));
      while (static_cast<double>(front + take * w) < limit && take < equal) take++;
      while (take > 1 && static_cast<double>(front + (take - 1) * w) >= limit) take--;
      return min(take, equal);
    };
    constexpr int kPer = kList / kSampleThreads;
    // The row's logits in bins [lo, hi] (part >= 0: in that part of the one bin) and not below
    // `floor_value`, as keys in s.merged, the largest first.  Returns their number; more than
    // kList of them are not listed.
    auto collect = [&](int which, int lo, int hi, int part, float floor_value) -> unsigned {
      // most logits lie far from the bins: a comparison tells
      float low, high;
      bounds(lo, hi, floor_value, &low, &high);
      for (int i0 = tid; i0 < n; i0 += 8 * kSampleThreads) {
        float v[8];
        bool some = false;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int i = i0 + j * kSampleThreads;
          v[j] = i < n ? slice[i] : -INFINITY;
          some |= v[j] >= low && v[j] <= high;
        }
        if (!some) continue;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if (!(v[j] >= low && v[j] <= high)) continue;
          const float p = place(v[j]);
          const int b = static_cast<int>(p);
          if (b < lo || b > hi) continue;
          if (part >= 0 && static_cast<int>((p - static_cast<float>(b)) * kBins) != part) continue;
          const unsigned at = atomicAdd(&s.listed[which], 1u);
          if (at < kList) s.list[at] = sample_key(v[j]);
        }
      }
      sync();  // after it nobody reads counts and weights of a bin any more
      unsigned lens[split], size = 0;
#pragma unroll
      for (int k = 0; k < split; k++) {
        lens[k] = split > 1 ? peer_u32(&s.listed[which], k) : s.listed[which];
        size += lens[k];
      }
      if (size > kList) return size;
      uint32_t got[kPer];
      unsigned at = 0;
#pragma unroll
      for (int j = 0; j < kPer; j++) got[j] = 0;
#pragma unroll
      for (int k = 0; k < split; k++) {
#pragma unroll
        for (int j = 0; j < kPer; j++) {
          const unsigned i = tid + j * kSampleThreads - at;
          if (i < lens[k]) got[j] = split > 1 ? peer_u32(&s.list[i], k) : s.list[i];
        }
        at += lens[k];
      }
      // bitonic sort (zeros, no logit's key, behind)
      unsigned m = 32;
      while (m < size) m <<= 1;
#pragma unroll
      for (int j = 0; j < kPer; j++)
        if (tid + j * kSampleThreads < m) s.merged[tid + j * kSampleThreads] = got[j];
      __syncthreads();
      for (unsigned len = 2; len <= m; len <<= 1)
        for (unsigned gap = len >> 1; gap > 0; gap >>= 1) {
          if (tid < m / 2) {
            const unsigned p0 = 2 * tid - (tid & (gap - 1)), p1 = p0 + gap;
            const uint32_t x0 = s.merged[p0], x1 = s.merged[p1];
            if ((x0 < x1) == ((p0 & len) == 0)) {
              s.merged[p0] = x1;
              s.merged[p1] = x0;
            }
          }
          // up to 64 entries one warp does it all
          if (m > 64)
            __syncthreads();
          else
            __syncwarp();
        }
      __syncthreads();
      return size;
    };
    // Of the first `stay` of the `size` keys in s.merged, with weight `acc` before them: those
    // that have less than `limit` in front (limit >= 0), or with share >= 0 less than that share
    // of their own weight.  Sets the results of a search.
    auto choose = [&](unsigned size, unsigned stay, u64 acc, double limit, double share) {
      if (limit >= 0.0 || share >= 0.0) {
        u64 w[kPer], sum = 0, front;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
          const unsigned i = tid * kPer + j;
          w[j] = i < stay ? weigher(key_value(s.merged[i])) : 0;
          sum += w[j];
        }
        const u64 all = scan(sum, &front);
        if (share >= 0.0) limit = share * static_cast<double>(all);
        unsigned kept = 0;
        u64 f = acc + front;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
          kept += __syncthreads_count(tid * kPer + j < stay && static_cast<double>(f) < limit);
          f += w[j];
        }
        stay = max(kept, 1u);
      }
      const uint32_t key = s.merged[stay - 1];
      unsigned above = 0, equal = 0;
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        const unsigned i = tid * kPer + j;
        above += __syncthreads_count(i < size && s.merged[i] > key);
        equal += __syncthreads_count(i < size && s.merged[i] == key);
      }
      if (tid == 0) {
        s.edge = key;
        s.take = stay - above;
        s.equals = equal;
        s.need = s.take < equal ? s.take : kAll;
      }
      __syncthreads();
    };
    // The edge within bin s.bin (of s.size logits): the `want`-th largest of the bin, or with
    // limit >= 0 the last one that has less than `limit` in front of it, `acc` being the weight
    // of the bins before.  Sets s.edge, s.equals (logits equal to it), s.take (how many of them
    // stay) and s.need (the same, kAll if all do).
    auto search = [&](int which, bool weights, unsigned want, u64 acc, double limit) {
      const int bin = s.bin;
      const float floor_value = edge ? key_value(edge) : -INFINITY;
      int part = -1;
      if (s.size > kList && bin < kBins - 1) {
        // many logits in the bin: the same once more, in parts of the bin
        clear();
        histogram(weights, floor_value, bin);
        const bool here = limit < 0.0 ? count_before < want && want <= count_before + my_count
                                      : static_cast<double>(acc + mass_before) < limit &&
                                            static_cast<double>(acc + mass_before + my_mass) >= limit;
        if (here) {
          s.bin = tid;
          s.size = my_count;
          s.before = static_cast<unsigned>(count_before);
          s.above = mass_before;
        }
        __syncthreads();
        part = s.bin;
        want -= limit < 0.0 ? s.before : 0u;
        acc += s.above;
      }
      const unsigned in_part = s.size;
      if (in_part <= kList) {
        const unsigned size = collect(which, bin, bin, part, floor_value);
        choose(size, limit >= 0.0 ? size : want, acc, limit, -1.0);
        return;
      }
      // still many (equal ones, or the open bin): by the digits of their bits
      uint32_t prefix = 0;
      u64 heavy = 0;
      for (int shift = 24; shift >= 0; shift -= 8) {
        sync();  // everyone has read the digits of the round before
        if (tid < 256) s.mass[tid] = s.count[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kSampleThreads) {
          const float v = slice[i];
          if (v == -INFINITY || v < floor_value || bin_of(v) != bin) continue;
          if (part >= 0 && static_cast<int>((place(v) - static_cast<float>(bin)) * kBins) != part) continue;
          const uint32_t k = sample_key(v);
          if (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
          atomicAdd(&s.count[(k >> shift) & 255], 1u);
          if (weights) {
            add_mass((k >> shift) & 255, weigher(v));
          }
        }
        sync();
        unsigned c = 0;
        u64 w = 0, c_before, w_before;
        const int digit = 255 - tid;  // largest digit first
        if (tid < 256) gather(digit, weights, &c, &w);
        const u64 c_all = scan(c, &c_before);
        scan(w, &w_before);
        bool here = c > 0;
        if (limit < 0.0) {
          here = here && c_before < want && want <= c_before + c;
        } else {
          const double front = static_cast<double>(acc + heavy + w_before);
          here = here && front < limit &&
                 (static_cast<double>(acc + heavy + w_before + w) >= limit || c_before + c == c_all);
        }
        if (here) {
          s.edge = prefix | static_cast<uint32_t>(digit) << shift;
          s.before = static_cast<unsigned>(c_before);
          s.above = w_before;
          s.need = c;
        }
        __syncthreads();
        prefix = s.edge;
        want -= s.before;
        heavy += s.above;
        __syncthreads();
      }
      if (tid == 0) {
        const unsigned equal = s.need;
        const unsigned take = limit < 0.0 ? want : take_of(acc + heavy, weigher(key_value(prefix)), equal, limit);
        s.take = take;
        s.equals = equal;
        s.need = take < equal ? take : kAll;
      }
      __syncthreads();
    };

    bool done = false;
    if (by_count && top_k <= kList / 2) {
      // The top_k-th largest of the threads' maxima is not above the top_k-th largest logit, and
      // few logits lie between the two: everything from its bin on goes to the list.
      if (best > -INFINITY) atomicAdd(&s.count[bin_of(best)], 1u);
      sync();
      gather(tid, false, &my_count, &my_mass);
      all_count = scan(my_count, &count_before);
      const u64 want = top_k;
      if (want <= all_count) {
        if (count_before < want && want <= count_before + my_count) s.bin = tid;
        __syncthreads();
        const unsigned size = collect(0, 0, s.bin, -1, -INFINITY);
        if (size <= kList) {
          choose(size, top_k, 0, -1.0, by_mass ? fmax(static_cast<double>(top_p), 0.0) : -1.0);
          edge = s.edge;
          need = s.need;
          done = true;
        }
      } else {
        sync();  // everyone has read the counts
      }
      if (!done) {
        __syncthreads();
        s.mass[tid] = s.count[tid] = 0;
        __syncthreads();
      }
    }
    u64 dropped = 0;  // weight of the logits equal to the edge that top-k leaves out
    if (by_count && !done) {
      histogram(false, -INFINITY, -1);
      const u64 want = top_k;
      if (want < all_count) {
        if (count_before < want && want <= count_before + my_count) {
          s.bin = tid;
          s.size = my_count;
          s.before = static_cast<unsigned>(count_before);
        }
        __syncthreads();
        search(1, false, static_cast<unsigned>(want - s.before), 0, -1.0);
        edge = s.edge;
        need = s.need;
        dropped = (s.equals - s.take) * weigher(key_value(edge));
      }
      if (by_mass) clear();
    }
    if (by_mass && !done) {
      histogram(true, edge ? key_value(edge) : -INFINITY, -1);
      const double limit = fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(all_mass - dropped);
      if (limit > 0.0) {
        // the bin in which the weight reaches the limit
        if (static_cast<double>(mass_before) < limit && static_cast<double>(mass_before + my_mass) >= limit) {
          s.bin = tid;
          s.size = my_count;
          s.sum = mass_before;
        }
        __syncthreads();
        const u64 acc = s.sum;
        search(2, true, 0, acc, limit);
        if (s.edge > edge) {
          edge = s.edge;
          need = s.need;
        } else if (s.edge == edge) {
          need = min(need, s.need);
        }
      } else {  // the first token only
        edge = sample_key(top);
        need = 1;
      }
    }
  }
  // -------------------------------------------------------------------- 3. the draw
  const u64 least = min_p > 0.0f ? static_cast<u64>(ceil(fmin(static_cast<double>(min_p), 1.0) *
                                                         static_cast<double>(kOne)))
                                 : 0;
  const float edge_value = edge == 0 ? -INFINITY : key_value(edge);
  const int run = ((n + kSampleThreads - 1) / kSampleThreads) | 1;  // odd: no bank conflicts
  const int i0 = min(n, tid * run), i1 = min(n, i0 + run);
  u64 eq_before = 0;
  if (need != kAll) {  // ids equal to the edge in front of the thread's
    u64 eq = 0;
    for (int i = i0; i < i1; i++) eq += slice[i] == edge_value;
    const u64 all = scan(eq, &eq_before);
    if (split > 1) {
      if (tid == 0) s.equal = static_cast<unsigned>(all);
      sync();
#pragma unroll
      for (int c = 0; c < split; c++) {
        const unsigned v = peer_u32(&s.equal, c);
        if (c < rank) eq_before += v;
      }
    }
  }
  const bool all_kept = edge == 0 && least == 0;
  // weights of four ids from i on, those beyond the thread's run 0; *rank_of counts the ids
  // equal to the edge
  auto weights_at = [&](int i, u64 (&w)[4], u64 *rank_of) {
    float v[4];
    bool in[4], some = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      v[j] = i + j < i1 ? slice[i + j] : -INFINITY;
      in[j] = v[j] > -INFINITY && v[j] >= edge_value;
      if (need != kAll && in[j] && v[j] == edge_value && (*rank_of)++ >= need) in[j] = false;
      some |= in[j];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = 0;
    if (!some) return;
    weigher.biased(v, w);
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = in[j] && w[j] - Weigher::kBias >= least ? w[j] - Weigher::kBias : 0;
  };
  u64 mass = 0, before, r = eq_before, w4[4];
  int i = i0;
  if (all_kept) {
    u64 biases = 0;
    for (; i + 4 <= i1; i += 4) {
      const float v[4] = {slice[i], slice[i + 1], slice[i + 2], slice[i + 3]};
      weigher.biased(v, w4);
      mass += (w4[0] + w4[1]) + (w4[2] + w4[3]);
      biases += 4 * Weigher::kBias;
    }
    mass -= biases;
  }
  for (; i < i1; i += 4) {
    weights_at(i, w4, &r);
    mass += (w4[0] + w4[1]) + (w4[2] + w4[3]);
  }
  const u64 own = scan(mass, &before);
  u64 total = own;
  if (split > 1) {
    if (tid == 0) s.sum = own;
    sync();
    u64 sums[split];
#pragma unroll
    for (int c = 0; c < split; c++) sums[c] = peer_u64(&s.sum, c);
    total = 0;
#pragma unroll
    for (int c = 0; c < split; c++) {
      if (c < rank) before += sums[c];
      total += sums[c];
    }
  }
  // nobody leaves while its shared memory is read; what follows needs none of the others
  if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const float u = u0 > 0.0f ? fminf(u0, 0.99999994f) : 0.0f;
  const u64 target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(total));
  // the thread in whose run the target falls has its warp walk the run, an id per lane
  const unsigned here = __ballot_sync(0xffffffffu, before <= target && target < before + mass);
  if (here) {
    const int owner = __ffs(here) - 1;
    const int from = __shfl_sync(0xffffffffu, i0, owner), to = __shfl_sync(0xffffffffu, i1, owner);
    u64 sum = __shfl_sync(0xffffffffu, before, owner);
    u64 rank_of = __shfl_sync(0xffffffffu, eq_before, owner);
    for (int at = from; at < to; at += 32) {
      const float v = at + lane < to ? slice[at + lane] : -INFINITY;
      const unsigned equal = __ballot_sync(0xffffffffu, v == edge_value);
      bool in = v > -INFINITY && v >= edge_value;
      if (need != kAll && v == edge_value) in = in && rank_of + __popc(equal & ((1u << lane) - 1u)) < need;
      rank_of += __popc(equal);
      u64 w = weigher(v);
      if (!in || w < least) w = 0;
#pragma unroll
      for (int i = 1; i < 32; i <<= 1) {
        const u64 o = __shfl_up_sync(0xffffffffu, w, i);
        if (lane >= i) w += o;
      }
      const unsigned past = __ballot_sync(0xffffffffu, sum + w > target);
      if (past) {
        if (lane == 0) a.next[row] = id0 + at + __ffs(past) - 1;
        break;
      }
      sum += __shfl_sync(0xffffffffu, w, 31);
    }
  }
  if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Shared memory of a CTA that holds `logits` of them (their start is moved by up to 3, see step 1).
constexpr size_t sample_smem(int logits) { return (static_cast<size_t>(logits) + 4) * sizeof(float); }

template <typename T>
static int sample_launch(const gptoss_sample_args_t &a, int sms, cudaStream_t st) {
  // CTAs per row: as few as let two CTAs share an SM, more while that leaves SMs without work
  int split = 1;
  auto per_cta = [&](int c) { return ((a.vocab + c - 1) / c + 7) & ~7; };
  while (split < kSampleMaxSplit && per_cta(split) > kSamplePart) split *= 2;
  while (split < kSampleMaxSplit && static_cast<long long>(a.n_rows) * split * 2 <= sms && per_cta(split) > 4096)
    split *= 2;
  const int per = per_cta(split);
  const size_t smem = sample_smem(per);
  const long long grid = static_cast<long long>(a.n_rows) * split;
  if (grid > INT32_MAX) return decode_error(GPTOSS_E_CAPACITY, "sample: too many rows for one launch");
  void (*kernel)(const gptoss_sample_args_t, int) =
      split == 1 ? sample_kernel<T, 1>
                 : (split == 2 ? sample_kernel<T, 2> : (split == 4 ? sample_kernel<T, 4> : sample_kernel<T, 8>));
  // The attribute belongs to the kernel and not to this launch, and another thread may be about to
  // launch it for another vocabulary: always the most that it is ever launched with.
  const size_t most = sample_smem(split < kSampleMaxSplit ? kSamplePart : kSampleMaxVocab / kSampleMaxSplit);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kernel, a, per);
  }
  return launch_result("sample", e);
}

}  // namespace gptoss

using namespace gptoss;

extern "C" int gptoss_decode_sample(const gptoss_sample_args_t *args, void *stream) {
  if (!args) return decode_error(GPTOSS_E_INVALID, "sample: null argument");
  const gptoss_sample_args_t &a = *args;
  if (a.n_rows < 0 || a.vocab <= 0) return decode_error(GPTOSS_E_INVALID, "sample: negative number of rows or no vocabulary");
  if (a.dtype < GPTOSS_DTYPE_BF16 || a.dtype > GPTOSS_DTYPE_FP32)
    return decode_error(GPTOSS_E_INVALID, "sample: unknown dtype %d", a.dtype);
  if (a.vocab > kSampleMaxVocab)
    return decode_error(GPTOSS_E_CAPACITY, "sample: vocabulary %d is above 262144", a.vocab);
  if (a.stride < a.vocab) return decode_error(GPTOSS_E_INVALID, "sample: the row stride is shorter than the vocabulary");
  if (a.n_rows == 0) return GPTOSS_OK;
  if (!a.logits || !a.u || !a.next) return decode_error(GPTOSS_E_INVALID, "sample: null buffer");
  if (!aligned(a.logits, a.dtype == GPTOSS_DTYPE_FP32 ? 4 : 2))
    return decode_error(GPTOSS_E_INVALID, "sample: logits are not a multiple of their element size");
  OnDeviceOf dev(a.next, "sample: next");
  if (dev.code) return dev.code;
  const int sms = sm_count(dev.device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.dtype == GPTOSS_DTYPE_FP32) return sample_launch<float>(a, sms, st);
  if (a.dtype == GPTOSS_DTYPE_BF16) return sample_launch<bf16>(a, sms, st);
  return sample_launch<__half>(a, sms, st);
}
