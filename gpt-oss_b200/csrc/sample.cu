// The next token of every row from its logits and a given uniform number:
// gptoss_decode_sample in include/gptoss_decode_b200.h.
//
// The kept set is a prefix of the order (logit descending, id ascending), so it is one
// threshold: all logits above a value and the first few ids among those equal to it.  The
// thresholds of top-k (a count) and top-p (a weight) are found digit by digit on the logits'
// ordered bit patterns; nothing is sorted.  Weights are integers (multiples of 2^-44), so
// every sum is exact whatever its order, and a draw is the same for any split of the row.
//
// One CTA per row.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "decode_ops.h"
#include "engine.h"

namespace gptoss {

typedef unsigned long long u64;

constexpr int kSampleThreads = 1024;
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // sample_key(-infinity)
constexpr uint32_t kKeyPosInf = 0xff800000u;  // sample_key(+infinity)

// Order-preserving bits of a logit: NaN as -infinity, -0 as +0.
__device__ __forceinline__ uint32_t sample_key(float x) {
  if (!(x == x)) return kKeyNegInf;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ float logit_at(const float *p) { return *p; }
__device__ __forceinline__ float logit_at(const bf16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float logit_at(const __half *p) { return __half2float(*p); }

// exp((x - max) / T) in units of 2^-44.
__device__ __forceinline__ u64 weight_of(uint32_t key, uint32_t max_key, double inv_t) {
  if (key == max_key) return 1ull << 44;
  if (max_key == kKeyPosInf || key == kKeyNegInf) return 0;
  const double d = static_cast<double>(key_value(key)) - static_cast<double>(key_value(max_key));
  return static_cast<u64>(exp(d * inv_t) * 17592186044416.0 + 0.5);
}

// Sum over the block of v; every thread gets the exclusive prefix in *before.
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
  u64 base = 0, total = 0;
  for (int w = 0; w < kSampleThreads / 32; w++) {
    if (w == warp) base = total;
    total += scratch[w];
  }
  __syncthreads();
  *before = base + inc - v;
  return total;
}

struct SampleShared {
  u64 mass[256];
  unsigned count[256];
  u64 scratch[kSampleThreads / 32];
  u64 best;
  uint32_t prefix;
  u64 acc;
  unsigned need;
  int pick;
};

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const gptoss_sample_args_t a) {
  __shared__ SampleShared s;
  const int row = blockIdx.x, tid = threadIdx.x;
  if (a.pos && a.pos[row] < 0) {
    if (tid == 0) a.next[row] = -1;
    return;
  }
  const T *x = static_cast<const T *>(a.logits) + row * a.stride;
  const int V = a.vocab;
  // largest logit, lowest id among equals
  if (tid == 0) s.best = 0;
  __syncthreads();
  u64 best = 0;
  for (int i = tid; i < V; i += kSampleThreads) {
    const u64 k = static_cast<u64>(sample_key(logit_at(x + i))) << 32 | (0xffffffffu - i);
    best = max(best, k);
  }
  atomicMax(&s.best, best);
  __syncthreads();
  const uint32_t max_key = static_cast<uint32_t>(s.best >> 32);
  const int max_id = static_cast<int>(0xffffffffu - static_cast<uint32_t>(s.best));
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  if (!(temp > 0.0f) || max_key == kKeyNegInf) {
    if (tid == 0) a.next[row] = max_key == kKeyNegInf ? 0 : max_id;
    return;
  }
  const double inv_t = 1.0 / static_cast<double>(temp);
  const int top_k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f;
  const float min_p = a.min_p ? a.min_p[row] : 0.0f;
  // kept: keys above `edge`, and the first `need` ids of those equal to it
  uint32_t edge = 0;
  unsigned need = 0xffffffffu;
  for (int mode = 0; mode < 2; mode++) {  // 0: top-k by count, 1: top-p by weight
    if (mode == 0 && (top_k <= 0 || top_k >= V)) continue;
    if (mode == 1 && !(top_p < 1.0f)) continue;
    double limit = 0.0;
    if (mode == 1) {
      u64 mine = 0, eq = 0, before;
      for (int i = tid; i < V; i += kSampleThreads) {
        const uint32_t k = sample_key(logit_at(x + i));
        if (k > edge) mine += weight_of(k, max_key, inv_t);
        if (k == edge) eq++;
      }
      u64 total = block_scan(mine, &before, s.scratch);
      eq = block_scan(eq, &before, s.scratch);
      total += min(eq, static_cast<u64>(need)) * weight_of(edge, max_key, inv_t);
      limit = fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(total);
    }
    if (tid == 0) {
      s.prefix = 0;
      s.acc = 0;
      s.need = top_k;
    }
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSampleThreads) s.mass[i] = s.count[i] = 0;
      __syncthreads();
      const uint32_t prefix = s.prefix;
      for (int i = tid; i < V; i += kSampleThreads) {
        const uint32_t k = sample_key(logit_at(x + i));
        if (k < edge || (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
        atomicAdd(&s.count[(k >> shift) & 255], 1u);
        if (mode == 1) atomicAdd(&s.mass[(k >> shift) & 255], weight_of(k, max_key, inv_t));
      }
      __syncthreads();
      if (tid == 0) {
        int last = 0;
        for (int b = 255; b >= 0; b--) {
          if (!s.count[b]) continue;
          last = b;
          if (mode == 0) {
            if (s.need <= s.count[b]) break;
            s.need -= s.count[b];
          } else {
            if (static_cast<double>(s.acc + s.mass[b]) >= limit) break;
            s.acc += s.mass[b];
          }
        }
        s.prefix |= static_cast<uint32_t>(last) << shift;
        if (mode == 1 && shift == 0) {
          const u64 w = weight_of(s.prefix, max_key, inv_t);
          unsigned n = 1;
          if (w > 0) {
            const double q = (limit - static_cast<double>(s.acc)) / static_cast<double>(w);
            n = q < 1.0 ? 1u : static_cast<unsigned>(fmin(q, 262144.0));
            while (static_cast<double>(s.acc + n * w) < limit) n++;
            while (n > 1 && static_cast<double>(s.acc + (n - 1) * w) >= limit) n--;
          }
          s.need = min(n, s.prefix == edge ? need : s.count[last]);
        }
      }
      __syncthreads();
    }
    edge = s.prefix;
    need = s.need;
    __syncthreads();
  }
  // running sums in the order of the ids: a thread owns a run of consecutive ids
  const int per = (V + kSampleThreads - 1) / kSampleThreads;
  const int i0 = min(V, tid * per), i1 = min(V, i0 + per);
  const double least = min_p > 0.0f ? fmin(static_cast<double>(min_p), 1.0) * 17592186044416.0 : 0.0;
  u64 eq = 0, eq_before, mass = 0, before;
  for (int i = i0; i < i1; i++) eq += sample_key(logit_at(x + i)) == edge;
  block_scan(eq, &eq_before, s.scratch);
  for (int pass = 0; pass < 2; pass++) {
    u64 total = 0, target = 0;
    if (pass == 1) {
      total = block_scan(mass, &before, s.scratch);
      const float u0 = a.u[row];
      const float u = u0 > 0.0f ? fminf(u0, 0.99999994f) : 0.0f;
      target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(total));
      if (!(before <= target && target < before + mass)) return;
    }
    u64 run = before, rank = eq_before;
    for (int i = i0; i < i1; i++) {
      const uint32_t k = sample_key(logit_at(x + i));
      if (k < edge || (k == edge && rank++ >= need)) continue;
      const u64 w = weight_of(k, max_key, inv_t);
      if (static_cast<double>(w) < least) continue;
      if (pass == 0) {
        mass += w;
      } else {
        run += w;
        if (run > target) {
          a.next[row] = i;
          return;
        }
      }
    }
  }
}

}  // namespace gptoss

using namespace gptoss;

extern "C" int gptoss_decode_sample(const gptoss_sample_args_t *args, void *stream) {
  if (!args) return decode_error(GPTOSS_E_INVALID, "sample: null argument");
  const gptoss_sample_args_t &a = *args;
  if (a.n_rows < 0 || a.vocab <= 0) return decode_error(GPTOSS_E_INVALID, "sample: negative number of rows or no vocabulary");
  if (a.dtype < GPTOSS_DTYPE_BF16 || a.dtype > GPTOSS_DTYPE_FP32)
    return decode_error(GPTOSS_E_INVALID, "sample: unknown dtype %d", a.dtype);
  if (a.vocab > (1 << 18))
    return decode_error(GPTOSS_E_CAPACITY, "sample: vocabulary %d is above 262144", a.vocab);
  if (a.stride < a.vocab) return decode_error(GPTOSS_E_INVALID, "sample: the row stride is shorter than the vocabulary");
  if (a.n_rows == 0) return GPTOSS_OK;
  if (!a.logits || !a.u || !a.next) return decode_error(GPTOSS_E_INVALID, "sample: null buffer");
  if (!aligned(a.logits, a.dtype == GPTOSS_DTYPE_FP32 ? 4 : 2))
    return decode_error(GPTOSS_E_INVALID, "sample: logits are not a multiple of their element size");
  OnDeviceOf dev(a.next, "sample: next");
  if (dev.code) return dev.code;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.dtype == GPTOSS_DTYPE_FP32)
    sample_kernel<float><<<a.n_rows, kSampleThreads, 0, st>>>(a);
  else if (a.dtype == GPTOSS_DTYPE_BF16)
    sample_kernel<bf16><<<a.n_rows, kSampleThreads, 0, st>>>(a);
  else
    sample_kernel<__half><<<a.n_rows, kSampleThreads, 0, st>>>(a);
  return launch_result("sample");
}
