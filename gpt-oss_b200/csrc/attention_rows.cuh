// Shared by the attention kernels: which sequence a slot of query rows belongs to, 16-bit
// packing, reads of another CTA's shared memory, the final factor of a row.
#pragma once
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "decode_ops.h"
#include "engine.h"
#include "umma_2sm.cuh"

namespace gptoss {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bf16 *) { return pack_bf16(lo, hi); }
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __half *) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t cta) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(cta));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void ld_cluster_f32x4(uint32_t addr, uint32_t cta, float *v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(cta));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "r"(remote)
               : "memory");
}
// What a row's sum of p v is multiplied with: 1 / (l + 2^(sink' - m)); 0 where no key was seen.
__device__ __forceinline__ float row_factor(float m, float l, const float *sinks, int head) {
  if (m == -INFINITY) return 0.f;
  if (!sinks) return 1.f / l;
  const float sink = sinks[head] * kLog2e;
  const float all = fmaxf(m, sink);
  const float f = fast_exp2(m - all);
  return f / (l * f + fast_exp2(sink - all));
}

// Query rows of one sequence and the keys that they see.
struct AttnRows {
  int q_row0;        // first query row
  int tokens;        // query tokens, at most the span
  long long kv_row0; // first key seen (row of k)
  int first_pos;     // position of the first query token relative to that key
  int keys;          // keys from that one to the last that any of the tokens sees
};

// Slots: a slot covers `span` tokens; sequence i's slots start at q_start[i] / span + i, which
// leaves room for a partial slot per sequence and needs no prefix sum.  One warp finds the
// slot's sequence by counting the starts at or before it, 128 of them at a time: among more
// sequences every 128th part is looked at first.  The slots (of all KV heads) together check
// every entry of q_start, 32 each; starts that do not ascend give some sequence or none, never
// rows outside the tensors.  Returns (warp-uniform, all lanes get the rows) whether there is
// anything to do for the slot.
__device__ __forceinline__ bool attn_find_rows(const gptoss_attention_args_t &a, int span, int slot,
                                               int kvh, int lane, AttnRows *rows) {
  const long long mine = (static_cast<long long>(slot) * a.n_kv_heads + kvh) * 32 + lane;
  int from = 0, to = 0;
  if (mine < a.n_seqs) {
    from = __ldg(a.q_start + mine);
    to = __ldg(a.q_start + mine + 1);
  }
  int below = 0, among = a.n_seqs;
  while (true) {
    const int step = (among - 1) / 128 + 1;
    int n = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const long long at = static_cast<long long>(lane + 32 * k) * step;
      if (at < among) {
        const int i = below + static_cast<int>(at);
        n += __ldg(a.q_start + i) / span <= slot - i;
      }
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (step == 1) {
      below += n;
      break;
    }
    if (n == 0) break;  // (only among all of them, and then the first start is not 0)
    below += (n - 1) * step;
    among = min(step, among - (n - 1) * step);
  }
  if (from < 0 || to < from || to > a.n_tokens) set_status(a.status, kStatusBadIndex);
  const int seq = below - 1;
  if (seq < 0) return false;
  const int q0 = __ldg(a.q_start + seq), q1 = __ldg(a.q_start + seq + 1);
  const long long start = __ldg(a.kv_start + seq);
  const int len = __ldg(a.kv_len + seq);
  if (q0 < 0 || q1 < q0 || q1 > a.n_tokens) return false;
  const long long t0 = static_cast<long long>(slot - (q0 / span + seq)) * span;
  const int len_q = q1 - q0;
  if (t0 < 0 || t0 >= len_q) return false;
  if (len < 0 || start < 0 || start > a.n_kv_rows - len) {
    set_status(a.status, kStatusBadIndex);
    return false;
  }
  rows->tokens = static_cast<int>(min(static_cast<long long>(span), len_q - t0));
  const long long pos = static_cast<long long>(len) - len_q + t0;  // of the first token
  const long long lo = a.window > 0 ? max(0ll, pos - a.window + 1) : 0;
  rows->q_row0 = q0 + static_cast<int>(t0);
  rows->kv_row0 = start + lo;
  rows->first_pos = static_cast<int>(pos - lo);
  rows->keys = static_cast<int>(max(lo, pos + rows->tokens) - lo);
  return true;
}

}  // namespace gptoss
