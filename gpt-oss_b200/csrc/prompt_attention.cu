// Attention of packed query rows over K / V rows: gptoss_decode_prompt_attention in
// include/gptoss_decode_b200.h.
//
// One warp per (query row, query head): the lanes hold the head's elements, keys come one
// after the other, and a running maximum and sum (fp32) make it one pass.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "decode_ops.h"
#include "engine.h"

namespace gptoss {

__device__ __forceinline__ float load_f32(const bf16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f32(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ void store_f32(bf16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f32(__half *p, float v) { *p = __float2half_rn(v); }

template <typename T, int D>
__global__ void __launch_bounds__(256) prompt_attention_kernel(const gptoss_attention_args_t a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int row = static_cast<int>(w / a.n_q_heads), h = static_cast<int>(w % a.n_q_heads);
  if (row >= a.n_tokens) return;
  // the sequence of this row
  int seq = -1, q0 = 0, q1 = 0;
  for (int i = 0; i < a.n_seqs; i++) {
    q0 = a.q_start[i];
    q1 = a.q_start[i + 1];
    if (q0 < 0 || q1 < q0 || q1 > a.n_tokens) {
      set_status(a.status, kStatusBadIndex);
      continue;
    }
    if (row >= q0 && row < q1) {
      seq = i;
      break;
    }
  }
  if (seq < 0) return;
  const long long start = a.kv_start[seq];
  const int len = a.kv_len[seq];
  if (len < 0 || start < 0 || start > a.n_kv_rows - len) {
    set_status(a.status, kStatusBadIndex);
    return;
  }
  const int p = len - (q1 - q0) + (row - q0);
  const int t0 = a.window > 0 ? max(0, p - a.window + 1) : 0;
  const int kvh = h / (a.n_q_heads / a.n_kv_heads);
  const T *q = static_cast<const T *>(a.q) + row * a.q_stride + h * D;
  const T *k = static_cast<const T *>(a.k) + start * a.k_stride + kvh * D;
  const T *v = static_cast<const T *>(a.v) + start * a.v_stride + kvh * D;
  float qr[E], o[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    qr[e] = load_f32(q + lane + 32 * e) * a.scale;
    o[e] = 0.f;
  }
  float m = a.sinks ? a.sinks[h] : -INFINITY, l = a.sinks ? 1.f : 0.f;
  for (int t = t0; t <= p; t++) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) s += qr[e] * load_f32(k + t * a.k_stride + lane + 32 * e);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    const float mn = fmaxf(m, s);
    const float keep = __expf(m - mn), pr = __expf(s - mn);
    l = l * keep + pr;
    m = mn;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = o[e] * keep + pr * load_f32(v + t * a.v_stride + lane + 32 * e);
  }
  T *out = static_cast<T *>(a.out) + row * a.out_stride + h * D;
#pragma unroll
  for (int e = 0; e < E; e++) store_f32(out + lane + 32 * e, p < 0 ? 0.f : o[e] / l);
}

template <typename T>
static void attention_launch(const gptoss_attention_args_t &a, cudaStream_t st) {
  const long long warps = static_cast<long long>(a.n_tokens) * a.n_q_heads;
  const unsigned grid = static_cast<unsigned>((warps + 7) / 8);
  if (a.head_dim == 32)
    prompt_attention_kernel<T, 32><<<grid, 256, 0, st>>>(a);
  else if (a.head_dim == 64)
    prompt_attention_kernel<T, 64><<<grid, 256, 0, st>>>(a);
  else
    prompt_attention_kernel<T, 128><<<grid, 256, 0, st>>>(a);
}

}  // namespace gptoss

using namespace gptoss;

extern "C" int gptoss_decode_prompt_attention(const gptoss_attention_args_t *args, void *stream) {
  if (!args) return decode_error(GPTOSS_E_INVALID, "prompt_attention: null argument");
  const gptoss_attention_args_t &a = *args;
  if (a.n_tokens < 0 || a.n_seqs < 0 || a.n_kv_rows < 0 || a.window < 0 || a.max_kv_len < 0)
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: negative size");
  if (a.dtype != GPTOSS_DTYPE_BF16 && a.dtype != GPTOSS_DTYPE_FP16)
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: dtype must be bf16 or fp16");
  if (a.head_dim != 32 && a.head_dim != 64 && a.head_dim != 128)
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: head_dim must be 32, 64 or 128");
  if (a.n_kv_heads <= 0 || a.n_q_heads <= 0 || a.n_q_heads % a.n_kv_heads ||
      a.n_q_heads / a.n_kv_heads > 128 || a.n_kv_heads > 1024)
    return decode_error(GPTOSS_E_INVALID,
                        "prompt_attention: n_q_heads must be a multiple of n_kv_heads, at most 128 times it");
  if (!(a.scale > 0.f) || !isfinite(a.scale))
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: scale must be positive and finite");
  const long long dq = static_cast<long long>(a.n_q_heads) * a.head_dim;
  const long long dkv = static_cast<long long>(a.n_kv_heads) * a.head_dim;
  if (a.q_stride < dq || a.out_stride < dq || a.k_stride < dkv || a.v_stride < dkv)
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: a row stride is shorter than the row");
  // 16-byte rows for the tensor maps, whose strides are below 2^40 bytes
  auto bad = [](long long stride) { return stride % 8 != 0 || stride >= (1ll << 38); };
  if (bad(a.q_stride) || bad(a.k_stride) || bad(a.v_stride) || bad(a.out_stride))
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: row strides must be multiples of 8 elements");
  if (a.n_kv_rows > INT32_MAX)
    return decode_error(GPTOSS_E_CAPACITY, "prompt_attention: more than 2^31 - 1 K / V rows");
  if (a.n_tokens == 0 || a.n_seqs == 0) return GPTOSS_OK;
  if (!a.q || !a.out || !a.q_start || !a.kv_start || !a.kv_len || (a.n_kv_rows > 0 && (!a.k || !a.v)))
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: null buffer");
  if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16))
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: q, k, v and out must be 16-byte aligned");
  OnDeviceOf dev(a.out, "prompt_attention: out");
  if (dev.code) return dev.code;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.dtype == GPTOSS_DTYPE_BF16)
    attention_launch<bf16>(a, st);
  else
    attention_launch<__half>(a, st);
  return launch_result("prompt_attention");
}
