// Rotary positions on packed rows with the append to the KV cache:
// gptoss_decode_rope_append in include/gptoss_decode_b200.h.
//
// A CTA takes kTok rows.  The angles of a row are the same for all of its heads, so they are
// computed once per row into shared memory and every head reads them there; the angle is
// formed in fp64 - position times frequency is exact to 2^-53 and its fraction of a turn is
// taken before anything is rounded to fp32, so a position of a million is as accurate as
// position 1 - for 32 angles per row of 5120 elements that costs nothing.  The rest is a
// copy: every element is read once and written once, in 16-byte vectors where sizes, strides
// and addresses allow it (V elements per vector, else one element at a time).
#include <cuda_fp16.h>

#include "common.cuh"
#include "decode_ops.h"
#include "engine.h"

namespace gptoss {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float *o) { *o = v; }
__device__ __forceinline__ void from_f32(float v, bf16 *o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half *o) { *o = __float2half_rn(v); }

// N elements moved at once, aligned to A elements.
template <typename T, int N, int A>
struct __align__(sizeof(T) * A) Pack {
  T e[N];
};

constexpr int kRopeThreads = 256;

// T: element type, V: elements per access, IL: interleaved pairs (with V = 1 an item of the
// rotated part is still a pair, read element by element).
template <typename T, int V, bool IL>
__global__ void __launch_bounds__(kRopeThreads)
rope_append_kernel(const gptoss_rope_args_t a, int rows_per_cta) {
  extern __shared__ float2 cs[];  // [rows_per_cta][half]
  constexpr int R = IL && V < 2 ? 2 : V;  // elements of one rotated item
  typedef Pack<T, R, V> PR;
  typedef Pack<T, V, V> P;
  const int half = a.rotary_dim >> 1, D = a.head_dim;
  const int row0 = blockIdx.x * rows_per_cta;
  const int rows = min(rows_per_cta, a.n_rows - row0);
  for (int i = threadIdx.x; i < rows * half; i += kRopeThreads) {
    const int r = i / half, j = i - r * half;
    const int p = a.pos[row0 + r];
    if (p < 0) continue;
    float s, c;
    if (a.angle_f32) {
      const float ang = static_cast<float>(p) * a.inv_freq[j];
      c = cosf(ang);
      s = sinf(ang);
    } else {
      const double turns = static_cast<double>(p) * static_cast<double>(a.inv_freq[j]) *
                           0.15915494309189533577;  // 1 / (2 pi)
      sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    }
    cs[i] = make_float2(c * a.concentration, s * a.concentration);
  }
  __syncthreads();
  // Items of one row: per q and k head the accesses of its rotated part (two for a pair of
  // half-split vectors) and of its copied part, then the accesses of v.
  const int rot_items = (IL ? a.rotary_dim : half) / R;
  const int head_items = rot_items + (D - a.rotary_dim) / V;
  const int qh = a.q ? a.n_q_heads : 0, kh = a.k ? a.n_kv_heads : 0;
  const int qk_items = (qh + kh) * head_items;
  const int items = qk_items + (a.v ? a.n_kv_heads * (D / V) : 0);
  for (int i = blockIdx.y * kRopeThreads + threadIdx.x; i < rows * items;
       i += gridDim.y * kRopeThreads) {
    const int r = i / items, it = i - r * items;
    const int row = row0 + r;
    if (a.pos[row] < 0) continue;
    long long slot = row;
    if (it >= qh * head_items) {
      if (a.slots) slot = a.slots[row];
      if (slot < 0 || slot >= a.n_slots) continue;
    }
    const T *src;
    T *dst;
    if (it >= qk_items) {
      const int e = (it - qk_items) * V;
      src = static_cast<const T *>(a.v) + row * a.v_stride + e;
      dst = static_cast<T *>(a.v_cache) + slot * a.v_cache_stride + e;
      *reinterpret_cast<P *>(dst) = *reinterpret_cast<const P *>(src);
      continue;
    }
    const int head = it / head_items, x = it - head * head_items;
    if (head < qh) {
      src = static_cast<const T *>(a.q) + row * a.q_stride + static_cast<size_t>(head) * D;
      dst = static_cast<T *>(a.q_out) + row * a.q_out_stride + static_cast<size_t>(head) * D;
    } else {
      src = static_cast<const T *>(a.k) + row * a.k_stride + static_cast<size_t>(head - qh) * D;
      dst = static_cast<T *>(a.k_cache) + slot * a.k_cache_stride + static_cast<size_t>(head - qh) * D;
    }
    if (x >= rot_items) {
      const int e = a.rotary_dim + (x - rot_items) * V;
      *reinterpret_cast<P *>(dst + e) = *reinterpret_cast<const P *>(src + e);
      continue;
    }
    const float2 *ang = cs + r * half;
    if (IL) {
      const int e = x * R;
      const PR in = *reinterpret_cast<const PR *>(src + e);
      PR out;
#pragma unroll
      for (int u = 0; u < R; u += 2) {
        const float2 t = ang[(e + u) >> 1];
        const float x1 = to_f32(in.e[u]), x2 = to_f32(in.e[u + 1]);
        from_f32(x1 * t.x - x2 * t.y, &out.e[u]);
        from_f32(x2 * t.x + x1 * t.y, &out.e[u + 1]);
      }
      *reinterpret_cast<PR *>(dst + e) = out;
    } else {
      const int e = x * R;
      const PR lo = *reinterpret_cast<const PR *>(src + e);
      const PR hi = *reinterpret_cast<const PR *>(src + half + e);
      PR olo, ohi;
#pragma unroll
      for (int u = 0; u < R; u++) {
        const float2 t = ang[e + u];
        const float x1 = to_f32(lo.e[u]), x2 = to_f32(hi.e[u]);
        from_f32(x1 * t.x - x2 * t.y, &olo.e[u]);
        from_f32(x2 * t.x + x1 * t.y, &ohi.e[u]);
      }
      *reinterpret_cast<PR *>(dst + e) = olo;
      *reinterpret_cast<PR *>(dst + half + e) = ohi;
    }
  }
}

// Every address that the kernel forms with `v` elements per access is a multiple of the
// access's bytes.
static bool rope_vector_fits(const gptoss_rope_args_t &a, int v, int size) {
  const int unit = a.interleaved ? a.rotary_dim : a.rotary_dim / 2;
  if (unit % v || a.head_dim % v || (a.head_dim - a.rotary_dim) % v) return false;
  const size_t bytes = static_cast<size_t>(v) * size;
  auto ok = [&](const void *p, long long stride) {
    return !p || (aligned(p, bytes) && stride % v == 0);
  };
  return ok(a.q, a.q_stride) && ok(a.q_out, a.q_out_stride) && ok(a.k, a.k_stride) &&
         ok(a.k_cache, a.k_cache_stride) && ok(a.v, a.v_stride) && ok(a.v_cache, a.v_cache_stride);
}

template <typename T, int V>
static void rope_launch(const gptoss_rope_args_t &a, dim3 grid, int rows_per_cta, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(rows_per_cta) * (a.rotary_dim / 2) * sizeof(float2);
  if (a.interleaved)
    rope_append_kernel<T, V, true><<<grid, kRopeThreads, smem, st>>>(a, rows_per_cta);
  else
    rope_append_kernel<T, V, false><<<grid, kRopeThreads, smem, st>>>(a, rows_per_cta);
}

}  // namespace gptoss

using namespace gptoss;

extern "C" int gptoss_decode_rope_append(const gptoss_rope_args_t *args, void *stream) {
  if (!args) return decode_error(GPTOSS_E_INVALID, "rope_append: null argument");
  const gptoss_rope_args_t &a = *args;
  if (a.n_rows < 0 || a.n_slots < 0) return decode_error(GPTOSS_E_INVALID, "rope_append: negative size");
  if (a.dtype < GPTOSS_DTYPE_BF16 || a.dtype > GPTOSS_DTYPE_FP32)
    return decode_error(GPTOSS_E_INVALID, "rope_append: unknown dtype %d", a.dtype);
  if (a.head_dim <= 0 || a.head_dim > 1024 || a.rotary_dim <= 0 || a.rotary_dim > a.head_dim ||
      a.rotary_dim % 2)
    return decode_error(GPTOSS_E_INVALID,
                        "rope_append: head_dim %d must be in 1..1024 and rotary_dim %d even and in 2..head_dim",
                        a.head_dim, a.rotary_dim);
  if (!a.q && !a.k && !a.v) return decode_error(GPTOSS_E_INVALID, "rope_append: q, k and v are all NULL");
  if (!a.q != !a.q_out || !a.k != !a.k_cache || !a.v != !a.v_cache)
    return decode_error(GPTOSS_E_INVALID, "rope_append: an input without its output, or the reverse");
  if ((a.q && (a.n_q_heads <= 0 || a.n_q_heads > 1024)) ||
      ((a.k || a.v) && (a.n_kv_heads <= 0 || a.n_kv_heads > 1024)))
    return decode_error(GPTOSS_E_INVALID, "rope_append: head counts must be in 1..1024");
  const long long dq = static_cast<long long>(a.n_q_heads) * a.head_dim;
  const long long dkv = static_cast<long long>(a.n_kv_heads) * a.head_dim;
  if ((a.q && (a.q_stride < dq || a.q_out_stride < dq)) ||
      (a.k && (a.k_stride < dkv || a.k_cache_stride < dkv)) ||
      (a.v && (a.v_stride < dkv || a.v_cache_stride < dkv)))
    return decode_error(GPTOSS_E_INVALID, "rope_append: a row stride is shorter than the row");
  if ((a.k || a.v) && !a.slots && a.n_slots < a.n_rows)
    return decode_error(GPTOSS_E_INVALID, "rope_append: without slots the cache needs a row for every input row");
  if (a.k && a.k == a.k_cache && (a.slots || a.k_stride != a.k_cache_stride))
    return decode_error(GPTOSS_E_INVALID, "rope_append: k in place needs slots == NULL and equal strides");
  if (a.v && a.v == a.v_cache && (a.slots || a.v_stride != a.v_cache_stride))
    return decode_error(GPTOSS_E_INVALID, "rope_append: v in place needs slots == NULL and equal strides");
  if (a.q && a.q == a.q_out && a.q_stride != a.q_out_stride)
    return decode_error(GPTOSS_E_INVALID, "rope_append: q in place needs equal strides");
  if (a.n_rows == 0) return GPTOSS_OK;
  if (!a.pos || !a.inv_freq) return decode_error(GPTOSS_E_INVALID, "rope_append: pos or inv_freq is NULL");
  const int size = a.dtype == GPTOSS_DTYPE_FP32 ? 4 : 2;
  auto off = [&](const void *p) { return !aligned(p, size); };
  if (off(a.q) || off(a.k) || off(a.v) || off(a.q_out) || off(a.k_cache) || off(a.v_cache))
    return decode_error(GPTOSS_E_INVALID, "rope_append: a pointer is not a multiple of its element size");
  OnDeviceOf dev(a.q_out ? a.q_out : (a.k_cache ? a.k_cache : a.v_cache), "rope_append: output");
  if (dev.code) return dev.code;
  // Rows per CTA: one angle per thread at most, and enough CTAs to fill the GPU before a CTA
  // takes a second row; few rows are split over CTAs along their heads instead.
  const int sms = sm_count(dev.device);
  int rows_per_cta = 1;
  while (rows_per_cta < 8 && a.n_rows >= 4 * rows_per_cta * sms) rows_per_cta *= 2;
  const int gx = (a.n_rows + rows_per_cta - 1) / rows_per_cta;
  int gy = 1;
  const dim3 grid(gx, gy);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.dtype == GPTOSS_DTYPE_FP32) {
    if (rope_vector_fits(a, 4, 4))
      rope_launch<float, 4>(a, grid, rows_per_cta, st);
    else
      rope_launch<float, 1>(a, grid, rows_per_cta, st);
  } else if (a.dtype == GPTOSS_DTYPE_BF16) {
    if (rope_vector_fits(a, 8, 2))
      rope_launch<bf16, 8>(a, grid, rows_per_cta, st);
    else if (rope_vector_fits(a, 4, 2))
      rope_launch<bf16, 4>(a, grid, rows_per_cta, st);
    else
      rope_launch<bf16, 1>(a, grid, rows_per_cta, st);
  } else {
    if (rope_vector_fits(a, 8, 2))
      rope_launch<__half, 8>(a, grid, rows_per_cta, st);
    else if (rope_vector_fits(a, 4, 2))
      rope_launch<__half, 4>(a, grid, rows_per_cta, st);
    else
      rope_launch<__half, 1>(a, grid, rows_per_cta, st);
  }
  return launch_result("rope_append");
}
