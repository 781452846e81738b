// Rotary positions on packed rows with the append to the KV cache:
// gptoss_decode_rope_append in include/gptoss_decode_b200.h.
//
// A CTA takes up to kRopeRows rows.  The angles of a row are the same for all of its heads, so they are
// computed once per row into shared memory and every head reads them there; the angle is
// formed in fp64 - position times frequency is exact to 2^-53 and its fraction of a turn is
// taken before anything is rounded to fp32, so a position of a million is as accurate as
// position 1 - for 32 angles per row of 5120 elements that costs nothing.  The rest is a
// copy: every element is read once and written once, in 16-byte vectors where sizes, strides
// and addresses allow it (V elements per vector, else one element at a time).
#include <cuda_fp16.h>

#include <string.h>

#include <algorithm>

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

// What one access moves, by its bytes; elements are taken out of it by copies of its bits
// (loads of a struct of 16-bit elements are split into 8 bytes).
template <int kBytes> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<2> { typedef uint16_t type; };

constexpr int kRopeRows = 8;  // rows of a CTA, at most

// T: element type, V: elements per access, IL: interleaved pairs.
//
// A row's work is cut into items: per q and k head the accesses of its rotated part (half-split:
// pairs of accesses; interleaved with V = 1: pairs too) and of its copied part, then the
// accesses of v.  A thread takes the same item of every row of the CTA, so that what an item is
// - two divisions - is found once.  What bounds the kernel is the bytes in flight: interleaved,
// a thread has four rows' loads on their way (30011 rows of 32 + 2 x 4 heads of 128, half of
// each rotated: 134 us with one, 106 us with four, 94 us at a copy's rate); half-split, one row's
// two loads and twice as many threads per SM are the better way to have them (8191 rows of 64 + 2
// x 8 heads of 64: 33 us, against 39 us with four rows and half as many threads; 26 us at a copy's
// rate).  Eight CTAs of 256 threads leave 32 registers, of which the 16-byte accesses spill some
// (100 bytes stored, 40 loaded).
template <typename T, int V, bool IL>
__global__ void __launch_bounds__(IL ? 384 : 256, IL ? 3 : 8)
rope_append_kernel(const gptoss_rope_args_t a, int rows_per_cta) {
  constexpr int kAhead = IL ? 4 : 1;
  constexpr int R = IL && V < 2 ? 2 : V;    // elements of one rotated item
  constexpr int kLoads = IL ? R / V : 2;    // its accesses
  typedef typename Raw<sizeof(T) * V>::type P;
  extern __shared__ float2 cs[];  // [rows_per_cta][half]
  __shared__ long long slots[kRopeRows];
  __shared__ int live[kRopeRows];
  const int half = a.rotary_dim >> 1, D = a.head_dim;
  const int row0 = blockIdx.x * rows_per_cta;
  const int rows = min(rows_per_cta, a.n_rows - row0);
  const int rot_items = (IL ? a.rotary_dim : half) / R;
  const int head_items = rot_items + (D - a.rotary_dim) / V;
  const int qh = a.q ? a.n_q_heads : 0, kh = a.k ? a.n_kv_heads : 0;
  const int qk_items = (qh + kh) * head_items;
  const int items = qk_items + (a.v ? a.n_kv_heads * (D / V) : 0);
  // the thread's item: where it comes from and goes to, and whether it is rotated
  const T *src;
  T *dst;
  long long src_stride, dst_stride;
  int x;  // index of the item in the rotated part
  bool rotate, to_cache;
  auto find_item = [&](int it) {
    int first;
    x = 0;
    rotate = false;
    to_cache = true;
    if (it >= qk_items) {
      first = (it - qk_items) * V;
      src = static_cast<const T *>(a.v);
      dst = static_cast<T *>(a.v_cache);
      src_stride = a.v_stride;
      dst_stride = a.v_cache_stride;
    } else {
      const int head = it / head_items;
      x = it - head * head_items;
      rotate = x < rot_items;
      const int in_head = rotate ? x * R : a.rotary_dim + (x - rot_items) * V;
      if (head < qh) {
        first = head * D + in_head;
        src = static_cast<const T *>(a.q);
        dst = static_cast<T *>(a.q_out);
        src_stride = a.q_stride;
        dst_stride = a.q_out_stride;
        to_cache = false;
      } else {
        first = (head - qh) * D + in_head;
        src = static_cast<const T *>(a.k);
        dst = static_cast<T *>(a.k_cache);
        src_stride = a.k_stride;
        dst_stride = a.k_cache_stride;
      }
    }
    src += row0 * src_stride + first;
    dst += first;
  };
  const int apart = IL ? V : half;  // distance of an item's second access
  P in[kAhead][kLoads];
  auto load = [&](int r0) {  // of the CTA's first row where there is no other (it exists)
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const T *at = src + (r0 + u < rows ? r0 + u : 0) * src_stride;
      in[u][0] = *reinterpret_cast<const P *>(at);
      if (kLoads > 1 && rotate) in[u][kLoads - 1] = *reinterpret_cast<const P *>(at + apart);
    }
  };
  // the first loads are on their way while the angles are made
  const bool busy = static_cast<int>(threadIdx.x) < items;
  if (busy) {
    find_item(threadIdx.x);
    load(0);
  }
  if (threadIdx.x < rows) {
    const int row = row0 + threadIdx.x;
    live[threadIdx.x] = a.pos[row] >= 0;
    const long long slot = a.slots ? a.slots[row] : row;
    slots[threadIdx.x] = slot >= 0 && slot < a.n_slots ? slot : -1;
  }
  for (int i = threadIdx.x; i < rows * half; i += blockDim.x) {
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
  for (int it = threadIdx.x; it < items; it += blockDim.x) {
    const bool again = it >= static_cast<int>(blockDim.x);
    if (again) find_item(it);
    const int angle0 = IL ? x * (R / 2) : x * R;
    for (int r0 = 0; r0 < rows; r0 += kAhead) {
      if (again || r0 > 0) load(r0);
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const int r = r0 + u;
        if (r >= rows || !live[r]) continue;
        const long long to = to_cache ? slots[r] : row0 + r;
        if (to < 0) continue;
        T *out = dst + to * dst_stride;
        if (rotate) {
          const float2 *ang = cs + r * half + angle0;
          T e[kLoads * V];
#pragma unroll
          for (int j = 0; j < kLoads; j++) memcpy(e + j * V, &in[u][j], sizeof(P));
#pragma unroll
          for (int j = 0; j < kLoads * V / 2; j++) {
            T *e1 = e + (IL ? 2 * j : j), *e2 = e + (IL ? 2 * j + 1 : V + j);
            const float2 t = ang[j];
            const float x1 = to_f32(*e1), x2 = to_f32(*e2);
            from_f32(x1 * t.x - x2 * t.y, e1);
            from_f32(x2 * t.x + x1 * t.y, e2);
          }
#pragma unroll
          for (int j = 0; j < kLoads; j++) memcpy(&in[u][j], e + j * V, sizeof(P));
          if (kLoads > 1) *reinterpret_cast<P *>(out + apart) = in[u][kLoads - 1];
        }
        *reinterpret_cast<P *>(out) = in[u][0];
      }
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
static int rope_launch(const gptoss_rope_args_t &a, int sms, cudaStream_t st) {
  // rows per CTA: enough CTAs for two waves before a CTA takes more rows
  int rows_per_cta = 1;
  while (rows_per_cta < kRopeRows && a.n_rows / (4 * rows_per_cta) >= sms) rows_per_cta *= 2;
  const int grid = (a.n_rows - 1) / rows_per_cta + 1;
  // threads: the items of a row in as few equal passes as fit
  const int most = a.interleaved ? 384 : 256;
  const int unit = a.interleaved ? (V < 2 ? 2 : V) : 2 * V;
  const int per_head = a.rotary_dim / unit + (a.head_dim - a.rotary_dim) / V;
  const int items = ((a.q ? a.n_q_heads : 0) + (a.k ? a.n_kv_heads : 0)) * per_head +
                    (a.v ? a.n_kv_heads * (a.head_dim / V) : 0);
  const int passes = (items + most - 1) / most;
  const int threads = std::max(32, (((items + passes - 1) / passes) + 31) & ~31);
  const size_t smem = static_cast<size_t>(rows_per_cta) * (a.rotary_dim / 2) * sizeof(float2);
  auto kernel = a.interleaved ? rope_append_kernel<T, V, true> : rope_append_kernel<T, V, false>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  return launch_result("rope_append", cudaLaunchKernelEx(&cfg, kernel, a, rows_per_cta));
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
  const int sms = sm_count(dev.device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.dtype == GPTOSS_DTYPE_FP32)
    return rope_vector_fits(a, 4, 4) ? rope_launch<float, 4>(a, sms, st) : rope_launch<float, 1>(a, sms, st);
  if (a.dtype == GPTOSS_DTYPE_BF16) {
    if (rope_vector_fits(a, 8, 2)) return rope_launch<bf16, 8>(a, sms, st);
    if (rope_vector_fits(a, 4, 2)) return rope_launch<bf16, 4>(a, sms, st);
    return rope_launch<bf16, 1>(a, sms, st);
  }
  if (rope_vector_fits(a, 8, 2)) return rope_launch<__half, 8>(a, sms, st);
  if (rope_vector_fits(a, 4, 2)) return rope_launch<__half, 4>(a, sms, st);
  return rope_launch<__half, 1>(a, sms, st);
}
