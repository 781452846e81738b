// Attention of sequences with a few query rows each (single tokens of a decode step):
// the other kernel behind gptoss_decode_prompt_attention.
//
// The work is reading K and V once; the arithmetic is small, and what counts is how many bytes
// are on their way at any time.  A job is 16 rows - 16 / group tokens times the query heads
// that share a KV head - which is one m16n8k16 tile, and the keys that they see.  Each of the
// CTA's warps takes every kWarps-th block of keys through a ring of its own (cp.async, no
// barrier between warps), keeps its own running maximum, sum and O, and the partial results are
// joined at the end: the warps' in shared memory, and where a cluster shares a job's keys the
// CTAs' through distributed shared memory, always in the same order.
//
// The tcgen05 kernel of prompt_attention.cu needs 128 rows per tile and several hand-shakes per
// block of keys; on 8 rows its warps wait for each other most of the time.
//
// What bounds it: the read of K and V.  One token each of 64 sequences with 1 to 7747 keys, 64/8
// heads of 64: 98 to 102 us with the same inputs, 105 with new ones for every call, 79 to 74 % of a
// copy's rate (the last jobs run alone); one token of 131071 keys: 59 us, 69 % (its 8 clusters of
// 16 CTAs are 128 CTAs, two to an SM, and leave SMs idle).  A ring of three blocks per warp, by
// those two and 256 sequences of 512 keys: 98, 59 and 66 us; of two 97, 72 and 58; of four, where
// an SM holds fewer CTAs, 93, 82 and 103.  Clusters of 8 take 75 us for the long token.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attention_rows.cuh"

namespace gptoss {

constexpr int kTokenWarps = 4;
constexpr int kTokenThreads = kTokenWarps * 32;
constexpr int kTokenSplit = 16;  // CTAs of a cluster that share a job's keys, at most

template <int D>
struct TokenShape {
  static constexpr int kKeys = D == 128 ? 16 : 32;     // keys of a block
  static constexpr int kPitch = D * 2 + 16;            // padded row: ldmatrix without conflicts
  static constexpr int kBlockBytes = kKeys * kPitch;   // of K, of V
  static constexpr int kStages = 3;
  static constexpr int kWarpBytes = kStages * 2 * kBlockBytes;
  static constexpr int kSmemBytes = kTokenWarps * kWarpBytes;
  static_assert(16 * D * 4 <= kWarpBytes, "a warp's partial output takes its ring's place");
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bf16 *) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half *) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes to shared memory, zeros where `there` is false
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0)
               : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kTokenThreads)
token_attention_kernel(const gptoss_attention_args_t a, int group, int span, int n_slots, int split) {
  typedef TokenShape<D> S;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ AttnRows job;
  __shared__ int found;
  __shared__ float warp_m[kTokenWarps][16], warp_l[kTokenWarps][16];
  __shared__ float part_m[16], part_l[16];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = split > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int unit = blockIdx.x / split;
  const int slot = unit / a.n_kv_heads, kvh = unit - slot * a.n_kv_heads;
  if (warp == 0) {
    AttnRows r;
    const bool yes = attn_find_rows(a, span, slot, kvh, lane, &r);
    if (lane == 0) {
      found = yes;
      if (yes) job = r;
    }
  }
  __syncthreads();
  if (!found) return;  // the whole cluster alike
  const int blocks = (job.keys + S::kKeys - 1) / S::kKeys;
  const int blk0 = static_cast<int>(static_cast<long long>(blocks) * rank / split);
  const int blk1 = static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / split);
  const int rows = job.tokens * group;
  const int g = lane >> 2, t4 = lane & 3;  // fragment rows g and g + 8, column pair t4

  const float c = a.scale * kLog2e;
  const int last_min = job.first_pos;
  const int first_max =
      a.window > 0 ? static_cast<int>(max(static_cast<long long>(job.first_pos) + job.tokens - a.window, -1ll)) : 0;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, base[2] = {0.f, 0.f};
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

  unsigned char *ring = smem + warp * S::kWarpBytes;
  const uint32_t ring_s = smem_u32(ring);
  // A lane copies the same 16 bytes of every kRows-th key of a block; its pointers run ahead
  // of the block at work, so a copy costs an addition and its issue.
  constexpr int kChunks = D / 8, kRows = 32 / kChunks;
  const int copy_row = lane / kChunks, copy_e = lane - copy_row * kChunks;
  const uint32_t copy_dst = ring_s + copy_row * S::kPitch + copy_e * 16;
  const long long key0 = static_cast<long long>(blk0 + warp) * S::kKeys + copy_row;
  const long long head0 = static_cast<long long>(kvh) * D + 8 * copy_e;
  const T *kp = static_cast<const T *>(a.k) + (job.kv_row0 + key0) * a.k_stride + head0;
  const T *vp = static_cast<const T *>(a.v) + (job.kv_row0 + key0) * a.v_stride + head0;
  const long long k_rows = kRows * a.k_stride, v_rows = kRows * a.v_stride;
  const long long k_skip = (kTokenWarps - 1) * S::kKeys * a.k_stride;  // to the warp's next block
  const long long v_skip = (kTokenWarps - 1) * S::kKeys * a.v_stride;
  auto fetch = [&](int b, int stage) {  // block b (none past the end) and the group's end
    const uint32_t dst = copy_dst + stage * 2 * S::kBlockBytes;
    if (b < blk1 && (b + 1) * S::kKeys <= job.keys) {
#pragma unroll
      for (int u = 0; u < S::kKeys / kRows; u++) {
        copy16(dst + u * kRows * S::kPitch, kp, true);
        copy16(dst + u * kRows * S::kPitch + S::kBlockBytes, vp, true);
        kp += k_rows;
        vp += v_rows;
      }
      kp += k_skip;
      vp += v_skip;
    } else if (b < blk1) {  // the last block: zeros in place of what lies past the last key
#pragma unroll
      for (int u = 0; u < S::kKeys / kRows; u++) {
        const bool there = b * S::kKeys + copy_row + u * kRows < job.keys;
        copy16(dst + u * kRows * S::kPitch, there ? kp : static_cast<const T *>(a.k), there);
        copy16(dst + u * kRows * S::kPitch + S::kBlockBytes, there ? vp : static_cast<const T *>(a.v), there);
        kp += k_rows;
        vp += v_rows;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < S::kStages - 1; s++) fetch(blk0 + warp + s * kTokenWarps, s);
  // Q as the MMA's row operand, straight from global memory
  uint32_t qa[D / 16][4];
  int last[2], first[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = g + 8 * h, tk = r / group;
    last[h] = job.first_pos + tk;
    first[h] = a.window > 0 ? static_cast<int>(max(static_cast<long long>(last[h]) - a.window + 1, -1ll)) : 0;
    const T *q = static_cast<const T *>(a.q) + static_cast<long long>(job.q_row0 + tk) * a.q_stride +
                 static_cast<long long>(kvh * group + r - tk * group) * D;
#pragma unroll
    for (int k = 0; k < D / 16; k++) {
      qa[k][h] = r < rows ? __ldg(reinterpret_cast<const uint32_t *>(q + 16 * k + 2 * t4)) : 0u;
      qa[k][2 + h] = r < rows ? __ldg(reinterpret_cast<const uint32_t *>(q + 16 * k + 8 + 2 * t4)) : 0u;
    }
  }
  int stage = 0;
  for (int b = blk0 + warp; b < blk1; b += kTokenWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
    __syncwarp();
    fetch(b + (S::kStages - 1) * kTokenWarps, stage == 0 ? S::kStages - 1 : stage - 1);
    const uint32_t kb = ring_s + stage * 2 * S::kBlockBytes, vb = kb + S::kBlockBytes;
    float s[S::kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < S::kKeys / 8; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; k++)
#pragma unroll
      for (int n = 0; n < S::kKeys / 16; n++) {
        uint32_t f[4];
        ldsm4(kb + (16 * n + (lane >> 4) * 8 + (lane & 7)) * S::kPitch + (2 * k + ((lane >> 3) & 1)) * 16, f);
        mma16(s[2 * n], qa[k], f[0], f[1], static_cast<T *>(nullptr));
        mma16(s[2 * n + 1], qa[k], f[2], f[3], static_cast<T *>(nullptr));
      }
    if ((b + 1) * S::kKeys - 1 > last_min || b * S::kKeys < first_max) {
      const int key = b * S::kKeys + 2 * t4;
#pragma unroll
      for (int n = 0; n < S::kKeys / 8; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int h = e >> 1, t = key + 8 * n + (e & 1);
          if (t > last[h] || t < first[h]) s[n][e] = -INFINITY;
        }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < S::kKeys / 8; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) top[h] = fmaxf(top[h], fmaxf(s[n][2 * h], s[n][2 * h + 1]));
    bool moved = false;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      top[h] *= c;
      moved |= top[h] > m[h] + 8.f;
    }
    // the maximum only moves when it grows by more than 8 (see prompt_attention.cu)
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float mn = fmaxf(m[h], top[h]);
        const float keep = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - mn);
        m[h] = mn;
        base[h] = mn == -INFINITY ? 0.f : mn;
        l[h] *= keep;
#pragma unroll
        for (int n = 0; n < D / 8; n++) {
          o[n][2 * h] *= keep;
          o[n][2 * h + 1] *= keep;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < S::kKeys / 8; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[n][e] = fast_exp2(fmaf(s[n][e], c, -base[e >> 1]));
        l[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int k = 0; k < S::kKeys / 16; k++) {
      uint32_t pa[4];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        pa[h] = pack16(s[2 * k][2 * h], s[2 * k][2 * h + 1], static_cast<T *>(nullptr));
        pa[2 + h] = pack16(s[2 * k + 1][2 * h], s[2 * k + 1][2 * h + 1], static_cast<T *>(nullptr));
      }
#pragma unroll
      for (int n = 0; n < D / 8; n += 2) {
        uint32_t f[4];
        ldsm4_t(vb + (16 * k + ((lane >> 3) & 1) * 8 + (lane & 7)) * S::kPitch + (n + (lane >> 4)) * 16, f);
        mma16(o[n], pa, f[0], f[1], static_cast<T *>(nullptr));
        mma16(o[n + 1], pa, f[2], f[3], static_cast<T *>(nullptr));
      }
    }
    __syncwarp();  // the block is read before its slot is filled again
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
  // the warp's part: O where its ring was, rows of D floats
#pragma unroll
  for (int h = 0; h < 2; h++) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t4 == 0) {
      warp_m[warp][g + 8 * h] = m[h];
      warp_l[warp][g + 8 * h] = l[h];
    }
#pragma unroll
    for (int n = 0; n < D / 8; n++)
      *reinterpret_cast<float2 *>(ring + ((g + 8 * h) * D + 8 * n + 2 * t4) * 4) =
          make_float2(o[n][2 * h], o[n][2 * h + 1]);
  }
  __syncthreads();
  // the CTA's part, 4 elements a time, in the place of the first warp's
  for (int i = threadIdx.x; i < rows * (D / 4); i += kTokenThreads) {
    const int r = i / (D / 4), e = i - r * (D / 4);
    float all = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kTokenWarps; w++) all = fmaxf(all, warp_m[w][r]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kTokenWarps; w++) {
      const float mw = warp_m[w][r];
      if (mw == -INFINITY) continue;
      const float f = fast_exp2(mw - all);
      const float4 v = *reinterpret_cast<const float4 *>(smem + w * S::kWarpBytes + (r * D + 4 * e) * 4);
      sum += warp_l[w][r] * f;
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
    }
    if (split == 1) {
      const int tk = r / group, head = kvh * group + r - tk * group;
      const float f = row_factor(all, sum, a.sinks, head);
      T *out = static_cast<T *>(a.out) + static_cast<long long>(job.q_row0 + tk) * a.out_stride +
               static_cast<long long>(head) * D + 4 * e;
      *reinterpret_cast<uint2 *>(out) = make_uint2(pack16(acc.x * f, acc.y * f, static_cast<T *>(nullptr)),
                                                   pack16(acc.z * f, acc.w * f, static_cast<T *>(nullptr)));
    } else {
      *reinterpret_cast<float4 *>(smem + (r * D + 4 * e) * 4) = acc;
      if (e == 0) {
        part_m[r] = all;
        part_l[r] = sum;
      }
    }
  }
  if (split == 1) return;
  cluster_barrier_all();
  for (int i = rank * kTokenThreads + threadIdx.x; i < rows * (D / 4); i += split * kTokenThreads) {
    const int r = i / (D / 4), e = i - r * (D / 4);
    float all = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f}, mr[kTokenSplit];
#pragma unroll
    for (int k = 0; k < kTokenSplit; k++) {
      mr[k] = k < split ? ld_cluster_f32(smem_u32(&part_m[r]), k) : -INFINITY;
      all = fmaxf(all, mr[k]);
    }
#pragma unroll
    for (int k = 0; k < kTokenSplit; k++) {
      if (mr[k] == -INFINITY) continue;
      const float f = fast_exp2(mr[k] - all);
      float v[4];
      ld_cluster_f32x4(smem_u32(smem + (r * D + 4 * e) * 4), k, v);
      sum += ld_cluster_f32(smem_u32(&part_l[r]), k) * f;
#pragma unroll
      for (int j = 0; j < 4; j++) acc[j] += v[j] * f;
    }
    const int tk = r / group, head = kvh * group + r - tk * group;
    const float f = row_factor(all, sum, a.sinks, head);
    T *out = static_cast<T *>(a.out) + static_cast<long long>(job.q_row0 + tk) * a.out_stride +
             static_cast<long long>(head) * D + 4 * e;
    *reinterpret_cast<uint2 *>(out) = make_uint2(pack16(acc[0] * f, acc[1] * f, static_cast<T *>(nullptr)),
                                                 pack16(acc[2] * f, acc[3] * f, static_cast<T *>(nullptr)));
  }
  cluster_barrier_all();  // nobody leaves while its shared memory is read
}

// Whether the device takes clusters of 16 of this kernel (a part of a GPU may not); asked once
// per device.
template <typename T, int D>
static bool takes_16() {
  static std::atomic<int> known[64];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return false;
  int state = known[device].load(std::memory_order_relaxed);
  if (state == 0) {
    typedef TokenShape<D> S;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(kTokenThreads);
    cfg.dynamicSmemBytes = S::kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 16;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    const bool yes = cudaOccupancyMaxActiveClusters(&clusters, token_attention_kernel<T, D>, &cfg) == cudaSuccess &&
                     clusters > 0;
    if (!yes) cudaGetLastError();
    state = yes ? 2 : 1;
    known[device].store(state, std::memory_order_relaxed);
  }
  return state == 2;
}

template <typename T, int D>
static int token_launch(const gptoss_attention_args_t &a, int sms, cudaStream_t st) {
  typedef TokenShape<D> S;
  const int group = a.n_q_heads / a.n_kv_heads, span = 16 / group;
  const long long slots = a.n_tokens / span + static_cast<long long>(a.n_seqs);
  if (slots > INT32_MAX) return decode_error(GPTOSS_E_CAPACITY, "prompt_attention: too many rows and sequences");
  long long most = a.max_kv_len > 0 ? a.max_kv_len : INT32_MAX;
  if (a.window > 0) most = std::min(most, static_cast<long long>(a.window) + span);
  // Share a job's keys while the CTAs (two per SM) do not fill the GPU, down to two blocks per
  // warp; sequences have at most one job on average, so there are about n_seqs jobs per head.
  const long long jobs = static_cast<long long>(a.n_seqs) * a.n_kv_heads;
  const long long blocks = (most + S::kKeys - 1) / S::kKeys;
  int split = 1;
  while (split < kTokenSplit && jobs * split * 2 <= 2 * sms && blocks >= 4 * kTokenWarps * split) split *= 2;
  auto kernel = token_attention_kernel<T, D>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes);
  if (e == cudaSuccess && split > 8) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && !takes_16<T, D>()) split = 8;
  }
  const long long grid = slots * a.n_kv_heads * split;
  if (grid > INT32_MAX) return decode_error(GPTOSS_E_CAPACITY, "prompt_attention: too many rows for one launch");
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kTokenThreads);
    cfg.dynamicSmemBytes = S::kSmemBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kernel, a, group, span, static_cast<int>(slots), split);
  }
  return launch_result("prompt_attention", e);
}

template <typename T>
static int token_for(const gptoss_attention_args_t &a, int sms, cudaStream_t st) {
  if (a.head_dim == 32) return token_launch<T, 32>(a, sms, st);
  if (a.head_dim == 64) return token_launch<T, 64>(a, sms, st);
  return token_launch<T, 128>(a, sms, st);
}

int launch_token_attention(const gptoss_attention_args_t &a, int sms, cudaStream_t st) {
  return a.dtype == GPTOSS_DTYPE_BF16 ? token_for<bf16>(a, sms, st) : token_for<__half>(a, sms, st);
}

}  // namespace gptoss
