// Attention of packed query rows over K / V rows: gptoss_decode_prompt_attention in
// include/gptoss_decode_b200.h.
//
//   o = sum_t p_t v_t / (sum_t p_t + 2^(sink' - m)),   p_t = 2^(c q.k_t - m),  c = scale log2 e
//
// A tile is 128 rows of one MMA: kTok = 128 / group query tokens times the `group` query heads
// that share a KV head, so K and V are read once for the whole group and a sequence of a few
// tokens still fills rows.  A CTA owns two tiles (A and B, consecutive tokens) of one sequence
// and KV head and runs them over the same stream of blocks of 128 keys:
//   warps 0-3, 4-7  softmax of tile A, of tile B: a thread owns a row (a TMEM lane)
//   warp 8          TMA: Q of both tiles once, then K and V blocks into two rings
//   warp 9          TMEM allocation and the MMAs, S = Q K^T and O += P V
// S comes from TMEM into registers whole (128 per thread), so the row maximum costs no second
// read; P goes back to TMEM as the MMA's 16-bit row operand, V is read in place as an N-major
// operand.  The maximum that scales a row is only moved when it grows by more than 8 (a factor
// of 256; fp32 sums and 16-bit floating-point P lose nothing by that), so O is rarely rescaled
// and the thread that owns the row does it itself.
//
// What bounds it: an exponential per (row, key), 16 per cycle and SM, is 1024 cycles per tile
// and block; the two MMAs take 256 each at head_dim 64 and 512 each at 128.  Two tiles keep
// the exponentials going while the other tile's MMAs run; at head_dim <= 64 there is room in
// TMEM for P beside S, and the next S is computed while P is still being made.
//
// Few tiles and long contexts: a cluster of up to 8 CTAs shares one pair of tiles, each taking
// an equal run of key blocks; the partial (m, l, O) are joined through distributed shared
// memory, in rank order, so the result does not depend on timing and no workspace is needed.
//
// Probabilities are rounded to the 16-bit type for the second product (tensor cores take both
// operands in one type); their sum is taken in fp32 before that rounding.
#include <cuda.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "decode_ops.h"
#include "engine.h"
#include "umma_2sm.cuh"

namespace gptoss {

constexpr int kAttnThreads = 320;
constexpr int kKeys = 128;            // keys per block
constexpr int kAttnTmemCols = 512;
constexpr int kAttnMaxSplit = 8;      // CTAs of a cluster that share a pair of tiles

template <int D>
struct AttnShape {
  static constexpr int kBox = D < 64 ? D : 64;            // elements of one swizzled row
  static constexpr int kPanels = D / kBox;                // 64-wide panels of a head
  static constexpr int kPanelBytes = 128 * kBox * 2;      // 128 rows of a panel
  static constexpr int kTileBytes = kPanels * kPanelBytes;
  static constexpr int kStages = D == 128 ? 2 : 4;        // K blocks and V blocks in flight
  static constexpr int kRingBytes = kStages * kTileBytes;
  // P beside S in TMEM (S 2 x 128 columns, P 2 x 64, O 2 x D), or in S's place
  static constexpr bool kApart = D <= 64;
  static constexpr int kColP = kApart ? 256 : 0;
  static constexpr int kStrideP = kApart ? 64 : 128;
  static constexpr int kColO = kApart ? 384 : 256;
  static constexpr int kStrideO = kApart ? 64 : 128;
  static constexpr int kOperandBytes = 2 * kTileBytes + 2 * kRingBytes;
  // fp32 partial outputs of both tiles take the operands' place in a split launch
  static constexpr int kSmemBytes = 1024 + (kOperandBytes > 256 * D * 4 ? kOperandBytes : 256 * D * 4);
};

struct AttnBarriers {
  uint64_t q_full[2], s_full[2], s_free[2], p_full[2], o_full[2], v_tail;
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
};

// Which rows a CTA works on, found once by one warp.
struct AttnJob {
  int seq;                // -1: nothing to do
  int q_row0;             // first query row of the pair of tiles
  int tokens[2];          // valid tokens of the tiles
  int kv_row0;            // first key of block 0 (row of k)
  int first_pos;          // position of the first query token, relative to block 0's first key
  int keys;               // keys from block 0's first to the last that the pair sees
  int begin[2], end[2];   // blocks of each tile, within this CTA's share
  int blk0, blk1;         // blocks of this CTA
};

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
// one CTA, M operand in tensor memory
__device__ __forceinline__ void umma_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *smem_dst, const void *tmap, uint64_t *bar, int c0,
                                            int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];"
      :
      : "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)),
        "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t cta) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(cta));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// A wait whose outcome the whole warp shares (what follows is issued by the converged warp).
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
}

// Shared-memory descriptors of operands that TMA wrote with rows of kBox elements and the
// matching swizzle: groups of 8 rows are 8 * row bytes apart.  For an operand read along its
// rows (K major) the leading offset is unused; for one read across them (V: N major) it is the
// distance of the 64-wide panels.
template <int D>
__device__ __forceinline__ uint64_t attn_desc(uint32_t addr) {
  typedef AttnShape<D> S;
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr & 0x3ffff) >> 4);
  d |= static_cast<uint64_t>(S::kPanels > 1 ? S::kPanelBytes >> 4 : 1) << 16;
  d |= static_cast<uint64_t>((8 * S::kBox * 2) >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(S::kBox == 64 ? 2 : 4) << 61;
  return d;
}
// fp32 accumulator, 16-bit operands; b_n_major: V
__host__ __device__ constexpr uint32_t attn_idesc(bool fp16, int n, bool b_n_major) {
  return (1u << 4) | (fp16 ? 0u : (1u << 7) | (1u << 10)) | (b_n_major ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}

__device__ __forceinline__ void ld_cluster_f32x4(uint32_t addr, uint32_t cta, float *v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(cta));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "r"(remote)
               : "memory");
}
// Byte offset of 16-byte piece `piece` of fp32 row `row` among the partial outputs.
template <int D>
__device__ __forceinline__ uint32_t part_offset(int row, int piece) {
  return static_cast<uint32_t>((row * (D / 4) + (piece ^ (row & 7))) * 16);
}
// What a row's sum of p v is multiplied with: 1 / (l + 2^(sink' - m)); 0 where no key was seen.
__device__ __forceinline__ float row_factor(float m, float l, const float *sinks, int head) {
  if (m == -INFINITY) return 0.f;
  if (!sinks) return 1.f / l;
  const float sink = sinks[head] * 1.4426950408889634f;
  const float all = fmaxf(m, sink);
  const float f = fast_exp2(m - all);
  return f / (l * f + fast_exp2(sink - all));
}

// Slots: a pair of tiles covers 2 * tok tokens; sequence i's pairs start at slot
// q_start[i] / (2 tok) + i, which leaves room for a partial pair per sequence and needs no
// prefix sum.  One warp finds the slot's sequence by counting the starts at or before it.
__device__ void attn_find_job(const gptoss_attention_args_t &a, int tok, int slot, int rank, int split,
                              int lane, AttnJob *job) {
  const int pair = 2 * tok;
  int below = 0;
  bool broken = false;
  for (int i0 = 0; i0 < a.n_seqs; i0 += 32) {
    const int i = i0 + lane;
    bool hit = false;
    if (i < a.n_seqs) {
      const int q0 = a.q_start[i];
      broken |= q0 < 0 || a.q_start[i + 1] < q0 || a.q_start[i + 1] > a.n_tokens;
      hit = q0 / pair + i <= slot;
    }
    below += __popc(__ballot_sync(0xffffffffu, hit));
  }
  if (broken) set_status(a.status, kStatusBadIndex);
  if (lane != 0) return;
  job->seq = -1;
  job->blk0 = job->blk1 = 0;
  for (int x = 0; x < 2; x++) job->tokens[x] = job->begin[x] = job->end[x] = 0;
  const int seq = below - 1;
  if (seq < 0) return;
  const int q0 = a.q_start[seq], q1 = a.q_start[seq + 1];
  if (q0 < 0 || q1 < q0 || q1 > a.n_tokens) return;
  const long long t0 = static_cast<long long>(slot - (q0 / pair + seq)) * pair;
  const int len_q = q1 - q0;
  if (t0 < 0 || t0 >= len_q) return;
  const long long start = a.kv_start[seq];
  const int len = a.kv_len[seq];
  if (len < 0 || start < 0 || start > a.n_kv_rows - len) {
    set_status(a.status, kStatusBadIndex);
    return;
  }
  const int n_tok = static_cast<int>(min(static_cast<long long>(pair), len_q - t0));
  const long long pos = static_cast<long long>(len) - len_q + t0;  // of the pair's first token
  const long long lo = a.window > 0 ? max(0ll, pos - a.window + 1) : 0;
  const long long hi = max(lo, pos + n_tok);  // one past the last key that the pair sees
  const int blocks = static_cast<int>((hi - lo + kKeys - 1) / kKeys);
  job->seq = seq;
  job->q_row0 = q0 + static_cast<int>(t0);
  job->kv_row0 = static_cast<int>(start + lo);
  job->first_pos = static_cast<int>(pos - lo);
  job->keys = static_cast<int>(hi - lo);
  job->blk0 = static_cast<int>(static_cast<long long>(blocks) * rank / split);
  job->blk1 = static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / split);
  for (int x = 0; x < 2; x++) {
    const int n = min(max(n_tok - x * tok, 0), tok);
    job->tokens[x] = n;
    if (n == 0) continue;
    const long long p = pos + x * tok;  // the tile's first token
    const long long from = a.window > 0 ? max(0ll, p - a.window + 1) - lo : 0;
    const long long to = p + n - lo;    // may be <= 0
    const int b = static_cast<int>(from / kKeys);
    const int e = to > 0 ? static_cast<int>((to + kKeys - 1) / kKeys) : 0;
    job->begin[x] = max(b, job->blk0);
    job->end[x] = max(job->begin[x], min(e, job->blk1));
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kAttnThreads, 1)
prompt_attention_kernel(const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const gptoss_attention_args_t a,
                        int group, int tok, int n_slots, int split) {
  typedef AttnShape<D> S;
  constexpr bool kHalf = !std::is_same<T, bf16>::value;
  extern __shared__ unsigned char smem_raw[];
  __shared__ AttnBarriers bar;
  __shared__ AttnJob job;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_word;
  __shared__ float part_m[256], part_l[256];
  unsigned char *smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  unsigned char *sm_q = smem, *sm_k = smem + 2 * S::kTileBytes, *sm_v = sm_k + S::kRingBytes;
  volatile int *abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = split > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  // the last slots first: a long prompt's last tiles see the most keys
  const int unit = blockIdx.x / split;
  const int slot = n_slots - 1 - unit / a.n_kv_heads, kvh = unit % a.n_kv_heads;

  if (warp == 9) {
    tmem_alloc(&tmem_holder, kAttnTmemCols);
    tmem_relinquish();
  } else if (warp == 8) {
    attn_find_job(a, tok, slot, rank, split, lane, &job);
  } else if (threadIdx.x == 0) {
    for (int x = 0; x < 2; x++) {
      mbar_init(&bar.q_full[x], 1);
      mbar_init(&bar.s_full[x], 1);
      mbar_init(&bar.s_free[x], 4);
      mbar_init(&bar.p_full[x], 4);
      mbar_init(&bar.o_full[x], 1);
    }
    mbar_init(&bar.v_tail, 1);
    for (int s = 0; s < S::kStages; s++) {
      mbar_init(&bar.k_full[s], 1);
      mbar_init(&bar.k_empty[s], 1);
      mbar_init(&bar.v_full[s], 1);
      mbar_init(&bar.v_empty[s], 1);
    }
    abort_word = 0;
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;

  float m = -INFINITY, l = 0.f;  // a softmax thread's row
  if (job.seq >= 0 && warp == 8) {
    // ---------------------------------------------------------------- loads
    const int n = job.blk1 - job.blk0;
    if (n > 0 && elect_one()) {
      for (int x = 0; x < 2; x++) {
        if (job.begin[x] >= job.end[x]) continue;
        mbar_arrive_expect_tx(&bar.q_full[x], static_cast<uint32_t>(S::kPanels) * tok * group * S::kBox * 2);
        for (int p = 0; p < S::kPanels; p++)
          tma_load_3d(sm_q + x * S::kTileBytes + p * S::kPanelBytes, &map_q, &bar.q_full[x],
                      p * S::kBox, kvh * group, job.q_row0 + x * tok);
      }
    }
    bool ok = true;
    for (int i = 0; i < n && ok; i++) {
      const int st = i % S::kStages;
      const uint32_t free_parity = (static_cast<uint32_t>(i / S::kStages) & 1u) ^ 1u;
      const int rel = (job.blk0 + i) * kKeys;
      const bool tail = rel + kKeys > job.keys;
      ok = warp_wait(&bar.k_empty[st], free_parity, abort_flag);
      if (ok && elect_one()) {
        mbar_arrive_expect_tx(&bar.k_full[st], S::kTileBytes);
        for (int p = 0; p < S::kPanels; p++)
          tma_load_3d(sm_k + st * S::kTileBytes + p * S::kPanelBytes, &map_k, &bar.k_full[st],
                      p * S::kBox, kvh, job.kv_row0 + rel);
      }
      ok = ok && warp_wait(&bar.v_empty[st], free_parity, abort_flag);
      // The last block may reach past the last key: what lies there may be anything, and 0
      // times NaN is NaN, so those rows of V are cleared before the block is handed on.
      uint64_t *landed = tail ? &bar.v_tail : &bar.v_full[st];
      unsigned char *v = sm_v + st * S::kTileBytes;
      if (ok && elect_one()) {
        mbar_arrive_expect_tx(landed, S::kTileBytes);
        for (int p = 0; p < S::kPanels; p++)
          tma_load_3d(v + p * S::kPanelBytes, &map_v, landed, p * S::kBox, kvh, job.kv_row0 + rel);
      }
      if (ok && tail) {
        ok = warp_wait(landed, 0, abort_flag);
        constexpr int kRowChunks = S::kBox * 2 / 16;
        for (int p = 0; ok && p < S::kPanels; p++)
          for (int c = (job.keys - rel) * kRowChunks + lane; c < kKeys * kRowChunks; c += 32)
            *reinterpret_cast<uint4 *>(v + p * S::kPanelBytes + c * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.v_full[st]);
      }
      if (!ok) {
        set_status(a.status, kStatusWaitTimeoutProducer);
        *abort_flag = 1;
      }
    }
  } else if (job.seq >= 0 && warp == 9) {
    // ---------------------------------------------------------------- MMAs
    constexpr uint32_t idesc_s = attn_idesc(kHalf, kKeys, false);
    constexpr uint32_t idesc_o = attn_idesc(kHalf, D, true);
    const uint64_t desc_q = attn_desc<D>(smem_u32(sm_q));
    const uint64_t desc_k = attn_desc<D>(smem_u32(sm_k));
    const uint64_t desc_v = attn_desc<D>(smem_u32(sm_v));
    const int b0 = job.blk0, n = job.blk1 - job.blk0;
    int s_done[2] = {0, 0}, o_done[2] = {0, 0};  // products issued per tile
    bool ok = true;
    auto active = [&](int x, int i) { return b0 + i >= job.begin[x] && b0 + i < job.end[x]; };
    auto scores = [&](int x, int i) {  // S_x = Q_x K_i^T
      const int st = i % S::kStages;
      if (s_done[x] == 0) ok = ok && warp_wait(&bar.q_full[x], 0, abort_flag);
      // S is free again once its readers have it in registers; where P takes its place, the
      // product that read that P was issued before (products run in the order of issue)
      if (S::kApart && s_done[x] > 0)
        ok = ok && warp_wait(&bar.s_free[x], (s_done[x] - 1) & 1, abort_flag);
      if (!ok) return;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
          constexpr int kPerPanel = S::kBox / 16;
          const uint32_t off = ((k / kPerPanel) * S::kPanelBytes + (k % kPerPanel) * 32) >> 4;
          umma_bf16(tmem + x * 128, desc_q + (x * S::kTileBytes >> 4) + off,
                    desc_k + (st * S::kTileBytes >> 4) + off, idesc_s, k != 0);
        }
        umma_commit(&bar.s_full[x]);
      }
      s_done[x]++;
    };
    auto values = [&](int x, int i) {  // O_x += P_x V_i
      const int st = i % S::kStages;
      ok = ok && warp_wait(&bar.p_full[x], o_done[x] & 1, abort_flag);
      if (!ok) return;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kKeys / 16; k++)
          umma_ta(tmem + S::kColO + x * S::kStrideO, tmem + S::kColP + x * S::kStrideP + k * 8,
                  desc_v + ((st * S::kTileBytes + k * 16 * S::kBox * 2) >> 4), idesc_o,
                  o_done[x] > 0 || k != 0);
        umma_commit(&bar.o_full[x]);
      }
      o_done[x]++;
    };
    auto wait_ring = [&](uint64_t *full, int i) {
      ok = ok && warp_wait(&full[i % S::kStages], (i / S::kStages) & 1, abort_flag);
    };
    // (nobody waits for the last ones)
    auto release = [&](uint64_t *empty, int i) {
      if (ok && i + S::kStages < n && elect_one()) umma_commit(&empty[i % S::kStages]);
    };
    if (n > 0) {
      wait_ring(bar.k_full, 0);
      for (int x = 0; x < 2; x++)
        if (active(x, 0)) scores(x, 0);
      release(bar.k_empty, 0);
    }
    for (int i = 0; i < n && ok; i++) {
      const bool more = i + 1 < n;
      if (S::kApart) {
        if (more) {
          wait_ring(bar.k_full, i + 1);
          for (int x = 0; x < 2; x++)
            if (active(x, i + 1)) scores(x, i + 1);
          release(bar.k_empty, i + 1);
        }
        wait_ring(bar.v_full, i);
        for (int x = 0; x < 2; x++)
          if (active(x, i)) values(x, i);
        release(bar.v_empty, i);
      } else {
        wait_ring(bar.v_full, i);
        if (more) wait_ring(bar.k_full, i + 1);
        for (int x = 0; x < 2; x++) {
          if (active(x, i)) values(x, i);
          if (more && active(x, i + 1)) scores(x, i + 1);
        }
        release(bar.v_empty, i);
        if (more) release(bar.k_empty, i + 1);
      }
    }
    if (!ok) {
      set_status(a.status, kStatusWaitTimeoutMma);
      *abort_flag = 1;
    }
  } else if (job.seq >= 0) {
    // ---------------------------------------------------------------- softmax
    const int x = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int rows = job.tokens[x] * group;
    const bool warp_live = quarter * 32 < rows;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t col_s = tmem + lanes + x * 128;
    const uint32_t col_p = tmem + lanes + S::kColP + x * S::kStrideP;
    const uint32_t col_o = tmem + lanes + S::kColO + x * S::kStrideO;
    const float c = a.scale * 1.4426950408889634f;
    // keys [first, last] relative to block 0, of this row and of the warp's rows together
    auto last_of = [&](int r) { return job.first_pos + x * tok + r / group; };
    const int last = last_of(row);
    const long long first_ll = a.window > 0 ? static_cast<long long>(last) - a.window + 1 : 0;
    const int first = static_cast<int>(max(first_ll, -1ll));
    const int last_min = __shfl_sync(0xffffffffu, last, 0);
    const int first_max = __shfl_sync(0xffffffffu, first, 31);
    bool ok = true;
    const int count = job.end[x] - job.begin[x];
    for (int i = 0; i < count; i++) {
      const int key0 = (job.begin[x] + i) * kKeys;
      uint32_t s[4][32];
      ok = warp_wait(&bar.s_full[x], i & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      float base = 0.f;
      if (warp_live) {
#pragma unroll
        for (int q = 0; q < 4; q++) tmem_ld32(col_s + 32 * q, s[q]);
#pragma unroll
        for (int q = 0; q < 4; q++) tmem_ld_wait32(s[q]);
      }
      if (S::kApart) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.s_free[x]);
      }
      float scale_o = 1.f;
      if (warp_live) {
        if (key0 + kKeys - 1 > last_min || key0 < first_max) {
#pragma unroll
          for (int q = 0; q < 4; q++)
#pragma unroll
            for (int e = 0; e < 32; e++) {
              const int t = key0 + 32 * q + e;
              if (t > last || t < first) s[q][e] = 0xff800000u;
            }
        }
        float mx[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          mx[q] = __uint_as_float(s[q][0]);
#pragma unroll
          for (int e = 1; e < 32; e++) mx[q] = fmaxf(mx[q], __uint_as_float(s[q][e]));
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
        if (top > m + 8.f) {
          scale_o = fast_exp2(m - top);
          l *= scale_o;
          m = top;
        }
        base = m == -INFINITY ? 0.f : m;
      }
      // the product of the block before has read P and written O
      if (i > 0) {
        ok = warp_wait(&bar.o_full[x], (i - 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
      }
      if (warp_live) {
        if (i > 0 && __any_sync(0xffffffffu, scale_o != 1.f)) {
#pragma unroll
          for (int d = 0; d < D; d += 16) {
            uint32_t o[16];
            tmem_ld16(col_o + d, o);
            tmem_ld_wait16(o);
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale_o);
            tmem_st16(col_o + d, o);
          }
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 4; q++) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float p0 = fast_exp2(fmaf(__uint_as_float(s[q][2 * e]), c, -base));
            const float p1 = fast_exp2(fmaf(__uint_as_float(s[q][2 * e + 1]), c, -base));
            sum[0] += p0;
            sum[1] += p1;
            p[e] = pack16(p0, p1, static_cast<T *>(nullptr));
          }
          tmem_st16(col_p + 16 * q, p);
        }
        l += sum[0] + sum[1];
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.p_full[x]);
    }
    if (ok && count > 0) ok = warp_wait(&bar.o_full[x], (count - 1) & 1, abort_flag);
    if (!ok) {
      set_status(a.status, kStatusWaitTimeoutEpilogue);
      *abort_flag = 1;
    }
    tc_fence_after();
  }
  // every copy and product of the CTA has been waited for above (unless a wait ran out)
  __syncthreads();
  if (*abort_flag) {
    const uint64_t t0 = global_timer_ns();  // let what is in flight land
    while (global_timer_ns() - t0 < 2000000ull) {
    }
    __syncthreads();
  }
  tc_fence_after();
  const int x = warp >> 2, quarter = warp & 3;
  const int row = quarter * 32 + lane;
  const int rows = warp < 8 && job.seq >= 0 ? job.tokens[x] * group : 0;
  if (quarter * 32 < rows && (split > 1 || !*abort_flag)) {
    const int head = kvh * group + row % group;
    const bool any = job.end[x] > job.begin[x];
    float f = 1.f;
    if (split == 1) f = row_factor(m, l, a.sinks, head);
    T *out = static_cast<T *>(a.out) +
             static_cast<long long>(job.q_row0 + x * tok + row / group) * a.out_stride +
             static_cast<long long>(head) * D;
    const uint32_t col_o = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + S::kColO + x * S::kStrideO;
    part_m[x * 128 + row] = m;
    part_l[x * 128 + row] = l;
#pragma unroll
    for (int d = 0; d < D; d += 16) {
      uint32_t o[16];
#pragma unroll
      for (int e = 0; e < 16; e++) o[e] = 0u;
      if (any) {
        tmem_ld16(col_o + d, o);
        tmem_ld_wait16(o);
      }
      if (split > 1) {
        // 16-byte pieces of a row are permuted by the row, so that a warp's rows spread over
        // the banks
#pragma unroll
        for (int e = 0; e < 4; e++)
          *reinterpret_cast<uint4 *>(smem + part_offset<D>(x * 128 + row, d / 4 + e)) =
              make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      } else if (row < rows) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
          w[e] = f == 0.f ? 0u
                          : pack16(__uint_as_float(o[2 * e]) * f, __uint_as_float(o[2 * e + 1]) * f,
                                   static_cast<T *>(nullptr));
        *reinterpret_cast<uint4 *>(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4 *>(out + d + 8) = make_uint4(w[4], w[5], w[6], w[7]);
      }
      __syncwarp();
    }
  }
  if (split > 1) {
    tc_fence_before();
    cluster_barrier_all();
    // the CTAs of the cluster share the rows out among their threads, 8 elements a time
    const int pieces = job.seq >= 0 ? (job.tokens[0] + job.tokens[1]) * group * (D / 8) : 0;
    for (int i = rank * kAttnThreads + threadIdx.x; i < pieces; i += split * kAttnThreads) {
      const int r = i / (D / 8), piece = i % (D / 8);
      const int rows_a = job.tokens[0] * group;
      const int tile = r >= rows_a, rt = r - tile * rows_a;
      const int pr = tile * 128 + rt;
      const int head = kvh * group + rt % group;
      float mr[kAttnMaxSplit], all = -INFINITY;
      for (int k = 0; k < split; k++) {
        mr[k] = ld_cluster_f32(smem_u32(&part_m[pr]), k);
        all = fmaxf(all, mr[k]);
      }
      float sum = 0.f, acc[8];
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] = 0.f;
      for (int k = 0; k < split; k++) {
        if (mr[k] == -INFINITY) continue;  // that CTA saw no key of this row
        const float w = fast_exp2(mr[k] - all);
        sum += ld_cluster_f32(smem_u32(&part_l[pr]), k) * w;
        float v[8];
        ld_cluster_f32x4(smem_u32(smem + part_offset<D>(pr, 2 * piece)), k, v);
        ld_cluster_f32x4(smem_u32(smem + part_offset<D>(pr, 2 * piece + 1)), k, v + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] += v[e] * w;
      }
      const float f = row_factor(all, sum, a.sinks, head);
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; e++)
        w[e] = pack16(acc[2 * e] * f, acc[2 * e + 1] * f, static_cast<T *>(nullptr));
      T *out = static_cast<T *>(a.out) +
               static_cast<long long>(job.q_row0 + tile * tok + rt / group) * a.out_stride +
               static_cast<long long>(head) * D + 8 * piece;
      *reinterpret_cast<uint4 *>(out) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    cluster_barrier_all();  // nobody leaves while its shared memory is read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kAttnTmemCols);
  }
}

template <typename T, int D>
static int attention_launch(const gptoss_attention_args_t &a, int sms, cudaStream_t st) {
  typedef AttnShape<D> S;
  const int group = a.n_q_heads / a.n_kv_heads, tok = 128 / group;
  const long long slots = a.n_tokens / (2 * tok) + static_cast<long long>(a.n_seqs);
  CUtensorMap map_q, map_k, map_v;
  std::string err;
  const bool fp16 = !std::is_same<T, bf16>::value;
  // without a K / V row no block is ever loaded; the maps still need an address
  const void *k = a.n_kv_rows ? a.k : a.q, *v = a.n_kv_rows ? a.v : a.q;
  const uint64_t rows = a.n_kv_rows ? a.n_kv_rows : 1;
  int rc = make_tmap_rows(&map_q, a.q, fp16, D, a.n_q_heads, a.n_tokens, a.q_stride, S::kBox, group,
                          tok, &err);
  if (!rc) rc = make_tmap_rows(&map_k, k, fp16, D, a.n_kv_heads, rows, a.k_stride, S::kBox, 1, kKeys, &err);
  if (!rc) rc = make_tmap_rows(&map_v, v, fp16, D, a.n_kv_heads, rows, a.v_stride, S::kBox, 1, kKeys, &err);
  if (rc) return decode_error(rc, "prompt_attention: %s", err.c_str());
  // Split the keys of a pair of tiles over a cluster while that leaves every CTA an SM of its
  // own and at least two blocks.
  long long most = a.max_kv_len > 0 ? a.max_kv_len : INT32_MAX;
  if (a.window > 0) most = std::min(most, static_cast<long long>(a.window) + 2 * tok);
  const long long blocks = (most + kKeys - 1) / kKeys;
  int split = 1;
  while (split < kAttnMaxSplit && slots * a.n_kv_heads * split * 2 <= sms && blocks >= 4 * split) split *= 2;
  const long long grid = slots * a.n_kv_heads * split;
  if (grid > INT32_MAX) return decode_error(GPTOSS_E_CAPACITY, "prompt_attention: too many rows for one launch");
  auto kernel = prompt_attention_kernel<T, D>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kAttnThreads);
    cfg.dynamicSmemBytes = S::kSmemBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kernel, map_q, map_k, map_v, a, group, tok, static_cast<int>(slots), split);
  }
  return launch_result("prompt_attention", e);
}

template <typename T>
static int attention_for(const gptoss_attention_args_t &a, int sms, cudaStream_t st) {
  if (a.head_dim == 32) return attention_launch<T, 32>(a, sms, st);
  if (a.head_dim == 64) return attention_launch<T, 64>(a, sms, st);
  return attention_launch<T, 128>(a, sms, st);
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
  // row coordinates of the copies, a block past the last row included, are 32-bit
  if (a.n_kv_rows > INT32_MAX - 2 * kKeys)
    return decode_error(GPTOSS_E_CAPACITY, "prompt_attention: more than 2^31 - 257 K / V rows");
  if (a.n_tokens == 0 || a.n_seqs == 0) return GPTOSS_OK;
  if (!a.q || !a.out || !a.q_start || !a.kv_start || !a.kv_len || (a.n_kv_rows > 0 && (!a.k || !a.v)))
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: null buffer");
  if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16))
    return decode_error(GPTOSS_E_INVALID, "prompt_attention: q, k, v and out must be 16-byte aligned");
  OnDeviceOf dev(a.out, "prompt_attention: out");
  if (dev.code) return dev.code;
  const int sms = sm_count(dev.device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a.dtype == GPTOSS_DTYPE_BF16 ? attention_for<bf16>(a, sms, st)
                                      : attention_for<__half>(a, sms, st);
}
