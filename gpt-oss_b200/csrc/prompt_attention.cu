// Attention of packed query rows over K / V rows: gptoss_decode_prompt_attention in
// include/gptoss_decode_b200.h.
//
//   o = sum_t p_t v_t / (sum_t p_t + 2^(sink' - m)),   p_t = 2^(c q.k_t - m),  c = scale log2 e
//
// A tile is 128 rows of one MMA: tok = 128 / group query tokens times the `group` query heads
// that share a KV head, so K and V are read once for the whole group and a sequence of a few
// tokens still fills rows.  A job is two tiles (consecutive tokens) of one sequence and KV head
// over the same stream of units of KEYS keys.  One CTA per SM:
//   warps 0-15   softmax, eight per tile: two warps share 32 rows, a thread has a row (a TMEM
//                lane) and half of a unit's keys
//   warp 16      the jobs (a CTA takes over the work of CTAs that have not started), TMA: Q of
//                both tiles, then K and V units into two rings
//   warps 17, 18 the MMAs of either tile, S = Q K^T a unit ahead of O += P V
// S comes from TMEM into registers whole, so the row maximum costs no second read, and S is
// free for the next unit's scores while P is being made; P goes back to TMEM as the MMA's
// 16-bit row operand, V is read in place as an N-major operand.  The maximum that scales a row
// is only moved when it grows by more than 8 (a factor of 256; fp32 sums and 16-bit
// floating-point P lose nothing by that), so O is rarely rescaled, and by its own softmax warps.
//
// What bounds it: an exponential per (row, key), 16 per cycle and SM.  64 keys of both tiles
// are 1024 cycles of exponentials against 256 of MMAs at head_dim 64 and 512 at 128; masking,
// maximum, scaling, sum and packing are issued beside them.  No pipe is full: one prompt of 8192
// tokens, 64/8 heads of 64, takes 690 to 725 us call after call, under the power limit (650 in a
// burst), which is 69 to 66 % (73) of the exponentials' rate; in a prompt of 4096 tokens the
// tensor pipe is at 36 % and the issue slots are at 61 %.  With units of 128 keys three of 16
// pairs of exponentials are computed on the FMA pipes.  That share is what measured best in this
// schedule: none takes 700 us (688 in a burst), four of 16 706 (666).  With units of 64 keys it
// gains nothing (one prompt of 4096 tokens, 32/4 heads of 128: 139 us, 0.99 PFLOP/s; 142 with two
// of 16).
//
// KEYS: 128 where TMEM holds S, P and O of both tiles (head_dim <= 64), 64 at 128.  A narrow
// window leaves most of a unit of 128 masked, so 64 are taken there too.  Time with 64 and 128
// keys of 10 packed prompts (13626 tokens), 64/8 heads of 64, by window: 32 tokens 112 and 119
// us, 128 127 and 147, 256 162 and 172, 512 222 and 220, 1024 321 and 309, 2048 460 and 436.
//
// Few tiles and long contexts: a cluster of up to 8 CTAs shares one pair of tiles, each taking
// an equal run of units; the partial (m, l, O) are joined through distributed shared memory, in
// rank order, so the result does not depend on timing and no workspace is needed.  Only as far
// as SMs would be idle otherwise: a cluster waits until that many SMs are free at once, and
// four packed pieces of prompts (3690 tokens, 32/4 heads of 128, contexts up to 16130) took 264
// us with whole jobs, 309 with every job in two parts and 471 in four.
//
// Jobs start in the order of their slots, the last one first.  Within a sequence that is the
// longest first, across sequences it is not: those four pieces take 259 us, and 336 with the one
// on 16130 keys at the front of the batch, which then starts last.
//
// Probabilities are rounded to the 16-bit type for the second product (tensor cores take both
// operands in one type); their sum is taken in fp32 before that rounding.
#include <cuda.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "attention_rows.cuh"

namespace gptoss {

constexpr int kAttnThreads = 640;
// Registers of a thread at launch: the bound on the threads leaves 65536 / 640, in steps of 8, and
// a kernel that moves registers between its warps is given all of them.  Those warps' shares.
constexpr int kAttnRegs = 65536 / kAttnThreads / 8 * 8;
constexpr int kAttnRegsSoftmax = 104, kAttnRegsOther = 64;
constexpr int kAttnSoftmaxWarps = 16;
static_assert(32 * kAttnSoftmaxWarps * kAttnRegsSoftmax + (kAttnThreads - 32 * kAttnSoftmaxWarps) * kAttnRegsOther <=
                  kAttnThreads * kAttnRegs,
              "the warps would wait for ever for registers that the launch did not bring");
constexpr int kAttnTmemCols = 512;
constexpr int kAttnMaxSplit = 8;      // CTAs of a cluster that share a pair of tiles
constexpr int kAttnNarrow = 512;      // widest window that takes units of 64 keys at head_dim <= 64
constexpr int kJobs = 4;              // jobs that may be at work in different warps

template <int D, int KEYS>
struct AttnShape {
  static constexpr int kBox = D < 64 ? D : 64;            // elements of one swizzled row
  static constexpr int kPanels = D / kBox;                // 64-wide panels of a head
  static constexpr int kQPanelBytes = 128 * kBox * 2;
  static constexpr int kPanelBytes = KEYS * kBox * 2;     // a panel of K or V
  static constexpr int kQBytes = kPanels * kQPanelBytes;
  static constexpr int kUnitBytes = kPanels * kPanelBytes;
  static constexpr int kStages = 4;                       // units of K and of V in flight
  static constexpr int kRingBytes = kStages * kUnitBytes;
  // TMEM columns: S of both tiles (KEYS each), P of both (KEYS / 2), O of both (D)
  static constexpr int kColP = 2 * KEYS;
  static constexpr int kColO = D == 128 ? 256 : 384;
  static_assert(3 * KEYS <= kColO && kColO + 2 * D <= kAttnTmemCols, "TMEM");
  // every kPolyStep-th of 16 pairs of exponentials is computed on the FMA pipes (17: none)
  static constexpr int kPolyStep = KEYS == 64 ? 17 : 5;
  static constexpr int kOperandBytes = 2 * kQBytes + 2 * kRingBytes;
  // fp32 partial outputs of both tiles take the operands' place in a split launch
  static constexpr int kSmemBytes = 1024 + (kOperandBytes > 256 * D * 4 ? kOperandBytes : 256 * D * 4);
};

struct AttnBarriers {
  uint64_t job_full[kJobs], job_empty[kJobs], steal;
  uint64_t q_full[2], q_empty[2], s_full[2], s_free[2], p_full[2], o_full[2], v_tail;
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
};

// The rows and keys of one job.
struct AttnJob {
  int kvh;                // KV head; -1: there are no more jobs
  int q_row0;             // first query row of the pair of tiles
  int tokens[2];          // valid tokens of the tiles
  int kv_row0;            // first key of unit 0 (row of k)
  int first_pos;          // position of the first query token, relative to unit 0's first key
  int keys;               // keys from unit 0's first to the last that the pair sees
  int begin[2], end[2];   // units of each tile, within this CTA's share
  int unit0, unit1;       // units of this CTA
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// two fp32 lanes in one instruction
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float2 f32x2_parts(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 2^x of two values in [-125, 127] on the FMA pipes: x = n + f with n the nearest integer (the
// addition of 1.5 * 2^23 rounds to it and leaves it in the low bits), 2^f by the polynomial of
// least relative error on [-1/2, 1/2] (Remez exchange; degree 3: 7.5e-5, degree 4: 2.6e-6),
// n added to the exponent.  Smaller x give 2^-125.
template <int kDegree>
__device__ __forceinline__ float2 poly_exp2(float2 x) {
  const uint64_t v = f32x2(fmaxf(x.x, -125.f), fmaxf(x.y, -125.f));
  const uint64_t magic = f32x2(12582912.f, 12582912.f), minus = f32x2(-1.f, -1.f);
  const uint64_t t = f32x2_add(v, magic);
  const uint64_t n = f32x2_add(t, f32x2(-12582912.f, -12582912.f));
  const uint64_t f = f32x2_fma(n, minus, v);
  uint64_t p;
  if (kDegree == 3) {
    p = f32x2_fma(f, f32x2(0.0551716685f, 0.0551716685f), f32x2(0.2426111251f, 0.2426111251f));
    p = f32x2_fma(p, f, f32x2(0.6932609677f, 0.6932609677f));
    p = f32x2_fma(p, f, f32x2(0.9999280572f, 0.9999280572f));
  } else {
    p = f32x2_fma(f, f32x2(0.0095701022f, 0.0095701022f), f32x2(0.0559178591f, 0.0559178591f));
    p = f32x2_fma(p, f, f32x2(0.2402474433f, 0.2402474433f));
    p = f32x2_fma(p, f, f32x2(0.6931217909f, 0.6931217909f));
    p = f32x2_fma(p, f, f32x2(0.9999992847f, 0.9999992847f));
  }
  const float2 r = f32x2_parts(p), m = f32x2_parts(t);
  return make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(m.x) << 23)),
                     __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(m.y) << 23)));
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

// A wait whose outcome the whole warp shares (what follows is issued by the converged warp).
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
}

// Shared-memory descriptors of operands that TMA wrote with rows of kBox elements and the
// matching swizzle: groups of 8 rows are 8 * row bytes apart.  For an operand read along its
// rows (K major) the leading offset is unused; for one read across them (V: N major) it is the
// distance of the 64-wide panels.
template <int D, int KEYS>
__device__ __forceinline__ uint64_t attn_desc(uint32_t addr) {
  typedef AttnShape<D, KEYS> S;
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

// Byte offset of 16-byte piece `piece` of fp32 row `row` among the partial outputs.
template <int D>
__device__ __forceinline__ uint32_t part_offset(int row, int piece) {
  return static_cast<uint32_t>((row * (D / 4) + (piece ^ (row & 7))) * 16);
}
// The job of a slot (a pair of tiles) and KV head, for this CTA's share of the keys.
template <int KEYS>
__device__ bool attn_find_job(const gptoss_attention_args_t &a, int tok, int slot, int kvh, int rank,
                              int split, int lane, AttnJob *job) {
  AttnRows r;
  if (!attn_find_rows(a, 2 * tok, slot, kvh, lane, &r)) return false;
  if (lane != 0) return true;
  const int units = (r.keys + KEYS - 1) / KEYS;
  job->kvh = kvh;
  job->q_row0 = r.q_row0;
  job->kv_row0 = static_cast<int>(r.kv_row0);
  job->first_pos = r.first_pos;
  job->keys = r.keys;
  job->unit0 = static_cast<int>(static_cast<long long>(units) * rank / split);
  job->unit1 = static_cast<int>(static_cast<long long>(units) * (rank + 1) / split);
  for (int x = 0; x < 2; x++) {
    const int n = min(max(r.tokens - x * tok, 0), tok);
    job->tokens[x] = n;
    job->begin[x] = job->end[x] = job->unit0;
    if (n == 0) continue;
    // relative to unit 0's first key: the tile's first token, the first key it sees
    const long long p = static_cast<long long>(r.first_pos) + x * tok;
    const long long from = a.window > 0 ? max(0ll, p - a.window + 1) : 0;
    const long long to = p + n;  // may be <= 0
    const int b = static_cast<int>(from / KEYS);
    const int e = to > 0 ? static_cast<int>((to + KEYS - 1) / KEYS) : 0;
    job->begin[x] = max(b, job->unit0);
    job->end[x] = max(job->begin[x], min(e, job->unit1));
  }
  return true;
}

// Asks for a CTA of this grid that has not started; the 16-byte answer says which one was
// taken out of the launch, or that there is none left (nothing may be asked after that).
__device__ __forceinline__ void steal_pair(void *answer, uint64_t *bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
      :
      : "r"(smem_u32(answer)), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool stolen_pair(const void *answer, uint32_t *pair) {
  uint32_t got, x;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t"
      "}"
      : "=r"(got), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  if (got) *pair = x;
  return got != 0;
}

// Position in a ring of N slots.
template <int N>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

template <typename T, int D, int KEYS>
__global__ void __launch_bounds__(kAttnThreads, 1)
prompt_attention_kernel(const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const gptoss_attention_args_t a,
                        int group, int tok, int n_slots, int split) {
  typedef AttnShape<D, KEYS> S;
  constexpr bool kHalf = !std::is_same<T, bf16>::value;
  extern __shared__ unsigned char smem_raw[];
  __shared__ AttnBarriers bar;
  __shared__ AttnJob jobs[kJobs];
  __shared__ __align__(16) unsigned char steal_answer[16];
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_word;
  __shared__ float exchange[2][2][2][128];  // [parity][tile][half of the columns][row]
  __shared__ float part_m[256], part_l[256];
  unsigned char *smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  unsigned char *sm_q = smem, *sm_k = smem + 2 * S::kQBytes, *sm_v = sm_k + S::kRingBytes;
  volatile int *abort_flag = &abort_word;
  // (through a shuffle, so that the compiler knows what the warp shares)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = split > 1 ? static_cast<int>(cluster_cta_rank()) : 0;

  if (warp == 17) {
    tmem_alloc(&tmem_holder, kAttnTmemCols);
    tmem_relinquish();
  } else if (warp == 16) {
    if (elect_one()) {
      tma_prefetch_desc(&map_q);
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
  } else if (threadIdx.x == 0) {
    for (int j = 0; j < kJobs; j++) {
      mbar_init(&bar.job_full[j], 1);
      mbar_init(&bar.job_empty[j], kAttnSoftmaxWarps + 2);
    }
    mbar_init(&bar.steal, 1);
    mbar_init(&bar.v_tail, 1);
    for (int x = 0; x < 2; x++) {
      mbar_init(&bar.q_full[x], 1);
      mbar_init(&bar.q_empty[x], 1);
      mbar_init(&bar.s_full[x], 1);
      mbar_init(&bar.s_free[x], kAttnSoftmaxWarps / 2);
      mbar_init(&bar.p_full[x], kAttnSoftmaxWarps / 2);
      mbar_init(&bar.o_full[x], 1);
    }
    for (int s = 0; s < S::kStages; s++) {
      mbar_init(&bar.k_full[s], 1);
      mbar_init(&bar.k_empty[s], 2);
      mbar_init(&bar.v_full[s], 1);
      mbar_init(&bar.v_empty[s], 2);
    }
    abort_word = 0;
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_holder, 0);

  float m = -INFINITY, l = 0.f;  // a softmax thread's row
  int part_rows = 0;             // split launch: rows of this thread's tile, whether it had keys
  bool part_any = false;
  bool ok = true;
  int code = kStatusOk;
  Ring<kJobs> jr;
  // whether there is a job in jobs[jr.slot] (false too when a wait ran out: ok is false then)
  auto have_job = [&]() {
    ok = ok && warp_wait(&bar.job_full[jr.slot], jr.phase, abort_flag);
    return ok && jobs[jr.slot].kvh >= 0;
  };
  auto done_job = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar.job_empty[jr.slot]);
    jr.next();
  };

  // Registers: 640 threads were launched with 96 each (61440); the four warps that hold no
  // tiles keep 64 and the sixteen that do take 104 (128 * 64 + 512 * 104 = 61440).
  if (warp >= kAttnSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAttnRegsOther));
    if (warp == 16) {
      // -------------------------------------------------------------- jobs and loads
      // The grid has a CTA (with a split: a cluster) per pair of tiles; this CTA does its own
      // and then, one at a time, those of CTAs that have not started, in their order.  It asks
      // for the next one only when the last loads of this one are due, so that a long job does
      // not keep another waiting.
      code = kStatusWaitTimeoutProducer;
      uint32_t pair = blockIdx.x / split, steal_phase = 0, q_phase[2] = {1u, 1u}, tail_phase = 0;
      Ring<S::kStages> ring;
      bool have = true, asked = false;
      auto ask = [&]() {
        if (asked || split > 1) return;
        asked = true;
        if (elect_one()) steal_pair(steal_answer, &bar.steal);
        __syncwarp();
      };
      auto answer = [&]() {
        have = false;
        if (!asked) return;
        asked = false;
        ok = ok && warp_wait(&bar.steal, steal_phase, abort_flag);
        steal_phase ^= 1u;
        have = ok && stolen_pair(steal_answer, &pair);
        __syncwarp();
      };
      while (ok) {
        ok = warp_wait(&bar.job_empty[jr.slot], jr.phase ^ 1u, abort_flag);
        AttnJob &job = jobs[jr.slot];
        bool found = false;
        while (ok && have && !found) {
          // the last slots first: a long prompt's last tiles see the most keys
          const uint32_t up = pair / a.n_kv_heads;
          found = attn_find_job<KEYS>(a, tok, n_slots - 1 - static_cast<int>(up),
                                static_cast<int>(pair - up * a.n_kv_heads), rank, split, lane, &job);
          if (!found) {
            ask();
            answer();
          }
        }
        if (!ok) break;
        if (!found && lane == 0) job.kvh = -1;  // the end
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.job_full[jr.slot]);
        if (!found) break;
        jr.next();
        auto load_q = [&](int x) {
          if (job.begin[x] >= job.end[x]) return;
          ok = ok && warp_wait(&bar.q_empty[x], q_phase[x], abort_flag);
          q_phase[x] ^= 1u;
          if (ok && elect_one()) {
            mbar_arrive_expect_tx(&bar.q_full[x], static_cast<uint32_t>(S::kPanels) * tok * group * S::kBox * 2);
            for (int p = 0; p < S::kPanels; p++)
              tma_load_3d(sm_q + x * S::kQBytes + p * S::kQPanelBytes, &map_q, &bar.q_full[x],
                          p * S::kBox, job.kvh * group, job.q_row0 + x * tok);
          }
          __syncwarp();
        };
        load_q(0);
        const int unit0 = job.unit0, unit1 = job.unit1;
        for (int u = unit0; ok && u < unit1; u++) {
          const int rel = u * KEYS;
          const bool tail = rel + KEYS > job.keys;
          unsigned char *k = sm_k + ring.slot * S::kUnitBytes, *v = sm_v + ring.slot * S::kUnitBytes;
          ok = warp_wait(&bar.k_empty[ring.slot], ring.phase ^ 1u, abort_flag);
          if (ok && elect_one()) {
            mbar_arrive_expect_tx(&bar.k_full[ring.slot], S::kUnitBytes);
            for (int p = 0; p < S::kPanels; p++)
              tma_load_3d(k + p * S::kPanelBytes, &map_k, &bar.k_full[ring.slot], p * S::kBox,
                          job.kvh, job.kv_row0 + rel);
          }
          __syncwarp();
          if (u == unit0) load_q(1);
          if (u + S::kStages >= unit1) ask();
          ok = ok && warp_wait(&bar.v_empty[ring.slot], ring.phase ^ 1u, abort_flag);
          // The last unit may reach past the last key: what lies there may be anything, and 0
          // times NaN is NaN, so those rows of V are cleared before the unit is handed on.
          uint64_t *landed = tail ? &bar.v_tail : &bar.v_full[ring.slot];
          if (ok && elect_one()) {
            mbar_arrive_expect_tx(landed, S::kUnitBytes);
            for (int p = 0; p < S::kPanels; p++)
              tma_load_3d(v + p * S::kPanelBytes, &map_v, landed, p * S::kBox, job.kvh, job.kv_row0 + rel);
          }
          __syncwarp();
          if (ok && tail) {
            ok = warp_wait(landed, tail_phase, abort_flag);
            tail_phase ^= 1u;
            constexpr int kRowChunks = S::kBox * 2 / 16;
            for (int p = 0; ok && p < S::kPanels; p++)
              for (int c = (job.keys - rel) * kRowChunks + lane; c < KEYS * kRowChunks; c += 32)
                *reinterpret_cast<uint4 *>(v + p * S::kPanelBytes + c * 16) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.v_full[ring.slot]);
          }
          ring.next();
        }
        ask();
        answer();
      }
    } else if (warp < 19) {
      // -------------------------------------------------------------- MMAs
      // A warp per tile issues; the tiles never wait for each other's softmax.
      code = kStatusWaitTimeoutMma;
      constexpr uint32_t idesc_s = attn_idesc(kHalf, KEYS, false);
      constexpr uint32_t idesc_o = attn_idesc(kHalf, D, true);
      const uint64_t desc_q = attn_desc<D, KEYS>(smem_u32(sm_q));
      const uint64_t desc_k = attn_desc<D, KEYS>(smem_u32(sm_k));
      const uint64_t desc_v = attn_desc<D, KEYS>(smem_u32(sm_v));
      Ring<S::kStages> kr, vr;
      const int x = warp - 17;
      const uint64_t dq = desc_q + (x * S::kQBytes >> 4);
      uint32_t q_phase = 0, free_phase = 1, p_phase = 0;
      for (; have_job(); done_job()) {
        const AttnJob &job = jobs[jr.slot];
        const int begin = job.begin[x], end = job.end[x], unit0 = job.unit0, unit1 = job.unit1;
        auto scores = [&](int u) {  // S = Q K_u^T
          ok = ok && warp_wait(&bar.k_full[kr.slot], kr.phase, abort_flag);
          const bool active = u >= begin && u < end;
          if (active) {
            if (u == begin) {
              ok = ok && warp_wait(&bar.q_full[x], q_phase, abort_flag);
              q_phase ^= 1u;
            }
            // free once its readers have the last S in registers
            ok = ok && warp_wait(&bar.s_free[x], free_phase, abort_flag);
            free_phase ^= 1u;
            tc_fence_after();
          }
          if (ok && elect_one()) {
            if (active) {
              const uint64_t dk = desc_k + (kr.slot * S::kUnitBytes >> 4);
#pragma unroll
              for (int k = 0; k < D / 16; k++) {
                constexpr int kPerPanel = S::kBox / 16;
                umma_bf16(tmem + x * KEYS,
                          dq + (((k / kPerPanel) * S::kQPanelBytes + (k % kPerPanel) * 32) >> 4),
                          dk + (((k / kPerPanel) * S::kPanelBytes + (k % kPerPanel) * 32) >> 4),
                          idesc_s, k != 0);
              }
              umma_commit(&bar.s_full[x]);
              if (u == end - 1) umma_commit(&bar.q_empty[x]);
            }
            umma_commit(&bar.k_empty[kr.slot]);
          }
          __syncwarp();
          kr.next();
        };
        auto values = [&](int u) {  // O += P V_u
          ok = ok && warp_wait(&bar.v_full[vr.slot], vr.phase, abort_flag);
          const bool active = u >= begin && u < end;
          if (active) {
            ok = ok && warp_wait(&bar.p_full[x], p_phase, abort_flag);
            p_phase ^= 1u;
            tc_fence_after();
          }
          if (ok && elect_one()) {
            if (active) {
              const uint64_t dv = desc_v + (vr.slot * S::kUnitBytes >> 4);
#pragma unroll
              for (int k = 0; k < KEYS / 16; k++)
                umma_ta(tmem + S::kColO + x * D, tmem + S::kColP + x * (KEYS / 2) + k * 8,
                        dv + ((k * 16 * S::kBox * 2) >> 4), idesc_o, k != 0 ? 1u : (u > begin ? 1u : 0u));
            }
            umma_commit(&bar.v_empty[vr.slot]);
            // last: who has waited for it has waited for everything before it
            if (active) umma_commit(&bar.o_full[x]);
          }
          __syncwarp();
          vr.next();
        };
        for (int u = unit0; ok && u <= unit1; u++) {  // the scores a unit ahead of the values
          if (u < unit1) scores(u);
          if (u > unit0) values(u - 1);
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAttnRegsSoftmax));
    code = kStatusWaitTimeoutEpilogue;
    // two warps per 32 rows: a thread has a row and half of a unit's keys
    constexpr int kMine = KEYS / 2, kParts = kMine / 32;
    const int x = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int row_tok = row / group;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t col_s = tmem + lanes + x * KEYS + half * kMine;
    const uint32_t col_p = tmem + lanes + S::kColP + x * (KEYS / 2) + half * (kMine / 2);
    const uint32_t col_o = tmem + lanes + S::kColO + x * D + half * (D / 2);
    const float c = a.scale * kLog2e;
    uint32_t s_phase = 0, o_phase = 0, parity = 0;
    // Hands over a value of the thread's row and returns that of the thread with the row's other
    // keys.  The barrier has no limit of its own: a warp that gives up raises the abort flag,
    // which is looked at before every call, and arrives once in its partner's place.
    const int pair_barrier = 1 + x * 4 + quarter;
    auto both = [&](float mine) {
      exchange[parity][x][half][row] = mine;
      named_barrier_sync(pair_barrier, 64);
      const float other = exchange[parity][x][half ^ 1][row];
      parity ^= 1u;
      return other;
    };
    for (; have_job(); done_job()) {
      const AttnJob &job = jobs[jr.slot];
      const int rows = job.tokens[x] * group;
      const bool warp_live = quarter * 32 < rows;
      const int begin = job.begin[x], n = job.end[x] - begin;
      // keys [first, last] relative to unit 0, of this row and of the warp's rows together
      const int last = job.first_pos + x * tok + row_tok;
      const long long first_ll = a.window > 0 ? static_cast<long long>(last) - a.window + 1 : 0;
      const int first = static_cast<int>(max(first_ll, -1ll));
      const int last_min = __shfl_sync(0xffffffffu, last, 0);
      const int first_max = __shfl_sync(0xffffffffu, first, 31);
      // one bit per key, so that masking a key costs a bit test and a select
      auto seen_keys = [&](int q, int key0) {
        const int lo = first - key0 - 32 * q, hi = last - key0 - 32 * q;
        const uint32_t from = lo <= 0 ? 0xffffffffu : (lo > 31 ? 0u : 0xffffffffu << lo);
        const uint32_t upto = hi >= 31 ? 0xffffffffu : (hi < 0 ? 0u : (2u << hi) - 1u);
        return from & upto;
      };
      m = -INFINITY;
      l = 0.f;
      for (int i = 0; i < n; i++) {
        ok = warp_wait(&bar.s_full[x], s_phase, abort_flag) && !*abort_flag;
        s_phase ^= 1u;
        if (!ok) break;
        tc_fence_after();
        uint32_t s[kParts][32], p[kParts][16];
        if (warp_live) {
#pragma unroll
          for (int q = 0; q < kParts; q++) tmem_ld32(col_s + 32 * q, s[q]);
#pragma unroll
          for (int q = 0; q < kParts; q++) tmem_ld_wait32(s[q]);
        }
        float scale_o = 1.f;
        if (warp_live) {
          const int key0 = (begin + i) * KEYS + half * kMine;
          const bool masked = key0 + kMine - 1 > last_min || key0 < first_max;
          if (masked) {
#pragma unroll
            for (int q = 0; q < kParts; q++) {
              const uint32_t seen = seen_keys(q, key0);
#pragma unroll
              for (int e = 0; e < 32; e++)
                if (!(seen & (1u << e))) s[q][e] = 0xff800000u;
            }
          }
          float mx[2 * kParts];
#pragma unroll
          for (int q = 0; q < 2 * kParts; q++) {
            const uint32_t *v = &s[q >> 1][(q & 1) * 16];
            mx[q] = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
#pragma unroll
            for (int e = 2; e < 16; e += 2)
              mx[q] = max3(mx[q], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
          }
          float top = fmaxf(mx[0], mx[1]);
          if (kParts > 1) top = fmaxf(top, fmaxf(mx[2 * kParts - 2], mx[2 * kParts - 1]));
          top *= c;
          top = fmaxf(top, both(top));
          // (the barrier in `both` has seen every lane's S in registers)
          tc_fence_before();
          if (lane == 0) mbar_arrive(&bar.s_free[x]);
          if (top > m + 8.f) {
            scale_o = fast_exp2(m - top);
            l *= scale_o;
            m = top;
          }
          const float base = m == -INFINITY ? 0.f : m;
          const uint64_t c2 = f32x2(c, c), base2 = f32x2(-base, -base);
          uint64_t sum = 0;
#pragma unroll
          for (int q = 0; q < kParts; q++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
              float2 y = f32x2_parts(f32x2_fma(
                  f32x2(__uint_as_float(s[q][2 * e]), __uint_as_float(s[q][2 * e + 1])), c2, base2));
              if (e % S::kPolyStep == S::kPolyStep - 1)
                y = poly_exp2<kHalf ? 4 : 3>(y);
              else
                y = make_float2(fast_exp2(y.x), fast_exp2(y.y));
              sum = f32x2_add(sum, f32x2(y.x, y.y));
              p[q][e] = pack16(y.x, y.y, static_cast<T *>(nullptr));
            }
          if (!kHalf && masked) {  // poly_exp2's 2^-125 (0 in fp16) of masked keys
#pragma unroll
            for (int q = 0; q < kParts; q++) {
              const uint32_t seen = seen_keys(q, key0);
#pragma unroll
              for (int e = S::kPolyStep - 1; e < 16; e += S::kPolyStep)
                p[q][e] &= (seen & (1u << (2 * e)) ? 0xffffu : 0u) | (seen & (2u << (2 * e)) ? 0xffff0000u : 0u);
            }
          }
          const float2 sums = f32x2_parts(sum);
          l += sums.x + sums.y;
        }
        if (!warp_live && lane == 0) mbar_arrive(&bar.s_free[x]);
        if (i > 0) {  // the product of the unit before has read P and written O
          ok = warp_wait(&bar.o_full[x], o_phase, abort_flag);
          o_phase ^= 1u;
          if (!ok) break;
          tc_fence_after();
        }
        if (warp_live) {
          if (i > 0 && __any_sync(0xffffffffu, scale_o != 1.f)) {
#pragma unroll
            for (int d = 0; d < D / 2; d += 16) {
              uint32_t o[16];
              tmem_ld16(col_o + d, o);
              tmem_ld_wait16(o);
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale_o);
              tmem_st16(col_o + d, o);
            }
          }
#pragma unroll
          for (int q = 0; q < kParts; q++) tmem_st16(col_p + 16 * q, p[q]);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_full[x]);
      }
      const bool any = n > 0;
      if (ok && any) {
        ok = warp_wait(&bar.o_full[x], o_phase, abort_flag);
        o_phase ^= 1u;
        tc_fence_after();
      }
      if (warp_live) {
        ok = ok && !*abort_flag;
        if (ok) {
          l += both(l);
        } else {
          *abort_flag = 1;
          __threadfence_block();
          asm volatile("bar.arrive %0, 64;" ::"r"(pair_barrier) : "memory");
        }
      }
      if (split > 1) {
        part_rows = rows;
        part_any = any;
        continue;  // a split launch has one job per CTA; its parts are joined below
      }
      if (!ok || !warp_live) continue;
      const int head = job.kvh * group + row - row_tok * group;
      const float f = row_factor(m, l, a.sinks, head);
      T *out = static_cast<T *>(a.out) +
               static_cast<long long>(job.q_row0 + x * tok + row_tok) * a.out_stride +
               static_cast<long long>(head) * D + half * (D / 2);
#pragma unroll
      for (int d = 0; d < D / 2; d += 16) {
        uint32_t o[16];
#pragma unroll
        for (int e = 0; e < 16; e++) o[e] = 0u;
        if (any) {
          tmem_ld16(col_o + d, o);
          tmem_ld_wait16(o);
        }
        if (row < rows) {
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
      tc_fence_before();
    }
  }
  if (!ok) {
    set_status(a.status, code);
    *abort_flag = 1;
  }
  // every copy and product of the CTA has been waited for above (unless a wait ran out)
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const uint64_t t0 = global_timer_ns();  // let what is in flight land
    while (global_timer_ns() - t0 < 2000000ull) {
    }
    __syncthreads();
  }
  tc_fence_after();
  if (split > 1) {
    const int x = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    if (quarter * 32 < part_rows) {
      const uint32_t col_o = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + S::kColO + x * D + half * (D / 2);
      if (half == 0) {
        part_m[x * 128 + row] = m;
        part_l[x * 128 + row] = l;
      }
      if (part_any) {
#pragma unroll
        for (int d = 0; d < D / 2; d += 16) {
          uint32_t o[16];
          tmem_ld16(col_o + d, o);
          tmem_ld_wait16(o);
          // 16-byte pieces of a row are permuted by the row, so that a warp's rows spread
          // over the banks
#pragma unroll
          for (int e = 0; e < 4; e++)
            *reinterpret_cast<uint4 *>(smem + part_offset<D>(x * 128 + row, (half * (D / 2) + d) / 4 + e)) =
                make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
    }
    tc_fence_before();
    cluster_barrier_all();
    // the CTAs of the cluster share the rows out among their threads, 8 elements a time (the
    // job's rows are the same in all of them)
    const AttnJob &job = jobs[0];
    const int pieces = job.kvh >= 0 ? (job.tokens[0] + job.tokens[1]) * group * (D / 8) : 0;
    for (int i = rank * kAttnThreads + threadIdx.x; i < pieces; i += split * kAttnThreads) {
      const int r = i / (D / 8), piece = i % (D / 8);
      const int rows_a = job.tokens[0] * group;
      const int tile = r >= rows_a, rt = r - tile * rows_a;
      const int pr = tile * 128 + rt;
      const int head = job.kvh * group + rt % group;
      float mr[kAttnMaxSplit], all = -INFINITY;
#pragma unroll
      for (int k = 0; k < kAttnMaxSplit; k++) {
        mr[k] = k < split ? ld_cluster_f32(smem_u32(&part_m[pr]), k) : -INFINITY;
        all = fmaxf(all, mr[k]);
      }
      float sum = 0.f, acc[8];
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] = 0.f;
#pragma unroll
      for (int k = 0; k < kAttnMaxSplit; k++) {
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
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem, kAttnTmemCols);
  }
}

template <typename T, int D, int KEYS>
static int attention_launch(const gptoss_attention_args_t &a, int sms, cudaStream_t st) {
  typedef AttnShape<D, KEYS> S;
  const int group = a.n_q_heads / a.n_kv_heads, tok = 128 / group;
  const long long slots = a.n_tokens / (2 * tok) + static_cast<long long>(a.n_seqs);
  if (slots > INT32_MAX) return decode_error(GPTOSS_E_CAPACITY, "prompt_attention: too many rows and sequences");
  // Kernel attributes first: a host thread that has made no CUDA call yet has no context, these
  // give it the device's, and the encoding of the tensor maps fails without one.
  auto kernel = prompt_attention_kernel<T, D, KEYS>;
  // with fewer registers than its warps share out they would wait for more for ever
  cudaFuncAttributes fa = {};
  cudaError_t e = cudaFuncGetAttributes(&fa, kernel);
  if (e == cudaSuccess && fa.numRegs != kAttnRegs)
    return decode_error(GPTOSS_E_STATE, "prompt_attention: built with %d registers, not %d", fa.numRegs, kAttnRegs);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes);
  if (e != cudaSuccess) return launch_result("prompt_attention", e);
  CUtensorMap map_q, map_k, map_v;
  std::string err;
  const bool fp16 = !std::is_same<T, bf16>::value;
  // without a K / V row no block is ever loaded; the maps still need an address
  const void *k = a.n_kv_rows ? a.k : a.q, *v = a.n_kv_rows ? a.v : a.q;
  const uint64_t rows = a.n_kv_rows ? a.n_kv_rows : 1;
  int rc = make_tmap_rows(&map_q, a.q, fp16, D, a.n_q_heads, a.n_tokens, a.q_stride, S::kBox, group,
                          tok, &err);
  if (!rc) rc = make_tmap_rows(&map_k, k, fp16, D, a.n_kv_heads, rows, a.k_stride, S::kBox, 1, KEYS, &err);
  if (!rc) rc = make_tmap_rows(&map_v, v, fp16, D, a.n_kv_heads, rows, a.v_stride, S::kBox, 1, KEYS, &err);
  if (rc) return decode_error(rc, "prompt_attention: %s", err.c_str());
  // Split the keys of a pair of tiles over a cluster while that leaves every CTA an SM of its
  // own and at least 256 keys.
  long long most = a.max_kv_len > 0 ? a.max_kv_len : INT32_MAX;
  if (a.window > 0) most = std::min(most, static_cast<long long>(a.window) + 2 * tok);
  const long long blocks = (most + 127) / 128;
  int split = 1;
  while (split < kAttnMaxSplit && slots * a.n_kv_heads * split * 2 <= sms && blocks >= 4 * split) split *= 2;
  const long long units = slots * a.n_kv_heads;
  const long long grid = units * split;
  if (grid > INT32_MAX) return decode_error(GPTOSS_E_CAPACITY, "prompt_attention: too many rows for one launch");
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
  return launch_result("prompt_attention", e);
}

// Few query rows per sequence go to the kernel of token_attention.cu: when a sequence has on
// average at most the tokens that fill 16 rows, one job there.  (64/8 heads of 64: one token each
// of 64 sequences with up to 7747 keys 152 us here and 98 there, one of 131071 keys 143 and 59.
// With more tokens a sequence that kernel reads its K and V once for every 16 rows.)  The choice
// holds for the whole call, so one kind pays where a call mixes them: a prompt of 4000 tokens and
// 63 single tokens on 8000 keys take 440 us here, 1070 there and 363 as two calls; with 4000
// single tokens on 512 keys beside it 1350 here, 1980 there and 1200 as two calls.
static bool rows_are_few(const gptoss_attention_args_t &a) {
  const int group = a.n_q_heads / a.n_kv_heads;
  return group <= 16 && a.n_tokens <= static_cast<long long>(a.n_seqs) * (16 / group);
}

template <typename T>
static int attention_for(const gptoss_attention_args_t &a, int sms, cudaStream_t st) {
  if (a.head_dim == 128) return attention_launch<T, 128, 64>(a, sms, st);
  const bool narrow = a.window > 0 && a.window <= kAttnNarrow;
  if (a.head_dim == 32)
    return narrow ? attention_launch<T, 32, 64>(a, sms, st) : attention_launch<T, 32, 128>(a, sms, st);
  return narrow ? attention_launch<T, 64, 64>(a, sms, st) : attention_launch<T, 64, 128>(a, sms, st);
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
  // row coordinates of the copies, a unit past the last row included, are 32-bit
  if (a.n_kv_rows > INT32_MAX - 256)
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
  if (rows_are_few(a)) return launch_token_attention(a, sms, st);
  return a.dtype == GPTOSS_DTYPE_BF16 ? attention_for<bf16>(a, sms, st)
                                      : attention_for<__half>(a, sms, st);
}
