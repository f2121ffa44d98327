// Block tables and slot maps of a paged cache, built on the GPU from the requests' lengths.
//
// With L_b tokens already in the cache and n_b new ones, sequence b has have_b = ceil(L_b / bs)
// blocks and takes need_b = ceil((L_b + n_b) / bs) - have_b more from the free list, in order of b:
// off_b = sum of need over the sequences before it (the list starts after the entries that earlier steps
// took, a count that stays on the GPU too). Packed token i of sequence b is new token
// t = i - cu[b] at position p = L_b + t, in block j = p / bs: the table's entry where j < have_b,
// else free[off_b + j - have_b]; its slot is block * bs + p % bs. The thread of a block's first
// token (p % bs == 0) writes the table entry, so every entry has one writer and no thread reads
// an entry that this launch writes.
//
// Work: 8 bytes out per token and 16 per sequence; at one decode step nothing but latency, so
// everything is one launch: each CTA scans (n, need) over all B sequences itself (B values from
// L2, a few hundred ns) instead of a second launch or a grid-wide wait, then finds its tokens'
// sequences by bisection of the scan in shared memory. 64 decode steps take 3.2 us of the
// GPU (calls in a graph), 509 sequences with 64 K new tokens 11.6.
#include "common.h"

namespace tllm {
namespace plan {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTokensPerCta = 2048;
constexpr int64_t kMaxSeqs = 16384;  // the scans of all sequences fit in shared memory

struct Args {
  int32_t *block_tables;
  const int32_t *seq_lens, *n_new, *free_blocks;
  const int32_t *free_start;  // [1]: entries of free_blocks that earlier steps took; null: none
  int32_t *slots, *positions, *cu, *new_lens, *taken;
  int B, n_free, max_tokens, block_size;
  int64_t max_blocks, sbt0, sbt1;
};

struct Seq {
  int64_t len, n, have, need;
  bool fits;
};

__device__ __forceinline__ Seq sequence(const Args &a, int b) {
  Seq s;
  s.len = max(__ldg(a.seq_lens + b), 0);
  s.n = max(__ldg(a.n_new + b), 0);
  s.have = (s.len + a.block_size - 1) / a.block_size;
  const int64_t want = (s.len + s.n + a.block_size - 1) / a.block_size;
  s.fits = want <= a.max_blocks;
  s.need = s.fits ? want - s.have : 0;
  return s;
}

__device__ __forceinline__ int32_t sat32(int64_t v) {
  return static_cast<int32_t>(v < 0x7fffffff ? v : 0x7fffffff);
}

// Inclusive scan over the warp.
__device__ __forceinline__ int64_t warp_scan(int64_t v, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += u;
  }
  return v;
}

__global__ void __launch_bounds__(kThreads) paged_plan_kernel(const Args a) {
  extern __shared__ int32_t s_cu[];  // [B + 1] new tokens before each sequence, then
  int32_t *s_off = s_cu + a.B + 1;   // [B] blocks taken before each sequence, or -1: refused
  __shared__ int64_t s_tok[kWarps], s_blk[kWarps];
  __shared__ int s_taken;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool first = blockIdx.x == 0;  // this CTA also writes the per-sequence results
  const int start = a.free_start ? min(max(__ldg(a.free_start), 0), a.n_free) : 0;
  const int32_t *free_blocks = a.free_blocks + start;
  const int n_free = a.n_free - start;

  // Each thread scans a run of consecutive sequences.
  const int per = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  int64_t tok = 0, blk = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = sequence(a, b);
    tok += s.n;
    blk += s.need;
  }
  const int64_t tok_in = warp_scan(tok, lane), blk_in = warp_scan(blk, lane);
  if (lane == 31) {
    s_tok[warp] = tok_in;
    s_blk[warp] = blk_in;
  }
  if (tid == 0) s_taken = 0;
  __syncthreads();
  int64_t tok_at = tok_in - tok, blk_at = blk_in - blk;
  for (int w = 0; w < warp; ++w) {
    tok_at += s_tok[w];
    blk_at += s_blk[w];
  }
  int took = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = sequence(a, b);
    const bool ok = s.fits && (s.need == 0 || blk_at + s.need <= n_free) &&
                    tok_at + s.n <= a.max_tokens;
    s_cu[b] = sat32(tok_at);
    s_off[b] = ok ? sat32(blk_at) : -1;
    if (ok && s.need > 0) took = static_cast<int>(blk_at + s.need);
    if (first) {
      a.cu[b] = sat32(tok_at);
      a.new_lens[b] = sat32(ok ? s.len + s.n : s.len);
    }
    tok_at += s.n;
    blk_at += s.need;
  }
  if ((b1 == a.B && b0 < b1) || (a.B == 0 && tid == 0)) {
    s_cu[a.B] = sat32(tok_at);
    if (first) a.cu[a.B] = sat32(tok_at);
  }
  // Admitted sequences that take blocks come before every refused one that would, so the last
  // one's end is the number of blocks taken.
  if (first && took > 0) atomicMax(&s_taken, took);
  __syncthreads();
  if (first && tid == 0) *a.taken = s_taken;

  const int end = min(a.max_tokens, (static_cast<int>(blockIdx.x) + 1) * kTokensPerCta);
  for (int i = blockIdx.x * kTokensPerCta + tid; i < end; i += kThreads) {
    if (i >= s_cu[a.B]) {  // past the last new token
      a.slots[i] = -1;
      a.positions[i] = 0;
      continue;
    }
    int lo = 0, hi = a.B;  // s_cu[lo] <= i < s_cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cu[mid] <= i) lo = mid; else hi = mid;
    }
    const int64_t len = max(__ldg(a.seq_lens + lo), 0);
    const int64_t pos = len + (i - s_cu[lo]);
    a.positions[i] = sat32(pos);
    const int off = s_off[lo];
    if (off < 0) {
      a.slots[i] = -1;
      continue;
    }
    const int64_t j = pos / a.block_size;
    const int in = static_cast<int>(pos - j * a.block_size);
    const int64_t have = (len + a.block_size - 1) / a.block_size;
    int32_t *entry = a.block_tables + lo * a.sbt0 + j * a.sbt1;
    const int32_t block = j < have ? *entry : __ldg(free_blocks + off + (j - have));
    if (in == 0) *entry = block;
    a.slots[i] = block < 0 ? -1 : sat32(static_cast<int64_t>(block) * a.block_size + in);
  }
}

}  // namespace
}  // namespace plan
}  // namespace tllm

extern "C" int tllm_paged_plan(int32_t *block_tables, const int32_t *seq_lens,
                               const int32_t *n_new, const int32_t *free_blocks, int32_t *slots,
                               int32_t *positions, int32_t *cu_seqlens, int32_t *new_lens,
                               int32_t *taken, int64_t B, int64_t max_blocks, int64_t n_free,
                               int64_t max_tokens, int64_t block_size, const int64_t *sbt,
                               void *stream) {
  return tllm_paged_plan_from(block_tables, seq_lens, n_new, free_blocks, nullptr, slots, positions,
                              cu_seqlens, new_lens, taken, B, max_blocks, n_free, max_tokens,
                              block_size, sbt, stream);
}

extern "C" int tllm_paged_plan_from(int32_t *block_tables, const int32_t *seq_lens,
                                    const int32_t *n_new, const int32_t *free_blocks,
                                    const int32_t *free_start, int32_t *slots, int32_t *positions,
                                    int32_t *cu_seqlens, int32_t *new_lens, int32_t *taken,
                                    int64_t B, int64_t max_blocks, int64_t n_free,
                                    int64_t max_tokens, int64_t block_size, const int64_t *sbt,
                                    void *stream) {
  using namespace tllm;
  clear_error();
  TLLM_CHECK_ARG(B >= 0 && max_blocks >= 0 && n_free >= 0 && max_tokens >= 0,
                 "paged_plan: negative dimension");
  TLLM_CHECK_ARG(block_size >= 1 && block_size < (1LL << 20), "paged_plan: block_size %lld out of range",
                 (long long)block_size);
  TLLM_CHECK_ARG(B <= plan::kMaxSeqs, "paged_plan: %lld sequences, at most %lld in one call",
                 (long long)B, (long long)plan::kMaxSeqs);
  TLLM_CHECK_ARG(n_free < (1LL << 31) && max_tokens < (1LL << 31) - plan::kTokensPerCta &&
                     max_blocks < (1LL << 31),
                 "paged_plan: problem too large");
  TLLM_CHECK_ARG(sbt, "paged_plan: null stride array");
  TLLM_CHECK_ARG(cu_seqlens && taken, "paged_plan: null output pointer");
  TLLM_CHECK_ARG(max_tokens == 0 || (slots && positions), "paged_plan: null output pointer");
  TLLM_CHECK_ARG(B == 0 || (seq_lens && n_new && new_lens), "paged_plan: null sequence pointer");
  TLLM_CHECK_ARG(B == 0 || max_blocks == 0 || block_tables, "paged_plan: null block table");
  TLLM_CHECK_ARG(n_free == 0 || free_blocks, "paged_plan: null free list");
  plan::Args a{};
  a.block_tables = block_tables;
  a.seq_lens = seq_lens;
  a.n_new = n_new;
  a.free_blocks = free_blocks;
  a.free_start = free_start;
  a.slots = slots;
  a.positions = positions;
  a.cu = cu_seqlens;
  a.new_lens = new_lens;
  a.taken = taken;
  a.B = static_cast<int>(B);
  a.n_free = static_cast<int>(n_free);
  a.max_tokens = static_cast<int>(max_tokens);
  a.block_size = static_cast<int>(block_size);
  a.max_blocks = max_blocks;
  a.sbt0 = sbt[0];
  a.sbt1 = sbt[1];
  const int smem = static_cast<int>((2 * B + 1) * sizeof(int32_t));
  if (smem > 40 * 1024) {
    KernelLaunchInfo info;
    const int rc = prepare_kernel(reinterpret_cast<const void *>(plan::paged_plan_kernel),
                                  static_cast<int>((2 * plan::kMaxSeqs + 1) * sizeof(int32_t)),
                                  plan::kThreads, 1, &info);
    if (rc) return rc;
  }
  const unsigned grid =
      static_cast<unsigned>(max_tokens > 0 ? (max_tokens + plan::kTokensPerCta - 1) / plan::kTokensPerCta : 1);
  plan::paged_plan_kernel<<<grid, plan::kThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
  return cuda_status(cudaGetLastError(), "paged_plan launch");
}
