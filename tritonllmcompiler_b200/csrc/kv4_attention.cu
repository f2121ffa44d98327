// Attention of new tokens over the 4-bit paged cache (kv4.cuh has the layout).
//
// Packed queries q [T, Hq, D]; sequence b owns rows cu[b] .. cu[b + 1], its n_b new tokens, already
// in the cache; token s of it sits at position len_b - n_b + s and, with causal, sees the keys up to
// its own. o = sum_t p_t v_t / sum_t p_t, p_t = 2^((q . k_t) scale log2(e) - m), k and v the values
// the cache stands for.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "kv4.cuh"
#include "ptx.cuh"

namespace tllm {

__device__ int g_kv4a_status = 0;

int kv4a_read_status(int *out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_kv4a_status, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyFromSymbol(kv4 attention status)");
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_kv4a_status, &zero, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyToSymbol(kv4 attention status)");
  *out = v;
  return TLLM_OK;
}

namespace kv4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 128;

struct Args {
  const void *q;
  const uint8_t *cache;
  const int32_t *block_tables, *lens, *cu;
  void *o;
  int64_t sq0, sq1, so0, so1, sblk, shead, sbt0, sbt1;
  int64_t T, num_blocks, max_blocks;
  int B, Hq, Hkv, G, log2_bs, causal;
  float scale_log2;
};

// One warp per query row; a lane holds D / 32 consecutive channels.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_attn_simple_kernel(const Args a) {
  using P = Piece<D>;
  constexpr int E = D / 32;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= a.T * a.Hq) return;
  const int lane = threadIdx.x & 31;
  const int64_t t = row / a.Hq;
  const int h = static_cast<int>(row % a.Hq), hk = h / a.G;
  T *o = static_cast<T *>(a.o) + t * a.so0 + h * a.so1 + lane * E;
  if (t < a.cu[0] || t >= a.cu[a.B]) {
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = from_f32<T>(0.f);
    return;
  }
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= t) lo = mid; else hi = mid;
  }
  const int64_t cap = a.max_blocks << a.log2_bs;
  const int64_t len = min(static_cast<int64_t>(max(a.lens[lo], 0)), cap);
  const int64_t pos = len - (a.cu[lo + 1] - a.cu[lo]) + (t - a.cu[lo]);
  const int64_t keys = a.causal ? min(pos + 1, len) : len;
  const T *q = static_cast<const T *>(a.q) + t * a.sq0 + h * a.sq1 + lane * E;
  float qf[E], acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qf[i] = to_f32<T>(q[i]);
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < keys; ++j) {
    int block = a.block_tables[lo * a.sbt0 + (j >> a.log2_bs) * a.sbt1];
    if (block < 0 || block >= a.num_blocks) {
      atomicCAS(&g_kv4a_status, 0, TLLM_DEV_BAD_INDEX);
      block = 0;
    }
    const int in = static_cast<int>(j & ((1 << a.log2_bs) - 1));
    const uint8_t *p = a.cache + block * a.sblk + hk * a.shead + (in / kPieceTokens) * P::BYTES;
    const int tok = in % kPieceTokens;
    auto half = [&](int at) { return __half2float(*reinterpret_cast<const __half *>(p + at)); };
    float s = 0.f, v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int d = lane * E + i, g = d / 32;
      const uint32_t kw = *reinterpret_cast<const uint32_t *>(p + P::k_word(tok, d / 8));
      const uint32_t vw = *reinterpret_cast<const uint16_t *>(p + P::v_bits(tok, g, (d % 32) / 4));
      const float kc = static_cast<float>((kw >> (4 * ((d % 8) >> 1) + 16 * (d & 1))) & 15u);
      const float vc = static_cast<float>((vw >> (4 * (d & 3))) & 15u);
      s = fmaf(qf[i], fmaf(kc, half(P::k_scale(tok, g)), half(P::k_zero(tok, g))), s);
      v[i] = fmaf(vc, half(P::v_scale(tok, g)), half(P::v_zero(tok, g)));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= a.scale_log2;
    const float m2 = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : exp2f(m - m2);
    const float w = exp2f(s - (m2 == -INFINITY ? 0.f : m2));
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = fmaf(acc[i], keep, w * v[i]);
    m = m2;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = from_f32<T>(acc[i] / l);
}

template <typename T, int D>
int launch(const Args &a, cudaStream_t st) {
  const int64_t rows = a.T * a.Hq;
  const unsigned grid = static_cast<unsigned>((rows + kThreads / 32 - 1) / (kThreads / 32));
  kv4_attn_simple_kernel<T, D><<<grid, kThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError(), "paged kv4 attention launch");
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace kv4
}  // namespace tllm

extern "C" size_t tllm_paged_kv4_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                                                     int64_t max_new, int64_t D, int64_t block_size,
                                                     int64_t max_blocks) {
  (void)B; (void)T; (void)Hq; (void)Hkv; (void)max_new; (void)D; (void)block_size; (void)max_blocks;
  return 0;
}

extern "C" int tllm_paged_kv4_attn(const void *q, const void *cache, const int32_t *block_tables,
                                   const int32_t *context_lens, const int32_t *cu_seqlens, void *o,
                                   void *workspace, size_t workspace_bytes, int64_t B, int64_t T,
                                   int64_t Hq, int64_t Hkv, int64_t max_new, int64_t D,
                                   int64_t block_size, int64_t max_blocks, int64_t num_blocks,
                                   const int64_t *sq, const int64_t *sc, const int64_t *sbt,
                                   const int64_t *so, float sm_scale, int causal, int dtype,
                                   void *stream) {
  using namespace tllm;
  using namespace tllm::kv4;
  (void)workspace;
  (void)workspace_bytes;
  clear_error();
  TLLM_CHECK_ARG(dtype == TLLM_DTYPE_F16 || dtype == TLLM_DTYPE_BF16,
                 "paged_kv4_attn: unsupported dtype %d", dtype);
  TLLM_CHECK_ARG(B >= 0 && T >= 0 && Hq >= 0 && Hkv >= 0 && max_new >= 0 && max_blocks >= 0 && num_blocks >= 0,
                 "paged_kv4_attn: negative dimension");
  TLLM_CHECK_ARG(D == 64 || D == 128, "paged_kv4_attn: head dim %lld not in {64,128}", (long long)D);
  TLLM_CHECK_ARG(block_size == 16 || block_size == 32 || block_size == 64,
                 "paged_kv4_attn: block_size %lld not in {16,32,64}", (long long)block_size);
  TLLM_CHECK_ARG(sq && sc && sbt && so, "paged_kv4_attn: null stride array");
  if (T == 0 || Hq == 0) return TLLM_OK;
  TLLM_CHECK_ARG(Hkv >= 1 && Hq % Hkv == 0, "paged_kv4_attn: %lld query heads do not group over %lld KV heads",
                 (long long)Hq, (long long)Hkv);
  TLLM_CHECK_ARG(q && o && cu_seqlens && (B == 0 || context_lens), "paged_kv4_attn: null tensor pointer");
  TLLM_CHECK_ARG(B == 0 || max_blocks == 0 || (block_tables && cache && num_blocks >= 1),
                 "paged_kv4_attn: null block table or empty cache");
  TLLM_CHECK_ARG(max_blocks * block_size < (1LL << 30) && num_blocks < (1LL << 31) && B < (1LL << 24) &&
                     Hq < (1LL << 20) && T < (1LL << 31) && T * Hq < (1LL << 31),
                 "paged_kv4_attn: problem too large");
  for (int i = 0; i < 2; ++i)
    TLLM_CHECK_ARG(sq[i] % 8 == 0 && so[i] % 8 == 0, "paged_kv4_attn: q/o strides must be multiples of 8 elements");
  TLLM_CHECK_ARG(sc[0] % 16 == 0 && sc[1] % 16 == 0, "paged_kv4_attn: cache strides must be multiples of 16 bytes");
  TLLM_CHECK_ARG(aligned16(q) && aligned16(o) && aligned16(cache), "paged_kv4_attn: tensors must be 16-byte aligned");
  Args a{};
  a.q = q;
  a.cache = static_cast<const uint8_t *>(cache);
  a.block_tables = block_tables;
  a.lens = context_lens;
  a.cu = cu_seqlens;
  a.o = o;
  a.sq0 = sq[0];
  a.sq1 = sq[1];
  a.so0 = so[0];
  a.so1 = so[1];
  a.sblk = sc[0];
  a.shead = sc[1];
  a.sbt0 = sbt[0];
  a.sbt1 = sbt[1];
  a.T = T;
  a.num_blocks = num_blocks;
  a.max_blocks = max_blocks;
  a.B = static_cast<int>(B);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.G = static_cast<int>(Hq / Hkv);
  a.log2_bs = block_size == 16 ? 4 : (block_size == 32 ? 5 : 6);
  a.causal = causal ? 1 : 0;
  a.scale_log2 = sm_scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TLLM_DTYPE_F16) return D == 64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
  return D == 64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
}
