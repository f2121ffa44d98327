// Writing K/V rows into the 4-bit paged cache by slot, and reading rows back (kv4.cuh has the
// layout).
//
// A group of 32 channels x of one token and head becomes
//   s = fp16((max - min) * (1 / 15)), z = fp16(min), code = clamp(rint((x - z) * (s > 0 ? 1 / s : 0)), 0, 15),
// each step one IEEE fp32 operation (no contraction), so the codes do not depend on the compiler.
// s and z are fp16: 11 bits put the reconstruction within 1 / 2048 of the group's range of where
// exact ones would, a fraction of the half step of 1 / 30, for 4 bytes per 16 bytes of codes. A
// group with a NaN or an infinity, or beyond fp16's range, reads back as NaN or infinities.
//
// Bound: HBM, 2 bytes in and 0.625 out per element (the other way round when reading back). D / 8
// consecutive lanes hold a row of K and the same row of V, one 16-byte vector of each; minimum and
// maximum take two shuffles within the four lanes of a group. A lane's V codes belong to two
// chunks of the layout, so pairs of lanes exchange halves and each lane stores one whole word.
// No two lanes write the same byte, so tokens of one piece may be appended in any order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "kv4.cuh"
#include "ptx.cuh"
#include "rmsnorm_rope.cuh"

namespace tllm {

__device__ int g_kv4_status = 0;

int kv4_read_status(int *out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_kv4_status, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyFromSymbol(kv4 status)");
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyToSymbol(kv4 status)");
  *out = v;
  return TLLM_OK;
}

namespace kv4 {
namespace {

using namespace rr;

constexpr int kThreads = 256;

struct Args {
  const void *k, *v;  // append: [T, H, D] in, gather: out; strides in elements
  int64_t skt, skh, svt, svh;
  uint8_t *cache;
  int64_t sblk, shead;  // bytes
  const int32_t *slots;
  int64_t T;
  int H;
  int log2_bs;
  int64_t num_slots;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The codes of the lane's 8 channels (channel i at bits 4 i) and its group's scale and zero. All
// four lanes of the group take part.
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], __half &s, __half &z) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  z = __float2half_rn(lo);
  const float sf = __half2float(s), zf = __half2float(z);
  const float inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], zf), inv)), 0.f), 15.f);  // NaN: 0
    codes |= static_cast<uint32_t>(c) << (4 * i);
  }
  return codes;
}

// Channels j at bits 4 j -> bits 4 (j / 2) + 16 (j % 2).
__device__ __forceinline__ uint32_t split_parity(uint32_t c) {
  uint32_t even = c & 0x0f0f0f0fu, odd = (c >> 4) & 0x0f0f0f0fu;
  even = (even | (even >> 4)) & 0x00ff00ffu;
  odd = (odd | (odd >> 4)) & 0x00ff00ffu;
  even = (even | (even >> 8)) & 0xffffu;
  odd = (odd | (odd >> 8)) & 0xffffu;
  return even | (odd << 16);
}

__device__ __forceinline__ uint8_t *piece_of(const Args &a, int64_t slot, int h, int bytes) {
  const int64_t in = slot & ((1 << a.log2_bs) - 1);
  return a.cache + (slot >> a.log2_bs) * a.sblk + h * a.shead + (in / kPieceTokens) * bytes;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(const Args a, uint32_t rows) {
  using P = Piece<D>;
  constexpr int LANES = D / 8;
  const uint32_t raw = (blockIdx.x * kThreads + threadIdx.x) / LANES;
  bool ok = raw < rows;  // lanes past the end recompute the last row (for the shuffles)
  const uint32_t row = ok ? raw : rows - 1;
  const uint32_t t = row / a.H;
  const int h = row % a.H;
  const int x = threadIdx.x % LANES;
  const int64_t slot = __ldg(a.slots + t);
  const T *kp = static_cast<const T *>(a.k) + static_cast<int64_t>(t) * a.skt + h * a.skh + 8 * x;
  const T *vp = static_cast<const T *>(a.v) + static_cast<int64_t>(t) * a.svt + h * a.svh + 8 * x;
  const uint4 kr = ld_stream(kp), vr = ld_stream(vp);
  if (slot >= a.num_slots && ok) atomicCAS(&g_kv4_status, 0, TLLM_DEV_BAD_INDEX);
  ok = ok && slot >= 0 && slot < a.num_slots;
  float kf[8], vf[8];
  unpack8<T>(kr, kf);
  unpack8<T>(vr, vf);
  __half ks, kz, vs, vz;
  const uint32_t kc = split_parity(quantise(kf, ks, kz));
  const uint32_t vc = quantise(vf, vs, vz);
  // Lane x = 4 g + m has V channels 32 g + 8 m + {0..7}: chunks n = 2 m (low half) and 2 m + 1. It
  // stores chunk n = x / (W / 2), groups 2 y and 2 y + 1 with y = x % (W / 2).
  constexpr int Y = P::W / 2;
  const int n = x / Y, y = x % Y;
  const int base = threadIdx.x & 31 & ~(LANES - 1);
  const uint32_t g0 = __shfl_sync(0xffffffffu, vc, base + 8 * y + (n >> 1));
  const uint32_t g1 = __shfl_sync(0xffffffffu, vc, base + 8 * y + 4 + (n >> 1));
  const uint32_t vw = __byte_perm(g0, g1, (n & 1) ? 0x7632 : 0x5410);
  if (!ok) return;
  uint8_t *p = piece_of(a, slot, h, P::BYTES);
  const int tok = static_cast<int>(slot & (kPieceTokens - 1));
  *reinterpret_cast<uint32_t *>(p + P::k_word(tok, x)) = kc;
  *reinterpret_cast<uint32_t *>(p + P::v_bits(tok, 2 * y, n)) = vw;
  const int g = x >> 2;
  switch (x & 3) {
    case 0: *reinterpret_cast<__half *>(p + P::k_scale(tok, g)) = ks; break;
    case 1: *reinterpret_cast<__half *>(p + P::k_zero(tok, g)) = kz; break;
    case 2: *reinterpret_cast<__half *>(p + P::v_scale(tok, g)) = vs; break;
    default: *reinterpret_cast<__half *>(p + P::v_zero(tok, g)) = vz; break;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_gather_kernel(const Args a, uint32_t rows) {
  using P = Piece<D>;
  constexpr int LANES = D / 8;
  const uint32_t row = (blockIdx.x * kThreads + threadIdx.x) / LANES;
  if (row >= rows) return;
  const uint32_t t = row / a.H;
  const int h = row % a.H;
  const int x = threadIdx.x % LANES;
  const int64_t slot = __ldg(a.slots + t);
  if (slot >= a.num_slots) atomicCAS(&g_kv4_status, 0, TLLM_DEV_BAD_INDEX);
  float kf[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, vf[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < a.num_slots) {
    const uint8_t *p = piece_of(a, slot, h, P::BYTES);
    const int tok = static_cast<int>(slot & (kPieceTokens - 1));
    const int g = x >> 2, n = 2 * (x & 3);
    const uint32_t kc = *reinterpret_cast<const uint32_t *>(p + P::k_word(tok, x));
    const uint32_t v0 = *reinterpret_cast<const uint16_t *>(p + P::v_bits(tok, g, n));
    const uint32_t v1 = *reinterpret_cast<const uint16_t *>(p + P::v_bits(tok, g, n + 1));
    const uint32_t vc = v0 | (v1 << 16);
    const float ks = __half2float(*reinterpret_cast<const __half *>(p + P::k_scale(tok, g)));
    const float kz = __half2float(*reinterpret_cast<const __half *>(p + P::k_zero(tok, g)));
    const float vs = __half2float(*reinterpret_cast<const __half *>(p + P::v_scale(tok, g)));
    const float vz = __half2float(*reinterpret_cast<const __half *>(p + P::v_zero(tok, g)));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      kf[j] = fmaf(static_cast<float>((kc >> (4 * (j >> 1) + 16 * (j & 1))) & 15u), ks, kz);
      vf[j] = fmaf(static_cast<float>((vc >> (4 * j)) & 15u), vs, vz);
    }
  }
  T *ko = static_cast<T *>(const_cast<void *>(a.k)) + static_cast<int64_t>(t) * a.skt + h * a.skh + 8 * x;
  T *vo = static_cast<T *>(const_cast<void *>(a.v)) + static_cast<int64_t>(t) * a.svt + h * a.svh + 8 * x;
  st_stream(ko, pack8<T>(kf));
  st_stream(vo, pack8<T>(vf));
}

template <typename T, int D>
int launch(const Args &a, bool append, cudaStream_t st) {
  const int64_t rows = a.T * a.H;
  const unsigned grid = static_cast<unsigned>((rows * (D / 8) + kThreads - 1) / kThreads);
  if (append) kv4_append_kernel<T, D><<<grid, kThreads, 0, st>>>(a, static_cast<uint32_t>(rows));
  else kv4_gather_kernel<T, D><<<grid, kThreads, 0, st>>>(a, static_cast<uint32_t>(rows));
  return cuda_status(cudaGetLastError(), append ? "paged kv4 append launch" : "paged kv4 gather launch");
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int entry(const char *op, bool append, const void *k, const void *v, void *cache,
          const int32_t *slots, int64_t T, int64_t H, int64_t D, int64_t block_size,
          int64_t num_blocks, const int64_t *sk, const int64_t *sv, const int64_t *sc, int dtype,
          void *stream) {
  clear_error();
  TLLM_CHECK_ARG(T >= 0 && H >= 0 && num_blocks >= 0, "%s: negative dimension", op);
  TLLM_CHECK_ARG(D == 64 || D == 128, "%s: head dim %lld not in {64,128}", op, (long long)D);
  TLLM_CHECK_ARG(block_size == 16 || block_size == 32 || block_size == 64,
                 "%s: block_size %lld not in {16,32,64}", op, (long long)block_size);
  TLLM_CHECK_ARG(dtype == TLLM_DTYPE_F16 || dtype == TLLM_DTYPE_BF16, "%s: unsupported dtype %d", op,
                 dtype);
  TLLM_CHECK_ARG(sk && sv && sc, "%s: null stride array", op);
  if (T * H == 0) return TLLM_OK;
  TLLM_CHECK_ARG(k && v && slots && (cache || num_blocks == 0), "%s: null tensor pointer", op);
  TLLM_CHECK_ARG(H < (1LL << 20) && T < (1LL << 31) && T * H * (D / 8) < (1LL << 32) - kThreads &&
                     num_blocks < (1LL << 31),
                 "%s: problem too large", op);
  for (int i = 0; i < 2; ++i)
    TLLM_CHECK_ARG(sk[i] % 8 == 0 && sv[i] % 8 == 0, "%s: strides must be multiples of 8 elements", op);
  TLLM_CHECK_ARG(sc[0] % 16 == 0 && sc[1] % 16 == 0, "%s: cache strides must be multiples of 16 bytes", op);
  TLLM_CHECK_ARG(aligned16(k) && aligned16(v) && aligned16(cache), "%s: tensors must be 16-byte aligned", op);
  Args a{};
  a.k = k;
  a.v = v;
  a.skt = sk[0];
  a.skh = sk[1];
  a.svt = sv[0];
  a.svh = sv[1];
  a.cache = static_cast<uint8_t *>(cache);
  a.sblk = sc[0];
  a.shead = sc[1];
  a.slots = slots;
  a.T = T;
  a.H = static_cast<int>(H);
  a.log2_bs = block_size == 16 ? 4 : (block_size == 32 ? 5 : 6);
  a.num_slots = num_blocks * block_size;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TLLM_DTYPE_F16) return D == 64 ? launch<__half, 64>(a, append, st) : launch<__half, 128>(a, append, st);
  return D == 64 ? launch<__nv_bfloat16, 64>(a, append, st) : launch<__nv_bfloat16, 128>(a, append, st);
}

}  // namespace
}  // namespace kv4
}  // namespace tllm

extern "C" int tllm_paged_kv4_append(const void *k, const void *v, void *cache, const int32_t *slots,
                                     int64_t T, int64_t H, int64_t D, int64_t block_size,
                                     int64_t num_blocks, const int64_t *sk, const int64_t *sv,
                                     const int64_t *sc, int dtype, void *stream) {
  return tllm::kv4::entry("paged_kv4_append", true, k, v, cache, slots, T, H, D, block_size,
                          num_blocks, sk, sv, sc, dtype, stream);
}

extern "C" int tllm_paged_kv4_gather(const void *cache, const int32_t *slots, void *k, void *v,
                                     int64_t T, int64_t H, int64_t D, int64_t block_size,
                                     int64_t num_blocks, const int64_t *sk, const int64_t *sv,
                                     const int64_t *sc, int dtype, void *stream) {
  return tllm::kv4::entry("paged_kv4_gather", false, k, v, const_cast<void *>(cache), slots, T, H, D,
                          block_size, num_blocks, sk, sv, sc, dtype, stream);
}
