// Writing K/V rows into the 4-bit paged cache by slot, and reading rows back (kv4.cuh has the
// layout).
//
// A group of 32 channels x of one token and head becomes
//   s = fp16((max - min) * (1 / 15)), z = fp16(min), code = clamp(rint((x - z) * (s > 0 ? 1 / s : 0)), 0, 15),
// each step one IEEE fp32 operation (no contraction), so the codes do not depend on the compiler. Where
// all of the group is within fp16's range but 15 s + z rounds past its end (a scale that was rounded up), s is
// one fp16 step less, so that every code stands for a number of that range.
// s and z are fp16: 11 bits put the reconstruction within 1 / 2048 of the group's range of where
// exact ones would, a fraction of the half step of 1 / 30, for 4 bytes per 16 bytes of codes. A
// group with a NaN, an infinity or a value that fp16 has no room for gets the scale NaN, so that all of it
// reads back as NaN, here and in attention: its zero may be finite, and so may both, and then some of what it
// stands for could be a number in one kernel and none in another.
//
// Bound: HBM, 2 bytes in and 0.625 out per element (the other way round when reading back), if the
// arithmetic stays at a few instructions per element. So a lane that writes holds a whole group of
// K or of V (64 bytes): minimum and maximum are packed 16-bit operations without shuffles, there is
// one reciprocal per group, differences and products are fp32 pairs, rounding and conversion are one
// addition, and a group whose ends round into 0 .. 15 needs no clamps inside. 16001 tokens of 8
// heads of 128: 27 us, 3 TB/s (a lane per 8 channels of both, each clamped and converted: 32 us). The
// lanes' 64 registers leave 32 warps an SM, and what one token writes is 8 to 16 bytes at a time,
// so latency and partial sectors hold it now, not issue. Reading back needs no group in one lane: 8
// channels of K and V each make wide coalesced stores, 20 us and 4 TB/s for the same rows (a group per
// lane: 28). No two lanes write the same byte, so tokens of one piece may be appended in any order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

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

// Packed minimum and maximum that keep NaNs.
__device__ __forceinline__ __half2 min2(__half2 a, __half2 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __half2 max2(__half2 a, __half2 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 min2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 max2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
template <typename T>
struct Two;
template <>
struct Two<__half> {
  using type = __half2;
};
template <>
struct Two<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

constexpr float kRound = 12582912.f;  // 1.5 * 2^23: y + kRound has y, rounded to even, in its low bits
// Sum of 16^i times the bits of kRound over four codes: what Horner's rule over the raw sums adds.
constexpr uint32_t kRoundBits = 0x4b400000u;
constexpr uint32_t kRoundFour = kRoundBits * 0x1111u;

constexpr float kPastHalf = 65520.f;  // rounds to infinity in fp16

// A group's 32 channels, two a word: its scale and zero, and sums[i] = kRoundBits + code i.
template <typename T>
__device__ __forceinline__ void quantise(const uint32_t (&w)[16], __half &s, __half &z, uint32_t (&sums)[32]) {
  using T2 = typename Two<T>::type;
  T2 lo2 = *reinterpret_cast<const T2 *>(&w[0]), hi2 = lo2;
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    const T2 v = *reinterpret_cast<const T2 *>(&w[i]);
    lo2 = min2(lo2, v);
    hi2 = max2(hi2, v);
  }
  const float2 l = Pack2<T>::unpack(*reinterpret_cast<const uint32_t *>(&lo2));
  const float2 h = Pack2<T>::unpack(*reinterpret_cast<const uint32_t *>(&hi2));
  // A NaN in either half has to stay.
  const float lo = l.x <= l.y ? l.x : (l.y < l.x ? l.y : __fadd_rn(l.x, l.y));
  const float hi = h.x >= h.y ? h.x : (h.y > h.x ? h.y : __fadd_rn(h.x, h.y));
  s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  z = __float2half_rn(lo);
  const float zf = __half2float(z);
  if (!(lo > -kPastHalf && hi < kPastHalf)) s = __ushort_as_half(0x7fff);  // NaN
  else if (__fmaf_rn(15.f, __half2float(s), zf) >= kPastHalf) s = __ushort_as_half(__half_as_ushort(s) - 1);
  const float sf = __half2float(s);
  const float inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
  // All steps are monotonic: if the ends stay inside, so does everything between.
  const bool inside = __fmul_rn(__fsub_rn(lo, zf), inv) >= -0.5f && __fmul_rn(__fsub_rn(hi, zf), inv) < 15.5f;
  const uint64_t mz = f2_pack(-zf, -zf), inv2 = f2_pack(inv, inv);
  if (inside) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 f = Pack2<T>::unpack(w[i]);
      float a, b;
      f2_unpack(f2_mul(f2_add(f2_pack(f.x, f.y), mz), inv2), a, b);
      sums[2 * i] = __float_as_uint(__fadd_rn(a, kRound));  // (a packed sum is contracted with the product)
      sums[2 * i + 1] = __float_as_uint(__fadd_rn(b, kRound));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 f = Pack2<T>::unpack(w[i]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float y = __fmul_rn(__fsub_rn(e ? f.y : f.x, zf), inv);
        sums[2 * i + e] = __float_as_uint(__fadd_rn(fminf(fmaxf(y, 0.f), 15.f), kRound));  // NaN: 0
      }
    }
  }
}

// Four codes at bits 0, 4, 8, 12.
__device__ __forceinline__ uint32_t four(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return ((d * 16u + c) * 16u + b) * 16u + a - kRoundFour;
}

__device__ __forceinline__ uint8_t *piece_of(const Args &a, int64_t slot, int h, int bytes) {
  const int64_t in = slot & ((1 << a.log2_bs) - 1);
  return a.cache + (slot >> a.log2_bs) * a.sblk + h * a.shead + (in / kPieceTokens) * bytes;
}

// 2 W lanes a row: the W groups of K, then those of V.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(const Args a, uint32_t rows) {
  using P = Piece<D>;
  constexpr int LANES = 2 * P::W;
  const uint32_t row = (blockIdx.x * kThreads + threadIdx.x) / LANES;
  if (row >= rows) return;
  const uint32_t t = row / a.H;
  const int h = row % a.H;
  const int g = threadIdx.x % P::W;
  const bool is_v = (threadIdx.x % LANES) >= P::W;
  const int64_t slot = __ldg(a.slots + t);
  const T *src = is_v ? static_cast<const T *>(a.v) + static_cast<int64_t>(t) * a.svt + h * a.svh
                      : static_cast<const T *>(a.k) + static_cast<int64_t>(t) * a.skt + h * a.skh;
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src + kGroup * g + 8 * i));  // a line is read in four goes: keep it
    w[4 * i] = v.x;
    w[4 * i + 1] = v.y;
    w[4 * i + 2] = v.z;
    w[4 * i + 3] = v.w;
  }
  if (slot >= a.num_slots) atomicCAS(&g_kv4_status, 0, TLLM_DEV_BAD_INDEX);
  if (slot < 0 || slot >= a.num_slots) return;
  __half s, z;
  uint32_t c[32];
  quantise<T>(w, s, z, c);
  uint8_t *p = piece_of(a, slot, h, P::BYTES);
  const int tok = static_cast<int>(slot & (kPieceTokens - 1));
  if (is_v) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
      *reinterpret_cast<uint16_t *>(p + P::v_bits(tok, g, n)) =
          static_cast<uint16_t>(four(c[4 * n], c[4 * n + 1], c[4 * n + 2], c[4 * n + 3]));
    *reinterpret_cast<__half *>(p + P::v_scale(tok, g)) = s;
    *reinterpret_cast<__half *>(p + P::v_zero(tok, g)) = z;
  } else {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<uint32_t *>(p + P::k_word(tok, 4 * g + x)) =
          four(c[8 * x], c[8 * x + 2], c[8 * x + 4], c[8 * x + 6]) +
          (four(c[8 * x + 1], c[8 * x + 3], c[8 * x + 5], c[8 * x + 7]) << 16);
    *reinterpret_cast<__half *>(p + P::k_scale(tok, g)) = s;
    *reinterpret_cast<__half *>(p + P::k_zero(tok, g)) = z;
  }
}

// Two codes (bits 0-3 of the halves of w) as a pair of T: code * s + z.
template <typename T>
__device__ __forceinline__ uint32_t values(uint32_t w, uint64_t s2, uint64_t z2) {
  const uint32_t h = w & 0x000f000fu;
  // Integers under the exponent of 2^23, less 2^23: no conversion instruction.
  const float a = __uint_as_float(0x4b000000u | (h & 15u)) - 8388608.f;
  const float b = __uint_as_float(0x4b000000u | (h >> 16)) - 8388608.f;
  float x, y;
  f2_unpack(f2_fma(f2_pack(a, b), s2, z2), x, y);
  return Pack2<T>::pack(x, y);
}

// A lane per 8 channels of both rows.
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
  uint4 ko = make_uint4(0u, 0u, 0u, 0u), vo = ko;
  if (slot >= 0 && slot < a.num_slots) {
    const uint8_t *p = piece_of(a, slot, h, P::BYTES);
    const int tok = static_cast<int>(slot & (kPieceTokens - 1));
    const int g = x >> 2, n = 2 * (x & 3);
    const uint32_t kc = *reinterpret_cast<const uint32_t *>(p + P::k_word(tok, x));
    const uint32_t v0 = *reinterpret_cast<const uint16_t *>(p + P::v_bits(tok, g, n));
    const uint32_t v1 = *reinterpret_cast<const uint16_t *>(p + P::v_bits(tok, g, n + 1));
    const float ks = __half2float(*reinterpret_cast<const __half *>(p + P::k_scale(tok, g)));
    const float kz = __half2float(*reinterpret_cast<const __half *>(p + P::k_zero(tok, g)));
    const float vs = __half2float(*reinterpret_cast<const __half *>(p + P::v_scale(tok, g)));
    const float vz = __half2float(*reinterpret_cast<const __half *>(p + P::v_zero(tok, g)));
    const uint64_t ks2 = f2_pack(ks, ks), kz2 = f2_pack(kz, kz), vs2 = f2_pack(vs, vs), vz2 = f2_pack(vz, vz);
    ko = make_uint4(values<T>(kc, ks2, kz2), values<T>(kc >> 4, ks2, kz2), values<T>(kc >> 8, ks2, kz2),
                    values<T>(kc >> 12, ks2, kz2));
    vo = make_uint4(values<T>(v0 | (v0 << 12), vs2, vz2), values<T>((v0 >> 8) | (v0 << 4), vs2, vz2),
                    values<T>(v1 | (v1 << 12), vs2, vz2), values<T>((v1 >> 8) | (v1 << 4), vs2, vz2));
  }
  st_stream(static_cast<T *>(const_cast<void *>(a.k)) + static_cast<int64_t>(t) * a.skt + h * a.skh + 8 * x, ko);
  st_stream(static_cast<T *>(const_cast<void *>(a.v)) + static_cast<int64_t>(t) * a.svt + h * a.svh + 8 * x, vo);
}

template <typename T, int D>
int launch(const Args &a, bool append, cudaStream_t st) {
  const int64_t rows = a.T * a.H;
  const int lanes = append ? 2 * Piece<D>::W : D / 8;
  const unsigned grid = static_cast<unsigned>((rows * lanes + kThreads - 1) / kThreads);
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
  // The largest slot stands for all those that int32 has no number for (paged_plan saturates).
  a.num_slots = std::min<int64_t>(num_blocks * block_size, INT32_MAX);
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
