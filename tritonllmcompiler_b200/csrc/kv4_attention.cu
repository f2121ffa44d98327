// Attention of new tokens over the 4-bit paged cache (kv4.cuh has the layout).
//
// Packed queries q [T, Hq, D]; sequence b owns rows cu[b] .. cu[b + 1], its n_b new tokens, already
// in the cache; token s of it sits at position len_b - n_b + s and, with causal, sees the keys up to
// its own. o = sum_t p_t v_t / sum_t p_t, p_t = 2^((q . k_t) scale log2(e) - m), k and v the values
// the cache stands for.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

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
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 32;   // tokens a warp takes at a time: two pieces
constexpr int kStages = 2;  // tiles of a warp in shared memory

enum : int { SITE_TILE = 0x41 };

struct Args {
  const void *q;
  const uint8_t *cache;
  const int32_t *block_tables, *lens, *cu;
  void *o;
  float *ws_ml;   // [row tiles][splits][rows of a tile][2] (maximum in log2 units, sum)
  float *ws_acc;  // [row tiles][splits][rows of a tile][D]
  int64_t sq0, sq1, so0, so1, sblk, shead, sbt0, sbt1;
  int64_t T, num_blocks, max_blocks;
  int B, Hkv, G, log2_bs, causal, max_new;
  int n_rt, splits, chunk;  // row tiles per sequence and KV head; key splits and their tokens
  float scale_log2;
};

// Where a CTA works: sequence b, row tile rt (rows r0 .. r0 + nr of the n_q * G rows, row r being new
// token r / G of query head hk * G + r % G), and how many keys its rows see.
struct Place {
  int b, rt, hk, r0, nr, row0, n_q, len, seen;
};

__device__ __forceinline__ int row_keys(const Args &a, const Place &p, int r) {
  return a.causal ? min(max(p.len - p.n_q + r / a.G + 1, 0), p.len) : p.len;
}

template <int ROWS>
__device__ __forceinline__ bool locate(const Args &a, int b, int rt, int hk, Place &p) {
  p.b = b;
  p.rt = rt;
  p.hk = hk;
  const int lim = static_cast<int>(a.T);
  p.row0 = min(max(__ldg(a.cu + b), 0), lim);
  p.n_q = min(max(__ldg(a.cu + b + 1), p.row0), lim) - p.row0;
  p.r0 = rt * ROWS;
  p.nr = min(ROWS, p.n_q * a.G - p.r0);
  if (p.nr <= 0) return false;
  p.len = static_cast<int>(min(static_cast<int64_t>(max(__ldg(a.lens + b), 0)), a.max_blocks << a.log2_bs));
  p.seen = row_keys(a, p, p.r0 + p.nr - 1);
  return true;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transposes an 8 x 8 matrix of 16-bit values held as an MMA fragment.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) { return Pack2<__half>::pack(a, b); }

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 .. 127

template <int N>
__device__ __forceinline__ void lds_words(const uint8_t *p, uint32_t (&w)[N]) {
  static_assert(N == 1 || N == 2 || N == 4, "vector width");
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  }
}

// The W fp16 scales of one token as fp32.
template <int W>
__device__ __forceinline__ void lds_scales(const uint8_t *p, float (&s)[W]) {
  uint32_t w[W / 2];
  lds_words<W / 2>(p, w);
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    const float2 f = Pack2<__half>::unpack(w[i]);
    s[2 * i] = f.x;
    s[2 * i + 1] = f.y;
  }
}

// Four fp16 pairs from a word of two times four codes: x[0], x[2] are the codes of bits 0-3 and 8-11 of
// each half times 2^-24, x[1], x[3] those of bits 4-7 and 12-15 times 2^-20 (subnormal numbers: the
// codes' own bits, exact, without a conversion).
__device__ __forceinline__ void spread(uint32_t w, uint32_t (&x)[4]) {
  x[0] = w & 0x000f000fu;
  x[1] = w & 0x00f000f0u;
  w >>= 8;
  x[2] = w & 0x000f000fu;
  x[3] = w & 0x00f000f0u;
}

// Few query rows per KV head (decode, speculative tokens): ROWS = 8 * NT rows a CTA.
//
// A CTA takes `chunk` tokens of one sequence and KV head; its four warps take tiles of 32 tokens in
// turn, each with its own ring of bulk copies (a page's K and V of one head are contiguous), its own
// running maximum and sum, and no barrier until they are added up at the end.
//
// Both products run as 16 x 8 x 16 MMAs with the cache as the 16-row operand, so 8 query rows fill
// them: S^T = K Q^T and O^T = V^T P^T. The operands from the cache are the codes themselves, as fp16
// subnormals masked out of the words (spread), which is exact; scales and zeros enter where they are
// cheap:
//   q . k = sum_g s_g (sum_{d in g} q_d c_d) + sum_g z_g (sum_{d in g} q_d): one FMA per group and
//           score on the products' fp32 results; the zeros are one more MMA with the sums of q, held as
//           high and low fp16 parts;
//   o_d   = sum_t (p_t s_{t,g}) c_{t,d} + sum_t p_t z_{t,g}: the weights times the scales are rounded
//           to fp16 per group, after a common power of two (from the largest scale met so far) that
//           keeps them in fp16's normal range; the zeros are one more MMA with 16 x 8 results.
// q is brought to [2^9, 2^10) by a power of two per row and is exact in fp16 from either type.
// An S^T result becomes a P^T operand by transposing 8 x 8 blocks in registers (movmatrix).
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3) kv4_split_kernel(const Args a) {
  using P = Piece<D>;
  constexpr int W = P::W;
  constexpr int ROWS = 8 * NT;
  constexpr int TILE_BYTES = 2 * P::BYTES;
  constexpr int RING = kStages * TILE_BYTES;
  static_assert(RING >= ROWS * D * 4, "a warp's results reuse its ring");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_bar[kWarps][kStages];
  __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
  __shared__ int s_abort;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, cq = lane & 3;  // fragment row (token, channel or query row) and column pair

  // ---- place ----
  const int64_t main_ctas = static_cast<int64_t>(a.B) * a.n_rt * a.splits * a.Hkv;
  if (blockIdx.x >= main_ctas) {  // the last CTA clears the rows that belong to no sequence
    const int64_t from = a.B > 0 ? min(max(static_cast<int64_t>(__ldg(a.cu + a.B)), int64_t{0}), a.T) : 0;
    const int64_t n = (a.T - from) * a.Hkv * a.G * (D / 8);
    for (int64_t i = tid; i < n; i += kThreads) {
      const int64_t row = i / (D / 8);
      T *o = static_cast<T *>(a.o) + (from + row / (a.Hkv * a.G)) * a.so0 + (row % (a.Hkv * a.G)) * a.so1;
      *reinterpret_cast<uint4 *>(o + (i % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int idx = static_cast<int>(blockIdx.x);
  const int hk = idx % a.Hkv;
  const int split = idx / a.Hkv % a.splits;
  const int brt = idx / a.Hkv / a.splits;
  Place pl;
  if (!locate<ROWS>(a, brt / a.n_rt, brt % a.n_rt, hk, pl)) return;
  if (pl.n_q > a.max_new && tid == 0) atomicCAS(&g_kv4a_status, 0, TLLM_DEV_BAD_INDEX);
  const int t0 = split * a.chunk;
  const int n = max(min(pl.seen - t0, a.chunk), 0);
  if (n == 0 && split > 0) return;  // the merge knows; split 0 always runs, for rows without keys
  const int n_tiles = (n + kTile - 1) / kTile;
  const int nk = n_tiles > warp ? (n_tiles - warp + kWarps - 1) / kWarps : 0;  // this warp's tiles

  if (tid == 0) {
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(smem_u32(&s_bar[0][0] + i), 1);
    s_abort = 0;
    fence_mbar_init();
  }
  __syncthreads();

  // ---- the warp's ring: tile k is tile warp + kWarps * k of the chunk ----
  uint8_t *ring = smem + warp * RING;
  int page0 = 0, page1 = 0;  // lane l: pages of tile 32 i + l
  auto issue = [&](int k) {
    if ((k & 31) == 0) {
      const int tok = t0 + (warp + kWarps * (k + lane)) * kTile;
      auto page = [&](int t) -> int {
        if (t >= pl.seen) return 0;
        const int p = __ldg(a.block_tables + pl.b * a.sbt0 + (t >> a.log2_bs) * a.sbt1);
        if (p >= 0 && p < a.num_blocks) return p;
        atomicCAS(&g_kv4a_status, 0, TLLM_DEV_BAD_INDEX);
        return 0;
      };
      if (k + lane < nk) {
        page0 = page(tok);
        page1 = a.log2_bs == 4 ? page(tok + kPieceTokens) : page0;
      }
    }
    const int64_t p0 = __shfl_sync(0xffffffffu, page0, k & 31);
    const int64_t p1 = __shfl_sync(0xffffffffu, page1, k & 31);
    if (lane == 0) {
      const int at = (warp + kWarps * k) * kTile;
      const bool both = n - at > kPieceTokens;
      const uint32_t bar = smem_u32(&s_bar[warp][k % kStages]);
      const uint32_t dst = smem_u32(ring + (k % kStages) * TILE_BYTES);
      const uint8_t *head = a.cache + hk * a.shead;
      mbar_arrive_expect_tx(bar, both ? TILE_BYTES : P::BYTES);
      if (a.log2_bs == 4) {
        bulk_load(dst, head + p0 * a.sblk, P::BYTES, bar);
        if (both) bulk_load(dst + P::BYTES, head + p1 * a.sblk, P::BYTES, bar);
      } else {
        const int piece = ((t0 + at) & ((1 << a.log2_bs) - 1)) / kPieceTokens;
        bulk_load(dst, head + p0 * a.sblk + piece * P::BYTES, both ? TILE_BYTES : P::BYTES, bar);
      }
    }
  };
  for (int k = 0; k < kStages && k < nk; ++k) issue(k);

  // ---- q: B fragments of Q^T, and each row's sums over the groups ----
  uint32_t qb[NT][W][4];  // words w: pairs {0,1}, {2,3} 2^-4, {4,5}, {6,7} 2^-4 of channels 32 w + 8 cq
  uint32_t qs[NT];
  float rs[NT][2];  // score factor of query rows 8 j + 2 cq, + 1
  int lim[NT][2];   // keys (from t0) that they see
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int row = pl.r0 + 8 * j + r;
    const bool ok = 8 * j + r < pl.nr;
    float f[W][8], top = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (ok)
        raw = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (pl.row0 + row / a.G) * a.sq0 +
                                                    (hk * a.G + row % a.G) * a.sq1 + 32 * w + 8 * cq));
      const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = Pack2<T>::unpack(u[i]);
        f[w][2 * i] = x.x;
        f[w][2 * i + 1] = x.y;
        top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // An infinite row keeps its infinities; a zero or subnormal one is scaled by 2^109 at most.
    const int e = max((__float_as_int(top) >> 23) - 127, -100);
    const float up = pow2(9 - e);
    float hi[W], lo[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[w][i] *= up;
        sum += f[w][i];
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      hi[w] = __half2float(__float2half_rn(sum));
      lo[w] = sum - hi[w];
      qb[j][w][0] = pack_half(f[w][0], f[w][1]);
      qb[j][w][1] = pack_half(f[w][2] * 0.0625f, f[w][3] * 0.0625f);
      qb[j][w][2] = pack_half(f[w][4], f[w][5]);
      qb[j][w][3] = pack_half(f[w][6] * 0.0625f, f[w][7] * 0.0625f);
    }
    // K index of the zeros' MMA: group g of the high parts, then of the low ones.
    qs[j] = 0;
#pragma unroll
    for (int i = 0; i < W; i += 2) {
      if (cq == i / 2) qs[j] = pack_half(hi[i], hi[i + 1]);
      if (cq == W / 2 + i / 2) qs[j] = pack_half(lo[i], lo[i + 1]);
    }
    const float down = pow2(e - 9) * a.scale_log2;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      rs[j][c] = __shfl_sync(0xffffffffu, down, 4 * (2 * cq + c));
      const int rr = 8 * j + 2 * cq + c;
      lim[j][c] = rr < pl.nr ? row_keys(a, pl, pl.r0 + rr) - t0 : n;
    }
  }
  const int lim_all = min(row_keys(a, pl, pl.r0) - t0, n);  // below this every row sees every key

  float acc[W][2][NT][4];  // O^T: [group][half][row tile]: channels 32 g + 4 r + 2 half (+ 1 in 2, 3)
  float accz[NT][4];       // zeros: row g of lane group r = g
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      accz[j][i] = 0.f;
#pragma unroll
      for (int g = 0; g < W; ++g) acc[g][0][j][i] = acc[g][1][j][i] = 0.f;
    }
    m[j][0] = m[j][1] = -INFINITY;
    l[j][0] = l[j][1] = 0.f;
  }
  int v_exp = 0;  // exponent field of the largest V scale so far

  auto scale_acc = [&](const float (&f)[NT][2]) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < W; ++g) {
          acc[g][0][j][i] *= f[j][i & 1];
          acc[g][1][j][i] *= f[j][i & 1];
        }
  };

  // One tile. kMask: some row does not see all of its 32 tokens.
  auto tile = [&](uint8_t *base, int at, auto mask_tag) {
    constexpr bool kMask = decltype(mask_tag)::value;
    if constexpr (kMask) {
      // Slots past the last key may hold anything: their V scales and zeros become 0. A zero that is
      // no number, in a token that only some rows see, would reach every row through its MMA; its
      // scale is then no number either, and alone marks the rows that do see it.
      uint8_t *pb = base + (lane >> 4) * P::BYTES;
      const int tok = lane & 15;
      const bool past = at + lane >= n;
#pragma unroll
      for (int g = 0; g < W; ++g) {
        uint16_t *z = reinterpret_cast<uint16_t *>(pb + P::v_zero(tok, g));
        if (past) *reinterpret_cast<uint16_t *>(pb + P::v_scale(tok, g)) = 0;
        if (past || (*z & 0x7c00u) == 0x7c00u) *z = 0;
      }
      __syncwarp();
    }
    // ---- scores ----
    float x[2][NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t *pb = base + h * P::BYTES;
      uint32_t z0 = 0, z1 = 0;
      if (W == 4 || cq < 2) {
        const uint8_t *zp = pb + P::k_zero(r, 0) + 4 * (cq % (W / 2));
        z0 = *reinterpret_cast<const uint32_t *>(zp);
        z1 = *reinterpret_cast<const uint32_t *>(zp + 8 * 2 * W);
      }
      uint32_t k0[W], k1[W];
      lds_words<W>(pb + P::K_CODES + r * (D / 2) + cq * (4 * W), k0);
      lds_words<W>(pb + P::K_CODES + (r + 8) * (D / 2) + cq * (4 * W), k1);
      float s0[W], s1[W];
      lds_scales<W>(pb + P::k_scale(r, 0), s0);
      lds_scales<W>(pb + P::k_scale(r + 8, 0), s1);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        x[h][j][0] = x[h][j][1] = x[h][j][2] = x[h][j][3] = 0.f;
        mma16816(x[h][j], z0, z1, 0u, 0u, qs[j], 0u);
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t u0[4], u1[4];
        spread(k0[w], u0);
        spread(k1[w], u1);
        const float f0 = s0[w] * 16777216.f, f1 = s1[w] * 16777216.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816(c, u0[0], u1[0], u0[1], u1[1], qb[j][w][0], qb[j][w][1]);
          mma16816(c, u0[2], u1[2], u0[3], u1[3], qb[j][w][2], qb[j][w][3]);
          x[h][j][0] = fmaf(f0, c[0], x[h][j][0]);
          x[h][j][1] = fmaf(f0, c[1], x[h][j][1]);
          x[h][j][2] = fmaf(f1, c[2], x[h][j][2]);
          x[h][j][3] = fmaf(f1, c[3], x[h][j][3]);
        }
      }
    }
    // ---- softmax: a lane has tokens r, r + 8 of each piece for rows 2 cq, 2 cq + 1 ----
    float m2[NT][2];
    bool grew = false;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = m[j][c];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float &v = x[h][j][c + 2 * i];
            v *= rs[j][c];
            if constexpr (kMask)
              if (at + 16 * h + r + 8 * i >= lim[j][c]) v = -INFINITY;
            top = fmaxf(top, v);
          }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        m2[j][c] = top;
        grew |= top > m[j][c];
      }
    if (__any_sync(0xffffffffu, grew)) {
      float f[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          f[j][c] = m[j][c] == -INFINITY ? 1.f : ex2_approx(m[j][c] - m2[j][c]);  // 1: nothing summed yet
          m[j][c] = m2[j][c];
          l[j][c] *= f[j][c];
          accz[j][c] *= f[j][c];
          accz[j][c + 2] *= f[j][c];
        }
      scale_acc(f);
    }
    // ---- the largest V scale of the tile ----
    {
      uint32_t v[W / 2], top = 0;
      lds_words<W / 2>(base + (lane >> 4) * P::BYTES + P::V_SCALE + (lane & 15) * 2 * W, v);
#pragma unroll
      for (int i = 0; i < W / 2; ++i) {
        const uint32_t u = v[i] & 0x7fff7fffu;
        top = __vmaxu2(top, u & __vcmpltu2(u, 0x7c007c00u));  // infinities and NaNs do not count
      }
      top = max(top & 0xffffu, top >> 16) >> 10;
      const int e = static_cast<int>(__reduce_max_sync(0xffffffffu, top));  // 0 .. 30
      if (e > v_exp) {
        float f[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) f[j][0] = f[j][1] = pow2(v_exp - e);
        scale_acc(f);
        v_exp = e;
      }
    }
    const float up = pow2(23 - v_exp);  // weight times scale times up < 2^9
    // ---- weights and O^T ----
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t *pb = base + h * P::BYTES;
      float s0[W], s1[W];
      lds_scales<W>(pb + P::v_scale(r, 0), s0);
      lds_scales<W>(pb + P::v_scale(r + 8, 0), s1);
      uint32_t z0 = 0, z2 = 0;
      if (r < W) {
        const uint8_t *zp = pb + P::v_zero(2 * cq, r);
        z0 = *reinterpret_cast<const uint32_t *>(zp);
        z2 = *reinterpret_cast<const uint32_t *>(zp + 16);
      }
      // Token pairs cq and cq + 4; W / 2 words of each token.
      const uint8_t *vp = pb + P::V_CODES + cq * D + (r ^ P::swizzle(cq)) * P::CHUNK;
      uint32_t v0[W], v1[W];
      lds_words<W>(vp, v0);
      lds_words<W>(vp + 4 * D, v1);
      float pf[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float mu = m[j][i & 1] == -INFINITY ? 0.f : m[j][i & 1];
          pf[j][i] = ex2_approx(x[h][j][i] - mu);
          l[j][i & 1] += pf[j][i];
        }
        const uint32_t b0 = transpose8(pack_half(pf[j][0], pf[j][1]));
        const uint32_t b1 = transpose8(pack_half(pf[j][2], pf[j][3]));
        mma16816(accz[j], z0, 0u, z2, 0u, b0, b1);
#pragma unroll
        for (int i = 0; i < 4; ++i) pf[j][i] *= up;
      }
#pragma unroll
      for (int g = 0; g < W; ++g) {
        const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
        uint32_t u0[4], u1[4];
        spread(__byte_perm(v0[g / 2], v0[W / 2 + g / 2], sel), u0);
        spread(__byte_perm(v1[g / 2], v1[W / 2 + g / 2], sel), u1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float w0 = pf[j][0] * s0[g], w1 = pf[j][1] * s0[g], w2 = pf[j][2] * s1[g], w3 = pf[j][3] * s1[g];
          if constexpr (kMask) {  // a hidden token's scale may be no number
            if (pf[j][0] == 0.f) w0 = 0.f;
            if (pf[j][1] == 0.f) w1 = 0.f;
            if (pf[j][2] == 0.f) w2 = 0.f;
            if (pf[j][3] == 0.f) w3 = 0.f;
          }
          const uint32_t b0 = transpose8(pack_half(w0, w1));
          const uint32_t b1 = transpose8(pack_half(w2, w3));
          mma16816(acc[g][0][j], u0[0], u0[1], u1[0], u1[1], b0, b1);
          mma16816(acc[g][1][j], u0[2], u0[3], u1[2], u1[3], b0, b1);
        }
      }
    }
  };

  bool ok = true;
  int k = 0;
  for (; k < nk && ok; ++k) {
    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_bar[warp][k % kStages]), (k / kStages) & 1, &s_abort,
                                           &g_kv4a_status, TLLM_DEV_WAIT_TIMEOUT + SITE_TILE));
    if (!ok) break;
    const int at = (warp + kWarps * k) * kTile;
    uint8_t *base = ring + (k % kStages) * TILE_BYTES;
    if (at + kTile > lim_all) {
      tile(base, at, std::true_type{});
      fence_proxy_async_smem();  // the tile was written to; a later copy may follow
    } else {
      tile(base, at, std::false_type{});
    }
    __syncwarp();
    if (k + kStages < nk) issue(k + kStages);
  }
  // After a wait that gave up: the copies in flight still write to this CTA's memory.
  for (int i = k; !ok && i < nk && i < k + kStages; ++i) {
    const long long since = clock64();
    while (!mbar_try_wait(smem_u32(&s_bar[warp][i % kStages]), (i / kStages) & 1) &&
           clock64() - since < kWaitLimitCycles) {
    }
  }

  // ---- the warps' results, through their rings ----
  const float f1 = pow2(1 + v_exp), f2 = pow2(v_exp - 3);  // 2^24 / up and 2^20 / up
  float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = 8 * j + 2 * cq + c;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], off);
      if (r == 0) {
        s_m[warp][row] = m[j][c];
        s_l[warp][row] = l[j][c];
      }
#pragma unroll
      for (int g = 0; g < W; ++g) {
        const float z = __shfl_sync(0xffffffffu, accz[j][c], 4 * g + cq);
        *reinterpret_cast<float4 *>(mine + row * D + 32 * g + 4 * r) =
            make_float4(fmaf(acc[g][0][j][c], f1, z), fmaf(acc[g][0][j][c + 2], f2, z),
                        fmaf(acc[g][1][j][c], f1, z), fmaf(acc[g][1][j][c + 2], f2, z));
      }
    }
  __syncthreads();
  const int64_t slot0 = ((static_cast<int64_t>(brt) * a.Hkv + hk) * a.splits + split) * ROWS;
  for (int i = tid; i < pl.nr * (D / 8); i += kThreads) {
    const int row = i / (D / 8), d = (i % (D / 8)) * 8;
    float top = s_m[0][row];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][row]);
    float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (s_m[w][row] == -INFINITY) continue;  // this warp has nothing for the row
      const float f = ex2_approx(s_m[w][row] - top);
      const float4 *p = reinterpret_cast<const float4 *>(smem + w * RING) + (row * D + d) / 4;
      const float4 x = p[0], y = p[1];
      sum = fmaf(s_l[w][row], f, sum);
      v[0] = fmaf(x.x, f, v[0]); v[1] = fmaf(x.y, f, v[1]); v[2] = fmaf(x.z, f, v[2]); v[3] = fmaf(x.w, f, v[3]);
      v[4] = fmaf(y.x, f, v[4]); v[5] = fmaf(y.y, f, v[5]); v[6] = fmaf(y.z, f, v[6]); v[7] = fmaf(y.w, f, v[7]);
    }
    if (a.splits == 1) {
      const int rr = pl.r0 + row;
      T *o = static_cast<T *>(a.o) + (pl.row0 + rr / a.G) * a.so0 + (hk * a.G + rr % a.G) * a.so1 + d;
      uint4 out;
      out.x = Pack2<T>::pack(v[0] / sum, v[1] / sum);
      out.y = Pack2<T>::pack(v[2] / sum, v[3] / sum);
      out.z = Pack2<T>::pack(v[4] / sum, v[5] / sum);
      out.w = Pack2<T>::pack(v[6] / sum, v[7] / sum);
      *reinterpret_cast<uint4 *>(o) = out;
    } else {
      float4 *p = reinterpret_cast<float4 *>(a.ws_acc + (slot0 + row) * D + d);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
      if (d == 0) *reinterpret_cast<float2 *>(a.ws_ml + 2 * (slot0 + row)) = make_float2(top, sum);
    }
  }
}

// One warp per query row: adds up the splits that have keys for its row tile.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kThreads) kv4_merge_kernel(const Args a) {
  constexpr int E = D / 32;
  const int64_t row_all = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t tile = row_all / ROWS;
  const int row = static_cast<int>(row_all % ROWS);
  if (tile >= static_cast<int64_t>(a.B) * a.n_rt * a.Hkv) return;
  const int hk = static_cast<int>(tile % a.Hkv), brt = static_cast<int>(tile / a.Hkv);
  Place pl;
  if (!locate<ROWS>(a, brt / a.n_rt, brt % a.n_rt, hk, pl) || row >= pl.nr) return;
  const int used = max((pl.seen + a.chunk - 1) / a.chunk, 1);
  const float2 *ml = reinterpret_cast<const float2 *>(a.ws_ml) + tile * a.splits * ROWS + row;
  const float *acc = a.ws_acc + (tile * a.splits * ROWS + row) * D + lane * E;
  float top = -INFINITY;
  for (int s = lane; s < used; s += 32) top = fmaxf(top, ml[s * ROWS].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  float sum = 0.f, v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < used; ++s) {
    const float2 x = ml[s * ROWS];
    const float f = x.x == -INFINITY ? 0.f : ex2_approx(x.x - top);
    sum = fmaf(x.y, f, sum);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = fmaf(acc[static_cast<int64_t>(s) * ROWS * D + i], f, v[i]);
  }
  const int rr = pl.r0 + row;
  T *o = static_cast<T *>(a.o) + (pl.row0 + rr / a.G) * a.so0 + (hk * a.G + rr % a.G) * a.so1 + lane * E;
#pragma unroll
  for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t *>(o + i) = Pack2<T>::pack(v[i] / sum, v[i + 1] / sum);
}

struct Plan {
  int nt = 1, n_rt = 1, splits = 1, chunk = 128;
  size_t ml_bytes = 0, ws_bytes = 0;
};

// Row tiles of 8 rows where all of a sequence's rows fit one, else of 16; key splits for four waves
// of CTAs, in chunks between 128 tokens (a tile per warp) and 2048.
Plan make_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t max_new, int64_t D, int64_t block_size,
               int64_t max_blocks) {
  Plan p;
  const int64_t rows = std::max<int64_t>(max_new, 1) * (Hq / Hkv);
  p.nt = rows <= 8 ? 1 : 2;
  p.n_rt = static_cast<int>((rows + 8 * p.nt - 1) / (8 * p.nt));
  const int64_t tiles = B * p.n_rt * Hkv, most = max_blocks * block_size;
  const int64_t want = 16LL * (sm_count() > 0 ? sm_count() : 148);
  int64_t chunk = 2048;
  while (chunk > 128 && tiles * ((most + chunk - 1) / chunk) < want) chunk /= 2;
  p.chunk = static_cast<int>(chunk);
  p.splits = static_cast<int>(std::max<int64_t>((most + chunk - 1) / chunk, 1));
  if (p.splits > 1) {
    const size_t slots = static_cast<size_t>(tiles) * p.splits * 8 * p.nt;
    p.ml_bytes = (slots * 2 * sizeof(float) + 255) / 256 * 256;
    p.ws_bytes = p.ml_bytes + slots * D * sizeof(float);
  }
  return p;
}

template <typename T, int D, int NT>
int launch(const Args &a, cudaStream_t st) {
  auto kern = kv4_split_kernel<T, D, NT>;
  constexpr int smem = kWarps * kStages * 2 * Piece<D>::BYTES;
  KernelLaunchInfo info;
  const int rc = prepare_kernel(reinterpret_cast<const void *>(kern), smem, kThreads, 1, &info);
  if (rc) return rc;
  const int64_t tiles = static_cast<int64_t>(a.B) * a.n_rt * a.Hkv;
  kern<<<static_cast<unsigned>(tiles * a.splits + 1), kThreads, smem, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_status(e, "paged kv4 attention launch");
  if (a.splits > 1 && tiles > 0) {
    const unsigned grid = static_cast<unsigned>((tiles * 8 * NT + kWarps - 1) / kWarps);
    kv4_merge_kernel<T, D, 8 * NT><<<grid, kThreads, 0, st>>>(a);
    e = cudaGetLastError();
  }
  return cuda_status(e, "paged kv4 attention merge launch");
}

template <typename T>
int launch_d(const Args &a, int64_t D, int nt, cudaStream_t st) {
  if (D == 64) return nt == 1 ? launch<T, 64, 1>(a, st) : launch<T, 64, 2>(a, st);
  return nt == 1 ? launch<T, 128, 1>(a, st) : launch<T, 128, 2>(a, st);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace kv4
}  // namespace tllm

extern "C" size_t tllm_paged_kv4_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                                                     int64_t max_new, int64_t D, int64_t block_size,
                                                     int64_t max_blocks) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || max_new < 0 || D <= 0 || block_size <= 0 || max_blocks <= 0)
    return 0;
  return tllm::kv4::make_plan(B, Hq, Hkv, max_new, D, block_size, max_blocks).ws_bytes;
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
  a.Hkv = static_cast<int>(Hkv);
  a.G = static_cast<int>(Hq / Hkv);
  a.log2_bs = block_size == 16 ? 4 : (block_size == 32 ? 5 : 6);
  a.causal = causal ? 1 : 0;
  a.scale_log2 = sm_scale * kLog2e;
  a.max_new = static_cast<int>(std::min<int64_t>(max_new, T));
  const Plan pl = make_plan(B, Hq, Hkv, a.max_new, D, block_size, max_blocks);
  TLLM_CHECK_ARG(B * pl.n_rt * Hkv * pl.splits < (1LL << 31) - 1, "paged_kv4_attn: grid too large");
  a.n_rt = pl.n_rt;
  a.splits = pl.splits;
  a.chunk = pl.chunk;
  if (pl.ws_bytes > 0) {
    if (!workspace || workspace_bytes < pl.ws_bytes)
      return fail(TLLM_ERR_WORKSPACE, "paged_kv4_attn: workspace of %zu bytes needed, %zu given", pl.ws_bytes,
                  workspace_bytes);
    TLLM_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
                   "paged_kv4_attn: workspace must be 256-byte aligned");
    a.ws_ml = static_cast<float *>(workspace);
    a.ws_acc = reinterpret_cast<float *>(static_cast<char *>(workspace) + pl.ml_bytes);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == TLLM_DTYPE_F16 ? launch_d<__half>(a, D, pl.nt, st) : launch_d<__nv_bfloat16>(a, D, pl.nt, st);
}
