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

#include "kv4_attention.cuh"

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

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 32;   // tokens a warp takes at a time: two pieces
constexpr int kStages = 2;  // tiles of a warp in shared memory
constexpr int kMergeLoads = 8;  // parts a merging warp reads at a time
constexpr int kMinTiles = 2;  // a warp's least run of tiles
// Places of the line that a segment's queries, results and start take (64 and 300 requests of 512 .. 8192 keys, four
// of 65,536 .. 131,072 with up to 32 rows, from a cold L2: none 110, 390 and 194 us, 3 105, 368 and 191, 4 103, 365 and
// 191, 6 103, 368 and 187).
constexpr int kExtra = 4;
// Query rows per sequence and KV head up to which kv4_split_kernel runs. 64 requests of 512 .. 8192 keys, split
// and prefill kernel: 16 rows 163 and 265 us, 32 rows 300 and 268, 48 rows 429 and 271; four of 100,000 keys,
// 32 rows: 286 and 294. (Rows alone, so a batch of many requests with 17 to 32 rows each is up to 12 % from the
// better of the two.)
constexpr int kSplitRows = 32;

// CTAs of the split kernel per SM: what its registers allow without spilling much. One row tile of 8 (64 requests of
// 512 .. 8192 keys, a row tile of 4 rows): three CTAs 103 us, four, in 128 registers, 112. Two (the same requests with
// 16 rows; four of 65,536 .. 131,072 keys): two CTAs 163 and 189 us, three, in 168 registers, 179 and 212.
__host__ __device__ constexpr int resident(int nt) { return nt == 1 ? 3 : 2; }

// Units of the products with the codes (fp16 subnormals) and with the zeros. The sums of q are split into two fp16
// parts, 22 bits: in the codes' unit the low part would be a subnormal, and the sum a multiple of half a q unit.
constexpr float kCodeUnit = 1.f / 16777216.f, kSumUnit = 1.f / 16.f;

enum : int { SITE_TILE = 0x41 };

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
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// v[r % W] without an indexed register.
template <int W>
__device__ __forceinline__ uint32_t pick(const uint32_t (&v)[W], int r) {
  if constexpr (W == 2) return (r & 1) ? v[1] : v[0];
  else return (r & 2) ? ((r & 1) ? v[3] : v[2]) : ((r & 1) ? v[1] : v[0]);
}

// Four fp16 pairs from a word of two times four codes: x[0], x[2] are the codes of bits 0-3 and 8-11 of
// each half times 2^-24, x[1], x[3] those of bits 4-7 and 12-15 times 2^-20 (subnormal numbers: the
// codes' own bits, exact, without a conversion).
__device__ __forceinline__ void spread(uint32_t w, uint32_t (&x)[4]) {
  x[0] = w & 0x000f000fu;
  x[1] = w & 0x00f000f0u;
  w = __byte_perm(w, 0u, 0x4341);  // the upper bytes of the halves
  x[3] = w & 0x00f000f0u;
  x[2] = sub_half2(w, x[3]);  // exact, and not on the logic pipe, which is the busier one
}

// Few query rows per KV head (decode, speculative tokens): ROWS = 8 * NT rows a row tile.
//
// A worker of the line (kv4_attention.cuh) is a warp, and the grid one wave of CTAs. A warp works by
// itself: its own ring of bulk copies (a page's K and V of one head are contiguous), its own running
// maximum and sum. A row tile that lies whole in a run is stored at once; otherwise each warp stores
// its part, and kv4_merge_kernel adds the parts up. (CTAs of one row tile and 1024 keys each, as
// before, spent 5 us of latency per CTA in starting and joining: 115 against 101 us for 64 requests of
// U[512, 8192], 32 heads over 8.)
//
// Both products run as 16 x 8 x 16 MMAs with the cache as the 16-row operand, so 8 query rows fill
// them: S^T = K Q^T and O^T = V^T P^T. The operands from the cache are the codes themselves, as fp16
// subnormals masked out of the words (spread), which is exact; scales and zeros enter where they are
// cheap:
//   q . k = sum_g s_g (sum_{d in g} q_d c_d) + sum_g z_g (sum_{d in g} q_d): one FMA per group and
//           score on the products' fp32 results; the zeros are one more MMA with the sums of q, held as
//           high and low fp16 parts. q is brought to [2^12, 2^13) by a power of two per row and is
//           exact in fp16 from either type (elements 2^-25 of the row's largest or less aside), so scores are
//           exact but for fp32 sums and the sums' 22 bits: within 2^-20 of the sizes of their terms.
//   o_d   = sum_t (p_t s_{t,g}) (c_{t,d} - 8) + sum_t p_t (z_{t,g} + 8 s_{t,g}): weights are fp16, and
//           fp16 again after the scale (packed products on the transposed weights, a third of the
//           instructions of fp32 ones). The second sum is one more MMA. The 8 centres both sums on
//           0: without it two sums of twice the size cancel, with 2.4 times the rounding errors, and over
//           100,000 keys the MMAs' truncating sums alone doubled the error of a bf16 output. (z + 8 s is rounded
//           to fp16, an error of 2^-12 of the group's middle.) For fp16
//           outputs the low parts that the rounding after the scale leaves out are multiplied too
//           (error 1.4 times that of rounding the output, against 1.6, for 5 % of the time).
// Weights are 2^(x - mu) with mu = m - k: k <= 12 keeps the weights times the scales in fp16's normal
// range whatever the size of V (from the largest scale met), and m follows the maximum only
// when it grows by more than 2^3 (weights and products stay under 2^15).
// An S^T result becomes a P^T operand by transposing 8 x 8 blocks in registers (movmatrix).
//
// Bound: HBM by bytes (1.25 D per token and head), but nothing is saturated: latency between the few warps that the
// registers allow holds it. 64 decode steps of U[512, 8192] keys, 32 heads over 8 of 128, fp16: 101 us, 3.9 TB/s, with
// 11 warps an SM half of the HBM's peak, 55 % of the issue slots, 45 % of the integer and 33 % of the tensor pipe; four
// requests of 65,536 .. 131,072 keys with up to 32 rows: 183 us, with 8 warps half of the issue slots and 38 % of the
// tensor pipe (each code is turned into operands once for 16 rows).
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, resident(NT)) kv4_split_kernel(const Args a) {
  using P = Piece<D>;
  constexpr int W = P::W;
  constexpr int ROWS = 8 * NT;
  constexpr bool kLow = std::is_same<T, __half>::value;  // weights times scales with their low parts
  constexpr int TILE_BYTES = 2 * P::BYTES;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_bar[kWarps][kStages];
  __shared__ LineScan<kThreads, kWarps> s_line;
  __shared__ int s_abort;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, cq = lane & 3;  // fragment row (token, channel or query row) and column pair

  if (tid == 0) {
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(smem_u32(&s_bar[0][0] + i), 1);
    s_abort = 0;
    fence_mbar_init();
  }
  int64_t per, total;
  const bool over = scan_line<ROWS, kTile, kExtra>(a, s_line, kMinTiles, per, total, &g_kv4a_status);
  other_rows<T, D>(a, over);
  const int worker = blockIdx.x * kWarps + warp;
  if (lane == 0) a.ws_open[worker].workers = 0;
  int64_t pos = worker * per;
  const int64_t end = min(pos + per, total);
  Segment sg;
  if (pos >= end || !first_segment<ROWS, kTile, kExtra>(a, s_line.seq[warp], s_line.rt[warp], s_line.off[warp], end - pos, sg)) return;
  const Place &pl = sg.pl;
  bool at_start = true;  // the worker's first segment

  // ---- the warp's ring ----
  uint8_t *ring = smem + warp * (kStages * TILE_BYTES);
  // This warp's fragments of q, kept out of the registers: [row tile of 8][word][lane].
  uint4 *qf = reinterpret_cast<uint4 *>(smem + kWarps * kStages * TILE_BYTES) + warp * (NT * W * 32);
  uint32_t taken = 0;        // tiles taken from the ring so far, over all segments
  int page0 = 0, page1 = 0;  // lane l: pages of the segment's tile 32 i + l
  // Starts the copy of the segment's tile k, `ahead` tiles after the next one to be taken.
  auto issue = [&](int k, int ahead) {
    if ((k & 31) == 0) {
      const int tok = (sg.first + k + lane) * kTile;
      auto page = [&](int t) -> int {
        if (t >= pl.seen) return 0;
        const int p = __ldg(a.block_tables + pl.b * a.sbt0 + (t >> a.log2_bs) * a.sbt1);
        if (p >= 0 && p < a.num_blocks) return p;
        atomicCAS(&g_kv4a_status, 0, TLLM_DEV_BAD_INDEX);
        return 0;
      };
      if (k + lane < sg.count) {
        page0 = page(tok);
        if (a.log2_bs == 4) page1 = page(tok + kPieceTokens);
      }
    }
    if (lane == (k & 31)) {  // the lane that has the pages
      const int tok = (sg.first + k) * kTile;
      const bool both = pl.seen - tok > kPieceTokens;
      const uint32_t stage = (taken + ahead) % kStages;
      const uint32_t bar = smem_u32(&s_bar[warp][stage]), dst = smem_u32(ring) + stage * TILE_BYTES;
      const uint8_t *src = a.cache + sg.hk * a.shead + page0 * a.sblk;
      mbar_arrive_expect_tx(bar, both ? TILE_BYTES : P::BYTES);
      if (a.log2_bs == 4) {
        bulk_load(dst, src, P::BYTES, bar);
        if (both) bulk_load(dst + P::BYTES, a.cache + sg.hk * a.shead + page1 * a.sblk, P::BYTES, bar);
      } else {
        const int piece = (tok & ((1 << a.log2_bs) - 1)) / kPieceTokens;
        bulk_load(dst, src + piece * P::BYTES, both ? TILE_BYTES : P::BYTES, bar);
      }
    }
  };
  auto prime = [&] {
    for (int k = 0; k < kStages && k < sg.count && pl.seen > 0; ++k) issue(k, k);
  };
  prime();

  while (true) {
  // ---- q: B fragments of Q^T, and each row's sums over the groups ----
  uint32_t qs[NT];
  float rs[NT][2];  // score factor (log2 units) of query rows 8 j + 2 cq, + 1
  int lim[NT][2];   // keys that they see
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
                                                    (sg.hk * a.G + row % a.G) * a.sq1 + 32 * w + 8 * cq));
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
    // An infinite row keeps its infinities; a zero or subnormal one is scaled by 2^112 at most.
    const int e = max((__float_as_int(top) >> 23) - 127, -100);
    const float up = pow2(12 - e);
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
      sum *= kSumUnit;  // |sum| < 2^14
      hi[w] = __half2float(__float2half_rn(sum));
      lo[w] = sum - hi[w];
      // pairs {0,1}, {2,3} 2^-4, {4,5}, {6,7} 2^-4 of channels 32 w + 8 cq
      qf[(j * W + w) * 32 + lane] =
          make_uint4(pack_half(f[w][0], f[w][1]), pack_half(f[w][2] * 0.0625f, f[w][3] * 0.0625f),
                     pack_half(f[w][4], f[w][5]), pack_half(f[w][6] * 0.0625f, f[w][7] * 0.0625f));
    }
    // K index of the zeros' MMA: group g of the high parts, then of the low ones.
    qs[j] = 0;
#pragma unroll
    for (int i = 0; i < W; i += 2) {
      if (cq == i / 2) qs[j] = pack_half(hi[i], hi[i + 1]);
      if (cq == W / 2 + i / 2) qs[j] = pack_half(lo[i], lo[i + 1]);
    }
    const float down = pow2(e) * (4096.f * a.scale_log2);  // 2^(e - 12) for q, 2^24 for the codes' unit
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      rs[j][c] = __shfl_sync(0xffffffffu, down, 4 * (2 * cq + c));
      const int rr = 8 * j + 2 * cq + c;
      lim[j][c] = rr < pl.nr ? row_keys(a, pl, pl.r0 + rr) : pl.seen;
    }
  }
  const int lim_all = row_keys(a, pl, pl.r0);  // below this every row sees every key

  float acc[W][2][NT][4];  // O^T: [group][half][row tile]: channels 32 g + 4 r + 2 half (+ 1 in 2, 3)
  float accz[NT][4];       // zeros: row g of lane group r = g
  float m[NT][2], mu[NT][2], l[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      accz[j][i] = 0.f;
#pragma unroll
      for (int g = 0; g < W; ++g) acc[g][0][j][i] = acc[g][1][j][i] = 0.f;
    }
    m[j][0] = m[j][1] = -INFINITY;
    mu[j][0] = mu[j][1] = l[j][0] = l[j][1] = 0.f;
  }
  int v_exp = 0;  // exponent field of the largest V scale so far

  // One tile. kMask: some row does not see all of its 32 tokens.
  auto tile = [&](uint8_t *base, int at, auto mask_tag) {
    constexpr bool kMask = decltype(mask_tag)::value;
    if constexpr (kMask) {
      // Slots past the last key may hold anything, and a group without numbers must not reach rows that do not
      // see its token (0 times infinity is no number): their V scales and zeros become 0, and the rows that
      // see the token get NaN, through the sum that all channels of the group have.
      const bool past = at + lane >= pl.seen;
      uint8_t *pb = base + (lane >> 4) * P::BYTES;
      uint32_t none = 0;
#pragma unroll
      for (int g = 0; g < W; ++g) {
        uint16_t *sp = reinterpret_cast<uint16_t *>(pb + P::v_scale(lane & 15, g));
        uint16_t *zp = reinterpret_cast<uint16_t *>(pb + P::v_zero(lane & 15, g));
        const bool number = (fma_half2(*sp, 0x4800u, *zp) & 0x7fffu) < 0x7c00u;  // z + 8 s
        if (!past && !number) none |= 1u << g;
        if (past || !number) *sp = *zp = 0;
      }
      for (uint32_t left = __ballot_sync(0xffffffffu, none != 0); left != 0; left &= left - 1) {
        const int t = __ffs(left) - 1;
        if ((__shfl_sync(0xffffffffu, none, t) >> (r % W)) & 1u) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (at + t < lim[j][c]) accz[j][c] = __int_as_float(0x7fc00000);
        }
      }
      __syncwarp();
    }
    // ---- scores ----
    float x[2][NT][4];
    uint32_t k0[2][W], k1[2][W], s0[2][W / 2], s1[2][W / 2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t *pb = base + h * P::BYTES;
      load_words<W>(pb + P::K_CODES + r * (D / 2) + cq * (4 * W), k0[h]);
      load_words<W>(pb + P::K_CODES + (r + 8) * (D / 2) + cq * (4 * W), k1[h]);
      load_words<W / 2>(pb + P::k_scale(r, 0), s0[h]);
      load_words<W / 2>(pb + P::k_scale(r + 8, 0), s1[h]);
      uint32_t z0 = 0, z1 = 0;
      if (W == 4 || cq < 2) {
        const uint8_t *zp = pb + P::k_zero(r, 0) + 4 * (cq % (W / 2));
        z0 = *reinterpret_cast<const uint32_t *>(zp);
        z1 = *reinterpret_cast<const uint32_t *>(zp + 8 * 2 * W);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        x[h][j][0] = x[h][j][1] = x[h][j][2] = x[h][j][3] = 0.f;
        mma16816(x[h][j], z0, z1, 0u, 0u, qs[j], 0u);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[h][j][i] *= kCodeUnit / kSumUnit;
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      uint4 qb[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) qb[j] = qf[(j * W + w) * 32 + lane];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t u0[4], u1[4];
        spread(k0[h][w], u0);
        spread(k1[h][w], u1);
        const float2 p0 = Pack2<__half>::unpack(s0[h][w / 2]), p1 = Pack2<__half>::unpack(s1[h][w / 2]);
        const float f0 = (w & 1) ? p0.y : p0.x, f1 = (w & 1) ? p1.y : p1.x;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816(c, u0[0], u1[0], u0[1], u1[1], qb[j].x, qb[j].y);
          mma16816(c, u0[2], u1[2], u0[3], u1[3], qb[j].z, qb[j].w);
          x[h][j][0] = fmaf(f0, c[0], x[h][j][0]);
          x[h][j][1] = fmaf(f0, c[1], x[h][j][1]);
          x[h][j][2] = fmaf(f1, c[2], x[h][j][2]);
          x[h][j][3] = fmaf(f1, c[3], x[h][j][3]);
        }
      }
    }
    // ---- references: a lane has tokens r, r + 8 of each piece for rows 2 cq, 2 cq + 1 ----
    bool grew = false;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x[h][j][c + 2 * i] *= rs[j][c];
            if constexpr (kMask)
              if (at + 16 * h + r + 8 * i >= lim[j][c]) x[h][j][c + 2 * i] = -INFINITY;
          }
        grew |= fmaxf(fmaxf(x[0][j][c], x[0][j][c + 2]), fmaxf(x[1][j][c], x[1][j][c + 2])) > m[j][c];
      }
    int e;  // exponent field of the tile's largest V scale
    {
      uint32_t v[W / 2], big = 0;
      load_words<W / 2>(base + (lane >> 4) * P::BYTES + P::V_SCALE + (lane & 15) * 2 * W, v);
#pragma unroll
      for (int i = 0; i < W / 2; ++i) big = __vmaxu2(big, v[i] & 0x7fff7fffu);
      e = static_cast<int>(__reduce_max_sync(0xffffffffu, max(big & 0xffffu, big >> 16)) >> 10);
      if (e == 31) {  // infinities and NaNs do not count
        big = 0;
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          const uint32_t u = v[i] & 0x7fff7fffu;
          big = __vmaxu2(big, u & __vcmpltu2(u, 0x7c007c00u));
        }
        e = static_cast<int>(__reduce_max_sync(0xffffffffu, max(big & 0xffffu, big >> 16)) >> 10);
      }
    }
    if (__any_sync(0xffffffffu, grew) || e > v_exp) {
      v_exp = max(v_exp, e);
      const float shift = static_cast<float>(min(12, 26 - v_exp));
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = fmaxf(fmaxf(x[0][j][c], x[0][j][c + 2]), fmaxf(x[1][j][c], x[1][j][c + 2]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          // m is the reference's maximum and the 2^3 that a weight may grow beyond it.
          const bool had = m[j][c] != -INFINITY;
          if (top > m[j][c]) m[j][c] = top + 3.f;
          const float to = m[j][c] == -INFINITY ? 0.f : m[j][c] - 3.f - shift;
          const float f = had ? ex2_approx(mu[j][c] - to) : 1.f;
          mu[j][c] = to;
          l[j][c] *= f;
          accz[j][c] *= f;
#pragma unroll
          for (int g = 0; g < W; ++g) {
            acc[g][0][j][c] *= f;
            acc[g][0][j][c + 2] *= f;
            acc[g][1][j][c] *= f;
            acc[g][1][j][c + 2] *= f;
          }
        }
    }
    // ---- weights and O^T ----
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t *pb = base + h * P::BYTES;
      // Token pairs cq and cq + 4: scales of both tokens per group, zeros of group r % W, codes.
      uint32_t sw[W], s0[W], s1[W];
      load_words<W>(pb + P::v_scale(2 * cq, 0), sw);
#pragma unroll
      for (int g = 0; g < W; ++g) s0[g] = __byte_perm(sw[g / 2], sw[W / 2 + g / 2], (g & 1) ? 0x7632 : 0x5410);
      load_words<W>(pb + P::v_scale(2 * cq + 8, 0), sw);
#pragma unroll
      for (int g = 0; g < W; ++g) s1[g] = __byte_perm(sw[g / 2], sw[W / 2 + g / 2], (g & 1) ? 0x7632 : 0x5410);
      const uint8_t *zp = pb + P::v_zero(2 * cq, r % W);
      uint32_t z0 = *reinterpret_cast<const uint32_t *>(zp), z1 = *reinterpret_cast<const uint32_t *>(zp + 16);
      z0 = fma_half2(pick<W>(s0, r), 0x48004800u, z0);  // z + 8 s
      z1 = fma_half2(pick<W>(s1, r), 0x48004800u, z1);
      const uint8_t *vp = pb + P::V_CODES + cq * D + (r ^ P::swizzle(cq)) * P::CHUNK;
      uint32_t v0[W], v1[W];
      load_words<W>(vp, v0);
      load_words<W>(vp + 4 * D, v1);
      uint32_t b0[NT], b1[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = ex2_approx(x[h][j][i] - mu[j][i & 1]);
          l[j][i & 1] += p[i];
        }
        b0[j] = transpose8(pack_half(p[0], p[1]));
        b1[j] = transpose8(pack_half(p[2], p[3]));
        mma16816(accz[j], z0, 0u, z1, 0u, b0[j], b1[j]);
      }
#pragma unroll
      for (int g = 0; g < W; ++g) {
        const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
        uint32_t u0[4], u1[4];
        spread(__byte_perm(v0[g / 2], v0[W / 2 + g / 2], sel), u0);
        spread(__byte_perm(v1[g / 2], v1[W / 2 + g / 2], sel), u1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // -8 in the two units
          u0[i] = add_half2(u0[i], (i & 1) ? 0x80808080u : 0x80088008u);
          u1[i] = add_half2(u1[i], (i & 1) ? 0x80808080u : 0x80088008u);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint32_t w0 = mul_half2(b0[j], s0[g]), w1 = mul_half2(b1[j], s1[g]);
          mma16816(acc[g][0][j], u0[0], u0[1], u1[0], u1[1], w0, w1);
          mma16816(acc[g][1][j], u0[2], u0[3], u1[2], u1[3], w0, w1);
          if constexpr (kLow) {  // what the products' rounding left out, exactly
            const uint32_t r0 = fma_half2(b0[j], s0[g], w0 ^ 0x80008000u);
            const uint32_t r1 = fma_half2(b1[j], s1[g], w1 ^ 0x80008000u);
            mma16816(acc[g][0][j], u0[0], u0[1], u1[0], u1[1], r0, r1);
            mma16816(acc[g][1][j], u0[2], u0[3], u1[2], u1[3], r0, r1);
          }
        }
      }
    }
  };

  bool ok = true;
  for (int k = 0; k < sg.count && pl.seen > 0; ++k, ++taken) {
    const uint32_t stage = taken % kStages, bar = smem_u32(&s_bar[warp][stage]), parity = (taken / kStages) & 1;
    if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
      ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, &s_abort, &g_kv4a_status, TLLM_DEV_WAIT_TIMEOUT + SITE_TILE));
    if (!ok) {
      // The copies in flight still write to this CTA's memory: give them their time, then leave.
      for (int i = 0; i < kStages && k + i < sg.count; ++i) {
        const long long since = clock64();
        while (!mbar_try_wait(smem_u32(&s_bar[warp][(taken + i) % kStages]), ((taken + i) / kStages) & 1) &&
               clock64() - since < kWaitLimitCycles) {
        }
      }
      return;
    }
    const int at = (sg.first + k) * kTile;
    uint8_t *base = ring + stage * TILE_BYTES;
    if (at + kTile > lim_all) {
      tile(base, at, std::true_type{});
      fence_proxy_async_smem();  // the tile was written to; a later copy may follow
    } else {
      tile(base, at, std::false_type{});
    }
    __syncwarp();
    if (k + kStages < sg.count) issue(k + kStages, kStages);
  }

  // ---- this segment's results; the next one's copies go out first ----
  const Segment done = sg;
  const int64_t done_pos = pos;
  pos += sg.rest;
  const bool more = next_segment<ROWS, kTile, kExtra>(a, end - pos, sg);
  if (more) prime();
  const bool whole = done.count == done.nt;
  const int64_t slot = 2 * static_cast<int64_t>(worker) + (at_start ? 0 : 1);
  if (!whole && done.first == 0 && lane == 0)
    a.ws_open[worker] = Open{static_cast<int>((done_pos + done.rest - 1) / per) - worker + 1, static_cast<int>(slot),
                             done.hk, done.pl.row0, done.pl.r0, done.pl.nr, 0, 0};
  const float f1 = pow2(24), f2 = pow2(20);  // the units of the two kinds of rows
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = 8 * j + 2 * cq + c;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], off);
      const int rr = done.pl.r0 + row;
      const float inv = 1.f / l[j][c];  // no key: 0 / 0
#pragma unroll
      for (int g = 0; g < W; ++g) {
        const float z = __shfl_sync(0xffffffffu, accz[j][c], 4 * g + cq);
        const float4 v = make_float4(fmaf(acc[g][0][j][c], f1, z), fmaf(acc[g][0][j][c + 2], f2, z),
                                     fmaf(acc[g][1][j][c], f1, z), fmaf(acc[g][1][j][c + 2], f2, z));
        if (row >= done.pl.nr) continue;
        if (whole) {
          T *o = static_cast<T *>(a.o) + (done.pl.row0 + rr / a.G) * a.so0 + (done.hk * a.G + rr % a.G) * a.so1;
          *reinterpret_cast<uint2 *>(o + 32 * g + 4 * r) =
              make_uint2(Pack2<T>::pack(v.x * inv, v.y * inv), Pack2<T>::pack(v.z * inv, v.w * inv));
        } else {
          *reinterpret_cast<float4 *>(a.ws_acc + (slot * ROWS + row) * D + 32 * g + 4 * r) = v;
        }
      }
      if (!whole && r == 0)  // (a sum that is no number counts)
        a.ws_ml[slot * ROWS + row] = make_float2(l[j][c] == 0.f ? -INFINITY : mu[j][c], l[j][c]);
    }
  if (!more) break;
  at_start = false;
  }
}

// A CTA per worker and 8 rows: the row tile that starts in its last segment and goes on in later workers, if
// any. Its first part is in that worker's slot, the others in the first slots of the workers after it.
// A warp adds up a row; each lane weighs one of 32 parts, so the parts' loads do not wait for one
// another, and 8 are in flight. Launched while the main kernel ends, it waits for it first.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256, 1) kv4_merge_kernel(const Args a) {
  constexpr int E = D / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int worker = blockIdx.x, lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int4 *info = reinterpret_cast<const int4 *>(a.ws_open + worker);
  const int4 o0 = info[0], o1 = info[1];
  const Open open = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, 0, 0};
  if (open.workers <= 1 || row >= open.nr) return;
  auto at = [&](int i) { return (i == 0 ? static_cast<int64_t>(open.slot) : 2LL * (worker + i)) * ROWS + row; };
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < open.workers) ml = a.ws_ml[at(lane)];
  float top = ml.x;
  for (int i = lane + 32; i < open.workers; i += 32) top = fmaxf(top, a.ws_ml[at(i)].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  float sum = 0.f, v[E];
#pragma unroll
  for (int d = 0; d < E; ++d) v[d] = 0.f;
  for (int i0 = 0; i0 < open.workers; i0 += 32) {
    if (i0 > 0) ml = i0 + lane < open.workers ? a.ws_ml[at(i0 + lane)] : make_float2(-INFINITY, 0.f);
    const float f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - top);
    sum = fmaf(ml.y, f, sum);
    const int n = min(32, open.workers - i0);
    for (int i1 = 0; i1 < n; i1 += kMergeLoads) {
      uint32_t x[kMergeLoads][E];
#pragma unroll
      for (int i = 0; i < kMergeLoads; ++i) {
        if (i1 + i < n) {
          const uint8_t *acc = reinterpret_cast<const uint8_t *>(a.ws_acc + at(i0 + i1 + i) * D + lane * E);
          load_words<E>(acc, x[i]);
        } else {
#pragma unroll
          for (int d = 0; d < E; ++d) x[i][d] = 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < kMergeLoads; ++i) {
        const float fi = __shfl_sync(0xffffffffu, f, (i1 + i) & 31);  // (0 past the last part)
#pragma unroll
        for (int d = 0; d < E; ++d) v[d] = fmaf(__uint_as_float(x[i][d]), fi, v[d]);
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  const int rr = open.r0 + row;
  T *o = static_cast<T *>(a.o) + (open.row0 + rr / a.G) * a.so0 + (open.hk * a.G + rr % a.G) * a.so1 + lane * E;
#pragma unroll
  for (int d = 0; d < E; d += 2) *reinterpret_cast<uint32_t *>(o + d) = Pack2<T>::pack(v[d] / sum, v[d + 1] / sum);
}

struct Plan {
  int nt = 1, n_rt = 1, ctas = 0;  // nt: 8-row tiles of a row tile, 0 for the prefill kernel
  int workers = 0;
  size_t ml_at = 0, acc_at = 0, ws_bytes = 0;
};

// Row tiles of 8 rows where all of a sequence's rows fit one, else of 16, and the prefill kernel above
// kSplitRows rows; one wave of CTAs, fewer where they would not all have tiles.
Plan make_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t max_new, int64_t D, int64_t block_size,
               int64_t max_blocks) {
  Plan p;
  const int64_t rows = std::max<int64_t>(max_new, 1) * (Hq / Hkv);
  p.nt = rows <= 8 ? 1 : (rows <= kSplitRows ? 2 : 0);
  const int row_tile = p.nt > 0 ? 8 * p.nt : kPrefillRows, tile = p.nt > 0 ? kTile : 128;
  p.n_rt = static_cast<int>((rows + row_tile - 1) / row_tile);
  const int64_t sms = sm_count() > 0 ? sm_count() : 148;
  const int64_t most = B * p.n_rt * Hkv * std::max<int64_t>((max_blocks * block_size + tile - 1) / tile, 1);
  const int64_t each = p.nt > 0 ? kWarps * kMinTiles : 1;  // a CTA's least run
  p.ctas = static_cast<int>(std::max<int64_t>(1, std::min(p.nt > 0 ? resident(p.nt) * sms : sms, (most + each - 1) / each)));
  p.workers = p.ctas * (p.nt > 0 ? kWarps : 1);
  const size_t workers = static_cast<size_t>(p.workers), rows_all = 2 * workers * row_tile;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  p.ml_at = up(workers * sizeof(Open));
  p.acc_at = up(p.ml_at + rows_all * sizeof(float2));
  p.ws_bytes = p.acc_at + rows_all * D * sizeof(float);
  return p;
}

template <typename T, int D, int ROWS>
int launch_merge(const Args &a, cudaStream_t st) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.workers, ROWS / 8);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kv4_merge_kernel<T, D, ROWS>, a), "paged kv4 attention merge launch");
}

template <typename T, int D, int NT>
int launch(const Args &a, cudaStream_t st) {
  auto kern = kv4_split_kernel<T, D, NT>;
  constexpr int smem = kWarps * (kStages * 2 * Piece<D>::BYTES + NT * Piece<D>::W * 512);
  KernelLaunchInfo info;
  int rc = prepare_kernel(reinterpret_cast<const void *>(kern), smem, kThreads, 1, &info);
  if (rc) return rc;
  kern<<<a.workers / kWarps, kThreads, smem, st>>>(a);
  rc = cuda_status(cudaGetLastError(), "paged kv4 attention launch");
  return rc ? rc : launch_merge<T, D, 8 * NT>(a, st);
}

template <typename T, int D>
int launch_nt(const Args &a, int nt, int dtype, cudaStream_t st) {
  if (nt == 1) return launch<T, D, 1>(a, st);
  if (nt == 2) return launch<T, D, 2>(a, st);
  const int rc = launch_prefill(a, D, dtype, st);
  return rc ? rc : launch_merge<T, D, kPrefillRows>(a, st);
}

template <typename T>
int launch_d(const Args &a, int64_t D, int nt, int dtype, cudaStream_t st) {
  return D == 64 ? launch_nt<T, 64>(a, nt, dtype, st) : launch_nt<T, 128>(a, nt, dtype, st);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace kv4
}  // namespace tllm

extern "C" size_t tllm_paged_kv4_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                                                     int64_t max_new, int64_t D, int64_t block_size,
                                                     int64_t max_blocks) {
  if (B < 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || max_new < 0 || D <= 0 || block_size <= 0 || max_blocks < 0)
    return 0;
  return tllm::kv4::make_plan(B, Hq, Hkv, std::min(max_new, T), D, block_size, max_blocks).ws_bytes;
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
  TLLM_CHECK_ARG(static_cast<int64_t>(pl.n_rt) * Hkv < (1LL << 31), "paged_kv4_attn: problem too large");
  a.n_rt = pl.n_rt;
  a.workers = pl.workers;
  if (!workspace || workspace_bytes < pl.ws_bytes)
    return fail(TLLM_ERR_WORKSPACE, "paged_kv4_attn: workspace of %zu bytes needed, %zu given", pl.ws_bytes,
                workspace_bytes);
  TLLM_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
                 "paged_kv4_attn: workspace must be 256-byte aligned");
  char *ws = static_cast<char *>(workspace);
  a.ws_open = reinterpret_cast<Open *>(ws);
  a.ws_ml = reinterpret_cast<float2 *>(ws + pl.ml_at);
  a.ws_acc = reinterpret_cast<float *>(ws + pl.acc_at);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == TLLM_DTYPE_F16 ? launch_d<__half>(a, D, pl.nt, dtype, st) : launch_d<__nv_bfloat16>(a, D, pl.nt, dtype, st);
}
