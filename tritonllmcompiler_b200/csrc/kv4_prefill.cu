// Attention over the 4-bit paged cache for many query rows per KV head (prefill chunks): tcgen05 on
// tiles of 128 query rows and 128 keys, the keys and values brought to fp16 on the way.
//
// A worker of the line (kv4_attention.cuh) is a CTA, one per SM; row tiles have 128 rows, key tiles
// 128 keys. Work goes through rings:
//   warp 17       copies: the tile's pages, K and V of one head, by bulk copies into the raw ring
//   warps 8-15    unpack, a piece of 16 tokens each: code * scale + zero in fp16 (11 bits: an error of
//                 2^-12 of a value against the half step of 1/30 of its group's range that 4 bits
//                 cost), stored swizzled as the K and V operands
//   warp 16       TMEM allocation and the lane that issues the UMMAs: S = Q K^T into one of two TMEM
//                 buffers (the next tile's overlaps this tile's softmax), O += P V with P from TMEM
//   warps 0-7     two threads per query row, 64 keys of a tile each: q to fp16 (bf16 rows by a power of
//                 two that keeps them in its range), softmax with a lazy rescale of O (2^8), results
// K, V and the weights are fp16 operands, rounded once each (2^-12 of a value, 2^-12 of a weight). With fp16 outputs
// that doubles the error of rounding the output alone, and scores are off by some 2^-12 of their spread: by 0.005 where
// they have a standard deviation of 29 (K of size 8, q of size 4). bf16 outputs do not show it.
// V's columns are stored in the order 0 4 1 5 2 6 3 7 of every eight channels (the order in which one
// mask yields pairs) and put right where O is read. The V rows of a last tile past the context are
// zeros. A V group whose scale, zero or largest value (15 s + z) is no fp16 number is stored as zeros too and
// noted in a mask per token, and the rows that see the token get NaN in its channels: a product would spread it to
// rows that do not.
//
// Bound: tensor products, 4 Hq D flops per visible pair, if K and V were 16-bit. They are 4-bit, so each tile
// of 128 keys is unpacked for every 128 rows: 8 requests of up to 512 new tokens in up to 4096, 32 heads over
// 8 of 128, bf16: 177 us, 472 TFLOP/s. A tile takes some 3200 cycles, 2800 of them each for its softmax and,
// beside it, its unpacking; half of the issue slots, 43 % of the integer pipe and a quarter of the tensor
// pipe are busy, so latency between few warps holds it. What was slower on the same requests: part of the powers
// of two by a polynomial (+9 to 15 %), twice the unpacking warps (+15 %), a row's 64 scores in registers at
// once (+6 %), two row tiles a CTA that share a tile's unpacking (+27 %).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "kv4_attention.cuh"

namespace tllm {

__device__ int g_kv4p_status = 0;

int kv4p_read_status(int *out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_kv4p_status, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyFromSymbol(kv4 prefill status)");
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_kv4p_status, &zero, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyToSymbol(kv4 prefill status)");
  *out = v;
  return TLLM_OK;
}

namespace kv4 {
namespace {

constexpr int BM = kPrefillRows;
constexpr int BN = 128;
// Places of the line that a segment's queries, results and empty pipeline take: 13,000 cycles, tiles 3,200 each.
// (8 requests of up to 512 new tokens in up to 4096, from a cold L2: none 224 us, 2 196, 3 190, 4 184, 5 183.)
constexpr int kExtra = 4;
constexpr int kPieces = BN / kPieceTokens;
constexpr int kRowThreads = 256;  // two per query row
constexpr int kHalf = BN / 2;     // keys of a tile per thread of a row
constexpr int kUnpackWarps = 8;
constexpr int kRawStages = 3;     // tiles of the cache on their way or being unpacked (shared memory holds no more)
constexpr int kUmmaWarp = 16, kCopyWarp = 17;
constexpr int kThreads = 18 * 32;
static_assert(kUnpackWarps == kPieces, "a piece of a tile per unpacking warp");
constexpr int TMEM_COLS = 512;
constexpr int O_COL = 256;  // S buffers at columns [0, 128) and [128, 256)
constexpr int P_COL = 384;  // P buffers at columns [384, 448) and [448, 512)
constexpr float kLazyRescaleLog2 = 8.0f;
// Weights are 2^(x + 7 - m): with the 2^8 that x may grow beyond m they stay within fp16, and those of 2^-21 of the
// largest keep their 11 bits (without the 2^7, many keys of such weights beside one of weight 1 lost 4 % and more of
// their sum). Beyond kHuge the 7 would be rounded.
constexpr float kWeightLog2 = 7.0f;
constexpr float kHuge = 1048576.f;
__device__ __forceinline__ float weight_shift(float m) {
  return m == -INFINITY ? 0.f : (fabsf(m) < kHuge ? kWeightLog2 : 0.f) - m;
}

enum : int {
  SITE_Q = 0x51,
  SITE_RAWFULL = 0x52,
  SITE_RAWEMPTY = 0x53,
  SITE_KFULL = 0x54,
  SITE_KEMPTY = 0x55,
  SITE_VFULL = 0x56,
  SITE_VEMPTY = 0x57,
  SITE_SFULL = 0x58,
  SITE_PFULL = 0x59,
  SITE_PVDONE = 0x5a,
  SITE_OFREE = 0x5b,
  SITE_SEMPTY = 0x5c,
  SITE_PAIR = 0x5d,
};

template <int D>
struct Geo {
  static constexpr int CHUNKS = D * 2 / 128;  // 128-byte swizzle spans per row
  static constexpr int CHUNK_BYTES = BM * 128;
  static constexpr int TILE_BYTES = CHUNKS * CHUNK_BYTES;
  static constexpr int RAW_BYTES = kPieces * Piece<D>::BYTES;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = TILE_BYTES;
  static constexpr int V_OFF = K_OFF + 2 * TILE_BYTES;
  static constexpr int RAW_OFF = V_OFF + 2 * TILE_BYTES;
  static constexpr int BAD_OFF = RAW_OFF + kRawStages * RAW_BYTES;  // [2][BN] bytes: groups of V without numbers
  static constexpr int ANY_OFF = BAD_OFF + 2 * BN;         // [2][kUnpackWarps] bytes: any in the piece
  static constexpr int MAX_OFF = ANY_OFF + 2 * kUnpackWarps;  // [2][2][BM] floats between a row's threads
  static constexpr int BAR_OFF = MAX_OFF + 4 * BM * 4;
  static constexpr int SMEM_BYTES = BAR_OFF + 256 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024 && BAR_OFF % 8 == 0, "shared memory plan");
};

constexpr uint32_t kSwizzle128 = 2;

// Descriptors of a tile's k-steps differ from the first one's by a constant in the address field (the
// issuing lane is on the critical path). Q, K: 16 channels of a row; V: 16 rows.
__device__ __forceinline__ uint64_t kmajor_base(uint32_t base) { return make_sdesc(base, 16, 8 * 128, kSwizzle128); }
template <int D>
__device__ __forceinline__ constexpr uint64_t kmajor_step(int k) {
  return static_cast<uint64_t>(((k / 4) * Geo<D>::CHUNK_BYTES + (k % 4) * 32) >> 4);
}
template <int D>
__device__ __forceinline__ uint64_t vmajor_base(uint32_t base) {
  return make_sdesc(base, Geo<D>::CHUNK_BYTES, 8 * 128, kSwizzle128);
}
constexpr uint64_t kVmajorStep = (16 * 128) >> 4;

// Byte of 16-byte unit u (of 8 per 128-byte span) of a tile's row.
__device__ __forceinline__ int unit_at(int row, int u) { return row * 128 + ((u ^ (row & 7)) << 4); }

// One half of a word in both (the compiler takes it as an operand's modifier).
__device__ __forceinline__ uint32_t twice(uint32_t v, bool high) {
  const __half2 h = *reinterpret_cast<const __half2 *>(&v);
  const __half2 r = high ? __high2half2(h) : __low2half2(h);
  return *reinterpret_cast<const uint32_t *>(&r);
}

// The 8 codes of a word (4 in each half) to fp16 values code * s + z; x[i] holds the codes at bits 4 i of
// both halves. A code c under the exponent of 1024 is 1024 + c (or 1024 + 16 c); the difference is exact.
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t s, uint32_t z, uint32_t (&x)[4]) {
  constexpr uint32_t kExp = 0x64006400u;
  const uint32_t hi = __byte_perm(w, 0u, 0x4341);  // the upper bytes of the halves
  x[0] = add_half2((w & 0x000f000fu) | kExp, 0xe400e400u);                     // - 1024
  x[1] = fma_half2((w & 0x00f000f0u) | kExp, 0x2c002c00u, 0xd400d400u);        // / 16 - 64
  x[2] = add_half2((hi & 0x000f000fu) | kExp, 0xe400e400u);
  x[3] = fma_half2((hi & 0x00f000f0u) | kExp, 0x2c002c00u, 0xd400d400u);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fma_half2(x[i], s, z);
}

constexpr uint32_t kFifteen = 0x4b804b80u;  // the largest code, in fp16
// Pieces in which a V scale or zero has at least this size (2184) have their groups looked at one by one: below
// it, 15 s + z is less than 16 * 2184 and a number. (Each lane over all its groups in registers, eight times
// the code: 199 us where a lane per group, through shared memory, takes 184 on the requests above.)
constexpr uint32_t kLook = 0x6844u;

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) kv4_prefill_kernel(const Args a) {
  using P = Piece<D>;
  using G = Geo<D>;
  constexpr int W = P::W;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + G::BAR_OFF);
  uint64_t *q_full = bars + 0;
  uint64_t *k_full = bars + 1;     // [2]
  uint64_t *k_empty = bars + 3;    // [2]
  uint64_t *v_full = bars + 5;     // [2]
  uint64_t *v_empty = bars + 7;    // [2]
  uint64_t *s_full = bars + 9;     // [2]
  // (Two, as of all barriers with a phase per tile: a phase must not pass unseen, and the next tile's
  // weights can be complete before this tile's wait has looked.)
  uint64_t *p_full = bars + 11;    // [2]
  uint64_t *pv_done = bars + 13;   // [2], as s_full by the tile's parity
  uint64_t *o_free = bars + 15;
  uint64_t *s_empty = bars + 16;   // [2]
  uint64_t *pair = bars + 18;      // [4]
  uint64_t *raw_full = bars + 22;                // [kRawStages]
  uint64_t *raw_empty = raw_full + kRawStages;   // [kRawStages]
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(raw_empty + kRawStages);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
  __shared__ LineScan<kThreads, 1> s_line;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(q_full), kRowThreads);
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&k_full[s]), kUnpackWarps);
      mbar_init(smem_u32(&k_empty[s]), 1);
      mbar_init(smem_u32(&v_full[s]), kUnpackWarps);
      mbar_init(smem_u32(&v_empty[s]), 1);
      mbar_init(smem_u32(&s_full[s]), 1);
      mbar_init(smem_u32(&s_empty[s]), kRowThreads);
      mbar_init(smem_u32(&p_full[s]), kRowThreads);
      mbar_init(smem_u32(&pv_done[s]), 1);
    }
    for (int s = 0; s < kRawStages; ++s) {
      mbar_init(smem_u32(&raw_full[s]), 1);
      mbar_init(smem_u32(&raw_empty[s]), kUnpackWarps);
    }
    for (int s = 0; s < 4; ++s) mbar_init(smem_u32(&pair[s]), 64);
    mbar_init(smem_u32(o_free), kRowThreads);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kUmmaWarp) {
    tmem_alloc(smem_u32(tmem_holder), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  int64_t per, total;
  const bool over = scan_line<BM, BN, kExtra>(a, s_line, 1, per, total, &g_kv4p_status);  // (synchronises the CTA)
  tc_fence_after();
  other_rows<T, D>(a, over);
  const uint32_t tmem_base = *tmem_holder;
  const uint32_t sQ = smem_u32(smem + G::Q_OFF);
  const uint32_t sK = smem_u32(smem + G::K_OFF);
  const uint32_t sV = smem_u32(smem + G::V_OFF);
  const int worker = blockIdx.x;
  int64_t pos = worker * per;
  const int64_t end = min(pos + per, total);
  if (threadIdx.x == 0) a.ws_open[worker].workers = 0;

  // Every role walks the same segments; `it` counts the key tiles of all of them.
  Segment sg;
  bool more = pos < end && first_segment<BM, BN, kExtra>(a, s_line.seq[0], s_line.rt[0], s_line.off[0], end - pos, sg);
  auto advance = [&] {
    pos += sg.rest;
    more = next_segment<BM, BN, kExtra>(a, end - pos, sg);
  };
  auto tiles = [&] { return sg.pl.seen > 0 ? sg.count : 0; };
  auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
    return mbar_wait(smem_u32(bar), parity, abort_flag, &g_kv4p_status, TLLM_DEV_WAIT_TIMEOUT + site);
  };

  if (warp >= 8 && warp < 8 + kUnpackWarps) {
    // ------------------------------ unpacking ------------------------------
    const int piece = warp - 8;
    bool ok = true;
    uint32_t it = 0;
    for (; more && ok; advance()) {
      const int n = tiles();
      for (int j = 0; j < n; ++j, ++it) {
        const uint32_t st = it & 1, empty = ((it >> 1) & 1) ^ 1, rst = it % kRawStages;
        // Tokens of this warp's piece that are keys (the others were not loaded, or hold anything).
        const int valid = min(max(sg.pl.seen - (sg.first + j) * BN - piece * kPieceTokens, 0), kPieceTokens);
        uint8_t *raw = smem + G::RAW_OFF + rst * G::RAW_BYTES + piece * P::BYTES;
        ok = __all_sync(0xffffffffu, wait(&raw_full[rst], (it / kRawStages) & 1, SITE_RAWFULL) && wait(&k_empty[st], empty, SITE_KEMPTY));
        if (!ok) break;
        if (valid > 0) {
          uint8_t *tile = smem + G::K_OFF + st * G::TILE_BYTES;
          const int cq = lane & 3;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // Eight lanes of one store phase: four units of rows t and t + 4, apart in the swizzle.
            const int t = half * 8 + ((lane >> 2) & 1) * 4 + (lane >> 3), row = piece * kPieceTokens + t;
            uint32_t code[W], sc[W / 2], ze[W / 2];
            load_words<W>(raw + P::K_CODES + t * (D / 2) + cq * (4 * W), code);
            load_words<W / 2>(raw + P::k_scale(t, 0), sc);
            load_words<W / 2>(raw + P::k_zero(t, 0), ze);
#pragma unroll
            for (int w = 0; w < W; ++w) {
              uint32_t x[4];
              unpack_word(code[w], twice(sc[w / 2], w & 1), twice(ze[w / 2], w & 1), x);
              *reinterpret_cast<uint4 *>(tile + (w / 2) * G::CHUNK_BYTES + unit_at(row, 4 * (w & 1) + cq)) =
                  make_uint4(x[0], x[1], x[2], x[3]);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&k_full[st]));

        ok = __all_sync(0xffffffffu, wait(&v_empty[st], empty, SITE_VEMPTY));
        if (!ok) break;
        {
          uint8_t *tile = smem + G::V_OFF + st * G::TILE_BYTES;
          const int m = lane & 3;  // channels 32 g + 8 m + {0..7}
          const int pr = ((lane >> 2) & 1) * 2 + ((lane >> 3) & 1) + ((lane >> 4) & 1) * 4;
          uint32_t c0[W], c1[W], sc[W], ze[W];  // [token][two groups a word], [token][..], zeros [group]: two tokens
          const uint8_t *vp = raw + P::V_CODES + pr * D + ((2 * m) ^ P::swizzle(pr)) * P::CHUNK;
          load_words<W>(vp, c0);
          load_words<W>(vp + P::CHUNK, c1);
          load_words<W>(raw + P::v_scale(2 * pr, 0), sc);
          uint32_t big = 0;
#pragma unroll
          for (int g = 0; g < W; ++g) {
            ze[g] = *reinterpret_cast<const uint32_t *>(raw + P::v_zero(2 * pr, g));
            big = __vmaxu2(big, __vmaxu2(sc[g] & 0x7fff7fffu, ze[g] & 0x7fff7fffu));
          }
          // Tokens past the last key, or some value that is no number: zeros, and a note of the latter.
          uint32_t bad = 0;  // bits g: token 2 pr, bits 8 + g: the next one
          const bool odd = valid < kPieceTokens || max(big & 0xffffu, big >> 16) >= kLook;
          const bool any_odd = __any_sync(0xffffffffu, odd);
          if (any_odd) {
            __syncwarp();
            if (m < W) {  // of the lanes that share two tokens, each looks at a group
#pragma unroll 1
              for (int e = 0; e < 2; ++e) {
                uint16_t *sp = reinterpret_cast<uint16_t *>(raw + P::v_scale(2 * pr + e, m));
                uint16_t *zp = reinterpret_cast<uint16_t *>(raw + P::v_zero(2 * pr + e, m));
                const uint32_t top = fma_half2(*sp, kFifteen, *zp);
                const bool past = 2 * pr + e >= valid;
                const bool none = (*zp & 0x7fffu) >= 0x7c00u || (top & 0x7fffu) >= 0x7c00u;
                if (!past && none) bad |= 1u << (8 * e + m);
                if (past || none) *sp = *zp = 0;
              }
            }
            bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
            bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
            __syncwarp();
            load_words<W>(raw + P::v_scale(2 * pr, 0), sc);
#pragma unroll
            for (int g = 0; g < W; ++g) ze[g] = *reinterpret_cast<const uint32_t *>(raw + P::v_zero(2 * pr, g));
          }
#pragma unroll
          for (int g = 0; g < W; ++g) {
            const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
            const int unit = 4 * (g & 1) + m, row = piece * kPieceTokens + 2 * pr;
            uint8_t *chunk = tile + (g / 2) * G::CHUNK_BYTES;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t x[4];
              unpack_word(__byte_perm(c0[e * (W / 2) + g / 2], c1[e * (W / 2) + g / 2], sel),
                          twice(sc[e * (W / 2) + g / 2], g & 1), twice(ze[g], e), x);
              *reinterpret_cast<uint4 *>(chunk + unit_at(row + e, unit)) = make_uint4(x[0], x[1], x[2], x[3]);
            }
          }
          const bool any = any_odd && __any_sync(0xffffffffu, bad != 0);
          if (any && m == 0)
            *reinterpret_cast<uint16_t *>(smem + G::BAD_OFF + st * BN + piece * kPieceTokens + 2 * pr) = static_cast<uint16_t>(bad);
          if (lane == 0) smem[G::ANY_OFF + st * kUnpackWarps + piece] = any;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&v_full[st]));
          mbar_arrive(smem_u32(&raw_empty[rst]));
        }
      }
    }
  } else if (warp >= 8) {
    if (warp == kCopyWarp) {
      // ------------------------------ copies ------------------------------
      const int per_page = (1 << a.log2_bs) / kPieceTokens;
      bool ok = true;
      uint32_t it = 0;
      for (; more && ok; advance()) {
        const int n = tiles();
        const int32_t *bt = a.block_tables + sg.pl.b * a.sbt0;
        // Lane i: page i of a tile, read one tile ahead.
        auto page_of = [&](int j) -> int {
          const int tok = (sg.first + j) * BN + (lane << a.log2_bs);
          if (j >= n || (lane << a.log2_bs) >= BN || tok >= sg.pl.seen) return -1;
          const int p = __ldg(bt + static_cast<int64_t>(tok >> a.log2_bs) * a.sbt1);
          if (p >= 0 && p < a.num_blocks) return p;
          atomicCAS(&g_kv4p_status, 0, TLLM_DEV_BAD_INDEX);
          return 0;
        };
        int page = page_of(0);
        for (int j = 0; j < n; ++j, ++it) {
          const uint32_t st = it % kRawStages;
          const int here = page;
          page = page_of(j + 1);
          ok = __all_sync(0xffffffffu, wait(&raw_empty[st], ((it / kRawStages) & 1) ^ 1, SITE_RAWEMPTY));
          if (!ok) break;
          const int pieces = min((sg.pl.seen - (sg.first + j) * BN + kPieceTokens - 1) / kPieceTokens, kPieces);
          const uint32_t bar = smem_u32(&raw_full[st]);
          if (lane == 0) mbar_arrive_expect_tx(bar, pieces * P::BYTES);
          __syncwarp();
          if (here >= 0) {
            const int at = lane * per_page;  // the page's first piece in the tile
            bulk_load(smem_u32(smem + G::RAW_OFF) + st * G::RAW_BYTES + at * P::BYTES,
                      a.cache + static_cast<int64_t>(here) * a.sblk + sg.hk * a.shead,
                      min(per_page, pieces - at) * P::BYTES, bar);
          }
        }
      }
      if (!ok) {
        // The copies in flight still write to this CTA's memory: give them their time.
        for (uint32_t i = it > kRawStages ? it - kRawStages : 0; i < it; ++i) {
          const long long since = clock64();
          while (!mbar_try_wait(smem_u32(&raw_full[i % kRawStages]), (i / kRawStages) & 1) && clock64() - since < kWaitLimitCycles) {
          }
        }
      }
    } else if (lane == 0) {
      // ------------------------------ UMMAs ------------------------------
      const uint32_t idesc_qk = make_idesc_f16(BM, BN, false, false, false);
      const uint32_t idesc_pv = make_idesc_f16(BM, D, false, false, true);
      bool ok = true;
      uint32_t it = 0, seg = 0;
      for (; more && ok; advance()) {
        const int n = tiles();
        if (n == 0) continue;
        auto issue_qk = [&](uint32_t i) {
          const uint64_t qd = kmajor_base(sQ), kd = kmajor_base(sK + (i & 1) * G::TILE_BYTES);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_f16_ss(tmem_base + (i & 1) * BN, qd + kmajor_step<D>(k), kd + kmajor_step<D>(k), idesc_qk,
                        k != 0 ? 1u : 0u);
          umma_commit(smem_u32(&s_full[i & 1]));
          umma_commit(smem_u32(&k_empty[i & 1]));
        };
        auto next_qk = [&](uint32_t i) {
          ok = wait(&k_full[i & 1], (i >> 1) & 1, SITE_KFULL) && wait(&s_empty[i & 1], ((i >> 1) & 1) ^ 1, SITE_SEMPTY);
          if (!ok) return;
          tc_fence_after();
          issue_qk(i);
        };
        ok = wait(q_full, seg & 1, SITE_Q);
        for (int j = 0; j < 2 && j < n && ok; ++j) next_qk(it + j);
        for (int j = 0; j < n && ok; ++j, ++it) {
          const uint32_t st = it & 1;
          ok = (j > 0 || seg == 0 || wait(o_free, (seg - 1) & 1, SITE_OFREE)) &&
               wait(&v_full[st], (it >> 1) & 1, SITE_VFULL) && wait(&p_full[st], (it >> 1) & 1, SITE_PFULL);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = vmajor_base<D>(sV + st * G::TILE_BYTES);
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            umma_f16_ts(tmem_base + O_COL, tmem_base + P_COL + st * kHalf + k * 8, vd + k * kVmajorStep, idesc_pv,
                        (j | k) != 0 ? 1u : 0u);
          umma_commit(smem_u32(&v_empty[st]));
          umma_commit(smem_u32(&pv_done[st]));
          if (j + 2 < n) next_qk(it + 2);
        }
        ++seg;
      }
    }
  } else {
    // ------------------------------ rows ------------------------------
    const int quad = warp & 3, half = warp >> 2;  // TMEM lanes 32 quad ..., keys 64 half ...
    const int row = quad * 32 + lane;             // = TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t o_tm = tmem_base + lane_off + O_COL;
    float *s_max = reinterpret_cast<float *>(smem + G::MAX_OFF);
    // A number from each of the row's two threads to the other: warps quad and quad + 4 meet. (On a
    // barrier whose wait is bounded; after one that gave up, the next wait for work leaves.)
    uint32_t meets = 0;
    auto other = [&](float v) -> float {
      float *at = s_max + (meets & 1) * 2 * BM;
      at[half * BM + row] = v;
      mbar_arrive(smem_u32(&pair[quad]));
      wait(&pair[quad], meets & 1, SITE_PAIR);
      ++meets;
      return at[(half ^ 1) * BM + row];
    };
    // A scale of 0 is a zero q (a hidden score is -infinity, which a factor of 0 would spoil).
    const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
    const float sign = a.scale_log2 > 0.f ? 1.f : (a.scale_log2 < 0.f ? -1.f : 0.f);
    // Brings this thread's half of the segment's q row into shared memory; returns the factor of its scores.
    constexpr int kUnits = D / 16;
    auto load_q = [&]() -> float {
      uint4 raw[kUnits];
      const bool in = row < sg.pl.nr;
      const int rr = sg.pl.r0 + row;
      const T *q = static_cast<const T *>(a.q) + (sg.pl.row0 + rr / a.G) * a.sq0 + (sg.hk * a.G + rr % a.G) * a.sq1 + half * (D / 2);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) raw[u] = in ? __ldg(reinterpret_cast<const uint4 *>(q) + u) : make_uint4(0, 0, 0, 0);
      float up = sign, down = scale;
      if constexpr (kBF16) {
        uint32_t big = 0;  // the exponents of bf16 are those of fp32: the largest magnitude's top bits
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          big = __vmaxu2(big, __vmaxu2(raw[u].x & 0x7fff7fffu, raw[u].y & 0x7fff7fffu));
          big = __vmaxu2(big, __vmaxu2(raw[u].z & 0x7fff7fffu, raw[u].w & 0x7fff7fffu));
        }
        const int mine = static_cast<int>(max(big & 0xffffu, big >> 16) >> 7) - 127;
        const int e = max(max(mine, static_cast<int>(other(static_cast<float>(mine)))), -100);
        up = pow2(12 - e) * sign;
        down = pow2(e) * (scale / 4096.f);
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Pack2<T>::unpack(w[i]);
          w[i] = pack_half(f.x * up, f.y * up);
        }
        const int at = half * kUnits + u;
        *reinterpret_cast<uint4 *>(smem + G::Q_OFF + (at / 8) * G::CHUNK_BYTES + unit_at(row, at % 8)) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
      fence_proxy_async_smem();
      mbar_arrive(smem_u32(q_full));
      return down;
    };
    bool ok = true, at_start = true;
    uint32_t it = 0;
    float rs = more && tiles() > 0 ? load_q() : 0.f;
    while (more && ok) {
      const int n = tiles();
      // Rows past the last one see all keys, as most others do: hiding costs a warp 800 cycles a tile.
      const int keys = row < sg.pl.nr ? row_keys(a, sg.pl, sg.pl.r0 + row) : sg.pl.seen;
      float m_use = -INFINITY, l_run = 0.f;
      uint32_t bad = 0;  // groups of V without numbers that the row sees
      for (int j = 0; j < n; ++j, ++it) {
        const uint32_t sb = it & 1;
        ok = __all_sync(0xffffffffu, wait(&s_full[sb], (it >> 1) & 1, SITE_SFULL));
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_tm = tmem_base + lane_off + sb * BN, p_tm = tmem_base + lane_off + P_COL + sb * kHalf;
        const int k0 = (sg.first + j) * BN, mine0 = k0 + half * kHalf;
        // 32 scores at a time in registers; the first 32 are read again for their weights.
        uint32_t sr[32];
        auto scores = [&](int c) {
          tmem_ld32(s_tm + half * kHalf + c, sr);
          if (mine0 + c + 32 > keys) {
#pragma unroll
            for (int t = 0; t < 32; ++t)
              if (mine0 + c + t >= keys) sr[t] = __float_as_uint(-INFINITY);
          }
        };
        float mx = -INFINITY;
        ok = __all_sync(0xffffffffu, wait(&v_full[sb], (it >> 1) & 1, SITE_VFULL));  // (for the notes below)
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kHalf; c += 32) {
          scores(c);
          float mx4[4] = {mx, __uint_as_float(sr[0]), __uint_as_float(sr[1]), __uint_as_float(sr[2])};
#pragma unroll
          for (int t = 3; t < 31; t += 2)
            mx4[(t >> 1) & 3] = max3f(mx4[(t >> 1) & 3], __uint_as_float(sr[t]), __uint_as_float(sr[t + 1]));
          mx = max3f(max3f(mx4[0], mx4[1], mx4[2]), mx4[3], __uint_as_float(sr[31]));
        }
        mx = rs * fmaxf(mx, other(mx));
        float alpha = 1.0f;
        bool rescale = false;
        if (m_use == -INFINITY) {
          m_use = mx;  // nothing accumulated yet (every earlier P of this row was 0)
        } else if (mx > m_use + kLazyRescaleLog2) {
          alpha = ex2_approx(weight_shift(mx) - weight_shift(m_use));
          m_use = mx;
          rescale = true;
        }
        const float neg_m = weight_shift(m_use);
        // The exponents below are exact products less the rounded maximum, which is within half an ulp of
        // its own product; where that is a good part of a unit and more, round the products first.
        const bool huge = __any_sync(0xffffffffu, fabsf(m_use) >= kHuge && m_use != -INFINITY);
        const float factor = huge ? 1.f : rs;
        const uint64_t scale2 = f2_pack(factor, factor);
        const uint64_t negm2 = f2_pack(neg_m, neg_m);
        uint64_t ps2[2] = {0ull, 0ull};
#pragma unroll
        for (int c = kHalf - 32; c >= 0; c -= 32) {
          if (c < kHalf - 32) scores(c);
          if (huge) {
#pragma unroll
            for (int t = 0; t < 32; ++t) sr[t] = __float_as_uint(__uint_as_float(sr[t]) * rs);
          }
          uint32_t pk[16];
#pragma unroll
          for (int t = 0; t < 32; t += 2) {
            const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(sr[t]), __uint_as_float(sr[t + 1])), scale2, negm2);
            float x0, x1;
            f2_unpack(x2, x0, x1);
            const float p0 = ex2_approx(x0);
            const float p1 = ex2_approx(x1);
            ps2[(t >> 1) & 1] = f2_add(ps2[(t >> 1) & 1], f2_pack(p0, p1));
            pk[t >> 1] = pack_half(p0, p1);
          }
          tmem_st16(p_tm + (half * kHalf + c) / 2, pk);
        }
        // The scores are read: their buffer may take the next but one tile's.
        tc_fence_before();
        mbar_arrive(smem_u32(&s_empty[sb]));
        float ps[4];
        f2_unpack(ps2[0], ps[0], ps[1]);
        f2_unpack(ps2[1], ps[2], ps[3]);
        l_run = l_run * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
        if (__any_sync(0xffffffffu, rescale)) {
          // O is stable once the previous tile's P V has completed. (Only here, and at the segment's end,
          // are these barriers waited for: two tiles earlier their P V had completed before S came.)
          ok = __all_sync(0xffffffffu, wait(&pv_done[sb ^ 1], ((it - 1) >> 1) & 1, SITE_PVDONE));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
            uint32_t r[32];
            tmem_ld32(o_tm + c, r);
#pragma unroll
            for (int t = 0; t < 32; ++t) r[t] = __float_as_uint(__uint_as_float(r[t]) * alpha);
            tmem_st32(o_tm + c, r);
          }
        }
        // V's groups without numbers: the notes are overwritten only after this tile's P V.
        if (*reinterpret_cast<const volatile uint64_t *>(smem + G::ANY_OFF + sb * kUnpackWarps) != 0) {
#pragma unroll 1
          for (int t = 0; t < BN && k0 + t < keys; ++t)
            if (smem[G::ANY_OFF + sb * kUnpackWarps + t / kPieceTokens]) bad |= smem[G::BAD_OFF + sb * BN + t];
        }
        tc_fence_before();
        mbar_arrive(smem_u32(&p_full[sb]));
      }
      if (!ok) break;
      // ---- the next segment's q goes in first: this one's products with Q are complete ----
      const Segment done = sg;
      const int64_t done_pos = pos;
      const float done_l = l_run + other(l_run);
      advance();
      if (more && tiles() > 0) rs = load_q();
      // ---- results: this thread's half of the channels ----
      if (n > 0) {
        ok = __all_sync(0xffffffffu, wait(&pv_done[(it - 1) & 1], ((it - 1) >> 1) & 1, SITE_PVDONE));
        if (!ok) break;
        tc_fence_after();
      }
      const bool whole = done.count == done.nt, in = row < done.pl.nr;
      const int64_t slot = (2 * static_cast<int64_t>(worker) + (at_start ? 0 : 1)) * BM + row;
      const int rr = done.pl.r0 + row;
      const float inv = 1.f / done_l;  // no key: 0 / 0
      T *o = static_cast<T *>(a.o) + (done.pl.row0 + rr / a.G) * a.so0 + (done.hk * a.G + rr % a.G) * a.so1;
#pragma unroll 1
      for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
        uint32_t r[32];
        if (n > 0) {
          tmem_ld32(o_tm + c, r);
        } else {
#pragma unroll
          for (int t = 0; t < 32; ++t) r[t] = 0u;
        }
        if (bad & (1u << (c / 32))) {
#pragma unroll
          for (int t = 0; t < 32; ++t) r[t] = 0x7fc00000u;  // NaN
        }
        if (!in) continue;
#pragma unroll
        for (int t = 0; t < 32; t += 8) {
          float v[8];  // columns 2 i + h hold channels i + 4 h
#pragma unroll
          for (int i = 0; i < 8; ++i) v[(i >> 1) + 4 * (i & 1)] = __uint_as_float(r[t + i]);
          if (whole) {
            uint4 pk;
            pk.x = Pack2<T>::pack(v[0] * inv, v[1] * inv);
            pk.y = Pack2<T>::pack(v[2] * inv, v[3] * inv);
            pk.z = Pack2<T>::pack(v[4] * inv, v[5] * inv);
            pk.w = Pack2<T>::pack(v[6] * inv, v[7] * inv);
            *reinterpret_cast<uint4 *>(o + c + t) = pk;
          } else {
            float4 *p = reinterpret_cast<float4 *>(a.ws_acc + slot * D + c + t);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      if (n > 0) {
        tc_fence_before();
        mbar_arrive(smem_u32(o_free));
      }
      if (!whole && in && half == 0)
        a.ws_ml[slot] = make_float2(done_l == 0.f ? -INFINITY : -weight_shift(m_use), done_l);
      if (!whole && done.first == 0 && threadIdx.x == 0)
        a.ws_open[worker] = Open{static_cast<int>((done_pos + done.rest - 1) / per) - worker + 1,
                                 2 * worker + (at_start ? 0 : 1), done.hk, done.pl.row0, done.pl.r0, done.pl.nr, 0, 0};
      at_start = false;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kUmmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <typename T, int D>
int launch(const Args &a, cudaStream_t st) {
  auto kern = kv4_prefill_kernel<T, D>;
  KernelLaunchInfo info;
  const int rc = prepare_kernel(reinterpret_cast<const void *>(kern), Geo<D>::SMEM_BYTES, kThreads, 1, &info);
  if (rc) return rc;
  kern<<<a.workers, kThreads, Geo<D>::SMEM_BYTES, st>>>(a);
  return cuda_status(cudaGetLastError(), "paged kv4 prefill launch");
}

}  // namespace

int launch_prefill(const Args &a, int64_t D, int dtype, cudaStream_t st) {
  if (dtype == TLLM_DTYPE_F16) return D == 64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
  return D == 64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
}

}  // namespace kv4
}  // namespace tllm
