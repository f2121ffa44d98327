// Layout of the 4-bit paged KV cache, shared by the kernels that write, read back and attend
// over it.
//
// A block (page) of one KV head is block_size / 16 pieces of 16 tokens, 20 * D bytes each and
// contiguous: one bulk copy brings everything attention needs of those tokens. Groups of 32
// channels of one token share a scale and a zero (fp16): value = code * scale + zero (a scale that is NaN: a group without numbers).
//   [ 0 D,  8 D)  K codes, D / 2 bytes per token. The 32-bit word [lane 4][w D / 32] holds channels
//                 32 w + 8 lane + j, channel j at bits 4 (j / 2) + 16 (j % 2): lane c of a quad
//                 reads its codes of all groups in one vector, and a mask of two nibbles at
//                 the same place of both halves gives two neighbouring channels of an MMA operand.
//   [ 8 D,  9 D)  K scales [token][group]
//   [ 9 D, 10 D)  K zeros [token][group]
//   [10 D, 18 D)  V codes, D bytes per pair of tokens: 8 chunks of D / 8 bytes, at place
//                 n ^ swizzle(pair) the chunk of channels 32 g + 4 n + j of every group g, 16 bits per
//                 group with channel j at bits 4 j, first token then second. The swizzle spreads the
//                 pairs that a quad of lanes reads at once over the shared-memory banks.
//   [18 D, 19 D)  V scales [token][group]
//   [19 D, 20 D)  V zeros [group][token]
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace tllm {
namespace kv4 {

constexpr int kGroup = 32;
constexpr int kPieceTokens = 16;

template <int D>
struct Piece {
  static_assert(D == 64 || D == 128, "head dim");
  static constexpr int W = D / kGroup;  // groups per token
  static constexpr int BYTES = 20 * D;
  static constexpr int K_CODES = 0;
  static constexpr int K_SCALE = 8 * D;
  static constexpr int K_ZERO = 9 * D;
  static constexpr int V_CODES = 10 * D;
  static constexpr int V_SCALE = 18 * D;
  static constexpr int V_ZERO = 19 * D;
  static constexpr int CHUNK = D / 8;  // bytes of a V chunk: two tokens
  static __host__ __device__ constexpr int swizzle(int pair) {
    return D == 128 ? 2 * (pair & 3) : 4 * ((pair >> 1) & 1);
  }
  // Word of channels [8 x, 8 x + 8) of token t.
  static __host__ __device__ constexpr int k_word(int t, int x) {
    return K_CODES + t * (D / 2) + 4 * ((x & 3) * W + (x >> 2));
  }
  // The 16 bits of channels [32 g + 4 n, + 4) of token t.
  static __host__ __device__ constexpr int v_bits(int t, int g, int n) {
    return V_CODES + (t >> 1) * D + (n ^ swizzle(t >> 1)) * CHUNK + (t & 1) * (CHUNK / 2) + 2 * g;
  }
  static __host__ __device__ constexpr int k_scale(int t, int g) { return K_SCALE + 2 * (t * W + g); }
  static __host__ __device__ constexpr int k_zero(int t, int g) { return K_ZERO + 2 * (t * W + g); }
  static __host__ __device__ constexpr int v_scale(int t, int g) { return V_SCALE + 2 * (t * W + g); }
  static __host__ __device__ constexpr int v_zero(int t, int g) { return V_ZERO + 2 * (g * 16 + t); }
};

}  // namespace kv4
}  // namespace tllm
