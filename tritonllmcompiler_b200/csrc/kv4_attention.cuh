// What the kernels of attention over the 4-bit paged cache share: arguments, the line of key tiles
// and its division among workers, and packed fp16 arithmetic.
#pragma once

#include <cuda_fp16.h>
#include <stddef.h>
#include <stdint.h>

#include "common.h"
#include "kv4.cuh"
#include "ptx.cuh"

namespace tllm {
namespace kv4 {

constexpr float kLog2e = 1.4426950408889634f;

// A row tile of several workers: rows [r0, r0 + nr) of the sequence that starts at row0.
struct __align__(16) Open {
  int workers, slot, hk, row0;  // workers 0: none; the first part's slot
  int r0, nr, pad0, pad1;
};

struct Args {
  const void *q;
  const uint8_t *cache;
  const int32_t *block_tables, *lens, *cu;
  void *o;
  // Partial results: two slots per worker (its first segment, its last), and per worker the row tile
  // that starts in its last segment and goes on in the next workers.
  Open *ws_open;    // [workers]
  float2 *ws_ml;    // [slots][rows of a tile]: reference in log2 units, sum
  float *ws_acc;    // [slots][rows of a tile][D]
  int64_t sq0, sq1, so0, so1, sblk, shead, sbt0, sbt1;
  int64_t T, num_blocks, max_blocks;
  int B, Hkv, G, log2_bs, causal, max_new;
  int n_rt, workers;  // row tiles per sequence and KV head; how many share the line
  float scale_log2;
};

// A row tile: rows r0 .. r0 + nr of the n_q * G rows of sequence b and a KV head hk, row r being new
// token r / G of query head hk * G + r % G, and how many keys they see.
struct Place {
  int b, rt, r0, nr, row0, n_q, len, seen;
};

__device__ __forceinline__ int row_keys(const Args &a, const Place &p, int r) {
  return a.causal ? min(max(p.len - p.n_q + r / a.G + 1, 0), p.len) : p.len;
}

template <int ROWS>
__device__ __forceinline__ bool locate(const Args &a, int b, int rt, Place &p) {
  p.b = b;
  p.rt = rt;
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

// Key tiles of a row tile; one where its rows see nothing, so that somebody writes them.
template <int TILE>
__device__ __forceinline__ int key_tiles(const Place &p) {
  return max((p.seen + TILE - 1) / TILE, 1);
}

// All key tiles of all row tiles form one line: sequences, in them row tiles of ROWS rows, in them KV
// heads, in them tiles of TILE keys. Each worker takes an equal run of it (within a tile), whatever
// the lengths are; a run's parts of one row tile are its segments.
struct Segment {
  Place pl;
  int hk, nt;        // KV head; key tiles of the row tile
  int first, count;  // the segment's key tiles
};

template <int THREADS, int WPC>
struct LineScan {
  int64_t warp[THREADS / 32];
  int64_t off[WPC];  // tiles before the run's start in its sequence
  int seq[WPC];
};

template <int ROWS, int TILE>
__device__ __forceinline__ int64_t tiles_of_sequence(const Args &a, int b, int *status) {
  int64_t t = 0;
  Place p;
  for (int rt = 0; rt < a.n_rt && locate<ROWS>(a, b, rt, p); ++rt) t += key_tiles<TILE>(p);
  if (p.n_q > a.max_new) atomicCAS(status, 0, TLLM_DEV_BAD_INDEX);
  return t * a.Hkv;
}

// Finds the runs of the CTA's WPC workers: a scan over the sequences, done by every CTA, so that it
// needs no launch of its own. All threads; leaves with the CTA synchronised.
template <int ROWS, int TILE, int THREADS, int WPC>
__device__ __forceinline__ void scan_line(const Args &a, LineScan<THREADS, WPC> &s, int min_tiles, int64_t &per,
                                          int64_t &total, int *status) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int share = (a.B + THREADS - 1) / THREADS;
  const int b0 = min(tid * share, a.B), b1 = min(b0 + share, a.B);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles_of_sequence<ROWS, TILE>(a, b, status);
  int64_t upto = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += u;
  }
  if (lane == 31) s.warp[warp] = upto;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) upto += s.warp[w];
    total += s.warp[w];
  }
  per = max((total + a.workers - 1) / a.workers, static_cast<int64_t>(min_tiles));
  for (int w = 0; w < WPC; ++w) {
    int64_t off = (static_cast<int64_t>(blockIdx.x) * WPC + w) * per - (upto - mine);
    if (off < 0 || off >= mine) continue;
    for (int b = b0; b < b1; ++b) {
      const int64_t t = tiles_of_sequence<ROWS, TILE>(a, b, status);
      if (off < t) {
        s.seq[w] = b;
        s.off[w] = off;
        break;
      }
      off -= t;
    }
  }
  __syncthreads();
}

// The segment that starts `off` tiles into sequence b; false past the last sequence, which cannot
// be while lengths stay as they were scanned.
template <int ROWS, int TILE>
__device__ __forceinline__ bool first_segment(const Args &a, int b, int64_t off, int64_t left, Segment &g) {
  for (int rt = 0; b < a.B;) {
    if (locate<ROWS>(a, b, rt, g.pl)) {
      g.nt = key_tiles<TILE>(g.pl);
      if (off < static_cast<int64_t>(g.nt) * a.Hkv) {
        g.hk = static_cast<int>(off / g.nt);
        g.first = static_cast<int>(off % g.nt);
        g.count = static_cast<int>(min(static_cast<int64_t>(g.nt - g.first), left));
        return true;
      }
      off -= static_cast<int64_t>(g.nt) * a.Hkv;
    }
    if (++rt == a.n_rt) {
      rt = 0;
      ++b;
    }
  }
  return false;
}

template <int ROWS, int TILE>
__device__ __forceinline__ bool next_segment(const Args &a, int64_t left, Segment &g) {
  if (left <= 0) return false;
  g.first = 0;
  if (++g.hk == a.Hkv) {
    g.hk = 0;
    int b = g.pl.b, rt = g.pl.rt;
    do {
      if (++rt == a.n_rt) {
        rt = 0;
        ++b;
      }
      if (b >= a.B) return false;
    } while (!locate<ROWS>(a, b, rt, g.pl));
    g.nt = key_tiles<TILE>(g.pl);
  }
  g.count = static_cast<int>(min(static_cast<int64_t>(g.nt), left));
  return true;
}

// Rows that belong to no sequence are cleared, by all threads of the grid.
template <typename T, int D>
__device__ __forceinline__ void clear_rows(const Args &a) {
  const int64_t from = a.B > 0 ? min(max(static_cast<int64_t>(__ldg(a.cu + a.B)), int64_t{0}), a.T) : 0;
  const int hq = a.Hkv * a.G;
  const int64_t n = (a.T - from) * hq * (D / 8), step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += step) {
    const int64_t row = i / (D / 8);
    T *o = static_cast<T *>(a.o) + (from + row / hq) * a.so0 + (row % hq) * a.so1;
    *reinterpret_cast<uint4 *>(o + (i % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) { return Pack2<__half>::pack(a, b); }

__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma_half2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t add_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t sub_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 .. 127

template <int N>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[N]) {
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

// Launches the kernel for many query rows per KV head (kv4_prefill.cu): row tiles of kPrefillRows
// rows, a CTA a worker.
constexpr int kPrefillRows = 128;
int launch_prefill(const Args &a, int64_t D, int dtype, cudaStream_t st);

}  // namespace kv4
}  // namespace tllm
