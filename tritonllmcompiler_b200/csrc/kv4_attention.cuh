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

// A row tile: rows r0 .. r0 + nr of the n_q * G rows of sequence b (of those of its first max_new tokens, where it
// has more) and a KV head hk, row r being new token r / G of query head hk * G + r % G, and how many keys they see.
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
  p.nr = min(ROWS, min(p.n_q, a.max_new) * a.G - p.r0);
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
// heads, in them EXTRA places for what a row tile costs besides its keys (queries, results, the way
// there) and then tiles of TILE keys. Each worker takes an equal run of it (within a place), whatever the
// lengths are; a run's parts of one row tile are its segments.
struct Segment {
  Place pl;
  int hk, nt;        // KV head; key tiles of the row tile
  int first, count;  // the segment's key tiles
  int rest;          // places from the segment's start to the end of the row tile
};

template <int THREADS, int WPC>
struct LineScan {
  int64_t warp[THREADS / 32];
  int64_t off[WPC];  // places before the run's start in its row tile (of all KV heads)
  int seq[WPC], rt[WPC];
};

// Finds the runs of the CTA's WPC workers: a scan over all sequences' row tiles, done by every CTA, so that
// it needs no launch of its own (a thread per row tile: per sequence, 16 row tiles in turn took 4 us). All
// threads; leaves with the CTA synchronised. Returns whether some sequence has more than max_new tokens.
template <int ROWS, int TILE, int EXTRA, int THREADS, int WPC>
__device__ __forceinline__ bool scan_line(const Args &a, LineScan<THREADS, WPC> &s, int min_tiles, int64_t &per,
                                          int64_t &total, int *status) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t n = static_cast<int64_t>(a.B) * a.n_rt, share = (n + THREADS - 1) / THREADS;
  const int64_t i0 = min(tid * share, n);
  const int count = static_cast<int>(min(share, n - i0)), first_b = static_cast<int>(i0 / a.n_rt);
  const int first_rt = static_cast<int>(i0 - static_cast<int64_t>(first_b) * a.n_rt);
  bool over = false;
  // Calls visit(b, rt, places) for this thread's row tiles until it returns false.
  auto each = [&](auto visit) {
    int b = first_b, rt = first_rt;
    for (int i = 0; i < count; ++i) {
      Place p;
      const int64_t places = locate<ROWS>(a, b, rt, p) ? static_cast<int64_t>(key_tiles<TILE>(p) + EXTRA) * a.Hkv : 0;
      if (rt == 0 && p.n_q > a.max_new) {
        atomicCAS(status, 0, TLLM_DEV_BAD_INDEX);
        over = true;
      }
      if (!visit(b, rt, places)) return;
      if (++rt == a.n_rt) {
        rt = 0;
        ++b;
      }
    }
  };
  int64_t mine = 0;
  each([&](int, int, int64_t places) {
    mine += places;
    return true;
  });
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
    each([&](int b, int rt, int64_t places) {
      if (off < places) {
        s.seq[w] = b;
        s.rt[w] = rt;
        s.off[w] = off;
        return false;
      }
      off -= places;
      return true;
    });
  }
  return __syncthreads_or(over);
}

// The segment that starts `off` places into row tile rt of sequence b; false if the run ends before its keys
// (the next worker has them all), or if there is none (not while lengths stay as they were scanned).
template <int ROWS, int TILE, int EXTRA>
__device__ __forceinline__ bool first_segment(const Args &a, int b, int rt, int64_t off, int64_t left, Segment &g) {
  if (!locate<ROWS>(a, b, rt, g.pl)) return false;
  g.nt = key_tiles<TILE>(g.pl);
  const int places = g.nt + EXTRA;
  g.hk = static_cast<int>(off / places);
  if (g.hk >= a.Hkv) return false;
  const int at = static_cast<int>(off % places);
  g.first = max(at - EXTRA, 0);
  g.rest = places - at;
  g.count = static_cast<int>(min(static_cast<int64_t>(g.nt - g.first), left - max(EXTRA - at, 0)));
  return g.count > 0;
}

template <int ROWS, int TILE, int EXTRA>
__device__ __forceinline__ bool next_segment(const Args &a, int64_t left, Segment &g) {
  left -= EXTRA;
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
  g.rest = g.nt + EXTRA;
  g.count = static_cast<int>(min(static_cast<int64_t>(g.nt), left));
  return true;
}

// Rows from .. to - 1 of the output become `bits`, by threads i0, i0 + step, ...
template <typename T, int D>
__device__ __forceinline__ void fill_rows(const Args &a, int64_t from, int64_t to, uint32_t bits, int64_t i0, int64_t step) {
  const int hq = a.Hkv * a.G;
  const int64_t n = (to - from) * hq * (D / 8);
  for (int64_t i = i0; i < n; i += step) {
    const int64_t row = i / (D / 8);
    T *o = static_cast<T *>(a.o) + (from + row / hq) * a.so0 + (row % hq) * a.so1;
    *reinterpret_cast<uint4 *>(o + (i % (D / 8)) * 8) = make_uint4(bits, bits, bits, bits);
  }
}

// The rows that no row tile has, by all threads of the grid: those before the first sequence and past the last
// one become zeros, and (over: there are some) those of tokens past a sequence's first max_new NaN.
template <typename T, int D>
__device__ __forceinline__ void other_rows(const Args &a, bool over) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  auto row = [&](int b) { return min(max(static_cast<int64_t>(__ldg(a.cu + b)), int64_t{0}), a.T); };
  fill_rows<T, D>(a, a.B > 0 ? row(a.B) : 0, a.T, 0u, i0, step);
  if (a.B > 0) fill_rows<T, D>(a, 0, row(0), 0u, i0, step);
  if (over)
    for (int b = blockIdx.x; b < a.B; b += gridDim.x)
      fill_rows<T, D>(a, row(b) + a.max_new, row(b + 1), 0x7fff7fffu, threadIdx.x, blockDim.x);
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
