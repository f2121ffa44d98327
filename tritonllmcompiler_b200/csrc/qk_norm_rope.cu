// RMS norm of every query and key head with the rotation by positions of several axes in the
// same pass, and its backward pass.
//
// With r = 1 / sqrt(mean(x^2) + eps) and y = x r w, the rotary pair i (of D / 2) of token t turns
// by the angle of row pos[a(i)][t], column i of the cos/sin tables:
//   z_i = y_i c - y_{i+D/2} s,  z_{i+D/2} = y_{i+D/2} c + y_i s.
// Backward, with dy = the rotation of dz by the opposite angle and g = dy w:
//   dx = r (g - x r^2 mean(g x)),  dw = sum over the rows of dy x r.
// Everything is fp32 from the loaded values to one rounding at the store. (rmsnorm_rope rounds y
// before the rotation, as the operator it replaces does; that is not repeated here.)
//
// Bound: HBM, 2 x 2 bytes an element forward and 3 x 2 backward. A row of D elements belongs to
// D / 16 consecutive lanes, each with one 16-byte vector of each half, so a pair never leaves its
// thread and the row sums take log2(D / 16) shuffles. A lane group takes R heads of one token in
// turn, so positions, cos and sin are read once for R rows, and all R rows are requested before
// the first is used. From a cold L2, 40 heads of 128: 16,384 tokens 72 us, 4.7 TB/s forward; 8192 tokens
// 64 us, 4.0 TB/s backward (two heads a group: more spill, and three blocks per SM instead of two
// took 91 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.h"
#include "ptx.cuh"
#include "rmsnorm_rope.cuh"

namespace tllm {

__device__ int g_qknr_status = 0;

int qknr_read_status(int *out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_qknr_status, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyFromSymbol(qk norm rope status)");
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_qknr_status, &zero, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyToSymbol(qk norm rope status)");
  *out = v;
  return TLLM_OK;
}

namespace qknr {
namespace {

using namespace rr;

constexpr int kThreads = 256;

// One of the two tensors (queries or keys).
struct Part {
  const void *x;   // [T, H, D], strides sxt, sxh
  const void *w;   // [D]
  void *out;       // forward: z; backward: dx (strides sot, soh)
  const void *dz;  // backward (strides sdt, sdh)
  int64_t sxt, sxh, sot, soh, sdt, sdh;
  int H;
};

struct Args {
  Part part[2];
  const float *cos, *sin;
  const int32_t *pos;  // [axes, T], stride spos between axes
  int64_t scos, ssin, spos;
  uint32_t axis[4];  // axis of each rotary pair, 2 bits each
  int64_t T;
  int64_t rope_rows;
  float eps;
  float *ws;  // backward: [blocks][D] partial sums of dw, the queries' blocks first
  void *dw[2];
  int blocks[2];
};

// cos and sin of the 8 rotary pairs c .. c + 7 of token t. One vector load each where the pairs
// have one axis, as with sections that are multiples of 8; a load per pair otherwise.
__device__ __forceinline__ void load_turn(const Args &a, int64_t t, int c, float (&cs)[8],
                                          float (&sn)[8]) {
  const uint32_t ax = (a.axis[c >> 4] >> ((2 * c) & 31)) & 0xffffu;
  auto row_of = [&](uint32_t axis) -> int64_t {
    const int p = __ldg(a.pos + axis * a.spos + t);
    if (p >= 0 && p < a.rope_rows) return p;
    atomicCAS(&g_qknr_status, 0, TLLM_DEV_BAD_INDEX);
    return 0;
  };
  if (ax == (ax & 3u) * 0x5555u) {
    const int64_t row = row_of(ax & 3u);
    const float4 *cp = reinterpret_cast<const float4 *>(a.cos + row * a.scos + c);
    const float4 *sp = reinterpret_cast<const float4 *>(a.sin + row * a.ssin + c);
    const float4 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
    cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w;
    cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
    sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w;
    sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t row = row_of((ax >> (2 * i)) & 3u);
      cs[i] = __ldg(a.cos + row * a.scos + c + i);
      sn[i] = __ldg(a.sin + row * a.ssin + c + i);
    }
  }
}

template <int TPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = TPR / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

template <typename T, int D, int R>
__global__ void __launch_bounds__(kThreads, 2) qk_norm_rope_kernel(const Args a, uint32_t groups) {
  constexpr int TPR = D / 16;
  constexpr int HALF = D / 2;
  // A group past the end recomputes the last one (the row sums shuffle) and stores nothing.
  const uint32_t raw = (blockIdx.x * kThreads + threadIdx.x) / TPR;
  const bool valid = raw < groups;
  const uint32_t gi = valid ? raw : groups - 1;
  const int c = static_cast<int>(threadIdx.x % TPR) * 8;
  const uint32_t gq = a.part[0].H / R, per = gq + a.part[1].H / R;
  const int64_t t = gi / per;
  const uint32_t at = gi % per;
  const Part &p = a.part[at < gq ? 0 : 1];
  const int h0 = (at < gq ? at : at - gq) * R;
  const T *x = static_cast<const T *>(p.x) + t * p.sxt + h0 * p.sxh + c;
  uint4 x1r[R], x2r[R];
#pragma unroll
  for (int u = 0; u < R; ++u) {
    x1r[u] = ld_stream(x + u * p.sxh);
    x2r[u] = ld_stream(x + u * p.sxh + HALF);
  }
  float cs[8], sn[8], w1[8], w2[8];
  load_turn(a, t, c, cs, sn);
  load8<T>(static_cast<const T *>(p.w) + c, w1);
  load8<T>(static_cast<const T *>(p.w) + HALF + c, w2);
  T *o = static_cast<T *>(p.out) + t * p.sot + h0 * p.soh + c;
#pragma unroll
  for (int u = 0; u < R; ++u) {
    float x1[8], x2[8];
    unpack8<T>(x1r[u], x1);
    unpack8<T>(x2r[u], x2);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x1[i], x1[i], fmaf(x2[i], x2[i], ss));
    const float r = rsqrtf(row_sum<TPR>(ss) * (1.0f / D) + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y1 = x1[i] * r * w1[i], y2 = x2[i] * r * w2[i];
      x1[i] = y1 * cs[i] - y2 * sn[i];
      x2[i] = y2 * cs[i] + y1 * sn[i];
    }
    if (valid) {
      st_stream(o + u * p.soh, pack8<T>(x1));
      st_stream(o + u * p.soh + HALF, pack8<T>(x2));
    }
  }
}

// Blocks [0, blocks[0]) take the queries' rows and the rest the keys'. Each lane group walks its
// part's (token, R heads) groups in a fixed stride, keeping its 16 columns of dw in registers; a
// block adds its groups up in shared memory in a fixed order and stores one row of partial sums,
// which dw_kernel adds up in block order, so dw does not depend on timing.
template <typename T, int D, int R>
__global__ void __launch_bounds__(kThreads, 2) qk_norm_rope_bwd_kernel(const Args a) {
  constexpr int TPR = D / 16;
  constexpr int HALF = D / 2;
  constexpr int NG = kThreads / TPR;  // lane groups of a block
  __shared__ float s_dw[kThreads / 32][D];
  const int which = blockIdx.x < a.blocks[0] ? 0 : 1;
  const Part &p = a.part[which];
  const int block = static_cast<int>(blockIdx.x) - (which ? a.blocks[0] : 0);
  const int c = static_cast<int>(threadIdx.x % TPR) * 8;
  const uint32_t per = p.H / R;
  const int64_t groups = a.T * per;
  const int64_t step = static_cast<int64_t>(a.blocks[which]) * NG;
  float w1[8], w2[8], dw1[8], dw2[8];
  load8<T>(static_cast<const T *>(p.w) + c, w1);
  load8<T>(static_cast<const T *>(p.w) + HALF + c, w2);
#pragma unroll
  for (int i = 0; i < 8; ++i) dw1[i] = dw2[i] = 0.f;
  // All lane groups of a warp make the same number of turns (the row sums shuffle over full
  // warps); a group past the end computes its part's last rows and counts and stores nothing.
  for (int64_t base = static_cast<int64_t>(block) * NG; base < groups; base += step) {
    const int64_t raw = base + threadIdx.x / TPR;
    const bool valid = raw < groups;
    const uint32_t gi = static_cast<uint32_t>(valid ? raw : groups - 1);
    const int64_t t = gi / per;
    const int h0 = static_cast<int>(gi % per) * R;
    const T *x = static_cast<const T *>(p.x) + t * p.sxt + h0 * p.sxh + c;
    const T *dz = static_cast<const T *>(p.dz) + t * p.sdt + h0 * p.sdh + c;
    uint4 x1r[R], x2r[R], d1r[R], d2r[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      x1r[u] = ld_stream(x + u * p.sxh);
      x2r[u] = ld_stream(x + u * p.sxh + HALF);
      d1r[u] = ld_stream(dz + u * p.sdh);
      d2r[u] = ld_stream(dz + u * p.sdh + HALF);
    }
    float cs[8], sn[8];
    load_turn(a, t, c, cs, sn);
    T *o = static_cast<T *>(p.out) + t * p.sot + h0 * p.soh + c;
#pragma unroll
    for (int u = 0; u < R; ++u) {
      float x1[8], x2[8], d1[8], d2[8];
      unpack8<T>(x1r[u], x1);
      unpack8<T>(x2r[u], x2);
      unpack8<T>(d1r[u], d1);
      unpack8<T>(d2r[u], d2);
      float ss = 0.f, gx = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss = fmaf(x1[i], x1[i], fmaf(x2[i], x2[i], ss));
        const float y1 = d1[i] * cs[i] + d2[i] * sn[i];
        const float y2 = d2[i] * cs[i] - d1[i] * sn[i];
        d1[i] = y1;
        d2[i] = y2;
        gx = fmaf(y1 * w1[i], x1[i], fmaf(y2 * w2[i], x2[i], gx));
      }
      ss = row_sum<TPR>(ss);
      gx = row_sum<TPR>(gx);
      const float r = rsqrtf(ss * (1.0f / D) + a.eps);
      const float k = r * r * (gx * (1.0f / D));
      if (valid) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dw1[i] = fmaf(d1[i], x1[i] * r, dw1[i]);
          dw2[i] = fmaf(d2[i], x2[i] * r, dw2[i]);
          x1[i] = r * (d1[i] * w1[i] - x1[i] * k);
          x2[i] = r * (d2[i] * w2[i] - x2[i] * k);
        }
        st_stream(o + u * p.soh, pack8<T>(x1));
        st_stream(o + u * p.soh + HALF, pack8<T>(x2));
      }
    }
  }
  // The groups of a warp, then the warps of the block.
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int off = TPR; off < 32; off <<= 1) {
      dw1[i] += __shfl_xor_sync(0xffffffffu, dw1[i], off);
      dw2[i] += __shfl_xor_sync(0xffffffffu, dw2[i], off);
    }
    if (lane < TPR) {
      s_dw[warp][c + i] = dw1[i];
      s_dw[warp][HALF + c + i] = dw2[i];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int wi = 0; wi < kThreads / 32; ++wi) v += s_dw[wi][d];
    a.ws[static_cast<int64_t>(blockIdx.x) * D + d] = v;
  }
}

// 16 columns of one part's dw: 16 threads a column add every 16th block's partial sum.
template <typename T>
__global__ void __launch_bounds__(kThreads) dw_kernel(const Args a, int D) {
  __shared__ float s[16][17];
  const int which = blockIdx.y;
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const float *ws = a.ws + (which ? static_cast<int64_t>(a.blocks[0]) * D : 0) + blockIdx.x * 16 + col;
  float v = 0.f;
#pragma unroll 8
  for (int b = slice; b < a.blocks[which]; b += 16) v += ws[static_cast<int64_t>(b) * D];
  s[slice][col] = v;
  __syncthreads();
  if (slice == 0) {
#pragma unroll
    for (int i = 1; i < 16; ++i) v += s[i][col];
    static_cast<T *>(a.dw[which])[blockIdx.x * 16 + col] = from_f32<T>(v);
  }
}

// The largest R <= most that divides both head counts and still leaves every SM `full` threads.
int heads_per_group(const Args &a, int64_t D, int most, int64_t full) {
  const int64_t sms = sm_count() > 0 ? sm_count() : 148;
  const int64_t lanes = a.T * (a.part[0].H + a.part[1].H) * (D / 16);
  for (int R = most; R > 1; R /= 2)
    if (a.part[0].H % R == 0 && a.part[1].H % R == 0 && lanes >= R * sms * full) return R;
  return 1;
}

template <typename T, int D>
int forward_d(const Args &a, cudaStream_t st) {
  // (16,384 tokens of 40 heads of 128: four heads a lane group 78 us, eight 71.)
  const int R = heads_per_group(a, D, 8, 512);
  const int64_t groups = a.T * ((a.part[0].H + a.part[1].H) / R);
  const unsigned grid = static_cast<unsigned>((groups * (D / 16) + kThreads - 1) / kThreads);
  const uint32_t g = static_cast<uint32_t>(groups);
  if (R == 8) qk_norm_rope_kernel<T, D, 8><<<grid, kThreads, 0, st>>>(a, g);
  else if (R == 4) qk_norm_rope_kernel<T, D, 4><<<grid, kThreads, 0, st>>>(a, g);
  else if (R == 2) qk_norm_rope_kernel<T, D, 2><<<grid, kThreads, 0, st>>>(a, g);
  else qk_norm_rope_kernel<T, D, 1><<<grid, kThreads, 0, st>>>(a, g);
  return cuda_status(cudaGetLastError(), "qk_norm_rope launch");
}

// Blocks of the backward pass: eight per SM at most (four waves; with the two that fit at once, and no
// new ones to start while others end, 8192 tokens took 79 us instead of 65), shared between queries
// and keys by their rows.
void plan_blocks(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int (&blocks)[2]) {
  const int64_t sms = sm_count() > 0 ? sm_count() : 148;
  const int64_t rows[2] = {T * Hq, T * Hkv}, all = rows[0] + rows[1];
  const int64_t groups = kThreads / (D / 16);  // rows a block takes at once
  for (int i = 0; i < 2; ++i) {
    const int64_t share = (8 * sms * rows[i] + all - 1) / std::max<int64_t>(all, 1);
    blocks[i] = static_cast<int>(std::min(share, (rows[i] + groups - 1) / groups));
  }
}

template <typename T, int D>
int backward_d(const Args &a, cudaStream_t st) {
  const int R = heads_per_group(a, D, 2, 512);
  const unsigned grid = a.blocks[0] + a.blocks[1];
  if (grid > 0) {
    if (R == 2) qk_norm_rope_bwd_kernel<T, D, 2><<<grid, kThreads, 0, st>>>(a);
    else qk_norm_rope_bwd_kernel<T, D, 1><<<grid, kThreads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_status(e, "qk_norm_rope backward launch");
  }
  dw_kernel<T><<<dim3(D / 16, 2), kThreads, 0, st>>>(a, D);
  return cuda_status(cudaGetLastError(), "qk_norm_rope weight gradient launch");
}

template <typename T>
int run(const Args &a, int64_t D, bool bwd, cudaStream_t st) {
  switch (D) {
    case 16: return bwd ? backward_d<T, 16>(a, st) : forward_d<T, 16>(a, st);
    case 32: return bwd ? backward_d<T, 32>(a, st) : forward_d<T, 32>(a, st);
    case 64: return bwd ? backward_d<T, 64>(a, st) : forward_d<T, 64>(a, st);
    default: return bwd ? backward_d<T, 128>(a, st) : forward_d<T, 128>(a, st);
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check(const char *op, const Args &a, int64_t Hq, int64_t Hkv, int64_t D, int64_t axes,
          const uint32_t *axis_of_pair, const int64_t *const (&strides)[6], int dtype) {
  TLLM_CHECK_ARG(a.T >= 0 && Hq >= 0 && Hkv >= 0, "%s: negative dimension", op);
  TLLM_CHECK_ARG(D == 16 || D == 32 || D == 64 || D == 128, "%s: head dim %lld not in {16,32,64,128}",
                 op, (long long)D);
  TLLM_CHECK_ARG(dtype == TLLM_DTYPE_F16 || dtype == TLLM_DTYPE_BF16, "%s: unsupported dtype %d", op,
                 dtype);
  TLLM_CHECK_ARG(axes >= 1 && axes <= 4, "%s: %lld position axes not in 1..4", op, (long long)axes);
  TLLM_CHECK_ARG(axis_of_pair, "%s: null pair axes", op);
  for (int i = 0; i < D / 2; ++i)
    TLLM_CHECK_ARG(static_cast<int64_t>((axis_of_pair[i / 16] >> (2 * (i % 16))) & 3u) < axes,
                   "%s: rotary pair %d has no such axis", op, i);
  TLLM_CHECK_ARG(Hq < (1LL << 20) && Hkv < (1LL << 20) && a.T < (1LL << 31) &&
                     a.T * (Hq + Hkv) * (D / 16) < (1LL << 32) - kThreads,
                 "%s: problem too large", op);
  for (const int64_t *s : strides) {
    if (!s) continue;
    TLLM_CHECK_ARG(s[0] % 8 == 0 && s[1] % 8 == 0, "%s: strides must be multiples of 8 elements", op);
  }
  if (a.T * (Hq + Hkv) == 0) return TLLM_OK;
  TLLM_CHECK_ARG(a.cos && a.sin && a.pos, "%s: null table or positions", op);
  TLLM_CHECK_ARG(a.rope_rows >= 1, "%s: empty cos/sin table", op);
  TLLM_CHECK_ARG(a.scos % 4 == 0 && a.ssin % 4 == 0 && aligned16(a.cos) && aligned16(a.sin),
                 "%s: cos/sin rows must be 16-byte aligned", op);
  for (const Part &p : a.part) {
    if (p.H == 0) continue;
    TLLM_CHECK_ARG(p.x && p.w && p.out, "%s: null tensor pointer", op);
    TLLM_CHECK_ARG(aligned16(p.x) && aligned16(p.w) && aligned16(p.out) && aligned16(p.dz),
                   "%s: tensors must be 16-byte aligned", op);
  }
  return TLLM_OK;
}

void fill(Args &a, int64_t T, int64_t Hq, int64_t Hkv, const float *cos, const float *sin,
          const int32_t *positions, int64_t rope_rows, int64_t scos, int64_t ssin, int64_t spos,
          const uint32_t *axis_of_pair, int64_t D, float eps) {
  a.part[0].H = static_cast<int>(Hq);
  a.part[1].H = static_cast<int>(Hkv);
  a.cos = cos;
  a.sin = sin;
  a.pos = positions;
  a.scos = scos;
  a.ssin = ssin;
  a.spos = spos;
  a.T = T;
  a.rope_rows = rope_rows;
  a.eps = eps;
  if (axis_of_pair)
    for (int i = 0; i < (D / 2 + 15) / 16 && i < 4; ++i) a.axis[i] = axis_of_pair[i];
}

}  // namespace
}  // namespace qknr
}  // namespace tllm

extern "C" int tllm_qk_norm_rope(const void *q, const void *k, const void *wq, const void *wk,
                                 const float *cos, const float *sin, const int32_t *positions,
                                 void *q_out, void *k_out, int64_t T, int64_t Hq, int64_t Hkv,
                                 int64_t D, int64_t rope_rows, int64_t scos, int64_t ssin,
                                 int64_t axes, int64_t spos, const uint32_t *axis_of_pair,
                                 const int64_t *sq, const int64_t *sk, const int64_t *sqo,
                                 const int64_t *sko, float eps, int dtype, void *stream) {
  using namespace tllm;
  using namespace tllm::qknr;
  clear_error();
  TLLM_CHECK_ARG(sq && sk && sqo && sko, "qk_norm_rope: null stride array");
  Args a{};
  fill(a, T, Hq, Hkv, cos, sin, positions, rope_rows, scos, ssin, spos, axis_of_pair, D, eps);
  a.part[0] = Part{q, wq, q_out, nullptr, sq[0], sq[1], sqo[0], sqo[1], 0, 0, a.part[0].H};
  a.part[1] = Part{k, wk, k_out, nullptr, sk[0], sk[1], sko[0], sko[1], 0, 0, a.part[1].H};
  const int64_t *const strides[6] = {sq, sk, sqo, sko, nullptr, nullptr};
  const int rc = check("qk_norm_rope", a, Hq, Hkv, D, axes, axis_of_pair, strides, dtype);
  if (rc) return rc;
  if (T * (Hq + Hkv) == 0) return TLLM_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == TLLM_DTYPE_F16 ? run<__half>(a, D, false, st) : run<__nv_bfloat16>(a, D, false, st);
}

extern "C" size_t tllm_qk_norm_rope_bwd_workspace_size(int64_t T, int64_t Hq, int64_t Hkv, int64_t D) {
  if (T <= 0 || Hq < 0 || Hkv < 0 || D < 16 || T * (Hq + Hkv) == 0) return 0;
  int blocks[2];
  tllm::qknr::plan_blocks(T, Hq, Hkv, D, blocks);
  return static_cast<size_t>(blocks[0] + blocks[1]) * D * sizeof(float);
}

extern "C" int tllm_qk_norm_rope_bwd(const void *dq_out, const void *dk_out, const void *q,
                                     const void *k, const void *wq, const void *wk,
                                     const float *cos, const float *sin, const int32_t *positions,
                                     void *dq, void *dk, void *dwq, void *dwk, void *workspace,
                                     size_t workspace_bytes, int64_t T, int64_t Hq, int64_t Hkv,
                                     int64_t D, int64_t rope_rows, int64_t scos, int64_t ssin,
                                     int64_t axes, int64_t spos, const uint32_t *axis_of_pair,
                                     const int64_t *sdqo, const int64_t *sdko, const int64_t *sq,
                                     const int64_t *sk, const int64_t *sdq, const int64_t *sdk,
                                     float eps, int dtype, void *stream) {
  using namespace tllm;
  using namespace tllm::qknr;
  clear_error();
  TLLM_CHECK_ARG(sdqo && sdko && sq && sk && sdq && sdk, "qk_norm_rope_bwd: null stride array");
  Args a{};
  fill(a, T, Hq, Hkv, cos, sin, positions, rope_rows, scos, ssin, spos, axis_of_pair, D, eps);
  a.part[0] = Part{q, wq, dq, dq_out, sq[0], sq[1], sdq[0], sdq[1], sdqo[0], sdqo[1], a.part[0].H};
  a.part[1] = Part{k, wk, dk, dk_out, sk[0], sk[1], sdk[0], sdk[1], sdko[0], sdko[1], a.part[1].H};
  const int64_t *const strides[6] = {sq, sk, sdq, sdk, sdqo, sdko};
  const int rc = check("qk_norm_rope_bwd", a, Hq, Hkv, D, axes, axis_of_pair, strides, dtype);
  if (rc) return rc;
  TLLM_CHECK_ARG(dwq && dwk, "qk_norm_rope_bwd: null weight gradient");
  for (const Part &p : a.part)
    TLLM_CHECK_ARG(p.H == 0 || T == 0 || p.dz, "qk_norm_rope_bwd: null output gradient");
  if (T * (Hq + Hkv) > 0) plan_blocks(T, Hq, Hkv, D, a.blocks);
  const size_t need = tllm_qk_norm_rope_bwd_workspace_size(T, Hq, Hkv, D);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(TLLM_ERR_WORKSPACE, "qk_norm_rope_bwd: workspace of %zu bytes needed, %zu given", need,
                workspace_bytes);
  TLLM_CHECK_ARG(need == 0 || aligned16(workspace), "qk_norm_rope_bwd: workspace must be 16-byte aligned");
  a.ws = static_cast<float *>(workspace);
  a.dw[0] = dwq;
  a.dw[1] = dwk;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == TLLM_DTYPE_F16 ? run<__half>(a, D, true, st) : run<__nv_bfloat16>(a, D, true, st);
}
