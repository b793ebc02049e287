// race_norm.cu -- root-mean-square norm with the residual's addition, its
// backward pass, and its form with 8-bit results.
//
//   h = x + residual;  r = 1 / sqrt(mean(h^2) + eps);  y = h r w
//   g = dy w;  dx = dh + r (g - h r^2 mean(g h));  dw = sum over rows of dy h r
//
// Both passes are bound by memory: forward 3 rows moved (x, residual, h) and
// one written (y, or a quarter to a half of it in 8 bits), backward 3 read and one
// written.  So a row is read once and held in registers between its sum and its
// use: a warp holds up to 1024 columns (32 values a lane), wider rows are
// spread over 4, 16 or 32 warps of one CTA.  Columns come in spans of 256 for each warp,
// two 8-bit blocks, so a block's maximum never leaves its warp: with vector
// loads a lane holds 8 consecutive columns and half a warp holds a block,
// otherwise (odd widths or strides) lane l holds columns l, l + 32, ... and the
// whole warp holds a block in four of its eight values.
//
// bfloat16 rows are short (1.5 KB at 768 columns), so a warp that loads one, waits,
// sums and stores keeps too few bytes on their way.  The grid is what the SMs
// hold at once and a warp walks rows; with vector loads the next rows are on their way
// before the current one is summed, in registers (forward, one row) or shared
// memory (backward, one or two).  Measured, bfloat16 with residual: 65536 x 768 forward
// 71 us (5.6 TB/s), to 8 bits 61 us (5.8), backward with dweight 82 us (4.9); one row a
// warp and no row ahead took 79, 83 and 112 to 158.  float32 rows are on their way in
// enough registers by themselves; which form takes which rows stands beside the launches,
// with both sides measured (float32 with residual: 65104 x 768 forward 124 us, 6.5 TB/s,
// to 8 bits 101 us, 6.4; 87232 x 768 backward 180 us, 5.9).
#include <algorithm>
#include <atomic>

#include "race_api.h"
#include "race_lowp.cuh"

namespace race {
namespace norm {

using namespace lowp;

struct FwdArgs {
  const void* x; int64_t ldx;
  const void* res; int64_t ldr;
  const void* w; int wbf16;
  void* y; int64_t ldy;
  void* h; int64_t ldh;
  uint8_t* codes; int64_t ldc;
  float* scales; int64_t sr, sb;
  float* rstd;
  int64_t rows; int width;
  float eps;
};

struct BwdArgs {
  const void* dy; int64_t lddy;
  const void* dh; int64_t lddh;
  const void* h; int64_t ldh;
  const void* w; int wbf16;
  const float* rstd;
  void* dx; int64_t lddx;
  float* part;            // [CTAs][width]
  int64_t rows; int width;
};

// column of value i of span s
template <int VEC>
__device__ __forceinline__ int col_of(int s, int lane, int i) {
  return 256 * s + (VEC ? 8 * lane + i : 32 * i + lane);
}

// VEC 0: single elements.  1: vectors, which need every row's base on 16 bytes and
// width % 8 == 0.  2: the same with width % 8 == 4, float32 alone (and a weight of that
// type): the last lane that holds columns holds four.
template <typename T, int VEC>
__device__ __forceinline__ void load_span(const T* row, int s, int lane, int width, float (&v)[8]) {
  if constexpr (VEC) {
    const int c = 256 * s + 8 * lane;
    if (VEC == 1 ? c < width : c + 8 <= width) {
      load8(row + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      if constexpr (VEC == 2 && sizeof(T) == 4) {
        if (c < width) {
          const float4 f = *reinterpret_cast<const float4*>(row + c);
          v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<VEC>(s, lane, i);
      v[i] = c < width ? to_f32(row[c]) : 0.f;
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_span(T* row, int s, int lane, int width, const float (&v)[8]) {
  if constexpr (VEC) {
    const int c = 256 * s + 8 * lane;
    if (VEC == 1 ? c < width : c + 8 <= width) {
      store8(row + c, v);
    } else if constexpr (VEC == 2 && sizeof(T) == 4) {
      if (c < width) *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<VEC>(s, lane, i);
      if (c < width) row[c] = from_f32<T>(v[i]);
    }
  }
}

// A warp's spans of a row as they were loaded: 4 (bfloat16) or 8 registers a span.
template <typename T, int V, int VEC>
struct Raw {
  uint4 u[V][sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* row, int w0, int wpr, int lane, int width) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = 256 * (j * wpr + w0) + 8 * lane;
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; ++q)
        u[j][q] = (VEC == 1 ? c : c + 4 * q) < width ? *reinterpret_cast<const uint4*>(row + c + q * (16 / (int)sizeof(T)))
                            : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void get(int j, float (&v)[8]) const {
    load8(reinterpret_cast<const T*>(&u[j][0]), v);
  }
};

template <int VEC>
__device__ __forceinline__ void load_weight(const void* w, int wbf16, int s, int lane, int width,
                                            float (&v)[8]) {
  if (wbf16)
    load_span<bf16, VEC>(static_cast<const bf16*>(w), s, lane, width, v);
  else
    load_span<float, VEC>(static_cast<const float*>(w), s, lane, width, v);
}

__device__ __forceinline__ float warp_sum(float a) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  return a;
}

// Sum over the WPR warps of a row, in the order of the warps.  `slot` alternates
// between calls, so that one barrier serves each.
template <int WPR>
__device__ __forceinline__ float row_sum(float a, float (*slot)[32], int which) {
  a = warp_sum(a);
  if constexpr (WPR > 1) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[which][warp] = a;
    __syncthreads();
    a = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) a += slot[which][i];
  }
  return a;
}

constexpr int threads_of(int wpr) { return wpr == 1 ? 128 : 32 * wpr; }

// WALK: whether a row's warps go on to further rows.
template <typename T, int VEC, int V, int WPR, bool Q, bool WALK>
__global__ void __launch_bounds__(threads_of(WPR), WPR == 32 && !VEC && Q ? 1 : 0) k_rms_fwd(const FwdArgs a) {
  __shared__ float slot[2][32];
  constexpr int RPC = threads_of(WPR) / (32 * WPR);
  constexpr bool AHEAD = WALK && VEC && V * sizeof(T) <= 8;   // the next row waits in registers
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w0 = warp % WPR;
  const int64_t step = (int64_t)gridDim.x * RPC;
  int64_t row = (int64_t)blockIdx.x * RPC + warp / WPR;     // the same for a row's warps
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.res);
  Raw<T, V, VEC> nx, nr;
  if (AHEAD && row < a.rows) {
    nx.load(x + row * a.ldx, w0, WPR, lane, a.width);
    if (res != nullptr) nr.load(res + row * a.ldr, w0, WPR, lane, a.width);
  }
  int which = 0;
  for (; row < a.rows; row = WALK ? row + step : a.rows) {
    float h[V][8];
    if constexpr (AHEAD) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        nx.get(j, h[j]);
        if (res != nullptr) {
          float t[8];
          nr.get(j, t);
#pragma unroll
          for (int i = 0; i < 8; ++i) h[j][i] += t[i];
        }
      }
      if (row + step < a.rows) {
        nx.load(x + (row + step) * a.ldx, w0, WPR, lane, a.width);
        if (res != nullptr) nr.load(res + (row + step) * a.ldr, w0, WPR, lane, a.width);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) load_span<T, VEC>(x + row * a.ldx, j * WPR + w0, lane, a.width, h[j]);
      if (res != nullptr) {
        // single elements of one row: all of the residual's on their way before the first is added
        constexpr int G = WALK || VEC || WPR == 32 ? 1 : V;
#pragma unroll
        for (int j0 = 0; j0 < V; j0 += G) {
          float t[G][8];
#pragma unroll
          for (int j = 0; j < G; ++j) load_span<T, VEC>(res + row * a.ldr, (j0 + j) * WPR + w0, lane, a.width, t[j]);
#pragma unroll
          for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) h[j0 + j][i] += t[j][i];
        }
      }
    }
    if (res != nullptr) {
      T* o = static_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
      for (int j = 0; j < V; ++j) store_span<T, VEC>(o, j * WPR + w0, lane, a.width, h[j]);
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(h[j][i], h[j][i], ss);
    ss = row_sum<WPR>(ss, slot, which);
    which ^= 1;
    const float rs = 1.f / sqrtf(ss / (float)a.width + a.eps);
    if (a.rstd != nullptr && lane == 0 && w0 == 0) a.rstd[row] = rs;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int s = j * WPR + w0;
      if (256 * s >= a.width) break;           // the same for the whole warp
      float w[8];
      load_weight<VEC>(a.w, a.wbf16, s, lane, a.width, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] = h[j][i] * rs * w[i];
      if constexpr (!Q) {
        store_span<T, VEC>(static_cast<T*>(a.y) + row * a.ldy, s, lane, a.width, h[j]);
      } else {
        uint8_t* c = a.codes + row * a.ldc;
        float* sc = a.scales + row * a.sr;
        if constexpr (VEC) {
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) m = max(m, mag(h[j][i]));
          const float sv = scale_of(max_over(m, 16));
          const int c0 = 256 * s + 8 * lane;
          // columns past the width hold zeros; the pitch is a multiple of 16
          if (c0 < ((a.width + 15) & ~15)) {
            *reinterpret_cast<uint2*>(c + c0) = code8(h[j], 1.f / sv);
            if ((lane & 15) == 0) sc[(2 * s + (lane >> 4)) * a.sb] = sv;
          }
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = max(m, mag(h[j][4 * b + i]));
            const float sv = scale_of(max_over(m, 32));
            const float inv = 1.f / sv;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int cc = col_of<0>(s, lane, 4 * b + i);
              // the row's pitch is a multiple of 16: the rest of its last 16 bytes is zeroed
              if (cc < ((a.width + 15) & ~15))
                c[cc] = (uint8_t)code2(h[j][4 * b + i] * inv, 0.f);
            }
            if (lane == 0 && 256 * s + 128 * b < a.width) sc[(2 * s + b) * a.sb] = sv;
          }
        }
      }
    }
  }
}

// The CTA of the backward pass: eight warps where a warp holds a row, so that few
// partial sums of dweight remain.
constexpr int bwd_threads(int wpr) { return wpr == 1 ? 256 : 32 * wpr; }
// The staged form (can_stage says where): the three rows wait in shared memory, STAGES
// rows deep, each lane copying and reading its own 16 bytes (so no barrier): one row
// ahead in registers took 171 of them at three spans and left 8 warps an SM.
template <typename T, int V, int WPR>
struct Staged {
  static constexpr int PART = (int)sizeof(T) / 2 * 512;          // bytes of a warp's span: 16 or 32 a lane
  static constexpr int ROW = 3 * V * PART;
  static constexpr int STAGES = ROW <= 4608 ? 3 : 2;
  static constexpr int WARPS = bwd_threads(WPR) / 32;
  static constexpr int BYTES = WARPS * STAGES * ROW;
  static constexpr int FIT = 225 * 1024 / (BYTES + 1024);
  static constexpr int MOST = WPR == 1 ? 3 : WPR == 4 ? 6 : 1;
  static constexpr int BLOCKS = FIT < 1 ? 1 : FIT < MOST ? FIT : MOST;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

template <typename T, int V, int WPR>
__global__ void __launch_bounds__(bwd_threads(WPR), Staged<T, V, WPR>::BLOCKS) k_rms_bwd_staged(const BwdArgs a) {
  using L = Staged<T, V, WPR>;
  extern __shared__ __align__(16) uint8_t rows[];
  __shared__ float slot[2][32];
  constexpr int RPC = bwd_threads(WPR) / (32 * WPR), Q = (int)sizeof(T) / 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w0 = warp % WPR;
  const int64_t step = (int64_t)gridDim.x * RPC;
  uint8_t* mine = rows + warp * (L::STAGES * L::ROW) + 16 * lane;
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(mine);
  const T *dyp = static_cast<const T*>(a.dy), *hp = static_cast<const T*>(a.h), *dhp = static_cast<const T*>(a.dh);
  float dw[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = 0.f;
  // the row's three parts, span by span; chunk q of a lane's columns 512 bytes on
  const auto bring = [&](int64_t r, int stage) {
    if (r < a.rows) {
      const uint32_t to = at + stage * L::ROW;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = 256 * (j * WPR + w0) + 8 * lane;
        const bool in = c < a.width;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int e = in ? c + q * 4 : 0;
          copy16(to + (0 * V + j) * L::PART + 512 * q, dyp + r * a.lddy + e, in);
          copy16(to + (1 * V + j) * L::PART + 512 * q, hp + r * a.ldh + e, in);
          if (dhp != nullptr) copy16(to + (2 * V + j) * L::PART + 512 * q, dhp + r * a.lddh + e, in);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");       // one group a row, empty or not
  };
  const auto get = [&](int stage, int part, int j, float (&v)[8]) {
    const uint8_t* p = mine + stage * L::ROW + (part * V + j) * L::PART;
    uint4 u[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) u[q] = *reinterpret_cast<const uint4*>(p + 512 * q);
    load8(reinterpret_cast<const T*>(u), v);
  };
  int which = 0, stage = 0;
  int64_t row = (int64_t)blockIdx.x * RPC + warp / WPR;
#pragma unroll
  for (int s = 0; s < L::STAGES - 1; ++s) bring(row + s * step, s);
  for (; row < a.rows; row += step) {
    const float rs = a.rstd[row];
    bring(row + (L::STAGES - 1) * step, stage == 0 ? L::STAGES - 1 : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(L::STAGES - 1) : "memory");
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float w[8], g[8], h[8];
      load_weight<1>(a.w, a.wbf16, j * WPR + w0, lane, a.width, w);
      get(stage, 0, j, g);
      get(stage, 1, j, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[j][i] = fmaf(g[i], h[i] * rs, dw[j][i]);
        dot = fmaf(g[i] * w[i], h[i], dot);
      }
    }
    dot = row_sum<WPR>(dot, slot, which);
    which ^= 1;
    const float c = dot / (float)a.width * rs * rs;
    T* dx = static_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float w[8], g[8], h[8];
      load_weight<1>(a.w, a.wbf16, j * WPR + w0, lane, a.width, w);
      get(stage, 0, j, g);
      get(stage, 1, j, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = rs * (g[i] * w[i] - h[i] * c);
      if (dhp != nullptr) {
        get(stage, 2, j, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] += h[i];
      }
      store_span<T, 1>(dx, j * WPR + w0, lane, a.width, g);
    }
    stage = stage == L::STAGES - 1 ? 0 : stage + 1;
  }
  float* part = a.part + (int64_t)blockIdx.x * a.width;
  if constexpr (RPC == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = col_of<1>(j * WPR + w0, lane, i);
        if (c < a.width) part[c] = dw[j][i];
      }
  } else {
    // the CTA's warps hold the same columns of different rows
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    float(*red)[256] = reinterpret_cast<float(*)[256]>(rows);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) red[warp][col_of<1>(0, lane, i)] = dw[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < 256; c += 32 * RPC) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < RPC; ++r) t += red[r][c];
        if (256 * j + c < a.width) part[256 * j + c] = t;
      }
    }
  }
}

// CTAs of the unstaged form that an SM holds
constexpr int bwd_blocks(int wpr, int v) { return wpr == 1 ? v == 1 ? 3 : 2 : wpr == 4 ? 4 : 1; }

// Where rows wait in shared memory.  A bfloat16 row is short, and several of them have to
// be on their way; a float32 row of more than 96 columns is on its way in enough
// registers by itself, and its second reading from shared memory costs more than the
// wait.  67 M elements with dh, staged against not: float32 1046872 x 64 373 and 403 us,
// 523432 x 128 283 and 241, 261712 x 256 267 and 175, 65424 x 1024 294 and 179, 16352 x 4096
// 309 and 191; bfloat16 10904 x 6144 157 and 192, 8176 x 8192 133 and 161, 4088 x 16384
// 142 and 152 (without dh 8178 x 8192 123 and 116).
template <typename T, int VEC, int V, int WPR>
constexpr bool can_stage() { return VEC == 1 && (sizeof(T) == 2 ? WPR <= 16 : V == 1 && WPR == 1); }
constexpr int kStagedFloats = 96;

template <typename T, int VEC, int V, int WPR>
__global__ void __launch_bounds__(bwd_threads(WPR), bwd_blocks(WPR, V)) k_rms_bwd(const BwdArgs a) {
  __shared__ float slot[2][32];
  constexpr int RPC = bwd_threads(WPR) / (32 * WPR);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w0 = warp % WPR;
  const int64_t step = (int64_t)gridDim.x * RPC;
  const T *dyp = static_cast<const T*>(a.dy), *hp = static_cast<const T*>(a.h), *dhp = static_cast<const T*>(a.dh);
  float dw[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = 0.f;
  int which = 0;
  int64_t row = (int64_t)blockIdx.x * RPC + warp / WPR;
  for (; row < a.rows; row += step) {
    const T* dy = dyp + row * a.lddy;
    const T* hr = hp + row * a.ldh;
    const float rs = a.rstd[row];
    float g[V][8], h[V][8];
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) load_span<T, VEC>(dy, j * WPR + w0, lane, a.width, g[j]);
#pragma unroll
    for (int j = 0; j < V; ++j) load_span<T, VEC>(hr, j * WPR + w0, lane, a.width, h[j]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float w[8];
      load_weight<VEC>(a.w, a.wbf16, j * WPR + w0, lane, a.width, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[j][i] = fmaf(g[j][i], h[j][i] * rs, dw[j][i]);
        g[j][i] *= w[i];
        dot = fmaf(g[j][i], h[j][i], dot);
      }
    }
    dot = row_sum<WPR>(dot, slot, which);
    which ^= 1;
    const float c = dot / (float)a.width * rs * rs;
    T* dx = static_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[j][i] = rs * (g[j][i] - h[j][i] * c);
      if (dhp != nullptr) {
        float t[8];
        load_span<T, VEC>(dhp + row * a.lddh, j * WPR + w0, lane, a.width, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[j][i] += t[i];
      }
      store_span<T, VEC>(dx, j * WPR + w0, lane, a.width, g[j]);
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * a.width;
  if constexpr (RPC == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = col_of<VEC>(j * WPR + w0, lane, i);
        if (c < a.width) part[c] = dw[j][i];
      }
  } else {
    // the CTA's warps hold the same columns of different rows
    __shared__ float red[RPC][256];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) red[warp][col_of<VEC>(0, lane, i)] = dw[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < 256; c += 32 * RPC) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < RPC; ++r) t += red[r][c];
        if (256 * j + c < a.width) part[256 * j + c] = t;
      }
    }
  }
}

// dweight[c] = sum over the CTAs' partial rows, in their order within 32 strands
__global__ void __launch_bounds__(1024) k_rms_dweight(const float* __restrict__ part, int parts,
                                                      int width, void* __restrict__ dw, int wbf16) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, strand = threadIdx.x >> 5;
  float t = 0.f;
  if (c < width)
    for (int p = strand; p < parts; p += 32) t += part[(int64_t)p * width + c];
  red[strand][lane] = t;
  __syncthreads();
  // warp `strand` sums column `strand` of the 32
  t = warp_sum(red[lane][strand]);
  const int o = blockIdx.x * 32 + strand;
  if (lane == 0 && o < width) {
    if (wbf16)
      static_cast<bf16*>(dw)[o] = from_f32<bf16>(t);
    else
      static_cast<float*>(dw)[o] = t;
  }
}

// CTAs of the backward pass, one partial row of dweight each: at most what
// the SMs hold at once, no more than there are rows
int bwd_ctas(const race_norm_desc_t* d, int wpr) {
  const int rpc = bwd_threads(wpr) / (32 * wpr);
  const int64_t most = (d->rows + rpc - 1) / rpc;
  // no more than either form keeps on an SM: the workspace goes by this number
  const int64_t fill = (int64_t)api_sm_count() * (wpr == 1 ? 3 : wpr == 4 ? 6 : 1);
  return (int)(most < fill ? most : fill);
}

int warps_per_row(int64_t width) {
  return width <= 1024 ? 1 : width <= 4096 ? 4 : width <= 16384 ? 16 : 32;
}

// CTAs of a kernel that the SMs hold at once
template <typename K>
int64_t resident(K kernel, int threads, std::atomic<int>& held) {
  int n = held.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess || n < 1) n = 1;
    held.store(n, std::memory_order_relaxed);
  }
  return (int64_t)n * api_sm_count();
}

template <typename T, int VEC, int V, int WPR, bool Q, bool WALK>
void launch_fwd_as(const FwdArgs& a, cudaStream_t s) {
  constexpr int RPC = threads_of(WPR) / (32 * WPR);
  int64_t grid = (a.rows + RPC - 1) / RPC;
  if constexpr (WALK) {
    static std::atomic<int> held;
    grid = std::min(grid, resident(&k_rms_fwd<T, VEC, V, WPR, Q, true>, threads_of(WPR), held));
  }
  k_rms_fwd<T, VEC, V, WPR, Q, WALK><<<(unsigned)grid, threads_of(WPR), 0, s>>>(a);
}

// Rows walked, or a CTA's rows alone.  Walking pays where a row leaves too few bytes on
// their way: bfloat16, and narrow float32.  Otherwise the CTAs that come and go keep
// more of them, and the registers that the loop takes cost more than it saves; a loop
// over 64 values a thread spills.  50 M elements with residual, walked and not, to x's
// type and (after the stroke) to 8 bits, in us:
//   float32           781250 x 64 160, 170 / 193, 204    390625 x 128 127, 120 / 114, 119
//                     195312 x 256 150, 122 / 118, 98    48828 x 1024 149, 128 / 110, 102
//                     12207 x 4096 147, 128 / 112, 109   1525 x 32768 555, 237 / 596, 222
//   bfloat16          1525 x 32768 341, 128 / 322, 133
//   float32, single   196078 x 255 144, 174 / 148, 183   97847 x 511 134, 124 / 132, 134
//   elements          49950 x 1001 138, 122 / 133, 125 (without residual 71, 65 / 65, 93)
//                     9994 x 5003 223, 138 / 249, 170    3050 x 16390 1153, 328 / 333, 507
//   bfloat16, single  49950 x 1001 93, 91 / 112, 123     31230 x 1601 148, 147 / 199, 183
//   elements          9994 x 5003 233, 240 / 255, 273    3050 x 16390 1040, 281 / 354, 433
template <typename T, int VEC, int V, int WPR, bool Q>
void launch_fwd_by(const FwdArgs& a, cudaStream_t s) {
  if constexpr (sizeof(T) == 4 && WPR == 1 && (V == 1 || !VEC)) {
    if (a.width < (VEC ? (Q ? 160 : 96) : (Q ? 1025 : 384)))
      launch_fwd_as<T, VEC, V, WPR, Q, true>(a, s);
    else
      launch_fwd_as<T, VEC, V, WPR, Q, false>(a, s);
  } else {
    constexpr bool WALK = WPR == 32 ? !VEC && Q : sizeof(T) == 2 && (VEC || WPR != 4);
    launch_fwd_as<T, VEC, V, WPR, Q, WALK>(a, s);
  }
}
template <typename T, int VEC, int V, int WPR>
void launch_fwd(const FwdArgs& a, cudaStream_t s) {
  if (a.codes != nullptr)
    launch_fwd_by<T, VEC, V, WPR, true>(a, s);
  else
    launch_fwd_by<T, VEC, V, WPR, false>(a, s);
}
// grid: the CTAs launched, one partial row of dweight each.
template <typename T, int VEC, int V, int WPR>
int launch_bwd(const BwdArgs& a, int most, int& grid, cudaStream_t s) {
  if constexpr (can_stage<T, VEC, V, WPR>()) {
    if (sizeof(T) == 2 || a.width <= kStagedFloats) {
      using L = Staged<T, V, WPR>;
      static std::atomic<uint64_t> ready;
      RACE_CALL(api_allow_smem(reinterpret_cast<const void*>(&k_rms_bwd_staged<T, V, WPR>), L::BYTES, ready));
      grid = std::min(most, L::BLOCKS * api_sm_count());
      k_rms_bwd_staged<T, V, WPR><<<grid, bwd_threads(WPR), L::BYTES, s>>>(a);
      return RACE_OK;
    }
  }
  if constexpr (sizeof(T) == 4 || !can_stage<T, VEC, V, WPR>()) {
    grid = std::min(most, bwd_blocks(WPR, V) * api_sm_count());
    k_rms_bwd<T, VEC, V, WPR><<<grid, bwd_threads(WPR), 0, s>>>(a);
  }
  return RACE_OK;
}

// The spans a warp holds (V) follow from the width; the form of single elements and
// the widest rows are built once.
template <typename F>
void pick(bool f32, int vec, int wpr, int v, F&& f) {
#define RACE_AS(T, VEC, V, W) \
  f(T(), std::integral_constant<int, VEC>(), std::integral_constant<int, V>(), std::integral_constant<int, W>())
#define RACE_PICK(V, W)                                                     \
  if (wpr == W && (vec != 0 || V == (W == 32 ? 8 : 4)) && v <= V) {         \
    if (vec == 2) return RACE_AS(float, 2, V, W);                           \
    if (vec == 1) return f32 ? RACE_AS(float, 1, V, W) : RACE_AS(bf16, 1, V, W); \
    if constexpr (V == (W == 32 ? 8 : 4))                                   \
      return f32 ? RACE_AS(float, 0, V, W) : RACE_AS(bf16, 0, V, W);        \
  }
  RACE_PICK(1, 1) RACE_PICK(2, 1) RACE_PICK(3, 1) RACE_PICK(4, 1)
  RACE_PICK(2, 4) RACE_PICK(3, 4) RACE_PICK(4, 4)
  RACE_PICK(2, 16) RACE_PICK(3, 16) RACE_PICK(4, 16)
  RACE_PICK(8, 32)
#undef RACE_PICK
#undef RACE_AS
}

// The form of the loads (see load_span) for rows whose bases allow vectors.
int vec_of(const race_norm_desc_t* d, bool aligned) {
  if (!aligned) return 0;
  if (d->width % 8 == 0) return 1;
  return d->width % 4 == 0 && d->dtype == RACE_F32 && d->weight_dtype == RACE_F32 ? 2 : 0;
}

bool aligned16(const void* p, int64_t ld, int es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0;
}

int check_desc(const race_norm_desc_t* d) {
  if (d == nullptr || d->rows < 0 || d->width < 1) return RACE_ERR_INVALID;
  if (d->dtype != RACE_F32 && d->dtype != RACE_BF16) return RACE_ERR_INVALID;
  if (d->weight_dtype != RACE_F32 && d->weight_dtype != RACE_BF16) return RACE_ERR_INVALID;
  if (d->width > 65536 || d->rows >= (int64_t(1) << 31)) {
    api_note("norm: width above 65536 or 2^31 rows and more");
    return RACE_ERR_UNSUPPORTED;
  }
  return RACE_OK;
}

int check_rows(const race_norm_desc_t* d, race_rows_t r, bool wanted) {
  if (r.data == nullptr) return wanted ? RACE_ERR_INVALID : RACE_OK;
  if (reinterpret_cast<uintptr_t>(r.data) % (d->dtype == RACE_F32 ? 4 : 2) != 0) return RACE_ERR_ALIGN;
  return d->rows <= 1 || r.ld >= d->width || r.ld == 0 ? RACE_OK : RACE_ERR_INVALID;
}

}  // namespace norm
}  // namespace race

using namespace race;

extern "C" int race_rms_norm(const race_norm_desc_t* desc, race_rows_t x, race_rows_t residual,
                             const void* weight, race_rows_t y, race_blocks_t y8, race_rows_t h,
                             float* rstd, cudaStream_t stream) {
  ApiCall call;
  RACE_CALL(norm::check_desc(desc));
  if (desc->rows == 0) return RACE_OK;
  if (weight == nullptr || (y.data == nullptr) == (y8.codes == nullptr)) return RACE_ERR_INVALID;
  RACE_CALL(norm::check_rows(desc, x, true));
  RACE_CALL(norm::check_rows(desc, residual, false));
  RACE_CALL(norm::check_rows(desc, y, false));
  RACE_CALL(norm::check_rows(desc, h, residual.data != nullptr));
  if (!api_aligned(weight, desc->weight_dtype == RACE_F32 ? 4 : 2) || !api_aligned(rstd, 4)) return RACE_ERR_ALIGN;
  if ((y.data != nullptr && y.ld < desc->width && desc->rows > 1) ||
      (residual.data != nullptr && h.ld < desc->width && desc->rows > 1))
    return RACE_ERR_INVALID;                 // results may not overlap
  if (y8.codes != nullptr) {
    if (y8.scales == nullptr) return RACE_ERR_INVALID;
    if (!api_aligned(y8.codes, 16) || y8.ld % 16 != 0 || !api_aligned(y8.scales, 4)) return RACE_ERR_ALIGN;
    if (y8.ld < desc->width) return RACE_ERR_INVALID;
  }
  RACE_CALL(api_bind(stream));
  norm::FwdArgs a{x.data, x.ld, residual.data, residual.ld, weight, desc->weight_dtype == RACE_BF16,
                  y.data, y.ld, h.data, h.ld, static_cast<uint8_t*>(y8.codes), y8.ld, y8.scales,
                  y8.stride_row, y8.stride_block, rstd, desc->rows, (int)desc->width, desc->eps};
  const bool f32 = desc->dtype == RACE_F32;
  const int es = f32 ? 4 : 2;
  const bool aligned = norm::aligned16(x.data, x.ld, es) && norm::aligned16(weight, 0, 1) &&
                   (residual.data == nullptr || (norm::aligned16(residual.data, residual.ld, es) &&
                                                 norm::aligned16(h.data, h.ld, es))) &&
                   (y.data == nullptr || norm::aligned16(y.data, y.ld, es));
  const int wpr = norm::warps_per_row(desc->width);
  const int v = (int)((desc->width + 256 * wpr - 1) / (256 * wpr));
  norm::pick(f32, norm::vec_of(desc, aligned), wpr, v, [&](auto t, auto ve, auto vv, auto ww) {
    norm::launch_fwd<decltype(t), decltype(ve)::value, decltype(vv)::value, decltype(ww)::value>(a, stream);
  });
  api_log(y8.codes != nullptr ? "rms_fwd_8bit" : "rms_fwd");
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
}

extern "C" size_t race_rms_norm_workspace(const race_norm_desc_t* desc) {
  if (norm::check_desc(desc) != RACE_OK) return 0;
  const int ctas = norm::bwd_ctas(desc, norm::warps_per_row(desc->width));
  return (size_t)(ctas > 0 ? ctas : 1) * (size_t)desc->width * sizeof(float);
}

extern "C" int race_rms_norm_backward(const race_norm_desc_t* desc, race_rows_t dy, race_rows_t dh,
                                      race_rows_t h, const void* weight, const float* rstd,
                                      race_rows_t dx, void* dweight, void* workspace,
                                      size_t workspace_bytes, cudaStream_t stream) {
  ApiCall call;
  RACE_CALL(norm::check_desc(desc));
  const bool any = desc->rows > 0;
  if (weight == nullptr || dweight == nullptr || (any && rstd == nullptr)) return RACE_ERR_INVALID;
  RACE_CALL(norm::check_rows(desc, dy, any));
  RACE_CALL(norm::check_rows(desc, dh, false));
  RACE_CALL(norm::check_rows(desc, h, any));
  RACE_CALL(norm::check_rows(desc, dx, any));
  const int ws = desc->weight_dtype == RACE_F32 ? 4 : 2;
  if (!api_aligned(weight, ws) || !api_aligned(dweight, ws) || !api_aligned(rstd, 4) || !api_aligned(workspace, 16))
    return RACE_ERR_ALIGN;
  if (desc->rows > 1 && dx.ld < desc->width) return RACE_ERR_INVALID;
  RACE_CALL(api_bind(stream));
  const int wb = desc->weight_dtype == RACE_BF16;
  if (!any) {
    const cudaError_t e = cudaMemsetAsync(dweight, 0, (size_t)desc->width * (wb ? 2 : 4), stream);
    return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
  }
  if (workspace == nullptr || workspace_bytes < race_rms_norm_workspace(desc)) return RACE_ERR_WORKSPACE;
  norm::BwdArgs a{dy.data, dy.ld, dh.data, dh.ld, h.data, h.ld, weight, wb, rstd, dx.data, dx.ld,
                  static_cast<float*>(workspace), desc->rows, (int)desc->width};
  const bool f32 = desc->dtype == RACE_F32;
  const int es = f32 ? 4 : 2;
  const bool aligned = norm::aligned16(dy.data, dy.ld, es) && norm::aligned16(h.data, h.ld, es) &&
                   norm::aligned16(dx.data, dx.ld, es) && norm::aligned16(weight, 0, 1) &&
                   (dh.data == nullptr || norm::aligned16(dh.data, dh.ld, es));
  const int wpr = norm::warps_per_row(desc->width);
  const int v = (int)((desc->width + 256 * wpr - 1) / (256 * wpr));
  const int most = norm::bwd_ctas(desc, wpr);
  int grid = 0, rc = RACE_OK;
  norm::pick(f32, norm::vec_of(desc, aligned), wpr, v, [&](auto t, auto ve, auto vv, auto ww) {
    rc = norm::launch_bwd<decltype(t), decltype(ve)::value, decltype(vv)::value, decltype(ww)::value>(a, most, grid, stream);
  });
  RACE_CALL(rc);
  api_log("rms_bwd");
  norm::k_rms_dweight<<<(unsigned)((desc->width + 31) / 32), 1024, 0, stream>>>(
      a.part, grid, a.width, dweight, wb);
  api_log("rms_dweight");
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
}
