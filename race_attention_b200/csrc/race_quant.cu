// race_quant.cu -- quantisation to 8 bits with one scale for each 128 elements
// of a row (and of a column), or for each 128 x 128 block.
//
// A training pass needs every operand twice: its rows for one product and its
// columns, transposed, for the other.  Reading x once for both halves the
// pass, which memory bounds (bf16: 2 bytes read and 2 written per element).
// A CTA takes a 128 x 128 tile, a whole block in either direction; thread
// (ty, tx) holds rows 8 ty .. 8 ty + 7 of columns 8 tx .. 8 tx + 7 in registers, so the tile
// never passes through shared memory at full width: the maxima of the eight rows
// are taken over the 16 lanes of a half warp in one exchange that leaves each
// pair of lanes with one row (and one reciprocal to form), a column's over the
// thread's rows and then eight warps.  Transposed codes are packed eight rows to a word pair in
// registers and cross shared memory as bytes (16 KB), written out in whole
// 128-byte rows.  Measured, 65536 x 2304 bfloat16: rows 69 us (6.5 TB/s), rows and
// columns 104 us (5.8), square blocks with their transpose 99 us; float32 rows and
// columns 141 us (6.4).  Odd widths or strides are read element by element:
// 65536 x 2303 rows 206 us and both 263 (bfloat16, 2.2 TB/s), 169 and 237 (float32, 4.5).
#include "race_api.h"
#include "race_lowp.cuh"

namespace race {
namespace quant {

using namespace lowp;

struct Args {
  const void* x; int64_t ld;
  int64_t rows, cols;
  uint8_t* rc; int64_t ldr; float* rs; int64_t rsr, rsb;   // by rows
  uint8_t* cc; int64_t ldc; float* cs; int64_t csr, csb;   // by columns, transposed
};

constexpr int NT = 256;

// The thread's 8 x 8 values.  bfloat16 stays packed (32 registers in place of
// 64, which lets three CTAs share an SM) and its maxima are taken two at a time.
template <typename T>
struct Tile;

template <>
struct Tile<float> {
  float v[8][8];
  __device__ __forceinline__ void load(int i, const float* p) { load8(p, v[i]); }
  __device__ __forceinline__ void set(int i, int j, float x) { v[i][j] = x; }
  __device__ __forceinline__ float get(int i, int j) const { return v[i][j]; }
  // magnitudes are compared as they are; a column word holds one of them
  static constexpr int CW = 8;
  static __device__ __forceinline__ uint32_t bits(uint32_t m) { return m; }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  __device__ __forceinline__ uint32_t row_max(int i) const {
    uint32_t m = mag(v[i][0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = max(m, mag(v[i][j]));
    return m;
  }
  __device__ __forceinline__ uint32_t col_max(int j) const {
    uint32_t m = mag(v[0][j]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, mag(v[i][j]));
    return m;
  }
};

template <>
struct Tile<bf16> {
  uint32_t w[8][4];
  __device__ __forceinline__ void load(int i, const bf16* p) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
  }
  __device__ __forceinline__ void set(int i, int j, float x) {
    const uint32_t b = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(x));
    w[i][j >> 1] = (j & 1) ? (w[i][j >> 1] & 0xffffu) | b << 16 : b;   // even columns are set first
  }
  __device__ __forceinline__ float get(int i, int j) const {
    return __uint_as_float((j & 1) ? w[i][j >> 1] & 0xffff0000u : w[i][j >> 1] << 16);
  }
  // magnitudes are compared as 16-bit integers, two to a word
  static constexpr int CW = 4;
  static __device__ __forceinline__ uint32_t bits(uint32_t m) { return m << 16; }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  __device__ __forceinline__ uint32_t two(int i, int q) const { return w[i][q] & 0x7fff7fffu; }
  __device__ __forceinline__ uint32_t row_max(int i) const {
    const uint32_t m = larger(larger(two(i, 0), two(i, 1)), larger(two(i, 2), two(i, 3)));
    return max(m & 0xffffu, m >> 16);
  }
  __device__ __forceinline__ uint32_t col_max(int q) const {
    uint32_t m = two(0, q);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = larger(m, two(i, q));
    return m;
  }
};

// The maxima over a half warp of eight values a lane: every step hands half of the
// values over, so that eight exchanges do, and lane tx ends with that of row tx / 2.
__device__ __forceinline__ uint32_t max_of_row(const uint32_t (&m)[8], int tx) {
  uint32_t a[4], b[2], c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a[i] = max(tx & 8 ? m[4 + i] : m[i], __shfl_xor_sync(0xffffffffu, tx & 8 ? m[i] : m[4 + i], 8));
#pragma unroll
  for (int i = 0; i < 2; ++i)
    b[i] = max(tx & 4 ? a[2 + i] : a[i], __shfl_xor_sync(0xffffffffu, tx & 4 ? a[i] : a[2 + i], 4));
  c = max(tx & 2 ? b[1] : b[0], __shfl_xor_sync(0xffffffffu, tx & 2 ? b[0] : b[1], 2));
  return max(c, __shfl_xor_sync(0xffffffffu, c, 1));
}

template <typename T>
__device__ __forceinline__ uint2 code_row(const Tile<T>& t, int i, float inv) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = t.get(i, j);
  return code8(v, inv);
}

// Three CTAs an SM where 80 registers hold a thread's values and codes: float32 by rows
// and columns takes 122 (square blocks of 21700 x 2303 float32 with their transpose 66 us;
// 80 with the 94 registers that the compiler takes by itself).
template <typename T, bool VEC, bool SQUARE, bool ROWS, bool COLS>
__global__ void __launch_bounds__(NT, sizeof(T) == 2 || SQUARE ? 3 : 2) k_quantize(const Args a) {
  __shared__ __align__(16) uint2 tile[COLS ? 128 * 16 : 1];   // [column][8-row group], swizzled
  constexpr int CW = Tile<T>::CW;                              // words of 8 columns' maxima
  __shared__ uint32_t wmax[8][COLS && !SQUARE ? 16 * CW : 1];
  __shared__ float cinv[COLS && !SQUARE ? 128 : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tx = tid & 15, ty = tid >> 4;
  // column tiles run fastest: a row's bytes are read by neighbouring CTAs
  const int64_t r0 = (int64_t)blockIdx.y * 128, c0 = (int64_t)blockIdx.x * 128;
  const int64_t r = r0 + 8 * ty, c = c0 + 8 * tx;
  const T* x = static_cast<const T*>(a.x) + r * a.ld + c;
  Tile<T> v;
  if (VEC && r0 + 128 <= a.rows && c0 + 128 <= a.cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v.load(i, x + i * a.ld);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (VEC && r + i < a.rows && c + 8 <= a.cols) {
        v.load(i, x + i * a.ld);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v.set(i, j, r + i < a.rows && c + j < a.cols ? to_f32(x[i * a.ld + j]) : 0.f);
      }
    }
  }
  if constexpr (COLS && !SQUARE) {
    uint32_t m[CW];
#pragma unroll
    for (int q = 0; q < CW; ++q) {
      m[q] = v.col_max(q);
      m[q] = Tile<T>::larger(m[q], __shfl_xor_sync(0xffffffffu, m[q], 16));
    }
    if (lane < 16)
#pragma unroll
      for (int q = 0; q < CW; ++q) wmax[warp][CW * tx + q] = m[q];
    __syncthreads();
    if (tid < 16 * CW) {
      uint32_t t = wmax[0][tid];
#pragma unroll
      for (int w = 1; w < 8; ++w) t = Tile<T>::larger(t, wmax[w][tid]);
#pragma unroll
      for (int z = 0; z < 8 / CW; ++z) {                       // bfloat16: two columns a word
        const int col = tid * (8 / CW) + z;
        const float s = scale_of(Tile<T>::bits(CW == 8 ? t : z ? t >> 16 : t & 0xffffu));
        cinv[col] = 1.f / s;
        if (c0 + col < a.cols) a.cs[(c0 + col) * a.csr + blockIdx.y * a.csb] = s;
      }
    }
  }
  uint2 code[SQUARE ? 8 : 1];
  if constexpr (SQUARE) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, v.row_max(i));
    m = max_over(m, 32);
    if (lane == 0) wmax[warp][0] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, wmax[w][0]);
    const float s = scale_of(Tile<T>::bits(m)), inv = 1.f / s;
    if (tid == 0) {
      if (ROWS) a.rs[blockIdx.y * a.rsr + blockIdx.x * a.rsb] = s;
      if (COLS && a.cs != nullptr) a.cs[blockIdx.x * a.csr + blockIdx.y * a.csb] = s;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = code_row(v, i, inv);
  }
  if constexpr (ROWS) {
    // the pitch is a multiple of 16: whole 8-byte groups fit
    const bool in = c < ((a.cols + 15) & ~int64_t(15));
    float rinv = 0.f;
    if constexpr (!SQUARE) {
      uint32_t m[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) m[i] = v.row_max(i);
      const float s = scale_of(Tile<T>::bits(max_of_row(m, tx)));
      rinv = 1.f / s;
      if ((tx & 1) == 0 && r + (tx >> 1) < a.rows) a.rs[(r + (tx >> 1)) * a.rsr + blockIdx.x * a.rsb] = s;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint2 q;
      if constexpr (SQUARE) {
        q = code[i];
      } else {
        q = code_row(v, i, __shfl_sync(0xffffffffu, rinv, 2 * i, 16));
      }
      if (r + i < a.rows && in) *reinterpret_cast<uint2*>(a.rc + (r + i) * a.ldr + c) = q;
    }
  }
  if constexpr (COLS) {
    if constexpr (!SQUARE) __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint2 p;
      if constexpr (SQUARE) {
        // byte j of the eight rows' codes
        const int sh = 8 * (j & 3);
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = ((j < 4 ? code[i].x : code[i].y) >> sh) & 0xffu;
        p.x = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
        p.y = b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24;
      } else {
        const float inv = cinv[8 * tx + j];
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = v.get(i, j);
        p = code8(t, inv);
      }
      // lanes of one column group fall on 16 different word pairs
      tile[(8 * tx + j) * 16 + (ty ^ tx)] = p;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int id = q * NT + tid, col = id >> 3, seg = id & 7;   // 16 rows each
      const int64_t rr = r0 + 16 * seg;
      if (c0 + col < a.cols && rr < a.rows) {
        const int t = col >> 3;
        const uint4 u = *reinterpret_cast<const uint4*>(&tile[col * 16 + ((2 * seg) ^ (t & ~1))]);
        // an odd column group holds the pair in reverse
        *reinterpret_cast<uint4*>(a.cc + (c0 + col) * a.ldc + rr) =
            (t & 1) ? make_uint4(u.z, u.w, u.x, u.y) : u;
      }
    }
  }
}

template <typename T, bool VEC>
void launch(const Args& a, bool square, cudaStream_t s) {
  const dim3 grid((unsigned)((a.cols + 127) / 128), (unsigned)((a.rows + 127) / 128));
  const bool r = a.rc != nullptr, c = a.cc != nullptr;
  if (square) {
    if (r && c) k_quantize<T, VEC, true, true, true><<<grid, NT, 0, s>>>(a);
    else if (r) k_quantize<T, VEC, true, true, false><<<grid, NT, 0, s>>>(a);
    else k_quantize<T, VEC, true, false, true><<<grid, NT, 0, s>>>(a);
  } else {
    if (r && c) k_quantize<T, VEC, false, true, true><<<grid, NT, 0, s>>>(a);
    else if (r) k_quantize<T, VEC, false, true, false><<<grid, NT, 0, s>>>(a);
    else k_quantize<T, VEC, false, false, true><<<grid, NT, 0, s>>>(a);
  }
}

int check_blocks(race_blocks_t b, int64_t cols, bool scales) {
  if (b.codes == nullptr) return RACE_OK;
  if (scales && b.scales == nullptr) return RACE_ERR_INVALID;
  if (!api_aligned(b.codes, 16) || b.ld % 16 != 0 || !api_aligned(b.scales, 4)) return RACE_ERR_ALIGN;
  return b.ld >= cols ? RACE_OK : RACE_ERR_INVALID;
}

}  // namespace quant
}  // namespace race

using namespace race;

extern "C" int race_quantize(race_rows_t x, int32_t dtype, int64_t rows, int64_t cols,
                             int32_t square, race_blocks_t by_rows, race_blocks_t by_cols,
                             cudaStream_t stream) {
  ApiCall call;
  if (rows < 0 || cols < 0 || (dtype != RACE_F32 && dtype != RACE_BF16)) return RACE_ERR_INVALID;
  if (rows == 0 || cols == 0) return RACE_OK;
  if (by_rows.codes == nullptr && by_cols.codes == nullptr) return RACE_ERR_INVALID;
  RACE_CALL(quant::check_blocks(by_rows, cols, true));
  RACE_CALL(quant::check_blocks(by_cols, rows, !square || by_rows.codes == nullptr));
  const int es = dtype == RACE_F32 ? 4 : 2;
  if (x.data == nullptr || (rows > 1 && x.ld < 0)) return RACE_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(x.data) % es != 0) return RACE_ERR_ALIGN;
  if (rows > 65535 * int64_t(128) || cols >= (int64_t(1) << 31)) {
    api_note("quantize: more than 8388480 rows");
    return RACE_ERR_UNSUPPORTED;
  }
  RACE_CALL(api_bind(stream));
  const quant::Args a{x.data, x.ld, rows, cols,
                      static_cast<uint8_t*>(by_rows.codes), by_rows.ld, by_rows.scales,
                      by_rows.stride_row, by_rows.stride_block,
                      static_cast<uint8_t*>(by_cols.codes), by_cols.ld, by_cols.scales,
                      by_cols.stride_row, by_cols.stride_block};
  const bool vec = reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.ld * es % 16 == 0;
  if (es == 4)
    vec ? quant::launch<float, true>(a, square != 0, stream) : quant::launch<float, false>(a, square != 0, stream);
  else
    vec ? quant::launch<lowp::bf16, true>(a, square != 0, stream) : quant::launch<lowp::bf16, false>(a, square != 0, stream);
  api_log(square ? "quantize_square" : "quantize");
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
}
