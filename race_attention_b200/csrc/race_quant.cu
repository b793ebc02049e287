// race_quant.cu -- quantisation to 8 bits with one scale for each 128 elements
// of a row (and of a column), or for each 128 x 128 block.
//
// A training pass needs every operand twice: its rows for one product and its
// columns, transposed, for the other.  Reading x once for both halves the
// pass, which memory bounds (bf16: 2 bytes read and 2 written per element).
// A CTA takes a 128 x 128 tile, a whole block in either direction; thread
// (ty, tx) holds rows 8 ty .. 8 ty + 7 of columns 8 tx .. 8 tx + 7 in registers, so the tile
// never passes through shared memory at full width: a row's maximum is taken
// over the 16 lanes of a half warp, a column's over the thread's rows and then
// eight warps.  Transposed codes are packed eight rows to a word pair in
// registers and cross shared memory as bytes (16 KB), written out in whole
// 128-byte rows.
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

template <typename T, bool VEC, bool SQUARE, bool ROWS, bool COLS>
__global__ void __launch_bounds__(NT) k_quantize(const Args a) {
  __shared__ __align__(16) uint2 tile[COLS ? 128 * 16 : 1];   // [column][8-row group], swizzled
  __shared__ uint32_t wmax[8][COLS && !SQUARE ? 128 : 1];
  __shared__ float cinv[COLS && !SQUARE ? 128 : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tx = tid & 15, ty = tid >> 4;
  // column tiles run fastest: a row's bytes are read by neighbouring CTAs
  const int64_t r0 = (int64_t)blockIdx.y * 128, c0 = (int64_t)blockIdx.x * 128;
  const int64_t r = r0 + 8 * ty, c = c0 + 8 * tx;
  const T* x = static_cast<const T*>(a.x) + r * a.ld + c;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (VEC && r + i < a.rows && c + 8 <= a.cols) {
      load8(x + i * a.ld, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[i][j] = r + i < a.rows && c + j < a.cols ? to_f32(x[i * a.ld + j]) : 0.f;
    }
  }
  uint2 code[8];
  if constexpr (SQUARE) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, mag(v[i][j]));
    m = max_over(m, 32);
    if (lane == 0) wmax[warp][0] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, wmax[w][0]);
    const float s = scale_of(m), inv = 1.f / s;
    if (tid == 0) {
      if (ROWS) a.rs[blockIdx.y * a.rsr + blockIdx.x * a.rsb] = s;
      if (COLS && a.cs != nullptr) a.cs[blockIdx.x * a.csr + blockIdx.y * a.csb] = s;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = code8(v[i], inv);
  } else if constexpr (ROWS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, mag(v[i][j]));
      const float s = scale_of(max_over(m, 16));
      if (tx == 0 && r + i < a.rows) a.rs[(r + i) * a.rsr + blockIdx.x * a.rsb] = s;
      code[i] = code8(v[i], 1.f / s);
    }
  }
  if constexpr (ROWS) {
#pragma unroll
    for (int i = 0; i < 8; ++i)   // the pitch is a multiple of 16: whole 8-byte groups fit
      if (r + i < a.rows && c < ((a.cols + 15) & ~int64_t(15)))
        *reinterpret_cast<uint2*>(a.rc + (r + i) * a.ldr + c) = code[i];
  }
  if constexpr (COLS) {
    if constexpr (!SQUARE) {
      uint32_t m[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m[j] = mag(v[0][j]);
#pragma unroll
        for (int i = 1; i < 8; ++i) m[j] = max(m[j], mag(v[i][j]));
        m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
      }
      if (lane < 16)
#pragma unroll
        for (int j = 0; j < 8; ++j) wmax[warp][8 * tx + j] = m[j];
      __syncthreads();
      if (tid < 128) {
        uint32_t t = wmax[0][tid];
#pragma unroll
        for (int w = 1; w < 8; ++w) t = max(t, wmax[w][tid]);
        const float s = scale_of(t);
        cinv[tid] = 1.f / s;
        if (c0 + tid < a.cols) a.cs[(c0 + tid) * a.csr + blockIdx.y * a.csb] = s;
      }
      __syncthreads();
    }
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
        for (int i = 0; i < 8; ++i) t[i] = v[i][j];
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
  if (reinterpret_cast<uintptr_t>(b.codes) % 16 != 0 || b.ld % 16 != 0) return RACE_ERR_ALIGN;
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
