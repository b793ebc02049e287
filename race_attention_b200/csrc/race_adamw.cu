// race_adamw.cu -- one AdamW step over many tensors in one launch, states in 32
// or in 8 bits.
//
//   p -= lr wd p;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p -= lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Nothing is used twice, so memory bounds the step: float32 with 32-bit states
// moves 28 bytes a parameter (96.0 M parameters 395 us, 6.8 TB/s; a copy, which writes as
// much as it reads where the step writes 12 bytes of 28, reaches 6.4), with 8-bit
// states 16.1 (258 us, 6.0 TB/s; 277 where other work had filled the cache), bfloat16 with
// 32-bit states 22 (337 us, 6.3).  bfloat16 with 8-bit states moves 10.1 and is bound by
// its 90 instructions a parameter, half of them logic (184 M: 509 us, 3.7 TB/s).  The tensors'
// addresses travel in the kernel's parameters (up to 360 tensors in the 32 KB
// that a launch carries), so a step needs no copy to the device; the step's count,
// learning rate and noise travel with them, which is why a capture is refused: each
// replay would repeat them.  A CTA finds its 2048 elements by bisection over the running chunk
// counts.  A thread holds 8 consecutive elements, half a warp one 128-element
// block of the states.
//
// 8-bit states.  m and sqrt(v) are held as e4m3 codes with one scale for each
// 128 elements (the root halves v's range of exponents).  Codes are 6 to 12 %
// apart while b2 = 0.999 moves sqrt(v) by at most 0.05 % of itself downwards a
// step, so rounding to nearest would never let a state decay; the states are
// rounded up or down with the probability of the part cut off instead, which is
// right on average.  A second moment above zero is held as at least the
// smallest code: as zero, it would leave eps alone in the denominator.
// bfloat16 parameters (2^-9 of themselves apart) are rounded the same way.
// The noise is a hash of the element's index, the seed and t, two odd
// multipliers (2^32 over the golden ratio; the fraction of sqrt(2)) between shifts.
// m takes its lower half, the root its upper half, and the parameter the lower half
// under the next key, which for an even key is that of m's neighbour: each rounding
// is right on average, but the two are not independent.
#include <cmath>
#include <type_traits>

#include "race_api.h"
#include "race_lowp.cuh"

namespace race {
namespace adamw {

using namespace lowp;

constexpr int NT = 256;
constexpr int kChunk = 8 * NT;         // elements of a CTA at a time
constexpr int kRounds = 4;             // of the 8-bit form with bfloat16 parameters
constexpr uint32_t kGolden = 0x9E3779B1u, kRootTwo = 0x6A09E667u;

struct Item {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* ms;
  float* vs;
  int64_t n;
  uint32_t first;
  uint32_t key;            // seed and step
  float step_size;         // lr / (1 - b1^t)
  float root_scale;        // 1 / sqrt(1 - b2^t)
  int flags;               // 1: bf16, 2: vector access
};

template <int N>
struct Args {
  int count;
  float keep;              // 1 - lr wd
  float b1, c1, b2, c2, eps;
  int32_t end[N];          // chunks up to and with tensor i
  Item item[N];
};

// h of the noise h ^ (h >> 16): its upper half is h's own
__device__ __forceinline__ uint32_t noise(uint32_t i_xor_key) {
  const uint32_t h = i_xor_key * kGolden;
  return (h ^ (h >> 15)) * kRootTwo;
}
__device__ __forceinline__ uint32_t lower(uint32_t h) { return (h ^ (h >> 16)) & 0xffffu; }

// y in [0, 448] up or down to the 8-bit format, r of 65536ths deciding (r20 = 16 r):
// below 2^-6 the format's steps are even, as they are for every number of the
// binade that adding 2^-6 moves y to.  Whether y is below comes from a saturated
// product, 0 or 1 (2^-6 - y is 2^-30 at least if it is above zero): the logic units
// are the bound here, the multipliers are not.  A y that rounding put one place
// above 448 still gives 448.
__device__ __forceinline__ float dither(float y, uint32_t r20) {
  const float low = __saturatef(fmaf(y, -0x1p40f, 0x1p34f));
  const uint32_t b = __float_as_uint(fmaf(low, 0.015625f, y)) + r20;
  return fmaf(low, -0.015625f, __uint_as_float(b & ~0xfffffu));
}

// to two units of the last place, infinite for zero
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// the larger magnitude, NaN if one is
__device__ __forceinline__ float max_mag(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

template <typename T>
__device__ __forceinline__ void load_some(const T* p, bool vec, int n, float (&v)[8]) {
  if (vec && n >= 8) {
    load8(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, bool vec, int n, const float (&v)[8]) {
  if (vec && n >= 8) {
    store8(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = from_f32<T>(v[i]);
}

// Pairs of values go through the two-wide multiply and add.
struct Eight {
  float2 v[4];
  __device__ __forceinline__ float get(int i) const { return i & 1 ? v[i >> 1].y : v[i >> 1].x; }
};

// sums of two products that are rounded first (a two-wide sum would be fused with them)
__device__ __forceinline__ float2 add_apart(float2 a, float2 b) {
  return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y));
}

// eight codes as values
__device__ __forceinline__ Eight decode(uint2 u, float s) {
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? u.x : u.y;
    const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * (i & 1))), __NV_E4M3);
    e.v[i] = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&hr)), make_float2(s, s));
  }
  return e;
}

// Holds a state's eight values of this lane.  ROOT: they are roots, at least
// zero, and take the upper half of the noise.
template <bool ROOT>
__device__ __forceinline__ void hold(void* p, float* scales, int64_t at, bool live, const Eight& x,
                                     const uint32_t (&h)[8], int lane) {
  float a = max_mag(x.v[0].x, x.v[0].y);
#pragma unroll
  for (int i = 1; i < 4; ++i) a = max_mag(a, max_mag(x.v[i].x, x.v[i].y));
  const float s = scale_of(max_over(__float_as_uint(a), 16)), inv = 1.f / s;
  if (!live) return;
  float c[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float yy[2] = {x.v[i].x * inv, x.v[i].y * inv};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t r = h[2 * i + q];
      if constexpr (ROOT) {
        // upper half of the noise, four places up; above zero at least the smallest code
        // (a root above zero over the largest scale is 2^-130 or more)
        const float d = dither(yy[q], (r >> 12) & 0xffff0u);
        c[2 * i + q] = fmaxf(d, fminf(yy[q] * 0x1p127f, 0.001953125f));
      } else {
        c[2 * i + q] = copysignf(dither(fabsf(yy[q]), lower(r) << 4), yy[q]);
      }
    }
  }
  *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p) + at) = code8(c, 1.f);
  if ((lane & 15) == 0) scales[at / kBlock] = s;
}

// The tensor that chunk `chunk` belongs to: bisection over the running counts.
template <int N>
__device__ __forceinline__ int tensor_of(const Args<N>& a, int chunk) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (chunk < a.end[mid]) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// m, v, the root and the parameters after the step; each operation of the states
// is rounded on its own, so that a restatement in elementary 32-bit operations
// gives the same states, bit for bit.  FAST: with 8-bit states arithmetic is the
// bound; the quotient may be two units of its last place off, far inside a step
// of either format.
template <bool FAST, int N>
__device__ __forceinline__ void update(const Args<N>& a, float ss, float rs, float (&p)[8], const float (&g)[8],
                                       Eight& m, Eight& v, Eight& root) {
  const float2 b1 = make_float2(a.b1, a.b1), c1 = make_float2(a.c1, a.c1);
  const float2 b2 = make_float2(a.b2, a.b2), c2 = make_float2(a.c2, a.c2);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 gg = make_float2(g[2 * i], g[2 * i + 1]);
    m.v[i] = add_apart(__fmul2_rn(b1, m.v[i]), __fmul2_rn(c1, gg));
    v.v[i] = add_apart(__fmul2_rn(b2, v.v[i]), __fmul2_rn(__fmul2_rn(c2, gg), gg));
    root.v[i] = make_float2(sqrtf(v.v[i].x), sqrtf(v.v[i].y));
    const float2 den = __ffma2_rn(root.v[i], make_float2(rs, rs), make_float2(a.eps, a.eps));
    const float2 q = FAST ? __fmul2_rn(m.v[i], make_float2(reciprocal(den.x), reciprocal(den.y)))
                          : make_float2(m.v[i].x / den.x, m.v[i].y / den.y);
    const float2 r = __ffma2_rn(make_float2(-ss, -ss), q,
                                __fmul2_rn(make_float2(p[2 * i], p[2 * i + 1]), make_float2(a.keep, a.keep)));
    p[2 * i] = r.x;
    p[2 * i + 1] = r.y;
  }
}

// bfloat16 parameters, up or down; ik: first index ^ key
__device__ __forceinline__ void store_half(bf16* o, bool whole, int n, float (&p)[8], uint32_t ik) {
  float zero = 0.f;                          // NaN as soon as one of the eight is not finite
#pragma unroll
  for (int i = 0; i < 8; ++i) zero = fmaf(p[i], 0.f, zero);
  if (zero == 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __uint_as_float(__float_as_uint(p[i]) + lower(noise(ik ^ i)));
  } else {                                   // infinities and NaN keep their bits
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(p[i]) < __int_as_float(0x7f800000))
        p[i] = __uint_as_float(__float_as_uint(p[i]) + lower(noise(ik ^ i)));
  }
  if (whole) {                               // the upper halves are the result
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __byte_perm(__float_as_uint(p[2 * i]), __float_as_uint(p[2 * i + 1]), 0x7632);
    *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) o[i] = __ushort_as_bfloat16((unsigned short)(__float_as_uint(p[i]) >> 16));
  }
}

// 32-bit states: 2048 elements a CTA
template <int N>
__global__ void __launch_bounds__(NT) k_adamw(const __grid_constant__ Args<N> a) {
  const int chunk = blockIdx.x, lo = tensor_of(a, chunk);
  const Item& it = a.item[lo];
  const int64_t at = (int64_t)(chunk - (lo > 0 ? a.end[lo - 1] : 0)) * kChunk + 8 * (int64_t)threadIdx.x;
  const int n = (int)min((int64_t)8, max((int64_t)0, it.n - at));    // elements of this thread
  const bool vec = it.flags & 2, half = it.flags & 1;
  float p[8], g[8], t[8];
  if (half) {
    load_some(static_cast<const bf16*>(it.p) + at, vec, n, p);
    load_some(static_cast<const bf16*>(it.g) + at, vec, n, g);
  } else {
    load_some(static_cast<const float*>(it.p) + at, vec, n, p);
    load_some(static_cast<const float*>(it.g) + at, vec, n, g);
  }
  Eight m, v, root;
  load_some(static_cast<const float*>(it.m) + at, true, n, t);
#pragma unroll
  for (int i = 0; i < 4; ++i) m.v[i] = make_float2(t[2 * i], t[2 * i + 1]);
  load_some(static_cast<const float*>(it.v) + at, true, n, t);
#pragma unroll
  for (int i = 0; i < 4; ++i) v.v[i] = make_float2(t[2 * i], t[2 * i + 1]);
  update<false>(a, it.step_size, it.root_scale, p, g, m, v, root);
  if (half)
    store_half(static_cast<bf16*>(it.p) + at, vec && n >= 8, n, p, (it.first + (uint32_t)at) ^ (it.key + 1));
  else
    store_some(static_cast<float*>(it.p) + at, vec, n, p);
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = m.get(i);
  store_some(static_cast<float*>(it.m) + at, true, n, t);
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = v.get(i);
  store_some(static_cast<float*>(it.v) + at, true, n, t);
}

// What a thread of the 8-bit form loads for eight elements, unconverted.
template <bool HALF>
struct Ahead {
  uint4 p[HALF ? 1 : 2], g[HALF ? 1 : 2];
  uint2 m, v;
  float sm, sv;
};

// 8-bit states.  Finding the tensor and its addresses takes a microsecond of
// dependent reads, a fifth of the time where arithmetic is the bound (184 M bfloat16
// parameters in 97 tensors 677 us, in one tensor 548): bfloat16 parameters go
// through kRounds times 2048 elements a CTA, the next ones loaded before the current
// ones are computed (514 us).  float32 moves 16 bytes a parameter, memory is the
// bound again, and one round with more CTAs is faster (by 11 % at 100.7 M).
template <int N, bool HALF>
__device__ __forceinline__ void steps8(const Args<N>& a, const Item& it, int64_t c0) {
  using T = typename std::conditional<HALF, bf16, float>::type;
  constexpr int R = HALF ? kRounds : 1;
  const int lane = threadIdx.x & 31;
  const int64_t total = it.n, padded = (total + kBlock - 1) & ~(int64_t)(kBlock - 1);
  const bool vec = it.flags & 2;
  T* const p0 = static_cast<T*>(it.p);
  const T* const g0 = static_cast<const T*>(it.g);
  const uint8_t* const m0 = static_cast<const uint8_t*>(it.m);
  const uint8_t* const v0 = static_cast<const uint8_t*>(it.v);
  float *const ms = it.ms, *const vs = it.vs;
  const uint32_t first = it.first, key = it.key;
  const float ss = it.step_size, rs = it.root_scale;
  Ahead<HALF> next;
  const auto load = [&](int64_t at) {
    if (vec && at + 8 <= total) {
#pragma unroll
      for (int q = 0; q < (HALF ? 1 : 2); ++q) {
        next.p[q] = *reinterpret_cast<const uint4*>(p0 + at + q * 4);
        next.g[q] = *reinterpret_cast<const uint4*>(g0 + at + q * 4);
      }
    }
    const bool live = at < padded;           // a state's block is whole even where the tensor ends inside it
    next.m = live ? *reinterpret_cast<const uint2*>(m0 + at) : make_uint2(0, 0);
    next.v = live ? *reinterpret_cast<const uint2*>(v0 + at) : make_uint2(0, 0);
    next.sm = live ? ms[at / kBlock] : 0.f;
    next.sv = live ? vs[at / kBlock] : 0.f;
  };
  int64_t at = c0 + 8 * (int64_t)threadIdx.x;
  load(at);
#pragma unroll 1
  for (int round = 0; round < R; ++round, at += kChunk) {
    if (c0 + round * (int64_t)kChunk >= total) break;      // the same for the whole CTA
    const int n = (int)min((int64_t)8, max((int64_t)0, total - at));
    const bool live = at < padded, whole = vec && n >= 8;
    float p[8], g[8];
    if (whole) {
      load8(reinterpret_cast<const T*>(next.p), p);
      load8(reinterpret_cast<const T*>(next.g), g);
    } else {
      load_some(p0 + at, false, n, p);
      load_some(g0 + at, false, n, g);
    }
    Eight m = decode(next.m, next.sm), v = decode(next.v, next.sv), root;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.v[i] = __fmul2_rn(v.v[i], v.v[i]);
    if (round + 1 < R) load(at + kChunk);
    update<true>(a, ss, rs, p, g, m, v, root);
    const uint32_t i0 = first + (uint32_t)at;              // a multiple of 8: i0 + i = i0 ^ i
    if constexpr (HALF)
      store_half(p0 + at, whole, n, p, i0 ^ (key + 1));
    else
      store_some(p0 + at, vec, n, p);
    uint32_t h[8];
    const uint32_t ik = i0 ^ key;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = noise(ik ^ i);
    if (n < 8) {                             // past the tensor: held as zero
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (2 * i >= n) m.v[i].x = root.v[i].x = 0.f;
        if (2 * i + 1 >= n) m.v[i].y = root.v[i].y = 0.f;
      }
    }
    hold<false>(it.m, ms, at, live, m, h, lane);
    hold<true>(it.v, vs, at, live, root, h, lane);
  }
}

// One type of parameters a launch: the two forms need 48 and 67 registers.  The
// compiler would take 50 for float32, which leaves four CTAs an SM in place of five
// (96.0 M parameters 295 us in place of 277).
template <int N, bool HALF>
__global__ void __launch_bounds__(NT, HALF ? 3 : 5) k_adamw8(const __grid_constant__ Args<N> a) {
  const int chunk = blockIdx.x, lo = tensor_of(a, chunk);
  const int64_t c0 = (int64_t)(chunk - (lo > 0 ? a.end[lo - 1] : 0)) * kChunk;
  steps8<N, HALF>(a, a.item[lo], c0 * (HALF ? kRounds : 1));
}

// Launches over the tensors `t[i]`, i in `pick`.
template <int N>
int launch(const race_adamw_desc_t* d, const race_adamw_tensor_t* t, const int64_t* pick, int count, cudaStream_t s) {
  static_assert(sizeof(Args<N>) <= 32764, "a launch carries 32764 bytes of parameters");
  Args<N> a;
  a.keep = (float)(1.0 - d->lr * d->weight_decay);
  a.b1 = (float)d->beta_one;
  a.c1 = (float)(1.0 - d->beta_one);
  a.b2 = (float)d->beta_two;
  a.c2 = (float)(1.0 - d->beta_two);
  a.eps = (float)d->eps;
  const bool eight = d->state_bits == 8, half = t[pick[0]].dtype == RACE_BF16;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const race_adamw_tensor_t& x = t[pick[i]];
    const int32_t step = x.step + 1;
    Item& it = a.item[i];
    it.p = x.param;
    it.g = x.grad;
    it.m = x.exp_avg;
    it.v = x.exp_avg_sq;
    it.ms = x.exp_avg_scale;
    it.vs = x.exp_avg_sq_scale;
    it.n = x.numel;
    it.first = (uint32_t)x.first;
    it.key = d->seed + kGolden * (uint32_t)step;
    it.step_size = (float)(d->lr / (1.0 - std::pow(d->beta_one, step)));
    it.root_scale = (float)(1.0 / std::sqrt(1.0 - std::pow(d->beta_two, step)));
    const bool vec = reinterpret_cast<uintptr_t>(x.param) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(x.grad) % 16 == 0;
    it.flags = (x.dtype == RACE_BF16 ? 1 : 0) | (vec ? 2 : 0);
    const int64_t each = eight && half ? kChunk * kRounds : kChunk;
    chunks += (x.numel + each - 1) / each;
    if (chunks >= (int64_t(1) << 31)) {
      api_note("adamw: 2^42 elements and more in one launch");
      return RACE_ERR_UNSUPPORTED;
    }
    a.end[i] = (int32_t)chunks;
  }
  a.count = count;
  if (!eight)
    k_adamw<N><<<(unsigned)chunks, NT, 0, s>>>(a);
  else if (half)
    k_adamw8<N, true><<<(unsigned)chunks, NT, 0, s>>>(a);
  else
    k_adamw8<N, false><<<(unsigned)chunks, NT, 0, s>>>(a);
  api_log(eight ? "adamw_8bit" : "adamw");
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
}

constexpr int kFew = 40, kMany = 360;

}  // namespace adamw
}  // namespace race

using namespace race;

extern "C" int race_adamw(const race_adamw_desc_t* desc, const race_adamw_tensor_t* tensors,
                          int64_t count, cudaStream_t stream) {
  ApiCall call;
  if (desc == nullptr || count < 0 || (count > 0 && tensors == nullptr)) return RACE_ERR_INVALID;
  if (desc->state_bits != 8 && desc->state_bits != 32) return RACE_ERR_INVALID;
  if (!(desc->beta_one >= 0 && desc->beta_one < 1) || !(desc->beta_two >= 0 && desc->beta_two < 1) ||
      !(desc->eps >= 0))
    return RACE_ERR_INVALID;
  for (int64_t i = 0; i < count; ++i) {
    const race_adamw_tensor_t& t = tensors[i];
    if (t.numel < 0 || t.step < 0 || t.first % 8 != 0 || (t.dtype != RACE_F32 && t.dtype != RACE_BF16))
      return RACE_ERR_INVALID;
    if (t.numel == 0) continue;
    if (t.param == nullptr || t.grad == nullptr || t.exp_avg == nullptr || t.exp_avg_sq == nullptr)
      return RACE_ERR_INVALID;
    if (desc->state_bits == 8 && (t.exp_avg_scale == nullptr || t.exp_avg_sq_scale == nullptr))
      return RACE_ERR_INVALID;
    const int es = t.dtype == RACE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(t.param) % es != 0 || reinterpret_cast<uintptr_t>(t.grad) % es != 0 ||
        reinterpret_cast<uintptr_t>(t.exp_avg) % 16 != 0 || reinterpret_cast<uintptr_t>(t.exp_avg_sq) % 16 != 0 ||
        (desc->state_bits == 8 && (!api_aligned(t.exp_avg_scale, 4) || !api_aligned(t.exp_avg_sq_scale, 4))))
      return RACE_ERR_ALIGN;
  }
  if (count == 0) return RACE_OK;
  bool capturing = false;
  RACE_CALL(api_bind(stream, &capturing));
  if (capturing) {
    api_note("adamw: a graph would repeat this step's count, learning rate and noise; call it outside the capture");
    return RACE_ERR_UNSUPPORTED;
  }
  // 32-bit states take both types in one launch, 8-bit states one after the other
  for (int type = 0; type < (desc->state_bits == 8 ? 2 : 1); ++type) {
    int64_t pick[adamw::kMany];
    int n = 0;
    for (int64_t i = 0; i <= count; ++i) {
      if (i < count && tensors[i].numel > 0 &&
          (desc->state_bits == 32 || tensors[i].dtype == (type == 0 ? RACE_BF16 : RACE_F32)))
        pick[n++] = i;
      if (n == adamw::kMany || (i == count && n > 0)) {
        RACE_CALL(n <= adamw::kFew ? adamw::launch<adamw::kFew>(desc, tensors, pick, n, stream)
                                   : adamw::launch<adamw::kMany>(desc, tensors, pick, n, stream));
        n = 0;
      }
    }
  }
  return RACE_OK;
}
