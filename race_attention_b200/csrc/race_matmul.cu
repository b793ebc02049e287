// race_matmul.cu -- product of 8-bit operands with a float32 scale for each 128
// elements along the contraction, on the 5th-generation tensor cores.
//
//   y[m][n] = sum over blocks j of  sa[m][j] sb[n][j]  sum_{k in block j} a[m][k] b[n][k]
//
// The inner sum is one tcgen05 chain (kind::f8f6f4, 4 instructions of K = 32)
// into tensor memory; since the scales change with j, each 128-long partial is
// read back, scaled in 32 bits and added to a sum held in registers
// ("promoted"), while the tensor core already fills the other half of tensor memory.  Codes
// arrive by TMA with the 128-byte swizzle: a 128-byte row is one block, and one
// swizzle atom, of the contraction.  Rows and columns past the operands' ends
// arrive as zeros.
//
// k_mm_split: one 128 x NT tile per cluster of C CTAs which split the contraction;
// the weight (b) takes the M side of the instruction, so that few tokens waste
// little of it, and the C partial tiles are joined over distributed shared
// memory in the order of the ranks.  Products with few rows or few tiles go here.
//
// k_mm_pair: persistent pairs of CTAs, 256 x 256 tiles (tcgen05.mma.cta_group::2: each CTA
// brings 128 rows of both operands, so a block costs 32 KB of loads where a
// lone CTA's 128 x 256 tile costs 48).  Warp 0 loads, warp 1 of the first CTA issues the
// instructions, eight warps promote: a thread sums half a row of the tile, 128
// columns, in registers.  A block takes the tensor core 450 cycles (four
// instructions of 112) and the promotion 420, most of it loads from tensor memory;
// tensor memory holds two accumulators, so one block is promoted while the
// next is multiplied.  The way round takes 950 cycles a block: its completion is
// seen by the promoting warps of both CTAs some 300 cycles later, and the second
// CTA's arrival takes as long to come back; waits are four instructions long
// because each stands in that way.  At full load the power cap is the bound, at
// six blocks a tile too: 16384 x 8192 x 4096 takes 501 us from a cold start (2193 TFLOP/s,
// 1965 MHz) and 575 kept up (1910, 1480 MHz, 990 W), 65536 x 2304 x 768 162 us (1435,
// 1680 MHz, 1000 W); one 128 x 128 tile a CTA took 1551 for the first.  Sixteen promoting
// warps took 637 (they share the schedulers with the issuing warp), halves of 128
// columns with four accumulators 869, with an issuing warp each 535.  Where b has a
// scale for each row (dw) an element takes two multiplications in place of one, and
// promotion is the bound: 4736 x 4096 x 8192 231 us, with square blocks 159.  Results
// leave through shared memory by TMA, 128 bytes of a row at a time.
#include <atomic>

#include "race_api.h"
#include "race_lowp.cuh"
#include "race_t5.cuh"

namespace race {
namespace mm {

using namespace lowp;
using t5::bar_expect_tx;
using t5::bar_init;
using t5::bar_wait;
using t5::fence_after;
using t5::fence_before;
using t5::saddr;

constexpr int kPolls = 1 << 22;

struct Args {
  const float* sa; int64_t sar, sab;     // scales of a: rows of the result
  const float* sb; int64_t sbr, sbb;     // scales of b: columns of the result
  void* y; int64_t ldy; int ybf16;
  int64_t m, n;
  int kb;                                // 128-long blocks of the contraction
  int ranks;                             // k_mm_split: CTAs of a cluster
  int polls;
  unsigned* status;
};

// e4m3 x e4m3 -> fp32, both operands K-major
template <int M, int N>
__host__ __device__ constexpr uint32_t idesc8() {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void mma8(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc));
}

__device__ __forceinline__ void tma2(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                     uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

// One lane of a converged warp.  The code behind it keeps its descriptors and
// addresses in uniform registers, which the tensor core's and the copy engine's
// instructions take: behind `lane == 0` each instruction costs 70 cycles of
// moves instead.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0;
}
// Up to 64 polls in a loop of four instructions: the warps share their
// scheduler with promoting ones, each instruction of a wait costs them a turn.
__device__ __forceinline__ bool spin(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, 64;\n"
      "AGAIN:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra THROUGH;\n\t"
      "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra AGAIN;\n"
      "THROUGH:\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait; gives up early once another thread has (see bar_wait).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort, int polls) {
  if (polls >= 64) {
    if (spin(bar, parity)) return true;
    for (int i = 64; i < polls && *abort == 0; i += 64)
      if (spin(bar, parity)) return true;
    *abort = 1;
    return false;
  }
  return bar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(bar)), parity, abort, polls);
}

__device__ __forceinline__ void launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(saddr(bar)) : "memory");
}
__device__ __forceinline__ void bar_init_n(uint64_t* bar, int n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(saddr(bar)), "r"(n));
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t p;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(addr), "r"(rank));
  return p;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

__device__ __forceinline__ void put(const Args& a, int64_t row, int64_t col, float v) {
  if (a.ybf16)
    static_cast<bf16*>(a.y)[row * a.ldy + col] = from_f32<bf16>(v);
  else
    static_cast<float*>(a.y)[row * a.ldy + col] = v;
}

// The status word may lie in host memory; its bits are set by whole stores (a
// launch that fails reports from one thread per CTA, any of them will do).
__device__ __forceinline__ void report(unsigned* status, unsigned bits) {
  if (status == nullptr) return;
  volatile unsigned* w = status;
  *w = *w | bits;
  __threadfence_system();
}

// Waits, after a launch has given up and its instructions are done, for the arrivals
// of each barrier's last commit (the parity of an earlier one would be mistaken for
// a phase that never comes).
template <int S>
__device__ __forceinline__ bool settled(int sent, uint64_t* empty, uint64_t* tfull) {
  bool ok = true;
  for (int j = sent > S ? sent - S : 0; j < sent; ++j) {
    ok &= bar_wait(empty + j % S, (j / S) & 1);
    if (j >= sent - 2) ok &= bar_wait(tfull + (j & 1), (j >> 1) & 1);
  }
  return ok;
}

template <int NT>
struct Split {
  static constexpr int A = 128 * 128, B = NT * 128, STAGE = A + B;
  static constexpr int S = NT == 16 ? 5 : 4;                       // stages: two CTAs share an SM
  static constexpr int RED = NT * 128 * 4;                         // joined partial tile
  static constexpr int SCALES = S * STAGE;                         // [2][NT] floats
  static constexpr int BARS = SCALES + 2 * NT * 4;                 // full, empty [S]; tfull, tempty [2]; drain
  static constexpr int MISC = BARS + (2 * S + 5) * 8;              // tmem base, abort word, work that stays in flight
  static constexpr int BYTES = MISC + 16 + 1024;                   // + alignment
  static constexpr int COLS = 2 * NT < 32 ? 32 : 2 * NT;
  // Few tokens: a launch takes 4 us and its preparation one of them, which runs
  // while the launch before it ends (1 x 2304 x 768 4.1 -> 3.3 us in a row of launches,
  // 16 x 8192 x 8192 from memory 16.0 -> 15.0; 64 tokens lose, 8.3 -> 9.0).
  static constexpr bool EARLY = NT <= 32;
  static_assert(RED <= S * STAGE, "the partial tile takes the stages' place");
};

constexpr int kSplitThreads = 192;
constexpr int kMaxCluster = 8;

template <int NT, bool SQ>
__global__ void __launch_bounds__(kSplitThreads)
    k_mm_split(const __grid_constant__ CUtensorMap mapw, const __grid_constant__ CUtensorMap mapx,
               const Args a) {
  using L = Split<NT>;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = raw + ((1024 - (saddr(raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::BARS);
  uint64_t* empty = full + L::S;
  uint64_t* tfull = empty + L::S;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* misc = reinterpret_cast<uint32_t*>(sm + L::MISC);
  volatile uint32_t* abort = misc + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // ranks are a power of two; divisions by them would stand before the first load
  const int C = a.ranks, lc = __popc(C - 1), tile = (int)blockIdx.x >> lc, rank = (int)blockIdx.x & (C - 1);
  const int64_t n0 = (int64_t)blockIdx.y * 128, m0 = (int64_t)tile * NT;
  const int k0 = (int)((int64_t)a.kb * rank >> lc), k1 = (int)((int64_t)a.kb * (rank + 1) >> lc);
  const int blocks = k1 - k0;

  if (tid == 0) {
    for (int i = 0; i < L::S; ++i) {
      bar_init_n(full + i, 1);
      bar_init_n(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init_n(tfull + i, 1);
      bar_init_n(tempty + i, 4);
    }
    bar_init(drain);                                               // + the fence for all
    *abort = 0;
    misc[2] = 0;
  }
  if (warp == 1) t5::tmem_alloc<L::COLS>(misc);
  fence_before();
  __syncthreads();
  fence_after();
  if constexpr (L::EARLY) {
    // this CTA has its tensor memory, so the next launch's CTAs may take theirs;
    // its own inputs are complete once the launch before it is
    launch_dependents();
    wait_prerequisites();
  }
  const uint32_t tm = misc[0];
  const uint32_t full0 = saddr(full), empty0 = saddr(empty);
  float* red = reinterpret_cast<float*>(sm);                       // [NT][128]
  int sent = 0;                                                    // blocks whose copies (warp 0) or instructions (warp 1) are issued

  if (warp == 0) {
    const uint32_t dst = saddr(sm);
    bool ok = true;
    for (; sent < blocks; ++sent) {
      const int i = sent, s = i % L::S;
      if (i >= L::S) ok = wait(empty0 + 8 * s, ((i / L::S) - 1) & 1, abort, a.polls);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (elect()) {
        bar_expect_tx(full + s, L::STAGE);
        tma2(dst + s * L::STAGE, &mapw, (k0 + i) * 128, (int)n0, full0 + 8 * s);
        tma2(dst + s * L::STAGE + L::A, &mapx, (k0 + i) * 128, (int)m0, full0 + 8 * s);
      }
      __syncwarp();
    }
    // the last commits reach this CTA's barriers before it leaves
    for (int j = sent > L::S ? sent - L::S : 0; ok && j < sent; ++j)
      ok = wait(empty0 + 8 * (j % L::S), (j / L::S) & 1, abort, a.polls);
  } else if (warp == 1) {
    const uint64_t da = t5::desc_sw128(sm, 0), db = t5::desc_sw128(sm + L::A, 0);
    const uint32_t tempty0 = saddr(tempty);
    for (; sent < blocks; ++sent) {
      const int i = sent, s = i % L::S, b = i & 1;
      const bool ok = wait(full0 + 8 * s, (i / L::S) & 1, abort, a.polls) &&
                      (i < 2 || wait(tempty0 + 8 * b, ((i >> 1) - 1) & 1, abort, a.polls));
      if (!__all_sync(0xffffffffu, ok)) break;
      fence_after();
      if (elect()) {
        const uint64_t at = (uint64_t)(s * (L::STAGE >> 4));
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma8(tm + b * NT, da + at + 2 * ks, db + at + 2 * ks, idesc8<128, NT>(), ks > 0);
        t5::commit(tfull + b);
        t5::commit(empty + s);
      }
      __syncwarp();
    }
  } else {
    // row of the tile (weight row) = tensor-memory lane; columns = tokens
    const int quarter = warp & 3, row = 32 * quarter + lane, pt = tid - 64;
    const uint32_t lanes = tm + ((uint32_t)(32 * quarter) << 16), tf = saddr(tfull);
    float* sx = reinterpret_cast<float*>(sm + L::SCALES);
    const int64_t wr = SQ ? blockIdx.y : (n0 + row < a.n ? n0 + row : a.n - 1);
    const float* sw = a.sb + wr * a.sbr + k0 * a.sbb;
    const bool tok = pt < NT && m0 + pt < a.m;
    const float* sxg = a.sa + (tok ? m0 + pt : 0) * a.sar + k0 * a.sab;
    float nx = tok ? __ldg(sxg) : 0.f;
    float nw = __ldg(sw);
    float acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = 0.f;
    for (int i = 0; i < blocks; ++i) {
      const int b = i & 1;
      const float w = nw;
      float* sxb = sx + b * NT;
      if (pt < NT) sxb[pt] = nx;
      asm volatile("bar.sync 1, 128;" ::: "memory");               // the four warps, scales in place
      if (i + 1 < blocks) {
        if (tok) nx = __ldg(sxg + (i + 1) * a.sab);
        nw = __ldg(sw + (i + 1) * a.sbb);
      }
      // a wait that ran out leaves garbage here, which is not stored
      wait(tf + 8 * b, (i >> 1) & 1, abort, a.polls);
      __syncwarp();
      fence_after();
#pragma unroll
      for (int c = 0; c < NT; c += 16) {
        float v[16];
        t5::tld16(lanes + b * NT + c, v);
        t5::tld_wait();
        if (c + 16 == NT) {
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(tempty + b);
        }
#pragma unroll
        for (int q = 0; q < 16; q += 2) {
          const float2 s2 = __fmul2_rn(*reinterpret_cast<const float2*>(sxb + c + q), make_float2(w, w));
          const float2 r = __ffma2_rn(s2, make_float2(v[q], v[q + 1]), make_float2(acc[c + q], acc[c + q + 1]));
          acc[c + q] = r.x;
          acc[c + q + 1] = r.y;
        }
      }
    }
    // every copy into the stages has been used: they now hold the partial tile
    asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
    for (int j = 0; j < NT; ++j) red[j * 128 + row] = acc[j];
  }
  __syncthreads();
  const bool failed = *abort != 0;                                 // final: every role has ended
  if (failed) {
    // A wait ran out, this role's own or another's.  What is in flight ends before
    // the memory that it reaches is given back: the copies, then the instructions
    // (the lane that issued them commits once more) and their arrivals.
    bool ok = true;
    if (warp == 0) {
      for (int j = sent > L::S ? sent - L::S : 0; j < sent; ++j) ok &= bar_wait(full + j % L::S, (j / L::S) & 1);
    } else if (warp == 1) {
      if (elect()) t5::commit(drain);
      __syncwarp();
      ok = bar_wait(drain, 0) && settled<L::S>(sent, empty, tfull);
    }
    if (!ok) misc[2] = 1;
    __syncthreads();
    if (tid == 0) report(a.status, t5::kErrTimeout | (misc[2] != 0 ? t5::kErrStuck : 0));
  }
  if (warp == 1) t5::tmem_free<L::COLS>(tm);
  if (C > 1) cluster_sync();
  // The ranks share the tile's tokens; a thread joins four weight rows of one,
  // all partials on their way at once, summed in the order of the ranks.
  if (!failed) {
    const int q = tid & 31;
    const int64_t col = n0 + 4 * q;
    const bool vec = a.ldy % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && col + 4 <= a.n;
    const int64_t left = a.m - m0;
    const int rows = left < NT ? (int)left : NT;
    for (int j = rank + C * (tid >> 5); j < rows; j += C * (kSplitThreads / 32)) {
      const uint32_t at = saddr(red + j * 128 + 4 * q);
      float4 t;
      if (C == 1) {
        t = *reinterpret_cast<const float4*>(red + j * 128 + 4 * q);
      } else {
        float4 v[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < C) v[r] = ld_cluster4(map_rank(at, r));
        t = v[0];
#pragma unroll
        for (int r = 1; r < kMaxCluster; ++r)
          if (r < C) {
            t.x += v[r].x; t.y += v[r].y; t.z += v[r].z; t.w += v[r].w;
          }
      }
      if (vec && a.ybf16) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(t.x, t.y), hi = __floats2bfloat162_rn(t.z, t.w);
        *reinterpret_cast<uint2*>(static_cast<bf16*>(a.y) + (m0 + j) * a.ldy + col) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else if (vec) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.y) + (m0 + j) * a.ldy + col) = t;
      } else {
        const float e[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (col + z < a.n) put(a, m0 + j, col + z, e[z]);
      }
    }
  }
  if (C > 1) {
    __syncwarp();
    cluster_sync();                                                // peers may still be reading
  }
}

template <int NT>
int launch_split(const Args& a, const CUtensorMap& mw, const CUtensorMap& mx, bool square,
                 cudaStream_t s) {
  void (*fn)(CUtensorMap, CUtensorMap, Args) =
      square ? k_mm_split<NT, true> : k_mm_split<NT, false>;
  static std::atomic<uint64_t> ready[2];
  RACE_CALL(api_allow_smem(reinterpret_cast<const void*>(fn), Split<NT>::BYTES, ready[square]));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.ranks * ((a.m + NT - 1) / NT)), (unsigned)((a.n + 127) / 128));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = Split<NT>::BYTES;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)a.ranks;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = Split<NT>::EARLY ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, mw, mx, a);
  api_log("mm_split");
  return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
}

// ------------------------------------------------------------------ pairs of CTAs

struct PairArgs {
  Args a;
  int tiles_m, tiles_n;    // 256 x 256 tiles
  int splits;              // of the contraction
  uint32_t group_mul;      // x / (kGroup tiles_n) = x group_mul >> 32 >> group_shift
  int group_shift;
  float* part;             // splits > 1: [split][m][n] partial results
  int store;               // 1: results leave by TMA (map y), 0: element by element
};

constexpr int kPairThreads = 384;                                  // a warpgroup that loads and issues, two that promote
constexpr int kGroup = 8;                                          // row tiles walked together

template <bool SQ>
struct Pair {
  static constexpr int A = 128 * 128, STAGE = 2 * A;               // this CTA's rows of a and of b
  static constexpr int S = SQ ? 5 : 4;
  static constexpr int OUT = S * STAGE;                            // [8 warps][2] boxes of 32 x 128 bytes
  static constexpr int SCALES = OUT + 16 * 4096;                   // rows of b: [8 warps][2][128] floats
  static constexpr int BARS = SCALES + (SQ ? 0 : 8192);            // full, empty [S]; tfull, tempty [2]; drain
  static constexpr int MISC = BARS + (2 * S + 5) * 8;              // tmem base, abort word, blocks loaded, blocks multiplied,
  static constexpr int BYTES = MISC + 32 + 1024;                   // work that stays in flight
  static_assert(BYTES <= 232448, "227 KB of shared memory");
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// into this CTA's shared memory, counted by a barrier of either CTA of the pair
__device__ __forceinline__ void tma2_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma2_store(const CUtensorMap* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(src)
               : "memory");
}
__device__ __forceinline__ void store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void mma8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc));
}
// one arrival at the same barrier of both CTAs once the instructions so far are done
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          saddr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
struct Item {
  int m, n, k0, k1, split;
};
// blocks [k0, k1) of item i's contraction; whole contractions need no division
__device__ __forceinline__ void range_of(const PairArgs& p, int i, int& k0, int& k1) {
  if (p.splits == 1) {
    k0 = 0;
    k1 = p.a.kb;
  } else {
    const int split = i / (p.tiles_m * p.tiles_n);
    k0 = (int)((int64_t)p.a.kb * split / p.splits);
    k1 = (int)((int64_t)p.a.kb * (split + 1) / p.splits);
  }
}
__device__ __forceinline__ Item item_of(const PairArgs& p, int i) {
  const int tiles = p.tiles_m * p.tiles_n;
  Item t;
  t.split = p.splits == 1 ? 0 : i / tiles;
  const int r = i - t.split * tiles;
  const int g = (int)((((uint64_t)r * p.group_mul) >> 32) >> p.group_shift), first = g * kGroup;
  const int rows = min(kGroup, p.tiles_m - first), l = r - first * p.tiles_n;
  t.n = rows == kGroup ? l / kGroup : l / rows;
  t.m = first + l - t.n * rows;
  range_of(p, i, t.k0, t.k1);
  return t;
}

template <bool SQ>
__global__ void __launch_bounds__(kPairThreads, 1)
    k_mm_pair(const __grid_constant__ CUtensorMap mapa, const __grid_constant__ CUtensorMap mapb,
              const __grid_constant__ CUtensorMap mapy, const PairArgs p) {
  using L = Pair<SQ>;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = raw + ((1024 - (saddr(raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::BARS);
  uint64_t* empty = full + L::S;
  uint64_t* tfull = empty + L::S;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* misc = reinterpret_cast<uint32_t*>(sm + L::MISC);
  volatile uint32_t* abort = misc + 1;
  const Args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const int items = p.tiles_m * p.tiles_n * p.splits;

  if (tid == 0) {
    for (int i = 0; i < L::S; ++i) {
      bar_init_n(full + i, 1);
      bar_init_n(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init_n(tfull + i, 1);
      bar_init_n(tempty + i, 16);                                  // eight warps of both CTAs
    }
    bar_init(drain);
    misc[1] = 0;
    misc[2] = 0;
    misc[3] = 0;
    misc[4] = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(saddr(misc)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  const uint32_t tm = misc[0];

  // 384 x 168 registers at launch = 128 x 40 + 256 x 232
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    const uint32_t full0 = saddr(full), empty0 = saddr(empty);
    int s = 0;                                                     // stage, and its barriers' phase
    uint32_t ph = 0;
    bool ok = true;
    if (warp == 0) {
      const uint32_t dst = saddr(sm), bar0 = map_rank(full0, 0);
      int it = 0;
      for (int i = cluster; ok && i < items; i += clusters) {
        const Item t = item_of(p, i);
        const int ra = t.m * 256 + (int)rank * 128, rb = t.n * 256 + (int)rank * 128;
        for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
          if (it >= L::S) ok = wait(empty0 + 8 * s, ph ^ 1, abort, a.polls);
          if (!__all_sync(0xffffffffu, ok)) break;
          if (elect()) {
            if (rank == 0) bar_expect_tx(full + s, 2 * L::STAGE);
            tma2_pair(dst + s * L::STAGE, &mapa, kb * 128, ra, bar0 + 8 * s);
            tma2_pair(dst + s * L::STAGE + L::A, &mapb, kb * 128, rb, bar0 + 8 * s);
          }
          __syncwarp();
          if (++s == L::S) {
            s = 0;
            ph ^= 1;
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      if (lane == 0) misc[2] = it;
      // the last commits reach this CTA's barriers before it leaves
      for (int j = it > L::S ? it - L::S : 0; ok && j < it; ++j)
        ok = wait(empty0 + 8 * (j % L::S), (j / L::S) & 1, abort, a.polls);
    } else if (warp == 1 && rank == 0) {
      const uint64_t da = t5::desc_sw128(sm, 0), db = t5::desc_sw128(sm + L::A, 0);
      const uint32_t tempty0 = saddr(tempty);
      int it = 0;
      for (int i = cluster; ok && i < items; i += clusters) {
        int k0, k1;
        range_of(p, i, k0, k1);
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int b = it & 1;
          ok = wait(full0 + 8 * s, ph, abort, a.polls) &&
               (it < 2 || wait(tempty0 + 8 * b, ((it >> 1) - 1) & 1, abort, a.polls));
          if (!__all_sync(0xffffffffu, ok)) break;
          fence_after();
          if (elect()) {
            // a stage is 16-byte units further on, a K = 32 step 32 bytes inside the swizzle atom
            const uint64_t at = (uint64_t)(s * (L::STAGE >> 4));
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma8_pair(tm + b * 256, da + at + 2 * ks, db + at + 2 * ks, idesc8<256, 256>(), ks > 0);
            commit_pair(tfull + b);
            commit_pair(empty + s);
          }
          __syncwarp();
          if (++s == L::S) {
            s = 0;
            ph ^= 1;
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      if (lane == 0) misc[3] = it;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quarter = warp & 3, part = (warp - 4) >> 2, row = 32 * quarter + lane;
    const uint32_t lanes = tm + ((uint32_t)(32 * quarter) << 16) + 128 * part;
    const uint32_t te = map_rank(saddr(tempty), 0), tf = saddr(tfull);
    uint8_t* box = sm + L::OUT + (warp - 4) * 8192;
    float* sbs = reinterpret_cast<float*>(sm + L::SCALES) + 256 * (warp - 4);
    int it = 0;
    // A tile's scales: this thread's row of a, and of b the 128 columns' block
    // (square) or columns lane, 32 + lane, ...: each warp keeps its own copy of the
    // 128, so that no barrier stands between blocks.  The next tile and its first
    // scales are found during this one's first block: in the epilogue they would
    // stand in the way.
    constexpr int NB = SQ ? 1 : 4;
    const float *sa = nullptr, *nsa = nullptr, *sb[NB] = {}, *nsb[NB] = {};
    float na = 0.f, fa = 0.f, nb[NB] = {}, fb[NB] = {};
    Item next = item_of(p, cluster);
    const auto fetch = [&]() {
      const int64_t mr = (int64_t)next.m * 256 + rank * 128 + row, n0 = (int64_t)next.n * 256 + 128 * part;
      nsa = a.sa + (mr < a.m ? mr : a.m - 1) * a.sar + next.k0 * a.sab;
      fa = __ldg(nsa);
#pragma unroll
      for (int q = 0; q < NB; ++q) {
        nsb[q] = a.sb + (SQ ? min(n0, a.n - 1) / 128 : min(n0 + 32 * q + lane, a.n - 1)) * a.sbr + next.k0 * a.sbb;
        fb[q] = __ldg(nsb[q]);
      }
    };
    if (cluster < items) fetch();
    for (int i = cluster; i < items; i += clusters) {
      const Item t = next;
      const int64_t mr = (int64_t)t.m * 256 + rank * 128 + row;    // this thread's row of the result
      const int64_t n0 = (int64_t)t.n * 256 + 128 * part;          // its first column
      sa = nsa;
      na = fa;
#pragma unroll
      for (int q = 0; q < NB; ++q) {
        sb[q] = nsb[q];
        nb[q] = fb[q];
      }
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.f;
      for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
        const int b = it & 1;
        const float ca = na, cb = nb[0];
        float* sbb = sbs + 128 * b;
        if constexpr (!SQ) {
#pragma unroll
          for (int q = 0; q < NB; ++q) sbb[32 * q + lane] = nb[q];
          __syncwarp();
        }
        if (kb + 1 < t.k1) {
          sa += a.sab;
          na = __ldg(sa);
#pragma unroll
          for (int q = 0; q < NB; ++q) {
            sb[q] += a.sbb;
            nb[q] = __ldg(sb[q]);
          }
        }
        if (kb == t.k0 && i + clusters < items) {
          next = item_of(p, i + clusters);
          fetch();
        }
        // rows of b: 16 columns' scales at a time, read while the columns before them
        // are added (their latency would otherwise stand before each addition)
        float4 w[2][4];
        if constexpr (!SQ) {
#pragma unroll
          for (int q = 0; q < 4; ++q) w[0][q] = *reinterpret_cast<const float4*>(sbb + 4 * q);
        }
        // a wait that ran out leaves garbage here, which is not stored
        wait(tf + 8 * b, (it >> 1) & 1, abort, a.polls);
        __syncwarp();
        fence_after();
        const float sc = ca * cb;
        // the next 16 columns are on their way while these are added
        float v[2][16];
        t5::tld16(lanes + b * 256, v[0]);
#pragma unroll
        for (int c = 0; c < 128; c += 16) {
          const int cur = (c >> 4) & 1;
          t5::tld_wait();
          if (c < 112) {
            t5::tld16(lanes + b * 256 + c + 16, v[cur ^ 1]);
            if constexpr (!SQ) {
#pragma unroll
              for (int q = 0; q < 4; ++q) w[cur ^ 1][q] = *reinterpret_cast<const float4*>(sbb + c + 16 + 4 * q);
            }
          } else {
            fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(te + 8 * b);
          }
#pragma unroll
          for (int q = 0; q < 16; q += 2) {
            float2 s2 = make_float2(sc, sc);
            if constexpr (!SQ) {
              const float4 f = w[cur][q >> 2];
              s2 = __fmul2_rn(make_float2(ca, ca), q & 2 ? make_float2(f.z, f.w) : make_float2(f.x, f.y));
            }
            const float2 r = __ffma2_rn(s2, make_float2(v[cur][q], v[cur][q + 1]),
                                        make_float2(acc[c + q], acc[c + q + 1]));
            acc[c + q] = r.x;
            acc[c + q + 1] = r.y;
          }
        }
      }
      if (*abort != 0) continue;
      // Two boxes of 32 rows x 128 bytes at a time (bfloat16: all 128 columns), 16-byte
      // chunk c of row r at c ^ (r % 8).  They leave by TMA, or, where the result's
      // rows do not start on 16 bytes and for partial results (whose rows a ragged
      // tile must not leave), row by row with a lane to a column.
      const int r0 = (int)(mr - lane);
      const bool tma = p.splits == 1 && p.store;
      if (p.splits == 1 && a.ybf16) {
        if (lane == 0) store_wait_read();                          // the last tile's stores have read the boxes
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(acc[8 * c + 2 * q], acc[8 * c + 2 * q + 1]);
            w[q] = *reinterpret_cast<const uint32_t*>(&h);
          }
          *reinterpret_cast<uint4*>(box + (c >> 3) * 4096 + lane * 128 + (((c & 7) ^ (lane & 7)) << 4)) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (tma) {
          t5::fence_async_smem();
          __syncwarp();
          if (lane == 0 && r0 < a.m) {
            if (n0 < a.n) tma2_store(&mapy, (int)n0 * 2, r0, saddr(box));
            if (n0 + 64 < a.n) tma2_store(&mapy, (int)n0 * 2 + 128, r0, saddr(box) + 4096);
          }
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        } else {
          __syncwarp();
          bf16* o = static_cast<bf16*>(a.y) + r0 * a.ldy + n0;
          const int rows = (int)min((int64_t)32, a.m - r0), cols = (int)min((int64_t)128, a.n - n0);
          for (int r = 0; r < rows; ++r, o += a.ldy)
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const int c = lane + 32 * h;
              if (c < cols)
                o[c] = *reinterpret_cast<const bf16*>(box + (h >> 1) * 4096 + r * 128 +
                                                      ((((c >> 3) & 7) ^ (r & 7)) << 4) + (c & 7) * 2);
            }
          __syncwarp();
        }
      } else {
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          if (lane == 0) store_wait_read();
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 16; ++c)
            *reinterpret_cast<float4*>(box + (c >> 3) * 4096 + lane * 128 + (((c & 7) ^ (lane & 7)) << 4)) =
                make_float4(acc[32 * g + 4 * c], acc[32 * g + 4 * c + 1], acc[32 * g + 4 * c + 2],
                            acc[32 * g + 4 * c + 3]);
          const int64_t col = n0 + 32 * g;
          if (tma) {
            t5::fence_async_smem();
            __syncwarp();
            if (lane == 0 && r0 < a.m) {
              if (col < a.n) tma2_store(&mapy, (int)col * 4, r0, saddr(box));
              if (col + 32 < a.n) tma2_store(&mapy, (int)col * 4 + 128, r0, saddr(box) + 4096);
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          } else {
            __syncwarp();
            const int64_t ld = p.splits > 1 ? a.n : a.ldy;
            float* o = (p.splits > 1 ? p.part + (int64_t)t.split * a.m * a.n : static_cast<float*>(a.y)) + r0 * ld + col;
            const int rows = (int)min((int64_t)32, a.m - r0), cols = (int)min((int64_t)64, a.n - col);
            for (int r = 0; r < rows; ++r, o += ld)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (lane + 32 * h < cols)
                  o[lane + 32 * h] = *reinterpret_cast<const float*>(box + h * 4096 + r * 128 +
                                                                     (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
            __syncwarp();
          }
        }
      }
    }
    if (lane == 0) store_wait_read();
  }
  __syncthreads();
  cluster_sync();
  // Every role of both CTAs has ended.  Where a wait of either ran out, what is in
  // flight ends before one of them leaves or gives memory back.
  const bool mine = *abort != 0;
  const uint32_t other = ld_cluster_u32(map_rank(saddr(misc + 1), rank ^ 1));
  if (mine || other != 0) {                                        // the same for the pair
    bool ok = true;
    if (warp == 0 && rank == 0 && lane == 0) {
      // the copies: the first CTA's barriers count both CTAs' bytes, so it settles
      // what only one of them issued
      const int i0 = (int)misc[2], i1 = (int)ld_cluster_u32(map_rank(saddr(misc + 2), 1));
      const int lo = min(i0, i1), hi = max(i0, i1);
      for (int j = lo; j < hi; ++j) {
        uint64_t* f = full + j % L::S;
        if (j < i0)
          asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(saddr(f)),
                       "r"(L::STAGE)
                       : "memory");
        else
          bar_expect_tx(f, L::STAGE);
      }
      for (int j = hi > L::S ? hi - L::S : 0; j < hi; ++j) ok &= bar_wait(full + j % L::S, (j / L::S) & 1);
    } else if (warp == 1) {
      // the instructions (the lane that issued them commits once more) and their
      // arrivals at both CTAs' barriers
      if (rank == 0 && elect()) commit_pair(drain);
      __syncwarp();
      ok = bar_wait(drain, 0) && settled<L::S>((int)ld_cluster_u32(map_rank(saddr(misc + 3), 0)), empty, tfull);
    }
    if (!ok) misc[4] = 1;
    __syncthreads();
    if (tid == 0) report(a.status, (mine ? t5::kErrTimeout : 0) | (misc[4] != 0 ? t5::kErrStuck : 0));
  }
  __syncthreads();
  cluster_sync();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tm));
}

// result = sum over the splits of their partial results, in their order
__global__ void __launch_bounds__(256) k_mm_join(const float* __restrict__ part, int splits, const Args a) {
  const int64_t total = a.m * a.n;
  const int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (i >= total) return;
  if (total % 4 == 0) {                      // then every split starts on 16 bytes
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(part + s * total + i));
      t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
    }
    const float r[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) put(a, (i + j) / a.n, (i + j) % a.n, r[j]);
  } else {
    for (int64_t e = i; e < i + 4 && e < total; ++e) {
      float t = 0.f;
      for (int s = 0; s < splits; ++s) t += part[s * total + e];
      put(a, e / a.n, e % a.n, t);
    }
  }
}

template <bool SQ>
int launch_pair(const PairArgs& p, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& my,
                cudaStream_t s) {
  static std::atomic<uint64_t> ready;
  RACE_CALL(api_allow_smem(reinterpret_cast<const void*>(&k_mm_pair<SQ>), Pair<SQ>::BYTES, ready));
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.splits;
  const int64_t pairs = api_sm_count() / 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2u * (unsigned)(items < pairs ? items : pairs));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = Pair<SQ>::BYTES;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, &k_mm_pair<SQ>, ma, mb, my, p);
  api_log("mm_pair");
  if (e == cudaSuccess && p.splits > 1) {
    const int64_t quads = (p.a.m * p.a.n + 3) / 4;
    k_mm_join<<<(unsigned)((quads + 255) / 256), 256, 0, s>>>(p.part, p.splits, p.a);
    api_log("mm_join");
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
}

// How a product is cut: the cheaper of the two kernels by their measured times
// (148 SMs, operands in L2; kb = blocks of the contraction).
//   k_mm_split: 4 us and 0.39 us a block while every CTA has an SM; beyond that 330
//     tile-blocks a us, a tile's start and end as long as 2.5 of its blocks
//     (1024 x 2304 x 768 7.8 us, 2048 x 1536 x 768 12.2, 16384 x 384 x 384 14.5).  Joining a
//     cluster's ranks costs 1.6 us for 64 tokens and 0.4 us for 16, eight ranks 0.4 more;
//     each rank taken off saves its blocks (33 x 768 x 3000 7.0 us for 4 ranks, 6.0 for 8;
//     16 x 8192 x 8192 25.8, 15.5, 11.7, 16.0 for 1, 2, 4, 8).  Two of a cluster's ranks on one SM
//     start 1.7 us later and take 0.48 us a block, eight of them join in 1.6 us more:
//     that pays where a rank keeps many blocks (128 x 8192 x 8192 22.4 us against 29.5 without,
//     256 x 4096 x 4096 14.5 and 16.7, 256 x 2304 x 768 11.0 and 6.3).
//   k_mm_pair: 6.4 us, and 0.45 us a block and 1 us a tile for every round of the 74
//     pairs (2048 x 1536 x 768 8.9 us, 1024 x 4096 x 4096 20.2); a contraction cut in
//     s adds 2.5 us and the partial results' way at 5 TB/s.
struct Plan {
  bool pair;
  int nt, c;               // k_mm_split: token columns of a tile, CTAs of a cluster
  int tiles_m, tiles_n, splits;
};

Plan plan_of(int64_t m, int64_t n, int64_t k) {
  Plan p{};
  const int64_t kb = (k + 127) / 128, sms = api_sm_count(), pairs = sms / 2;
  p.nt = m <= 16 ? 16 : m <= 32 ? 32 : 64;
  const double join = p.nt == 64 ? 1.6 : 0.4;
  const int64_t tiles = ((n + 127) / 128) * ((m + p.nt - 1) / p.nt);
  double split = 1e30, pair = 1e30;
  for (int c = 1; c <= kMaxCluster && 2 * c <= 3 * kb; c *= 2) {
    if (c > 1 && tiles * c > 2 * sms) break;
    const bool two = p.nt == 64 && c > 1 && tiles * c > sms;         // CTAs of one SM
    const double each = 4.0 + (two ? 1.7 : 0.0) + (two ? 0.48 : 0.39) * (double)((kb + c - 1) / c) +
                        (c > 1 ? join : 0.0) + (c > 4 ? (two ? 1.6 : 0.4) : 0.0);
    const double all = 2.0 + (double)tiles * ((double)kb + 2.5) / 330.0 * (p.nt == 64 ? 1.0 : 0.5);
    const double t = each > all ? each : all;
    if (t < split) {
      split = t;
      p.c = c;
    }
  }
  p.tiles_m = (int)((m + 255) / 256);
  p.tiles_n = (int)((n + 255) / 256);
  p.splits = 1;
  const int64_t big = (int64_t)p.tiles_m * p.tiles_n;
  if (m > 128 && n > 128)
    for (int s = 1; s <= 32 && s <= kb && (s == 1 || big < 4 * pairs); ++s) {
      const double rounds = (double)((big * s + pairs - 1) / pairs);
      const double t = 6.4 + rounds * (0.45 * (double)((kb + s - 1) / s) + 1.0) +
                       (s > 1 ? 2.5 + s * (double)(m * n) * 4 / 5e6 : 0.0);
      if (t < pair) {
        pair = t;
        p.splits = s;
      }
    }
  p.pair = pair < split;
  return p;
}

int check(const race_matmul_desc_t* d) {
  if (d == nullptr || d->m < 0 || d->n < 0 || d->k < 0 || d->wait_polls < 0) return RACE_ERR_INVALID;
  if (d->out_dtype != RACE_F32 && d->out_dtype != RACE_BF16) return RACE_ERR_INVALID;
  if (d->m > (int64_t(1) << 30) || d->n > (int64_t(1) << 22) || d->k > (int64_t(1) << 30)) {
    api_note("matmul: m or k above 2^30, n above 2^22");
    return RACE_ERR_UNSUPPORTED;
  }
  return RACE_OK;
}

int check_operand(race_blocks_t b, int64_t rows, int64_t k) {
  if (b.codes == nullptr || b.scales == nullptr) return RACE_ERR_INVALID;
  if (!api_aligned(b.codes, 16) || b.ld % 16 != 0 || b.ld <= 0 || !api_aligned(b.scales, 4)) return RACE_ERR_ALIGN;
  return b.ld >= k || rows <= 1 ? RACE_OK : RACE_ERR_INVALID;
}

}  // namespace mm
}  // namespace race

using namespace race;

extern "C" size_t race_scaled_matmul_workspace(const race_matmul_desc_t* desc) {
  if (mm::check(desc) != RACE_OK || desc->m == 0 || desc->n == 0 || desc->k == 0) return 0;
  const mm::Plan p = mm::plan_of(desc->m, desc->n, desc->k);
  return p.pair && p.splits > 1 ? (size_t)p.splits * (size_t)desc->m * (size_t)desc->n * sizeof(float) : 0;
}

extern "C" int race_scaled_matmul(const race_matmul_desc_t* desc, race_blocks_t a, race_blocks_t b,
                                  race_rows_t result, uint32_t* status, void* workspace,
                                  size_t workspace_bytes, cudaStream_t stream) {
  ApiCall call;
  RACE_CALL(mm::check(desc));
  if (desc->m == 0 || desc->n == 0) return RACE_OK;
  const int es = desc->out_dtype == RACE_F32 ? 4 : 2;
  if (result.data == nullptr || (desc->m > 1 && result.ld < desc->n)) return RACE_ERR_INVALID;
  if (!api_aligned(result.data, es) || !api_aligned(status, 4)) return RACE_ERR_ALIGN;
  if (desc->k > 0) {
    RACE_CALL(mm::check_operand(a, desc->m, desc->k));
    RACE_CALL(mm::check_operand(b, desc->n, desc->k));
    if (!api_aligned(workspace, 16)) return RACE_ERR_ALIGN;          // partial results are read four at a time
  }
  RACE_CALL(api_bind(stream));
  if (desc->k == 0) {   // an empty sum
    const cudaError_t e = cudaMemset2DAsync(result.data, (size_t)(desc->m > 1 ? result.ld : desc->n) * es, 0,
                                            (size_t)desc->n * es, (size_t)desc->m, stream);
    return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
  }
  mm::Args g{a.scales, a.stride_row, a.stride_block, b.scales, b.stride_row, b.stride_block,
             result.data, result.ld, desc->out_dtype == RACE_BF16, desc->m, desc->n,
             (int)((desc->k + 127) / 128), 1, desc->wait_polls > 0 ? desc->wait_polls : mm::kPolls, status};
  const mm::Plan plan = mm::plan_of(desc->m, desc->n, desc->k);
  g.ranks = plan.c;
  const bool square = desc->b_square != 0;
  CUtensorMap ma, mb;
  if (plan.pair) {
    const size_t need = plan.splits > 1 ? (size_t)plan.splits * desc->m * desc->n * sizeof(float) : 0;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return RACE_ERR_WORKSPACE;
    CUtensorMap my;
    const bool store = reinterpret_cast<uintptr_t>(result.data) % 16 == 0 && result.ld * es % 16 == 0;
    if (!api_encode_bytes(&ma, a.codes, desc->m, desc->k, a.ld, 128) ||
        !api_encode_bytes(&mb, b.codes, desc->n, desc->k, b.ld, 128) ||
        !(store ? api_encode_bytes(&my, result.data, desc->m, desc->n * es, result.ld * es, 32)
                : api_encode_bytes(&my, a.codes, desc->m, desc->k, a.ld, 32)))
      return RACE_ERR_UNSUPPORTED;
    // x / d for 0 <= x < 2^31: with 2^s < d <= 2^(s + 1), mul = ceil(2^(32 + s) / d) < 2^32
    const uint64_t d = (uint64_t)mm::kGroup * plan.tiles_n;
    int shift = 0;
    while ((uint64_t(2) << shift) < d) ++shift;
    const uint32_t mul = (uint32_t)(((uint64_t(1) << (32 + shift)) + d - 1) / d);
    const mm::PairArgs p{g, plan.tiles_m, plan.tiles_n, plan.splits, mul, shift,
                         static_cast<float*>(workspace), store};
    return square ? mm::launch_pair<true>(p, ma, mb, my, stream)
                  : mm::launch_pair<false>(p, ma, mb, my, stream);
  }
  if (!api_encode_bytes(&mb, b.codes, desc->n, desc->k, b.ld, 128) ||
      !api_encode_bytes(&ma, a.codes, desc->m, desc->k, a.ld, plan.nt))
    return RACE_ERR_UNSUPPORTED;
  switch (plan.nt) {
    case 16: return mm::launch_split<16>(g, mb, ma, square, stream);
    case 32: return mm::launch_split<32>(g, mb, ma, square, stream);
    default: return mm::launch_split<64>(g, mb, ma, square, stream);
  }
}
