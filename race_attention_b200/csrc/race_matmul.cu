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
// memory in the order of the ranks.  Few launches' worth of tiles, or few rows, go here.
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
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t p;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(p) : "memory");
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

template <int NT>
struct Split {
  static constexpr int A = 128 * 128, B = NT * 128, STAGE = A + B;
  static constexpr int S = NT >= 128 ? 6 : 5;                      // stages
  static constexpr int RED = NT * 128 * 4;                         // joined partial tile
  static constexpr int DATA = S * STAGE > RED ? S * STAGE : RED;
  static constexpr int SCALES = DATA;                              // [2][NT] floats
  static constexpr int BARS = SCALES + 2 * NT * 4;                 // full, empty [S]; tfull, tempty [2]; drain
  static constexpr int MISC = BARS + (2 * S + 5) * 8;              // tmem base, abort word
  static constexpr int BYTES = MISC + 16 + 1024;                   // + alignment
  static constexpr int COLS = 2 * NT < 32 ? 32 : 2 * NT;
};

constexpr int kSplitThreads = 192;

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
  const int C = (int)gridDim.x, rank = (int)blockIdx.x;            // the cluster spans x
  const int64_t n0 = (int64_t)blockIdx.y * 128, m0 = (int64_t)blockIdx.z * NT;
  const int k0 = (int)((int64_t)a.kb * rank / C), k1 = (int)((int64_t)a.kb * (rank + 1) / C);
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
  }
  if (warp == 1) t5::tmem_alloc<L::COLS>(misc);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tm = misc[0];

  float acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = 0.f;

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < blocks; ++i) {
        const int s = i % L::S;
        if (i >= L::S && !bar_wait(empty + s, ((i / L::S) - 1) & 1, abort, a.polls)) break;
        bar_expect_tx(full + s, L::STAGE);
        const uint32_t dst = saddr(sm) + s * L::STAGE;
        tma2(dst, &mapw, (k0 + i) * 128, (int)n0, saddr(full + s));
        tma2(dst + L::A, &mapx, (k0 + i) * 128, (int)m0, saddr(full + s));
      }
      if (i < blocks)                                              // gave up: copies in flight land first
        for (int j = i > L::S ? i - L::S : 0; j < i; ++j)
          if (!bar_wait(full + j % L::S, (j / L::S) & 1)) report(a.status, t5::kErrStuck);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int i = 0;
      for (; i < blocks; ++i) {
        const int s = i % L::S, b = i & 1;
        if (i >= 2 && !bar_wait(tempty + b, ((i >> 1) - 1) & 1, abort, a.polls)) break;
        if (!bar_wait(full + s, (i / L::S) & 1, abort, a.polls)) break;
        fence_after();
        const uint8_t* st = sm + s * L::STAGE;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma8(tm + b * NT, t5::desc_sw128(st, ks), t5::desc_sw128(st + L::A, ks), idesc8<128, NT>(),
               ks > 0);
        t5::commit(empty + s);
        t5::commit(tfull + b);
      }
      if (i < blocks) {
        t5::commit(drain);
        if (!bar_wait(drain, 0)) report(a.status, t5::kErrStuck);
      }
    }
  } else {
    // row of the tile (weight row) = tensor-memory lane; columns = tokens
    const int quarter = warp & 3, row = 32 * quarter + lane, pt = tid - 64;
    float* sx = reinterpret_cast<float*>(sm + L::SCALES);
    const int64_t wr = SQ ? blockIdx.y : (n0 + row < a.n ? n0 + row : a.n - 1);
    const float* sw = a.sb + wr * a.sbr + k0 * a.sbb;
    const bool tok = pt < NT && m0 + pt < a.m;
    const float* sxg = a.sa + (tok ? m0 + pt : 0) * a.sar + k0 * a.sab;
    float nx = tok && blocks > 0 ? __ldg(sxg) : 0.f;
    float nw = blocks > 0 ? __ldg(sw) : 0.f;
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
      // a thread that gives up leaves through the same barriers as the rest
      const bool ok = bar_wait(tfull + b, (i >> 1) & 1, abort, a.polls);
      if (__any_sync(0xffffffffu, !ok)) continue;
      fence_after();
      constexpr int G = NT < 32 ? NT : 32;
#pragma unroll
      for (int c = 0; c < NT; c += G) {
        float v[G];
#pragma unroll
        for (int q = 0; q < G; q += 16) {
          float (&vq)[16] = *reinterpret_cast<float (*)[16]>(&v[q]);
          t5::tld16(tm + ((uint32_t)(32 * quarter) << 16) + b * NT + c + q, vq);
        }
        t5::tld_wait();
        if (c + G == NT) {
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(tempty + b);
        }
#pragma unroll
        for (int q = 0; q < G; q += 4) {
          const float4 s4 = *reinterpret_cast<const float4*>(sxb + c + q);
          acc[c + q] = fmaf(s4.x * w, v[q], acc[c + q]);
          acc[c + q + 1] = fmaf(s4.y * w, v[q + 1], acc[c + q + 1]);
          acc[c + q + 2] = fmaf(s4.z * w, v[q + 2], acc[c + q + 2]);
          acc[c + q + 3] = fmaf(s4.w * w, v[q + 3], acc[c + q + 3]);
        }
      }
    }
  }
  __syncthreads();
  const bool failed = *abort != 0;
  if (failed && tid == 0) report(a.status, t5::kErrTimeout);
  if (warp == 1) t5::tmem_free<L::COLS>(tm);

  const int quarter = warp & 3, row = 32 * quarter + lane;
  const int64_t col = n0 + row;
  if (C == 1) {
    if (warp >= 2 && col < a.n && !failed) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (m0 + j < a.m) put(a, m0 + j, col, acc[j]);
    }
    return;
  }
  // every copy into the stages has been used: they now hold the partial tile
  float* red = reinterpret_cast<float*>(sm);
  if (warp >= 2) {
#pragma unroll
    for (int j = 0; j < NT; ++j) red[j * 128 + row] = acc[j];
  }
  __syncwarp();
  cluster_sync();
  if (warp >= 2 && !failed) {
    for (int j = rank; j < NT; j += C) {
      if (m0 + j >= a.m) break;
      float t = 0.f;
      for (int r = 0; r < C; ++r) t += ld_cluster(saddr(red + j * 128 + row), r);
      if (col < a.n) put(a, m0 + j, col, t);
    }
  }
  __syncwarp();
  cluster_sync();                                                  // peers may still be reading
}

// Opts a kernel in to its shared memory, once on each device.
int allow_smem(const void* fn, int bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return api_cuda_fail(e);
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (ready.load(std::memory_order_relaxed) & bit) return RACE_OK;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return api_cuda_fail(e);
  ready.fetch_or(bit, std::memory_order_relaxed);
  return RACE_OK;
}

template <int NT>
int launch_split(const Args& a, const CUtensorMap& mw, const CUtensorMap& mx, bool square, int c,
                 cudaStream_t s) {
  void (*fn)(CUtensorMap, CUtensorMap, Args) =
      square ? k_mm_split<NT, true> : k_mm_split<NT, false>;
  static std::atomic<uint64_t> ready[2];
  RACE_CALL(allow_smem(reinterpret_cast<const void*>(fn), Split<NT>::BYTES, ready[square]));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)c, (unsigned)((a.n + 127) / 128), (unsigned)((a.m + NT - 1) / NT));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = Split<NT>::BYTES;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)c;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, mw, mx, a);
  api_log("mm_split");
  return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
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
  if (reinterpret_cast<uintptr_t>(b.codes) % 16 != 0 || b.ld % 16 != 0 || b.ld <= 0)
    return RACE_ERR_ALIGN;
  return b.ld >= k || rows <= 1 ? RACE_OK : RACE_ERR_INVALID;
}

}  // namespace mm
}  // namespace race

using namespace race;

extern "C" size_t race_scaled_matmul_workspace(const race_matmul_desc_t* desc) {
  return mm::check(desc) == RACE_OK ? 0 : 0;
}

extern "C" int race_scaled_matmul(const race_matmul_desc_t* desc, race_blocks_t a, race_blocks_t b,
                                  race_rows_t result, uint32_t* status, void* workspace,
                                  size_t workspace_bytes, cudaStream_t stream) {
  (void)workspace;
  (void)workspace_bytes;
  ApiCall call;
  RACE_CALL(mm::check(desc));
  if (desc->m == 0 || desc->n == 0) return RACE_OK;
  const int es = desc->out_dtype == RACE_F32 ? 4 : 2;
  if (result.data == nullptr || (desc->m > 1 && result.ld < desc->n)) return RACE_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(result.data) % es != 0) return RACE_ERR_ALIGN;
  RACE_CALL(api_bind(stream));
  if (desc->k == 0) {   // an empty sum
    const cudaError_t e = cudaMemset2DAsync(result.data, (size_t)(desc->m > 1 ? result.ld : desc->n) * es, 0,
                                            (size_t)desc->n * es, (size_t)desc->m, stream);
    return e == cudaSuccess ? RACE_OK : api_cuda_fail(e);
  }
  RACE_CALL(mm::check_operand(a, desc->m, desc->k));
  RACE_CALL(mm::check_operand(b, desc->n, desc->k));
  mm::Args g{a.scales, a.stride_row, a.stride_block, b.scales, b.stride_row, b.stride_block,
             result.data, result.ld, desc->out_dtype == RACE_BF16, desc->m, desc->n,
             (int)((desc->k + 127) / 128), desc->wait_polls > 0 ? desc->wait_polls : mm::kPolls, status};
  const int nt = desc->m <= 16 ? 16 : desc->m <= 32 ? 32 : desc->m <= 64 ? 64 : 128;
  CUtensorMap mw, mx;
  if (!api_encode_bytes(&mw, b.codes, desc->n, desc->k, b.ld, 128) ||
      !api_encode_bytes(&mx, a.codes, desc->m, desc->k, a.ld, nt))
    return RACE_ERR_UNSUPPORTED;
  // split the contraction while the tiles leave SMs idle
  const int64_t tiles = ((desc->n + 127) / 128) * ((desc->m + nt - 1) / nt);
  int c = 1;
  while (c < 8 && tiles * c * 2 <= 2 * (int64_t)api_sm_count() && c * 2 <= g.kb) c *= 2;
  if ((desc->m + nt - 1) / nt > 65535 || (desc->n + 127) / 128 > 65535) {
    api_note("matmul: more than 65535 tiles along one side");
    return RACE_ERR_UNSUPPORTED;
  }
  switch (nt) {
    case 16: return mm::launch_split<16>(g, mw, mx, desc->b_square != 0, c, stream);
    case 32: return mm::launch_split<32>(g, mw, mx, desc->b_square != 0, c, stream);
    case 64: return mm::launch_split<64>(g, mw, mx, desc->b_square != 0, c, stream);
    default: return mm::launch_split<128>(g, mw, mx, desc->b_square != 0, c, stream);
  }
}
