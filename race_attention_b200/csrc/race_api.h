// race_api.h -- what the entry points in other translation units share with
// race_capi.cu: the call scope (kernel log, error text), the binding of the
// stream's device and the tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "race_b200.h"

namespace race {

void api_begin();
void api_end();
// Makes the stream's device current; *capturing: whether the stream is being captured.
int api_bind(cudaStream_t stream, bool* capturing = nullptr);
int api_cuda_fail(cudaError_t e);             // records the text, returns RACE_ERR_CUDA
void api_log(const char* kernel);             // adds a launch to race_last_kernels()
int api_sm_count();
void api_note(const char* text);              // text behind RACE_ERR_UNSUPPORTED

// The outermost entry point of a call opens one of these.
struct ApiCall {
  ApiCall() { api_begin(); }
  ~ApiCall() { api_end(); }
  ApiCall(const ApiCall&) = delete;
  ApiCall& operator=(const ApiCall&) = delete;
};

// 2-D tensor map of bytes: `cols` bytes a row, rows `ld` bytes apart, boxes of
// box_rows x 128 bytes with the 128-byte swizzle, zeros outside.
bool api_encode_bytes(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld,
                      int box_rows);

// Opts a kernel in to its shared memory, once on each device.
inline int api_allow_smem(const void* fn, int bytes, std::atomic<uint64_t>& ready) {
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

// p lies on a multiple of `bytes` (a null pointer does)
inline bool api_aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

#define RACE_CALL(x)                 \
  do {                               \
    const int rc_ = (x);             \
    if (rc_ != RACE_OK) return rc_;  \
  } while (0)

}  // namespace race
