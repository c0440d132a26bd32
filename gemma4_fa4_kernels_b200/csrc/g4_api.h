// What the C-ABI files share: error reporting, launch accounting, device facts.
// Defined in capi.cu.
#pragma once

#include <cuda_runtime.h>

namespace g4 {

// Kernel ids of g4_launch_count / g4_profile_read (names: capi.cu).
enum KernelId {
  kKFwd = 0,
  kKBwdPre,
  kKBwdDq,
  kKBwdDkv,
  kKPlan,
  kKMask,
  kKScore,
  kKGemmDv,
  kKGemmDk,
  kKGemmDq,
  kKFwdScore,
  kKFwdPv,
  kKDecode,
  kKDecodeCombine,
  kKPrepFwd,
  kKPrepBwd,
  kKPrepDw,
  kKSelftest,
  kKGemmDvDk,
  kKCast,
  kKMerge,
  kKAdd,
  kKDecodeShort,
  kKReset,
  kKKv8Attn,
  kKKv8Merge,
  kKKv8Append,
  kKKv8Read,
  kKKv8Chunk,
  kKPagesPlan,
  kKPagesApply,
  kKCount
};

// Brackets one launch: counts it and, when profiling, records events around it.
class LaunchScope {
 public:
  LaunchScope(int id, cudaStream_t st);
  ~LaunchScope();

 private:
  int id_;
  cudaStream_t st_;
  cudaEvent_t a_{}, b_{};
  bool timed_ = false;
};

// Record the calling thread's last error; both return the status to hand back.
int api_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int api_cuda_fail(cudaError_t e, const char* what);
void api_clear_error();
// SM count of the current device (148 when no device is visible).
int api_sm_count();

}  // namespace g4
