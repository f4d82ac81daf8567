// Arguments shared by the kernels of q4k_paged_attention.
#pragma once
#include <stdint.h>

#include "kv_cache.cuh"

namespace q4k {

constexpr uint32_t kAttendMaxCtas = 512;  // two counters each; kMergeGroup^2 parts and more
static_assert(2 * kAttendMaxCtas <= kSplitCounters, "arrival counters");

struct AttendArgs {
  KvCache c;
  KvBatch b;
  const void* q;
  void* out;
  uint64_t q_stride, out_stride;
  uint32_t group;     // query heads per key head
  uint32_t window;    // 0: none
  uint32_t max_rows;  // sequences with more rows a key head are another kernel's (0: none are)
  float scale_log2;   // softmax scale * log2(e)
  float* work;        // parts of cut units: 2 per CTA
  size_t work_bytes;
  uint32_t* counters;
  uint32_t* status;
};

// Rows of a sequence and key head above which the prompt kernel takes it.
constexpr uint32_t kPromptRows = 64;

// The prompt kernel (kv_prompt.cu): sequences with more than a.max_rows rows, f16 and bf16.
cudaError_t launch_prompt(const AttendArgs& a, uint32_t dtype, uint32_t spin, int device, cudaStream_t s);

}  // namespace q4k
