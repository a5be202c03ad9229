// fqkv_kv4.cuh -- parameter blocks and host launcher declarations of the paged 4-bit
// key/value cache (layout: include/fused_rmsnorm_qkv.h, fqkv_kv4_cache).
#pragma once

#include <cuda_runtime.h>

#include "fqkv_device.cuh"

namespace fqkv {

constexpr int kKv4Rec = 16;           // tokens per record
constexpr int kKv4CounterBytes = 4096;  // arrival counters at the head of the attention workspace
constexpr int kKv4MaxGrid = 320;      // CTAs of the split attention kernel, at most
constexpr int kKv4PromptMaxGrid = 160;  // and of the prompt kernel

// A record's byte offsets for head_dim D and NG groups: keys at 0, values at 8 D, the keys'
// parameters at 16 D, the values' at 16 D + 64 NG.
__host__ __device__ constexpr int kv4_record_bytes(int D, int NG) { return 16 * D + 128 * NG; }

struct Kv4Cache {
  uint8_t* data;
  int64_t n_blocks;
  int n_kv, D, P, group;
};

struct Kv4PlanParams {
  const int* ctx;
  const int* add;
  int64_t R;
  int* table;
  int64_t table_stride, width;
  const int* free_blocks;
  int64_t free_capacity;
  const int* n_free;
  int P;
  int64_t T;
  int *query_start, *positions, *slots, *seq_lens, *n_free_out, *refused;
};

struct Kv4AppendParams {
  Kv4Cache c;
  const uint16_t *k, *v;
  int64_t k_b, k_s, k_h, v_b, v_s, v_h;  // element strides
  int64_t T, S;
  const int* slots;
};

struct Kv4GatherParams {
  Kv4Cache c;
  uint16_t *k, *v;
  int64_t T;
  const int* slots;
};

struct Kv4AttnParams {
  Kv4Cache c;
  const uint16_t* q;
  int64_t q_r, q_t, q_h;          // element strides
  const int* query_start;         // nullable: every request has S queries
  int64_t T, S;
  int R, n_q, G;                  // G = query heads per KV head
  const int* table;
  int64_t table_stride;
  int width;
  const int* seq_lens;
  int window;                     // 0: none
  float scale_log2;               // score scale * log2(e)
  uint16_t* out;
  int64_t o_t;
  int* counters;
  float* partial;
  int withhold;                   // FQKV_FLAG_TEST_WITHHOLD: one arrival of CTA 0 is left out
};

cudaError_t launch_kv4_plan(const Kv4PlanParams& p, bool pdl, cudaStream_t stream);
cudaError_t launch_kv4_append(const Kv4AppendParams& p, bool bf16, bool pdl, cudaStream_t stream);
cudaError_t launch_kv4_gather(const Kv4GatherParams& p, bool bf16, bool pdl, cudaStream_t stream);
cudaError_t launch_kv4_attn_split(const Kv4AttnParams& p, int sms, bool bf16, bool pdl, cudaStream_t stream);
int64_t kv4_split_partial_bytes(int D);
cudaError_t launch_kv4_attn_prompt(const Kv4AttnParams& p, int sms, bool bf16, bool pdl, cudaStream_t stream);
int64_t kv4_prompt_partial_bytes(int D);

template <typename... KArgs, typename... Args>
cudaError_t kv4_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, bool pdl, cudaStream_t stream,
                       Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

cudaError_t ensure_smem_attr(const void* func, size_t bytes);  // fqkv_api.cu

// Host-side error reporting and device query of the C boundary (fqkv_api.cu).
int api_fail(int code, const char* msg);
int api_cuda_fail(cudaError_t e, const char* what);
int api_sm100(int* sms);  // SM count of the current device, or FQKV_ERR_DEVICE

}  // namespace fqkv
