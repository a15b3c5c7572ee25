// The entry points of libcerebro_hip.so that csrc/torch/nodes.cpp calls: included by
// their definitions (dense.hip, distill.hip, toplogits.hip) and by the caller, so a
// changed argument on one side does not compile.  Two names each: bf16 and, with
// _f32, fp32 elements behind the void pointers.  All return a hipError_t, the _ws
// functions a workspace size, -1 for sizes out of range.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

#define CER_DENSE_FWD(NAME)                                                                        \
  int NAME(const void* x, int64_t ldx, const void* w, int64_t ws, const void* b, int64_t bs,       \
           const void* r, int64_t ldr, void* y, void* d, int M, int N, int K, int G, int act,      \
           float* part, int64_t part_floats, hipStream_t st)
#define CER_DENSE_BWD(NAME)                                                                        \
  int NAME(const void* dy, const void* d, void* dz, const void* x, int64_t ldx, const void* w,     \
           int64_t ws, void* dx, float* gw, int64_t gs, float* gb, int64_t gbs, int M, int N,      \
           int K, int G, int act, float* part, int64_t part_floats, hipStream_t st)
#define CER_DISTILL_FWD(NAME)                                                                      \
  int NAME(const void* z, int64_t ldz, const int* labels, const void* val, int val_f32,            \
           int64_t val_gs, int64_t val_bs, const int* idx, int64_t idx_gs, int64_t idx_bs,         \
           const float* alpha, float alpha0, const float* tau, float tau0, float* stats, void* dz, \
           float* loss, float* acc, int B, int G, int N, int K, float* ws, int64_t ws_floats,      \
           hipStream_t st)
#define CER_DISTILL_BWD(NAME)                                                                      \
  int NAME(const void* z, int64_t ldz, const int* labels, const void* val, int val_f32,            \
           int64_t val_gs, int64_t val_bs, const int* idx, int64_t idx_gs, int64_t idx_bs,         \
           const float* alpha, float alpha0, const float* tau, float tau0, const float* dloss,     \
           float* stats, void* dz, int B, int G, int N, int K, hipStream_t st)
#define CER_TOP_LOGITS(NAME)                                                                       \
  int NAME(const void* z, int64_t ldz, void* val, int* idx, int B, int G, int N, int K,            \
           int64_t* ws, int64_t ws_n, hipStream_t st)

extern "C" {
CER_DENSE_FWD(cer_dense_fwd);
CER_DENSE_FWD(cer_dense_fwd_f32);
CER_DENSE_BWD(cer_dense_bwd);
CER_DENSE_BWD(cer_dense_bwd_f32);
int64_t cer_dense_ws(int kind, int M, int N, int K, int G, int is_bf16, int act);
CER_DISTILL_FWD(cer_distill_fwd);
CER_DISTILL_FWD(cer_distill_fwd_f32);
CER_DISTILL_BWD(cer_distill_bwd);
CER_DISTILL_BWD(cer_distill_bwd_f32);
int64_t cer_distill_ws(int B, int G, int N, int is_bf16);
CER_TOP_LOGITS(cer_top_logits);
CER_TOP_LOGITS(cer_top_logits_f32);
int64_t cer_top_ws(int B, int G, int N, int K, int is_bf16);
}
