// sd_paged.h -- internal interface of the paged K/V cache (sd_paged.cu) and its attention (sd_pattn.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "specdec_b200.h"

namespace sd {
int check_pages(const sd_pages* p, const char* what);
int check_kv_pool(const sd_kv_pool* p, const char* what);
// The entry points' work on checked arguments of device dev (the current one), with the error word to record in.
int launch_pages_plan(const sd_pages* p, const int32_t* kv_len, const int32_t* q_len, int q_stride, int pos0, int n_tokens,
                      int32_t* q_start, int32_t* slots, int32_t* positions, int32_t* missing, int* err, cudaStream_t st);
int launch_paged_attention(const sd_attn_args* a, int dev, int* err, cudaStream_t st);
// The current device, checked against the one that holds p.
int paged_device(const void* p, const char* what, int* dev);
}  // namespace sd
