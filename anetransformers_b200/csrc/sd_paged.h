// sd_paged.h -- internal interface of the paged K/V cache (sd_paged.cu) and its attention (sd_pattn.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "specdec_b200.h"

namespace sd {
int check_pages(const sd_pages* p, const char* what);
int check_kv_pool(const sd_kv_pool* p, const char* what);
// The current device, checked against the one that holds p.
int paged_device(const void* p, const char* what, int* dev);
}  // namespace sd
