// The forms of the products with weights of four bits.
#pragma once

#include <cuda_runtime.h>

namespace ksa {

constexpr int kI4WMostRows = 32, kI4WMostParts = 8;

// Up to 32 rows with a pitch lda >= K.
int int4_linear_wide(const void* A, const void* codes, const void* meta, void* C, int M, int N, int K, int group, int pitch, long long lda, long long ldc,
                     cudaStream_t st);

}  // namespace ksa
