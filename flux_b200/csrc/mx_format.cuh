// Layout of microscaled 4-bit matrices in memory (the OCP MX format MXFP4), shared by quantisation and products.
#pragma once
#include <cuda_runtime.h>

namespace fluxb {

constexpr int kMxBlock = 32;           // values that share a scale
constexpr int kMxGroupK = 128;         // values of K whose scales fill a cell
constexpr int kMxSfBytes = 512;        // scales of 128 rows x 128 values of K

// The scales of a matrix [rows, k] are blocks of 512 bytes, [ceil(rows / 128)][ceil(k / 128)], each 128 rows
// x 4 scales: row r at (r % 32) * 16 + r / 32 % 4 * 4. Scales past k / 32 in the last cell are zero; rows past the end hold
// anything.
__host__ __device__ __forceinline__ long long mx_sf_offset(long long row, int kg, int groups) {
  return ((row >> 7) * groups + kg) * kMxSfBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

}  // namespace fluxb
