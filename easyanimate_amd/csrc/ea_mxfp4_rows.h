// Row arithmetic of the microscaled 4-bit kernels that host code can evaluate too (plain C++: no HIP header).
#pragma once
#include <cstdint>

#ifdef __HIPCC__
#define EA_ROWS_HD __host__ __device__ __forceinline__
#else
#define EA_ROWS_HD inline
#endif

// gemm256_mxfp4_w4_kernel: byte offset, inside a K tile's scales (8 bytes a row), of a lane's 16-byte request for rows `row` and row + 1
// of an operand of `rows` (>= 2) rows.  Rows past the end read the last two again.  A pair that begins WITH the last row takes the 8 bytes
// behind it along: the next K tile's first row, or, in the last K tile, MXW4_SCALE_PAD bytes that the buffer must have.
constexpr int MXW4_SCALE_PAD = 8;
EA_ROWS_HD int mxw4_scale_offset(const int64_t row, const int64_t rows) { return (int)((row < rows ? row : rows - 2) * 8); }
