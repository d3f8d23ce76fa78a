// Host-side construction of TMA tensor maps without linking libcuda: the driver's encoder is looked up
// through the runtime (cudaGetDriverEntryPoint).  Encoding is pure host arithmetic (no device work, no
// allocation), so it is safe inside stream capture.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace b2 {

// 2-D row-major tensor [rows, cols] of `elem_bytes`-byte elements with box [box_rows, box_cols].
// The base address and the row pitch (cols * elem_bytes) must be multiples of 16 bytes.
bool make_tensor_map_2d(CUtensorMap* out, CUtensorMapDataType dt, int elem_bytes, const void* ptr, uint64_t rows,
                        uint64_t cols, uint32_t box_rows, uint32_t box_cols, CUtensorMapSwizzle swz);

// bf16 tensor of four dimensions, innermost first, with strides in elements (multiples of 8) for the outer three, read in boxes of
// box[0] x box[1] elements of the inner two with the 128-byte swizzle.
bool make_tensor_map_4d(CUtensorMap* out, const void* ptr, const uint64_t (&dims)[4], const uint64_t (&strides)[3],
                        const uint32_t (&box)[2]);

}  // namespace b2
