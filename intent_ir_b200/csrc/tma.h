// Tensor maps for the bulk tensor copies (built in gemm.cu).
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace ib200 {
int make_byte_map(CUtensorMap* map, const void* base, int64_t rows, int64_t row_bytes, int box_rows);
}  // namespace ib200
