// Tensor maps for bulk copies (host side).
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace b200 {

// Matrices of one launch: how many and how far apart (elements); count == 0 asks for a 2-D map.
struct BatchDim {
    int64_t count = 0;
    int64_t stride = 0;
    uint32_t box = 1;  // matrices per copy
};

// Tensor map over a column-major matrix: dim0 (contiguous) has `inner` elements, dim1 has `outer`
// elements `ld` elements apart; batched problems add dim2 = matrix of the batch (box extent 1 unless asked for).
int encode_map_2d(CUtensorMap* tm, CUtensorMapDataType dt, int elem_bytes, const void* base, int64_t inner,
                  int64_t outer, int64_t ld, uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle sw,
                  const char* what, BatchDim batch = BatchDim());

inline CUtensorMapDataType map_type(int type) {  // B200_F16 / B200_F32 / B200_BF16
    return type == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : (type == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
}

}  // namespace b200
