// Internal launch interface of what quantises rows to 8-bit integers (int8_rows.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sdxl_hip {

struct I8RowsParams {
    const void *x, *gamma, *beta;  // gamma null: the rows themselves, else their LayerNorm
    int8_t* q;
    float* q_scale;
    int64_t rows, cols, ld_x, ld_q;  // ld_x: elements, ld_q: bytes
    int64_t q_cols;                  // codes are written up to here, zeros past the last column
    float eps;
};

hipError_t launch_i8_rows(const I8RowsParams& p, bool bf16, hipStream_t stream);

}  // namespace sdxl_hip
