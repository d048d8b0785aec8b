// The expert layer's launches for one code type (moe_ops.cu holds the entry point, moe_product.cu a unit for each type).
#pragma once

#include "host_common.h"
#include "moe_kernels.cuh"

namespace b200 {

int launch_moe_int4(const MoeParams& params, bool n_major, int sm_count, cudaStream_t stream);
int launch_moe_int8(const MoeParams& params, bool n_major, int sm_count, cudaStream_t stream);

}  // namespace b200
