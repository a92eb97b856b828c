// Launchers of the AdamW step's kernels (adamw.hip; called by adamw_capi.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "mft/adamw.h"

namespace mft {

size_t adamw_workspace(int32_t n);
// Tensors without values or a gradient are left out.
hipError_t launch_adamw(const mft_adamw_desc& d, int32_t n, const mft_adamw_tensor* tensors, int64_t* step, float* norm,
                        void* workspace, hipStream_t st);

}  // namespace mft
