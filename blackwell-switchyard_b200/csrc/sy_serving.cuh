// sy_serving.cuh -- launchers of the serving kernels (append, attention over
// pages, sampling), called by the entry points in sy_serving_abi.cu after
// their arguments were checked.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/switchyard_b200.h"

namespace sy {

struct ServingDev {
  int device = 0;
  int sms = 0;
};

cudaError_t launch_append(const sy_append_kv_args& a, cudaStream_t st);

int64_t attend_workspace(const sy_attend_args& a, const ServingDev& dev);
cudaError_t launch_attend(const sy_attend_args& a, const ServingDev& dev, cudaStream_t st);

cudaError_t launch_sample(const sy_sample_args& a, cudaStream_t st);

}  // namespace sy
