// Attention of prompt chunks on the fifth-generation tensor cores (kv4_prompt.cu), as l3m_kv4_attend_dev uses it.
#pragma once
#include <cuda_runtime.h>
#include "../../include/l3m_kernels.h"

namespace l3m {

bool prompt_fits(const l3m_kv4 *c, const l3m_kv4_attend *a);       // from the integer fields alone
cudaError_t prompt_attend(const l3m_kv4 *c, const l3m_kv4_attend *a, cudaStream_t s);

}  // namespace l3m
