/* FP8-128 products (k3_fp8.hip), for the other translation units. */
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace k3 {

/* Scratch of k3_moe_fp8_128_gemm_bf16 (cols % 128 == 0). */
size_t fp8_scratch_bytes(uint32_t tokens, uint32_t rows, uint32_t cols);

}  // namespace k3
