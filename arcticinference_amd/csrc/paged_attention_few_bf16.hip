// The kernels of paged_attention_few.hpp for bf16 queries (a translation unit of their own: they take longest to build).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "paged_attention_few.hpp"

namespace arctic {
void few_launch_bf16(const FewParams &p, const FewShape &f, int kv, hipStream_t s) { few_launch<BF16>(p, f, kv, s); }
}  // namespace arctic
