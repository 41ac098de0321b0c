// The kernels of paged_attention_many.hpp for bf16 queries (a translation unit of their own: they take longest to build).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "paged_attention_many.hpp"

namespace arctic {
void many_launch_bf16(const ManyParams &p, const ManyShape &f, int kv, hipStream_t s) { many_launch<BF16>(p, f, kv, s); }
}  // namespace arctic
