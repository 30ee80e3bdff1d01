// The attention kernels over the paged KV cache, by rows x heads of one KV head of a request
// (host side; paged_attn.cu chooses).
#pragma once

#include "pages.hpp"

#include <cuda.h>

namespace navi::attn {

struct AttendArgs;

// rows x heads of a KV head up to which the kernel for few rows is taken
constexpr int FEW_ROWS = 32;

void attend_few(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, int dtype, int cache, int rows, int sms, cudaStream_t stream);
// q: rows x heads in boxes of 128 rows of one KV head, where a.q_boxes is set
void attend_many(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, const CUtensorMap & q, int dtype, int cache, int64_t rows, int sms, cudaStream_t stream);

} // namespace navi::attn
