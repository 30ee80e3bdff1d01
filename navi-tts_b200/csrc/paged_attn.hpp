// The attention kernels over the paged KV cache, by rows x heads of one KV head of a request
// (host side; paged_attn.cu chooses).
#pragma once

#include "pages.hpp"

#include <cuda.h>

namespace navi::attn {

struct AttendArgs;

void attend_few(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, int dtype, int cache, int rows, int sms, cudaStream_t stream);

} // namespace navi::attn
