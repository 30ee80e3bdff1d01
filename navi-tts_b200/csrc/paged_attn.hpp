// The attention kernels over the paged KV cache, by rows x heads of one KV head of a request
// (host side; paged_attn.cu chooses).
#pragma once

#include "pages.hpp"

#include <cuda.h>

namespace navi::attn {

struct AttendArgs;

// Which kernel: by rows x heads of one KV head, the most a request of the step has.
//   up to 16: few. K and V are read once and the products are short.
//   17 to 32: few while the step has fewer items (requests x KV heads) than the GPU has multiprocessors,
//     else many. Four trees of up to 16 rows, two heads each, KV 200 to 2048, f32: few 20.6 us,
//     many 25.7. 48 such requests, KV 255 to 8191: f16 103 and 95 us, f32 134 and 122.
//   above: many. 48 trees of up to 33 rows, KV 255 to 8191, f16: 97 to 104 us; the simple kernel before it
//     (mma.sync tiles of 64 rows, a block each) 394.
constexpr int FEW_ROWS = 16, FEW_ROWS_SHORT = 32;

void attend_few(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, int dtype, int cache, int rows, int sms, cudaStream_t stream);
// q: rows x heads in boxes of 128 rows of one KV head, where a.q_boxes is set
void attend_many(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, const CUtensorMap & q, int dtype, int cache, int64_t rows, int sms, cudaStream_t stream);

} // namespace navi::attn
