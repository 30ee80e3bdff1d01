// The attention kernels over the paged KV cache, by rows x heads of one KV head of a request
// (host side; paged_attn.cu chooses).
#pragma once

#include "pages.hpp"

#include <cuda.h>

namespace navi::attn {

struct AttendArgs;

// Which kernel: by rows x heads of one KV head, the most a request of the step may have (max_new; 48 single f16
// rows take 86 us with max_new 1, 94 with 8 and 117 with 16 or more).
//   up to 16: few. K and V are read once and the products are short.
//   17 to 32: few while the step has fewer items (requests x KV heads) than the GPU has multiprocessors,
//     else many. Lengths are on the device, so the rule does not see them. Trees of 9 to 16 rows, two heads each, 8 KV
//     heads, few and many: 4 over 200 to 2048 tokens f16 18.3 and 22.7 us, f32 20.5 and 26.7; 16 such f16 28.8 and
//     27.8, f32 35.2 and 39.1; 20 over 255 to 8191 tokens f16 71 and 55, f32 89 and 74; 48 such f16 134 and 118, f32
//     175 and 155. Below the bound long ones lose: 18 over 255 to 8191 tokens f16 63 and 52, f32 81 and 68.
//   above: many. 48 trees of up to 33 rows, KV 255 to 8191, f16: 98 to 108 us; the simple kernel before it
//     (mma.sync tiles of 64 rows, a block each) 394.
constexpr int FEW_ROWS = 16, FEW_ROWS_SHORT = 32;

void attend_few(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, int dtype, int cache, int rows, int sms, cudaStream_t stream);
// q: rows x heads in boxes of 128 rows of one KV head, where a.q_boxes is set
void attend_many(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, const CUtensorMap & q, int dtype, int cache, int64_t rows, int sms, cudaStream_t stream);

} // namespace navi::attn
