// Attention of a step's rows over the paged KV cache (navi_pages_attend).
//
//   out[j] = sum_k p[j][k] v[k] / l[j],  p[j][k] = exp(scale q[j] k[k] - m[j]),  l[j] = sum_k p[j][k]
//
// over the request's cached tokens k < ctx and those of the step's rows that row j sees: its
// ancestors and itself in a drafted tree (a bit mask), rows up to j in a chain. m is a running
// maximum, so one pass over the keys is enough; m, l and the sums are f32.
#include "paged_attn.hpp"
#include "paged_attn.cuh"

#include <string>

namespace navi {

void Pages::attend(const navi_step & s, int layer, const navi_attend_args & q, cudaStream_t stream) const {
    check_step(s, "pages attend");
    check_layer(layer, "pages attend");
    if (q.n_head < 1 || q.n_head > 4096 || q.n_head % d_.n_kv_head) fail("pages attend: n_head must be a positive multiple of n_kv_head", NAVI_E_ARG);
    if (!(q.dtype == d_.dtype || (q.dtype == NAVI_F32 && d_.dtype == NAVI_F16))) fail("pages attend: rows are of the cache's type, or NAVI_F32 for an f16 cache", NAVI_E_ARG);
    if (!(q.scale > 0.f) || q.scale > 1e30f) fail("pages attend: scale must be positive and finite", NAVI_E_ARG);
    if (s.n_req == 0 || s.max_rows == 0) return;
    const int D = d_.head_dim;
    const int64_t elt = q.dtype == NAVI_F32 ? 4 : 2, dense = static_cast<int64_t>(q.n_head) * D, in = q.q_stride ? q.q_stride : dense,
                  out = q.out_stride ? q.out_stride : dense;
    if (!q.q || !q.out) fail("pages attend: NULL rows", NAVI_E_ARG);
    if (in < dense || out < dense) fail("pages attend: a row stride is shorter than the row", NAVI_E_ARG);
    const auto off16 = [](const void * p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
    if (off16(q.q) || off16(q.out) || in * elt % 16 || out * elt % 16) fail("pages attend: rows must be 16-byte aligned", NAVI_E_ARG);
    NAVI_CUDA(cudaSetDevice(dev_->info().ordinal));
    const int sms = dev_->info().multiprocessors;
    const PagesScratch sc(dev_->scratch(stream, PagesScratch::bytes(sms)), sms);
    attn::AttendArgs a{};
    a.q = q.q;
    a.out = q.out;
    a.lse = q.lse;
    a.k = static_cast<const uint8_t *>(k_[static_cast<size_t>(layer)]);
    a.v = static_cast<const uint8_t *>(v_[static_cast<size_t>(layer)]);
    a.table = d_.table;
    a.req = s.req;
    a.ctx_len = s.ctx_len;
    a.cu_rows = s.cu_rows;
    a.status = s.status;
    a.mask = s.parent ? s.mask : nullptr;
    a.pieces = sc.pieces;
    a.arrived = sc.arrived;
    a.err = sc.err;
    a.q_stride = in;
    a.out_stride = out;
    a.scale = q.scale * 1.4426950408889634f;
    a.n_req = s.n_req;
    a.max_rows = s.max_rows;
    a.mask_words = s.mask_words;
    a.n_head = q.n_head;
    a.n_kv = d_.n_kv_head;
    a.group = q.n_head / d_.n_kv_head;
    a.head_dim = D;
    a.shift = shift_;
    a.n_pages = d_.n_pages;
    a.max_blocks = d_.max_blocks;
    a.max_requests = d_.max_requests;
    const int64_t most = std::min(s.max_new, s.max_rows);
    if (a.group > 1) a.group_mul = static_cast<uint32_t>(((1ull << 32) + static_cast<uint64_t>(a.group) - 1) / static_cast<uint64_t>(a.group));
    // a request that is not served may have all of max_rows: its rows are counted too, and written
    const int64_t all = static_cast<int64_t>(s.max_rows) + 512;
    if (all * a.group > INT32_MAX || ((a.group & (a.group - 1)) != 0 && all * a.group * a.group >= 1ll << 32))
        fail("pages attend: too many rows for this many heads to a KV head", NAVI_E_SHAPE);
    // the list of key tiles that the blocks divide: of requests that are served, and a tile for each 8 rows x heads that are not
    const int64_t rows = most * a.group <= attn::FEW_ROWS_SHORT ? 16 : 128, items = (most * a.group + rows - 1) / rows * d_.n_kv_head * s.n_req, tiles = (static_cast<int64_t>(d_.max_blocks) * d_.page_size + attn::KT - 1) / attn::KT + 2;
    if (items * tiles + (all * a.group / 8 + s.n_req) * 2 * d_.n_kv_head >= 1ll << 31) fail("pages attend: requests x heads x tokens pass 31 bits of key tiles", NAVI_E_SHAPE);
    const int64_t m = most * a.group;
    const size_t at = static_cast<size_t>(2 * layer);
    if (m <= attn::FEW_ROWS || (m <= attn::FEW_ROWS_SHORT && s.n_req * d_.n_kv_head < sms)) return attn::attend_few(a, page_maps_[at], page_maps_[at + 1], q.dtype, d_.dtype, static_cast<int>(m), sms, stream);
    // q by TMA where an item has two tiles of it, by a warp's loads where it has one: 48 trees of up to 33 rows
    // 101 us by loads and 105 by TMA. 8 chunks of 1000 rows went from 246 to 210 us in the step that brought
    // TMA and, with it, the waits before a pair of products.
    CUtensorMap qm{};
    if (q.dtype != NAVI_F32 && m > 128 && a.group <= 128 && (a.group & (a.group - 1)) == 0) {
        a.q_boxes = 1;
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(q.n_head), static_cast<cuuint64_t>(s.max_rows)};
        const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(in) * 2};
        const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(128 / a.group)};
        qm = swizzled_map(q.q, q.dtype, 3, dims, strides, box);
    }
    attn::attend_many(a, maps_[at], maps_[at + 1], qm, q.dtype, d_.dtype, m, sms, stream);
}

} // namespace navi
