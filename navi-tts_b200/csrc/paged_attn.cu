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

namespace {

using namespace navi::attn;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// c (16x8 f32) += a (16x16, row) b (16x8, col), operands of the cache's type C
template <class C> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<C, __half>)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
constexpr int ROWS = 64, KEYS = 64, WARPS = 4, THREADS = 128;

// A block takes 64 of a request's rows x heads of one KV head (4 warps of 16, the heads of a row
// next to one another) through all keys, 64 at a time, double-buffered by cp.async. T is the type
// of q and out, C the cache's. f32 rows enter the products as two f16 terms, q = hi + lo and
// p = hi + lo, against the exact cache values: about 22 bits. 16-bit rows are exact, and p is
// rounded once to the type that the result has. Shared-memory rows are swizzled by 16-byte
// pieces so that ldmatrix reads eight different banks.
template <class T, class C, int D>
__global__ void __launch_bounds__(THREADS) k_attend(const __grid_constant__ AttendArgs a, const uint8_t * kpool, const uint8_t * vpool) {
    constexpr bool SPLIT = std::is_same_v<T, float>;
    constexpr int CH = D / 8;                         // 16-byte pieces of a row
    constexpr uint32_t ROW = D * 2, TILE = KEYS * ROW;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t * qhi = smem, * qlo = qhi + ROWS * ROW, * kv = qhi + (SPLIT ? 2 : 1) * ROWS * ROW;
    const Request rq = request(a, blockIdx.z);
    const int g = blockIdx.y, m0 = blockIdx.x * ROWS, M = rq.n * a.group;   // M: rows x heads of the KV head
    if (m0 >= M) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    const auto swz = [](int row, int piece) { return static_cast<uint32_t>(row) * ROW + ((piece ^ (row & 7)) << 4); };
    const int n_keys = a.mask || rq.keys == 0 ? rq.keys : rq.ctx + min((m0 + ROWS - 1) / a.group + 1, rq.n);
    const int tiles = (n_keys + KEYS - 1) / KEYS;

    const auto load = [&](int kt) {
        uint8_t * kb = kv + (kt & 1) * 2 * TILE, * vb = kb + TILE;
        for (int x = tid; x < KEYS * CH; x += THREADS) {
            const int r = x / CH, c = x % CH, key = kt * KEYS + r;
            const uint32_t o = swz(r, c);
            if (key < n_keys) {
                const int page = min(max(rq.table[key >> a.shift], 0), a.n_pages - 1);
                const size_t at = ((((static_cast<size_t>(page) * a.n_kv + g) << a.shift) + (key & ((1 << a.shift) - 1))) * CH + c) * 16;
                cp_async16(kb + o, kpool + at);
                cp_async16(vb + o, vpool + at);
            } else {   // past the request's tokens: zeros, whatever the page holds there
                *reinterpret_cast<uint4 *>(kb + o) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4 *>(vb + o) = make_uint4(0, 0, 0, 0);
            }
        }
        cp_async_commit();
    };
    if (tiles > 0) load(0);
    for (int x = tid; x < ROWS * CH; x += THREADS) {
        const int r = x / CH, c = x % CH, m = m0 + r;
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if (m < M) {
            const T * src = static_cast<const T *>(a.q) + (rq.row0 + m / a.group) * a.q_stride + (g * a.group + m % a.group) * D + c * 8;
            if constexpr (SPLIT) {
                float f[8];
                *reinterpret_cast<float4 *>(f) = *reinterpret_cast<const float4 *>(src);
                *reinterpret_cast<float4 *>(f + 4) = *reinterpret_cast<const float4 *>(src + 4);
                uint32_t * h = &hi.x, * l = &lo.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    h[k] = pack<C>(f[2 * k], f[2 * k + 1]);
                    const float2 b = unpack<C>(h[k]);
                    l[k] = pack<C>(f[2 * k] - b.x, f[2 * k + 1] - b.y);
                }
            } else {
                hi = *reinterpret_cast<const uint4 *>(src);
            }
        }
        *reinterpret_cast<uint4 *>(qhi + swz(r, c)) = hi;
        if constexpr (SPLIT) *reinterpret_cast<uint4 *>(qlo + swz(r, c)) = lo;
    }

    const int w0 = warp * 16;
    int row[2];                                       // this thread's rows gq and gq + 8 of the warp, among the request's
#pragma unroll
    for (int x = 0; x < 2; ++x) row[x] = min((m0 + w0 + gq + 8 * x) / a.group, rq.n - 1);
    float o[D / 8][4], mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int x = 0; x < D / 8; ++x) o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.f;
    const uint32_t sqh = smem_addr(qhi), sql = smem_addr(qlo);
    for (int kt = 0; kt < tiles; ++kt) {
        if (kt + 1 < tiles) {
            load(kt + 1);
            cp_async_wait<1>();
        } else {
            cp_async_wait<0>();
        }
        __syncthreads();
        const uint32_t sk = smem_addr(kv + (kt & 1) * 2 * TILE), sv = sk + TILE;
        float s[KEYS / 8][4];
#pragma unroll
        for (int x = 0; x < KEYS / 8; ++x) s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t ah[4], al[4];
            const int ar = w0 + (lane & 15), ac = ks * 2 + (lane >> 4);
            ldsm4(ah, sqh + swz(ar, ac));
            if constexpr (SPLIT) ldsm4(al, sql + swz(ar, ac));
#pragma unroll
            for (int np = 0; np < KEYS / 16; ++np) {
                uint32_t b[4];
                ldsm4(b, sk + swz(np * 16 + (lane & 7) + (lane >> 4) * 8, ks * 2 + ((lane >> 3) & 1)));
                mma<C>(s[2 * np], ah, b[0], b[1]);
                mma<C>(s[2 * np + 1], ah, b[2], b[3]);
                if constexpr (SPLIT) {
                    mma<C>(s[2 * np], al, b[0], b[1]);
                    mma<C>(s[2 * np + 1], al, b[2], b[3]);
                }
            }
        }
        float m[2] = {mx[0], mx[1]};
        const bool plain = (kt + 1) * KEYS <= rq.ctx;   // every key of the tile is seen by every row
#pragma unroll
        for (int x = 0; x < KEYS / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = s[x][e] * a.scale;
                if (!plain) {
                    const int key = kt * KEYS + x * 8 + 2 * tq + (e & 1), at = key - rq.ctx, j = row[e >> 1];
                    bool seen = key < n_keys;
                    if (at >= 0 && seen)
                        seen = a.mask ? at < 64 * a.mask_words && (a.mask[static_cast<size_t>(rq.row0 + j) * a.mask_words + (at >> 6)] >> (at & 63) & 1) : at <= j;
                    v = seen ? v : -INFINITY;
                }
                s[x][e] = v;
                m[e >> 1] = fmaxf(m[e >> 1], v);
            }
        float al[2], mu[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            m[x] = fmaxf(m[x], __shfl_xor_sync(0xffffffffu, m[x], 1));
            m[x] = fmaxf(m[x], __shfl_xor_sync(0xffffffffu, m[x], 2));
            mu[x] = m[x] == -INFINITY ? 0.f : m[x];   // a row that has seen nothing yet
            al[x] = exp2_fast(mx[x] - mu[x]);
            mx[x] = m[x];
            l[x] *= al[x];
        }
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
            o[x][0] *= al[0]; o[x][1] *= al[0];
            o[x][2] *= al[1]; o[x][3] *= al[1];
        }
        uint32_t ph[KEYS / 16][4], pl[KEYS / 16][4];
#pragma unroll
        for (int x = 0; x < KEYS / 8; ++x) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float p0 = exp2_fast(s[x][2 * e] - mu[e]), p1 = exp2_fast(s[x][2 * e + 1] - mu[e]);
                l[e] += p0 + p1;
                const int at = (x & 1) * 2 + e;
                ph[x >> 1][at] = pack<C>(p0, p1);
                if constexpr (SPLIT) {
                    const float2 b = unpack<C>(ph[x >> 1][at]);
                    pl[x >> 1][at] = pack<C>(p0 - b.x, p1 - b.y);
                }
            }
        }
#pragma unroll
        for (int st = 0; st < KEYS / 16; ++st)
#pragma unroll
            for (int dp = 0; dp < D / 16; ++dp) {
                uint32_t b[4];
                ldsm4t(b, sv + swz(st * 16 + (lane & 15), dp * 2 + (lane >> 4)));
                mma<C>(o[2 * dp], ph[st], b[0], b[1]);
                mma<C>(o[2 * dp + 1], ph[st], b[2], b[3]);
                if constexpr (SPLIT) {
                    mma<C>(o[2 * dp], pl[st], b[0], b[1]);
                    mma<C>(o[2 * dp + 1], pl[st], b[2], b[3]);
                }
            }
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        const int m = m0 + w0 + gq + 8 * x;
        if (m >= M) continue;
        const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];
        const int j = m / a.group, h = g * a.group + m % a.group;
        T * dst = static_cast<T *>(a.out) + (rq.row0 + j) * a.out_stride + h * D;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
            const float u = o[d][2 * x] * inv, w = o[d][2 * x + 1] * inv;
            if constexpr (SPLIT) *reinterpret_cast<float2 *>(dst + d * 8 + 2 * tq) = make_float2(u, w);
            else *reinterpret_cast<uint32_t *>(dst + d * 8 + 2 * tq) = pack<C>(u, w);
        }
        if (a.lse && tq == 0)
            a.lse[static_cast<size_t>(rq.row0 + j) * a.n_head + h] = l[x] == 0.f ? -INFINITY : (mx[x] + log2f(l[x])) * 0.6931471805599453f;
    }
}

} // namespace

void Pages::attend(const navi_step & s, int layer, const navi_attend_args & q, cudaStream_t stream) const {
    check_step(s, "pages attend");
    if (layer < 0 || layer >= d_.n_layer) fail("pages attend: layer outside the cache", NAVI_E_ARG);
    if (q.n_head < 1 || q.n_head > 4096 || q.n_head % d_.n_kv_head) fail("pages attend: n_head must be a positive multiple of n_kv_head", NAVI_E_ARG);
    if (!(q.dtype == d_.dtype || (q.dtype == NAVI_F32 && d_.dtype == NAVI_F16))) fail("pages attend: rows are of the cache's type, or NAVI_F32 for an f16 cache", NAVI_E_ARG);
    if (!(q.scale > 0.f) || q.scale > 1e30f) fail("pages attend: scale must be positive and finite", NAVI_E_ARG);
    if (s.n_req == 0 || s.max_rows == 0 || s.max_new == 0) return;
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
    AttendArgs a{q.q, q.out, q.lse, d_.table, s.req, s.ctx_len, s.cu_rows, s.status, s.parent ? s.mask : nullptr, sc.pieces, sc.arrived, sc.err,
                 in, out, q.scale * 1.4426950408889634f, s.n_req, s.max_rows, s.mask_words, q.n_head, d_.n_kv_head, q.n_head / d_.n_kv_head, D, shift_,
                 d_.n_pages, d_.max_blocks, d_.max_requests};
    const CUtensorMap & km = maps_[static_cast<size_t>(2 * layer)], & vm = maps_[static_cast<size_t>(2 * layer + 1)];
    const int64_t m = static_cast<int64_t>(std::min(s.max_new, s.max_rows)) * a.group;
    if (m <= 32) return attend_few(a, km, vm, q.dtype, d_.dtype, static_cast<int>(m), sms, stream);
    const dim3 grid(static_cast<unsigned>((m + ROWS - 1) / ROWS), static_cast<unsigned>(d_.n_kv_head), static_cast<unsigned>(s.n_req));
    const auto go = [&](auto kernel, bool split) {
        const int smem = static_cast<int>(((split ? 2 : 1) * ROWS + 4 * KEYS) * D * 2);
        NAVI_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        kernel<<<grid, THREADS, static_cast<size_t>(smem), stream>>>(a, static_cast<const uint8_t *>(k_[static_cast<size_t>(layer)]), static_cast<const uint8_t *>(v_[static_cast<size_t>(layer)]));
    };
    if (q.dtype == NAVI_F32) D == 128 ? go(k_attend<float, __half, 128>, true) : go(k_attend<float, __half, 64>, true);
    else if (q.dtype == NAVI_F16) D == 128 ? go(k_attend<__half, __half, 128>, false) : go(k_attend<__half, __half, 64>, false);
    else D == 128 ? go(k_attend<__nv_bfloat16, __nv_bfloat16, 128>, false) : go(k_attend<__nv_bfloat16, __nv_bfloat16, 64>, false);
    NAVI_CUDA(cudaGetLastError());
}

} // namespace navi
