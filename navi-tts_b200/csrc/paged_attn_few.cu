// Attention over the paged KV cache for few rows of a request (paged_attn.cu): single tokens and
// small drafted trees, on mma.sync tiles.
#include "paged_attn.hpp"
#include "paged_attn.cuh"

namespace navi::attn {

namespace {

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
// A tile of 16 rows (8, where a block has no more) belongs to KQ warps, which divide a key tile of
// 128 between them, each with a running maximum and sums of its own until the segment ends; a
// ninth warp keeps a ring of tiles full by TMA. K and V are read once however many rows there are,
// so up to 32 rows the bound is HBM.
//
// f32 rows enter the products as two f16 terms, q = hi + lo and p = hi + lo, against the exact cache
// values: about 22 bits of q, and of weights down to 2^-17 of the largest (smaller ones to 2^-39 of
// it). With 8 rows the high terms are rows 0..7 of the 16 that a product has and the low ones rows
// 8..15, so that they cost nothing. The tensor cores' sums truncate: the low
// terms and each step's contribution are summed apart and added in f32. 16-bit rows are exact, and
// their p is two terms too in tiles of 8. With more rows it is rounded once to the type that the
// result has, 8 bits of bf16, 11 of f16 down to 2^-28 of the largest weight, about the result's own rounding:
// a second term there is products of its own (5 rows of two heads over 200,003 bf16 tokens 132 -> 135.5 us, 48 f16
// trees of up to 8 such rows 99 -> 107), in tiles of 8 none (48 single f16 rows 89.5 -> 87.7 us, without the spills).
//
// Measured on one B200: one request of 200,003 tokens, 5 rows, bf16: 129 to 135 us, 6.1 to 6.3 TB/s (a copy
// reaches 6.54). 48 single f16 rows over pages of 16: 84 to 88 us; with a box for each 64 dims of a page 92.7 where
// one box took 84.3. The tile's rows: 48 single rows, KV 255 to 8191, f32: 88 us in tiles of 8, 150 in tiles of 32; 30
// such, KV 255 to 2000, f16: 31 and 39. Four single rows at KV 512 take 11 us, of which the data are 1.3; what
// is left is launch and one trip to L2 after another: the work list, q and pages, the tile, the join.
template <class C> constexpr float LIFT = std::is_same_v<C, __half> ? 14.f : 0.f;   // f16 holds 65504

template <int D> struct FewSmem {
    static constexpr int STAGE = KT * D * 4;                    // K and V of a tile
    static constexpr int STAGES = D == 128 ? 3 : 6;
    static constexpr int JOIN = 8 * 16 * 64 * 4;                // eight warps' sums over 64 dims
    static constexpr int BYTES = 1024 + STAGES * STAGE + JOIN;  // 1024: to align the ring to the swizzle's 1024 bytes
};

// y and what the tokens that were cleared add to row m of a segment, if it sees them. Out of line: it seldom runs.
template <class T, class C, int D>
__device__ __noinline__ float4 with_bad(const AttendArgs & a, const Segment & s, const uint32_t * bad, int m, float ref, int dim, float4 y) {
    const int bad0 = s.ctx / KT * KT, j = by_group(a, s.m0 + m);
#pragma unroll 1
    for (int w = 0; w < 16; ++w)
#pragma unroll 1
        for (uint32_t left = bad[w]; left; left &= left - 1) {
            const int key = bad0 + 32 * w + __ffs(left) - 1;
            if (!(seen_bits(a, s, j, key - s.ctx, s.n_keys - key) & 1)) continue;
            const float w = token_weight<T, C, D>(a, s, m, key, ref);
            const C * v = token_at<C, D>(a, s, a.v, key) + dim;
            y.x += w * static_cast<float>(v[0]);
            y.y += w * static_cast<float>(v[1]);
            y.z += w * static_cast<float>(v[2]);
            y.w += w * static_cast<float>(v[3]);
        }
    return y;
}

template <class T, class C, int D, int ROWS>   // ROWS: 8, 16 or 32 rows of an item
__global__ void __launch_bounds__(288, 1) k_attend_few(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                                                       const __grid_constant__ CUtensorMap vmap) {
    constexpr bool SPLIT = std::is_same_v<T, float>, EIGHT = ROWS == 8;
    constexpr int RT = EIGHT ? 1 : ROWS / 16, KQ = 8 / RT, WK = KT / KQ;    // row tiles; warps and keys of a tile a warp takes
    constexpr int XR = EIGHT ? 1 : 2, MR = 8 * XR;                          // rows a thread and a warp have
    constexpr int KS = WK / 16;                                             // 16-key products a warp does at a time
    constexpr bool TERMS = SPLIT && !EIGHT;                                 // the low terms are products of their own
    using L = FewSmem<D>;
    extern __shared__ uint8_t raw[];
    uint8_t * ring = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    float4 * sums = reinterpret_cast<float4 *>(ring + L::STAGES * L::STAGE);
    // q lies where the warps' sums come when it is no longer read: [16 RT][D], the low terms of f32 rows in rows
    // 8..15 or, with more than 8 rows, in as many rows again
    uint8_t * qs = reinterpret_cast<uint8_t *>(sums);
    static_assert(2 * 32 * D * 2 <= L::JOIN);
    __shared__ __align__(8) uint64_t full[L::STAGES], empty[L::STAGES];
    __shared__ __align__(8) SegmentRing segs;
    __shared__ float stat[8][2][MR];
    __shared__ float q_scale[SPLIT ? ROWS : 1];   // f32 rows: each row's scale of the scores
    __shared__ uint32_t bad[16];   // tokens from the item's first masked tile on whose V is not finite
    __shared__ int red[9];
    __shared__ Share share;
    __shared__ volatile int abort_flag;
    __shared__ int is_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 8);
        }
        segs.init(8);
        fence_mbar_init();
    }
    __syncthreads();
    griddep_wait();
    griddep_launch_dependents();
    const bool one = a.n_req <= 32;
    if (!one) share_of_block<ROWS, 0, 288>(a, share, red);
    const Wait wait{&abort_flag, a.err};

    if (warp == 8) {
        Request first{};
        Share sh;
        if (one) {
            sh = share_of_warp<ROWS, 0>(a, first);
            if (lane == 0) share.d = sh.d;           // the other warps read it after a segment
        } else {
            sh = share;
            if (sh.u < sh.end) first = request(a, sh.i);
        }
        Walk<ROWS, 0> walk(a, sh, first);
        int n = 0;
        bool ok = true;
        const int kv = lane >> 4, nth = lane & 15;   // half a warp each for K and V; a box is a page: [D / 64][page][64]
#pragma unroll 1
        for (int k = 0; ok; ++k) {
            Segment s;
            const bool more = walk.next(s);
            int page = more && s.n_keys > 0 ? page_at(a, s, s.t0, nth) : -1;
            if (k >= SegmentRing::N) ok = __shfl_sync(0xffffffffu, lane == 0 ? wait(&segs.empty[k % SegmentRing::N], (k / SegmentRing::N - 1) & 1) : 0, 0);
            if (!ok) break;
            if (lane == 0) {
                segs.s[k % SegmentRing::N] = s;
                mbar_arrive(&segs.full[k % SegmentRing::N]);
            }
            if (!more) break;
            if (s.n_keys <= 0) continue;
#pragma unroll 1
            for (int t = s.t0; t < s.t0 + s.nt; ++t, ++n) {
                const int st = n % L::STAGES, next = t + 1 < s.t0 + s.nt ? page_at(a, s, t + 1, nth) : -1;
                if (n >= L::STAGES) ok = __shfl_sync(0xffffffffu, lane == 0 ? wait(&empty[st], (n / L::STAGES - 1) & 1) : 0, 0);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(2 * (tile_pages(a, s, t) << a.shift) * D * 2));
                __syncwarp();
                if (page >= 0)
                    tma_box_3d(ring + st * L::STAGE + kv * (L::STAGE / 2) + (nth << a.shift) * (D * 2), kv ? &vmap : &kmap, 0, (page * a.n_kv + s.g) << a.shift, 0,
                               &full[st]);
                page = next;
            }
        }
        // after an abort, whoever raised it, the copies still under way land before the block's shared memory goes
        named_sync(2, 288);
        if (abort_flag)
            for (int k = max(n - L::STAGES, 0); k < n; ++k) mbar_drain(&full[k % L::STAGES], (k / L::STAGES) & 1);
        return;
    }

    const int rt = warp / KQ, kq = warp % KQ, k0 = kq * WK;
    // A tile lies page after page, [D / 64][page][64]: rows of 128 bytes, their eight 16-byte pieces swizzled by the row.
    // The lanes of an ldmatrix read eight rows in a row from a multiple of 8 on, so the swizzle is the lane's own,
    // and piece 2 j + b of a row lies at one of four offsets. 16 keys never leave a page.
    uint32_t off_k[4], off_v[4];                      // b = (lane >> 3) & 1 for K, lane >> 4 for V and q
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        off_k[j] = ((2 * j + ((lane >> 3) & 1)) ^ (lane & 7)) << 4;
        off_v[j] = ((2 * j + (lane >> 4)) ^ (lane & 7)) << 4;
    }
    const uint32_t half = 128u << a.shift;            // from a page's first 64 dims to the next
    const auto place = [&](int key) { return static_cast<uint32_t>((key >> a.shift << a.shift) * (D * 2) + (key & ((1 << a.shift) - 1)) * 128); };
    uint32_t k_at[KS], v_at[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        k_at[k] = smem_addr(ring) + place(k0 + 16 * k) + ((lane & 7) + (lane >> 4) * 8) * 128;
        v_at[k] = smem_addr(ring) + L::STAGE / 2 + place(k0 + 16 * k) + (lane & 15) * 128;
    }
    const uint32_t q_at = smem_addr(qs) + (rt * 16 + (lane & 15)) * (D * 2);
    int n = 0;
#pragma unroll 1
    for (int sn = 0;; ++sn) {
        const bool got = wait(&segs.full[sn % SegmentRing::N], (sn / SegmentRing::N) & 1);
        if (tid < 16) bad[tid] = 0;
        // after an abort all warps leave together
        if (named_sync_or(1, 256, !got)) break;
        const Segment & s = segs.s[sn % SegmentRing::N];
        if (s.nt < 0) break;
        // q into shared memory, a thread 8 values, whole rows a warp
#pragma unroll 1
        for (int x = tid; x < ROWS * (D / 8); x += 256) {
            const int m = x / (D / 8), c = x % (D / 8);
            uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f), g = f;   // f32 rows
            if (m < s.m) {
                const T * src = row_at<const T>(a, a.q, a.q_stride, s, m) + c * 8;
                if constexpr (SPLIT) {
                    f = *reinterpret_cast<const float4 *>(src);
                    g = *reinterpret_cast<const float4 *>(src + 4);
                } else {
                    hi = *reinterpret_cast<const uint4 *>(src);
                }
            }
            if constexpr (SPLIT) {
                const uint32_t field = row_field(lanes_max<D / 8>(fmaxf(largest4(f), largest4(g))));
                const float up = row_up(field);
                split_pair<C>(f.x * up, f.y * up, hi.x, lo.x);
                split_pair<C>(f.z * up, f.w * up, hi.y, lo.y);
                split_pair<C>(g.x * up, g.y * up, hi.z, lo.z);
                split_pair<C>(g.z * up, g.w * up, hi.w, lo.w);
                if (c == 0) q_scale[m] = row_scale(a.scale, field);
            }
            uint8_t * dst = qs + m * (D * 2) + ((c ^ (m & 7)) << 4);
            *reinterpret_cast<uint4 *>(dst) = hi;
            if constexpr (SPLIT || EIGHT) *reinterpret_cast<uint4 *>(dst + (EIGHT ? 8 : ROWS) * D * 2) = lo;
        }
        named_sync(1, 256);
        float o[D / 8][2 * XR], mx[XR], l[XR], scale[XR];
        int row[XR];
#pragma unroll
        for (int x = 0; x < XR; ++x) {
            mx[x] = -INFINITY;
            l[x] = 0.f;
            scale[x] = SPLIT ? q_scale[SPLIT ? rt * 16 + gq + 8 * x : 0] : a.scale;
            row[x] = by_group(a, s.m0 + min(rt * 16 + gq + 8 * x, s.m - 1));
        }
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
#pragma unroll
            for (int e = 0; e < 2 * XR; ++e) o[d][e] = 0.f;
        const int n_keys = s.n_keys, ctx = s.ctx, tiles = n_keys > 0 ? s.nt : 0;
#pragma unroll 1
        for (int t = 0; t < tiles; ++t, ++n) {
            const int st = n % L::STAGES;
            const int first = (s.t0 + t) * KT + k0, valid = n_keys - first;   // this warp's keys of the tile
            if (!wait(&full[st], (n / L::STAGES) & 1)) break;
            if (valid > 0 && valid < WK) {   // V rows past the item's keys: zeros, whatever the page holds there
#pragma unroll 1
                for (int x = lane; x < (WK - valid) * (D / 8); x += 32) {
                    const int key = k0 + valid + x / (D / 8), c = x % (D / 8);
                    *reinterpret_cast<uint4 *>(ring + st * L::STAGE + L::STAGE / 2 + place(key) + (c >> 3) * half + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
            }
            if (valid > 0) {
                const bool masked = first + WK > ctx;       // some of these keys are new rows, or past the last
                uint32_t seen[XR];
                if (masked) {
#pragma unroll
                    for (int x = 0; x < XR; ++x) seen[x] = seen_bits(a, s, row[x], first - ctx, valid);
                }
                float sc[2 * KS][4] = {}, low[2 * KS][4] = {};
                const uint32_t stage = st * L::STAGE;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    uint32_t q[4], p[4], b[KS][4];
                    ldsm4(q, q_at + (ks >> 2) * 128 + off_v[ks & 3]);
                    if constexpr (TERMS) ldsm4(p, q_at + ROWS * D * 2 + (ks >> 2) * 128 + off_v[ks & 3]);
#pragma unroll
                    for (int k = 0; k < KS; ++k) ldsm4(b[k], stage + k_at[k] + (ks >> 2) * half + off_k[ks & 3]);
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        mma<C>(sc[2 * k], q, b[k][0], b[k][1]);
                        mma<C>(sc[2 * k + 1], q, b[k][2], b[k][3]);
                        if constexpr (TERMS) {
                            mma<C>(low[2 * k], p, b[k][0], b[k][1]);
                            mma<C>(low[2 * k + 1], p, b[k][2], b[k][3]);
                        }
                    }
                }
                if constexpr (SPLIT) {
#pragma unroll
                    for (int y = 0; y < 2 * KS; ++y)
#pragma unroll
                        for (int e = 0; e < 2 * XR; ++e) sc[y][e] += EIGHT ? sc[y][2 + e] : low[y][e];
                }
                if (masked) {
                    // tokens that not every row sees: those whose V is not finite are cleared, and come in by themselves at the end
                    const int key = k0 + lane % WK, bit = first + lane % WK - s.ctx / KT * KT;   // a lane a token, or half of one
                    uint8_t * at = ring + st * L::STAGE + L::STAGE / 2 + place(key);
                    uint32_t m = 0;
#pragma unroll 4
                    for (int c = lane / WK; c < D / 8; c += 32 / WK) m = magnitude(m, *reinterpret_cast<const uint4 *>(at + (c >> 3) * half + (((c + lane) & 7) << 4)));
                    // another warp may share the tokens and clear them meanwhile: it says so first, so who reads its zeros sees that too
                    if (not_finite<C>(m) && bit < 512) atomicOr(&bad[bit >> 5], 1u << (bit & 31));
                    __threadfence_block();
                    __syncwarp();
                    const bool clear = bit < 512 && (*const_cast<volatile uint32_t *>(&bad[bit >> 5]) >> (bit & 31) & 1);
                    if (__any_sync(0xffffffffu, clear)) {
                        if (lane < WK && clear) {
#pragma unroll 1
                            for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4 *>(at + (c >> 3) * half + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
#pragma unroll
                    for (int x = 0; x < XR; ++x)
#pragma unroll
                        for (int y = 0; y < 2 * KS; ++y)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (!(seen[x] >> (y * 8 + 2 * tq + e) & 1)) sc[y][2 * x + e] = -INFINITY;
                }
                float m[XR];
                bool more = false;
#pragma unroll
                for (int x = 0; x < XR; ++x) {
                    m[x] = -INFINITY;
#pragma unroll
                    for (int y = 0; y < 2 * KS; ++y) m[x] = fmaxf(m[x], fmaxf(sc[y][2 * x], sc[y][2 * x + 1]));
                    m[x] = fmaxf(m[x], __shfl_xor_sync(0xffffffffu, m[x], 1));
                    m[x] = reference(fmaxf(m[x], __shfl_xor_sync(0xffffffffu, m[x], 2)), scale[x], LIFT<C>);
                    more = more || m[x] > mx[x];
                }
                if (__any_sync(0xffffffffu, more)) {
#pragma unroll
                    for (int x = 0; x < XR; ++x) {
                        m[x] = fmaxf(m[x], mx[x]);
                        const float w = m[x] == -INFINITY ? 1.f : exp2_fast(mx[x] - m[x]);
                        mx[x] = m[x];
                        l[x] *= w;
#pragma unroll
                        for (int d = 0; d < D / 8; ++d) {
                            o[d][2 * x] *= w;
                            o[d][2 * x + 1] *= w;
                        }
                    }
                }
                uint32_t ph[KS][4] = {}, pl[KS][4];
#pragma unroll
                for (int x = 0; x < XR; ++x) {
                    const float ref = mx[x] == -INFINITY ? 0.f : mx[x];
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const float * v = sc[2 * k + y] + 2 * x;
                            const float p0 = exp2_fast(fmaf(v[0], scale[x], -ref)), p1 = exp2_fast(fmaf(v[1], scale[x], -ref));
                            l[x] += p0 + p1;
                            if constexpr (TERMS) split_pair<C>(p0, p1, ph[k][2 * y + x], pl[k][2 * y + x]);
                            else if constexpr (EIGHT) split_pair<C>(p0, p1, ph[k][2 * y], ph[k][2 * y + 1]);
                            else ph[k][2 * y + x] = pack<C>(p0, p1);
                        }
                }
#pragma unroll
                for (int dp = 0; dp < D / 16; ++dp) {
                    uint32_t b[KS][4];
#pragma unroll
                    for (int k = 0; k < KS; ++k) ldsm4t(b[k], stage + v_at[k] + (dp >> 2) * half + off_v[dp & 3]);
                    if constexpr (SPLIT || EIGHT) {
                        float c[2][4] = {};
                        if constexpr (TERMS) {
#pragma unroll
                            for (int k = 0; k < KS; ++k) {
                                mma<C>(c[0], pl[k], b[k][0], b[k][1]);
                                mma<C>(c[1], pl[k], b[k][2], b[k][3]);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            mma<C>(c[0], ph[k], b[k][0], b[k][1]);
                            mma<C>(c[1], ph[k], b[k][2], b[k][3]);
                        }
#pragma unroll
                        for (int y = 0; y < 2; ++y)
#pragma unroll
                            for (int e = 0; e < 2 * XR; ++e)   // a value of infinity is in the high terms' sum; the low ones' may be 0 or less
                                o[2 * dp + y][e] += !EIGHT || !(fabsf(c[y][e]) < INFINITY) ? c[y][e] : c[y][e] + c[y][2 + e];
                    } else {
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            mma<C>(o[2 * dp], ph[k], b[k][0], b[k][1]);
                            mma<C>(o[2 * dp + 1], ph[k], b[k][2], b[k][3]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }

        // the warps' sums of a row become one: W dims at a time through shared memory, [warp][MR][W / 4 x 4], the pieces of
        // 4 swizzled by row; then a thread has 4 dims of a row
        constexpr int W = EIGHT ? D : 64, Q = W / 4;
        static_assert(8 * MR * W * 4 <= L::JOIN);
#pragma unroll
        for (int x = 0; x < XR; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            if (tq == 0) {
                stat[warp][0][gq + 8 * x] = mx[x];
                stat[warp][1][gq + 8 * x] = l[x];
            }
        }
        const bool whole = is_whole(s);
        float4 * pc = reinterpret_cast<float4 *>(piece(a, blockIdx.x, s.t0 == 0));
        named_sync(1, 256);                                      // q is read
        const bool any_bad = __any_sync(0xffffffffu, bad[lane & 15] != 0);
#pragma unroll
        for (int h = 0; h < D / W; ++h) {
#pragma unroll
            for (int d = 0; d < W / 8; ++d)
#pragma unroll
                for (int x = 0; x < XR; ++x) {
                    float2 * p = reinterpret_cast<float2 *>(sums + (warp * MR + gq + 8 * x) * Q + ((2 * d + (tq >> 1)) ^ gq)) + (tq & 1);
                    *p = make_float2(o[W / 8 * h + d][2 * x], o[W / 8 * h + d][2 * x + 1]);
                }
            named_sync(1, 256);
#pragma unroll 1
            for (int x = tid; x < ROWS * Q; x += 256) {
                const int m = x / Q, q = x % Q, r = m % MR, w0 = m / MR * KQ;
                if (m >= s.m) break;
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int k = 0; k < KQ; ++k) top = fmaxf(top, stat[w0 + k][0][r]);
                const float ref = top == -INFINITY ? 0.f : top;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < KQ; ++k) {
                    const float w = exp2_fast(stat[w0 + k][0][r] - ref);
                    const float4 v = sums[((w0 + k) * MR + r) * Q + (q ^ (r & 7))];
                    sum += w * stat[w0 + k][1][r];
                    y.x += w * v.x; y.y += w * v.y; y.z += w * v.z; y.w += w * v.w;
                }
                if (any_bad) y = with_bad<T, C, D>(a, s, bad, m, ref, W * h + 4 * q, y);
                if (whole) {
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    T * dst = row_at<T>(a, a.out, a.out_stride, s, m) + W * h + 4 * q;
                    if constexpr (SPLIT) *reinterpret_cast<float4 *>(dst) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
                    else *reinterpret_cast<uint2 *>(dst) = make_uint2(pack<C>(y.x * inv, y.y * inv), pack<C>(y.z * inv, y.w * inv));
                    if (a.lse && h == 0 && q == 0) put_lse(a, s, m, top, sum);
                } else {
                    pc[(Q * h + q) * ROWS + m] = y;
                    if (h == 0 && q == 0) {
                        float * st = reinterpret_cast<float *>(pc) + ROWS * D + m;
                        st[0] = top;
                        st[ROWS] = sum;
                    }
                }
            }
            named_sync(1, 256);
        }
        if (!whole) {
            if (tid == 0) is_last = arrive_piece(a, share.d, s);
            named_sync(1, 256);
            if (is_last) join<T, C, ROWS, D, 256, ROWS / 8, ROWS == 8 ? 8 : 4>(a, share.d, s, tid);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&segs.empty[sn % SegmentRing::N]);
    }
    named_sync(2, 288);
}

template <class T, class C, int D> void few(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, int rows, int sms, cudaStream_t stream) {
    const auto go = [&](auto kernel) {
        allow_smem(kernel, FewSmem<D>::BYTES);
        NAVI_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(sms)), dim3(288), FewSmem<D>::BYTES, stream, a, k, v));
    };
    if (rows <= 8) go(k_attend_few<T, C, D, 8>);
    else if (rows <= 16) go(k_attend_few<T, C, D, 16>);
    else go(k_attend_few<T, C, D, 32>);
}

} // namespace

void attend_few(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, int dtype, int cache, int rows, int sms, cudaStream_t stream) {
    const bool wide = a.head_dim == 128;
    if (dtype == NAVI_F32) wide ? few<float, __half, 128>(a, k, v, rows, sms, stream) : few<float, __half, 64>(a, k, v, rows, sms, stream);
    else if (cache == NAVI_F16) wide ? few<__half, __half, 128>(a, k, v, rows, sms, stream) : few<__half, __half, 64>(a, k, v, rows, sms, stream);
    else wide ? few<__nv_bfloat16, __nv_bfloat16, 128>(a, k, v, rows, sms, stream) : few<__nv_bfloat16, __nv_bfloat16, 64>(a, k, v, rows, sms, stream);
}

} // namespace navi::attn
