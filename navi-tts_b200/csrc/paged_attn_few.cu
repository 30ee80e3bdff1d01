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
// RT tiles of 16 rows, 8 / RT warps to each, which divide a key tile of 128 between them, each with
// a running maximum and sums of its own until the item ends; a ninth warp keeps a ring of tiles
// full by TMA. K and V are read once however many rows there are, so up to 32 rows the bound is
// HBM. f32 rows enter the products as two f16 terms, q = hi + lo and p = hi + lo, against the
// exact cache values, about 22 bits; the tensor cores' sums truncate, so the low terms and each
// step's contribution are summed apart and added in f32. 16-bit rows are exact, and p is
// rounded once to the type that the result has.
template <int D> struct FewSmem {
    static constexpr int STAGE = KT * D * 4;                    // K and V of a tile
    static constexpr int STAGES = D == 128 ? 3 : 6;
    static constexpr int JOIN = 4 * 16 * D * 4;                 // four warps' sums
    static constexpr int BYTES = 1024 + STAGES * STAGE + JOIN;  // 1024: to align the ring to the swizzle's 1024 bytes
};

template <class T, class C, int D, int RT>
__global__ void __launch_bounds__(288, 1) k_attend_few(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                                                       const __grid_constant__ CUtensorMap vmap) {
    constexpr bool SPLIT = std::is_same_v<T, float>;
    constexpr int ROWS = 16 * RT, KQ = 8 / RT, WK = KT / KQ;    // WK: keys of a tile that a warp takes
    using L = FewSmem<D>;
    extern __shared__ uint8_t raw[];
    uint8_t * ring = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    float4 * sums = reinterpret_cast<float4 *>(ring + L::STAGES * L::STAGE);
    // q lies in the upper half of the warps' sums, which are idle while it is read: [ROWS][D], f32 rows twice
    uint8_t * qs = reinterpret_cast<uint8_t *>(sums) + L::JOIN / 2;
    static_assert(2 * 32 * D * 2 <= L::JOIN / 2);
    __shared__ __align__(8) uint64_t full[L::STAGES], empty[L::STAGES];
    __shared__ __align__(8) SegmentRing segs;
    __shared__ float stat[8][2][16];
    __shared__ int red[9];
    __shared__ Share sh;
    __shared__ int abort_flag, is_last;
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
    griddep_wait();
    griddep_launch_dependents();
    share_out<ROWS, 288>(a, sh, red);
    if (sh.u >= sh.end) return;
    const Wait wait{&abort_flag, a.err};

    if (warp == 8) {
        Walk<ROWS> walk(a, sh);
        int n = 0;
        bool ok = true;
        const int kv = lane >> 4, box = lane & 15;   // half a warp each for K and V
#pragma unroll 1
        for (int k = 0; ok; ++k) {
            Segment s;
            const bool more = walk.next(s);
            if (k >= SegmentRing::N) ok = __shfl_sync(0xffffffffu, lane == 0 ? wait(&segs.empty[k % SegmentRing::N], (k / SegmentRing::N - 1) & 1) : 0, 0);
            if (!ok) break;
            if (lane == 0) {
                segs.s[k % SegmentRing::N] = s;
                mbar_arrive(&segs.full[k % SegmentRing::N]);
            }
            if (!more) break;
            if (s.n_keys <= 0) continue;
            int page = page_of_box<D>(a, s, s.t0, box);
#pragma unroll 1
            for (int t = s.t0; t < s.t0 + s.nt; ++t, ++n) {
                const int st = n % L::STAGES, next = t + 1 < s.t0 + s.nt ? page_of_box<D>(a, s, t + 1, box) : -1;
                if (n >= L::STAGES) ok = __shfl_sync(0xffffffffu, lane == 0 ? wait(&empty[st], (n / L::STAGES - 1) & 1) : 0, 0);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(2 * (tile_pages(a, s, t) << a.shift) * D * 2));
                __syncwarp();
                load_box<D>(a, kv ? &vmap : &kmap, s, page, box, ring + st * L::STAGE + kv * (L::STAGE / 2), &full[st]);
                page = next;
            }
        }
        // after an abort the copies still under way land before the block's shared memory goes
        if (abort_flag)
            for (int k = max(n - L::STAGES, 0); k < n; ++k) mbar_drain(&full[k % L::STAGES], (k / L::STAGES) & 1);
        return;
    }

    const int rt = warp / KQ, kq = warp % KQ, k0 = kq * WK;
    const uint32_t ring_at = smem_addr(ring), q_at = smem_addr(qs);
    const auto at = [](uint32_t base, int key, int piece) { return base + (piece >> 3) * (KT * 128) + key * 128 + (((piece & 7) ^ (key & 7)) << 4); };
    const auto q_swz = [](int row, int piece) { return static_cast<uint32_t>(row * (D * 2) + ((piece ^ (row & 7)) << 4)); };
    int n = 0;
#pragma unroll 1
    for (int sn = 0;; ++sn) {
        const bool got = wait(&segs.full[sn % SegmentRing::N], (sn / SegmentRing::N) & 1);
        // after an abort all warps leave together
        if (named_sync_or(1, 256, !got)) break;
        const Segment & s = segs.s[sn % SegmentRing::N];
        if (s.nt < 0) break;
        // q into shared memory, a thread 8 values
#pragma unroll 1
        for (int x = tid; x < ROWS * (D / 8); x += 256) {
            const int m = x / (D / 8), c = x % (D / 8);
            uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
            if (m < s.m) {
                const T * src = row_at<const T>(a, a.q, a.q_stride, s, m) + c * 8;
                if constexpr (SPLIT) {
                    const float4 f = *reinterpret_cast<const float4 *>(src), g = *reinterpret_cast<const float4 *>(src + 4);
                    split_pair<C>(f.x, f.y, hi.x, lo.x);
                    split_pair<C>(f.z, f.w, hi.y, lo.y);
                    split_pair<C>(g.x, g.y, hi.z, lo.z);
                    split_pair<C>(g.z, g.w, hi.w, lo.w);
                } else {
                    hi = *reinterpret_cast<const uint4 *>(src);
                }
            }
            *reinterpret_cast<uint4 *>(qs + q_swz(m, c)) = hi;
            if constexpr (SPLIT) *reinterpret_cast<uint4 *>(qs + ROWS * D * 2 + q_swz(m, c)) = lo;
        }
        named_sync(1, 256);
        float o[D / 8][4], mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int x = 0; x < D / 8; ++x) o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.f;
        const int n_keys = s.n_keys, ctx = s.ctx, tiles = n_keys > 0 ? s.nt : 0;
#pragma unroll 1
        for (int t = 0; t < tiles; ++t, ++n) {
            const int st = n % L::STAGES;
            if (!wait(&full[st], (n / L::STAGES) & 1)) break;
            const uint32_t sk = ring_at + st * L::STAGE, sv = sk + L::STAGE / 2;
            const int first = (s.t0 + t) * KT + k0, valid = n_keys - first;   // this warp's keys of the tile
            if (valid > 0 && valid < WK) {   // V rows past the item's keys: zeros, whatever the page holds there
#pragma unroll 1
                for (int x = lane; x < (WK - valid) * (D / 8); x += 32) {
                    const int key = k0 + valid + x / (D / 8);
                    *reinterpret_cast<uint4 *>(ring + (at(sv, key, x % (D / 8)) - ring_at)) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
            }
            // 16 keys at a time
#pragma unroll 1
            for (int k = 0; k < WK && k < valid; k += 16) {
                float sc[2][4] = {}, low[2][4] = {};
#pragma unroll 4
                for (int ks = 0; ks < D / 16; ++ks) {
                    uint32_t b[4], qh[4];
                    ldsm4(qh, q_at + q_swz(rt * 16 + (lane & 15), ks * 2 + (lane >> 4)));
                    ldsm4(b, at(sk, k0 + k + (lane & 7) + (lane >> 4) * 8, ks * 2 + ((lane >> 3) & 1)));
                    mma<C>(sc[0], qh, b[0], b[1]);
                    mma<C>(sc[1], qh, b[2], b[3]);
                    if constexpr (SPLIT) {
                        ldsm4(qh, q_at + ROWS * D * 2 + q_swz(rt * 16 + (lane & 15), ks * 2 + (lane >> 4)));
                        mma<C>(low[0], qh, b[0], b[1]);
                        mma<C>(low[1], qh, b[2], b[3]);
                    }
                }
                if constexpr (SPLIT) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[0][e] += low[0][e];
                        sc[1][e] += low[1][e];
                    }
                }
                if (first + k + 16 > ctx) {   // some of these keys are new rows, or past the last
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int j = by_group(a, s.m0 + min(rt * 16 + gq + 8 * x, s.m - 1));
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!sees(a, s, first + k + (e >> 1) * 8 + 2 * tq + (e & 1), j)) sc[e >> 1][2 * x + (e & 1)] = -INFINITY;
                    }
                }
                float m[2];
                bool more = false;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    m[x] = fmaxf(fmaxf(sc[0][2 * x], sc[0][2 * x + 1]), fmaxf(sc[1][2 * x], sc[1][2 * x + 1]));
                    m[x] = fmaxf(m[x], __shfl_xor_sync(0xffffffffu, m[x], 1));
                    m[x] = fmaxf(m[x], __shfl_xor_sync(0xffffffffu, m[x], 2)) * a.scale;
                    more = more || m[x] > mx[x];
                }
                if (__any_sync(0xffffffffu, more)) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
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
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float ref = mx[x] == -INFINITY ? 0.f : mx[x];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float p0 = exp2_fast(fmaf(sc[y][2 * x], a.scale, -ref)), p1 = exp2_fast(fmaf(sc[y][2 * x + 1], a.scale, -ref));
                        l[x] += p0 + p1;
                        if constexpr (SPLIT) split_pair<C>(p0, p1, ph[2 * y + x], pl[2 * y + x]);
                        else ph[2 * y + x] = pack<C>(p0, p1);
                    }
                }
#pragma unroll
                for (int dp = 0; dp < D / 16; ++dp) {
                    uint32_t b[4];
                    ldsm4t(b, at(sv, k0 + k + (lane & 15), dp * 2 + (lane >> 4)));
                    if constexpr (SPLIT) {
                        float c[2][4] = {};
                        mma<C>(c[0], pl, b[0], b[1]);
                        mma<C>(c[1], pl, b[2], b[3]);
                        mma<C>(c[0], ph, b[0], b[1]);
                        mma<C>(c[1], ph, b[2], b[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[2 * dp][e] += c[0][e];
                            o[2 * dp + 1][e] += c[1][e];
                        }
                    } else {
                        mma<C>(o[2 * dp], ph, b[0], b[1]);
                        mma<C>(o[2 * dp + 1], ph, b[2], b[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }

        // the warps' sums of a row become one
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            if (tq == 0) {
                stat[warp][0][gq + 8 * x] = mx[x];
                stat[warp][1][gq + 8 * x] = l[x];
            }
        }
        named_sync(1, 256);
        float top[2], sum[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            top[x] = -INFINITY;
            sum[x] = 0.f;
#pragma unroll 4
            for (int k = 0; k < KQ; ++k) top[x] = fmaxf(top[x], stat[rt * KQ + k][0][gq + 8 * x]);
            const float ref = top[x] == -INFINITY ? 0.f : top[x];
#pragma unroll 4
            for (int k = 0; k < KQ; ++k) sum[x] += stat[rt * KQ + k][1][gq + 8 * x] * exp2_fast(stat[rt * KQ + k][0][gq + 8 * x] - ref);
            const float w = exp2_fast(mx[x] - ref);
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
                o[d][2 * x] *= w;
                o[d][2 * x + 1] *= w;
            }
        }
#pragma unroll 1
        for (int half = KQ / 2; half >= 1; half /= 2) {
            float4 * slot = sums + (kq % half * RT + rt) * (4 * D) + lane;
            if (kq >= half && kq < 2 * half) {
#pragma unroll
                for (int d = 0; d < D / 8; ++d) slot[d * 32] = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
            }
            named_sync(1, 256);
            if (kq < half) {
#pragma unroll
                for (int d = 0; d < D / 8; ++d) {
                    const float4 v = slot[d * 32];
                    o[d][0] += v.x; o[d][1] += v.y; o[d][2] += v.z; o[d][3] += v.w;
                }
            }
            if (half > 1) named_sync(1, 256);
        }
        const int whole = s.whole;
        if (kq == 0) {
            float * pc = piece(a, blockIdx.x, s.slot);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int m = rt * 16 + gq + 8 * x;
                if (m >= s.m) continue;
                if (whole) {
                    const float inv = sum[x] == 0.f ? 0.f : 1.f / sum[x];
                    T * dst = row_at<T>(a, a.out, a.out_stride, s, m) + 2 * tq;
#pragma unroll
                    for (int d = 0; d < D / 8; ++d) {
                        const float v = o[d][2 * x] * inv, w = o[d][2 * x + 1] * inv;
                        if constexpr (SPLIT) *reinterpret_cast<float2 *>(dst + d * 8) = make_float2(v, w);
                        else *reinterpret_cast<uint32_t *>(dst + d * 8) = pack<C>(v, w);
                    }
                    if (a.lse && tq == 0) put_lse(a, s, m, top[x], sum[x]);
                } else {
#pragma unroll
                    for (int d = 0; d < D / 8; ++d)
                        *reinterpret_cast<float2 *>(pc + ((2 * d + (tq >> 1)) * ROWS + m) * 4 + 2 * (tq & 1)) = make_float2(o[d][2 * x], o[d][2 * x + 1]);
                    if (tq == 0) {
                        pc[ROWS * D + m] = top[x];
                        pc[ROWS * D + ROWS + m] = sum[x];
                    }
                }
            }
        }
        if (!whole) {
            __threadfence();
            named_sync(1, 256);
            if (tid == 0) is_last = arrive_piece(a, s);
            named_sync(1, 256);
            if (is_last) join<T, C, ROWS, D, 256, 8, L::JOIN / 4>(a, s, tid, reinterpret_cast<float *>(sums));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&segs.empty[sn % SegmentRing::N]);
    }
}

template <class T, class C, int D> void few(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, int rows, int sms, cudaStream_t stream) {
    const auto go = [&](auto kernel) {
        NAVI_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, FewSmem<D>::BYTES));
        NAVI_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(sms)), dim3(288), FewSmem<D>::BYTES, stream, a, k, v));
    };
    if (rows <= 16) go(k_attend_few<T, C, D, 1>);
    else go(k_attend_few<T, C, D, 2>);
}

} // namespace

void attend_few(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, int dtype, int cache, int rows, int sms, cudaStream_t stream) {
    const bool wide = a.head_dim == 128;
    if (dtype == NAVI_F32) wide ? few<float, __half, 128>(a, k, v, rows, sms, stream) : few<float, __half, 64>(a, k, v, rows, sms, stream);
    else if (cache == NAVI_F16) wide ? few<__half, __half, 128>(a, k, v, rows, sms, stream) : few<__half, __half, 64>(a, k, v, rows, sms, stream);
    else wide ? few<__nv_bfloat16, __nv_bfloat16, 128>(a, k, v, rows, sms, stream) : few<__nv_bfloat16, __nv_bfloat16, 64>(a, k, v, rows, sms, stream);
}

} // namespace navi::attn
