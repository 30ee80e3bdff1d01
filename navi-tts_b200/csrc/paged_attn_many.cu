// Attention over the paged KV cache for many rows of a request (paged_attn.cu): larger drafted
// trees and chunks of prompts, on the tcgen05 tensor cores.
#include "paged_attn.hpp"
#include "paged_attn.cuh"
#include "tmem.cuh"
#include "umma.cuh"

namespace navi::attn {

namespace {

using namespace navi::umma;

// A block (one a multiprocessor) holds 128 or 256 rows x heads of an item. Two warpgroups do the
// softmax, a thread a row; one thread feeds the ring of K and V tiles by TMA, one issues the MMAs.
// Each warpgroup has its scores S (128 columns of tensor memory, its weights P written over them)
// and its sums O (D columns), so that while one does its softmax the tensor cores work for the
// other. With more than 128 rows the warpgroups take 128 rows each and share every K and V tile;
// with fewer they take the key tiles in turn, each with a maximum and sums of its own, and join
// them when the item ends.
//
// The MMA thread issues, for the pairs n = 0, 1, ... of (warpgroup n & 1, key tile):
//   S(0) S(1) | P V(0) S(2) | P V(1) S(3) | ...     each P V after its warpgroup has written P
// A commit covers all that was issued before it, so when S(n) is there P V(n - 2), the last to
// touch this warpgroup's O, is done too, and the warpgroup may rescale O. It does so only where
// a row's maximum grew by more than 2^LAZY: bf16 weights up to 2^8 are as exact, and sums are f32. f16 weights
// are 2^14 at first and up to 2^15 (LIFT + LAZY, of 65504), so that a long tail keeps its weights: see reference().
//
// f32 rows: q and p as two f16 terms each against the exact cache values, as in the kernel for few
// rows. Two tiles of q do not fit then, so their items have 128 rows. Bringing each row of q to f16's range costs
// 4 to 5 % there (48 trees of up to 33 f32 rows 125 -> 132 us, 8 chunks 422 -> 434).
//
// Measured on one B200: 8 chunks of 1000 bf16 rows over 511 to 4097 tokens: 199 to 224 us, 675 to 760 TFLOP/s;
// a plain matrix product reaches 1669. 128 rows x 128 keys take about 2000 cycles in the loop, their two products
// alone 1025 to 1136 in a loop of nothing else. 48 trees of up to 33 f16 rows over 255 to 8191 tokens in pages of
// 16: 98 to 108 us, 4.2 to 4.6 TB/s; counters for both: the tensor pipe 41 and 26 % of the cycles, ex2's pipe 42 and
// 26 %, so each waits for the other. The f32 variants spill 20 to 28 bytes a thread. Weights go over in two halves
// (48 trees 96 us; whole 97). Tried and slower: S in units of 64 keys with two buffers a warpgroup (279 us for the chunks, 210 then: an MMA of 64 columns
// takes as long as one of 128), an MMA warp for each warpgroup (222 us, 204 then).
// f16: LAZY 1, 2, 3, 5 and 8 with LIFT to match (15 - LAZY): 48 trees 99.8, 99.0, 98.6, 98.1 and 98.0 us, 8 chunks of
// f16 rows 219, 224, 218, 221 and 216, of f32 rows 431, 429 to 435, 417, 429 and 436 (410 to 419 without LIFT): the
// closest was taken.
template <class C> constexpr float LIFT = std::is_same_v<C, __half> ? 14.f : 0.f;
template <class C> constexpr float LAZY = std::is_same_v<C, __half> ? 1.f : 8.f;
constexpr int EXTRA = 1;                                        // what an item costs beside its key tiles, in key tiles. 48 trees with 0 to 3: 102, 102, 108, 113 us; 8 chunks 217, 210, 211, 209

template <class T, int D, int ROWS> struct ManySmem {
    static constexpr bool SPLIT = std::is_same_v<T, float>;
    static constexpr int QTILE = 128 * D * 2;                   // 128 rows, 16-bit: [D / 64][128][128 B], swizzled
    static constexpr int STAGE = KT * D * 2;                    // K or V of a key tile
    static constexpr int QTILES = SPLIT || ROWS > 128 ? 2 : 1;
    static constexpr int STAGES = D == 128 ? 7 - QTILES : 8;
    static constexpr int CONTROL = 3072;                        // ManyControl, and the tiles at 1024-byte boundaries
    static constexpr int BYTES = CONTROL + QTILES * QTILE + STAGES * STAGE;
    static_assert(BYTES <= 227 * 1024);
};

struct ManyControl {
    uint64_t full[8], empty[8], q_full, q_empty, s_full[2], p_full[2][2], o_full[2], drained, q_scaled[2];
    float stat[2][2][128];
    uint8_t q_field[2][128];     // f32 rows: row_field of this segment's and the next one's
    uint32_t bad[16];            // tokens from the first masked tile on whose V is not finite
    SegmentRing segs;
    int red[12];
    Share sh;
    uint32_t tmem_at;
    volatile int abort_flag;
    int is_last;
};

// K-major rows (Q, K): desc_kmajor_sw128 of umma.cuh. V is the B operand with its rows along the
// summed dimension (MN-major): atoms of 64 dims x 8 keys, the next 8 keys 1024 bytes on, the next 64
// dims `lbo` bytes on.
__device__ __forceinline__ uint64_t desc_mnmajor_sw128(uint32_t addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// kind::f16 with both operands f16 or both bf16, f32 sums; B along its rows when v_major
template <class C> constexpr uint32_t idesc(int M, int N, bool v_major) {
    constexpr uint32_t f = std::is_same_v<C, __nv_bfloat16> ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | (v_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
// The warp that issues the MMAs runs as one, so that descriptors stay in uniform registers (moving
// them there for every MMA cost more than the MMA); `leader` is set in one of its lanes.
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t id, bool accumulate, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(id), "r"(accumulate ? 1u : 0u), "r"(leader)
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t id, bool accumulate, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(id), "r"(accumulate ? 1u : 0u), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void commit_by(uint64_t * bar, uint32_t leader) {
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
                     smem_addr(bar)),
                 "r"(leader)
                 : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

template <class T, class C, int D, int ROWS>   // ROWS: 128 or 256 rows of an item
__global__ void __launch_bounds__(384, 1) k_attend_many(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                                                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap) {
    constexpr bool SPLIT = std::is_same_v<T, float>;
    using L = ManySmem<T, D, ROWS>;
    static_assert(sizeof(ManyControl) <= L::CONTROL && L::STAGES <= 8);
    extern __shared__ __align__(1024) uint8_t raw[];   // all of the block's shared memory: at a 1024-byte boundary
    ManyControl & S = *reinterpret_cast<ManyControl *>(raw);
    uint8_t * qs = raw + L::CONTROL, * ring = qs + L::QTILES * L::QTILE;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        S.abort_flag = 0;
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        mbar_init(&S.q_full, a.q_boxes ? 1 : 64);
        mbar_init(&S.q_empty, 1);
        for (int g = 0; g < 2; ++g) {
            mbar_init(&S.s_full[g], 1);
            mbar_init(&S.p_full[g][0], 128);
            mbar_init(&S.p_full[g][1], 128);
            mbar_init(&S.o_full[g], 1);
            mbar_init(&S.q_scaled[g], 64);
        }
        mbar_init(&S.drained, 1);
        S.segs.init(11);
        fence_mbar_init();
    }
    if (warp == 9) {
        tmem_alloc(&S.tmem_at, 512);
        tmem_relinquish();
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    griddep_wait();
    griddep_launch_dependents();
    const bool one = a.n_req <= 32;
    if (!one) share_of_block<ROWS, EXTRA, 384>(a, S.sh, S.red);
    const uint32_t tmem = S.tmem_at;
    const Wait wait{&S.abort_flag, a.err};
    int issued = 0;              // by this warp: tiles of K and V, or q of so many segments by TMA

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) {
            Request first{};
            Share sh;
            if (one) {
                sh = share_of_warp<ROWS, EXTRA>(a, first);
                if (lane == 0) S.sh.d = sh.d;                   // the other roles read it after a segment
            } else {
                sh = S.sh;
                if (sh.u < sh.end) first = request(a, sh.i);
            }
            Walk<ROWS, EXTRA> walk(a, sh, first);
            int n = 0;
            bool ok = true;
#pragma unroll 1
            for (int k = 0; ok; ++k) {
                Segment s;
                const bool more = walk.next(s);
                if (k >= SegmentRing::N) ok = __shfl_sync(0xffffffffu, lane == 0 ? wait(&S.segs.empty[k % SegmentRing::N], (k / SegmentRing::N - 1) & 1) : 0, 0);
                if (!ok) break;
                // a box is half of a page's dims (D = 128), so that a tile is halves of [KT][64] in 128-byte swizzled rows
                const int half = lane % (D / 64), nth = (lane & 15) / (D / 64);
                int page = more && s.n_keys > 0 ? page_at(a, s, s.t0, nth) : -1;
                if (lane == 0) {
                    S.segs.s[k % SegmentRing::N] = s;
                    mbar_arrive(&S.segs.full[k % SegmentRing::N]);
                }
                if (!more) break;
                if (s.n_keys <= 0) continue;
#pragma unroll 1
                for (int t = s.t0; t < s.t0 + s.nt && ok; ++t) {
                    const int next = t + 1 < s.t0 + s.nt ? page_at(a, s, t + 1, nth) : -1;
#pragma unroll 1
                    for (int kv = 0; kv < 2 && ok; ++kv) {
                        const int st = n % L::STAGES;
                        if (n >= L::STAGES) ok = __shfl_sync(0xffffffffu, lane == 0 ? wait(&S.empty[st], (n / L::STAGES - 1) & 1) : 0, 0);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&S.full[st], static_cast<uint32_t>((tile_pages(a, s, t) << a.shift) * D * 2));
                        __syncwarp();
                        if (lane < 16 && page >= 0)
                            tma_box_2d(ring + st * L::STAGE + half * (KT * 128) + (nth << a.shift) * 128, kv ? &vmap : &kmap, half * 64,
                                       (page * a.n_kv + s.g) << a.shift, &S.full[st]);
                        ++n;
                    }
                    page = next;
                }
            }
            issued = n;
        } else if (warp == 9) {
            constexpr uint32_t ID_S = idesc<C>(128, KT, false), ID_O = idesc<C>(128, D, true);
            const uint32_t leader = lane == 0, tm = static_cast<uint32_t>(uniform(static_cast<int>(tmem)));
            const uint64_t q_desc = desc_kmajor_sw128(smem_addr(qs)), k_desc = desc_kmajor_sw128(smem_addr(ring)), v_desc = desc_mnmajor_sw128(smem_addr(ring), KT * 128);
            const auto wait_all = [&](uint64_t * bar, int parity) { return __all_sync(0xffffffffu, wait(bar, static_cast<uint32_t>(parity))) != 0; };
            const auto all = [](bool x) { return __all_sync(0xffffffffu, x) != 0; };
            // places in the ring: stage and the parity of its turn
            struct Place {
                int st = 0, turn = 0;
                __device__ __forceinline__ void go(int by) {
                    st += by;
                    if (st >= L::STAGES) {
                        st -= L::STAGES;
                        turn ^= 1;
                    }
                }
            };
            Place kp, vp;                                  // the next K and V tile
            vp.go(1);
            int nq = 0, np0 = 0, np1 = 0;
            // The pairs of a segment. A barrier's answer takes a while, so those that a step needs are asked together, and
            // waited for one by one only if one of them says no. TWO: the warpgroups share the tiles, arithmetic is the bound,
            // and everything is there before the two products, which then follow one another. Otherwise HBM is the bound,
            // and P V, which frees a stage, does not wait for the next K.
            const auto run = [&](auto two_c, int P) {
                constexpr bool TWO = decltype(two_c)::value;
                // step n asks for the scores of pair n + 2 once P V of pair n is under way; the first two only ask
#pragma unroll 1
                for (int n = -2; n < P; ++n) {
                    const int g = n & 1, turn = (g ? np1 : np0) & 1, v_st = uniform(vp.st), k_st = uniform(kp.st);
                    const bool pv = n >= 0, next = n + 2 < P, opens = !TWO || g == 0, closes = !TWO || g == 1;   // a tile's first and last pair
                    const bool r_v = !pv || !opens || mbar_try_wait(&S.full[vp.st], vp.turn), r_k = !TWO || !next || !opens || mbar_try_wait(&S.full[kp.st], kp.turn);
                    const bool r_0 = !pv || mbar_try_wait(&S.p_full[g][0], turn), r_1 = !pv || mbar_try_wait(&S.p_full[g][1], turn);
                    if (!all(r_v && r_k && r_0)) {
                        if (pv && opens && !wait_all(&S.full[vp.st], vp.turn)) return false;
                        if (TWO && next && opens && !wait_all(&S.full[kp.st], kp.turn)) return false;
                        if (pv && !wait_all(&S.p_full[g][0], turn)) return false;
                    }
                    fence_after_sync();
                    if (pv) {
                        if (g) ++np1;
                        else ++np0;
                        const uint32_t d = tm + 256 + g * 128, p = tm + g * 128;
                        const uint64_t v = v_desc + static_cast<uint32_t>(v_st * (L::STAGE >> 4));
                        // the weights come in two halves: P V of the first may run while the second is still made
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (h == 1 && !all(r_1)) {
                                if (!wait_all(&S.p_full[g][1], turn)) return false;
                                fence_after_sync();
                            }
#pragma unroll
                            for (int term = 0; term < (SPLIT ? 2 : 1); ++term)
#pragma unroll
                                for (int ks = 4 * h; ks < 4 * h + 4; ++ks)
                                    mma_ts(d, p + (SPLIT ? (1 - term) * 64 : 0) + ks * 8, v + ks * (2048 >> 4), ID_O, n > 1 || term > 0 || ks > 0, leader);
                        }
                        if (n + 2 >= P) commit_by(&S.o_full[g], leader);
                        if (closes) {
                            commit_by(&S.empty[vp.st], leader);
                            vp.go(2);
                        }
                    }
                    if (next) {
                        if (!TWO) {
                            if (!wait_all(&S.full[kp.st], kp.turn)) return false;
                            fence_after_sync();
                        }
                        const uint32_t d = tm + g * 128;
                        const uint64_t q = q_desc + static_cast<uint32_t>(TWO ? g * (L::QTILE >> 4) : 0), k = k_desc + static_cast<uint32_t>(k_st * (L::STAGE >> 4));
#pragma unroll
                        for (int term = 0; term < (SPLIT ? 2 : 1); ++term)
#pragma unroll
                            for (int ks = 0; ks < D / 16; ++ks) {
                                constexpr int HALF = 128 * 128 >> 4;
                                const int o = (ks >> 2) * HALF + (ks & 3) * 2;
                                mma_ss(d, q + (SPLIT ? (1 - term) * (L::QTILE >> 4) : 0) + o, k + o, ID_S, term > 0 || ks > 0, leader);
                            }
                        commit_by(&S.s_full[g], leader);
                        if (n + 3 == P) commit_by(&S.q_empty, leader);
                        if (closes) {
                            commit_by(&S.empty[kp.st], leader);
                            kp.go(2);
                        }
                    }
                }
                return true;
            };
#pragma unroll 1
            for (int sn = 0;; ++sn) {
                if (!wait_all(&S.segs.full[sn % SegmentRing::N], (sn / SegmentRing::N) & 1)) break;
                const Segment & s = S.segs.s[sn % SegmentRing::N];
                const int s_nt = uniform(s.nt), s_m = uniform(s.m), nt = uniform(s.n_keys) > 0 ? s_nt : 0;
                if (s_nt < 0) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.segs.empty[sn % SegmentRing::N]);
                if (nt == 0) continue;
                if (!wait_all(&S.q_full, nq & 1)) break;
                ++nq;
                fence_after_sync();
                bool ok;
                if (ROWS > 128 && s_m > 128) ok = run(std::bool_constant<(ROWS > 128)>{}, 2 * nt);
                else ok = run(std::false_type{}, nt);
                if (!ok) break;
            }
            // nothing may still write the tensor memory when it is given back
            commit_by(&S.drained, leader);
            __syncwarp();
            mbar_drain(&S.drained, 0);
        } else if (warp >= 10) {
            // q of a segment into shared memory, as soon as no MMA reads the last one's: by TMA, the heads of a
            // row next to one another, or 64 threads, 16-byte pieces of 16-bit values, U of them at a time (f32
            // rows: the high terms, then the low ones)
            int nq = 0;
#pragma unroll 1
            for (int sn = 0;; ++sn) {
                bool ok = wait(&S.segs.full[sn % SegmentRing::N], (sn / SegmentRing::N) & 1);
                const Segment & it = S.segs.s[sn % SegmentRing::N];
                const bool has = ok && it.nt > 0 && it.n_keys > 0;
                if (has && nq > 0) ok = wait(&S.q_empty, (nq - 1) & 1);
                if (named_sync_or(2, 64, !ok) || it.nt < 0) break;   // after an abort both warps leave together
                if (has && a.q_boxes) {
                    ++nq;
                    issued = nq;
                    if (tid == 320) {
                        const int tiles = it.m > 128 ? 2 : 1;
                        mbar_arrive_expect_tx(&S.q_full, static_cast<uint32_t>(tiles * L::QTILE));
#pragma unroll 1
                        for (int x = 0; x < tiles * (D / 64); ++x) {
                            const int tile = x / (D / 64), h = x % (D / 64);
                            tma_box_3d(qs + tile * L::QTILE + h * (128 * 128), &qmap, h * 64, it.g * a.group, it.row0 + by_group(a, it.m0 + tile * 128), &S.q_full);
                        }
                    }
                } else if (has) {
                    ++nq;
                    constexpr int CH = D / 8, STEP = 64 / CH, U = SPLIT ? 4 : 8;   // pieces of a row; rows a pass
                    const int c = tid % CH, rows = it.m > 128 ? 256 : 128;
#pragma unroll 1
                    for (int m1 = (tid & 63) / CH; m1 < rows; m1 += U * STEP) {
                        uint4 v[U], w[SPLIT ? U : 1];
#pragma unroll
                        for (int k = 0; k < U; ++k) {
                            const int m = m1 + k * STEP;
                            v[k] = make_uint4(0, 0, 0, 0);
                            if constexpr (SPLIT) w[k] = v[k];
                            if (m < it.m) {
                                const uint4 * src = reinterpret_cast<const uint4 *>(row_at<const T>(a, a.q, a.q_stride, it, m) + c * 8);
                                v[k] = src[0];
                                if constexpr (SPLIT) w[k] = src[1];
                            }
                        }
#pragma unroll
                        for (int k = 0; k < U; ++k) {
                            const int m = m1 + k * STEP;
                            uint8_t * dst = qs + (m >> 7) * L::QTILE + (c >> 3) * (128 * 128) + (m & 127) * 128 + (((c & 7) ^ (m & 7)) << 4);
                            if constexpr (SPLIT) {
                                const float4 f = *reinterpret_cast<const float4 *>(&v[k]), g = *reinterpret_cast<const float4 *>(&w[k]);
                                const uint32_t field = row_field(lanes_max<CH>(fmaxf(largest4(f), largest4(g))));
                                const float up = row_up(field);
                                uint4 hi, lo;
                                split_pair<C>(f.x * up, f.y * up, hi.x, lo.x);
                                split_pair<C>(f.z * up, f.w * up, hi.y, lo.y);
                                split_pair<C>(g.x * up, g.y * up, hi.z, lo.z);
                                split_pair<C>(g.z * up, g.w * up, hi.w, lo.w);
                                if (c == 0) S.q_field[(nq - 1) & 1][m] = static_cast<uint8_t>(field);
                                *reinterpret_cast<uint4 *>(dst) = hi;
                                *reinterpret_cast<uint4 *>(dst + L::QTILE) = lo;
                            } else {
                                *reinterpret_cast<uint4 *>(dst) = v[k];
                            }
                        }
                    }
                    fence_proxy_async_smem();
                    mbar_arrive(&S.q_full);
                    if constexpr (SPLIT) mbar_arrive(&S.q_scaled[(nq - 1) & 1]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.segs.empty[sn % SegmentRing::N]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int wg = warp >> 2, r = tid & 127;
        const uint32_t lane_at = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lane_at + wg * 128, o_at = tmem + lane_at + 256 + wg * 128;
        int base = 0, ns = 0, no0 = 0, no1 = 0;
#pragma unroll 1
        for (int sn = 0;; ++sn) {
            const bool got = wait(&S.segs.full[sn % SegmentRing::N], (sn / SegmentRing::N) & 1);
            if (tid < 16) S.bad[tid] = 0;
            // after an abort all warps leave together
            if (named_sync_or(1, 256, !got)) break;
            const Segment & it = S.segs.s[sn % SegmentRing::N];
            if (it.nt < 0) break;
            const bool two = ROWS > 128 && it.m > 128;
            const int nt = it.n_keys > 0 ? it.nt : 0, n_keys = it.n_keys, ctx = it.ctx, t0 = it.t0;
            const int m = (two ? wg * 128 : 0) + r, j = by_group(a, it.m0 + min(m, it.m - 1));
            // every row of the warp sees the tokens before `open`
            const int open = ctx + (a.mask ? 0 : by_group(a, it.m0 + min((two ? wg * 128 : 0) + (warp & 3) * 32, it.m - 1)) + 1);
            const int open0 = ctx + (a.mask ? 0 : by_group(a, it.m0) + 1), bad0 = open0 / KT * KT;   // the same for the item; its first masked tile
            float top = -INFINITY, sum = 0.f, scale = a.scale;
            bool any = false;                             // this warpgroup has had a tile
            if (SPLIT && wg < nt) {   // this place is next written two segments on, behind the weights of this one
                wait(&S.q_scaled[no0 & 1], (no0 >> 1) & 1);
                scale = row_scale(a.scale, S.q_field[no0 & 1][r]);
            }
            for (int x = two ? 0 : wg; x < nt; x += two ? 1 : 2, ++ns) {
                if (!wait(&S.s_full[wg], ns & 1)) break;
                fence_after_sync();
                const int key0 = (t0 + x) * KT, left = n_keys - key0;
                if (key0 + KT > open0) {              // some of these tokens are not seen by every row of the item
                    const int idx = base + 2 * x + 1, st = idx % L::STAGES;
                    wait(&S.full[st], (idx / L::STAGES) & 1);
                    // V rows past the last token, whatever the page holds there, and those that are not finite: zeros. A thread a row
                    uint8_t * row = ring + st * L::STAGE + r * 128;
                    bool clear = r >= left;
                    if (!clear) {
                        uint32_t m = 0;
#pragma unroll
                        for (int c = 0; c < D / 8; ++c) m = magnitude(m, *reinterpret_cast<const uint4 *>(row + (c >> 3) * (KT * 128) + (((c + r) & 7) << 4)));
                        // the other warpgroup may share the tile and clear the row meanwhile: it says so first, so who reads
                        // its zeros sees that too
                        const int bit = key0 - bad0 + r;
                        if (bit < 512) {
                            if (not_finite<C>(m)) atomicOr(&S.bad[bit >> 5], 1u << (bit & 31));
                            __threadfence_block();
                            clear = *const_cast<volatile uint32_t *>(&S.bad[bit >> 5]) >> (bit & 31) & 1;
                        }
                    }
                    if (clear) {
#pragma unroll 1
                        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4 *>(row + (c >> 3) * (KT * 128) + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async_smem();
                    }
                }
                uint32_t s[KT];
                tmem_ld<64>(s_at, s);
                tmem_ld<64>(s_at + 64, s + 64);
                if (key0 + KT > open) {                   // some of these tokens are not seen by every row of the warp
#pragma unroll
                    for (int w = 0; w < KT / 32; ++w) {
                        const uint32_t b = seen_bits(a, it, j, key0 + 32 * w - ctx, left - 32 * w);
#pragma unroll
                        for (int k = 0; k < 32; ++k) s[32 * w + k] = b >> k & 1 ? s[32 * w + k] : __float_as_uint(-INFINITY);
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < KT; k += 2) mx[k / 2 & 3] = max3(mx[k / 2 & 3], __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
                const float best = reference(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), scale, LIFT<C>);
                if (!any) {
                    top = best;
                } else if (__any_sync(0xffffffffu, best > top + LAZY<C>)) {
                    const float now = fmaxf(best, top), w = now == -INFINITY ? 1.f : exp2_fast(top - now);
                    top = now;
                    sum *= w;
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_ld<32>(o_at + c, o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * w);
                        tmem_st<32>(o_at + c, o);
                    }
                }
                any = true;
                const float ref = top == -INFINITY ? 0.f : top;
                const float2 scale2 = make_float2(scale, scale), ref2 = make_float2(-ref, -ref);
                float2 part[2] = {};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t hi[32], lo[SPLIT ? 32 : 1];
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const int c = 64 * h + 2 * k;
                        const float2 e = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale2, ref2);
                        const float2 w = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                        part[k & 1] = __fadd2_rn(part[k & 1], w);
                        if constexpr (SPLIT) split_pair<C>(w.x, w.y, hi[k], lo[k]);
                        else hi[k] = pack<C>(w.x, w.y);
                    }
                    tmem_st<32>(s_at + 32 * h, hi);
                    if constexpr (SPLIT) tmem_st<32>(s_at + 64 + 32 * h, lo);
                    tmem_st_wait();
                    fence_before_sync();
                    mbar_arrive(&S.p_full[wg][h]);
                }
                sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
            }
            base += 2 * nt;
            // which warpgroup's sums there are: none where the rows see no key (a request that is not served); both
            // read both where they took the key tiles in turn
            const bool use0 = nt > 0 && (!two || wg == 0), use1 = two ? nt > 0 && wg == 1 : nt > 1;
            if (use0) wait(&S.o_full[0], no0 & 1);
            if (use1) wait(&S.o_full[1], no1 & 1);
            no0 += nt > 0;
            no1 += two ? nt > 0 : nt > 1;
            fence_after_sync();
            const bool whole = is_whole(it);
            float w0 = 1.f, w1 = 1.f;                     // what their O count
            int c_lo = 0, c_hi = D;                       // the columns that this warpgroup finishes
            if (!two) {
                S.stat[wg][0][r] = top;
                S.stat[wg][1][r] = sum;
                named_sync(1, 256);
                const float t0 = S.stat[0][0][r], t1 = S.stat[1][0][r];
                top = fmaxf(t0, t1);
                const float ref = top == -INFINITY ? 0.f : top;
                w0 = exp2_fast(t0 - ref);
                w1 = exp2_fast(t1 - ref);
                sum = S.stat[0][1][r] * w0 + S.stat[1][1][r] * w1;
                c_lo = wg * (D / 2);
                c_hi = c_lo + D / 2;
            }
            {
                float4 * pc = reinterpret_cast<float4 *>(piece(a, blockIdx.x, it.t0 == 0)) + m;
                const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
                const bool live = m < it.m;
                const bool bad = __any_sync(0xffffffffu, S.bad[lane & 15] != 0);   // tokens of this segment whose V was cleared
                T * dst = row_at<T>(a, a.out, a.out_stride, it, live ? m : 0);
                const bool wide = (reinterpret_cast<uintptr_t>(dst) & 31) == 0;   // rows are at least 16-byte aligned
                w0 *= inv;
                w1 *= inv;
#pragma unroll 1
                for (int c = c_lo; c < c_hi; c += 32) {
                    uint32_t o[32];
                    float v[32] = {};
                    if (use0) {
                        tmem_ld<32>(tmem + lane_at + 256 + c, o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(o[k]) * w0;
                    }
                    if (use1) {
                        tmem_ld<32>(tmem + lane_at + 384 + c, o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[k] += __uint_as_float(o[k]) * w1;
                    }
                    if (!live) continue;
                    if (bad) {
#pragma unroll 1
                        for (int w = 0; w < 16; ++w)
#pragma unroll 1
                            for (uint32_t left = S.bad[w]; left; left &= left - 1) {
                                const int key = bad0 + 32 * w + __ffs(left) - 1;
                                if (!(seen_bits(a, it, j, key - ctx, n_keys - key) & 1)) continue;
                                const float u = token_weight<T, C, D>(a, it, m, key, top == -INFINITY ? 0.f : top) * inv;
                                const C * vr = token_at<C, D>(a, it, a.v, key) + c;
#pragma unroll
                                for (int k = 0; k < 32; ++k) v[k] += u * static_cast<float>(vr[k]);
                            }
                    }
                    if (!whole) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4) pc[(c + k) / 4 * ROWS] = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                    } else if (wide) {
                        constexpr int W = SPLIT ? 8 : 16;
#pragma unroll
                        for (int k = 0; k < 32; k += W) {
                            uint32_t y[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                if constexpr (SPLIT) y[e] = __float_as_uint(v[k + e]);
                                else y[e] = pack<C>(v[k + 2 * e], v[k + 2 * e + 1]);
                            }
                            store32(dst + c + k, y);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; k += 4) {
                            if constexpr (SPLIT) *reinterpret_cast<float4 *>(dst + c + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                            else *reinterpret_cast<uint2 *>(dst + c + k) = make_uint2(pack<C>(v[k], v[k + 1]), pack<C>(v[k + 2], v[k + 3]));
                        }
                    }
                }
                if (live && (two || wg == 0)) {
                    if (whole) {
                        if (a.lse) put_lse(a, it, m, top, sum);
                    } else {
                        float * st = piece(a, blockIdx.x, it.t0 == 0) + ROWS * D + m;
                        st[0] = top;
                        st[ROWS] = sum;
                    }
                }
            }
            fence_before_sync();
            named_sync(1, 256);
            if (!whole) {
                if (tid == 0) S.is_last = arrive_piece(a, S.sh.d, it);
                named_sync(1, 256);
                if (S.is_last) join<T, C, ROWS, D, 256, 8, 2>(a, S.sh.d, it, tid);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.segs.empty[sn % SegmentRing::N]);
        }
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    // after an abort, whoever raised it, the copies still under way land before the block's shared memory goes
    if (S.abort_flag) {
        if (warp == 8)
            for (int k = max(issued - L::STAGES, 0); k < issued; ++k) mbar_drain(&S.full[k % L::STAGES], (k / L::STAGES) & 1);
        if (warp == 10 && issued > 0) mbar_drain(&S.q_full, (issued - 1) & 1);
    }
    if (warp == 9) {
        fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

template <class T, class C, int D>
void many(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, const CUtensorMap & q, int64_t rows, int sms, cudaStream_t stream) {
    const auto go = [&](auto kernel, int smem) {
        allow_smem(kernel, smem);
        NAVI_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(sms)), dim3(384), static_cast<size_t>(smem), stream, a, k, v, q));
    };
    if constexpr (!std::is_same_v<T, float>)
        if (rows > 128) return go(k_attend_many<T, C, D, 256>, ManySmem<T, D, 256>::BYTES);
    go(k_attend_many<T, C, D, 128>, ManySmem<T, D, 128>::BYTES);
}

} // namespace

void attend_many(const AttendArgs & a, const CUtensorMap & k, const CUtensorMap & v, const CUtensorMap & q, int dtype, int cache, int64_t rows, int sms, cudaStream_t stream) {
    const bool wide = a.head_dim == 128;
    if (dtype == NAVI_F32) wide ? many<float, __half, 128>(a, k, v, q, rows, sms, stream) : many<float, __half, 64>(a, k, v, q, rows, sms, stream);
    else if (cache == NAVI_F16) wide ? many<__half, __half, 128>(a, k, v, q, rows, sms, stream) : many<__half, __half, 64>(a, k, v, q, rows, sms, stream);
    else wide ? many<__nv_bfloat16, __nv_bfloat16, 128>(a, k, v, q, rows, sms, stream) : many<__nv_bfloat16, __nv_bfloat16, 64>(a, k, v, q, rows, sms, stream);
}

} // namespace navi::attn
