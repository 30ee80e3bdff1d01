// The paged KV cache: its pools and block tables, and the operators that plan a step, store its
// rows and commit the accepted branch of a drafted tree (include/navi_b200.h). The attention
// over the pages is in paged_attn.cu.
#include "pages.hpp"
#include "device.cuh"

#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cstring>
#include <string>
#include <type_traits>
#include <utility>

namespace navi {

CUtensorMap swizzled_map(const void * base, int dtype, int rank, const cuuint64_t * dims, const cuuint64_t * strides, const cuuint32_t * box) {
    // the driver entry point is looked up at run time, so the library loads without libcuda
    static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    if (!encode) {
        cudaDriverEntryPointQueryResult q{};
        void * fn = nullptr;
        NAVI_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess || !fn) fail("pages: cuTensorMapEncodeTiled unavailable", NAVI_E_CUDA);
        encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
    CUtensorMap m{};
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = encode(&m, dtype == NAVI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, static_cast<cuuint32_t>(rank),
                              const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fail("pages: cuTensorMapEncodeTiled failed (" + std::to_string(static_cast<int>(r)) + ")", NAVI_E_CUDA);
    return m;
}

namespace {

using namespace navi::dev;

// ---- plan ------------------------------------------------------------------------------------

struct PlanArgs {
    navi_step s;
    int32_t * table, * held, * free_pages, * n_free;
    int * ticket, * broken;
    int n_pages, shift, max_blocks, max_requests;
};
struct PlanLimited : PlanArgs {
    int positions;   // no row may be at this position or past it
};

constexpr int PLAN_THREADS = 256;

// Exclusive sum of one value per thread over the block, and the total; `red` holds a word per warp.
template <class T> __device__ __forceinline__ T block_scan(T v, T * red, T & total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) red[warp] = x;
    __syncthreads();
    T base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 32; ++w) {
        if (w < warp) base += red[w];
        total += red[w];
    }
    __syncthreads();
    return base + x - v;
}

// The last i with a[i] <= e, for a[0] = 0 <= e and a[] not decreasing.
__device__ __forceinline__ int owner(const int * a, int n, int e) {
    int lo = 0, hi = n;   // a[lo] <= e < a[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= e) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One launch. The step is a handful of sums over the requests and then independent items: rows,
// pages taken, pages given back. Every block does the sums over all requests itself (12 bytes a
// request, from L2 after the first block) and keeps them in shared memory, which costs less
// than a second launch or a wait between blocks; then the blocks share the items out. What the
// sums read (held, n_free) is written by the block that finishes last, so no block can see it
// half done: an arrival counter, no wait. A page that is taken from above the old stack top is
// one that this very call gives back; it is read where it still stands, in its owner's table
// row, whose entries past the need nobody writes. What bounds it is a chain of trips to L2: one for the
// inputs (asked for together, the parents of the block's rows with them), one for the pages, one to count
// the blocks. A plan and the plan that undoes it, launched in a row: 9 to 11 us for four single rows, 12 for 64
// trees of up to 61 rows (899 in all), 18 for a thousand prompts (218,522 rows).
// Args: PlanArgs, or PlanLimited for a talker's step.
template <class Args> __global__ void __launch_bounds__(PLAN_THREADS) k_pages_plan(const __grid_constant__ Args a) {
    constexpr bool LIMIT = std::is_same_v<Args, PlanLimited>;
    extern __shared__ int plan_smem[];
    __shared__ long long red64[PLAN_THREADS / 32];
    __shared__ int par[2 * PLAN_THREADS];
    __shared__ int last_block, taken_s;
    griddep_wait();
    griddep_launch_dependents();
    const int B = a.s.n_req, tid = threadIdx.x, MB = a.max_blocks;
    int * cu = plan_smem, * cg = cu + B + 1, * cs = cg + B, * st = cs + B;

    const int per = (B + PLAN_THREADS - 1) / PLAN_THREADS, i0 = min(B, tid * per), i1 = min(B, i0 + per);
    const long long cap = a.s.max_rows;
    // what is read of the thread's first four requests (all of them, up to 1024), and the parents of the block's first
    // rows and of as many before them, is asked for at once
    constexpr int R = 4;
    int n_r[R], ctx_r[R], tr_r[R], held_r[R], par1[2] = {-1, -1};
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int i = i0 + k;
        n_r[k] = i < i1 ? a.s.n_new[i] : 0;
        ctx_r[k] = i < i1 ? a.s.ctx_len[i] : 0;
        tr_r[k] = i < i1 ? a.s.req ? a.s.req[i] : i : -1;
    }
    const int block_row = blockIdx.x * PLAN_THREADS;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int r = block_row - PLAN_THREADS + k * PLAN_THREADS + tid;
        if (a.s.parent && r >= 0 && r < a.s.max_rows) par1[k] = a.s.parent[r];
    }
    const int F = min(max(*a.n_free, 0), a.n_pages);
#pragma unroll
    for (int k = 0; k < R; ++k) held_r[k] = tr_r[k] >= 0 && tr_r[k] < a.max_requests ? a.held[tr_r[k]] : -1;
    if (tid == 0) taken_s = 0;
    int top;
    {
        long long rows = 0, total;
#pragma unroll
        for (int k = 0; k < R; ++k) rows += max(n_r[k], 0);
        for (int i = i0 + R; i < i1; ++i) rows += max(a.s.n_new[i], 0);
        long long row = block_scan(rows, red64, total);
        if (tid == 0) cu[B] = static_cast<int>(min(total, cap));
        long long grow = 0, surplus = 0;
        const auto past = [&](int n, int ctx) {   // a chain's last row
            if constexpr (LIMIT) return !a.s.parent && n > 0 && ctx > a.positions - n;
            return false;
        };
        const auto sort = [&](int i, int n, int ctx, int tr, int held) {
            cu[i] = static_cast<int>(min(row, cap));
            row += max(n, 0);
            int status = NAVI_OK, g = 0, u = 0;
            const long long need = (static_cast<long long>(max(ctx, 0)) + max(n, 0) + (1 << a.shift) - 1) >> a.shift;
            if (n < 0 || ctx < 0 || tr < 0 || tr >= a.max_requests || held < 0 || held > MB) status = NAVI_E_ARG;
            else if (n > a.s.max_new || need > MB || row > cap || past(n, ctx)) status = NAVI_E_SHAPE;
            else {
                g = max(static_cast<int>(need) - held, 0);
                u = max(held - static_cast<int>(need), 0);
            }
            cg[i] = g;
            cs[i] = u;
            st[i] = status;
            grow += g;
            surplus += u;
        };
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (i0 + k < i1) sort(i0 + k, n_r[k], ctx_r[k], tr_r[k], held_r[k]);
        for (int i = i0 + R; i < i1; ++i) {
            const int tr = a.s.req ? a.s.req[i] : i;
            sort(i, a.s.n_new[i], a.s.ctx_len[i], tr, tr >= 0 && tr < a.max_requests ? a.held[tr] : -1);
        }
        long long all_grow, all_surplus, g = block_scan(grow, red64, all_grow), u = block_scan(surplus, red64, all_surplus);
        top = static_cast<int>(min(F + all_surplus, static_cast<long long>(a.n_pages)));
        int taken = 0;
        for (int i = i0; i < i1; ++i) {
            const int gi = cg[i], ui = cs[i];
            cg[i] = static_cast<int>(min(g, static_cast<long long>(INT_MAX)));
            cs[i] = static_cast<int>(min(u, static_cast<long long>(INT_MAX)));
            g += gi;
            u += ui;
            if (gi > 0) {
                if (g <= top) taken = static_cast<int>(g);
                else st[i] = NAVI_E_KV_FULL;
            }
        }
        if (taken > 0) atomicMax(&taken_s, taken);
    }
    __syncthreads();
    const int taken = taken_s, all_surplus = top - F;

    const auto need_of = [&](int i) { return (a.s.ctx_len[i] + max(a.s.n_new[i], 0) + (1 << a.shift) - 1) >> a.shift; };
    const auto table_row = [&](int i) { return a.table + static_cast<size_t>(a.s.req ? a.s.req[i] : i) * MB; };
    // the e-th page that is given back
    const auto given = [&](int e) {
        const int i = owner(cs, B, e);
        return table_row(i)[need_of(i) + e - cs[i]];
    };
    // the e-th page that is taken
    const auto taken_page = [&](int e) {
        const int at = top - 1 - e;
        return at < F ? a.free_pages[at] : given(top - 1 - at);
    };
    const int nb = gridDim.x, step = nb * PLAN_THREADS, first = blockIdx.x * PLAN_THREADS + tid;
    for (int e = first; e < all_surplus; e += step) {
        const int at = top - 1 - e;
        if (at >= F) a.free_pages[at] = given(e);
    }
    for (int e = first; e < taken; e += step) {
        const int i = owner(cg, B, e);
        table_row(i)[a.held[a.s.req ? a.s.req[i] : i] + e - cg[i]] = taken_page(e);
    }
    if (blockIdx.x == 0)
        for (int i = tid; i <= B; i += PLAN_THREADS) a.s.cu_rows[i] = cu[i];

    const int n_rows = cu[B];
    for (int r0 = blockIdx.x * PLAN_THREADS; r0 < n_rows; r0 += step) {
        const int r = r0 + tid;
        const int base = r0 - PLAN_THREADS;
        if (a.s.parent) {   // the parents of these rows, and of the 256 before them: a tree's first row is among those
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int at = base + k * PLAN_THREADS + tid;
                par[k * PLAN_THREADS + tid] = r0 == block_row ? par1[k] : at >= 0 && at < n_rows ? a.s.parent[at] : -1;
            }
            __syncthreads();
        }
        if (r >= n_rows) continue;
        const int i = owner(cu, B, r), j = r - cu[i], ctx = a.s.ctx_len[i];
        int depth = j;
        bool whole = true;
        if (a.s.parent) {
            const int at0 = cu[i] - base;              // the request's first row among the staged ones; below 0: too many rows, refused
            whole = at0 >= 0;
            int at = whole ? j : -1;
            depth = -1;
            if (a.s.mask_words == 1) {                 // the usual tree: one word
                uint64_t m = 0;
                while (at >= 0) {
                    ++depth;
                    m |= 1ull << (at & 63);
                    const int up = par[at0 + at];
                    whole = up >= -1 && up < at;
                    at = whole ? up : -1;
                }
                a.s.mask[r] = whole ? m : 0;
            } else {
                uint64_t m[NAVI_STEP_MAX_TREE / 64] = {};
                while (at >= 0) {
                    ++depth;
#pragma unroll
                    for (int w = 0; w < NAVI_STEP_MAX_TREE / 64; ++w)
                        if ((at >> 6) == w) m[w] |= 1ull << (at & 63);
                    const int up = par[at0 + at];
                    whole = up >= -1 && up < at;
                    at = whole ? up : -1;
                }
                for (int w = 0; w < a.s.mask_words; ++w) {
                    uint64_t v = 0;
#pragma unroll
                    for (int x = 0; x < NAVI_STEP_MAX_TREE / 64; ++x)
                        if (x == w) v = m[x];
                    a.s.mask[static_cast<size_t>(r) * a.s.mask_words + w] = whole ? v : 0;
                }
            }
        }
        int64_t slot = -1;
        if (st[i] == NAVI_OK && whole) {
            const int held = a.held[a.s.req ? a.s.req[i] : i], blk = (ctx + j) >> a.shift;
            const int page = blk < held ? table_row(i)[blk] : taken_page(cg[i] + blk - held);
            if (page >= 0 && page < a.n_pages) slot = (static_cast<int64_t>(page) << a.shift) + ((ctx + j) & ((1 << a.shift) - 1));
        }
        if constexpr (LIMIT) {
            if (a.s.parent && (!whole || ctx + depth >= a.positions)) atomicMax(a.broken + i, whole ? 1 : 2);
        } else {
            if (!whole) a.broken[i] = 2;
        }
        a.s.row_req[r] = i;
        a.s.pos[r] = ctx + depth;
        a.s.slot[r] = slot;
    }

    if (nb > 1) {
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            last_block = atomicAdd(a.ticket, 1) == nb - 1;
            __threadfence();
        }
        __syncthreads();
        if (!last_block) return;
    } else {
        __syncthreads();
    }
    for (int i = tid; i < B; i += PLAN_THREADS) {
        int status = st[i];
        if (status == NAVI_OK) a.held[a.s.req ? a.s.req[i] : i] = need_of(i);
        if (a.s.parent) {
            if (const int why = __ldcg(a.broken + i); why) {   // 2: a parent, 1: a position
                a.broken[i] = 0;
                if (status == NAVI_OK) status = LIMIT && why == 1 ? NAVI_E_SHAPE : NAVI_E_ARG;
            }
        }
        a.s.status[i] = status;
    }
    if (tid == 0) {
        *a.n_free = top - taken;
        *a.ticket = 0;
    }
}

// ---- store -----------------------------------------------------------------------------------

struct StoreArgs {
    const void * qkv;
    void * q_out;
    int64_t in_stride, out_stride;
    const int32_t * cu_rows, * pos;
    const int64_t * slot;
    const float * q_norm, * k_norm, * rope;
    uint8_t * k, * v;
    float eps;
    int n_req, max_rows, n_head, n_kv, shift, n_pages, rope_positions, parts;
};

// 8 bytes of T as pairs of floats (one pair of f32, two of 16-bit values), and back
template <class T> __device__ __forceinline__ void load8(const T * p, float2 * v) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    if constexpr (std::is_same_v<T, float>) {
        v[0] = make_float2(__uint_as_float(x.x), __uint_as_float(x.y));
    } else if constexpr (std::is_same_v<T, __half>) {
        v[0] = __half22float2(*reinterpret_cast<const __half2 *>(&x.x));
        v[1] = __half22float2(*reinterpret_cast<const __half2 *>(&x.y));
    } else {
        v[0] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&x.x));
        v[1] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&x.y));
    }
}
template <class T> __device__ __forceinline__ uint32_t pack2(float2 v) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __float22half2_rn(v);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __float22bfloat162_rn(v);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <class T, int N> __device__ __forceinline__ void store_pairs(T * p, const float2 * v) {
    if constexpr (std::is_same_v<T, float>) *reinterpret_cast<float2 *>(p) = v[0];
    else if constexpr (N == 1) *reinterpret_cast<uint32_t *>(p) = pack2<T>(v[0]);
    else *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(v[0]), pack2<T>(v[1]));
}

// A warp takes a share (1 / parts) of one row's heads. A lane holds 8 bytes of a head's first half and the
// 8 bytes that RoPE pairs them with in the second, so a head is D * sizeof(T) / 16 lanes, a warp reads 512
// bytes at a time and the rotation needs no exchange between lanes; only the sum of squares does. With the
// norm's weights in the coefficients, fixed for the row,
//   y0 = s (x0 (w0 c) - x1 (w1 sin)),  y1 = s (x0 (w0 sin) + x1 (w1 c)),  s = rsqrt(mean x^2 + eps).
// 11,722 bf16 rows of 16 + 8 + 8 heads: 44 us, 4.4 TB/s of reads and writes, 67 % of the measured copy
// rate. With a lane's 16 bytes in one half and the partner by shuffles it took 46.9, and 58.4
// before four loads were under way together. Loads ahead (2, 4, 8) and shares of a row to a warp were swept at
// this size: 44 to 59 us, four loads and whole rows the best.
template <class T, class C, int D> __global__ void __launch_bounds__(128) k_pages_store(const __grid_constant__ StoreArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int N = 4 / sizeof(T), LANES = D / (4 * N), HPW = 32 / LANES;   // pairs of floats in 8 bytes, lanes a head, heads a warp
    const int w = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    const int r = w / a.parts, part = w % a.parts;
    if (r >= a.max_rows) return;
    const int e0 = lane % LANES * (2 * N), H = a.n_head, total = H + 2 * a.n_kv;
    // the first heads are asked for before what the row's place and position lead to
    constexpr int U = 4;   // heads of a lane whose loads are under way together
    const int stride = a.parts * HPW, first = part * HPW + lane / LANES;
    const T * in = static_cast<const T *>(a.qkv) + r * a.in_stride + e0;
    float2 x0[U][N], x1[U][N];
    const auto load = [&](int h0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * stride;
            const T * src = in + static_cast<size_t>(h < total ? h : 0) * D;
            load8<T>(src, x0[u]);
            load8<T>(src + D / 2, x1[u]);
        }
    };
    load(first);
    const int64_t slot = a.slot[r];
    const int pos = a.pos[r];
    if (r >= a.cu_rows[a.n_req]) return;
    const bool known = !a.rope || (pos >= 0 && pos < a.rope_positions);
    T * qo = static_cast<T *>(a.q_out) + r * a.out_stride + e0;
    const int64_t page = slot >> a.shift, off = slot & ((1 << a.shift) - 1);
    const bool stored = slot >= 0 && page < a.n_pages && known;
    const size_t at = ((static_cast<size_t>(page) * a.n_kv << a.shift) + off) * D + e0;   // head 0 of the token
    C * k = reinterpret_cast<C *>(a.k) + at, * v = reinterpret_cast<C *>(a.v) + at;
    // [q or k][x0 -> y0, x1 -> y0, x0 -> y1, x1 -> y1]
    float2 co[2][4][N];
#pragma unroll
    for (int x = 0; x < N; ++x) {
        float2 c = make_float2(1.f, 1.f), s = make_float2(0.f, 0.f);
        if (a.rope && known) {
            const float * row = a.rope + static_cast<size_t>(pos) * D + e0 + 2 * x;
            c = make_float2(row[0], row[1]);
            s = make_float2(row[D / 2], row[D / 2 + 1]);
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const float * nw = g ? a.k_norm : a.q_norm;
            float2 w0 = make_float2(1.f, 1.f), w1 = w0;
            if (nw) {
                nw += e0 + 2 * x;
                w0 = make_float2(nw[0], nw[1]);
                w1 = make_float2(nw[D / 2], nw[D / 2 + 1]);
            }
            co[g][0][x] = __fmul2_rn(w0, c);
            co[g][1][x] = __fmul2_rn(w1, make_float2(-s.x, -s.y));
            co[g][2][x] = __fmul2_rn(w0, s);
            co[g][3][x] = __fmul2_rn(w1, c);
        }
    }
    for (int h0 = first; h0 - lane / LANES < total; h0 += U * stride) {
        if (h0 != first) load(h0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * stride;
            if (h - lane / LANES >= total) break;   // the same for the whole warp
            const bool is_q = h < H, is_v = h >= H + a.n_kv;
            float2 y0[N], y1[N];
            if (!__all_sync(0xffffffffu, is_v)) {
                float scale = 1.f;
                if (a.q_norm || a.k_norm) {
                    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
                    for (int x = 0; x < N; ++x) ss = __ffma2_rn(x0[u][x], x0[u][x], __ffma2_rn(x1[u][x], x1[u][x], ss));
                    float sum = ss.x + ss.y;
#pragma unroll
                    for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (is_q ? a.q_norm : a.k_norm) scale = rsqrtf(sum * (1.f / D) + a.eps);
                }
                const float2 s2 = make_float2(scale, scale);
#pragma unroll
                for (int x = 0; x < N; ++x) {
                    float2 m[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) m[y] = is_q ? co[0][y][x] : co[1][y][x];
                    y0[x] = __fmul2_rn(s2, __ffma2_rn(x0[u][x], m[0], __fmul2_rn(x1[u][x], m[1])));
                    y1[x] = __fmul2_rn(s2, __ffma2_rn(x0[u][x], m[2], __fmul2_rn(x1[u][x], m[3])));
                }
            }
            if (h >= total) continue;
            if (is_q) {
                if (!known) {
#pragma unroll
                    for (int x = 0; x < N; ++x) y0[x] = y1[x] = make_float2(0.f, 0.f);
                }
                T * dst = qo + static_cast<size_t>(h) * D;
                store_pairs<T, N>(dst, y0);
                store_pairs<T, N>(dst + D / 2, y1);
            } else if (stored) {
                C * dst = (is_v ? v : k) + (static_cast<size_t>(h - H - (is_v ? a.n_kv : 0)) << a.shift) * D;
                store_pairs<C, N>(dst, is_v ? x0[u] : y0);
                store_pairs<C, N>(dst + D / 2, is_v ? x1[u] : y1);
            }
        }
    }
}

// ---- commit ----------------------------------------------------------------------------------

struct CommitArgs {
    navi_step s;
    navi_commit_args c;
    uint8_t * k[NAVI_PAGES_MAX_LAYERS], * v[NAVI_PAGES_MAX_LAYERS];
    int * walked;                       // IN_PLACE: the blocks of a request that have walked
    int n_layer, n_kv, shift, chunks;   // chunks: 16-byte pieces of one head's row
    int n_pages;
};

constexpr int COMMIT_THREADS = 256;

// Block (i, z) walks request i's tree (every z the same walk: a few hundred ids from L2) and moves
// its share of the layers. The walk: each row looks whether its ids are the model's choice at its
// parent, the lowest such child of each node is kept, and one thread follows them from the root.
// The k-th accepted row is row path[k] >= k, so a thread that owns 16 bytes of a token's row and
// goes through the path in order never writes a place that a later step still has to read. Bound by the walk's
// trips to L2 (parents, ids, choices, slots) and then by the moves: four trees 7 us, as long as a launch;
// 64 trees through 28 layers 10.6 to 12.4 us, 3.3 to 3.9 TB/s. 16 bytes at a time with four moves ahead took
// it from 29 to 17.0 us, twice the blocks (8 for 4 times the multiprocessors) to 11.5; 16 times takes 12.1.
// IN_PLACE: next_token is root_target.
template <bool IN_PLACE> __global__ void __launch_bounds__(COMMIT_THREADS) k_pages_commit(const __grid_constant__ CommitArgs a) {
    __shared__ int child[NAVI_STEP_MAX_TREE + 1];
    __shared__ int path[NAVI_STEP_MAX_TREE];
    __shared__ int64_t from[NAVI_STEP_MAX_TREE], to[NAVI_STEP_MAX_TREE];
    __shared__ int count, moved;
    griddep_wait();
    griddep_launch_dependents();
    const int i = blockIdx.x, tid = threadIdx.x, W = a.c.width;
    const int r0 = a.s.cu_rows[i], n = min(a.s.cu_rows[i + 1] - r0, NAVI_STEP_MAX_TREE);
    const bool served = a.s.status[i] == NAVI_OK;
    for (int j = tid; j <= n; j += COMMIT_THREADS) child[j] = INT_MAX;
    __syncthreads();
    // 4 lanes compare a row's ids, 16 bytes at a time where they are that
    const bool vec = W % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.c.tokens) | reinterpret_cast<uintptr_t>(a.c.targets) | reinterpret_cast<uintptr_t>(a.c.root_target)) & 15) == 0;
    for (int x = tid; x < (n + COMMIT_THREADS / 4 - 1) / (COMMIT_THREADS / 4) * COMMIT_THREADS; x += COMMIT_THREADS) {
        const int j = x >> 2, part = x & 3;
        const int up = served && j < n ? a.s.parent[r0 + j] : -2;
        bool same = up >= -1 && up < j;
        if (same) {
            const int32_t * want = up >= 0 ? a.c.targets + static_cast<size_t>(r0 + up) * W : a.c.root_target + static_cast<size_t>(i) * W;
            const int32_t * have = a.c.tokens + static_cast<size_t>(r0 + j) * W;
            if (vec) {
                for (int y = part * 4; y < W; y += 16) {
                    const int4 p = *reinterpret_cast<const int4 *>(want + y), q = *reinterpret_cast<const int4 *>(have + y);
                    same = same && p.x == q.x && p.y == q.y && p.z == q.z && p.w == q.w;
                }
            } else {
                for (int y = part; y < W; y += 4) same = same && want[y] == have[y];
            }
        }
        const unsigned all = __ballot_sync(0xffffffffu, same);
        if (part == 0 && (all >> (tid & 31) & 15) == 15) atomicMin(&child[up + 1], j);
    }
    __syncthreads();
    if (tid == 0) {
        int at = 0, k = 0, m = -1;
        while (child[at] != INT_MAX) {
            const int j = child[at];
            if (j != k && m < 0) m = k;
            path[k++] = j;
            at = j + 1;
        }
        count = k;
        moved = m < 0 ? k : m;   // the first of the path that is not in its place
    }
    __syncthreads();
    const int k0 = moved, k1 = count;
    const int32_t * nx = k1 > 0 ? a.c.targets + static_cast<size_t>(r0 + path[k1 - 1]) * W : a.c.root_target + static_cast<size_t>(i) * W;
    int32_t * next = a.c.next_token + static_cast<size_t>(i) * W;
    if (IN_PLACE && tid >= COMMIT_THREADS - 32) {   // over the ids that the other blocks compare: by the last of them, when all have
        const int lane = tid & 31;
        int last = 0;
        if (lane == 0) {
            __threadfence();
            last = atomicAdd(a.walked + i, 1) == static_cast<int>(gridDim.y) - 1;
            if (last) a.walked[i] = 0;
        }
        if (__shfl_sync(0xffffffffu, last, 0))
            for (int x = lane; x < W; x += 32) next[x] = nx[x];
    }
    if (blockIdx.y == 0) {
        for (int j = tid; j < n; j += COMMIT_THREADS) a.c.path[r0 + j] = j < k1 ? path[j] : -1;
        if (n == NAVI_STEP_MAX_TREE)   // more rows are not served
            for (int j = r0 + n + tid; j < a.s.cu_rows[i + 1]; j += COMMIT_THREADS) a.c.path[j] = -1;
        if constexpr (!IN_PLACE)
            for (int x = tid; x < W; x += COMMIT_THREADS) next[x] = nx[x];
        if (tid == 0) {
            a.c.accepted[i] = k1;
            a.c.new_len[i] = a.s.ctx_len[i] + k1;
        }
    }
    if (k0 >= k1) return;
    // places of the moved rows: byte offset of head 0 in units of 16 bytes
    for (int k = k0 + tid; k < k1; k += COMMIT_THREADS) {
        const auto place = [&](int64_t slot) {
            const int64_t page = slot >> a.shift, off = slot & ((1 << a.shift) - 1);
            return slot >= 0 && page < a.n_pages ? ((page * a.n_kv << a.shift) + off) * a.chunks : -1;
        };
        from[k] = place(a.s.slot[r0 + path[k]]);
        to[k] = place(a.s.slot[r0 + k]);
    }
    __syncthreads();
    const int per = a.n_kv * a.chunks, items = a.n_layer * 2 * per;
    for (int x = blockIdx.y * COMMIT_THREADS + tid; x < items; x += gridDim.y * COMMIT_THREADS) {
        const int l = x / (2 * per), y = x % (2 * per), kv = y / per, z = y % per, h = z / a.chunks, c = z % a.chunks;
        uint4 * pool = reinterpret_cast<uint4 *>(kv ? a.v[l] : a.k[l]) + (static_cast<size_t>(h) << a.shift) * a.chunks + c;
        // places are written behind the ones that are read, so four reads go ahead of their writes
        for (int k = k0; k < k1; k += 4) {
            uint4 v[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
                if (k + y < k1 && from[k + y] >= 0) v[y] = pool[from[k + y]];
#pragma unroll
            for (int y = 0; y < 4; ++y)
                if (k + y < k1 && from[k + y] >= 0 && to[k + y] >= 0) pool[to[k + y]] = v[y];
        }
    }
}

// A pool as rows of head_dim values; a box is a page of one head: 64 dims of it, or all, half after half.
CUtensorMap pool_map(void * pool, const navi_pages_desc & d, bool whole) {
    const cuuint64_t rows = static_cast<cuuint64_t>(d.n_pages) * d.n_kv_head * d.page_size, halves = static_cast<cuuint64_t>(d.head_dim) / 64;
    const cuuint64_t row = static_cast<cuuint64_t>(d.head_dim) * 2;
    if (whole) {
        const cuuint64_t dims[3] = {64, rows, halves}, strides[2] = {row, 128};
        const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(d.page_size), static_cast<cuuint32_t>(halves)};
        return swizzled_map(pool, d.dtype, 3, dims, strides, box);
    }
    const cuuint64_t dims[2] = {64 * halves, rows}, strides[1] = {row};
    const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(d.page_size)};
    return swizzled_map(pool, d.dtype, 2, dims, strides, box);
}

bool overlap(const void * a, size_t na, const void * b, size_t nb) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return na > 0 && nb > 0 && x < y + nb && y < x + na;
}

bool aligned16(const void * p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

} // namespace

// ---- host side -------------------------------------------------------------------------------

std::unique_ptr<Pages> Pages::create(const Device & dev, const navi_pages_desc & d) {
    if (d.n_layer < 1 || d.n_layer > NAVI_PAGES_MAX_LAYERS) fail("pages: n_layer outside 1..NAVI_PAGES_MAX_LAYERS", NAVI_E_ARG);
    if (d.page_size != 16 && d.page_size != 32 && d.page_size != 64 && d.page_size != 128) fail("pages: page_size must be 16, 32, 64 or 128", NAVI_E_ARG);
    if (d.head_dim != 64 && d.head_dim != 128) fail("pages: the kernels are built for head_dim 64 and 128", NAVI_E_SHAPE);
    if (d.dtype != NAVI_F16 && d.dtype != NAVI_BF16) fail("pages: the cache is NAVI_F16 or NAVI_BF16", NAVI_E_ARG);
    if (d.n_kv_head < 1 || d.n_pages < 1 || d.max_blocks < 1) fail("pages: n_kv_head, n_pages and max_blocks must be positive", NAVI_E_ARG);
    if (d.max_requests < 1 || d.max_requests > NAVI_PAGES_MAX_REQUESTS) fail("pages: max_requests outside 1..NAVI_PAGES_MAX_REQUESTS", NAVI_E_ARG);
    // rows of all heads and pages are counted in 31 bits (tensor-map coordinates), a table row's tokens too
    if (static_cast<int64_t>(d.n_pages) * d.n_kv_head * d.page_size > INT32_MAX) fail("pages: n_pages * n_kv_head * page_size passes 31 bits", NAVI_E_SHAPE);
    if (static_cast<int64_t>(d.max_blocks) * d.page_size > INT32_MAX / 2) fail("pages: max_blocks * page_size passes 30 bits", NAVI_E_SHAPE);
    if (!d.k != !d.v) fail("pages: k and v are both given or both NULL", NAVI_E_ARG);
    const int given = !!d.table + !!d.held + !!d.free_pages + !!d.n_free;
    if (given != 0 && given != 4) fail("pages: table, held, free_pages and n_free are all given or all NULL", NAVI_E_ARG);
    if (d.k)
        for (int l = 0; l < d.n_layer; ++l)
            if (!aligned16(d.k[l]) || !aligned16(d.v[l])) fail("pages: a layer's pool is not 16-byte aligned", NAVI_E_ARG);
    std::unique_ptr<Pages> p(new Pages());
    dev.make_current();
    p->dev_ = &dev;
    p->d_ = d;
    while ((1 << p->shift_) < d.page_size) ++p->shift_;
    const auto take = [&](size_t bytes) {
        void * m = nullptr;
        NAVI_CUDA(cudaMalloc(&m, bytes));
        p->owned_.push_back(m);
        NAVI_CUDA(cudaMemset(m, 0, bytes));
        return m;
    };
    if (d.k) {
        p->k_.assign(d.k, d.k + d.n_layer);
        p->v_.assign(d.v, d.v + d.n_layer);
    } else {
        const size_t bytes = static_cast<size_t>(d.n_pages) * d.n_kv_head * d.page_size * d.head_dim * 2;
        for (int l = 0; l < d.n_layer; ++l) {
            p->k_.push_back(take(bytes));
            p->v_.push_back(take(bytes));
        }
    }
    p->d_.k = p->k_.data();
    p->d_.v = p->v_.data();
    for (int l = 0; l < d.n_layer; ++l)
        for (void * pool : {p->k_[static_cast<size_t>(l)], p->v_[static_cast<size_t>(l)]}) {
            p->maps_.push_back(pool ? pool_map(pool, d, false) : CUtensorMap{});
            p->page_maps_.push_back(pool ? pool_map(pool, d, true) : CUtensorMap{});
        }
    if (!given) {
        std::vector<int32_t> ids(static_cast<size_t>(d.n_pages));
        for (int i = 0; i < d.n_pages; ++i) ids[static_cast<size_t>(i)] = d.n_pages - 1 - i;
        p->d_.table = static_cast<int32_t *>(take(static_cast<size_t>(d.max_requests) * d.max_blocks * 4));
        p->d_.held = static_cast<int32_t *>(take(static_cast<size_t>(d.max_requests) * 4));
        p->d_.free_pages = static_cast<int32_t *>(take(ids.size() * 4));
        p->d_.n_free = static_cast<int32_t *>(take(4));
        NAVI_CUDA(cudaMemcpy(p->d_.free_pages, ids.data(), ids.size() * 4, cudaMemcpyHostToDevice));
        NAVI_CUDA(cudaMemcpy(p->d_.n_free, &d.n_pages, 4, cudaMemcpyHostToDevice));
    }
    // the zeros are written on the legacy stream, for which other streams (the engine's) do not wait
    if (!p->owned_.empty()) NAVI_CUDA(cudaStreamSynchronize(cudaStreamLegacy));
    return p;
}

Pages::~Pages() {
    if (!owned_.empty()) cudaSetDevice(dev_->info().ordinal);
    for (void * m : owned_) cudaFree(m);
}

void Pages::check_step(const navi_step & s, const char * who) const {
    const auto refuse = [&](const char * why, int status) { fail(std::string(who) + why, status); };
    if (s.n_req < 0 || s.n_req > d_.max_requests) refuse(": n_req outside 0..max_requests", NAVI_E_ARG);
    if (s.max_rows < 0 || s.max_new < 0) refuse(": max_rows and max_new must not be negative", NAVI_E_ARG);
    if (s.n_req == 0) return;
    if (!s.ctx_len || !s.n_new || !s.cu_rows || !s.status) refuse(": ctx_len, n_new, cu_rows and status are needed", NAVI_E_ARG);
    if (s.max_rows > 0 && (!s.row_req || !s.pos || !s.slot)) refuse(": row_req, pos and slot are needed", NAVI_E_ARG);
    if (s.parent) {
        if (s.max_new > NAVI_STEP_MAX_TREE) refuse(": a tree has at most NAVI_STEP_MAX_TREE rows", NAVI_E_SHAPE);
        if (s.mask_words < 0 || s.mask_words > NAVI_STEP_MAX_TREE / 64 || 64 * s.mask_words < s.max_new || (s.mask_words > 0 && !s.mask))
            refuse(": mask of 64 * mask_words >= max_new bits is needed with parent", NAVI_E_ARG);
    }
}

void Pages::check_layer(int layer, const char * who) const {
    if (layer < 0 || layer >= d_.n_layer) fail(std::string(who) + ": layer outside the cache", NAVI_E_ARG);
    if (!k_[static_cast<size_t>(layer)] || !v_[static_cast<size_t>(layer)]) fail(std::string(who) + ": the layer has no pool", NAVI_E_ARG);
}

void Pages::plan(const navi_step & s, cudaStream_t stream, int positions) const {
    check_step(s, "pages plan");
    if (s.n_req == 0) return;
    NAVI_CUDA(cudaSetDevice(dev_->info().ordinal));
    const int sms = dev_->info().multiprocessors;
    const PagesScratch sc(dev_->scratch(stream, PagesScratch::bytes(sms)), sms);
    PlanArgs a{s, d_.table, d_.held, d_.free_pages, d_.n_free, sc.ticket, sc.broken, d_.n_pages, shift_, d_.max_blocks, d_.max_requests};
    const size_t smem = (4 * static_cast<size_t>(s.n_req) + 1) * sizeof(int);
    static_assert((4 * static_cast<size_t>(NAVI_PAGES_MAX_REQUESTS) + 1) * sizeof(int) < 200 * 1024);
    const int blocks = std::clamp((s.max_rows + PLAN_THREADS - 1) / PLAN_THREADS, 1, 2 * sms);
    const auto go = [&](auto kernel, const auto & args) {
        if (smem > 40 * 1024)
            NAVI_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>((4 * NAVI_PAGES_MAX_REQUESTS + 1) * sizeof(int))));
        NAVI_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(PLAN_THREADS), smem, stream, args));
    };
    if (positions == INT_MAX) go(k_pages_plan<PlanArgs>, a);
    else go(k_pages_plan<PlanLimited>, PlanLimited{a, positions});
}

void Pages::store(const navi_step & s, int layer, const navi_store_args & q, cudaStream_t stream) const {
    check_step(s, "pages store");
    check_layer(layer, "pages store");
    if (q.n_head < 0 || q.n_head > 4096) fail("pages store: n_head outside 0..4096", NAVI_E_ARG);
    if (!(q.dtype == d_.dtype || (q.dtype == NAVI_F32 && d_.dtype == NAVI_F16))) fail("pages store: rows are of the cache's type, or NAVI_F32 for an f16 cache", NAVI_E_ARG);
    if (q.rope && q.rope_positions < 1) fail("pages store: rope_positions must be positive", NAVI_E_ARG);
    if (s.n_req == 0 || s.max_rows == 0) return;
    const int D = d_.head_dim, heads = q.n_head + 2 * d_.n_kv_head;
    const int64_t elt = q.dtype == NAVI_F32 ? 4 : 2, in = q.qkv_stride ? q.qkv_stride : static_cast<int64_t>(heads) * D,
                  out = q.q_out_stride ? q.q_out_stride : static_cast<int64_t>(q.n_head) * D;
    if (!q.qkv || (q.n_head > 0 && !q.q_out)) fail("pages store: NULL rows", NAVI_E_ARG);
    if (in < static_cast<int64_t>(heads) * D || out < static_cast<int64_t>(q.n_head) * D) fail("pages store: a row stride is shorter than the row", NAVI_E_ARG);
    if (!aligned16(q.qkv) || !aligned16(q.q_out) || in * elt % 16 || out * elt % 16) fail("pages store: rows must be 16-byte aligned", NAVI_E_ARG);
    // q over its own rows, or between them; any other overlap would write rows that are still to be read
    const bool same_rows = q.q_out == q.qkv && (in == out || s.max_rows == 1);
    if (q.n_head > 0 && !same_rows &&
        overlap(q.qkv, static_cast<size_t>((s.max_rows - 1) * in + static_cast<int64_t>(heads) * D) * elt, q.q_out,
                static_cast<size_t>((s.max_rows - 1) * out + static_cast<int64_t>(q.n_head) * D) * elt)) {
        const int64_t apart = (reinterpret_cast<intptr_t>(q.q_out) - reinterpret_cast<intptr_t>(q.qkv)) / elt, at = (apart % in + in) % in;
        if (in != out || at < static_cast<int64_t>(heads) * D || at + static_cast<int64_t>(q.n_head) * D > in)
            fail("pages store: q_out overlaps qkv otherwise than row for row (q_out_stride of rows in place is theirs)", NAVI_E_ARG);
    }
    NAVI_CUDA(cudaSetDevice(dev_->info().ordinal));
    StoreArgs a{q.qkv, q.q_out, in, out, s.cu_rows, s.pos, s.slot, q.q_norm, q.k_norm, q.rope, static_cast<uint8_t *>(k_[static_cast<size_t>(layer)]),
                static_cast<uint8_t *>(v_[static_cast<size_t>(layer)]), q.eps, s.n_req, s.max_rows, q.n_head, d_.n_kv_head, shift_, d_.n_pages, q.rope_positions, 1};
    // few rows: a row's heads go to several warps, down to one pass of a warp each
    const int per_warp = static_cast<int>(512 / (D * elt)), passes = (heads + per_warp - 1) / per_warp;
    while (a.parts * 2 <= passes && static_cast<int64_t>(s.max_rows) * a.parts < 16 * 4 * dev_->info().multiprocessors) a.parts *= 2;
    const int64_t warps = static_cast<int64_t>(s.max_rows) * a.parts;
    if (warps > INT32_MAX / 32) fail("pages store: too many rows", NAVI_E_SHAPE);
    const unsigned blocks = static_cast<unsigned>((warps + 3) / 4);
    const auto go = [&](auto kernel) { NAVI_CUDA(launch_pdl(kernel, dim3(blocks), dim3(128), 0, stream, a)); };
    if (q.dtype == NAVI_F32) D == 128 ? go(k_pages_store<float, __half, 128>) : go(k_pages_store<float, __half, 64>);
    else if (q.dtype == NAVI_F16) D == 128 ? go(k_pages_store<__half, __half, 128>) : go(k_pages_store<__half, __half, 64>);
    else D == 128 ? go(k_pages_store<__nv_bfloat16, __nv_bfloat16, 128>) : go(k_pages_store<__nv_bfloat16, __nv_bfloat16, 64>);
}

void Pages::commit(const navi_step & s, const navi_commit_args & c, cudaStream_t stream) const {
    check_step(s, "pages commit");
    if (c.width < 1) fail("pages commit: width must be positive", NAVI_E_ARG);
    if (s.n_req == 0) return;
    if (!s.parent) fail("pages commit: the step has no parent (there is no tree to walk)", NAVI_E_ARG);
    for (int l = 0; l < d_.n_layer; ++l) check_layer(l, "pages commit");
    if (!c.root_target || !c.accepted || !c.new_len || !c.next_token) fail("pages commit: NULL argument", NAVI_E_ARG);
    if (s.max_rows > 0 && (!c.tokens || !c.targets || !c.path)) fail("pages commit: NULL argument", NAVI_E_ARG);
    // Blocks of a request read its ids while another of them writes the outcome
    const size_t ids = static_cast<size_t>(s.max_rows) * c.width, reqs = static_cast<size_t>(s.n_req);
    const std::pair<const int32_t *, size_t> in[] = {{c.tokens, ids}, {c.targets, ids}, {c.root_target, reqs * c.width}},
                                             out[] = {{c.next_token, reqs * c.width}, {c.accepted, reqs}, {c.path, static_cast<size_t>(s.max_rows)}, {c.new_len, reqs}};
    const bool in_place = c.next_token == c.root_target;
    for (const auto & o : out)
        for (const auto & i : in)
            if (overlap(o.first, o.second * 4, i.first, i.second * 4) && !(in_place && o.first == c.next_token && i.first == c.root_target))
                fail("pages commit: the outcome overlaps the ids (next_token may be root_target)", NAVI_E_ARG);
    NAVI_CUDA(cudaSetDevice(dev_->info().ordinal));
    CommitArgs a{};
    if (in_place) a.walked = PagesScratch(dev_->scratch(stream, PagesScratch::bytes(dev_->info().multiprocessors)), dev_->info().multiprocessors).broken;
    a.s = s;
    a.c = c;
    for (int l = 0; l < d_.n_layer; ++l) {
        a.k[l] = static_cast<uint8_t *>(k_[static_cast<size_t>(l)]);
        a.v[l] = static_cast<uint8_t *>(v_[static_cast<size_t>(l)]);
    }
    a.n_layer = d_.n_layer;
    a.n_kv = d_.n_kv_head;
    a.shift = shift_;
    a.chunks = d_.head_dim / 8;
    a.n_pages = d_.n_pages;
    const int64_t items = static_cast<int64_t>(d_.n_layer) * 2 * d_.n_kv_head * a.chunks;
    if (items > INT32_MAX / 2) fail("pages commit: too many heads", NAVI_E_SHAPE);
    const int most = static_cast<int>((items + COMMIT_THREADS - 1) / COMMIT_THREADS);
    const int z = std::clamp(8 * dev_->info().multiprocessors / s.n_req, 1, std::min(most, 65535));
    NAVI_CUDA(launch_pdl(in_place ? k_pages_commit<true> : k_pages_commit<false>, dim3(static_cast<unsigned>(s.n_req), static_cast<unsigned>(z)), dim3(COMMIT_THREADS),
                         0, stream, a));
}

void Pages::check(cudaStream_t stream) const {
    NAVI_CUDA(cudaSetDevice(dev_->info().ordinal));
    const int sms = dev_->info().multiprocessors;
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    NAVI_CUDA(cudaStreamIsCapturing(stream, &capturing));
    if (capturing != cudaStreamCaptureStatusNone) fail("pages check: the stream is being captured", NAVI_E_ARG);
    std::vector<void *> blocks = dev_->captured_scratch();
    blocks.push_back(dev_->scratch(stream, PagesScratch::bytes(sms)));
    std::vector<int> err(blocks.size(), 0);
    for (size_t k = 0; k < blocks.size(); ++k)
        NAVI_CUDA(cudaMemcpyAsync(&err[k], PagesScratch(blocks[k], sms).err, sizeof(int), cudaMemcpyDeviceToHost, stream));
    NAVI_CUDA(cudaStreamSynchronize(stream));
    if (std::all_of(err.begin(), err.end(), [](int e) { return e == 0; })) return;
    NAVI_CUDA(cudaDeviceSynchronize());
    for (size_t k = 0; k < blocks.size(); ++k)   // counters of blocks that gave up
        if (err[k]) NAVI_CUDA(cudaMemsetAsync(PagesScratch(blocks[k], sms).ticket, 0, PagesScratch::ints(sms) * sizeof(int), stream));
    NAVI_CUDA(cudaStreamSynchronize(stream));
    fail("pages: a wait for a copy or a matrix product passed its deadline", NAVI_E_TIMEOUT);
}

} // namespace navi
