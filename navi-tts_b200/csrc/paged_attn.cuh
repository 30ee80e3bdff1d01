// What the attention kernels over the paged KV cache share (paged_attn.cu has the mathematics):
// the launch's arguments, how the blocks divide ragged requests between them, how the pieces of
// an item are joined, and how a tile of pages is brought to shared memory.
#pragma once

#include "device.cuh"
#include "pages.hpp"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace navi::attn {

using namespace navi::dev;

struct AttendArgs {
    const void * q;
    void * out;
    float * lse;
    const int32_t * table, * req, * ctx_len, * cu_rows, * status;
    const uint64_t * mask;       // nullptr: a chain
    float * pieces;              // the stream's scratch: unfinished sums, arrival counters, error word
    int * arrived, * err;
    int64_t q_stride, out_stride;
    float scale;                 // times log2(e)
    int n_req, max_rows, mask_words, n_head, n_kv, group, group_shift, head_dim, shift, n_pages, max_blocks, max_requests;
};

// What a block needs to know of one request.
struct Request {
    int row0, n, ctx, keys;      // first row, rows, cached tokens, tokens in all
    int table;                   // its row of the block table
};
__device__ __forceinline__ Request request(const AttendArgs & a, int i) {
    Request r;
    r.row0 = a.cu_rows[i];
    r.n = max(min(a.cu_rows[i + 1], a.max_rows) - r.row0, 0);
    r.ctx = a.ctx_len[i];
    r.table = a.req ? a.req[i] : i;
    const bool ok = a.status[i] == NAVI_OK && r.table >= 0 && r.table < a.max_requests && r.ctx >= 0 &&
                    static_cast<long long>(r.ctx) + r.n <= (static_cast<long long>(a.max_blocks) << a.shift);
    r.keys = ok ? r.ctx + r.n : 0;
    r.table = ok ? r.table : 0;
    return r;
}
// The requests from the block's first one on, in shared memory: a walk over items then costs no
// trip to L2 for each.
struct Window {
    static constexpr int N = 32;
    long long base;              // the first unit of request `first`
    int first, count;
    int row0[N], n[N], ctx[N], keys[N], table[N];
};
__device__ __forceinline__ Request request(const AttendArgs & a, const Window & w, int i) {
    const int k = i - w.first;
    if (k >= w.count) return request(a, i);
    return {w.row0[k], w.n[k], w.ctx[k], w.keys[k], w.table[k]};
}
__device__ __forceinline__ int by_group(const AttendArgs & a, int x) { return a.group_shift >= 0 ? x >> a.group_shift : x / a.group; }

template <class C> __device__ __forceinline__ uint32_t pack(float a, float b) {
    if constexpr (std::is_same_v<C, __half>) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <class C> __device__ __forceinline__ float2 unpack(uint32_t v) {
    if constexpr (std::is_same_v<C, __half>) return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
}
// 2^x by the hardware's approximation (two units of the last place); 2^-inf = 0
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- who does what ----------------------------------------------------------------------------
//
// The work of a launch is a list of units: for each request, each KV head and each tile of ROWS
// rows (rows x heads of the KV head, an item), the item's key tiles of KT keys, at least one.
// Lengths are on the device and ragged, so the blocks divide the list evenly themselves: block c
// of G takes the units [c W / G, (c + 1) W / G), whatever request they belong to. An item that
// falls to several blocks leaves its pieces (the sums and each row's maximum and sum, f32) in
// the stream's scratch, and the block that arrives last joins them in the blocks' order, so
// the result does not depend on who was last. A block has at most two such pieces: slot 0 for
// one that begins inside an item, slot 1 for one that only ends inside it.

constexpr int KT = 128;

// x / y of values that are not negative: the 64-bit division is the slow one
__device__ __forceinline__ long long cut(long long x, long long y) {
    return (x | y) >> 32 ? x / y : static_cast<long long>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y));
}

// This block's units [u, end) of total, and the item that holds the first.
struct Share {
    long long u, end, total;
    int blocks, i;               // blocks that have work; the request of unit u
    long long base;              // the request's first unit
};

struct Item {
    int i, g, rt;                // request, KV head, row tile
    int tiles, n_keys;           // key tiles (1 at least) and keys that its rows may see
    int m0, m;                   // its first row x head, and how many
    long long u0;                // its first unit
    Request rq;
};

template <int ROWS> __device__ __forceinline__ int row_tiles(const AttendArgs & a, const Request & r) { return (r.n * a.group + ROWS - 1) / ROWS; }
template <int ROWS> __device__ __forceinline__ int keys_of(const AttendArgs & a, const Request & r, int rt) {
    if (a.mask || r.keys == 0) return r.keys;
    return r.ctx + min(by_group(a, (rt + 1) * ROWS - 1) + 1, r.n);
}
__device__ __forceinline__ int tiles_of(int n_keys) { return max((n_keys + KT - 1) / KT, 1); }
// the units of one KV head of a request
template <int ROWS> __device__ __forceinline__ long long units_of(const AttendArgs & a, const Request & r) {
    const int rts = row_tiles<ROWS>(a, r);
    if (a.mask || r.keys == 0) return static_cast<long long>(rts) * tiles_of(r.keys);
    long long n = 0;
    for (int rt = 0; rt < rts; ++rt) n += tiles_of(keys_of<ROWS>(a, r, rt));
    return n;
}
template <int ROWS> __device__ __forceinline__ void open_tile(const AttendArgs & a, Item & it) {
    it.n_keys = keys_of<ROWS>(a, it.rq, it.rt);
    it.tiles = tiles_of(it.n_keys);
    it.m0 = it.rt * ROWS;
    it.m = min(it.rq.n * a.group - it.m0, ROWS);
}
template <int ROWS> __device__ __forceinline__ void next_item(const AttendArgs & a, const Window & win, Item & it) {
    it.u0 += it.tiles;
    if (++it.rt >= row_tiles<ROWS>(a, it.rq)) {
        it.rt = 0;
        if (++it.g >= a.n_kv) {
            it.g = 0;
            do it.rq = request(a, win, ++it.i);
            while (it.rq.n <= 0);   // more units follow, so a later request has rows
        }
    }
    open_tile<ROWS>(a, it);
}

// Every thread of the block takes part. It holds the block's only barriers before the roles part, so
// what the block's threads write to shared memory before the call is there for all after it.
// Up to 32 requests every warp does the sums by itself, a lane a request: one trip to L2 and no
// barrier between.
template <int ROWS, int THREADS> __device__ __forceinline__ void share_out(const AttendArgs & a, Window & win, Share & out, long long * red) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.n_req;
    const bool one = B <= 32;
    const int per = one ? 1 : (B + THREADS - 1) / THREADS, i0 = min(B, one ? lane : tid * per), i1 = min(B, i0 + per);
    long long mine = 0;
    Request r{};
    for (int i = i0; i < i1; ++i) {
        r = request(a, i);
        mine += units_of<ROWS>(a, r) * a.n_kv;
    }
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    long long base = x - mine, total = __shfl_sync(0xffffffffu, x, 31);
    if (!one) {
        if (lane == 31) red[warp] = x;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) base += red[w];
            total += red[w];
        }
    }
    Share sh;
    const long long G = min(static_cast<long long>(gridDim.x), total), c = blockIdx.x;
    sh.total = total;
    sh.blocks = static_cast<int>(G);
    sh.u = G ? cut(c * total, G) : 0;
    sh.end = c < G ? cut((c + 1) * total, G) : sh.u;
    const bool holds = c < G && sh.u >= base && sh.u < base + mine;
    if (one) {
        const int from = __ffs(__ballot_sync(0xffffffffu, holds)) - 1;
        sh.i = max(from, 0);
        sh.base = __shfl_sync(0xffffffffu, base, sh.i);
        if (warp == 0 && lane < B) {
            win.row0[lane] = r.row0;
            win.n[lane] = r.n;
            win.ctx[lane] = r.ctx;
            win.keys[lane] = r.keys;
            win.table[lane] = r.table;
        }
        if (tid == 0) {
            win.first = 0;
            win.count = B;
        }
    } else {
        if (holds) {
            int i = i0;
            long long b = base;
            for (;; ++i) {
                const long long n = units_of<ROWS>(a, request(a, i)) * a.n_kv;
                if (sh.u < b + n) break;
                b += n;
            }
            win.first = i;
            win.base = b;
        }
        __syncthreads();
        sh.i = win.first;
        sh.base = win.base;
        if (sh.u < sh.end && tid < Window::N) {
            const int count = min(Window::N, B - sh.i);
            if (tid < count) {
                const Request q = request(a, sh.i + tid);
                win.row0[tid] = q.row0;
                win.n[tid] = q.n;
                win.ctx[tid] = q.ctx;
                win.keys[tid] = q.keys;
                win.table[tid] = q.table;
            }
            if (tid == 0) win.count = count;
        }
    }
    if (tid == 0) out = sh;
    __syncthreads();
}
template <int ROWS> __device__ __forceinline__ Item first_item(const AttendArgs & a, const Window & win, const Share & sh) {
    Item it{};
    it.i = sh.i;
    it.rq = request(a, win, it.i);
    const long long per_head = units_of<ROWS>(a, it.rq);
    it.g = static_cast<int>(cut(sh.u - sh.base, per_head));
    it.u0 = sh.base + it.g * per_head;
    if (a.mask || it.rq.keys == 0) {   // every row tile has as many key tiles
        it.rt = static_cast<int>(cut(sh.u - it.u0, tiles_of(it.rq.keys)));
        it.u0 += static_cast<long long>(it.rt) * tiles_of(it.rq.keys);
    }
    open_tile<ROWS>(a, it);
    while (it.u0 + it.tiles <= sh.u) {
        it.u0 += it.tiles;
        ++it.rt;
        open_tile<ROWS>(a, it);
    }
    return it;
}
__device__ __forceinline__ int block_of(const Share & sh, long long unit) { return static_cast<int>(cut((unit + 1) * sh.blocks - 1, sh.total)); }

// A piece in the scratch: the rows' sums as float4 [D / 4][ROWS], then [ROWS] maxima and [ROWS] sums of weights.
__device__ __forceinline__ float * piece(const AttendArgs & a, int block, int slot) {
    return a.pieces + (static_cast<size_t>(block) * 2 + slot) * PagesScratch::PIECE_FLOATS;
}

// Row m of an item: where its q and its result are.
template <class T> __device__ __forceinline__ T * row_at(const AttendArgs & a, const void * base, int64_t stride, const Item & it, int m) {
    const int at = it.m0 + m, j = by_group(a, at);
    return static_cast<T *>(const_cast<void *>(base)) + (it.rq.row0 + j) * stride + static_cast<int64_t>(it.g * a.group + at - j * a.group) * a.head_dim;
}
__device__ __forceinline__ float * lse_at(const AttendArgs & a, const Item & it, int m) {
    const int at = it.m0 + m, j = by_group(a, at);
    return a.lse + static_cast<size_t>(it.rq.row0 + j) * a.n_head + it.g * a.group + at - j * a.group;
}
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f; }

// One thread of a block whose piece is written: whether it is the item's last.
__device__ __forceinline__ bool arrive_piece(const AttendArgs & a, const Share & sh, const Item & it) {
    const int c0 = block_of(sh, it.u0), c1 = block_of(sh, it.u0 + it.tiles - 1);
    if (atomicAdd(a.arrived + c0, 1) != c1 - c0) return false;
    a.arrived[c0] = 0;
    __threadfence();
    return true;
}

// Joins the pieces of an item, in order: THREADS threads of the block, all of them. First what each
// piece counts in each row goes to `weight` (CAP floats of shared memory), LANES lanes to a row,
// then the sums are read.
template <class T, class C, int ROWS, int D, int THREADS, int LANES, int CAP>
__device__ __forceinline__ void join(const AttendArgs & a, const Share & sh, const Item & it, int tid, float * weight) {
    const int c0 = block_of(sh, it.u0), np = block_of(sh, it.u0 + it.tiles - 1) - c0 + 1;
    const auto part = [&](int p) { return piece(a, c0 + p, p == 0); };
    const int most = CAP / np;                        // rows at a time: up to 256 blocks share an item
    for (int m0 = 0; m0 < it.m; m0 += most) {
        const int rows = min(most, it.m - m0), sub = tid % LANES;
        for (int r = tid / LANES; r < (rows + THREADS / LANES - 1) / (THREADS / LANES) * (THREADS / LANES); r += THREADS / LANES) {
            const bool live = r < rows;
            const int m = m0 + (live ? r : 0);
            float top = -INFINITY, l = 0.f;
#pragma unroll 4
            for (int p = sub; p < np; p += LANES) top = fmaxf(top, __ldcg(part(p) + ROWS * D + m));
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
            for (int p = sub; p < np; p += LANES) {
                const float w = exp2_fast(__ldcg(part(p) + ROWS * D + m) - ref);
                l += w * __ldcg(part(p) + ROWS * D + ROWS + m);
                if (live) weight[p * rows + r] = w;
            }
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            if (live)
                for (int p = sub; p < np; p += LANES) weight[p * rows + r] *= inv;
            if (live && sub == 0 && a.lse) *lse_at(a, it, m) = lse_of(top, l);
        }
        named_sync(1, THREADS);
        // a thread stays with its row: neighbours read neighbouring rows, the weights come without conflicts
        constexpr int QS = THREADS / ROWS > 0 ? THREADS / ROWS : 1, N = D / 4 / QS, U = N < 8 ? N : 8;
        static_assert(THREADS >= ROWS && N % U == 0);
        const int r = tid % ROWS, q0 = tid / ROWS;
        if (r < rows) {
            T * dst = row_at<T>(a, a.out, a.out_stride, it, m0 + r);
            for (int q = q0; q < D / 4; q += U * QS) {
                float4 s[U];
#pragma unroll
                for (int k = 0; k < U; ++k) s[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
                for (int p = 0; p < np; ++p) {
                    const float4 * src = reinterpret_cast<const float4 *>(part(p)) + m0 + r;
                    const float w = weight[p * rows + r];
                    float4 v[U];
#pragma unroll
                    for (int k = 0; k < U; ++k) v[k] = __ldcg(src + (q + k * QS) * ROWS);
#pragma unroll
                    for (int k = 0; k < U; ++k) {
                        s[k].x += w * v[k].x; s[k].y += w * v[k].y; s[k].z += w * v[k].z; s[k].w += w * v[k].w;
                    }
                }
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if constexpr (std::is_same_v<T, float>) *reinterpret_cast<float4 *>(dst + 4 * (q + k * QS)) = s[k];
                    else *reinterpret_cast<uint2 *>(dst + 4 * (q + k * QS)) = make_uint2(pack<C>(s[k].x, s[k].y), pack<C>(s[k].z, s[k].w));
                }
            }
        }
        named_sync(1, THREADS);
    }
}

// 32 bytes to global memory in one store: a whole sector
__device__ __forceinline__ void store32(void * p, const uint32_t * v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}

// ---- waits --------------------------------------------------------------------------------------
// Every wait for a copy or an MMA is bounded: past the deadline the block raises its abort flag and
// the scratch's error word (navi_pages_check), and every role leaves its loops.

constexpr unsigned long long DEADLINE_NS = 2000000000ull;

struct Wait {
    volatile int * abort;
    int * err;
    __device__ __forceinline__ bool operator()(uint64_t * bar, uint32_t parity) const {
        for (int k = 0; k < 64; ++k)
            if (mbar_try_wait(bar, parity)) return true;
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(bar, parity)) {
            if (*abort) return false;
            if (globaltimer() - t0 > DEADLINE_NS) {
                *abort = 1;
                atomicExch(err, 1);
                return false;
            }
        }
        return true;
    }
};

// The same wait for copies that nothing stops any more, after an abort.
__device__ __forceinline__ void mbar_drain(uint64_t * bar, uint32_t parity) {
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(bar, parity) && globaltimer() - t0 < 2 * DEADLINE_NS) {}
}

// Whether row j of the item's request sees token `key`.
__device__ __forceinline__ bool sees(const AttendArgs & a, const Item & it, int key, int j) {
    if (key >= it.n_keys) return false;
    const int at = key - it.rq.ctx;
    if (at < 0) return true;
    if (!a.mask) return at <= j;
    return at < 64 * a.mask_words && (__ldg(a.mask + static_cast<size_t>(it.rq.row0 + j) * a.mask_words + (at >> 6)) >> (at & 63) & 1);
}

// The pages that hold key tile t of an item, and the bytes of them that one pool contributes.
__device__ __forceinline__ int tile_pages(const AttendArgs & a, const Item & it, int t) {
    return (min(it.n_keys - t * KT, KT) + (1 << a.shift) - 1) >> a.shift;
}
// A warp brings them from a pool's map to dst: halves of 64 dims, each [KT][64] in 128-byte rows that
// the copy swizzles; only pages with keys of the item, so rows past them keep what they held.
// The bytes (tile_pages * page * D * 2) arrive on `bar`. Lane x has the x-th box of the tile, at
// most 16 of them (a page of 16 tokens, two halves), so the page ids, which it reads a tile ahead,
// cost one latency together and not one each.
template <int D> __device__ __forceinline__ int page_of_box(const AttendArgs & a, const Item & it, int t, int box) {
    const int p = box / (D / 64);
    return p < tile_pages(a, it, t) ? min(max(__ldg(a.table + static_cast<size_t>(it.rq.table) * a.max_blocks + (t * KT >> a.shift) + p), 0), a.n_pages - 1) : -1;
}
template <int D> __device__ __forceinline__ void load_box(const AttendArgs & a, const CUtensorMap * map, const Item & it, int page, int box, uint8_t * dst, uint64_t * bar) {
    const int p = box / (D / 64), h = box % (D / 64);
    if (page >= 0) tma_box_2d(dst + h * (KT * 128) + (p << a.shift) * 128, map, h * 64, (page * a.n_kv + it.g) << a.shift, bar);
}

} // namespace navi::attn
