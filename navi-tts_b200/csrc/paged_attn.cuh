// What the attention kernels over the paged KV cache share (paged_attn.cu has the mathematics):
// the launch's arguments, how the blocks divide ragged requests between them, how the pieces of
// an item are joined, and how a tile of pages is brought to shared memory.
#pragma once

#include "device.cuh"
#include "pages.hpp"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>
#include <set>
#include <type_traits>
#include <utility>

namespace navi::attn {

using namespace navi::dev;

// The kernels may be resident while plan and store still write what they read, before griddep_wait: no
// load here is of the kind that takes its data for constant over the kernel's life (ld.global.nc, __ldg).

struct AttendArgs {
    const void * q;
    void * out;
    float * lse;
    const uint8_t * k, * v;      // the layer's pools, for what does not come by TMA
    const int32_t * table, * req, * ctx_len, * cu_rows, * status;
    const uint64_t * mask;       // nullptr: a chain
    float * pieces;              // the stream's or graph's scratch: unfinished sums, arrival counters, error word
    int * arrived, * err;
    int64_t q_stride, out_stride;
    float scale;                 // times log2(e)
    uint32_t group_mul;          // 2^32 / group rounded up, 0 for 1
    // q_boxes: q comes as boxes of a tensor map (16-bit rows, group a power of two up to 128)
    int n_req, max_rows, mask_words, n_head, n_kv, group, q_boxes, head_dim, shift, n_pages, max_blocks, max_requests;
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
// A row x head of a request -> its row: x / group as a product, exact below 2^32 / group (the host checks).
__device__ __forceinline__ int by_group(const AttendArgs & a, int x) {
    return a.group_mul ? static_cast<int>(__umulhi(static_cast<uint32_t>(x), a.group_mul)) : x;
}

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
// two f32 values as pairs of 16-bit terms, v = hi + lo to about twice the bits
template <class C> __device__ __forceinline__ void split_pair(float x, float y, uint32_t & hi, uint32_t & lo) {
    hi = pack<C>(x, y);
    const float2 b = unpack<C>(hi);
    lo = pack<C>(x - b.x, y - b.y);
}
// A row of f32 q is brought to magnitudes of up to 2^15 by a power of two before the split, and its scores back by the
// inverse in their scale: f16 would take values from 65520 on as infinity and keep few bits of small ones.
// From the row's largest magnitude: the exponent field of that power, 2^(field - 127), 14..253 (127 if it is not finite).
__device__ __forceinline__ uint32_t row_field(float largest) {
    const uint32_t e = __float_as_uint(largest) >> 23;
    return e == 255 ? 127 : min(268 - e, 253u);
}
__device__ __forceinline__ float row_up(uint32_t field) { return __uint_as_float(field << 23); }
// The scale of such a row's scores. It stays above 0 and finite, as a score of -inf or 0 times it has to stay what it is.
__device__ __forceinline__ float row_scale(float scale, uint32_t field) {
    return fminf(fmaxf(scale * __uint_as_float((254 - field) << 23), 1.17549435e-38f), 3.40282347e38f);
}
__device__ __forceinline__ float largest4(float4 v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }
// The largest over N neighbouring lanes (N a power of two, lanes from a multiple of N on).
template <int N> __device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
    for (int o = 1; o < N; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
// 2^x by the hardware's approximation (two units of the last place); 2^-inf = 0
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The weights of a softmax enter the product with V as values of the cache's type. bf16 has f32's range; f16 would lose
// what is 2^-25 of the largest weight, whose sum over a long tail of keys counts (and which the sum of the
// weights, in f32, has). So with f16 the largest weight is 2^LIFT and not 1: the reference that scores are taken
// against is LIFT lower, in log2, which cancels in the division, in the join of pieces and in the log of the sum.
// Rounded up, the reference is never below max scale - LIFT, so that no weight passes 2^LIFT however large the scores.
__device__ __forceinline__ float reference(float best, float scale, float lift) { return __fmaf_ru(best, scale, -lift); }

// Lets a kernel have `bytes` of dynamic shared memory, asking the runtime once a kernel and device.
template <class... A> void allow_smem(void (*kernel)(A...), int bytes) {
    static std::mutex lock;
    static std::set<std::pair<int, const void *>> done;
    int dev = 0;
    NAVI_CUDA(cudaGetDevice(&dev));
    const std::lock_guard<std::mutex> hold(lock);
    const void * k = reinterpret_cast<const void *>(kernel);
    if (done.count({dev, k})) return;
    NAVI_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.insert({dev, k});
}

// ---- who does what ----------------------------------------------------------------------------
//
// The work of a launch is a list of units: for each request, each KV head and each tile of ROWS
// rows (rows x heads of the KV head, an item), the item's key tiles of KT keys, at least one,
// after EXTRA units that stand for what an item costs beside its tiles.
// Lengths are on the device and ragged, so the blocks divide the list evenly themselves,
// whatever request the units belong to. An item that falls to several blocks leaves its pieces
// (the sums and each row's maximum and sum, f32) in the scratch, and the block that
// arrives last joins them in the blocks' order, so the result does not depend on who was last. A
// block has at most two such pieces: slot 0 for one that begins inside an item, slot 1 for one
// that begins with the item and ends inside it. Arrivals are counted in key tiles at the item's
// first block.
//
// One warp of the block walks the list and hands each part of it (a segment: the block's key tiles
// of one item) to the others through a small ring in shared memory. The walk is long code that
// runs seldom; the roles that run often stay short, which for a step of a few microseconds
// matters more than anything else: its instructions are read once, from L2.

constexpr int KT = 128;

struct Segment {
    int row0, ctx, table, g;     // the request, the KV head
    int m0, m, n_keys;           // its first row x head, how many, the keys that they may see
    int t0, nt;                  // key tiles t0 .. t0 + nt - 1; nt -1: no more segments
    int u0, tiles;               // the item's key tiles among the units
};
__device__ __forceinline__ bool is_whole(const Segment & s) { return s.nt == s.tiles; }

template <int ROWS> __device__ __forceinline__ int row_tiles(const AttendArgs & a, const Request & r) { return (r.n * a.group + ROWS - 1) / ROWS; }
template <int ROWS> __device__ __forceinline__ int keys_of(const AttendArgs & a, const Request & r, int rt) {
    if (a.mask || r.keys == 0) return r.keys;
    return r.ctx + min(by_group(a, (rt + 1) * ROWS - 1) + 1, r.n);
}
__device__ __forceinline__ int tiles_of(int n_keys) { return max((n_keys + KT - 1) / KT, 1); }
// the units of one KV head of a request
template <int ROWS, int EXTRA> __device__ __forceinline__ int units_of(const AttendArgs & a, const Request & r) {
    const int rts = row_tiles<ROWS>(a, r);
    if (a.mask || r.keys == 0) return rts * (EXTRA + tiles_of(r.keys));
    int n = rts * EXTRA;
#pragma unroll 1
    for (int rt = 0; rt < rts; ++rt) n += tiles_of(keys_of<ROWS>(a, r, rt));
    return n;
}

// x / y of x >= 0, y > 0. (x + 1/2) / y is 1 / 2y away from an integer at least, the approximate quotient
// off by 2^-21 of itself at most: exact below 2^20.
__device__ __forceinline__ int quick_div(int x, int y) {
    return x < 1 << 20 ? static_cast<int>(__fdividef(static_cast<float>(x) + 0.5f, static_cast<float>(y))) : x / y;
}

// How the units divide: `more` blocks of `per` + 1 units, then blocks of `per`.
struct Division {
    int per, more;
    __device__ __forceinline__ int first(int block) const { return block * per + min(block, more); }
    __device__ __forceinline__ int block(int unit) const {
        const int x = unit - more * (per + 1);
        return x < 0 ? quick_div(unit, per + 1) : more + quick_div(x, per);
    }
};
// The division, this block's units [u, end), and the request i that holds the first of them and begins
// at unit `base`.
struct Share {
    Division d;
    int u, end, i, base;
};

__device__ __forceinline__ int warp_scan(int x) {   // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}
__device__ __forceinline__ void take(Share & sh, int total) {
    const int G = min(static_cast<int>(gridDim.x), total), c = blockIdx.x;
    sh.d = {0, 0};
    if (G > 0) {
        sh.d.per = quick_div(total, G);
        sh.d.more = total - sh.d.per * G;
    }
    sh.u = sh.d.first(c);
    sh.end = c < G ? sh.d.first(c + 1) : sh.u;
}
// Up to 32 requests a warp finds its block's share by itself, a lane a request. (The host has checked
// that the units fit 31 bits.)
template <int ROWS, int EXTRA> __device__ __forceinline__ Share share_of_warp(const AttendArgs & a, Request & first) {
    const int lane = threadIdx.x & 31;
    Request r{};
    if (lane < a.n_req) r = request(a, lane);
    const int mine = units_of<ROWS, EXTRA>(a, r) * a.n_kv, x = warp_scan(mine);
    Share sh;
    take(sh, __shfl_sync(0xffffffffu, x, 31));
    sh.i = max(__ffs(__ballot_sync(0xffffffffu, sh.u < x)) - 1, 0);   // the first request that ends after unit u
    sh.base = __shfl_sync(0xffffffffu, x - mine, sh.i);
    first.row0 = __shfl_sync(0xffffffffu, r.row0, sh.i);
    first.n = __shfl_sync(0xffffffffu, r.n, sh.i);
    first.ctx = __shfl_sync(0xffffffffu, r.ctx, sh.i);
    first.keys = __shfl_sync(0xffffffffu, r.keys, sh.i);
    first.table = __shfl_sync(0xffffffffu, r.table, sh.i);
    return sh;
}
// More: all THREADS threads of the block, each some requests in a row. What they wrote to shared memory
// before is there for all of them after it.
template <int ROWS, int EXTRA, int THREADS> __device__ __forceinline__ void share_of_block(const AttendArgs & a, Share & out, int * red) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.n_req;
    const int per = (B + THREADS - 1) / THREADS, i0 = min(B, tid * per), i1 = min(B, i0 + per);
    int mine = 0;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) mine += units_of<ROWS, EXTRA>(a, request(a, i)) * a.n_kv;
    const int x = warp_scan(mine);
    if (lane == 31) red[warp] = x;
    __syncthreads();
    int base = x - mine, total = 0;
#pragma unroll 1
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) base += red[w];
        total += red[w];
    }
    Share sh{};
    take(sh, total);
    const int u = sh.u;
    if (tid == 0) {
        out.d = sh.d;
        out.u = u;
        out.end = sh.end;
    }
    if (u < sh.end && u >= base && u < base + mine) {
        int i = i0;
#pragma unroll 1
        for (;; ++i) {
            const int n = units_of<ROWS, EXTRA>(a, request(a, i)) * a.n_kv;
            if (u < base + n) break;
            base += n;
        }
        out.i = i;
        out.base = base;
    }
    __syncthreads();
}

// The walk over the block's segments: next() fills in the next one; false when there is none.
template <int ROWS, int EXTRA> struct Walk {
    const AttendArgs & a;
    Share sh;
    Request r;
    int i, g, rt, u0, u, tiles, n_keys;   // u0: the item's first key tile

    __device__ __forceinline__ Walk(const AttendArgs & args, const Share & share, const Request & first) : a(args), sh(share), r(first) {
        i = sh.i;
        u = sh.u;
        if (u >= sh.end) return;
        const int per_head = units_of<ROWS, EXTRA>(a, r);
        g = quick_div(u - sh.base, per_head);
        u0 = sh.base + g * per_head + EXTRA;
        rt = 0;
        if (a.mask || r.keys == 0) {   // every row tile has as many key tiles
            const int each = EXTRA + tiles_of(r.keys);
            rt = quick_div(u - u0 + EXTRA, each);
            u0 += rt * each;
        }
        open();
        while (u0 + tiles <= u) {
            u0 += tiles + EXTRA;
            ++rt;
            open();
        }
    }
    __device__ __forceinline__ void open() {
        n_keys = keys_of<ROWS>(a, r, rt);
        tiles = tiles_of(n_keys);
    }
    __device__ __forceinline__ bool next(Segment & s) {
        if (u < sh.end && u >= u0 + tiles) {
            u0 += tiles + EXTRA;
            if (++rt >= row_tiles<ROWS>(a, r)) {
                rt = 0;
                if (++g >= a.n_kv) {
                    g = 0;
                    do r = request(a, ++i);
                    while (r.n <= 0);   // more units follow, so a later request has rows
                }
            }
            open();
        }
        if (u >= sh.end || u0 >= sh.end) {   // no more, or nothing but what an item costs beside its tiles
            s.nt = -1;
            return false;
        }
        u = max(u, u0);
        const int t1 = min(tiles, sh.end - u0);
        s.row0 = r.row0;
        s.ctx = r.ctx;
        s.table = r.table;
        s.g = g;
        s.m0 = rt * ROWS;
        s.m = min(r.n * a.group - s.m0, ROWS);
        s.n_keys = n_keys;
        s.t0 = u - u0;
        s.nt = t1 - s.t0;
        s.u0 = u0;
        s.tiles = tiles;
        u += s.nt;
        return true;
    }
};

// A piece in the scratch: the rows' sums as float4 [D / 4][ROWS], then [ROWS] maxima and [ROWS] sums of weights.
__device__ __forceinline__ float * piece(const AttendArgs & a, int block, int slot) {
    return a.pieces + (static_cast<size_t>(block) * 2 + slot) * PagesScratch::PIECE_FLOATS;
}

// Row m of a segment: where its q and its result are.
template <class T> __device__ __forceinline__ T * row_at(const AttendArgs & a, const void * base, int64_t stride, const Segment & s, int m) {
    const int at = s.m0 + m, j = by_group(a, at);
    return static_cast<T *>(const_cast<void *>(base)) + (s.row0 + j) * stride + static_cast<int64_t>(s.g * a.group + at - j * a.group) * a.head_dim;
}
__device__ __forceinline__ void put_lse(const AttendArgs & a, const Segment & s, int m, float top, float l) {
    const int at = s.m0 + m, j = by_group(a, at);
    a.lse[static_cast<size_t>(s.row0 + j) * a.n_head + s.g * a.group + at - j * a.group] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
}

// One thread of a block whose piece is written (and a barrier passed since): whether it is the item's last.
__device__ __forceinline__ bool arrive_piece(const AttendArgs & a, const Division & d, const Segment & s) {
    const int c0 = s.t0 == 0 ? static_cast<int>(blockIdx.x) : d.block(s.u0);
    __threadfence();
    if (atomicAdd(a.arrived + c0, s.nt) + s.nt != s.tiles) return false;
    a.arrived[c0] = 0;
    __threadfence();
    return true;
}

// Joins the pieces of an item, in order: THREADS threads of the block. A thread has U pieces of 4 dims of
// a row (neighbours have neighbouring rows) and reads P blocks' pieces at once, their maxima and sums
// with them: one trip to L2 for each P blocks.
template <class T, class C, int ROWS, int D, int THREADS, int U, int P>
__device__ __forceinline__ void join(const AttendArgs & a, const Division & d, const Segment & s, int tid) {
    const int c0 = d.block(s.u0), np = d.block(s.u0 + s.tiles - 1) - c0 + 1;
    constexpr int N = D / 4 / U;                      // threads of a row
#pragma unroll 1
    for (int x = tid; x < ROWS * N; x += THREADS) {
        const int r = x % ROWS, q = x / ROWS;
        if (r >= s.m) continue;
        float top = -INFINITY, l = 0.f;
        float4 y[U];
#pragma unroll
        for (int k = 0; k < U; ++k) y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int p0 = 0; p0 < np; p0 += P) {
            float m[P], w[P];
            float4 v[P][U];
            float best = top;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float * at = piece(a, c0 + min(p0 + p, np - 1), p0 + p == 0);
                m[p] = __ldcg(at + ROWS * D + r);
                w[p] = __ldcg(at + ROWS * D + ROWS + r);
#pragma unroll
                for (int k = 0; k < U; ++k) v[p][k] = __ldcg(reinterpret_cast<const float4 *>(at) + (q + k * N) * ROWS + r);
            }
#pragma unroll
            for (int p = 0; p < P; ++p) best = p0 + p < np ? fmaxf(best, m[p]) : best;
            const float ref = best == -INFINITY ? 0.f : best, old = exp2_fast(top - ref);
            top = best;
            l *= old;
#pragma unroll
            for (int k = 0; k < U; ++k) { y[k].x *= old; y[k].y *= old; y[k].z *= old; y[k].w *= old; }
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const bool there = p0 + p < np;       // no branch: the loads above stay together
                const float c = there ? exp2_fast(m[p] - ref) : 0.f;
                l += c * w[p];
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const float4 z = there ? v[p][k] : make_float4(0.f, 0.f, 0.f, 0.f);
                    y[k].x += c * z.x; y[k].y += c * z.y; y[k].z += c * z.z; y[k].w += c * z.w;
                }
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T * dst = row_at<T>(a, a.out, a.out_stride, s, r);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if constexpr (std::is_same_v<T, float>) *reinterpret_cast<float4 *>(dst + 4 * (q + k * N)) = make_float4(y[k].x * inv, y[k].y * inv, y[k].z * inv, y[k].w * inv);
            else *reinterpret_cast<uint2 *>(dst + 4 * (q + k * N)) = make_uint2(pack<C>(y[k].x * inv, y[k].y * inv), pack<C>(y[k].z * inv, y[k].w * inv));
        }
        if (q == 0 && a.lse) put_lse(a, s, r, top, l);
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
        return mbar_try_wait(bar, parity) || slow(bar, parity);
    }
    __device__ __forceinline__ bool slow(uint64_t * bar, uint32_t parity) const {
#pragma unroll 1
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

// Bits 0..31: whether row j of the request sees the tokens ctx + a .. ctx + a + 31 (a may be negative:
// those are cached tokens), of which `left` are the item's.
__device__ __forceinline__ uint32_t seen_bits(const AttendArgs & a, const Segment & it, int j, int at, int left) {
    if (left <= 0) return 0u;
    uint32_t b;
    if (at + 31 < 0) b = ~0u;
    else if (!a.mask) {
        const int n = j - at + 1;            // tokens from `at` up to row j itself
        b = n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
    } else {
        const uint64_t * m = a.mask + static_cast<size_t>(it.row0 + j) * a.mask_words;
        const int w = at >> 6;               // floor: -1 for the bits before row 0, all seen
        const uint64_t lo = w < 0 ? ~0ull : w < a.mask_words ? m[w] : 0ull;
        const uint64_t hi = w + 1 < a.mask_words ? m[w + 1] : 0ull;
        const int s = at & 63;
        b = static_cast<uint32_t>(s ? (lo >> s) | (hi << (64 - s)) : lo);
    }
    return left >= 32 ? b : b & ((1u << left) - 1u);
}

// The pages that hold key tile t, and the bytes of them that one pool contributes.
__device__ __forceinline__ int tile_pages(const AttendArgs & a, const Segment & s, int t) {
    return (min(s.n_keys - t * KT, KT) + (1 << a.shift) - 1) >> a.shift;
}
// A warp brings them from a pool's map by TMA, a box a lane; only pages with keys of the item, so rows
// past them keep what they held. The bytes (tile_pages * page * D * 2) arrive on a barrier. Every lane
// reads its page's id a tile ahead, so the ids cost one latency together and not one each.
__device__ __forceinline__ int page_at(const AttendArgs & a, const Segment & s, int t, int p) {
    return p < tile_pages(a, s, t) ? min(max(a.table[static_cast<size_t>(s.table) * a.max_blocks + (t * KT >> a.shift) + p], 0), a.n_pages - 1) : -1;
}

// ---- values that are not finite where a row does not look --------------------------------------
//
// A weight of zero times a V value that is infinite or NaN is NaN, so tokens that some rows do not see
// must not enter their product. Past the last token shared memory is cleared. Among the new rows
// (a sibling in the tree, a later row of the chain) every token is some row's own: in the tiles that
// have such tokens, those whose V is not finite are looked for and cleared too, and the rows that do
// see them add them from the pool, one by one. That is seldom; the looking costs the last tiles of an item
// 16 loads a thread.

// The larger of the magnitudes so far and those of 16 bytes, as pairs of 16-bit patterns.
__device__ __forceinline__ uint32_t magnitude(uint32_t m, uint4 v) {
    m = __vmaxu2(m, v.x & 0x7fff7fffu);
    m = __vmaxu2(m, v.y & 0x7fff7fffu);
    m = __vmaxu2(m, v.z & 0x7fff7fffu);
    return __vmaxu2(m, v.w & 0x7fff7fffu);
}
template <class C> __device__ __forceinline__ bool not_finite(uint32_t m) {
    constexpr uint32_t inf = std::is_same_v<C, __half> ? 0x7c00u : 0x7f80u;
    return (m & 0xffffu) >= inf || (m >> 16) >= inf;
}
// Token `key` of the segment's request and KV head in a pool.
template <class C, int D> __device__ __forceinline__ const C * token_at(const AttendArgs & a, const Segment & s, const uint8_t * pool, int key) {
    const int page = min(max(a.table[static_cast<size_t>(s.table) * a.max_blocks + (key >> a.shift)], 0), a.n_pages - 1);
    return reinterpret_cast<const C *>(pool) + (((static_cast<size_t>(page) * a.n_kv + s.g) << a.shift) + (key & ((1 << a.shift) - 1))) * D;
}

// The weight 2^(scale q k - ref) of row m of the segment and token `key`.
template <class T, class C, int D> __device__ __forceinline__ float token_weight(const AttendArgs & a, const Segment & s, int m, int key, float ref) {
    const T * q = row_at<const T>(a, a.q, a.q_stride, s, m);
    const C * k = token_at<C, D>(a, s, a.k, key);
    float z = 0.f;
#pragma unroll 1
    for (int d = 0; d < D; ++d) z += static_cast<float>(q[d]) * static_cast<float>(k[d]);
    return exp2_fast(fmaf(z, a.scale, -ref));
}

// The ring of segments: one warp fills it, every other role reads it.
struct SegmentRing {
    static constexpr int N = 4;
    Segment s[N];
    uint64_t full[N], empty[N];
    __device__ __forceinline__ void init(int readers) {
        for (int k = 0; k < N; ++k) {
            mbar_init(&full[k], 1);
            mbar_init(&empty[k], readers);
        }
    }
};

} // namespace navi::attn
