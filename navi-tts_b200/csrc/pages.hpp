// navi::Pages: the paged KV cache shared by many requests, and the four operators of a step
// (include/navi_b200.h, "paged KV cache and drafted trees"). No counterpart in the reference,
// whose cache is one contiguous block per stream (model/qwen3tts/talker.h:20-24).
#pragma once

#include "../../include/navi_b200.h"
#include "runtime.hpp"

#include <cuda.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <memory>
#include <vector>

namespace navi {

// A tensor map of 16-bit values (dtype NAVI_F16 or NAVI_BF16) whose boxes land in 128-byte swizzled
// rows of shared memory; values outside the tensor read as zero.
CUtensorMap swizzled_map(const void * base, int dtype, int rank, const cuuint64_t * dims, const cuuint64_t * strides, const cuuint32_t * box);

class Pages {
public:
    static std::unique_ptr<Pages> create(const Device & dev, const navi_pages_desc & d);
    ~Pages();
    Pages(const Pages &) = delete;

    const navi_pages_desc & desc() const { return d_; }
    // A request with a row at `positions` or past it is not served (NAVI_E_SHAPE).
    void plan(const navi_step & s, cudaStream_t stream, int positions = INT_MAX) const;
    void store(const navi_step & s, int layer, const navi_store_args & a, cudaStream_t stream) const;
    void attend(const navi_step & s, int layer, const navi_attend_args & a, cudaStream_t stream) const;
    void commit(const navi_step & s, const navi_commit_args & a, cudaStream_t stream) const;
    // Waits for the stream; throws NAVI_E_TIMEOUT when a kernel on it, or of a graph, gave up a wait since the last check.
    void check(cudaStream_t stream) const;

private:
    Pages() = default;
    // Throws NAVI_E_ARG / NAVI_E_SHAPE for a step that no call can take.
    void check_step(const navi_step & s, const char * who) const;
    // Throws NAVI_E_ARG for a layer that the cache has not, or has no pool of.
    void check_layer(int layer, const char * who) const;

    const Device * dev_ = nullptr;
    navi_pages_desc d_{};
    std::vector<void *> k_, v_;     // d_.k and d_.v point here
    std::vector<CUtensorMap> maps_, page_maps_;   // K, V of each layer: boxes of a page of one head, 64 dims or all
    std::vector<void *> owned_;
    int shift_ = 0;                 // log2(page_size)
};

// A block of scratch (Device::scratch), laid out for every operator that hands work from
// one block to another. All counters are zero between launches.
struct PagesScratch {
    static constexpr size_t PIECE_FLOATS = 256 * (128 + 2);          // attend: one block's unfinished item
    int * ticket, * broken, * arrived, * err;                        // ticket: plan, blocks that have finished; broken: plan, requests whose tree is refused; commit, blocks
    float * pieces;                                                  // two a block

    // `blocks`: the most blocks of a launch that leave pieces (one a multiprocessor)
    static size_t ints(int blocks) { return (1 + NAVI_PAGES_MAX_REQUESTS + static_cast<size_t>(blocks) + 1 + 63) / 64 * 64; }
    static size_t bytes(int blocks) { return ints(blocks) * sizeof(int) + 2 * static_cast<size_t>(blocks) * PIECE_FLOATS * sizeof(float); }
    PagesScratch(void * p, int blocks)
        : ticket(static_cast<int *>(p)), broken(ticket + 1), arrived(broken + NAVI_PAGES_MAX_REQUESTS), err(arrived + blocks),
          pieces(reinterpret_cast<float *>(ticket + ints(blocks))) {}
};

} // namespace navi
