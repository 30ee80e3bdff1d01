// navi::Pages: the paged KV cache shared by many requests, and the four operators of a step
// (include/navi_b200.h, "paged KV cache and drafted trees"). No counterpart in the reference,
// whose cache is one contiguous block per stream (model/qwen3tts/talker.h:20-24).
#pragma once

#include "../../include/navi_b200.h"
#include "runtime.hpp"

#include <cuda_runtime.h>

#include <cstdint>
#include <memory>
#include <vector>

namespace navi {

class Pages {
public:
    static std::unique_ptr<Pages> create(const Device & dev, const navi_pages_desc & d);
    ~Pages();
    Pages(const Pages &) = delete;

    const navi_pages_desc & desc() const { return d_; }
    void plan(const navi_step & s, cudaStream_t stream) const;
    void store(const navi_step & s, int layer, const navi_store_args & a, cudaStream_t stream) const;
    void attend(const navi_step & s, int layer, const navi_attend_args & a, cudaStream_t stream) const;
    void commit(const navi_step & s, const navi_commit_args & a, cudaStream_t stream) const;

private:
    Pages() = default;
    // Throws NAVI_E_ARG / NAVI_E_SHAPE for a step that no call can take.
    void check_step(const navi_step & s, const char * who) const;

    const Device * dev_ = nullptr;
    navi_pages_desc d_{};
    std::vector<void *> k_, v_;     // d_.k and d_.v point here
    std::vector<void *> owned_;
    int shift_ = 0;                 // log2(page_size)
};

// The scratch of one stream (Device::scratch), laid out for every operator that hands work from
// one block to another. All counters are zero between launches.
struct PagesScratch {
    static constexpr size_t TICKETS = 64;                                   // ints: launch-wide counters
    static constexpr size_t BROKEN = NAVI_PAGES_MAX_REQUESTS;               // ints: plan, a request with a bad parent
    static constexpr size_t BYTES = (TICKETS + BROKEN) * sizeof(int);
};

} // namespace navi
