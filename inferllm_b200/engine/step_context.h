// Building the device-side description of a step (StepContext) from the cache's plan: all index
// arrays go into one pinned staging buffer and one host-to-device copy.  Shared by the engine and by
// the sandbox in which single parts are run.
#pragma once
#include <vector>

#include "cache/cache.h"
#include "parts/parts.h"

namespace illm {

// The adapters of a step's tokens, and what is set aside for their plans (one per number of pieces of a projection).
struct StepAdapters {
    std::vector<int> index;                         // per token, -1: none
    std::vector<int> ranks;                         // per adapter
    AdapterPlanSizes sizes[kAdapterPieces];
    std::vector<int> packed_ranks(int pieces) const {
        std::vector<int> r = ranks;
        for (int& v : r) v *= pieces;
        return r;
    }
    size_t ints() const {
        size_t n = 0;
        for (const AdapterPlanSizes& s : sizes) n += (size_t)adapter_plan_layout(s).total;
        return n;
    }
};

// The common prefixes of a decode step's sequences and what is set aside for their plan.
struct StepPrefixes {
    std::vector<ops::PrefixGroup> groups;
    ops::PrefixPlanSizes sizes;
    int heads = 0;                  // query heads per kv head of the layers that use it
};

class StepContextBuilder {
public:
    StepContextBuilder(Device* dev, Runtime* rt);
    ~StepContextBuilder();
    // int32 elements of a step's buffer
    static size_t ints(int T, int B, int K, size_t n_groups, int width);
    // `into`: a device buffer of an earlier step of the same shape to fill again (the static input of
    // a captured graph); nullptr takes a fresh one from the step arena.  tables_dev gets, per paged
    // group of the cache, the device address of the step's page table [B, width].
    StepContext build(const SequenceCache& cache, const StepPlan& plan, const std::vector<int>& ids, const std::vector<int>& want_rows,
                      int* into, std::vector<const int*>* tables_dev, const StepAdapters* adapters = nullptr, const StepPrefixes* prefixes = nullptr);
    size_t last_upload_bytes = 0;

private:
    struct Stage { int* host = nullptr; size_t cap = 0; cudaEvent_t busy = nullptr; bool used = false; };
    Device* dev_;
    Runtime* rt_;
    Stage stages_[4];
    int next_ = 0;
};

}  // namespace illm
