// The generic decoder: embedding, blocks run in the order of the schedule, final norm, head.
//
// It is built from a ModelSpec alone: each layer's block arrangement, mixer, feed-forward and norms,
// the embedding and the head are looked up by kind in the part registries and built with the spec's
// parameters, so layers of one model may differ, a layer may run twice, and a layer may read another
// layer's cache.  The reference builds its module list the same way from a per-model construct_llm
// (src/graph/llama_like.cpp:54-109) and runs it in Graph::execute (src/core/graph.cpp:166-197).
#pragma once
#include <functional>
#include <map>
#include <memory>
#include <set>
#include <string>
#include <vector>

#include "parts/parts.h"

namespace illm {

class SequenceCache;

// The cache entry number of an embedding that keeps per-sequence state (schedule entries count from 0).
constexpr int kEmbeddingCacheEntry = -1;
// ModelSpec::reentry of this kind is no part: before a schedule entry marked `reenter` the embedding output is added to
// the stream (x <- x + x0, float32), instead of a map of the two joined.
constexpr const char* kReentryAddEmbedding = "add_embedding";
// A mixer's second entry (Mixer::aux_cache_request) has the number of its first plus this.
constexpr int kAuxCacheEntryBase = 1 << 20;

class DecoderModel {
public:
    // runtime == nullptr: the parts only declare their tensors (for checking a folder or writing a
    // random one without a device).
    DecoderModel(const ModelSpec& spec, Runtime* runtime);

    // Every tensor the model reads from a weight file, by its name there, in a fixed order.
    // (tensors declared optional only if asked: a weight file is checked with them, a random model has none)
    std::vector<std::pair<std::string, TensorDecl>> tensor_decls(bool include_optional = false) const;
    // `open(prefix)` gives the source of the tensors below a prefix; each part takes its own and packs
    // them, one part at a time.
    void load_tensors(const std::function<std::unique_ptr<TensorSource>(const std::string& prefix)>& open);
    // Cache entry number -> what its writing layer's mixer asks for.
    // int8: keys and values in eight bits wherever every layer that uses the entry can (Mixer::takes_int8_cache).
    std::map<int, CacheRequest> cache_requests(bool int8 = false) const;
    // Query heads per kv head of the layers that walk common prefixes once (Mixer::prefix_heads); 0: no layer does, or they differ.
    int prefix_heads() const;
    // The cache entries of those layers.
    std::set<int> prefix_entries() const;
    // Run the tokens of one step; float32 logits [ctx.K, vocab] (rows == 0 when nothing is wanted).
    Mat forward(const StepContext& ctx, const SequenceCache& cache, const std::vector<const int*>& tables_dev);
    // Low-rank adapters: the names (as in the weight file) of the matrices beside which they can stand, with their shapes; room
    // for `count` of rank up to `rank`; adapter i's factors by those names.
    std::map<std::string, std::vector<long long>> adapted() const;
    void make_adapters(int count, int rank);
    void put_adapter(int i, const AdapterFactors& f);
    // true if a one-token-per-sequence step launches the same kernels every time, i.e. no part reads
    // host-side fields of the step context.
    bool graph_safe() const;
    // true if a single prompt may be run with tokens appended behind its own (see Mixer::pad_safe).
    bool pad_safe() const;

    ModelSpec spec;
    Runtime* rt;

private:
    struct Layer {
        std::unique_ptr<Block> block;
        std::unique_ptr<Mixer> mixer;
        std::unique_ptr<FeedForward> ffn;
        std::map<std::string, std::unique_ptr<Norm>> norms;
    };
    std::vector<std::pair<std::string, Part*>> owners() const;
    std::unique_ptr<EmbeddingPart> embedding_;
    std::unique_ptr<FeedForward> reentry_;      // the map of [stream; embedding output] before the entries marked `reenter`
    std::vector<Layer> layers_;
    std::unique_ptr<Norm> final_norm_;
    std::unique_ptr<HeadPart> head_;
};

}  // namespace illm
