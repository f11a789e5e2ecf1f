#include "engine/engine.h"

#include <climits>
#include <algorithm>
#include <cmath>
#include <cstring>
#include <set>

#include "kernels/adapter_plan.h"
#include "util/log.h"
#include "weights/loader.h"

namespace illm {

EngineOptions EngineOptions::from_json(const Json& j) {
    EngineOptions o;
    if (!j.is_object()) return o;
    if (j.at("dtype").is_string()) o.dtype = j.at("dtype").as_string();
    if (j.at("device_id").is_int()) o.device_id = (int)j.at("device_id").as_int();
    if (j.has("max_tokens")) o.max_tokens = j.at("max_tokens").is_int() ? j.at("max_tokens").as_int() : 0;
    if (j.at("mem_fraction").is_number()) o.mem_fraction = j.at("mem_fraction").as_double();
    if (j.at("max_seq_len").is_int()) o.max_seq_len = j.at("max_seq_len").as_int();
    if (j.at("max_batch").is_int()) o.max_batch = (int)j.at("max_batch").as_int();
    if (j.at("page_size").is_int()) o.page_size = (int)j.at("page_size").as_int();
    if (j.at("max_adapters").is_int()) o.max_adapters = (int)j.at("max_adapters").as_int();
    if (j.at("adapter_rank").is_int()) o.adapter_rank = (int)j.at("adapter_rank").as_int();
    if (j.at("cuda_graphs").is_bool()) o.cuda_graphs = j.at("cuda_graphs").as_bool();
    if (j.at("gemm").is_string()) o.gemm = j.at("gemm").as_string();
    if (j.at("poison_freed_pages").is_bool()) o.poison_freed_pages = j.at("poison_freed_pages").as_bool();
    if (j.has("cache_dtype") && j.at("cache_dtype").is_string()) o.cache_dtype = j.at("cache_dtype").as_string();
    if (j.has("share_prefixes") && j.at("share_prefixes").is_bool()) o.share_prefixes = j.at("share_prefixes").as_bool();
    if (j.has("shared_prefix_bytes") && j.at("shared_prefix_bytes").is_number())      // (numbers of 19 digits come as float64)
        o.shared_prefix_bytes = j.at("shared_prefix_bytes").as_double() >= 9e18 ? LLONG_MAX : j.at("shared_prefix_bytes").as_int();
    if (j.at("stream").is_int()) o.stream = (void*)(uintptr_t)j.at("stream").as_int();
    return o;
}

struct Engine::GraphEntry {
    cudaGraphExec_t exec = nullptr;     // nullptr: the shape has been seen once and is captured the next time
    cudaGraph_t graph = nullptr;
    int* ctx_buf = nullptr;             // the step's index arrays: the static input of the graph
    LogitsRef out;
    long long launches = 0;
};

static DType engine_dtype(const std::string& name) {
    if (name == "bfloat16" || name == "bf16") return DType::BF16;
    if (name == "float32" || name == "fp32") return DType::F32;
    throw EngineError("dtype '" + name + "' is not supported (bfloat16 or float32)");
}

static long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

Engine::Engine(std::unique_ptr<ArchConfig> config, const EngineOptions& options) : config_(std::move(config)), options_(options) {
    const DType dtype = engine_dtype(options.dtype);
    if (options.page_size <= 0) throw EngineError("page_size must be positive");
    if (options.max_adapters < 0 || options.max_adapters > 4096) throw EngineError("max_adapters must be in [0, 4096]");
    if (options.max_adapters > 0 && (options.adapter_rank < 1 || options.adapter_rank > ADAPTER_GROUP * ADAPTER_MAX_GROUPS / kAdapterPieces))
        throw EngineError("adapter_rank must be in [1, " + std::to_string(ADAPTER_GROUP * ADAPTER_MAX_GROUPS / kAdapterPieces) + "]");
    if (options.cache_dtype != "auto" && options.cache_dtype != "int8") throw EngineError("cache_dtype '" + options.cache_dtype + "' is not supported (auto or int8)");
    device_.reset(new Device(options.device_id, (cudaStream_t)options.stream));
    device_->set_weights_settled(true);
    rt_.dev = device_.get();
    rt_.dtype = dtype;
    rt_.page_size = options.page_size;
    rt_.gemm = ops::gemm_backend_from_name(options.gemm);
    model_.reset(new DecoderModel(config_->model_spec(), &rt_));
    const ModelSpec& spec = model_->spec;
    const long long max_seq = std::min(options.max_seq_len > 0 ? options.max_seq_len : spec.max_positions, spec.max_positions);
    // (before the cache, which may take its share of what is left)
    if (options.max_adapters > 0) {
        if (model_->adapted().empty()) throw EngineError("max_adapters: no layer of this model runs low-rank adapters");
        model_->make_adapters(options.max_adapters, options.adapter_rank);
        adapter_ranks_.assign((size_t)options.max_adapters, 0);
    }
    const std::map<int, CacheRequest> requests = model_->cache_requests(options.cache_dtype == "int8");
    if (options.cache_dtype == "int8") {
        bool any = false;
        for (auto& r : requests) any = any || r.second.int8;
        if (!any) throw EngineError("cache_dtype int8: no layer of this model keeps its keys and values in eight bits");
    }
    prefix_heads_ = model_->prefix_heads();
    long long max_tokens = options.max_tokens;
    if (max_tokens <= 0) max_tokens = tokens_that_fit(options.mem_fraction);
    const int num_pages = (int)std::max<long long>(1, ceil_div(max_tokens, options.page_size));
    const int num_slots = options.max_batch > 0 ? options.max_batch : num_pages;
    cache_.reset(new SequenceCache(requests, num_slots, num_pages, options.page_size, max_seq, device_.get(), dtype,
                                   options.poison_freed_pages));
    for (int entry : model_->prefix_entries()) {
        if (cache_->kind_of(entry) != SequenceCache::KV) continue;
        const SequenceCache::PagedGroup& g = cache_->paged[(size_t)cache_->group_of(entry)];
        prefix_entries_.insert({g.request.n_kv_heads, (long long)(g.page_bytes + g.v_page_bytes), g.request.int8});
    }
    builder_.reset(new StepContextBuilder(device_.get(), &rt_));
    for (TokRead& t : tok_reads_) check_cuda(cudaEventCreateWithFlags(&t.done, cudaEventDisableTiming), "cudaEventCreate");
    // say once which attention kernels the model's layers get: a head size that the tensor-core kernels
    // do not take falls to the general kernel, which is right but far slower on prompts
    std::set<std::string> said;
    std::set<int> int8_layers;
    for (const ScheduleEntry& s : spec.schedule)
        if (cache_->kind_of(s.cache) == SequenceCache::KV && cache_->paged[(size_t)cache_->group_of(s.cache)].request.int8) int8_layers.insert(s.layer);
    if (options.cache_dtype == "int8") {
        size_t paged = 0, int8 = 0;
        for (const SequenceCache::PagedGroup& g : cache_->paged) paged += g.entries.size(), int8 += g.request.int8 ? g.entries.size() : 0;
        log_line(LogLevel::Info, "cache: %zu of %zu entries in eight bits", int8, paged);
    }
    for (size_t i = 0; i < spec.layers.size(); i++) {
        const LayerSpec& ls = spec.layers[i];
        if (ls.mixer.kind != "attention" || !ls.mixer.has("n_heads")) continue;
        // a layer with sinks, gates, biases or norms of its own takes the general path (ops::attention_ex), which this line does not describe
        if (ls.mixer.get_bool("sink", false) || ls.mixer.get_bool("qkv_bias", false) || ls.mixer.has("out_gate") || ls.mixer.has("qk_norm")) continue;
        const int nh = (int)ls.mixer.get_int("n_heads"), nkv = (int)ls.mixer.get_int("n_kv_heads", nh), d = (int)ls.mixer.get_int("head_dim", 0);
        const std::string what = ops::attention_kernels_for(dtype, nh, nkv, d, options.page_size, int8_layers.count((int)i) != 0);
        const std::string line = std::to_string(nh) + " heads over " + std::to_string(nkv) + " of size " + std::to_string(d) + ", pages of " +
                                 std::to_string(options.page_size) + ": " + what;
        if (!said.insert(line).second) continue;
        const bool slow = dtype == DType::BF16 && (what.find("prompts: generic") != std::string::npos || what.find("plain") != std::string::npos);
        log_line(slow ? LogLevel::Warning : LogLevel::Info, "attention, %s%s", line.c_str(),
                 !slow                        ? ""
                 : int8_layers.count((int)i) ? " (head sizes 64 and 128 with pages of a multiple of 64 and, for single tokens, up to 16 heads per kv head get the tensor-core kernels)"
                                             : " (head sizes 64 and 128 get the tensor-core kernels)");
    }
}

Engine::~Engine() {
    if (device_) {
        cudaSetDevice(device_->ordinal());
        cudaStreamSynchronize(device_->stream());
    }
    drop_graphs(false);
    builder_.reset();
    for (TokRead& t : tok_reads_) {
        if (t.host) device_->free_pinned(t.host);
        if (t.done) cudaEventDestroy(t.done);
    }
    cache_.reset();
    model_.reset();
}

std::unique_ptr<Engine> Engine::from_folder(const std::string& folder, const EngineOptions& options, const std::string& model_name) {
    std::unique_ptr<Engine> e(new Engine(config_from_folder(folder, model_name), options));
    e->load_folder(folder);
    return e;
}
std::unique_ptr<Engine> Engine::from_config(std::unique_ptr<ArchConfig> config, const EngineOptions& options, unsigned long long seed) {
    std::unique_ptr<Engine> e(new Engine(std::move(config), options));
    e->load_random(seed);
    return e;
}
void Engine::load_folder(const std::string& folder) {
    device_->make_current();
    load_model_weights(*model_, folder);
    loaded_ = true;
}
void Engine::load_random(unsigned long long seed) {
    device_->make_current();
    init_random_weights(*model_, seed);
    loaded_ = true;
}

long long Engine::tokens_that_fit(double fraction) const {
    const size_t elem = dtype_size(rt_.dtype);
    size_t weights = 0;
    for (auto& d : model_->tensor_decls()) weights += (size_t)d.second.numel() * elem;
    const size_t per_token = SequenceCache::bytes_per_token(model_->cache_requests(options_.cache_dtype == "int8"), rt_.dtype);
    const size_t free_b = device_->mem_free();
    if (per_token == 0) return options_.page_size;
    const double room = ((double)free_b - (double)weights) * fraction;
    if (room < (double)per_token * options_.page_size) {
        char msg[200];
        snprintf(msg, sizeof msg, "the weights (%.1f GiB) leave no room for a cache on this device (%.1f GiB free%s)",
                 weights / 1073741824.0, free_b / 1073741824.0, options_.max_adapters > 0 ? " beside the room for adapters" : "");
        throw EngineError(msg);
    }
    return (long long)(room / (double)per_token);
}

int Engine::new_sequence() {
    device_->make_current();
    return cache_->alloc_slot();
}
int Engine::fork_sequence(int slot, long long length) {
    device_->make_current();
    return cache_->fork_slot(slot, length);
}
void Engine::end_sequence(int slot) {
    device_->make_current();
    cache_->free_slot(slot);
}
long long Engine::sequence_length(int slot) const {
    if (!cache_->slots.is_held(slot)) throw CacheError("slot " + std::to_string(slot) + " is not live");
    return cache_->seq_len[(size_t)slot];
}
Limits Engine::limits() const { return Limits{cache_->num_slots, cache_->num_pages, cache_->page_size, cache_->max_seq_len}; }
int Engine::graphs_captured() const {
    int n = 0;
    for (auto& g : graphs_)
        if (g.second->exec) n++;
    return n;
}

size_t Engine::context_ints(int T, int B, int K) const {
    return StepContextBuilder::ints(T, B, K, cache_->paged.size(), cache_->width);
}

int Engine::add_adapter(const AdapterFactors& f) {
    device_->make_current();
    const auto free = std::find(adapter_ranks_.begin(), adapter_ranks_.end(), 0);
    if (free == adapter_ranks_.end())
        throw EngineError("there is room for " + std::to_string(adapter_ranks_.size()) + " adapters (EngineOptions::max_adapters), and all are in use");
    const auto names = model_->adapted();
    std::string wrong;
    int rank = 0;
    if (f.of.empty()) wrong = " it has no factors;";
    if (!std::isfinite(f.scale)) wrong += " its scale is not finite;";
    for (auto& o : f.of) {
        const AdapterFactors::One& one = o.second;
        auto it = names.find(o.first);
        if (it == names.end()) {
            wrong += " '" + o.first + "' is no projection that runs adapters;";
            continue;
        }
        if (one.n_out != it->second[0] || one.n_in != it->second[1])
            wrong += " '" + o.first + "' is [" + std::to_string(it->second[0]) + ", " + std::to_string(it->second[1]) + "], the factors are for [" +
                     std::to_string(one.n_out) + ", " + std::to_string(one.n_in) + "];";
        else if (one.r < 1 || one.r > options_.adapter_rank)
            wrong += " '" + o.first + "': rank " + std::to_string(one.r) + " is outside [1, " + std::to_string(options_.adapter_rank) + "];";
        else {
            // (the prompt product multiplies an adapter's second factor with the zeros of its neighbours' tokens)
            const float most = rt_.is_f32() ? 3.4028235e38f : 3.3895314e38f;       // the largest that stays finite
            bool finite = true;
            for (long long k = 0; k < one.r * one.n_in; k++) finite = finite && std::fabs(one.a[k]) <= most;
            for (long long k = 0; k < one.r * one.n_out; k++) finite = finite && std::fabs(one.b[k]) <= most;
            if (!finite) wrong += " '" + o.first + "' is not finite;";
        }
        rank = std::max(rank, one.r);
    }
    if (!wrong.empty()) throw EngineError("the adapter does not fit the model:" + wrong);
    AdapterFactors own = f;
    own.rank = rank;
    const int i = (int)(free - adapter_ranks_.begin());
    model_->put_adapter(i, own);
    adapter_ranks_[(size_t)i] = rank;
    return i;
}
void Engine::remove_adapter(int i) {
    if (i < 0 || i >= (int)adapter_ranks_.size() || adapter_ranks_[(size_t)i] == 0) throw EngineError("adapter " + std::to_string(i) + " is not there");
    adapter_ranks_[(size_t)i] = 0;
}
// What is set aside for the plans: as much as these tokens need, or (a captured step) as any step of its kind can.
void Engine::size_adapters(StepAdapters& a, bool fixed, bool one_sequence) const {
    for (int p = 1; p <= kAdapterPieces; p++) {
        const std::vector<int> ranks = a.packed_ranks(p);
        a.sizes[p - 1] = fixed ? ops::adapter_plan_bound((int)a.index.size(), (int)ranks.size(), p * options_.adapter_rank, one_sequence)
                               : ops::adapter_plan_sizes(a.index.data(), (int)a.index.size(), ranks.data(), (int)ranks.size());
    }
}

StepContext Engine::make_context(const StepPlan& plan, const std::vector<int>& ids, const std::vector<int>& want_rows, int* into,
                                 std::vector<const int*>* tables_dev, const StepAdapters* adapters, const StepPrefixes* prefixes) {
    StepContext ctx = builder_->build(*cache_, plan, ids, want_rows, into, tables_dev, adapters, prefixes);
    last_upload_bytes_ = builder_->last_upload_bytes;
    return ctx;
}

// The common prefixes of a decode step's sequences, where walking them once saves more than the second launch of it costs.  What the launches depend on
// (tiles, the splits that follow from the lengths) is rounded up, so that captured steps of growing sequences can be replayed.
bool Engine::find_prefixes(const StepPlan& plan, StepPrefixes* out) const {
    if (!prefix_heads_ || plan.slots.size() < 2 || plan.slots.size() > kSharedPrefixSequences) return false;
    long long saved = 0;        // positions
    for (auto& g : cache_->common_prefixes(plan.slots)) {
        saved += g.first * ((long long)g.second.size() - 1);
        ops::PrefixGroup group;
        group.prefix = g.first;
        group.members = g.second;
        out->groups.push_back(std::move(group));
    }
    if (out->groups.empty()) return false;
    for (const PrefixEntry& e : prefix_entries_)
        if (options_.shared_prefix_bytes >= 0 ? saved / cache_->page_size * e.page_bytes < options_.shared_prefix_bytes
                                              : !ops::shared_prefix_pays(saved * e.rows, (long long)plan.slots.size(), e.int8))
            return false;
    std::vector<int> lens;
    for (size_t i = 0; i < plan.slots.size(); i++) lens.push_back((int)(plan.past[i] + 1));
    out->heads = prefix_heads_;
    out->sizes = ops::prefix_plan_sizes(out->groups, lens.data(), (int)lens.size(), prefix_heads_);
    auto up = [](int n) {
        int p = 1;
        while (p < n) p *= 2;
        return p;
    };
    out->sizes.tiles = up(out->sizes.tiles);
    out->sizes.longest_rest = up(out->sizes.longest_rest);
    out->sizes.longest_prefix = up(out->sizes.longest_prefix);
    return true;
}

LogitsRef Engine::run_forward(const StepContext& ctx, const std::vector<const int*>& tables) {
    Mat logits = model_->forward(ctx, *cache_, tables);
    return LogitsRef{(const float*)logits.p, ctx.K, model_->spec.vocab_size};
}

// ---- the step

LogitsRef Engine::step(const std::vector<StepItem>& items, const int* device_ids) {
    if (!loaded_) throw EngineError("the model has no weights yet");
    if (items.empty()) throw EngineError("a step needs at least one sequence");
    device_->make_current();
    const long long V = vocab_size();
    std::vector<int> ids, want_rows, slots, q_lens;
    StepAdapters step_adapters, *adapters = nullptr;
    int off = 0;
    for (const StepItem& it : items) {
        const int n = (int)it.tokens.size();
        if (n == 0) throw EngineError("slot " + std::to_string(it.slot) + ": a step must bring at least one token");
        for (int tok : it.tokens)
            if (tok < 0 || tok >= V)
                throw EngineError("slot " + std::to_string(it.slot) + ": token id " + std::to_string(tok) + " is outside the vocabulary [0, " +
                                  std::to_string(V) + ")");
        for (int w : it.want) {
            if (w < 0 || w >= n)
                throw EngineError("slot " + std::to_string(it.slot) + ": wanted place " + std::to_string(w) + " is outside its " +
                                  std::to_string(n) + " tokens");
            want_rows.push_back(off + w);
        }
        if (it.adapter != -1) {
            if (it.adapter < 0 || it.adapter >= (int)adapter_ranks_.size() || adapter_ranks_[(size_t)it.adapter] == 0)
                throw EngineError("slot " + std::to_string(it.slot) + ": adapter " + std::to_string(it.adapter) + " is not there");
            adapters = &step_adapters;
        }
        step_adapters.index.insert(step_adapters.index.end(), it.tokens.size(), it.adapter);
        ids.insert(ids.end(), it.tokens.begin(), it.tokens.end());
        slots.push_back(it.slot);
        q_lens.push_back(n);
        off += n;
    }
    if (device_ids && ids.size() != items.size()) throw EngineError("device_ids needs one int32 id per item and items of one token each");
    if (adapters) adapters->ranks = adapter_ranks_;
    if (graph_safe_ < 0) graph_safe_ = model_->graph_safe() ? 1 : 0;
    if (options_.cuda_graphs && items.size() == 1 && ids.size() > 1 && ids.size() <= (size_t)kPromptGraphMaxTokens) {
        if (pad_safe_ < 0) pad_safe_ = model_->pad_safe() ? 1 : 0;
        LogitsRef out;
        if (pad_safe_ && prompt_step_graphed(items[0].slot, ids, want_rows, adapters, &out)) return out;
    }
    StepPlan plan = cache_->plan_step(slots, q_lens);
    LogitsRef logits;
    try {
        StepPrefixes step_prefixes;
        const StepPrefixes* prefixes = ids.size() == items.size() && find_prefixes(plan, &step_prefixes) ? &step_prefixes : nullptr;
        if (options_.cuda_graphs && ids.size() == items.size() && graph_safe_) {
            if (adapters) size_adapters(*adapters, true, false);
            logits = decode_step_graphed(plan, ids, want_rows, device_ids, adapters, prefixes);
        } else {
            if (adapters) size_adapters(*adapters, false, false);
            device_->arena_rewind();
            std::vector<const int*> tables;
            StepContext ctx = make_context(plan, ids, want_rows, nullptr, &tables, adapters, prefixes);
            if (device_ids)
                check_cuda(cudaMemcpyAsync((void*)ctx.ids, device_ids, ids.size() * sizeof(int), cudaMemcpyDeviceToDevice, device_->stream()),
                           "copying the step's token ids");
            logits = run_forward(ctx, tables);
        }
    } catch (...) {
        cache_->abandon_step(plan);     // the pages reserved for the step go back
        throw;
    }
    cache_->commit_step(plan);
    return logits;
}

void Engine::drop_graphs(bool keep_seen) {
    if (device_) cudaStreamSynchronize(device_->stream());
    for (auto it = graphs_.begin(); it != graphs_.end();) {
        GraphEntry& e = *it->second;
        if (!e.exec && keep_seen) {
            ++it;
            continue;
        }
        if (e.exec) cudaGraphExecDestroy(e.exec);
        if (e.graph) cudaGraphDestroy(e.graph);
        if (e.ctx_buf) device_->free_persistent(e.ctx_buf);
        it = graphs_.erase(it);
    }
}

// A kind of step is captured the second time it comes.  Kinds that never came again are forgotten together; they take no room from those that were captured.
void Engine::seen_once(const std::string& key) {
    if (graphs_.size() > (size_t)kKindsMost + kGraphsMost)
        for (auto it = graphs_.begin(); it != graphs_.end();) it = it->second->exec ? std::next(it) : graphs_.erase(it);
    graphs_[key].reset(new GraphEntry);
}

LogitsRef Engine::capture_and_run(const std::string& key, const StepPlan& plan, const std::vector<int>& ids,
                                  const std::vector<int>& want_rows, const int* device_ids, const StepAdapters* adapters, const StepPrefixes* prefixes) {
    if (graphs_captured() > kGraphsMost) drop_graphs(true);
    std::unique_ptr<GraphEntry> e(new GraphEntry);
    int T = 0;
    for (int q : plan.q_lens) T += q;
    e->ctx_buf = (int*)device_->alloc_persistent(
            (context_ints(T, (int)plan.slots.size(), (int)want_rows.size()) + (adapters ? (adapters->ints() + 3) / 4 * 4 : 0) + (prefixes ? (size_t)prefixes->sizes.ints() : 0)) *
                    sizeof(int),
            "the inputs of a captured step");
    device_->arena_rewind();
    std::vector<const int*> tables;
    StepContext ctx = make_context(plan, ids, want_rows, e->ctx_buf, &tables, adapters, prefixes);
    if (device_ids)
        check_cuda(cudaMemcpyAsync((void*)ctx.ids, device_ids, ids.size() * sizeof(int), cudaMemcpyDeviceToDevice, device_->stream()),
                   "copying the step's token ids");
    device_->synchronize();
    const long long before = ops::launch_count();
    std::unique_ptr<Capture> going_on(new Capture);
    cudaError_t rc = cudaStreamBeginCapture(device_->stream(), cudaStreamCaptureModeRelaxed);
    if (rc != cudaSuccess) {
        device_->free_persistent(e->ctx_buf);
        check_cuda(rc, "cudaStreamBeginCapture");
    }
    try {
        e->out = run_forward(ctx, tables);
    } catch (...) {
        cudaGraph_t broken = nullptr;
        cudaStreamEndCapture(device_->stream(), &broken);
        if (broken) cudaGraphDestroy(broken);
        cudaGetLastError();
        device_->free_persistent(e->ctx_buf);
        throw;
    }
    rc = cudaStreamEndCapture(device_->stream(), &e->graph);
    going_on.reset();
    device_->make_current();            // (what waited may have been another device's)
    if (rc == cudaSuccess) rc = cudaGraphInstantiate(&e->exec, e->graph, 0);
    if (rc != cudaSuccess) {
        if (e->graph) cudaGraphDestroy(e->graph);
        device_->free_persistent(e->ctx_buf);
        cudaGetLastError();
        check_cuda(rc, "capturing a step in a CUDA graph");
    }
    e->launches = ops::launch_count() - before;
    check_cuda(cudaGraphLaunch(e->exec, device_->stream()), "cudaGraphLaunch");
    LogitsRef out = e->out;
    graphs_[key] = std::move(e);
    return out;
}

LogitsRef Engine::replay(GraphEntry& e, const StepPlan& plan, const std::vector<int>& ids, const std::vector<int>& want_rows,
                         const int* device_ids, const StepAdapters* adapters, const StepPrefixes* prefixes) {
    std::vector<const int*> tables;
    StepContext ctx = make_context(plan, ids, want_rows, e.ctx_buf, &tables, adapters, prefixes);
    if (device_ids)
        check_cuda(cudaMemcpyAsync((void*)ctx.ids, device_ids, ids.size() * sizeof(int), cudaMemcpyDeviceToDevice, device_->stream()),
                   "copying the step's token ids");
    check_cuda(cudaGraphLaunch(e.exec, device_->stream()), "cudaGraphLaunch");
    ops::count_replayed_launches(e.launches);
    return e.out;
}

// A single prompt (or a further piece of one sequence) of up to 1,024 tokens: the host needs longer to
// issue the step's launches than the GPU to run them, so the step is padded to whole buckets of 64
// tokens, with tokens behind the real ones that no real token sees (what they leave in the sequence's
// pages lies behind its length and is overwritten by the tokens that follow), and the launches of a
// bucket are captured in a CUDA graph the second time it is seen.  Only where the padding needs no
// page that the step would not need anyway and stays within the longest sequence; false otherwise (the
// caller then runs the step as it is).  The logits of the real tokens do not depend on the padding
// beyond rounding, and in float32 not at all.
bool Engine::prompt_step_graphed(int slot, const std::vector<int>& ids_in, const std::vector<int>& want_rows, StepAdapters* adapters, LogitsRef* out) {
    SequenceCache& c = *cache_;
    const int T = (int)ids_in.size();
    const int padded = (int)ceil_div(T, kPromptBucket) * kPromptBucket;
    if (!c.slots.is_held(slot)) return false;
    const long long past = c.seq_len[(size_t)slot];
    if (past + padded > c.max_seq_len) return false;
    for (auto& g : c.paged)
        if (g.ledger->pages_needed(slot, past + padded) != g.ledger->pages_needed(slot, past + T)) return false;
    StepPlan plan = c.plan_step({slot}, {padded});
    std::vector<int> ids = ids_in;
    ids.resize((size_t)padded, 0);
    const std::string key = std::string(adapters ? "pa/" : "p/") + std::to_string(padded) + "/" + std::to_string(want_rows.size());
    try {
        if (adapters) {
            adapters->index.resize((size_t)padded, adapters->index.back());
            size_adapters(*adapters, true, true);
        }
        auto it = graphs_.find(key);
        if (it == graphs_.end()) {
            seen_once(key);
            device_->arena_rewind();
            std::vector<const int*> tables;
            StepContext ctx = make_context(plan, ids, want_rows, nullptr, &tables, adapters);
            *out = run_forward(ctx, tables);
        } else if (!it->second->exec) {
            *out = capture_and_run(key, plan, ids, want_rows, nullptr, adapters);
        } else {
            *out = replay(*it->second, plan, ids, want_rows, nullptr, adapters);
        }
    } catch (...) {
        c.abandon_step(plan);
        throw;
    }
    plan.q_lens = {T};          // the sequence grows by its real tokens only
    c.commit_step(plan);
    return true;
}

// One token per sequence: the launches of such a step are the same every time (all that changes lies
// in device memory), so the step is captured in a CUDA graph the second time a batch size is seen and
// replayed from then on.
LogitsRef Engine::decode_step_graphed(const StepPlan& plan, const std::vector<int>& ids, const std::vector<int>& want_rows,
                                      const int* device_ids, const StepAdapters* adapters, const StepPrefixes* prefixes) {
    std::string key = std::string(adapters ? "da/" : "d/") + std::to_string(ids.size()) + "/" + std::to_string(want_rows.size());
    if (prefixes)
        for (int n : {prefixes->sizes.tiles, prefixes->sizes.per_tile, prefixes->sizes.longest_prefix, prefixes->sizes.longest_rest}) key += "/" + std::to_string(n);
    auto it = graphs_.find(key);
    if (it == graphs_.end()) {
        seen_once(key);
        device_->arena_rewind();
        std::vector<const int*> tables;
        StepContext ctx = make_context(plan, ids, want_rows, nullptr, &tables, adapters, prefixes);
        if (device_ids)
            check_cuda(cudaMemcpyAsync((void*)ctx.ids, device_ids, ids.size() * sizeof(int), cudaMemcpyDeviceToDevice, device_->stream()),
                       "copying the step's token ids");
        return run_forward(ctx, tables);
    }
    if (!it->second->exec) return capture_and_run(key, plan, ids, want_rows, device_ids, adapters, prefixes);
    return replay(*it->second, plan, ids, want_rows, device_ids, adapters, prefixes);
}

void Engine::read_logits(const LogitsRef& logits, float* host) {
    if (logits.rows <= 0) return;
    check_cuda(cudaMemcpyAsync(host, logits.p, (size_t)logits.rows * logits.vocab * sizeof(float), cudaMemcpyDeviceToHost, device_->stream()),
               "reading the logits");
    device_->synchronize();
}

int Engine::read_tokens_async(const int* toks, int n) {
    const int ticket = tok_next_;
    tok_next_ = (tok_next_ + 1) % 4;
    TokRead& r = tok_reads_[ticket];
    if (r.cap < n) {
        if (r.host) device_->free_pinned(r.host);
        r.cap = std::max(n, 256);
        r.host = (int*)device_->alloc_pinned((size_t)r.cap * sizeof(int));
    }
    r.n = n;
    check_cuda(cudaMemcpyAsync(r.host, toks, (size_t)n * sizeof(int), cudaMemcpyDeviceToHost, device_->stream()), "reading sampled tokens");
    check_cuda(cudaEventRecord(r.done, device_->stream()), "cudaEventRecord");
    return ticket;
}
std::vector<int> Engine::finish_read(int ticket) {
    TokRead& r = tok_reads_[ticket & 3];
    check_cuda(cudaEventSynchronize(r.done), "waiting for sampled tokens");
    return std::vector<int>(r.host, r.host + r.n);
}

void Engine::warm_up(long long prompt_tokens, const std::vector<int>& batch_sizes) {
    const Limits lim = limits();
    const long long longest = std::min<long long>({prompt_tokens, lim.max_seq_len, (long long)lim.num_pages * lim.page_size});
    for (long long n = ops::kLibraryRowBucket; n <= longest; n += ops::kLibraryRowBucket) {
        bool full = false;
        for (int round = 0; round < (n <= kPromptGraphMaxTokens ? 2 : 1) && !full; round++) {     // the second sight of a bucket captures its graph
            int slot;
            try {
                slot = new_sequence();
            } catch (const CacheError&) {
                full = true;
                break;
            }
            try {
                StepItem it;
                it.slot = slot;
                it.tokens.assign((size_t)n, 0);
                it.want = {(int)n - 1};
                step({it});
            } catch (const CacheError&) {          // live sequences hold the pages: no larger size fits either
                full = true;
            }
            end_sequence(slot);
        }
        if (full) break;
    }
    for (int b : batch_sizes) {
        if (b < 1 || b > lim.max_batch || b > lim.num_pages || cache_->slots.n_free() < b) continue;
        std::vector<int> slots;
        for (int i = 0; i < b; i++) slots.push_back(new_sequence());
        try {
            for (int round = 0; round < 4; round++) {
                std::vector<StepItem> items;
                for (int s : slots) {
                    StepItem it;
                    it.slot = s;
                    it.tokens = {0};
                    it.want = {0};
                    items.push_back(it);
                }
                step(items);
            }
        } catch (const CacheError&) {
        }
        for (int s : slots) end_sequence(s);
    }
    device_->synchronize();
}

void Engine::check_device_errors() {
    auto words = device_->take_error_words();
    if (words.first) {
        const char* what;
        switch (words.first) {
            case 4: what = "a wait inside the tensor-core matrix product (gemm_tc, gemm_tc2) timed out"; break;
            case 5: what = "a wait inside the tensor-core prompt attention (attention_prefill_tc, attention_tiles) timed out"; break;
            case 6: what = "a tensor-core kernel found its shared memory misaligned and did not run"; break;
            case 7: what = "a wait inside the decode attention (attention_decode_ring, attention_pages) timed out"; break;
            case 8: what = "an attention kernel met a visible position whose page the sequence does not hold"; break;
            default: what = nullptr;
        }
        throw EngineError((what ? std::string(what) : "a tensor-core kernel reported error " + std::to_string(words.first)) +
                          ": the step's results are not valid");
    }
    if (words.second) {
        const char* what;
        switch (words.second) {
            case 1: what = "a token id outside the embedding table"; break;
            case 2: what = "a cache write to a page that the sequence does not hold"; break;
            case 3: what = "a position beyond the position table"; break;
            default: what = nullptr;
        }
        throw EngineError("a kernel reported " + (what ? std::string(what) : "error " + std::to_string(words.second)));
    }
}

}  // namespace illm
