#include "parts/adapted.h"

#include <algorithm>
#include <cmath>

#include "util/dtype.h"

namespace illm {

AdaptedProjection::AdaptedProjection(Runtime* rt, const char* what, long long n_in, std::vector<Piece> pieces, int count, int rank)
        : rt_(rt), n_in_(n_in), pieces_(std::move(pieces)) {
    for (const Piece& p : pieces_) n_out_ += p.rows;
    const int R = ((int)pieces_.size() * rank + ADAPTER_GROUP - 1) / ADAPTER_GROUP * ADAPTER_GROUP;
    if (R > ADAPTER_GROUP * ADAPTER_MAX_GROUPS)
        throw EngineError(std::string("adapters of rank ") + std::to_string(rank) + " beside " + what + ": " + std::to_string(pieces_.size()) +
                          " projections side by side have more than 256 ranks");
    if (rt->dtype == DType::BF16 && n_in % 8) throw EngineError(std::string("adapters beside ") + what + ": its inner size " + std::to_string(n_in) + " must be a multiple of 8 in bfloat16");
    if ((long long)count * R * (n_out_ / ADAPTER_GROUP + 1) >= (1ll << 31)) throw EngineError(std::string("adapters beside ") + what + ": too many rows");
    const size_t es = dtype_size(rt->dtype), a = (size_t)count * R * n_in * es, b = (size_t)count * R * n_out_ * es;
    a_ = DeviceBuffer(rt->dev, a, "the first factors of adapters");
    b_ = DeviceBuffer(rt->dev, b, "the second factors of adapters");
    scales_ = DeviceBuffer(rt->dev, (size_t)count * sizeof(float), "the scales of adapters");
    check_cuda(cudaMemsetAsync(a_.get(), 0, a, rt->dev->stream()), "clearing adapters");
    check_cuda(cudaMemsetAsync(b_.get(), 0, b, rt->dev->stream()), "clearing adapters");
    check_cuda(cudaMemsetAsync(scales_.get(), 0, (size_t)count * sizeof(float), rt->dev->stream()), "clearing adapters");
    set_.a = a_.get();
    set_.b = b_.get();
    set_.scales = (const float*)scales_.get();
    set_.count = count;
    set_.R = R;
}

void AdaptedProjection::put(int i, const AdapterFactors& f) {
    const int R = set_.R;
    std::vector<float> a((size_t)R * n_in_, 0.f), b((size_t)R * n_out_, 0.f);
    for (size_t p = 0; p < pieces_.size(); p++) {
        auto it = f.of.find(pieces_[p].name);
        if (it == f.of.end()) continue;
        const AdapterFactors::One& one = it->second;
        const long long at = (long long)p * f.rank;
        std::copy(one.a, one.a + (size_t)one.r * n_in_, a.begin() + at * n_in_);
        for (long long o = 0; o < pieces_[p].rows; o++) {
            const long long row = pieces_[p].row0 + o * pieces_[p].step;
            for (int r = 0; r < one.r; r++) {
                const long long k = at + r;
                b[(size_t)((k / ADAPTER_GROUP * n_out_ + row) * ADAPTER_GROUP + k % ADAPTER_GROUP)] = one.b[o * one.r + r];
            }
        }
    }
    const size_t es = dtype_size(rt_->dtype);
    auto upload = [&](const std::vector<float>& from, void* to) {
        std::vector<uint16_t> half;
        const void* src = from.data();
        if (rt_->dtype == DType::BF16) {
            half.resize(from.size());
            for (size_t k = 0; k < from.size(); k++) half[k] = f32_to_bf16_bits(from[k]);
            src = half.data();
        }
        // behind the steps that the stream holds; the host memory is free when the call returns
        check_cuda(cudaMemcpyAsync(to, src, from.size() * es, cudaMemcpyHostToDevice, rt_->dev->stream()), "uploading an adapter");
        rt_->dev->synchronize();
    };
    upload(a, (char*)a_.get() + (size_t)i * a.size() * es);
    upload(b, (char*)b_.get() + (size_t)i * b.size() * es);
    check_cuda(cudaMemcpyAsync((float*)scales_.get() + i, &f.scale, sizeof(float), cudaMemcpyHostToDevice, rt_->dev->stream()), "uploading an adapter's scale");
    rt_->dev->synchronize();
}

}  // namespace illm
