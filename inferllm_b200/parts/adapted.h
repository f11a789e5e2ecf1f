// Low-rank adapters beside a part's projections: their storage and how a request's factors are packed into it.
#pragma once
#include <string>
#include <vector>

#include "parts/parts.h"

namespace illm {

// One packed projection with room for adapters.  It consists of up to kAdapterPieces pieces (q, k, v; gate, up), each with a
// tensor name and rows of its own among the packed ones: row0, row0 + step, ...  An adapter's ranks are its pieces' side by side,
// piece p's at p * r, r the adapter's rank; a piece without factors has zeros there.
class AdaptedProjection {
public:
    struct Piece { std::string name; long long rows, row0, step; };
    AdaptedProjection() {}
    AdaptedProjection(Runtime* rt, const char* what, long long n_in, std::vector<Piece> pieces, int count, int rank);
    // Adapter i becomes these factors, of rank `r` for every piece.
    void put(int i, const AdapterFactors& f);
    bool empty() const { return set_.count == 0; }
    const AdapterSet& set() const { return set_; }
    // the step's plan for this projection
    const AdapterView& view(const StepView& ctx) const { return ctx.adapters[pieces_.size() - 1]; }

private:
    Runtime* rt_ = nullptr;
    long long n_in_ = 0, n_out_ = 0;
    std::vector<Piece> pieces_;
    DeviceBuffer a_, b_, scales_;
    AdapterSet set_;
};

}  // namespace illm
