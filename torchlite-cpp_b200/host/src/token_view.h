// The C-ABI view of tl::Tokens, for the layer's ops and nodes.
#pragma once

#include <tl/tokens.h>

#include <tlc.h>

#include <stdexcept>

namespace tl {

inline tlc_index index_of(const Tokens& t) {
    if (t.empty()) throw std::invalid_argument("Tokens: empty");
    if (t.sizes().size() > TLC_MAX_DIMS) throw std::invalid_argument("Tokens: more than 8 dims");
    tlc_index v{};
    v.ndim = static_cast<int32_t>(t.sizes().size());
    v.bits = 64;
    int64_t step = 1;
    for (int i = v.ndim - 1; i >= 0; --i) {
        v.sizes[i] = t.sizes()[i];
        v.strides[i] = step;
        step *= t.sizes()[i];
    }
    v.data = t.numel() > 0 ? const_cast<int64_t*>(t.device_data()) : nullptr;
    return v;
}

}  // namespace tl
