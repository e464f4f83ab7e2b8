// Token numbers of any shape, for tl::embedding and tl::token_logprobs
// (tl::Tensor holds floats alone).  Mirrored like a Tensor's storage: a host
// copy and a device copy, each made when it is first needed.
#pragma once

#include <cstdint>
#include <memory>
#include <vector>

namespace tl {

class Tokens {
  public:
    Tokens() = default;
    // `values` in row-major order; -1 marks padding
    Tokens(const std::vector<int64_t>& sizes, const std::vector<int64_t>& values);
    // contents undefined, on the device: the output of a GPU op
    static Tokens device_empty(const std::vector<int64_t>& sizes);

    const std::vector<int64_t>& sizes() const { return sizes_; }
    int64_t numel() const;
    bool empty() const { return !data_; }
    const std::vector<int64_t>& values() const;  // row-major, copied from the device if need be
    const int64_t* device_data() const;
    int64_t* device_out();                       // for a GPU op that writes every value

  private:
    struct Buffer;
    std::vector<int64_t> sizes_;
    std::shared_ptr<Buffer> data_;
};

}  // namespace tl
