// tl::Tokens: token numbers with mirrored host / device storage (see tokens.h).
#include <tl/tokens.h>

#include <tlc.h>

#include <new>
#include <stdexcept>
#include <string>

namespace tl {

namespace {

void check(int status, const char* what) {
    if (status == TLC_OK) return;
    if (status == TLC_ERR_OUT_OF_MEMORY) throw std::bad_alloc();
    throw std::runtime_error(std::string(what) + ": " + tlc_last_error());
}

int64_t count_of(const std::vector<int64_t>& sizes) {
    int64_t n = 1;
    for (int64_t s : sizes) {
        if (s < 0) throw std::invalid_argument("Tokens: negative size");
        n *= s;
    }
    return n;
}

}  // namespace

struct Tokens::Buffer {
    std::vector<int64_t> host;
    int64_t* dev = nullptr;
    int64_t n = 0;
    bool host_valid = false, dev_valid = false;
    ~Buffer() {
        if (dev) tlc_free(dev);
    }
    int64_t* device_raw() {
        if (!dev && n > 0) {
            void* p = nullptr;
            check(tlc_malloc(&p, sizeof(int64_t) * static_cast<size_t>(n)), "tlc_malloc");
            dev = static_cast<int64_t*>(p);
        }
        return dev;
    }
};

Tokens::Tokens(const std::vector<int64_t>& sizes, const std::vector<int64_t>& values) : sizes_(sizes) {
    const int64_t n = count_of(sizes);
    if (static_cast<int64_t>(values.size()) != n)
        throw std::invalid_argument("Tokens: " + std::to_string(values.size()) + " values for " + std::to_string(n) +
                                    " places");
    data_ = std::make_shared<Buffer>();
    data_->n = n;
    data_->host = values;
    data_->host_valid = true;
}

Tokens Tokens::device_empty(const std::vector<int64_t>& sizes) {
    Tokens t;
    t.sizes_ = sizes;
    t.data_ = std::make_shared<Buffer>();
    t.data_->n = count_of(sizes);
    t.data_->device_raw();
    t.data_->dev_valid = true;
    return t;
}

int64_t Tokens::numel() const { return data_ ? data_->n : 0; }

const std::vector<int64_t>& Tokens::values() const {
    if (!data_) throw std::invalid_argument("Tokens: empty");
    Buffer& b = *data_;
    if (!b.host_valid) {
        b.host.resize(static_cast<size_t>(b.n));
        if (b.n > 0) {
            check(tlc_memcpy(b.host.data(), b.dev, sizeof(int64_t) * b.n, 1, nullptr), "d2h");
            check(tlc_stream_synchronize(nullptr), "sync");
        }
        b.host_valid = true;
    }
    return b.host;
}

const int64_t* Tokens::device_data() const {
    if (!data_) throw std::invalid_argument("Tokens: empty");
    Buffer& b = *data_;
    int64_t* d = b.device_raw();
    if (!b.dev_valid && b.n > 0)
        check(tlc_memcpy(d, b.host.data(), sizeof(int64_t) * b.n, 0, nullptr), "h2d");
    b.dev_valid = true;
    return d;
}

int64_t* Tokens::device_out() {
    if (!data_) throw std::invalid_argument("Tokens: empty");
    data_->dev_valid = true;
    data_->host_valid = false;
    return data_->device_raw();
}

}  // namespace tl
