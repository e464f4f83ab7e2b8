// Tests of the tl:: layer's token-model ops (layer_norm, embedding,
// token_logprobs and their autograd nodes) against the formulas in 64 bits, and
// of a whole chain of them with matmul and flash attention.
//
//   tl_token_tests            all tests (needs a GPU)
//   tl_token_tests --cpu      only the exception tests (no GPU needed)
#include <tl/autograd.h>
#include <tl/ops.h>
#include <tl/tensor.h>
#include <tl/tokens.h>

#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <functional>
#include <iostream>
#include <stdexcept>
#include <string>
#include <vector>

#define CHECK(cond)                                                              \
    do {                                                                         \
        if (!(cond)) {                                                           \
            std::cerr << "FAIL: " #cond " at " __FILE__ ":" << __LINE__ << "\n"; \
            std::exit(1);                                                        \
        }                                                                        \
    } while (0)

template <typename F>
static void expect_invalid(F f, const char* part) {
    try {
        f();
    } catch (const std::invalid_argument& e) {
        CHECK(std::string(e.what()).find(part) != std::string::npos);
        return;
    }
    CHECK(!"expected std::invalid_argument");
}

static uint32_t g_state = 1u;
static float uniform() {
    g_state = g_state * 1664525u + 1013904223u;
    return ((g_state >> 8) & 0xFFFF) / 32768.0f - 1.0f;
}
static tl::Tensor random(const std::vector<int64_t>& sizes, float size = 1.0f) {
    tl::Tensor t(sizes);
    for (int64_t i = 0; i < t.numel(); ++i) t.data()[i] = size * uniform();
    return t;
}

static void test_errors() {
    expect_invalid([] { tl::Tokens({2, 2}, {1, 2, 3}); }, "3 values for 4 places");
    tl::Tokens none;
    tl::Tensor w({4, 3});
    expect_invalid([&] { tl::embedding(w, none); }, "empty");
    expect_invalid([&] { tl::embedding(tl::Tensor({4}), tl::Tokens({1}, {0})); }, "2-D");
    expect_invalid([&] { tl::layer_norm(tl::Tensor(std::vector<int64_t>{}), tl::Tensor(), tl::Tensor()); }, "1-D");
    expect_invalid([&] { tl::token_logprobs(w, none); }, "empty");
    expect_invalid([&] { tl::token_logprobs(w, tl::Tokens({4}, {0, 1, 2, 0}), 1.0f, -1); }, "top");
    // refused before any output is made
    expect_invalid([&] { tl::token_logprobs(w, tl::Tokens({4}, {0, 1, 2, 0}), 1.0f, 4); }, "vocabulary's size");
    expect_invalid([&] { tl::token_logprobs(w, tl::Tokens({4}, {0, 1, 2, 0}), 1.0f, 2147483647); }, "vocabulary's size");
    bool many = false;
    try {
        tl::token_logprobs(tl::Tensor({1, 50}), tl::Tokens({1}, {0}), 1.0f, 33);
    } catch (const std::runtime_error& e) {
        many = std::string(e.what()).find("at most 32") != std::string::npos;
    }
    CHECK(many);
    std::cout << "errors ok\n";
}

// Gradients of `f`, a sum in 64 bits, by central differences, against `grad`.
// The difference is off by h^2 / 6 times third derivatives of at most 1e3 and
// by 2^-52 |f| / h, the gradient by some hundred roundings of its terms.
static void against_differences(std::vector<double>& at, const std::function<double()>& f, const float* grad) {
    for (size_t i = 0; i < at.size(); ++i) {
        const double keep = at[i], h = 1e-5;
        at[i] = keep + h;
        const double up = f();
        at[i] = keep - h;
        const double down = f();
        at[i] = keep;
        const double d = (up - down) / (2 * h);
        CHECK(std::fabs(d - grad[i]) <= 3e-5 * std::fmax(1.0, std::fabs(d)));
    }
}

// A small language model, twice: on the device in fp32, and here in 64 bits.
//   h = embedding(tokens), a = layer_norm(h), q = a Wq, o = flash(q, a, a),
//   y = layer_norm(h + o), logits = y Wo; loss = -sum(logprobs) - 0.1 sum(entropy)
static void test_chain() {
    const int64_t S = 7, D = 12, V = 19;
    const std::vector<int64_t> tok = {3, 18, 3, 0, 7, -1, 3}, next = {18, 3, 0, 7, -1, 3, 11};
    tl::Tensor E = random({V, D}), w1 = random({D}, 0.5f), b1 = random({D}), Wq = random({D, D}, 0.5f), w2 = random({D}),
               Wo = random({D, V}, 0.5f);
    for (int64_t i = 0; i < D; ++i) w1.data()[i] += 1.0f, w2.data()[i] += 1.0f;
    std::vector<tl::Tensor*> params = {&E, &w1, &b1, &Wq, &w2, &Wo};
    for (auto* p : params) p->set_requires_grad(true);
    const float att = 0.3f, emb = 1.5f, temp = 0.9f;

    tl::Tokens t({S}, tok), n({S}, next);
    tl::Tensor h = tl::embedding(E, t, emb);
    tl::Tensor a = tl::layer_norm(h, w1, b1);
    tl::Tensor q = tl::matmul(a, Wq);
    tl::Tensor o = tl::flash_attention(q, a, a, att);
    tl::Tensor y = tl::layer_norm(tl::add(h, o), w2, tl::Tensor());
    tl::Tensor logits = tl::matmul(y, Wo);
    tl::TokenScores s = tl::token_logprobs(logits, n, temp, 3);
    tl::Tensor total = tl::add(tl::scale(s.logprobs, -1.0f), tl::scale(s.entropy, -0.1f));
    total.backward();

    std::vector<std::vector<double>> v(params.size());
    for (size_t k = 0; k < params.size(); ++k) v[k].assign(params[k]->data(), params[k]->data() + params[k]->numel());
    std::vector<double> lp(S), ent(S), lg(S * V);
    auto norm = [&](const std::vector<double>& x, const std::vector<double>& w, const double* b) {
        std::vector<double> r(S * D);
        for (int64_t i = 0; i < S; ++i) {
            double m = 0, var = 0;
            for (int64_t j = 0; j < D; ++j) m += x[i * D + j] / D;
            for (int64_t j = 0; j < D; ++j) var += (x[i * D + j] - m) * (x[i * D + j] - m) / D;
            for (int64_t j = 0; j < D; ++j)
                r[i * D + j] = (x[i * D + j] - m) / std::sqrt(var + 1e-5f) * w[j] + (b ? b[j] : 0.0);
        }
        return r;
    };
    auto model = [&]() {
        std::vector<double> x(S * D, 0.0), qq(S * D, 0.0), oo(S * D, 0.0);
        for (int64_t i = 0; i < S; ++i)
            if (tok[i] >= 0)
                for (int64_t j = 0; j < D; ++j) x[i * D + j] = (double)emb * v[0][tok[i] * D + j];
        std::vector<double> aa = norm(x, v[1], v[2].data());
        for (int64_t i = 0; i < S; ++i)
            for (int64_t j = 0; j < D; ++j)
                for (int64_t k = 0; k < D; ++k) qq[i * D + j] += aa[i * D + k] * v[3][k * D + j];
        for (int64_t i = 0; i < S; ++i) {
            std::vector<double> e(S);
            double l = 0;
            for (int64_t k = 0; k < S; ++k) {
                double dot = 0;
                for (int64_t j = 0; j < D; ++j) dot += qq[i * D + j] * aa[k * D + j];
                l += e[k] = std::exp(dot * (double)att);
            }
            for (int64_t k = 0; k < S; ++k)
                for (int64_t j = 0; j < D; ++j) oo[i * D + j] += e[k] / l * aa[k * D + j];
        }
        for (int64_t i = 0; i < S * D; ++i) oo[i] += x[i];
        std::vector<double> yy = norm(oo, v[4], nullptr);
        double f = 0;
        for (int64_t i = 0; i < S; ++i) {
            double l = 0, ex = 0;
            for (int64_t c = 0; c < V; ++c) {
                double z = 0;
                for (int64_t j = 0; j < D; ++j) z += yy[i * D + j] * v[5][j * V + c];
                lg[i * V + c] = z;
                l += std::exp(z * (double)temp);
                ex += std::exp(z * (double)temp) * z * (double)temp;
            }
            lp[i] = next[i] >= 0 ? lg[i * V + next[i]] * (double)temp - std::log(l) : 0.0;
            ent[i] = std::log(l) - ex / l;
            f += -lp[i] - 0.1f * ent[i];
        }
        return f;
    };
    model();
    // the chain's roundings: attention's products and exponentials are good to 1e-5 here
    for (int64_t i = 0; i < S; ++i) {
        CHECK(std::fabs(s.logprobs.data()[i] - lp[i]) <= 2e-5 * (1 + std::fabs(lp[i])));
        CHECK(std::fabs(s.entropy.data()[i] - ent[i]) <= 2e-5);
        double last = 1e300;
        for (int k = 0; k < 3; ++k) {
            const int64_t c = s.top_tokens.values()[i * 3 + k];
            CHECK(c >= 0 && c < V && lg[i * V + c] <= last);
            last = lg[i * V + c];
        }
    }
    for (size_t k = 0; k < params.size(); ++k) against_differences(v[k], model, params[k]->grad().data());
    std::cout << "chain ok\n";
}

static void test_gradients_add_up() {
    // a second use of the same table adds to its gradient; views are read in place
    tl::Tensor E = random({5, 4});
    E.set_requires_grad(true);
    tl::Tokens t({2, 2}, {0, 1, 1, -1});
    tl::Tensor y = tl::add(tl::embedding(E, t), tl::embedding(E, t, 2.0f));
    y.backward();
    const float want[5] = {3.0f, 6.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t i = 0; i < 20; ++i) CHECK(E.grad().data()[i] == want[i / 4]);

    tl::Tensor x = random({6, 3}), w = random({6}), b = random({6});
    tl::Tensor direct = tl::layer_norm(tl::transpose(x, 0, 1), w, b);
    tl::Tensor dense = tl::layer_norm(tl::transpose(x, 0, 1).contiguous(), w, b);
    for (int64_t i = 0; i < 18; ++i) CHECK(direct.data()[i] == dense.data()[i]);
    {
        tl::NoGradGuard guard;
        x.set_requires_grad(true);
        CHECK(!tl::layer_norm(x, tl::Tensor(), tl::Tensor()).grad_fn);
    }
    tl::Tensor none = tl::layer_norm(tl::Tensor({0, 6}), w, b);
    CHECK(none.numel() == 0);
    std::cout << "gradients ok\n";
}

int main(int argc, char** argv) {
    const bool cpu_only = argc > 1 && std::string(argv[1]) == "--cpu";
    test_errors();
    if (cpu_only) return 0;
    test_chain();
    test_gradients_add_up();
    std::cout << "all token tests passed\n";
    return 0;
}
