// test_ag_losses.cpp -- layer_norm, linear_cross_entropy and distill_topk in the ag:: graph on
// the GPU: numerical gradients (central differences of the forward, as for the other ops),
// accumulation, a norm whose output both losses read, forward mode, refusals, capture and
// replay, empty batches.  Prints PASS/FAIL per check; exits with the number of failures.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "ag/ag.hpp"

using namespace ag;

namespace {

int g_failures = 0;

void report(const char* name, bool ok, const std::string& detail = "") {
    std::printf("[%s] %s%s%s\n", ok ? "PASS" : "FAIL", name, detail.empty() ? "" : ": ",
                detail.c_str());
    std::fflush(stdout);
    if (!ok) ++g_failures;
}

std::vector<float> normal(size_t n, uint64_t seed, float sd = 1.0f) {
    std::mt19937_64 eng(seed);
    std::normal_distribution<float> d(0.0f, sd);
    std::vector<float> v(n);
    for (float& f : v) f = d(eng);
    return v;
}

Value leaf(const std::vector<float>& v, const std::vector<int64_t>& shape, const char* name) {
    Tensor t = Tensor::from_host_f32(v, shape);
    t.set_requires_grad(true);
    return make_tensor(t, name);
}

double sum_of(const Value& y) {
    double s = 0.0;
    for (float v : y.val().to_host_f32()) s += v;
    return s;
}

// |analytic - central difference of f| for every element of p.  f's fp32 forward is good to
// about 1e-6 of values of a few units, which over 2 h = 0.02 is 1e-4; the differences' own
// error is h^2 / 6 times third derivatives of a few units, another 1e-4.
void check_grad(const char* name, Value& p, const std::function<double()>& f,
                double tol = 1e-3) {
    const std::vector<float> grad = p.grad().to_host_f32(), orig = p.val().to_host_f32();
    const std::vector<int64_t> shape = p.val().shape();
    const float h = 1e-2f;
    double worst = 0.0;
    for (size_t i = 0; i < orig.size(); ++i) {
        std::vector<float> v = orig;
        v[i] = orig[i] + h;
        const double up = v[i];
        p.val() = Tensor::from_host_f32(v, shape);
        const double hi = f();
        v[i] = orig[i] - h;
        const double dn = v[i];
        p.val() = Tensor::from_host_f32(v, shape);
        const double lo = f();
        worst = std::max(worst, std::fabs((hi - lo) / (up - dn) - grad[i]));
    }
    p.val() = Tensor::from_host_f32(orig, shape);
    report(name, worst <= tol, "max |analytic - numerical| = " + std::to_string(worst));
}

bool throws(const std::function<void()>& f) {
    try {
        f();
    } catch (const std::runtime_error&) {
        return true;
    }
    return false;
}

void test_layer_norm() {
    Value x = leaf(normal(40, 1), {4, 10}, "x"), g = leaf(normal(10, 2), {10}, "g"),
          b = leaf(normal(10, 3), {1, 10}, "b");
    Tensor dy = Tensor::from_host_f32(normal(40, 4), {4, 10});
    auto f = [&] { return sum_of(layer_norm(x, g, b) * make_tensor(dy)); };
    backward(layer_norm(x, g, b), &dy);
    check_grad("layer_norm dx", x, f);
    check_grad("layer_norm dgamma", g, f);
    check_grad("layer_norm dbeta", b, f);
    const std::vector<float> once = g.grad().to_host_f32(), dx = x.grad().to_host_f32();
    backward(layer_norm(x, g, b), &dy);
    const std::vector<float> twice = g.grad().to_host_f32(), dx2 = x.grad().to_host_f32();
    bool same = true;
    for (size_t i = 0; i < once.size(); ++i) same = same && twice[i] == 2 * once[i];
    for (size_t i = 0; i < dx.size(); ++i) same = same && dx2[i] == 2 * dx[i];
    report("layer_norm gradients accumulate", same);

    nn::LayerNorm m(10);
    Value y = m(x);
    report("nn::LayerNorm starts as laynor", y.val().to_host_f32() == laynor(x).val().to_host_f32());
    backward(y);
    report("nn::LayerNorm has two parameters with fp32 gradients",
           m.parameters().size() == 2 && m.gamma.grad().dtype() == Dtype::Float32 &&
               m.beta.grad().to_host_f32() == std::vector<float>(10, 4.0f));

    // forward mode along (tx, tg, tb) against differences
    const std::vector<float> tx = normal(40, 5), tg = normal(10, 6), tb = normal(10, 7);
    const std::vector<float> xv = x.val().to_host_f32(), gv = g.val().to_host_f32(),
                             bv = b.val().to_host_f32();
    Tensor ty = jvp(layer_norm(x, g, b), {{x.node.get(), Tensor::from_host_f32(tx, {4, 10})},
                                          {g.node.get(), Tensor::from_host_f32(tg, {10})},
                                          {b.node.get(), Tensor::from_host_f32(tb, {1, 10})}});
    auto at = [&](float h) {
        auto move = [&](const std::vector<float>& v, const std::vector<float>& t) {
            std::vector<float> r = v;
            for (size_t i = 0; i < r.size(); ++i) r[i] += h * t[i];
            return r;
        };
        return layer_norm(leaf(move(xv, tx), {4, 10}, "x"), leaf(move(gv, tg), {10}, "g"),
                          leaf(move(bv, tb), {1, 10}, "b"))
            .val()
            .to_host_f32();
    };
    const float h = 2e-3f;
    const std::vector<float> hi = at(h), lo = at(-h), got = ty.to_host_f32();
    double worst = 0.0;
    for (size_t i = 0; i < got.size(); ++i)
        worst = std::max(worst, std::fabs((double(hi[i]) - lo[i]) / (2 * h) - got[i]));
    report("jvp of layer_norm == central differences", worst <= 1e-2, std::to_string(worst));
}

void test_cross_entropy() {
    Value x = leaf(normal(48, 11), {2, 2, 12}, "x"), w = leaf(normal(108, 12, 0.5f), {9, 12}, "w");
    const Indices labels = Indices::from_host({3, -100, 8, 0}, {2, 2});
    auto loss = [&] { return linear_cross_entropy(x, w, labels); };
    Value l = loss();
    report("linear_cross_entropy has a loss [..., 1] per row, 0 without a label",
           l.val().shape() == std::vector<int64_t>{2, 2, 1} && l.val().to_host_f32()[1] == 0.0f &&
               l.val().dtype() == Dtype::Float32);
    Tensor dy = Tensor::from_host_f32({0.5f, 7.0f, -1.25f, 2.0f}, {2, 2, 1});
    backward(l, &dy);
    auto f = [&] { return sum_of(loss() * make_tensor(dy)); };
    check_grad("linear_cross_entropy dx", x, f);
    check_grad("linear_cross_entropy dw", w, f);
    Value frozen = make_tensor(Tensor::from_host_f32(normal(108, 12, 0.5f), {9, 12}), "frozen");
    Value x2 = leaf(normal(48, 11), {2, 2, 12}, "x2");
    backward(linear_cross_entropy(x2, frozen, labels), &dy);
    report("a frozen head leaves dx as it was", x2.grad().to_host_f32() == x.grad().to_host_f32());
}

void test_distill() {
    Value z = leaf(normal(80, 21, 2.0f), {4, 20}, "z");
    const Indices index =
        Indices::from_host({1, 5, 19, 0, -1, 7, -1, -1, -1, 4, 4, 2}, {4, 3});
    const Tensor teacher = Tensor::from_host_f32(normal(12, 22), {4, 3});
    auto loss = [&] { return distill_topk(z, index, teacher, 1.5f); };
    Value l = loss();
    report("distill_topk has a loss [..., 1] per row, 0 without a teacher",
           l.val().shape() == std::vector<int64_t>{4, 1} && l.val().to_host_f32()[2] == 0.0f);
    Tensor dy = Tensor::from_host_f32(normal(4, 23), {4, 1});
    backward(l, &dy);
    check_grad("distill_topk dz", z, [&] { return sum_of(loss() * make_tensor(dy)); });
}

// A norm whose output both losses read: the label's through the head in pieces, the teacher's
// on the logits of a matmul with the same weights.
void test_together() {
    const int64_t R = 6, D = 16, V = 21;
    Value x = leaf(normal(R * D, 31), {R, D}, "x"), w = leaf(normal(V * D, 32, 0.4f), {V, D}, "w"),
          wt = leaf(normal(D * V, 33, 0.4f), {D, V}, "wt");
    nn::LayerNorm norm(D);
    const Indices labels = Indices::from_host({3, 20, -1, 0, 7, 7}, {R});
    const Indices index = Indices::from_host({1, 2, 3, 4, 5, 6, -1, -1, 9, 10, 11, -1}, {R, 2});
    const Tensor teacher = Tensor::from_host_f32(normal(2 * R, 34), {R, 2});
    auto losses = [&](Value& a, Value& b) {
        Value h = norm(x);
        a = linear_cross_entropy(h, w, labels);
        b = distill_topk(matmul(h, wt), index, teacher, 2.0f);
    };
    auto f = [&] {
        Value c, d;
        losses(c, d);
        return sum_of(c) + sum_of(d);
    };
    Value a, b, c, d;
    losses(a, b);
    backward(a);
    losses(c, d);  // a graph of its own: backward adds to the leaves' gradients
    backward(d, nullptr, true);
    check_grad("norm + both losses: dx", x, f);
    check_grad("norm + both losses: dgamma", norm.gamma, f);
    check_grad("norm + both losses: dbeta", norm.beta, f);
    check_grad("norm + both losses: dw of the head", w, f);
    check_grad("norm + both losses: dw of the logits", wt, f);
}

void test_refusals() {
    Value x = leaf(normal(24, 41), {2, 12}, "x"), w = leaf(normal(36, 42), {3, 12}, "w"),
          g = leaf(normal(12, 43), {12}, "g"), b = leaf(normal(12, 44), {12}, "b");
    const Indices two = Indices::from_host({0, 1}, {2}), three = Indices::from_host({0, 1, 2}, {3});
    const Tensor t = Tensor::from_host_f32({1.0f, 2.0f}, {2, 1});
    const Indices i21 = Indices::from_host({0, 1}, {2, 1});
    std::vector<uint16_t> bits(24, 0);
    Value xb = make_tensor(Tensor::from_host(bits.data(), {2, 12}, Dtype::BFloat16), "xb");
    report("layer_norm refuses wrong shapes, shared nodes and mixed dtypes",
           throws([&] { layer_norm(x, w, b); }) && throws([&] { layer_norm(x, g, g); }) &&
               throws([&] { layer_norm(xb, g, b); }) && throws([&] { layer_norm(x, Value(), b); }));
    report("linear_cross_entropy refuses wrong shapes, dtypes and missing labels",
           throws([&] { linear_cross_entropy(x, w, three); }) &&
               throws([&] { linear_cross_entropy(x, g, two); }) &&
               throws([&] { linear_cross_entropy(x, x, two); }) &&
               throws([&] { linear_cross_entropy(xb, w, two); }) &&
               throws([&] { linear_cross_entropy(x, w, Indices()); }));
    Value wb = make_tensor(Tensor::from_host(bits.data(), {2, 12}, Dtype::BFloat16), "wb");
    report("linear_cross_entropy refuses bf16 widths that are no multiple of 8",
           throws([&] { linear_cross_entropy(xb, wb, two); }));
    report("distill_topk refuses wrong shapes and temperatures",
           throws([&] { distill_topk(x, two, t); }) && throws([&] { distill_topk(x, i21, Tensor()); }) &&
               throws([&] { distill_topk(x, i21, Tensor::from_host_f32({1.0f}, {1, 1})); }) &&
               throws([&] { distill_topk(x, i21, t, 0.0f); }));
    report("the losses have no forward-mode rule and say so",
           throws([&] { jvp(linear_cross_entropy(x, w, two), {{x.node.get(), x.val()}}); }) &&
               throws([&] { jvp(distill_topk(x, i21, t), {{x.node.get(), x.val()}}); }));
    report("Indices refuses a wrong element count", throws([&] { Indices::from_host({1}, {2}); }));
}

void test_empty_batch() {
    Value x = leaf({}, {0, 12}, "x"), w = leaf(normal(36, 51), {3, 12}, "w"),
          g = leaf(normal(12, 52), {12}, "g"), b = leaf(normal(12, 53), {12}, "b");
    Value h = layer_norm(x, g, b);
    Value l = linear_cross_entropy(h, w, Indices::from_host({}, {0}));
    backward(l);
    bool zero = true;
    for (float v : w.grad().to_host_f32()) zero = zero && v == 0.0f;
    for (float v : g.grad().to_host_f32()) zero = zero && v == 0.0f;
    report("an empty batch gives zero gradients", l.val().numel() == 0 && zero);
}

// Forward and backward of all three captured and replayed on new inputs and labels, with an eager
// graph of the same leaves alive through the capture, and eager work between the replays.
void test_capture(Dtype dt) {
    const int64_t R = 96, D = 64, V = 700;
    auto tensor = [&](const std::vector<float>& v, std::vector<int64_t> shape, bool req = true) {
        Tensor t;
        if (dt == Dtype::Float32) {
            t = Tensor::from_host_f32(v, shape);
        } else {
            std::vector<uint16_t> bits(v.size());
            for (size_t i = 0; i < v.size(); ++i) {
                uint32_t u;
                std::memcpy(&u, &v[i], 4);
                bits[i] = static_cast<uint16_t>(u >> 16);
            }
            t = Tensor::from_host(bits.data(), shape, dt);
        }
        t.set_requires_grad(req);
        return t;
    };
    auto labels_of = [&](uint64_t seed) {
        std::mt19937_64 eng(seed);
        std::vector<int64_t> v(R);
        for (int64_t& l : v) l = static_cast<int64_t>(eng() % (V + V / 4)) - V / 4;
        return v;
    };
    GraphRunner runner(size_t(256) << 20);
    StreamGuard guard(runner.get_stream());
    const std::vector<float> gv = normal(D, 61), bv = normal(D, 62), wv = normal(V * D, 63, 0.3f);
    Tensor xt = tensor(normal(R * D, 60), {R, D});
    Indices lab = Indices::from_host(labels_of(1), {R});
    std::vector<int64_t> cols = labels_of(2);
    const Indices index = Indices::from_host(cols, {R, 1});
    const Tensor teacher = Tensor::from_host_f32(normal(R, 64), {R, 1});
    Tensor seed = Tensor::from_host_f32(normal(R, 65), {R, 1});
    Value x = make_tensor(xt, "x"), g = make_tensor(tensor(gv, {D}), "g"),
          b = make_tensor(tensor(bv, {D}), "b"), w = make_tensor(tensor(wv, {V, D}), "w");
    Value eager = linear_cross_entropy(layer_norm(x, g, b), w, lab);  // lives on
    Value z = make_tensor(tensor(normal(R * V, 66), {R, V}), "z");
    runner.begin_capture();
    Value l = linear_cross_entropy(layer_norm(x, g, b), w, lab);
    Value d = distill_topk(z, index, teacher, 2.0f);
    backward(l, &seed);
    backward(d, &seed);
    runner.end_capture();
    bool same = true;
    for (int rep = 0; rep < 3; ++rep) {
        xt.copy_from(tensor(normal(R * D, 70 + rep), {R, D}));
        lab.set_from_host(labels_of(80 + rep));
        Value ge = make_tensor(tensor(gv, {D}), "ge"), be = make_tensor(tensor(bv, {D}), "be"),
              we = make_tensor(tensor(wv, {V, D}), "we"),
              xe = make_tensor(tensor(normal(R * D, 70 + rep), {R, D}), "xe"),
              ze = make_tensor(tensor(normal(R * V, 66), {R, V}), "ze");
        Value le = linear_cross_entropy(layer_norm(xe, ge, be), we, lab);
        Value de = distill_topk(ze, index, teacher, 2.0f);
        backward(le, &seed);
        backward(de, &seed);
        if (!runner.replay()) same = false;
        (void)hipStreamSynchronize(runner.get_stream());
        same = same && l.val().to_host_f32() == le.val().to_host_f32() &&
               d.val().to_host_f32() == de.val().to_host_f32() &&
               x.grad().to_host_f32() == xe.grad().to_host_f32() &&
               g.grad().to_host_f32() == ge.grad().to_host_f32() &&
               b.grad().to_host_f32() == be.grad().to_host_f32() &&
               w.grad().to_host_f32() == we.grad().to_host_f32() &&
               z.grad().to_host_f32() == ze.grad().to_host_f32();
    }
    backward(eager, &seed);  // the graph from before the capture still runs
    report(dt == Dtype::Float32 ? "replays on new inputs and labels == eager (fp32)"
                                : "replays on new inputs and labels == eager (bf16)",
           same, "arena bytes used " + std::to_string(runner.arena_bytes_used()));
}

}  // namespace

int main() {
    try {
        test_layer_norm();
        test_cross_entropy();
        test_distill();
        test_together();
        test_refusals();
        test_empty_batch();
        test_capture(Dtype::Float32);
        test_capture(Dtype::BFloat16);
    } catch (const std::exception& e) {
        report("no exception", false, e.what());
    }
    std::printf("%d failure(s)\n", g_failures);
    return g_failures;
}
