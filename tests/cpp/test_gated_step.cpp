// The step between two blocks and the linear layer with 4-bit weights through the C++20 host layer: the MLP half of a block whose weights have 4 bits (modulated
// norm -> product with GELU -> product -> gated residual with the next norm) in bf16, each step against double arithmetic on what the step before stored; and
// refusals.
//   test_gated_step --cpu   refusals that need no GPU
//   test_gated_step         the GPU run
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "attention_ops.h"

extern "C" {
int orc_torch_randn_f32(uint64_t seed, size_t n, float* out);
void orc_f32_to_bf16_bits(const float* x, size_t n, uint16_t* out);
void orc_bf16_bits_to_f32(const uint16_t* x, size_t n, float* out);
}

using namespace bdamd;
using bt::Activation;
using bt::Norm;

static int g_failures = 0;
#define CHECK(cond)                                                              \
    do {                                                                         \
        if (!(cond)) { std::printf("CHECK failed %s:%d: %s\n", __FILE__, __LINE__, #cond); ++g_failures; } \
    } while (0)

template <typename F>
static bool throws_with(F&& f, const char* needle) {
    try { f(); } catch (const std::runtime_error& e) { return std::strstr(e.what(), needle) != nullptr; }
    return false;
}
static Tensor normal_bf16(uint64_t seed, int rows, int cols, float times = 1.f) {
    std::vector<float> x(std::max<size_t>(16, static_cast<size_t>(rows) * cols));
    orc_torch_randn_f32(seed, x.size(), x.data());
    for (float& v : x) v *= times;
    std::vector<uint16_t> bits(x.size());
    orc_f32_to_bf16_bits(x.data(), x.size(), bits.data());
    return Tensor::from_host(bits.data(), rows, cols, Dtype::BF16);
}
static std::vector<double> values(const Tensor& t) {
    const std::vector<std::uint8_t> raw = t.to_host_bytes();
    std::vector<float> f(t.size());
    orc_bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(raw.data()), f.size(), f.data());
    return std::vector<double>(f.begin(), f.end());
}

// 4-bit weights and what they stand for
struct Weight {
    int out, in, group;
    Tensor packed, scales, zeros;
    std::vector<double> w;      // (out, in)
    Weight(unsigned seed, int n, int k, int g, bool with_zeros) : out(n), in(k), group(g), w(static_cast<size_t>(n) * k) {
        auto next = [&] { return (seed = seed * 1664525u + 1013904223u) >> 8; };
        const int groups = (k + g - 1) / g;
        std::vector<std::uint8_t> q(static_cast<size_t>(n) * k / 2), z(static_cast<size_t>(groups) * n, 8);
        for (auto& v : q) v = static_cast<std::uint8_t>(next());
        if (with_zeros) {
            for (auto& v : z) v = static_cast<std::uint8_t>(next() % 16);
            zeros = Tensor::from_host(z.data(), groups, n, Dtype::INT8);
        }
        scales = normal_bf16(seed, groups, n, 1.f / (4.6f * std::sqrt(static_cast<float>(k))));
        const auto s = values(scales);
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < k; ++j) {
                const size_t at = static_cast<size_t>(i) * k + j, of = static_cast<size_t>(j / g) * n + i;
                w[at] = ((q[at / 2] >> (at % 2 * 4) & 15) - z[of]) * s[of];
            }
        bt::pack_int4(Tensor::from_host(q.data(), n, k / 2, Dtype::INT8), packed);
    }
    const Tensor* zero_points() const { return zeros.size() ? &zeros : nullptr; }
};
static double gelu(double v) { return 0.5 * v * std::erfc(-v / std::sqrt(2.0)); }
// One rounding to bf16 (2^-8 of the value), 2e-5 for an activation, and FP32 sums: a group's start at -z sum(x), up to 2 (128 + 4) additions for a block's 128 elements
// or fewer, each off by at most 2^-23 (the matrix instructions may cut off) of sum (q + 2 z) |x| <= 45 sum |x|; groups, blocks and the bias then meet with three
// roundings each
static void check_linear(const char* what, const Tensor& x, const Weight& w, const Tensor* bias, bool act, const Tensor* res, const Tensor& y) {
    CHECK(y.dtype == Dtype::BF16 && y.rows == x.rows && y.cols == w.out);
    const auto vx = values(x), vy = values(y), vs = values(w.scales);
    const auto vb = bias ? values(*bias) : std::vector<double>(w.out, 0.0), vr = res ? values(*res) : std::vector<double>(vy.size(), 0.0);
    int bad = 0;
    for (int r = 0; r < x.rows; ++r)
        for (int n = 0; n < w.out; ++n) {
            double s = vb[n], terms = std::fabs(vb[n]);
            for (int k = 0; k < w.in; ++k) {
                const double v = vx[static_cast<size_t>(r) * w.in + k];
                s += v * w.w[static_cast<size_t>(n) * w.in + k];
                terms += 45 * std::fabs(v * vs[static_cast<size_t>(k / w.group) * w.out + n]);
            }
            const size_t at = static_cast<size_t>(r) * w.out + n;
            const double ref = (act ? gelu(s) : s) + vr[at], sums = (4 * (128 + 4) + 3 * (w.scales.rows + w.in / 128 + 11)) / 16777216.0 * terms;
            if (!(std::fabs(vy[at] - ref) <= std::fabs(ref) / 256 + 1.13 * sums + 2e-5 * std::fabs(s) + std::fabs(vr[at]) / 8388608)) ++bad;      // (GELU's slope is at most 1.13)
        }
    if (bad) std::printf("%s: %d values are off\n", what, bad);
    CHECK(bad == 0);
}
static std::vector<double> normed(const std::vector<double>& v, int cols, bool layer, double eps) {
    std::vector<double> o(v.size());
    for (size_t r = 0; r < v.size() / cols; ++r) {
        double mean = 0, ss = 0;
        for (int c = 0; c < cols && layer; ++c) mean += v[r * cols + c] / cols;
        for (int c = 0; c < cols; ++c) ss += (v[r * cols + c] - mean) * (v[r * cols + c] - mean);
        for (int c = 0; c < cols; ++c) o[r * cols + c] = (v[r * cols + c] - mean) / std::sqrt(ss / cols + eps);
    }
    return o;
}
// One rounding to bf16, and 1e-5 of the terms for the FP32 statistics and factors (24 roundings and a sum of `cols` squares in partial sums: < 100 * 2^-24)
static void check_step(const char* what, const Tensor& x, const bt::GateAddNorm& p, const Tensor* sum, const Tensor* out) {
    const int cols = x.cols;
    const auto vx = values(x);
    auto at = [&](const Tensor* t, const std::vector<double>& v, size_t i, double none) {
        if (t == nullptr) return none;
        const size_t r = i / cols, per = t->rows > 1 ? x.rows / t->rows : x.rows;
        return v[r / per * cols + i % cols];
    };
    auto of = [](const Tensor* t) { return t ? values(*t) : std::vector<double>(); };
    const auto vg = of(p.gate), vp = of(p.post_gain), vn = of(p.gain), vs = of(p.scale), vt = of(p.shift);
    std::vector<double> h = vx;
    int bad = 0;
    if (p.branch) {
        auto b = values(*p.branch);
        if (p.post_norm != Norm::None) b = normed(b, cols, p.post_norm == Norm::Layer, p.post_eps);
        const auto vh = values(*sum);
        for (size_t i = 0; i < h.size(); ++i) {
            const double t = at(p.gate, vg, i, 1) * b[i] * at(p.post_gain, vp, i, 1), x0 = static_cast<double>(p.residual_scale) * vx[i];
            h[i] = x0 + t;
            if (!(std::fabs(vh[i] - h[i]) <= std::fabs(h[i]) / 256 + 1e-5 * (std::fabs(t) + std::fabs(x0)))) ++bad;
        }
        h = vh;      // (the norm is of what is stored)
    }
    if (out) {
        const auto vo = values(*out), n = normed(h, cols, p.norm == Norm::Layer, p.eps);
        for (size_t i = 0; i < h.size(); ++i) {
            const double t = n[i] * at(p.gain, vn, i, 1) * (1 + at(p.scale, vs, i, 0)), ref = t + at(p.shift, vt, i, 0);
            if (!(std::fabs(vo[i] - ref) <= std::fabs(ref) / 256 + 1e-5 * (std::fabs(t) + std::fabs(at(p.shift, vt, i, 0)) + std::fabs(at(p.gain, vn, i, 1) * (1 + std::fabs(at(p.scale, vs, i, 0))))))) ++bad;
        }
    }
    if (bad) std::printf("%s: %d values are off\n", what, bad);
    CHECK(bad == 0);
}

static void test_refusals() {
    Tensor x, y;
    x.device = Device::CPU;
    x.rows = 2; x.cols = 64; x.dtype = Dtype::BF16;
    CHECK(throws_with([&] { bt::gate_add_norm(x, {}, nullptr, &y); }, "gate_add_norm: tensor is on the CPU"));
    CHECK(throws_with([&] { bt::pack_int4(x, y); }, "pack_int4: tensor is on the CPU"));
    CHECK(throws_with([&] { bt::linear_int4(x, x, x, nullptr, 64, nullptr, Activation::None, nullptr, y); }, "linear_int4: tensor is on the CPU"));
}

static void test_half(int images, int per, int group, bool zeros) {
    const int D = 320, F = 1288, rows = images * per;
    const Tensor x = normal_bf16(21 + rows, rows, D), mod[3] = {normal_bf16(22, images, D, 0.5f), normal_bf16(23, images, D, 0.5f), normal_bf16(24, images, D)};
    const Tensor gain = normal_bf16(25, 1, D), b1 = normal_bf16(26, 1, F), b2 = normal_bf16(27, 1, D), each = normal_bf16(28, rows, D);
    const Weight w1(29, F, D, group, zeros), w2(30, D, F, group, zeros);
    Tensor n, u, v, h, o;
    bt::GateAddNorm first;
    first.norm = Norm::Layer; first.scale = &mod[0]; first.shift = &mod[1];
    bt::gate_add_norm(x, first, nullptr, &n);
    check_step("modulated norm", x, first, nullptr, &n);
    bt::linear_int4(n, w1.packed, w1.scales, w1.zero_points(), group, &b1, Activation::Gelu, nullptr, u);
    check_linear("first product", n, w1, &b1, true, nullptr, u);
    bt::linear_int4(u, w2.packed, w2.scales, w2.zero_points(), group, &b2, Activation::None, nullptr, v);
    check_linear("second product", u, w2, &b2, false, nullptr, v);
    bt::GateAddNorm next;
    next.branch = &v; next.gate = &mod[2]; next.post_norm = Norm::Rms; next.post_gain = &gain; next.residual_scale = 0.75f;
    next.norm = Norm::Rms; next.gain = &gain; next.shift = &each;
    bt::gate_add_norm(x, next, &h, &o);
    check_step("gated residual and norm", x, next, &h, &o);
    // into the operands: the stream and the branch, a product's residual
    Tensor x1 = normal_bf16(21 + rows, rows, D), v1;
    bt::linear_int4(u, w2.packed, w2.scales, w2.zero_points(), group, &b2, Activation::None, nullptr, v1);
    bt::GateAddNorm in_place = next;
    in_place.branch = &v1;
    bt::gate_add_norm(x1, in_place, &x1, &v1);
    CHECK(x1.to_host_bytes() == h.to_host_bytes() && v1.to_host_bytes() == o.to_host_bytes());
    Tensor y = normal_bf16(21 + rows, rows, D), z;
    bt::linear_int4(u, w2.packed, w2.scales, w2.zero_points(), group, nullptr, Activation::None, &x, z);
    check_linear("product with a residual", u, w2, nullptr, false, &x, z);
    bt::linear_int4(u, w2.packed, w2.scales, w2.zero_points(), group, nullptr, Activation::None, &y, y);
    CHECK(y.to_host_bytes() == z.to_host_bytes());
    // the last block: the sum alone
    bt::GateAddNorm last;
    last.branch = &v; last.gate = &mod[2];
    bt::gate_add_norm(x, last, &h, nullptr);
    check_step("the last sum", x, last, &h, nullptr);
    if (rows < 2) return;
    // refused before anything is resized
    Tensor gain1 = normal_bf16(25, 1, D), short_gate = normal_bf16(5, rows + 1, D);
    bt::GateAddNorm bad = next;
    bad.gate = &short_gate;
    CHECK(throws_with([&] { bt::gate_add_norm(x, bad, &h, &o); }, "gate must hold X's columns"));
    bad = next; bad.gain = &gain1;
    CHECK(throws_with([&] { bt::gate_add_norm(x, bad, &h, &gain1); }, "out is another operand"));
    CHECK(throws_with([&] { bt::gate_add_norm(x, bad, &h, &h); }, "sum is another operand"));
    bad.branch = &u;
    CHECK(throws_with([&] { bt::gate_add_norm(x, bad, &h, &o); }, "the branch must have"));
    CHECK(throws_with([&] { bt::gate_add_norm(x, next, &h, nullptr); }, "gate_add_norm"));      // a norm without an output
    CHECK(throws_with([&] { bt::linear_int4(u, w2.packed, w2.scales, w2.zero_points(), group, nullptr, Activation::None, nullptr, u); }, "Y is another operand"));
    CHECK(throws_with([&] { bt::linear_int4(n, w2.packed, w2.scales, w2.zero_points(), group, nullptr, Activation::None, nullptr, z); }, "scales must be"));
    CHECK(throws_with([&] { bt::linear_int4(u, w1.scales, w2.scales, w2.zero_points(), group, nullptr, Activation::None, nullptr, z); }, "packed weights"));
    CHECK(throws_with([&] { bt::linear_int4(u, w2.packed, w2.scales, &w1.packed, group, nullptr, Activation::None, nullptr, z); }, "zeros must be"));
    CHECK(throws_with([&] { bt::linear_int4(u, w2.packed, w2.scales, w2.zero_points(), 0, nullptr, Activation::None, nullptr, z); }, "scales must be"));
    CHECK(throws_with([&] { bt::linear_int4(u, w2.packed, w2.scales, w2.zero_points(), group, nullptr, Activation::None, &u, z); }, "the residual must have"));
    CHECK(throws_with([&] { bt::pack_int4(u, z); }, "bytes"));
    CHECK(gain1.cols == D && u.cols == F && z.to_host_bytes() == y.to_host_bytes());
}
// a contraction that several work groups share: twice the same bits, also where a larger problem has come between
static void test_shares() {
    const Tensor x = normal_bf16(41, 3, 8192), more = normal_bf16(42, 40, 8192);
    const Weight w(43, 64, 8192, 128, true), wide(44, 640, 8192, 64, false);
    Tensor y, y2, again;
    bt::linear_int4(x, w.packed, w.scales, &w.zeros, 128, nullptr, Activation::None, nullptr, y);
    check_linear("a long contraction", x, w, nullptr, false, nullptr, y);
    bt::linear_int4(more, wide.packed, wide.scales, nullptr, 64, nullptr, Activation::Silu, nullptr, y2);
    bt::linear_int4(x, w.packed, w.scales, &w.zeros, 128, nullptr, Activation::None, nullptr, again);
    CHECK(again.to_host_bytes() == y.to_host_bytes());
}

int main(int argc, char** argv) {
    test_refusals();
    if (argc < 2 || std::strcmp(argv[1], "--cpu") != 0) {
        test_half(1, 1, 128, false);
        test_half(3, 11, 64, true);
        test_half(2, 50, 32, false);
        test_shares();
    }
    if (g_failures) { std::printf("test_gated_step: %d failures\n", g_failures); return 1; }
    std::printf("test_gated_step: OK\n");
    return 0;
}
