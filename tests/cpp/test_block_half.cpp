// The 8-bit rows and the linear layer with an epilogue through the C++20 host layer: an MLP half of a block (norm -> first product -> rows ->
// second product with the residual) in bf16, each step against double arithmetic on what the step before stored; and refusals.
//   test_block_half --cpu   refusals that need no GPU
//   test_block_half         the GPU run
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
static Tensor normal_bf16(uint64_t seed, int rows, int cols) {
    std::vector<float> x(std::max<size_t>(16, static_cast<size_t>(rows) * cols));
    orc_torch_randn_f32(seed, x.size(), x.data());
    std::vector<uint16_t> bits(x.size());
    orc_f32_to_bf16_bits(x.data(), x.size(), bits.data());
    return Tensor::from_host(bits.data(), rows, cols, Dtype::BF16);
}
static std::vector<double> values(const Tensor& t) {
    const std::vector<std::uint8_t> raw = t.to_host_bytes();
    std::vector<double> v(t.size());
    if (t.dtype == Dtype::INT8) {
        for (size_t i = 0; i < v.size(); ++i) v[i] = static_cast<signed char>(raw[i]);
    } else if (t.dtype == Dtype::FP32) {
        for (size_t i = 0; i < v.size(); ++i) { float f; std::memcpy(&f, &raw[4 * i], 4); v[i] = f; }
    } else {
        std::vector<float> f(v.size());
        orc_bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(raw.data()), f.size(), f.data());
        std::copy(f.begin(), f.end(), v.begin());
    }
    return v;
}
// a weight as 8-bit rows: what quantize_rows_int8 makes of a bf16 one
struct Weight { Tensor q, scales; };
static Weight weight(uint64_t seed, int out, int in) {
    Weight w;
    bt::quantize_rows_int8(normal_bf16(seed, out, in), w.q, w.scales);
    return w;
}
static double gelu(double v) { return 0.5 * v * std::erfc(-v / std::sqrt(2.0)); }
// One rounding to bf16 (2^-8 of the value) and FP32 steps around an exact sum: 2e-5 for the GELU, 8 roundings of what is joined
static void check_linear(const char* what, const Tensor& x, const Tensor& xs, const Weight& w, const Tensor* bias, bool act, const Tensor* res, const Tensor& y) {
    const auto vx = values(x), vs = values(xs), vw = values(w.q), ws = values(w.scales), vy = values(y);
    const auto vb = bias ? values(*bias) : std::vector<double>(w.q.rows, 0.0), vr = res ? values(*res) : std::vector<double>(vy.size(), 0.0);
    int bad = 0;
    for (int r = 0; r < x.rows; ++r)
        for (int n = 0; n < w.q.rows; ++n) {
            double s = 0;
            for (int k = 0; k < x.cols; ++k) s += vx[static_cast<size_t>(r) * x.cols + k] * vw[static_cast<size_t>(n) * x.cols + k];
            const double scaled = s * vs[r] * ws[n], v = scaled + vb[n], a = act ? gelu(v) : v;
            const size_t at = static_cast<size_t>(r) * w.q.rows + n;
            const double ref = a + vr[at], joined = std::fabs(scaled) + std::fabs(vb[n]) + std::fabs(vr[at]);
            if (!(std::fabs(vy[at] - ref) <= std::fabs(ref) / 256 + 8 * joined / 16777216 + 2e-5 * std::fabs(a) + 1e-30)) ++bad;
        }
    if (bad) std::printf("%s: %d values are off\n", what, bad);
    CHECK(bad == 0);
}

static void test_refusals() {
    Tensor x, w, y;
    x.device = Device::CPU;
    x.rows = 2; x.cols = 64; x.dtype = Dtype::BF16;
    CHECK(throws_with([&] { bt::linear_act(x, nullptr, x, nullptr, nullptr, bt::Activation::None, nullptr, y); }, "linear_act: tensor is on the CPU"));
    CHECK(throws_with([&] { bt::quantize_rows_int8(x, y, w); }, "quantize_rows_int8: tensor is on the CPU"));
    CHECK(throws_with([&] { bt::add_rms_norm(x, nullptr, x, 1e-6f, y, w); }, "add_rms_norm: tensor is on the CPU"));
}

static void test_half(int rows) {
    const int D = 320, F = 1280;
    Tensor x = normal_bf16(11 + rows, rows, D), r = normal_bf16(12 + rows, rows, D), gain = normal_bf16(13, 1, D), b1 = normal_bf16(14, 1, F), b2 = normal_bf16(15, 1, D);
    Weight w1 = weight(16, F, D), w2 = weight(17, D, F);
    Tensor h, q, s, u, q2, s2, y, n;
    bt::add_rms_norm_int8(x, &r, gain, 1e-6f, h, q, s);
    bt::add_rms_norm(x, &r, gain, 1e-6f, h, n);
    const auto vx = values(x), vr = values(r), vg = values(gain), vh = values(h), vq = values(q), vs = values(s), vn = values(n);
    for (int i = 0; i < rows; ++i) {
        double ss = 0, most = 0;
        for (int c = 0; c < D; ++c) {
            const size_t at = static_cast<size_t>(i) * D + c;
            CHECK(std::fabs(vh[at] - (vx[at] + vr[at])) <= std::fabs(vx[at] + vr[at]) / 256);
            ss += vh[at] * vh[at];
            most = std::max(most, std::fabs(vh[at] * vg[c]));
        }
        const double inv = 1 / std::sqrt(ss / D + 1e-6);
        CHECK(std::fabs(vs[i] - most * inv / 127) <= 1e-5 * vs[i]);
        for (int c = 0; c < D; ++c) {
            const size_t at = static_cast<size_t>(i) * D + c;
            CHECK(vq[at] == std::nearbyint(127 * vh[at] * vg[c] / most));
            CHECK(std::fabs(vn[at] - vh[at] * vg[c] * inv) <= std::fabs(vn[at]) * (1.0 / 256 + 1e-5));
        }
    }
    bt::linear_act(q, &s, w1.q, &w1.scales, &b1, bt::Activation::Gelu, nullptr, u);
    CHECK(u.dtype == Dtype::BF16 && u.rows == rows && u.cols == F);
    check_linear("first product", q, s, w1, &b1, true, nullptr, u);
    bt::quantize_rows_int8(u, q2, s2);
    bt::linear_act(q2, &s2, w2.q, &w2.scales, &b2, bt::Activation::None, &h, y);
    check_linear("second product", q2, s2, w2, &b2, false, &h, y);
    // into the residual itself
    bt::linear_act(q2, &s2, w2.q, &w2.scales, &b2, bt::Activation::None, &h, h);
    CHECK(h.to_host_bytes() == y.to_host_bytes());
    // an output that is an operand: refused before anything is resized
    CHECK(throws_with([&] { bt::add_rms_norm_int8(x, &r, gain, 1e-6f, h, x, s); }, "out is another operand"));
    CHECK(throws_with([&] { bt::add_rms_norm_int8(x, &r, gain, 1e-6f, q, q, s); }, "sum is another operand"));
    CHECK(throws_with([&] { bt::add_rms_norm(x, &r, gain, 1e-6f, h, gain); }, "out is another operand"));
    CHECK(throws_with([&] { bt::quantize_rows_int8(u, u, s2); }, "out is another operand"));
    CHECK(throws_with([&] { bt::linear_act(u, nullptr, w2.q, &w2.scales, nullptr, bt::Activation::None, nullptr, u); }, "Y is another operand"));
    CHECK(values(x) == vx && gain.cols == D && u.cols == F);
    // 16-bit outputs in place
    Tensor x1 = normal_bf16(11 + rows, rows, D), r1 = normal_bf16(12 + rows, rows, D);
    bt::add_rms_norm(x1, &r1, gain, 1e-6f, r1, x1);
    CHECK(values(r1) == vh && values(x1) == vn);
    CHECK(throws_with([&] { bt::linear_act(q2, &s2, w2.q, nullptr, &b2, bt::Activation::None, &h, y); }, "INT8 weights"));
    CHECK(throws_with([&] { bt::linear_act(q2, &s2, w1.q, &w1.scales, nullptr, bt::Activation::None, &h, y); }, "same columns"));
    CHECK(throws_with([&] { bt::linear_act(q2, &s, w2.q, &w1.scales, &b2, bt::Activation::None, &h, y); }, "w_scales"));
}

int main(int argc, char** argv) {
    test_refusals();
    if (argc < 2 || std::strcmp(argv[1], "--cpu") != 0)
        for (int rows : {1, 33}) test_half(rows);
    if (g_failures) { std::printf("test_block_half: %d failures\n", g_failures); return 1; }
    std::printf("test_block_half: OK\n");
    return 0;
}
