// The C++20 host layer's scratch for linear layers whose contraction several work groups share (bt::linear_act): its first allocation, growth, calls that
// need less again, and graphs captured on a scratch that was outgrown since. INT8 rows and weights: the sums are exact, so every call of a problem gives the
// same bits, and those are checked against double arithmetic.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "attention_ops.h"

using namespace bdamd;

static int g_failures = 0;
#define CHECK(cond)                                                              \
    do {                                                                         \
        if (!(cond)) { std::printf("CHECK failed %s:%d: %s\n", __FILE__, __LINE__, #cond); ++g_failures; } \
    } while (0)

struct Problem {
    int M, N, K;
    std::vector<signed char> hx, hw;
    std::vector<float> hxs, hws;
    Tensor x, w, xs, ws, y;
    Problem(int m, int n, int k, unsigned seed) : M(m), N(n), K(k), hx(static_cast<size_t>(m) * k), hw(static_cast<size_t>(n) * k), hxs(m), hws(n) {
        auto next = [&] { return (seed = seed * 1664525u + 1013904223u) >> 8; };
        for (auto& v : hx) v = static_cast<signed char>(static_cast<int>(next() % 255) - 127);
        for (auto& v : hw) v = static_cast<signed char>(static_cast<int>(next() % 255) - 127);
        for (auto& v : hxs) v = (512 + next() % 512) / 65536.f;
        for (auto& v : hws) v = (512 + next() % 512) / 16777216.f;
        x = Tensor::from_host(hx.data(), M, K, Dtype::INT8);
        w = Tensor::from_host(hw.data(), N, K, Dtype::INT8);
        xs = Tensor::from_host(hxs.data(), M, 1, Dtype::FP32);
        ws = Tensor::from_host(hws.data(), N, 1, Dtype::FP32);
        y.resize(M, N, Dtype::BF16);      // (without bias and residual, Y says what type it is)
    }
    void run() { bt::linear_act(x, &xs, w, &ws, nullptr, bt::Activation::None, nullptr, y); }
    size_t scratch() const {
        mi_linear_act_args a;
        std::memset(&a, 0, sizeof(a));
        a.struct_size = sizeof(a);
        a.dtype = MI_DTYPE_BF16;
        a.x = x.data; a.w = w.data; a.y = y.data;
        a.x_scales = static_cast<const float*>(xs.data); a.w_scales = static_cast<const float*>(ws.data);
        a.rows = M; a.out_features = N; a.in_features = K;
        return mi_linear_act_scratch_bytes(&a);
    }
    // one rounding to bf16 (2^-8 of the value), and FP32 roundings of the sum, a product and a multiply-add with nothing
    void check(const char* what) {
        const std::vector<std::uint8_t> raw = y.to_host_bytes();
        int bad = 0;
        for (int r = 0; r < M; r += 1 + M / 16)
            for (int n = r % 3; n < N; n += 1 + N / 64) {
                long s = 0;
                for (int k = 0; k < K; ++k) s += hx[static_cast<size_t>(r) * K + k] * hw[static_cast<size_t>(n) * K + k];
                const double ref = static_cast<double>(s) * hxs[r] * hws[n];
                std::uint16_t half;
                std::memcpy(&half, &raw[2 * (static_cast<size_t>(r) * N + n)], 2);
                const std::uint32_t bits = static_cast<std::uint32_t>(half) << 16;
                float got;
                std::memcpy(&got, &bits, 4);
                if (!(std::fabs(got - ref) <= std::fabs(ref) * (1.0 / 256 + 4.0 / 16777216))) ++bad;
            }
        if (bad) std::printf("%s: %d values are off\n", what, bad);
        CHECK(bad == 0);
    }
};

static void clear(Problem& p) {
    const std::vector<std::uint8_t> zeros(p.y.bytes(), 0);
    CHECK(mi_memcpy_h2d(p.y.data, zeros.data(), zeros.size()) == 0);
}

int main() {
    hipStream_t stream;
    CHECK(hipStreamCreate(&stream) == hipSuccess);
    CHECK(mi_set_stream(stream) == 0);
    Problem small(46, 368, 32000, 1), middle(70, 1000, 32768, 2), large(333, 1000, 32768, 3);
    CHECK(small.scratch() > 0 && middle.scratch() > small.scratch() && large.scratch() > 2 * middle.scratch());
    small.run();      // the first allocation
    CHECK(mi_stream_synchronize(stream) == 0);
    small.check("first call");
    const std::vector<std::uint8_t> want = small.y.to_host_bytes();

    hipGraph_t graph;
    hipGraphExec_t exec;
    CHECK(hipStreamBeginCapture(stream, hipStreamCaptureModeThreadLocal) == hipSuccess);
    small.run();
    CHECK(hipStreamEndCapture(stream, &graph) == hipSuccess && hipGraphInstantiate(&exec, graph, nullptr, nullptr, 0) == hipSuccess);

    // growth twice, what is allocated in between taken by others, and the captured call again behind each
    std::vector<Tensor> others;
    for (Problem* p : {&middle, &large, &middle, &small}) {
        p->run();
        CHECK(mi_stream_synchronize(stream) == 0);
        p->check("after growth");
        for (int i = 0; i < 4; ++i) {
            std::vector<float> ones(small.scratch() / 4, 1.f);
            others.push_back(Tensor::from_host(ones.data(), 1, static_cast<int>(ones.size()), Dtype::FP32));
        }
        clear(small);
        CHECK(hipGraphLaunch(exec, stream) == hipSuccess && mi_stream_synchronize(stream) == 0);
        CHECK(small.y.to_host_bytes() == want);
        for (const Tensor& t : others) {
            const auto raw = t.to_host_bytes();
            const float one = 1.f;
            bool whole = true;
            for (size_t i = 0; i < raw.size(); i += 4) whole = whole && std::memcmp(&raw[i], &one, 4) == 0;
            CHECK(whole);
        }
    }
    // another stream has a scratch of its own: both run at once
    hipStream_t second;
    CHECK(hipStreamCreate(&second) == hipSuccess);
    Problem twin(46, 368, 32000, 4);
    for (int i = 0; i < 20; ++i) {
        CHECK(mi_set_stream(stream) == 0);
        small.run();
        CHECK(mi_set_stream(second) == 0);
        twin.run();
    }
    CHECK(mi_stream_synchronize(stream) == 0 && mi_stream_synchronize(second) == 0);
    CHECK(small.y.to_host_bytes() == want);
    twin.check("second stream");
    CHECK(mi_set_stream(nullptr) == 0);
    CHECK(hipGraphExecDestroy(exec) == hipSuccess && hipGraphDestroy(graph) == hipSuccess);
    if (g_failures) { std::printf("test_linear_act_scratch: %d failures\n", g_failures); return 1; }
    std::printf("test_linear_act_scratch: OK\n");
    return 0;
}
