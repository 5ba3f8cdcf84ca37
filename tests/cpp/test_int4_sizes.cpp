// bt::pack_int4's sizes without a GPU: what is refused leaves `packed` as it is, and no width passes an int. Tensors are views of addresses that nothing reads.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>

#include "attention_ops.h"

using namespace bdamd;

int main() {
    int failures = 0;
    auto at = [](std::uintptr_t a) { return reinterpret_cast<void*>(a); };
    const struct { int rows, cols; const char* said; } cases[] = {
        {20, 64, "multiples of 8"},                    // out_features
        {24, 66, "multiples of 8"},                    // in_features 132
        {16, 1 << 27, "in_features"},                  // a block's row of 2^31 bytes
        {16, (1 << 29) - 4, "in_features"},
        {16, (1 << 30) + 4, "in_features"},            // in_features past an int
        {0, 64, "in_features / 2"}, {16, 0, "in_features / 2"}};
    for (const auto& c : cases) {
        const Tensor q = Tensor::view(Device::GPU, at(1ul << 46), c.rows, c.cols, Dtype::INT8);
        Tensor packed = Tensor::view(Device::GPU, at(1ul << 45), 1 << 20, 1 << 11, Dtype::FP32);
        std::string said;
        try { bt::pack_int4(q, packed); } catch (const std::runtime_error& e) { said = e.what(); }
        if (said.find("pack_int4") == std::string::npos || said.find(c.said) == std::string::npos || packed.rows != 1 << 20 || packed.cols != 1 << 11 || packed.dtype != Dtype::FP32) {
            std::printf("q %d x %d: packed %d x %d, \"%s\"\n", c.rows, c.cols, packed.rows, packed.cols, said.c_str());
            ++failures;
        }
    }
    std::printf(failures ? "test_int4_sizes: %d failures\n" : "test_int4_sizes: OK\n", failures);
    return failures != 0;
}
