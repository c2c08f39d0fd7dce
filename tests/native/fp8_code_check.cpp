// fp8_act_code_short (objeta_amd/csrc/quant_rules.hpp) against fp8_act_code on every float, at a
// scale of 1 and at the factor 0 of a block that holds an infinity. Compiled by
// tests/test_fp8_code_cpu.py with g++ -fopenmp; prints the number of floats with different codes.
#include <cstdint>
#include <cstdio>

#include "quant_rules.hpp"

int main() {
    uint64_t n = 0;
#pragma omp parallel for reduction(+ : n) schedule(static)
    for (int64_t u = 0; u < (int64_t(1) << 32); ++u) {
        const float x = objeta::rules::u2f(static_cast<uint32_t>(u));
        n += objeta::rules::fp8_act_code(x, 1.0f) != objeta::rules::fp8_act_code_short(x, 1.0f);
        n += objeta::rules::fp8_act_code(x, 0.0f) != objeta::rules::fp8_act_code_short(x, 0.0f);
    }
    std::printf("%llu\n", static_cast<unsigned long long>(n));
    return 0;
}
