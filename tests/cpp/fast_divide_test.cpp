// Division by one product (ilgpu_b200/csrc/fast_divide.cuh) against the processor's own: all quotients around the multiples of a
// divisor where a wrong one would show, for all small divisors, those around powers of two and many others.
#include <cstdio>
#include <random>

#include "fast_divide.cuh"

static long g_failures = 0;

static void check(uint32_t d, uint32_t q) {
    const b200alg::FastDivide by(d);
    if (by(q) != q / d && ++g_failures < 20) std::printf("FAILED %u / %u = %u, not %u\n", q, d, by(q), q / d);
}

static void check(uint32_t d) {
    constexpr uint32_t kMost = (1u << 31) - 1;
    static std::mt19937 rng(1);
    check(d, 0u), check(d, kMost);
    const uint32_t whole = kMost / d;  // quotients there are
    auto around = [&](uint32_t multiple) {
        const uint64_t q = (uint64_t)multiple * d;
        for (int64_t at = (int64_t)q - 1; at <= (int64_t)q + 1; ++at)
            if (at >= 0 && at <= (int64_t)kMost) check(d, (uint32_t)at);
    };
    for (uint32_t i = 0; i < 3 && i <= whole; ++i) around(i), around(whole - i);
    for (int i = 0; i < 20; ++i) around(rng() % (whole + 1u));
}

int main() {
    for (uint32_t d = 1; d <= 100000; ++d) check(d);
    for (int s = 1; s <= 31; ++s)
        for (int64_t by = -40; by <= 40; ++by) {
            const int64_t d = ((int64_t)1 << s) + by;
            if (d >= 1 && d <= (int64_t)1 << 31) check((uint32_t)d);
        }
    std::mt19937 rng(2);
    for (int i = 0; i < 1000000; ++i) check((rng() >> (rng() % 31)) % (1u << 31) + 1u);
    for (uint32_t d : {1u, 2u, 3u, 7u, 115u, 1357u, 65535u, 65537u, (1u << 30) + 1u})  // every dividend of a stretch
        for (uint32_t q = 0; q < 3000000; ++q) check(d, q), check(d, (1u << 31) - 1u - q);
    if (g_failures) std::printf("%ld failures\n", g_failures);
    return g_failures != 0;
}
