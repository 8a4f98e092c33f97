// Host-only check of the paged cache's C++ wrappers (no GPU needed): an invalid-argument return becomes ROCmKernels::HipError with
// hipErrorInvalidValue, and the workspace size is returned. Prints one line per case; exit code = failures.
#include <ROCmKernels/Kernels/Cache/KeyValueCache.hpp>

#include <cstdio>
#include <functional>

namespace {
int failures = 0;

void expect_invalid(const char *name, const std::function<void()> &call) {
    try {
        call();
        std::printf("FAIL %s: no exception\n", name);
        ++failures;
    } catch (const ROCmKernels::HipError &error) {
        const bool ok = error.Status() == hipErrorInvalidValue;
        std::printf("%s %s: %s\n", ok ? "ok" : "FAIL", name, error.what());
        failures += ok ? 0 : 1;
    }
}
} // namespace

int main() {
    using namespace ROCmKernels::Kernels;
    const Strides s{0, 0, 0};
    alignas(16) float dummy[4] = {};
    const int numbers[4] = {};
    const KeyValueCache cache{dummy, dummy, dummy, 1, 16, 2, 32};
    const KeyValueCache odd{dummy, dummy, dummy, 1, 17, 2, 32};
    const CacheSequences one{numbers, numbers, numbers, 1, 1, 1, 1}, many{numbers, numbers, numbers, 1, 1, 4096, 4096};
    expect_invalid("CacheAppend null k", [&] { CacheAppend(nullptr, dummy, nullptr, nullptr, nullptr, nullptr, cache, one, 0, 0, s, s, s, s, s, s, DType::BFloat16); });
    expect_invalid("CacheAppend cos without sin", [&] { CacheAppend(dummy, dummy, nullptr, dummy, nullptr, nullptr, cache, one, 0, 1, s, s, s, s, s, s, DType::Float32); });
    expect_invalid("CacheForward odd page", [&] { CacheForward(dummy, odd, one, dummy, nullptr, 2, 0, -1, 0, s, s, DType::Float16, nullptr, 0); });
    expect_invalid("CacheForward no workspace", [&] { CacheForward(dummy, cache, many, dummy, nullptr, 2, 0, -1, 0, s, s, DType::Float16, nullptr, 0); });
    expect_invalid("CacheWorkspace heads", [&] { (void)CacheWorkspace(cache, one, 3, 0, DType::Float32); });
    if (CacheWorkspace(cache, one, 2, 0, DType::Float32) != 0 || CacheWorkspace(cache, many, 2, 0, DType::Float32) == 0) {
        std::printf("FAIL CacheWorkspace sizes\n");
        ++failures;
    }
    std::printf("%d failure(s)\n", failures);
    return failures;
}
