// The operators of a training step through the C++ host mirror (include/ilgpu_algorithms.hpp), against serial loops in
// double on the host, and their argument errors.  All inputs are small whole numbers or powers of two, so that lookup,
// gradient and clipping have to come out exactly.  Exit code 0 = all checks passed.
#include <cmath>
#include <cstdio>
#include <vector>

#include "ilgpu_algorithms.hpp"

using namespace ILGPU;
using namespace ILGPU::Algorithms;

static int g_checks = 0, g_failures = 0;
#define CHECK(cond)                                                                 \
    do {                                                                            \
        ++g_checks;                                                                 \
        if (!(cond)) { ++g_failures; std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); } \
    } while (0)
#define CHECK_THROWS(type, call)                     \
    do {                                             \
        bool thrown = false;                         \
        try { call; } catch (const type &) { thrown = true; } \
        CHECK(thrown);                               \
    } while (0)

template <typename T> std::unique_ptr<MemoryBuffer1D<T>> Upload(const Accelerator &acc, const std::vector<T> &h) {
    auto b = acc.Allocate1D<T>((int64_t)h.size());
    b->CopyFromCPU(h.data());
    return b;
}
template <typename T> std::vector<T> Download(const MemoryBuffer1D<T> &b) {
    std::vector<T> h(b.Length());
    b.CopyToCPU(h.data());
    return h;
}

static void EmbeddingTests(const Accelerator &acc, int n, int rows, int width) {
    AcceleratorStream stream;
    std::vector<__nv_bfloat16> table(rows * width);
    for (size_t i = 0; i < table.size(); ++i) table[i] = __float2bfloat16((float)((int)(i * 7 % 61) - 30));
    std::vector<int64_t> tokens(n);
    for (int i = 0; i < n; ++i) tokens[i] = (int64_t)(i * 13 % (rows + 2)) - 1;  // -1 and rows: none
    auto dtable = Upload(acc, table);
    auto dtokens = Upload(acc, tokens);
    auto out = acc.Allocate1D<float>(n * width), gradient = acc.Allocate1D<float>(rows * width);
    ArrayView2D<__nv_bfloat16> t(dtable->View(), rows, width);
    ArrayView2D<float> o(out->View(), n, width), g(gradient->View(), rows, width);
    CreateEmbedding<__nv_bfloat16, int64_t, float>(acc)(stream, t, dtokens->View(), o, 2.0);
    auto temp = acc.Allocate1D<int>(ComputeEmbeddingGradientTempStorageSize(acc, rows, width, n));
    auto backward = CreateEmbeddingGradient<int64_t, float, float>(acc);
    backward(stream, dtokens->View(), o, g, temp->View(), 0.5);
    acc.Synchronize();
    const auto got = Download(*out), back = Download(*gradient);
    std::vector<double> want(rows * width, 0.0);
    bool same = true;
    for (int i = 0; i < n; ++i)
        for (int c = 0; c < width; ++c) {
            const bool there = tokens[i] >= 0 && tokens[i] < rows;
            const float y = there ? 2.0f * __bfloat162float(table[tokens[i] * width + c]) : 0.0f;
            same = same && got[i * width + c] == y;
            if (there) want[tokens[i] * width + c] += 0.5 * y;
        }
    CHECK(same);
    for (size_t i = 0; i < want.size(); ++i) same = same && back[i] == want[i];
    CHECK(same);
    auto add = CreateEmbeddingGradient<int64_t, float, float>(acc, true);
    add(stream, dtokens->View(), o, g, temp->View(), 0.5);
    acc.Synchronize();
    const auto twice = Download(*gradient);
    for (size_t i = 0; i < want.size(); ++i) same = same && twice[i] == 2.0 * want[i];
    CHECK(same);
    ArrayView2D<float> few(out->View(), n - 1, width);
    CHECK_THROWS(ArgumentOutOfRangeException, (CreateEmbedding<__nv_bfloat16, int64_t, float>(acc)(stream, t, dtokens->View(), few, 1.0)));
    CHECK_THROWS(ArgumentNullException, (CreateEmbedding<__nv_bfloat16, int64_t, float>(acc)(stream, ArrayView2D<__nv_bfloat16>(), dtokens->View(), o, 1.0)));
    CHECK_THROWS(ArgumentOutOfRangeException, backward(stream, dtokens->View(), o, g, temp->View().SubView(0, 64), 1.0));
    CHECK_THROWS(ArgumentOutOfRangeException, ArrayView2D<float>(out->View(), n + 1, width));
}

static void GradientTests(const Accelerator &acc) {
    AcceleratorStream stream = AcceleratorStream::Create();
    auto a = Upload(acc, std::vector<float>(48, 3.0f));
    auto b = Upload(acc, std::vector<__half>(64, __float2half(4.0f)));
    auto c = acc.Allocate1D<__nv_bfloat16>(48);
    auto d = acc.Allocate1D<__half>(64);
    auto norm = acc.Allocate1D<float>(1);
    auto temp = acc.Allocate1D<int>(ComputeGradientNormTempStorageSize(acc, 2));
    const std::vector<ElementView> views{a->View(), b->View()}, outputs{c->View(), d->View()};
    GradientNorm(acc, stream, views, norm->View(), temp->View());
    stream.Synchronize();
    const double whole = std::sqrt(48 * 9.0 + 64 * 16.0);
    CHECK(std::fabs(Download(*norm)[0] - whole) <= 1e-5 * whole);
    GradientClip(acc, stream, views, &outputs, 1e9, norm->View(), temp->View());  // nothing to clip: converted
    stream.Synchronize();
    CHECK(__bfloat162float(Download(*c)[47]) == 3.0f && __half2float(Download(*d)[63]) == 4.0f);
    auto given = Upload(acc, std::vector<float>{8.0f});
    GradientScale(acc, stream, views, nullptr, 2.0, given->View());
    stream.Synchronize();
    CHECK(Download(*a)[0] == 0.75f && __half2float(Download(*b)[5]) == 1.0f);
    CHECK_THROWS(ArgumentOutOfRangeException, GradientClip(acc, stream, views, nullptr, -1.0, norm->View(), temp->View()));
    const std::vector<ElementView> one{c->View()};
    CHECK_THROWS(ArgumentOutOfRangeException, GradientClip(acc, stream, views, &one, 1.0, norm->View(), temp->View()));
    CHECK_THROWS(ArgumentNullException, GradientNorm(acc, stream, views, ArrayView<float>(), temp->View()));
}

static void BalanceTests(const Accelerator &acc, int tokens, int experts, int choices) {
    AcceleratorStream stream;
    std::vector<float> logits(tokens * experts);
    for (size_t i = 0; i < logits.size(); ++i) logits[i] = (float)((int)(i * 11 % 17) - 8) * 0.25f;
    std::vector<int32_t> chosen(tokens * choices);
    for (size_t i = 0; i < chosen.size(); ++i) chosen[i] = (int32_t)(i * 5 % experts);
    std::vector<uint8_t> mask(tokens);
    for (int t = 0; t < tokens; ++t) mask[t] = t % 4 != 3;
    auto dl = Upload(acc, logits);
    auto dc = Upload(acc, chosen);
    auto dm = Upload(acc, mask);
    auto loss = acc.Allocate1D<float>(1), p = acc.Allocate1D<float>(experts), gradient = acc.Allocate1D<float>(tokens * experts);
    auto counts = acc.Allocate1D<int32_t>(experts + 1);
    auto temp = acc.Allocate1D<int>(ComputeBalanceLossTempStorageSize(acc, experts, tokens));
    ArrayView2D<float> l(dl->View(), tokens, experts), g(gradient->View(), tokens, experts);
    ArrayView2D<int32_t> k(dc->View(), tokens, choices);
    BalanceLoss(acc, stream, l, k, dm->View(), 1.0, loss->View(), counts->View(), p->View(), temp->View());
    auto upstream = Upload(acc, std::vector<float>{(float)tokens});
    BalanceLossGradient(acc, stream, l, dm->View(), counts->View(), choices, 1.0, upstream->View(), g);
    acc.Synchronize();
    std::vector<double> soft(tokens * experts, 0.0), mean(experts, 0.0);
    std::vector<int32_t> often(experts + 1, 0);
    for (int t = 0; t < tokens; ++t) {
        if (!mask[t]) continue;
        ++often[experts];
        double whole = 0.0;
        for (int e = 0; e < experts; ++e) whole += std::exp((double)logits[t * experts + e]);
        for (int e = 0; e < experts; ++e) mean[e] += soft[t * experts + e] = std::exp((double)logits[t * experts + e]) / whole;
        for (int j = 0; j < choices; ++j) ++often[chosen[t * choices + j]];
    }
    double value = 0.0;
    for (int e = 0; e < experts; ++e) value += experts * (double)often[e] / choices / often[experts] * mean[e] / often[experts];
    CHECK(Download(*counts) == often);
    CHECK(std::fabs(Download(*loss)[0] - value) <= 1e-5 * value);
    const auto got = Download(*gradient);
    bool near = true;
    for (int t = 0; t < tokens; ++t) {
        double dot = 0.0;
        for (int e = 0; e < experts; ++e) dot += often[e] * soft[t * experts + e];
        for (int e = 0; e < experts; ++e) {
            const double factor = (double)tokens * experts / choices / often[experts] / often[experts];
            const double want = factor * soft[t * experts + e] * (often[e] - dot);
            near = near && std::fabs(got[t * experts + e] - want) <= 1e-5 * factor * soft[t * experts + e] * (often[e] + dot);
        }
    }
    CHECK(near);
    CHECK_THROWS(ArgumentOutOfRangeException, BalanceLoss(acc, stream, l, k, dm->View().SubView(0, tokens - 1), 1.0, loss->View(), counts->View(), p->View(), temp->View()));
    CHECK_THROWS(ArgumentOutOfRangeException, BalanceLossGradient(acc, stream, l, dm->View(), counts->View().SubView(0, experts), choices, 1.0, upstream->View(), g));
    CHECK_THROWS(B200AlgException, BalanceLossGradient(acc, stream, l, dm->View(), counts->View(), 0, 1.0, upstream->View(), g));
}

int main() {
    Accelerator acc;
    EmbeddingTests(acc, 1, 1, 1);
    EmbeddingTests(acc, 200, 40, 24);
    EmbeddingTests(acc, 3000, 130, 72);
    GradientTests(acc);
    BalanceTests(acc, 50, 6, 2);
    BalanceTests(acc, 3000, 64, 4);
    std::printf("%d checks, %d failures\n", g_checks, g_failures);
    return g_failures ? 1 : 0;
}
