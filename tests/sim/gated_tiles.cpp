// Host run of csrc/decoder/gated_tiles.hpp.
//   plan SMS FORM M N K   prints the plan of a product
//   mark                  what the CTAs of products that gave up leave: each element of the results NaN, once, and nothing beside them written
#include "../../csrc/decoder/gated_tiles.hpp"
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

using namespace dccl;

static int mark(int sms, int form, unsigned m, unsigned n, unsigned k, bool keep) {
    const GemmPlan p = plan_gemm(sms, form, m, n, k);
    const size_t stride = up_to(n, 4), planes = (size_t)p.splits * (form == INPUT_GRAD ? 1 : 2);
    std::vector<uint16_t> c[2] = {std::vector<uint16_t>((size_t)m * n + 8, 1), std::vector<uint16_t>((size_t)m * n + 8, 1)};
    std::vector<float> pre[2] = {std::vector<float>(m * stride + 8, 1.0f), std::vector<float>(m * stride + 8, 1.0f)}, partial(planes * m * stride + 8, 1.0f);
    const bool split = p.splits > 1;
    if (split && p.partial_bytes != planes * m * stride * sizeof(float)) return 1;
    const Tiling a = {m, n, p.tiles_m, p.tiles_n, p.batch, p.splits, p.k_blocks};
    const Results to = {c[0].data(), c[p.batch - 1].data(), keep ? pre[0].data() : nullptr, keep ? pre[1].data() : nullptr, stride, split ? partial.data() : nullptr, stride};
    const unsigned tiles = p.tiles_m * p.tiles_n * p.batch * p.splits, workers = p.pair ? sms / 2 : sms, ctas = tiles < workers ? tiles : workers, threads = 320;
    for (unsigned cta = 0; cta < ctas; cta++)
        for (unsigned rank = 0; rank < (p.pair ? 2u : 1u); rank++)
            for (unsigned t = 0; t < threads; t++)
                mark_incomplete(form, a, to, p.pair ? 2 * kTileM : kTileM, form == GATED ? p.columns / 2 : p.columns, rank, cta, ctas, t, threads);
    size_t wrong = 0;
    for (int w = 0; w < 2; w++) {
        const bool stored = !split && w < (int)p.batch;
        for (size_t i = 0; i < c[w].size(); i++) wrong += c[w][i] != (stored && i < (size_t)m * n ? kNoResult16 : 1);
        for (size_t i = 0; i < pre[w].size(); i++)
            wrong += keep && form == GATED && !split && i < m * stride && i % stride < n ? !std::isnan(pre[w][i]) : pre[w][i] != 1.0f;
    }
    for (size_t i = 0; i < partial.size(); i++) wrong += split && i < planes * m * stride && i % stride < n ? !std::isnan(partial[i]) : partial[i] != 1.0f;
    if (wrong) printf("%zu elements of form %d, %u x %u x %u\n", wrong, form, m, n, k);
    return wrong != 0;
}

int main(int argc, char** argv) {
    if (argc == 7 && !strcmp(argv[1], "plan")) {
        const GemmPlan p = plan_gemm(atoi(argv[2]), atoi(argv[3]), atoi(argv[4]), atoi(argv[5]), atoi(argv[6]));
        const unsigned tiles = p.tiles_m * p.tiles_n * p.batch * p.splits, workers = p.pair ? atoi(argv[2]) / 2 : atoi(argv[2]);
        printf("%d %d %u %u\n", p.pair, p.columns, p.splits, (tiles + workers - 1) / workers);
        return 0;
    }
    int wrong = 0;
    const unsigned sizes[][3] = {{1, 1, 1}, {129, 65, 64}, {300, 1033, 65}, {257, 191, 2048}, {1000, 48, 4000}, {64, 300, 8192}, {700, 2055, 500}};
    for (const auto& s : sizes)
        for (int form = GATED; form <= WEIGHT_GRAD; form++)
            for (const bool keep : {false, true}) wrong += mark(148, form, s[0], s[1], s[2], keep) + mark(12, form, s[0], s[1], s[2], keep);
    return wrong != 0;
}
