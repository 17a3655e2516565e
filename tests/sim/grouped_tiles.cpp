// Host run of csrc/experts/grouped_tiles.hpp.
//   (no arguments)               for many tables of starts, sound ones and others, the tiles of a product cover each element of its results once for each part of k, by rows of the
//                                right expert, and what the CTAs of a product that gave up leave is NaN in each of them and nothing beside
//   plan SMS FORM ROWS E M N K   prints the plan of a product
#include "../../csrc/experts/grouped_tiles.hpp"
#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace dccl;

static std::vector<unsigned> list(const Grouped& a, const int* starts) {
    std::vector<unsigned> first(listed_of(a) + 1);
    unsigned before = 0;
    for (unsigned i = 0; i < listed_of(a); i++) {
        first[i] = before;
        for (unsigned e = i * a.stride; e < (i + 1) * a.stride && e <= a.experts; e++) before += tall_of(starts, e, a);
    }
    first[listed_of(a)] = before;
    return first;
}

static int fail(const char* what, unsigned rows, unsigned experts, int form) {
    printf("%s: %u rows, %u experts, form %d\n", what, rows, experts, form);
    return 1;
}

static int check(int form, unsigned rows, unsigned experts, unsigned m, unsigned n, unsigned tall, unsigned columns, unsigned splits, const std::vector<int>& starts, bool sound) {
    Grouped a = {};
    a.rows = rows;
    a.experts = experts;
    a.m = m;
    a.n = n;
    a.tile_rows = tall;
    a.tile_columns = columns;
    a.tiles_m = form == EXPERTS_WEIGHT ? blocks_of(m, tall) : 0;
    a.tiles_n = By(blocks_of(n, columns));
    a.group = By(16 * a.tiles_n.d);
    a.expert = By(form == EXPERTS_WEIGHT ? a.tiles_m * a.tiles_n.d : 1);
    a.splits = By(splits);
    a.k_blocks = 5;
    a.stride = (experts + kListed) / kListed;
    a.most = (form == EXPERTS_WEIGHT ? experts * a.tiles_m : blocks_of(rows, tall) + experts + 1) * a.tiles_n.d * splits;
    if (listed_of(a) > kListed) return fail("list too long", rows, experts, form);
    const std::vector<unsigned> first = list(a, starts.data());
    const size_t height = grouped_rows(form, a);
    std::vector<int> seen(height * n, 0), blocks(splits > 1 || form == EXPERTS_WEIGHT ? experts * (rows / kTileK + 8) : 0, 0);
    const unsigned tiles = grouped_tiles(form, a, first.data());
    for (unsigned t = 0; t < tiles; t++) {
        const GroupedPlace p = grouped_place(form, t, a, first.data(), starts.data());
        if (p.expert > experts || p.rows > tall || (sound && !p.rows) || p.column >= n || p.split >= splits) return fail("place", rows, experts, form);
        const Span s = span_of(starts.data(), p.expert, experts, rows);
        if (form == EXPERTS_WEIGHT ? p.k_count && (p.k_from < s.from || p.k_from + p.k_count > s.from + s.count)
                                   : p.expert < experts ? p.k_from + p.k_count > 5 * kTileK : p.k_count != 0)
            return fail("k", rows, experts, form);
        if (p.row % 1 == 0 && p.column == 0 && form == EXPERTS_WEIGHT && p.row == 0 && sound)
            for (unsigned k = 0; k < p.k_count; k += kTileK) blocks[p.expert * (rows / kTileK + 8) + (p.k_from - s.from + k) / kTileK]++;
        for (unsigned r = 0; r < p.rows; r++) {
            const size_t at = grouped_row(form, p, r, a);
            if (at >= height || (form != EXPERTS_WEIGHT && sound && p.expert < experts && (p.row + r < (unsigned)starts[p.expert] || p.row + r >= (unsigned)starts[p.expert + 1])))
                return fail("row", rows, experts, form);
            for (unsigned c = p.column; c < n && c < p.column + columns; c++) seen[at * n + c]++;
        }
    }
    for (int s : seen)
        if (sound && s != (int)splits) return fail("covered", rows, experts, form);
    if (form == EXPERTS_WEIGHT && sound)
        for (unsigned e = 0; e < experts; e++)
            for (unsigned b = 0; b < rows / kTileK + 8; b++)
                if (blocks[e * (rows / kTileK + 8) + b] != (b * kTileK < (unsigned)(starts[e + 1] - starts[e]))) return fail("blocks", rows, experts, form);
    // as the CTAs of a launch would mark them
    const size_t stride = up_to(n, 4);
    std::vector<uint16_t> c(height * n + 8, 1);
    std::vector<float> z(height * stride + 8, 1.0f), partial(splits > 1 ? splits * height * stride + 8 : 0, 1.0f);
    const GroupedResults to = {c.data(), form == EXPERTS_FORWARD ? z.data() : nullptr, stride, partial.data(), stride};
    const unsigned ctas = tiles < 7 ? tiles : 7;
    for (unsigned cta = 0; cta < ctas; cta++)
        for (unsigned t = 0; t < 320; t++) grouped_mark(form, a, to, first.data(), starts.data(), cta, ctas, t, 320);
    for (size_t i = 0; i < c.size(); i++)
        if (c[i] != (splits == 1 && i < height * n && seen[i] ? kNoResult16 : 1)) return fail("marked", rows, experts, form);
    for (size_t i = 0; i < z.size() && sound; i++) {
        const size_t r = i / stride, col = i % stride;
        if ((z[i] != z[i]) != (splits == 1 && form == EXPERTS_FORWARD && r < rows && col < n && r < (size_t)starts[experts])) return fail("marked products", rows, experts, form);
    }
    for (size_t i = 0; i < partial.size(); i++) {
        const size_t line = i / stride, col = i % stride;
        if ((partial[i] != partial[i]) != (line < splits * height && col < n && (!sound || true) && seen[line % height * n + col] > 0)) return fail("marked parts", rows, experts, form);
    }
    return 0;
}

int main(int argc, char** argv) {
    if (argc == 9) {
        const GroupedPlan p = plan_grouped(atoi(argv[3]), atoi(argv[2]), atoi(argv[4]), atoi(argv[5]), atoi(argv[6]), atoi(argv[7]), atoi(argv[8]));
        printf("%u %u %u\n", p.tile_rows, p.tile_columns, p.splits);
        return 0;
    }
    srand(1);
    int wrong = 0;
    for (int round = 0; round < 300 && !wrong; round++) {
        const unsigned experts = 1 + (round % 5 == 0 ? rand() % 1024 : rand() % 12), rows = 1 + rand() % (round % 3 ? 700 : 3000);
        std::vector<int> starts(experts + 1);
        const unsigned used = round % 2 ? rows : rows - rand() % (rows + 1);
        for (unsigned e = 0; e <= experts; e++) starts[e] = e == 0 ? 0 : e == experts ? (int)used : (int)(used ? rand() % (used + 1) : 0);
        for (unsigned i = 1; i < experts; i++)      // in order
            for (unsigned j = i; j > 1 && starts[j] < starts[j - 1]; j--) { const int v = starts[j]; starts[j] = starts[j - 1]; starts[j - 1] = v; }
        const unsigned m = 1 + rand() % 300, n = 1 + rand() % 40, columns = 16, splits = round % 4 ? 1 : 1 + rand() % 4, tall = round % 7 == 3 ? 32 : round % 5 == 2 ? 256 : 128, high = tall < 128 ? 128 : tall;
        wrong |= check(EXPERTS_FORWARD, rows, experts, 0, n, tall, columns, splits, starts, true);
        wrong |= check(EXPERTS_INPUT, rows, experts, 0, n, high, columns, splits, starts, true);
        wrong |= check(EXPERTS_WEIGHT, rows, experts < 9 ? experts : 8, m, n, high, columns, splits, starts, true);
        for (int& s : starts) s = rand() % 5 ? s : (rand() % 2 ? -rand() : rand());       // numbers of nothing
        if (experts < 20) {
            wrong |= check(EXPERTS_FORWARD, rows, experts, 0, n, tall, columns, splits, starts, false);
            wrong |= check(EXPERTS_WEIGHT, rows, experts < 9 ? experts : 8, m, n, high, columns, splits, starts, false);
        }
    }
    if (!wrong) printf("OK\n");
    return wrong;
}
