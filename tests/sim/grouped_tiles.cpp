// Host run of csrc/experts/grouped_tiles.hpp: for many tables of starts, sound ones and others, the tiles of a product cover each element of its results once, by rows
// of the right expert, and what the CTAs of a product that gave up leave is NaN in each of them and nothing beside.
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
        for (unsigned e = i * a.stride; e < (i + 1) * a.stride && e <= a.experts; e++) before += tall_of(starts, e, a.experts, a.rows);
    }
    first[listed_of(a)] = before;
    return first;
}

static int fail(const char* what, unsigned rows, unsigned experts, int form) {
    printf("%s: %u rows, %u experts, form %d\n", what, rows, experts, form);
    return 1;
}

static int check(int form, unsigned rows, unsigned experts, unsigned m, unsigned n, unsigned columns, const std::vector<int>& starts, bool sound) {
    Grouped a = {};
    a.rows = rows;
    a.experts = experts;
    a.m = m;
    a.n = n;
    a.tiles_m = form == EXPERTS_WEIGHT ? blocks_of(m, kTileM) : 0;
    a.tiles_n = blocks_of(n, columns);
    a.k_blocks = 3;
    a.stride = (experts + kListed) / kListed;
    if (listed_of(a) > kListed) return fail("list too long", rows, experts, form);
    const std::vector<unsigned> first = list(a, starts.data());
    const size_t height = form == EXPERTS_WEIGHT ? (size_t)experts * m : rows;
    std::vector<int> seen(height * n, 0);
    const unsigned long long tiles = grouped_tiles(form, a, first.data());
    for (unsigned long long t = 0; t < tiles; t++) {
        const GroupedPlace p = grouped_place(form, t, columns, a, first.data(), starts.data());
        if (p.expert > experts || p.rows < 1 || p.rows > (unsigned)kTileM || p.column >= n) return fail("place", rows, experts, form);
        if (form == EXPERTS_WEIGHT ? p.k_from + p.k_count > rows || (sound && (p.k_from != (unsigned)starts[p.expert] || p.k_count != (unsigned)(starts[p.expert + 1] - starts[p.expert])))
                                   : (p.k_count != (p.expert < experts ? 3u * kTileK : 0u)))
            return fail("k", rows, experts, form);
        for (unsigned r = 0; r < p.rows; r++) {
            const size_t at = grouped_row(form, p, r, a);
            if (at + n > height * n || (form != EXPERTS_WEIGHT && sound && p.expert < experts && (p.row + r < (unsigned)starts[p.expert] || p.row + r >= (unsigned)starts[p.expert + 1])))
                return fail("row", rows, experts, form);
            for (unsigned c = p.column; c < n && c < p.column + columns; c++) seen[at + c]++;
        }
    }
    for (int s : seen)
        if (sound && s != 1) return fail("covered", rows, experts, form);
    // as the CTAs of a launch would mark them
    std::vector<uint16_t> c(height * n + 8, 1);
    const size_t stride = up_to(n, 4);
    std::vector<float> z(rows * stride + 8, 1.0f);
    const unsigned ctas = tiles < 7 ? (unsigned)tiles : 7;
    for (unsigned cta = 0; cta < ctas; cta++)
        for (unsigned t = 0; t < 320; t += 1)
            grouped_mark(form, a, columns, first.data(), starts.data(), c.data(), form == EXPERTS_FORWARD ? z.data() : nullptr, stride, cta, ctas, t, 320);
    for (size_t i = 0; i < c.size(); i++)
        if (c[i] != (i < height * n && seen[i] ? kNoResult16 : 1)) return fail("marked", rows, experts, form);
    for (size_t i = 0; i < z.size(); i++) {
        const size_t r = i / stride, col = i % stride;
        const bool want = form == EXPERTS_FORWARD && sound && r < rows && col < n && r < (size_t)starts[experts];
        if (sound && (z[i] != z[i]) != want) return fail("marked products", rows, experts, form);
    }
    return 0;
}

int main() {
    srand(1);
    int wrong = 0;
    for (int round = 0; round < 300 && !wrong; round++) {
        const unsigned experts = 1 + (round % 5 == 0 ? rand() % 1024 : rand() % 12), rows = rand() % (round % 3 ? 700 : 3000);
        std::vector<int> starts(experts + 1);
        const unsigned used = round % 2 ? rows : rows - (rows ? rand() % (rows + 1) : 0);
        std::vector<unsigned> cuts;
        for (unsigned e = 0; e <= experts; e++) starts[e] = e == 0 ? 0 : e == experts ? (int)used : (int)(used ? rand() % (used + 1) : 0);
        for (unsigned i = 1; i < experts; i++)      // in order
            for (unsigned j = i; j > 1 && starts[j] < starts[j - 1]; j--) { const int v = starts[j]; starts[j] = starts[j - 1]; starts[j - 1] = v; }
        const unsigned m = 1 + rand() % 300, n = 1 + rand() % 40, columns = 16;
        if (rows) {
            wrong |= check(EXPERTS_FORWARD, rows, experts, 0, n, columns, starts, true);
            wrong |= check(EXPERTS_INPUT, rows, experts, 0, n, columns, starts, true);
            wrong |= check(EXPERTS_WEIGHT, rows, experts < 9 ? experts : 8, m, n, columns, starts, true);
            for (int& s : starts) s = rand() % 5 ? s : (rand() % 2 ? -rand() : rand());       // numbers of nothing
            if (experts < 20) {
                wrong |= check(EXPERTS_FORWARD, rows, experts, 0, n, columns, starts, false);
                wrong |= check(EXPERTS_WEIGHT, rows, experts < 9 ? experts : 8, m, n, columns, starts, false);
            }
        }
    }
    if (!wrong) printf("OK\n");
    return wrong;
}
