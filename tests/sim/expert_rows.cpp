// Host run of csrc/experts/grouped_tiles.hpp: for many tables of where experts' rows start, also such as leave rows before the first, go back or are no rows at all, every row of the results is stored
// exactly once for each part of k, those of an expert by products with its weights and those of nobody as zeros, and every expert's rows are summed over once.
#include "../../csrc/experts/grouped_tiles.hpp"
#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace dccl;

struct Table { std::vector<unsigned> first; std::vector<int> starts; };

/** What list_tiles and order_starts leave. */
static Table list(const Grouped& a, const std::vector<int>& starts) {
    Table t = {{}, starts};
    bool back = false;
    for (unsigned e = 0; e <= a.experts; e++) back |= goes_back(starts.data(), e, a);
    unsigned reached = 0;
    for (unsigned e = 0; e <= a.experts && back; e++) {
        const unsigned start = row_within(starts[e], a.rows);
        reached = start > reached ? start : reached;
        t.starts[e] = (int)reached;
    }
    unsigned before = 0;
    for (unsigned i = 0; i < listed_of(a); i++) {
        t.first.push_back(before);
        for (unsigned e = i * a.stride; e < (i + 1) * a.stride && e <= a.experts; e++) before += tall_of(t.starts.data(), e, a);
    }
    t.first.push_back(before);
    return t;
}

static int fail(const char* what, const Grouped& a, int form) {
    printf("%s: %u rows, %u experts, form %d, tiles of %u\n", what, a.rows, a.experts, form, a.tile_rows);
    return 1;
}

static int check(int form, unsigned rows, unsigned experts, unsigned m, unsigned n, unsigned tall, unsigned splits, const std::vector<int>& starts) {
    Grouped a = {};
    a.rows = rows;
    a.experts = experts;
    a.m = m;
    a.n = n;
    a.tile_rows = tall;
    a.tile_columns = 16;
    a.tiles_m = form == EXPERTS_WEIGHT ? blocks_of(m, tall) : 0;
    a.tiles_n = By(blocks_of(n, 16));
    a.group = By(16 * a.tiles_n.d);
    a.expert = By(form == EXPERTS_WEIGHT ? a.tiles_m * a.tiles_n.d : 1);
    a.splits = By(splits);
    a.k_blocks = 5;
    a.stride = listed_by(experts);
    a.most = (form == EXPERTS_WEIGHT ? experts * a.tiles_m : blocks_of(rows, tall) + experts + 2) * a.tiles_n.d * splits;
    const Table t = list(a, starts);
    // whose each row is, from the table's meaning alone
    std::vector<unsigned> owner(rows, experts);
    unsigned at = 0;
    for (unsigned e = 0; e <= experts; e++) {
        const unsigned start = starts[e] < 0 ? 0 : (unsigned)starts[e] < rows ? (unsigned)starts[e] : rows;
        for (; at < start; at++) owner[at] = e ? e - 1 : experts;
    }
    if (form != EXPERTS_WEIGHT && (unsigned long long)t.first.back() * a.tiles_n.d * splits > a.most) return fail("more tiles than a launch has", a, form);
    std::vector<unsigned> stored(form == EXPERTS_WEIGHT ? (size_t)experts * m * n : (size_t)rows * n, 0), summed(rows, 0);
    for (unsigned i = 0; i < grouped_tiles(form, a, t.first.data()); i++) {
        const GroupedPlace p = grouped_place(form, i, a, t.first.data(), t.starts.data());
        if (p.expert > experts || !p.rows || p.rows > tall || p.column >= n || p.split >= splits) return fail("place", a, form);
        for (unsigned r = 0; r < p.rows; r++) {
            if (form != EXPERTS_WEIGHT && (p.row + r >= rows || owner[p.row + r] != p.expert)) return fail("a row of another", a, form);
            if (form == EXPERTS_WEIGHT && p.row + r >= m) return fail("row", a, form);
            for (unsigned c = p.column; c < n && c < p.column + 16; c++) stored[grouped_row(form, p, r, a) * n + c]++;
        }
        if (form != EXPERTS_WEIGHT) {
            if (p.expert == experts ? p.k_count != 0 : p.k_from + p.k_count > 5 * kTileK) return fail("k", a, form);
        } else {
            for (unsigned k = p.k_from; k < p.k_from + p.k_count; k++) {
                if (k >= rows || owner[k] != p.expert) return fail("k of another", a, form);
                summed[k] += p.row == 0 && p.column == 0;
            }
        }
    }
    for (unsigned s : stored)
        if (s != splits) return fail("stored", a, form);
    for (unsigned r = 0; r < rows && form == EXPERTS_WEIGHT; r++)
        if (summed[r] != (owner[r] < experts)) return fail("summed", a, form);
    return 0;
}

int main() {
    srand(2);
    int wrong = 0;
    for (int round = 0; round < 600 && !wrong; round++) {
        const unsigned experts = 1 + (round % 5 == 0 ? rand() % 1024 : rand() % 12), rows = 1 + rand() % (round % 3 ? 700 : 3000), splits = round % 4 ? 1 : 1 + rand() % 4;
        const unsigned tall = round % 7 == 3 ? 32 : round % 5 == 2 ? 256 : 128, high = tall < 128 ? 128 : tall, m = 1 + rand() % 300, n = 1 + rand() % 40;
        std::vector<int> starts(experts + 1);
        for (int& s : starts) s = rand() % (rows + 1);
        for (unsigned i = 1; i <= experts; i++)     // in order
            for (unsigned j = i; j > 0 && starts[j] < starts[j - 1]; j--) { const int v = starts[j]; starts[j] = starts[j - 1]; starts[j - 1] = v; }
        if (round % 3 == 1) starts[experts] = rows;
        if (round % 8 == 1) starts[0] = 0;
        wrong |= check(EXPERTS_FORWARD, rows, experts, 0, n, tall, splits, starts);
        wrong |= check(EXPERTS_INPUT, rows, experts, 0, n, high, splits, starts);
        wrong |= check(EXPERTS_WEIGHT, rows, experts, m, n, high, splits, starts);
        for (int& s : starts) s = rand() % 5 ? s : rand() % 3 ? rand() % (int)(rows + 1) : rand() % 2 ? -rand() : rand();        // some that go back, and numbers of nothing
        if (round % 2) starts[experts] = rand() % (rows + 1);
        wrong |= check(EXPERTS_FORWARD, rows, experts, 0, n, tall, splits, starts);
        wrong |= check(EXPERTS_INPUT, rows, experts, 0, n, high, splits, starts);
        wrong |= check(EXPERTS_WEIGHT, rows, experts, m, n, high, splits, starts);
    }
    if (!wrong) printf("OK\n");
    return wrong;
}
