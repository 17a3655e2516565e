/**
 * How the experts' products are cut into tiles by counts that only the device knows, and what a CTA that could not finish leaves behind. Nothing here needs
 * CUDA, so that tests run it on the host.
 */
#pragma once
#include "../decoder/gated_tiles.hpp"

namespace dccl {

enum GroupedForm {
    EXPERTS_FORWARD,        // h = act(x W^T): the rows of a tile are some of one expert's, its columns some of `out`
    EXPERTS_INPUT,          // dx = dz W: the columns are some of `width`
    EXPERTS_WEIGHT,         // dW = dz^T x: the rows of a tile are some of `out`, its columns some of `width`, and k are the expert's rows
};

struct Grouped {
    unsigned rows, experts;                 // of all
    unsigned m, n;                          // EXPERTS_WEIGHT: rows of one expert's result; columns of the result
    unsigned tiles_m, tiles_n, k_blocks;    // EXPERTS_WEIGHT: rows of tiles; columns of tiles; otherwise: blocks of k
    unsigned stride;                        // otherwise: experts of one entry of the list of tiles
};

/** The list has room for this many entries and the end: shared memory beside the tiles has no more. */
constexpr unsigned kListed = 256;

/** Rows of an expert, whatever the numbers are: inside of [0, rows), and none where the next starts before. The last is of nobody, and goes to the end. */
struct Span { unsigned from, count; };
DCCL_BOTH unsigned row_within(int v, unsigned rows) { return v < 0 ? 0 : (unsigned)v < rows ? (unsigned)v : rows; }
DCCL_BOTH Span span_of(const int* starts, unsigned e, unsigned experts, unsigned rows) {
    const unsigned from = row_within(starts[e], rows), to = e < experts ? row_within(starts[e + 1], rows) : rows;
    return {from, to > from ? to - from : 0};
}

DCCL_BOTH unsigned tall_of(const int* starts, unsigned e, unsigned experts, unsigned rows) { return (span_of(starts, e, experts, rows).count + kTileM - 1) / kTileM; }

/** Entries of the list: the experts and the rows of nobody, `stride` each. */
DCCL_BOTH unsigned listed_of(const Grouped& a) { return (a.experts + a.stride) / a.stride; }

/** One tile: rows [row, row + rows) of the result (EXPERTS_WEIGHT: of the expert's), columns from `column`, and the k that it adds up. */
struct GroupedPlace { unsigned expert, row, rows, column, k_from, k_count; };

/**
 * Tile number -> place, of tiles of kTileM x `columns`. first[i]: rows of tiles before expert i * stride, and all of them (the rows of nobody are the last
 * "expert"). Groups of 16 rows of tiles are walked column by column, so that the tiles of one moment share operands in L2.
 */
DCCL_BOTH GroupedPlace grouped_place(int form, unsigned long long tile, unsigned columns, const Grouped& a, const unsigned* first, const int* starts) {
    GroupedPlace p;
    unsigned tiles_m, within;
    if (form == EXPERTS_WEIGHT) {
        const unsigned per = a.tiles_m * a.tiles_n;
        p.expert = (unsigned)(tile / per);
        within = (unsigned)(tile % per);
        tiles_m = a.tiles_m;
    } else {
        unsigned low = 0, high = listed_of(a);
        while (high - low > 1) {
            const unsigned mid = (low + high) / 2;
            if ((unsigned long long)first[mid] * a.tiles_n <= tile) low = mid;
            else high = mid;
        }
        unsigned long long at = (unsigned long long)first[low] * a.tiles_n;
        p.expert = low * a.stride;
        tiles_m = tall_of(starts, p.expert, a.experts, a.rows);
        while (p.expert < a.experts && tile - at >= (unsigned long long)tiles_m * a.tiles_n) {
            at += (unsigned long long)tiles_m * a.tiles_n;
            tiles_m = tall_of(starts, ++p.expert, a.experts, a.rows);
        }
        within = (unsigned)(tile - at);
    }
    const unsigned group = within / (16 * a.tiles_n), top = group * 16, tall = tiles_m - top < 16 ? tiles_m - top : 16;
    within -= top * a.tiles_n;
    const unsigned m = top + within % tall;
    p.column = within / tall * columns;
    const Span s = span_of(starts, p.expert, a.experts, a.rows);
    if (form == EXPERTS_WEIGHT) {
        p.row = m * kTileM;
        p.rows = a.m - p.row < (unsigned)kTileM ? a.m - p.row : kTileM;
        p.k_from = s.from;
        p.k_count = s.count;
    } else {
        p.row = s.from + m * kTileM;
        // (starts that are not in order may give more tiles than can be counted)
        p.rows = m * kTileM >= s.count ? 0 : s.count - m * kTileM < (unsigned)kTileM ? s.count - m * kTileM : kTileM;
        p.k_from = 0;
        p.k_count = p.expert < a.experts ? a.k_blocks * kTileK : 0;
    }
    return p;
}

/** Tiles of a whole product. */
DCCL_BOTH unsigned long long grouped_tiles(int form, const Grouped& a, const unsigned* first) {
    return form == EXPERTS_WEIGHT ? (unsigned long long)a.experts * a.tiles_m * a.tiles_n : (unsigned long long)first[listed_of(a)] * a.tiles_n;
}

/** First element of a row of the result. */
DCCL_BOTH size_t grouped_row(int form, const GroupedPlace& p, unsigned row, const Grouped& a) { return ((size_t)(form == EXPERTS_WEIGHT ? p.expert : 0) * a.m + p.row + row) * a.n; }

/** NaN in all that one CTA stores (first tile, step), by each of its threads. */
DCCL_BOTH void grouped_mark(int form, const Grouped& a, unsigned columns, const unsigned* first, const int* starts, uint16_t* c, float* z, size_t z_stride, unsigned long long tile,
                            unsigned long long step, unsigned thread, unsigned threads) {
    for (const unsigned long long tiles = grouped_tiles(form, a, first); tile < tiles; tile += step) {
        const GroupedPlace p = grouped_place(form, tile, columns, a, first, starts);
        for (unsigned i = thread; i < p.rows * columns; i += threads) {
            const unsigned row = i / columns, column = p.column + i % columns;
            if (column >= a.n) continue;
            c[grouped_row(form, p, row, a) + column] = kNoResult16;
            if (z && p.expert < a.experts) z[(p.row + row) * z_stride + column] = __builtin_nanf("");
        }
    }
}

} // namespace dccl
