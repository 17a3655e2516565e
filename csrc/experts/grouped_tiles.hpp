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

/** Division of n < 2^31 by a number that the host knows, as Divisor of row_access.cuh does it. */
struct By {
    unsigned d, m, s;
    By() = default;
    explicit By(unsigned divisor) : d(divisor), s(0) {
        while (s < 31 && (1u << s) < d) s++;
        m = (unsigned)((((uint64_t)1 << (32 + s)) + d - 1) / d - ((uint64_t)1 << 32));
    }
    DCCL_BOTH unsigned quotient(unsigned n) const { return ((unsigned)((uint64_t)n * m >> 32) + n) >> s; }
};

struct Grouped {
    unsigned rows, experts;                 // of all
    unsigned m, n;                          // EXPERTS_WEIGHT: rows of one expert's result; columns of the result
    unsigned tile_rows, tile_columns;
    unsigned tiles_m, k_blocks;             // EXPERTS_WEIGHT: rows of tiles; otherwise: blocks of k
    unsigned stride;                        // otherwise: experts of one entry of the list of tiles
    unsigned most;                          // tiles, whatever the starts are
    By tiles_n, group, expert, splits;      // columns of tiles; tiles of 16 rows of them; EXPERTS_WEIGHT: of an expert; parts that the k of a tile is cut into
};

/** What a product leaves where: c of 16 bits, and in fp32 the products before their activation (EXPERTS_FORWARD), or the parts of a sum that is cut, [split][row][partial_stride]. */
struct GroupedResults { void* c; float* z; size_t z_stride; float* partial; size_t partial_stride; };

/** The list has room for this many entries and the end: shared memory beside the tiles has no more. */
constexpr unsigned kListed = 120;

/** Rows of an expert by starts in order, whatever the numbers are: inside of [0, rows). The last is of nobody, and goes to the end. (The rows before the first start are
 *  nobody's either; their tiles come behind those of the last.) */
struct Span { unsigned from, count; };
DCCL_BOTH unsigned row_within(int v, unsigned rows) { return v < 0 ? 0 : (unsigned)v < rows ? (unsigned)v : rows; }
DCCL_BOTH Span span_of(const int* starts, unsigned e, unsigned experts, unsigned rows) {
    const unsigned from = row_within(starts[e], rows), to = e < experts ? row_within(starts[e + 1], rows) : rows;
    return {from, to > from ? to - from : 0};
}

/** Whether the start behind this one lies before it. Such starts are put in order first, each as far as those ahead of it: so no row is of two experts. */
DCCL_BOTH bool goes_back(const int* starts, unsigned e, const Grouped& a) { return e < a.experts && row_within(starts[e + 1], a.rows) < row_within(starts[e], a.rows); }

/** Rows of tiles. */
DCCL_BOTH unsigned tall_of(unsigned rows, const Grouped& a) { return (rows + a.tile_rows - 1) / a.tile_rows; }
DCCL_BOTH unsigned tall_of(const int* starts, unsigned e, const Grouped& a) {
    return tall_of(span_of(starts, e, a.experts, a.rows).count, a) + (e == a.experts ? tall_of(row_within(starts[0], a.rows), a) : 0);
}

/** Experts of one entry, so that they and the rows of nobody have at most kListed. */
inline unsigned listed_by(unsigned experts) { return (experts + kListed) / kListed; }
/** Entries of the list: the experts and the rows of nobody, `stride` each. */
DCCL_BOTH unsigned listed_of(const Grouped& a) { return (a.experts + a.stride) / a.stride; }

/** One tile, or a part of it: rows [row, row + rows) of the result (EXPERTS_WEIGHT: of the expert's), columns from `column`, and the k that it adds up. */
struct GroupedPlace { unsigned expert, row, rows, column, k_from, k_count, split; };

/**
 * Tile number -> place. first[i]: rows of tiles before expert i * stride, and all of them (the rows of nobody are the last "expert"). Groups of 16 rows of tiles
 * are walked column by column, so that the tiles of one moment share operands in L2.
 */
DCCL_BOTH GroupedPlace grouped_place(int form, unsigned tile, const Grouped& a, const unsigned* first, const int* starts) {
    GroupedPlace p;
    unsigned tiles_m, within, part = a.splits.quotient(tile);
    p.split = tile - part * a.splits.d;
    if (form == EXPERTS_WEIGHT) {
        p.expert = a.expert.quotient(part);
        within = part - p.expert * a.expert.d;
        tiles_m = a.tiles_m;
    } else {
        unsigned low = 0, high = listed_of(a);
        while (high - low > 1) {
            const unsigned mid = (low + high) / 2;
            if ((unsigned long long)first[mid] * a.tiles_n.d <= part) low = mid;
            else high = mid;
        }
        unsigned long long at = (unsigned long long)first[low] * a.tiles_n.d;
        p.expert = low * a.stride;
        tiles_m = tall_of(starts, p.expert, a);
        while (p.expert < a.experts && part - at >= (unsigned long long)tiles_m * a.tiles_n.d) {
            at += (unsigned long long)tiles_m * a.tiles_n.d;
            tiles_m = tall_of(starts, ++p.expert, a);
        }
        within = (unsigned)(part - at);
    }
    const unsigned group = a.group.quotient(within), top = group * 16, tall = tiles_m - top < 16 ? tiles_m - top : 16;
    within -= group * a.group.d;
    const unsigned n = tall == 16 ? within / 16 : within / tall;
    unsigned m = top + within - n * tall;
    p.column = n * a.tile_columns;
    Span s = span_of(starts, p.expert, a.experts, a.rows);
    if (form != EXPERTS_WEIGHT && p.expert == a.experts && m >= tall_of(s.count, a)) {
        m -= tall_of(s.count, a);
        s = {0, row_within(starts[0], a.rows)};
    }
    unsigned count, blocks;
    if (form == EXPERTS_WEIGHT) {
        p.row = m * a.tile_rows;
        p.rows = a.m - p.row < a.tile_rows ? a.m - p.row : a.tile_rows;
        p.k_from = s.from;
        count = s.count;
    } else {
        p.row = s.from + m * a.tile_rows;
        p.rows = m * a.tile_rows >= s.count ? 0 : s.count - m * a.tile_rows < a.tile_rows ? s.count - m * a.tile_rows : a.tile_rows;
        p.k_from = 0;
        count = p.expert < a.experts ? a.k_blocks * kTileK : 0;
    }
    blocks = (count + kTileK - 1) / kTileK;
    if (a.splits.d > 1) {           // whole blocks for each part, in order
        const unsigned from = (unsigned)((uint64_t)blocks * p.split / a.splits.d) * kTileK, to = (unsigned)((uint64_t)blocks * (p.split + 1) / a.splits.d) * kTileK;
        p.k_from += from;
        count = (to < count ? to : count) - from;
    }
    p.k_count = count;
    return p;
}

/** Tiles of a whole product, parts of tiles counted each. */
DCCL_BOTH unsigned grouped_tiles(int form, const Grouped& a, const unsigned* first) {
    if (form == EXPERTS_WEIGHT) return a.most;
    const unsigned long long tiles = (unsigned long long)first[listed_of(a)] * a.tiles_n.d * a.splits.d;
    return tiles < a.most ? (unsigned)tiles : a.most;
}

/** Number of a row of the result. */
DCCL_BOTH size_t grouped_row(int form, const GroupedPlace& p, unsigned row, const Grouped& a) { return (size_t)(form == EXPERTS_WEIGHT ? p.expert : 0) * a.m + p.row + row; }
/** Rows of the result. */
DCCL_BOTH size_t grouped_rows(int form, const Grouped& a) { return form == EXPERTS_WEIGHT ? (size_t)a.experts * a.m : a.rows; }

/** NaN in all that one CTA stores (first tile, step), by each of its threads. What joins the parts hands the NaN of one on. */
DCCL_BOTH void grouped_mark(int form, const Grouped& a, const GroupedResults& to, const unsigned* first, const int* starts, unsigned tile, unsigned step, unsigned thread, unsigned threads) {
    for (const unsigned tiles = grouped_tiles(form, a, first); tile < tiles; tile += step) {
        const GroupedPlace p = grouped_place(form, tile, a, first, starts);
        for (unsigned i = thread; i < p.rows * a.tile_columns; i += threads) {
            const unsigned row = i / a.tile_columns, column = p.column + i % a.tile_columns;
            if (column >= a.n) continue;
            const size_t at = grouped_row(form, p, row, a);
            if (a.splits.d > 1) {
                to.partial[(p.split * grouped_rows(form, a) + at) * to.partial_stride + column] = __builtin_nanf("");
            } else {
                reinterpret_cast<uint16_t*>(to.c)[at * a.n + column] = kNoResult16;
                if (to.z && p.expert < a.experts) to.z[at * to.z_stride + column] = __builtin_nanf("");
            }
        }
    }
}

/**
 * What the loading thread of a CTA has under way, by the stages that its blocks go round: which barrier counts a stage's bytes, and the parity of their phase there. A block whose
 * rows are cleared before it is used (`tail`, of a pair of CTAs) lands on a barrier of its own, `landed`, and the other one, `full`, is completed by the other CTA's arrival alone.
 */
struct InFlight {
    unsigned filled = 0, tails = 0, turns = 0;      // blocks so far; stages whose last one was a tail, and that have had an odd number of them
    DCCL_BOTH void load(unsigned stage, bool tail) {
        filled++;
        tails = tail ? tails | 1u << stage : tails & ~(1u << stage);
        turns ^= (unsigned)tail << stage;
    }
    /** The blocks that may not have landed: the last ones, one of each stage. */
    DCCL_BOTH unsigned oldest(unsigned stages) const { return filled > stages ? filled - stages : 0; }
    DCCL_BOTH bool on_landed(unsigned block, unsigned stages) const { return tails >> block % stages & 1; }
    DCCL_BOTH unsigned parity(unsigned block, unsigned stages) const { return on_landed(block, stages) ? ~(turns >> block % stages) & 1 : block / stages & 1; }
};

/** Rows and columns of tiles, and the parts of k. More rows than a CTA's are those of two, which hold half of what makes the columns each. */
struct GroupedPlan {
    unsigned tile_rows, tile_columns, splits;
    unsigned held_rows() const { return tile_rows < kTileM ? tile_rows : kTileM; }
    unsigned held_columns() const { return tile_rows > kTileM ? tile_columns / 2 : tile_columns; }
};

/**
 * As if the experts had equal shares of the rows, which the host does not know, or, where that makes more tiles, shares about equal that fill half of their last one. What a
 * plan takes, in nanoseconds, is what one CTA takes for its tiles, or two that share some of 256 x 256: a block of k takes 390 for one of these, 450 for one of 128 x 256 and
 * 280 for 128 x 128 (with every SM at work 396, 450 and 275 measured), a tile about one microsecond more, but what its results take to be stored at least (4.2 and 3.7
 * measured at four blocks), and the start of pairs four more; parts are stored in fp32, and added up by another launch (products that need it are small for pairs).
 * 16384 rows of 8 experts, 2048 x 5632, by pairs and by single CTAs: h 249 us and 288, dx 247 and 273, dW 278 and 289; of 64 experts, 2048 x 768, h with GELU 71 and 78,
 * dW 93 and 77; 5 experts of some 140 rows, 1001 x 2731 fp16, which have half of a pair's rows, h 24 and 20.
 * Up to 32 rows of an expert, forward: tiles of 32 x 64. Then reading the weights is all there is to do, and the tile's own rows should not be most of what it loads.
 */
inline GroupedPlan plan_grouped(int form, int sms, size_t rows, size_t experts, size_t m, size_t n, size_t k) {
    const size_t busy = experts < rows ? experts : rows, each = busy ? (rows + busy - 1) / busy : 0;
    if (form == EXPERTS_FORWARD && each <= 32) return {32, 64, 1};
    const size_t blocks = blocks_of(form == EXPERTS_WEIGHT ? each : k, kTileK);
    const size_t results = form == EXPERTS_WEIGHT ? experts * m : rows;
    GroupedPlan best = {kTileM, 256, 1};
    double least = 0;
    const struct { unsigned rows, columns, block, least, once; } shapes[] = {{2 * kTileM, 256, 390, 4200, 4000}, {kTileM, 256, 450, 3700, 0}, {kTileM, 128, 280, 1900, 0}};
    for (const auto& s : shapes) {
        const size_t shares = (rows + busy * s.rows / 2) / s.rows, workers = s.rows > kTileM ? sms / 2 : sms;
        const size_t equal = busy * blocks_of(each, s.rows), high = form == EXPERTS_WEIGHT ? experts * blocks_of(m, s.rows) : busy < 2 || equal > shares ? equal : shares;
        for (unsigned splits = 1; workers && splits <= 16 && (splits == 1 || (s.rows == kTileM && splits * 4 <= blocks)); splits++) {
            const size_t tiles = high * blocks_of(n, s.columns) * splits, rounds = (tiles + workers - 1) / workers;
            if (splits > 1 && rounds > 4) break;
            const size_t tile = (blocks + splits - 1) / splits * s.block + 1000;
            double cost = (double)rounds * (tile < s.least ? s.least : tile) + s.once;
            if (splits > 1) cost += 3000 + (double)results * n * 8 * splits / 5000;
            if (!least || cost < least) { least = cost; best = {s.rows, s.columns, splits}; }
        }
    }
    return best;
}

} // namespace dccl
