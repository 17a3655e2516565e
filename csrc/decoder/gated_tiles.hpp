/**
 * How the products of a gated layer are cut into tiles, which CTA takes which, and what one that could not finish leaves behind. Nothing here
 * needs CUDA, so that tests run it on the host.
 */
#pragma once
#include <cstddef>
#include <cstdint>

#ifdef __CUDACC__
#define DCCL_BOTH __host__ __device__ __forceinline__
#else
#define DCCL_BOTH inline
#endif

namespace dccl {

enum Form {
    GATED,          // C = act(x Wg^T) .* (x Wu^T): both operands contiguous along k; the columns of a tile are half of Wg and half of Wu
    INPUT_GRAD,     // dx = dg Wg + du Wu: k runs through ffn twice; W is contiguous along the columns
    WEIGHT_GRAD,    // dW = dg^T x, du^T x: k are the tokens, both operands contiguous along rows and columns of the result
};

constexpr int kTileM = 128, kTileK = 64;

struct Tiling {
    unsigned m, n;                                                  // rows and columns of the result
    unsigned tiles_m, tiles_n, batch, splits, k_blocks;             // k_blocks: of one tile over all its k
};

struct Results {
    void *c0, *c1;                  // of 16 bits (c1: second of the batch)
    float *g, *u;                   // GATED: the products, or null
    size_t pre_stride;
    float* partial;                 // [split][batch or gate, up][m][partial_stride] where splits > 1
    size_t partial_stride;
};

DCCL_BOTH size_t up_to(size_t v, size_t step) { return (v + step - 1) / step * step; }
DCCL_BOTH unsigned blocks_of(size_t v, size_t block) { return (unsigned)((v + block - 1) / block); }

/** Tile number -> place. Groups of 16 rows of tiles are walked column by column, so that the tiles of one moment share operands in L2. */
struct Place { unsigned m, n, batch, split; };
DCCL_BOTH Place place_of(unsigned tile, const Tiling& a) {
    Place p;
    p.split = tile % a.splits;
    tile /= a.splits;
    const unsigned per_batch = a.tiles_m * a.tiles_n;
    p.batch = tile / per_batch;
    tile %= per_batch;
    const unsigned group = tile / (16 * a.tiles_n), first = group * 16, rows = a.tiles_m - first < 16 ? a.tiles_m - first : 16;
    tile -= first * a.tiles_n;
    p.m = first + tile % rows;
    p.n = tile / rows;
    return p;
}

constexpr uint16_t kNoResult16 = 0x7fff;        // a NaN of both 16-bit types

/** One row of 16-bit results, and of the products where they are kept, as NaN. */
DCCL_BOTH void mark_incomplete(void* h, float* g, float* u, size_t at, size_t pre_at) {
    reinterpret_cast<uint16_t*>(h)[at] = kNoResult16;
    if (g) g[pre_at] = u[pre_at] = __builtin_nanf("");
}

/** NaN in all that one CTA stores (rank: of a pair; first, step: its tiles), by each of its threads. k_join hands the NaN of a part on. */
DCCL_BOTH void mark_incomplete(int form, const Tiling& a, const Results& to, unsigned tile_rows, unsigned tile_columns, unsigned rank, unsigned first, unsigned step, unsigned thread,
                               unsigned threads) {
    for (unsigned tile = first; tile < a.tiles_m * a.tiles_n * a.batch * a.splits; tile += step) {
        const Place p = place_of(tile, a);
        for (unsigned i = thread; i < kTileM * tile_columns; i += threads) {
            const size_t row = (size_t)p.m * tile_rows + rank * kTileM + i / tile_columns, column = (size_t)p.n * tile_columns + i % tile_columns;
            if (row >= a.m || column >= a.n) continue;
            if (a.splits == 1) {
                mark_incomplete(p.batch ? to.c1 : to.c0, form == GATED ? to.g : nullptr, to.u, row * a.n + column, row * to.pre_stride + column);
            } else {
                const unsigned planes = form == GATED ? 2 : a.batch;
                for (unsigned w = 0; w < planes; w++)
                    if (form == GATED || w == p.batch) to.partial[(((size_t)p.split * planes + w) * a.m + row) * to.partial_stride + column] = __builtin_nanf("");
            }
        }
    }
}

/** Tiles of a product, 256 columns wide or 128, and the parts that its k is cut into. */
struct GemmPlan { bool pair; int columns; unsigned tiles_m, tiles_n, batch, splits, k_blocks; size_t partial_bytes; };

inline GemmPlan plan_gemm(int sms, int form, size_t m, size_t n, size_t k) {
    GemmPlan p;
    p.pair = m > kTileM;
    p.tiles_m = blocks_of(m, p.pair ? 2 * kTileM : kTileM);
    p.batch = form == WEIGHT_GRAD ? 2 : 1;
    p.k_blocks = blocks_of(k, kTileK) * (form == INPUT_GRAD ? 2 : 1);
    const unsigned workers = p.pair ? sms / 2 : sms;
    const auto tiles_of = [&](int columns) { return (size_t)p.tiles_m * blocks_of(n, form == GATED ? columns / 2 : columns) * p.batch; };
    // At least four blocks of k for a part. Forward and backward with 1, 2, 4, 8, and uncut: 129 x 2048 x 512 51, 42, 33, 33 and 37 us, 200 x 1000 x 384
    // 39, 32, 29, 29 and 30, 520 x 512 x 1024 41, 41, 38, 32 and 36; 1 x 2048 x 5632 55 with any and 93 uncut.
    const auto splits_of = [&](int columns) {
        const size_t tiles = tiles_of(columns), most = p.k_blocks / 4, s = workers / (tiles ? tiles : 1);
        return s > most ? (most ? most : 1) : s ? s : 1;
    };
    // Rounds of tiles, and what a round takes: a tile of half the width loads three quarters of the bytes, which is what these products wait for. Forward / with
    // the backward pass, bf16, all tiles of 128 and all of 256 columns: 200 x 1000 x 384 9.9 / 28.6 and 12.0 / 33.5 us, 300 x 2048 x 5632 36.6 / 109 and
    // 29.1 / 88, 2000 x 2048 x 5632 137 / 363 and 68 / 234. It misses where k is short: 545 x 520 x 816, cut in two at 256, 9.1 / 31.7 and 12.4 / 39.1.
    const auto cost = [&](int columns) { return (columns == 128 ? 3 : 4) * 64 * ((tiles_of(columns) + workers - 1) / workers) / splits_of(columns); };
    p.columns = cost(128) < cost(256) ? 128 : 256;
    p.tiles_n = blocks_of(n, form == GATED ? p.columns / 2 : p.columns);
    p.splits = (unsigned)splits_of(p.columns);
    p.partial_bytes = p.splits > 1 ? (size_t)p.splits * (form == INPUT_GRAD ? 1 : 2) * m * up_to(n, 4) * sizeof(float) : 0;
    return p;
}

/** Whether k_gated_few takes a call: for wider layers than it has CTAs for, splits of k read the weights faster. This kernel and the general one, bf16: 2048 x 5632,
 *  1 token 14.0 and 18.1 us, 40 tokens 15.4 and 16.8, 100 tokens 20.9 and 18.0, 128 tokens 21.8 and 18.8; 256 x 688, 16 tokens 5.0 and 5.8, 128 tokens 8.6 and 6.1;
 *  16 tokens of 8192 x 296, which the general one takes, 39.8 and 15.0, of 4096 x 576 22.2 and 11.6, of 2048 x 296 13.1 and 9.3. So both borders lie
 *  higher than they should. */
inline bool few_tokens(int sms, size_t tokens, size_t width, size_t ffn) {
    return tokens <= 128 && (width <= 4096 || 2 * blocks_of(ffn, 8) >= (size_t)sms);
}

/** Rows of each weight for one CTA of k_gated_few, two of which share an SM: as many CTAs as there is room for, in as few rounds as it takes,
 *  but not less than 32 rows while every SM has a CTA, since each CTA reads x as well (5632 rows: 32 take 13.7 us for one token and 16.9 for
 *  64, 24 take 14.3 and 19.9, and one CTA of 40 rows per SM 13.8 and 19.0). */
inline unsigned few_rows(int sms, size_t ffn) {
    const size_t room = 2 * (size_t)sms, rounds = (ffn + 64 * room - 1) / (64 * room);
    const unsigned rows = (unsigned)up_to((ffn + room * rounds - 1) / (room * rounds), 8);
    return rows < 32 && ffn >= 32 * (size_t)sms ? 32 : rows;
}

} // namespace dccl
