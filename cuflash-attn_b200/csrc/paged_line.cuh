#pragma once

// How the attention over a paged cache divides its work (paged_sm100.cu).
//
// A context is a run of query tokens with one key sequence: sequence b
// (ragged), or the shared prefix with every sequence's token, and each
// sequence's own keys with its one token (prefix decode).  The query heads of
// one K/V head (in chunks of gt <= 128 of them) are packed with the tokens
// into row tiles of tpt tokens x gt heads <= 128 rows.  A unit is one head chunk
// with two row tiles, with one where no second is left, or with few rows (at most
// few_rows in the whole context); it reads its keys and values once for all of its
// rows, up to 256, so a context's are read once per unit of a head chunk.  Its
// length is the number of keys its last token sees plus kUnitCost, doubled for two
// tiles; key block j (128 keys) lies at 128 j of it.  The units, one after the other (context, then head chunk, then
// row tiles), form a line that is cut into equal pieces, one per CTA.  There
// are two lines: units of row tiles, which the tensor cores bound, and units
// of few rows, which the loads of keys and values bound; CTA i takes piece i
// of the first and piece G - 1 - i of the second, so that few pieces of either
// kind do not meet on the same CTAs.  The lengths live in device memory, so
// every CTA works out the lines itself, in closed form per context (lengths
// linear in the keys rather than counted in blocks make the sum over a
// context's causal units an arithmetic series).  A piece that covers a whole
// ragged unit writes the result; all others write partials for a second
// kernel, and the piece with a unit's first block records which pieces those
// are.
//
// Plain integer code, host and device; small on purpose: the kernel's roles
// share the instruction caches, and unrolled or repeated copies of this code
// (divisions above all) made up a third of it.

#include <cuda_runtime.h>

#include "paged.cuh"

namespace cuflash {
namespace detail {

constexpr int kTileRows = 128;
constexpr int kBlockKeys = 128;

constexpr int kFewTile = 16;  // rows of a partial tile of few rows (ragged)

#ifdef __CUDACC__
#define CUFLASH_ROLLED _Pragma("unroll 1")
#else
#define CUFLASH_ROLLED
#endif

// What a unit costs besides its keys, in keys: 64 for the unused part of its last
// block, on average, and 1.5 blocks for the start and the end of a segment (3.3 us,
// where a block of two row tiles takes 2.2).  Too little, and the CTAs with short
// units are late.  With 127, 191, 255 and 383, per call in a graph: 16 mixed sequences
// 116.2, 114.6, 110.7 and 110.3 us, a prefix of 32768 keys before 128 sequences 154.4,
// 152.2, 150.7 and 154.9, one of 512 before 4 15.1, 14.7, 13.0 and 13.3.
constexpr int kUnitCost = 255;

enum UnitMode { kOneTile = 0, kTwoTiles = 1, kFew = 2 };
enum Line { kTiles = 0, kFewLine = 1 };

// One CTA's part of one unit.
struct Seg {
    int n_blk;      // key blocks; 0 ends the CTA's work
    int blk0;       // first key block
    int len;        // keys of the context
    int lim0;       // causal: last key the first token of tile 0 sees
    int tok0;       // first token of tile 0
    int tok_end;    // end of the context's tokens
    int head0;      // first query head
    int nh;         // query heads
    int hk;         // K/V head
    int ctx;        // sequence, or -1 for the shared prefix
    int mode;       // UnitMode
    int part_row;   // first partial row, -1: the whole unit, write the result
    int part_rows;  // rows of a partial tile
    int pad[3];
};
static_assert(sizeof(Seg) == 64, "Seg layout");

// How long a wait for a segment of n_blk blocks may last, in ticks of 1024 ns:
// `base`, the limit of a wait for a single block, and 64 for each block (they take
// 2 to 4 us).
__host__ __device__ __forceinline__ unsigned wait_ticks(unsigned base, int n_blk) {
    return base + 64u * static_cast<unsigned>(n_blk);
}

// The pieces of a unit: written by the one with its first block.  Prefix decode:
// of every unit; ragged: of the units that several pieces share, by piece.
struct Span {
    int first, last;
};
struct Split {
    int last;  // last piece of the unit, -1: none
    int tok0, tok_end, head0, nh, mode;
    int pad[2];
};

struct PagedLine {
    const int* prefix_len;
    const int* seq_lens;
    const int* cu_seqlens;
    int prefix_mode, causal;
    int num_tokens, B, hq, hkv, group;
    int gt, chunks, tpt;  // heads per tile, chunks of the group, tokens per tile
    int heads;            // head chunks: hkv * chunks
    int few_rows;         // contexts of at most this many rows are "few"
    int page_shift, max_prefix_pages, max_pages;
    int prefix_pairs;  // units per head chunk of the prefix
    int pieces;        // of each line: the CTAs of the launch
    int own_part_row;  // prefix decode: first partial row of the own-keys units
    int few_part_row;  // ragged: first partial row of units of few rows
    Span* span;        // prefix decode: [heads * prefix_pairs] prefix units, [B * heads] own
    Split* split;      // ragged: one per piece of each line
};

struct Ctx {
    int tok, ntok, len;
    int pairs;            // units per head chunk
    int last_mode;        // of the last one; the others have two tiles
    long long head_cost;  // line length of a head chunk
};

// Keys that the last token of a unit sees, at least 1 (ragged: a unit that sees
// none takes one masked block, which writes its rows).
__host__ __device__ __forceinline__ int unit_keys(const PagedLine& p, const Ctx& c, int pair) {
    int n = c.len;
    if (p.causal && pair < c.pairs - 1) n += (pair + 1) * 2 * p.tpt - c.ntok;
    return n > 0 ? n : 1;
}

__host__ __device__ __forceinline__ int unit_mode(const Ctx& c, int pair) {
    return pair < c.pairs - 1 ? static_cast<int>(kTwoTiles) : c.last_mode;
}

// Line length of the first n (two-tile) units of a head chunk: the sum over
// i = 1..n of max(off + i s, 1) + kUnitCost, doubled.
__host__ __device__ __forceinline__ long long pairs_cost(const PagedLine& p, const Ctx& c, int n) {
    const int s = p.causal ? 2 * p.tpt : 0;
    const int off = p.causal ? c.len - c.ntok : (c.len > 0 ? c.len : 1);
    int z = off < 0 ? -off / s : 0;  // units that see no key
    if (z > n) z = n;
    const long long m = n - z;
    const long long steps = (m * (m + 1)) / 2 + m * z;  // z + 1 + ... + n
    return 2 * (n * static_cast<long long>(kUnitCost) + z + m * off + steps * s);
}

__host__ __device__ __forceinline__ long long unit_length(const PagedLine& p, const Ctx& c, int pair) {
    return static_cast<long long>(unit_keys(p, c, pair) + kUnitCost) << (unit_mode(c, pair) == kTwoTiles);
}

// Context c: -1 is the shared prefix.
__host__ __device__ __forceinline__ Ctx load_ctx(const PagedLine& p, int c) {
    Ctx x;
    const bool shared = c < 0;
    x.len = clamp_len(shared ? *p.prefix_len : p.seq_lens[c],
                      (shared ? p.max_prefix_pages : p.max_pages) << p.page_shift);
    if (p.prefix_mode) {
        x.tok = shared ? 0 : c;
        x.ntok = shared ? p.B : 1;
    } else {
        x.tok = clamp_len(p.cu_seqlens[c], p.num_tokens);
        x.ntok = clamp_len(p.cu_seqlens[c + 1] - x.tok, p.num_tokens - x.tok);
    }
    const int tiles = (x.ntok + p.tpt - 1) / p.tpt;
    x.pairs = (tiles + 1) / 2;
    x.last_mode = (tiles & 1) == 0 ? kTwoTiles : (x.ntok * p.gt <= p.few_rows ? kFew : kOneTile);
    x.head_cost = 0;
    if (x.pairs > 0 && (x.len > 0 || !p.prefix_mode))
        x.head_cost = pairs_cost(p, x, x.pairs - 1) + unit_length(p, x, x.pairs - 1);
    return x;
}

// The line of a context's units: those of one context are all of one kind but
// the last, which has few rows only where it is the only one.
__host__ __device__ __forceinline__ int line_of(const Ctx& c) {
    return c.last_mode == kFew ? static_cast<int>(kFewLine) : static_cast<int>(kTiles);
}

// Length of a piece: at least a block of a two-tile unit, so that every piece
// between a unit's first and last one has a block of it.  (Longer ones make fewer
// partials to join, but a step costs more than that: one chunk of 33 tokens takes
// 17.7 us with 256, 21.6 with 384, 4 sequences behind 512 keys 12.8 and 14.7, and 16
// mixed sequences 111 either way.)
__host__ __device__ __forceinline__ long long piece_length(long long line, int pieces) {
    const int shift = line >> 31 ? 20 : 0;
    const long long per =
        static_cast<long long>(static_cast<unsigned>(line >> shift) / static_cast<unsigned>(pieces) + 1) << shift;
    return per < 2 * kBlockKeys ? 2 * kBlockKeys : per;
}

// y / d for quotients below 2^20: an estimate, put right.
__host__ __device__ __forceinline__ int quotient(long long y, long long d) {
#ifdef __CUDA_ARCH__
    int q = static_cast<int>(__fdividef(static_cast<float>(y), static_cast<float>(d)));
#else
    int q = static_cast<int>(static_cast<float>(y) / static_cast<float>(d));
#endif
    CUFLASH_ROLLED
    while (q * d > y) --q;
    CUFLASH_ROLLED
    while ((q + 1) * d <= y) ++q;
    return q;
}

// The piece of a line that CTA `cta` takes.
__host__ __device__ __forceinline__ int piece_index(const PagedLine& p, int line, int cta) {
    return line == kTiles ? cta : p.pieces - 1 - cta;
}

// Ragged: no unit starts in the CTA's pieces until its walk of them says so.  A
// CTA resets the records that its own walk writes, and no others: nothing orders
// it with another CTA, which may have walked its pieces before this one starts
// (where a kernel on another stream holds the SM), so a reset of that one's
// records would lose them, and with them the rows of the units they name.
__host__ __device__ __forceinline__ void reset_records(const PagedLine& p, int cta) {
    p.split[piece_index(p, kTiles, cta)].last = -1;
    p.split[p.pieces + piece_index(p, kFewLine, cta)].last = -1;
}

// Piece [x0, x1) of a line, unit by unit.
struct Walk {
    Ctx ctx;
    int c, hc, pair;           // context, head chunk, unit of it
    int line, piece, records;  // records: this walk writes them
    long long ub, x, x0, x1, per;  // line position of the unit, of the walk; the piece; its length
};

// Context c holds position x0 and starts at ctx_base.
__host__ __device__ __forceinline__ void walk_start(const PagedLine& p, Walk& w, const Ctx& ctx, int c,
                                                    long long ctx_base, long long x0, long long x1,
                                                    long long per, int line, int piece, bool records) {
    w.ctx = ctx;
    w.c = c;
    w.line = line;
    w.piece = piece;
    w.records = records;
    w.x = w.x0 = x0;
    w.x1 = x1;
    w.per = per;
    w.hc = quotient(x0 - ctx_base, ctx.head_cost);
    const long long base = ctx_base + w.hc * ctx.head_cost;
    int lo = 0, hi = ctx.pairs - 1;  // the last unit that does not start behind x0
    w.ub = base;
    CUFLASH_ROLLED
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        const long long at = base + pairs_cost(p, ctx, mid);
        if (at <= x0) {
            lo = mid;
            w.ub = at;
        } else {
            hi = mid - 1;
        }
    }
    w.pair = lo;
}

// The next segment; false at the end.  next_ctx(c, line, ctx): the first
// context behind c with units on the line.
template <typename NextCtx>
__host__ __device__ __forceinline__ bool walk_next(const PagedLine& p, Walk& w, Seg& sg,
                                                   const NextCtx& next_ctx) {
    CUFLASH_ROLLED
    while (w.x < w.x1) {
        const int mode = unit_mode(w.ctx, w.pair);
        const int keys = unit_keys(p, w.ctx, w.pair);
        const int nb = (keys + kBlockKeys - 1) / kBlockKeys;
        const int two = mode == kTwoTiles ? 1 : 0;
        const int sh = 7 + two;  // line length of a block: 128, doubled
        const int blk0 = static_cast<int>((w.x - w.ub + (1 << sh) - 1) >> sh);
        const long long end = (w.x1 - w.ub + (1 << sh) - 1) >> sh;
        const int blk1 = end < nb ? static_cast<int>(end) : nb;
        const bool some = blk1 > blk0;
        if (some) {
            sg.n_blk = blk1 - blk0;
            sg.blk0 = blk0;
            sg.len = w.ctx.len;
            sg.lim0 = w.ctx.len - w.ctx.ntok + w.pair * 2 * p.tpt;
            sg.tok0 = w.ctx.tok + w.pair * 2 * p.tpt;
            sg.tok_end = w.ctx.tok + w.ctx.ntok;
            sg.hk = p.chunks == 1 ? w.hc : w.hc / p.chunks;
            const int ch = w.hc - sg.hk * p.chunks;
            sg.head0 = sg.hk * p.group + ch * p.gt;
            sg.nh = p.group - ch * p.gt < p.gt ? p.group - ch * p.gt : p.gt;
            sg.ctx = w.c;
            sg.mode = mode;
            sg.part_rows = kTileRows;
            const bool first = blk0 == 0;
            int last = w.piece;
            if (first && blk1 < nb)
                last += quotient(w.ub + (static_cast<long long>(nb - 1) << sh) - w.x0, w.per);
            if (p.prefix_mode) {
                int u = w.hc * p.prefix_pairs + w.pair;
                if (w.c < 0) {
                    sg.part_row = (u + w.piece) * (2 * kTileRows);
                } else {
                    u = w.c * p.heads + w.hc;
                    sg.part_row = p.own_part_row + (u + w.piece) * p.gt;
                    sg.part_rows = p.gt;
                    u += p.heads * p.prefix_pairs;
                }
                if (first && w.records) p.span[u] = Span{w.piece, last};
            } else if (first && blk1 == nb) {
                sg.part_row = -1;
            } else {
                const int slot = 2 * w.piece + (first ? 1 : 0);
                sg.part_row = w.line == kFewLine ? p.few_part_row + slot * kFewTile : slot * (2 * kTileRows);
                if (w.line == kFewLine) sg.part_rows = kFewTile;
                if (first && w.records)
                    p.split[w.line * p.pieces + w.piece] =
                        Split{last, sg.tok0, sg.tok_end, sg.head0, sg.nh, mode, {0, 0}};
            }
        }
        w.ub += static_cast<long long>(keys + kUnitCost) << two;
        w.x = w.ub;
        if (++w.pair == w.ctx.pairs) {
            w.pair = 0;
            if (++w.hc == p.heads) {
                w.hc = 0;
                if (w.x < w.x1) w.c = next_ctx(w.c, w.line, w.ctx);
            }
        }
        if (some) return true;
    }
    return false;
}

// Row tiles of the query heads and tokens.
inline void set_tiles(PagedLine& p, int few_rows) {
    p.group = p.hq / p.hkv;
    p.chunks = (p.group + kTileRows - 1) / kTileRows;
    p.gt = (p.group + p.chunks - 1) / p.chunks;
    p.tpt = kTileRows / p.gt;
    p.heads = p.hkv * p.chunks;
    p.few_rows = few_rows;
    p.prefix_pairs = ((p.B + p.tpt - 1) / p.tpt + 1) / 2;
}

// Partial rows and record bytes of a launch of `grid` CTAs; false if the rows
// could pass 32 bits.  Going along a line, each segment starts a new unit, a
// new piece or both, so unit + piece numbers them; ragged, only a piece's first
// and last segment are partial.
inline bool set_parts(PagedLine& p, int grid, long long& rows, long long& records) {
    p.pieces = grid;
    const long long heads = p.heads;
    long long own = 0, few = 0;
    if (p.prefix_mode) {
        own = (heads * p.prefix_pairs + grid) * 2 * kTileRows;
        rows = own + (heads * p.B + grid) * p.gt;
        records = heads * (p.prefix_pairs + p.B) * static_cast<long long>(sizeof(Span));
    } else {
        few = 2LL * grid * 2 * kTileRows;
        rows = few + 2LL * grid * kFewTile;
        records = 2 * grid * static_cast<long long>(sizeof(Split));
    }
    if (rows > 0x7fffffffLL || heads * (p.prefix_pairs + static_cast<long long>(p.B)) > 0x7fffffffLL) return false;
    p.own_part_row = static_cast<int>(own);
    p.few_part_row = static_cast<int>(few);
    return true;
}

}  // namespace detail
}  // namespace cuflash
