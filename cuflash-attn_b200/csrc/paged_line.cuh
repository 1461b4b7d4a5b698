#pragma once

// How the attention over a paged cache divides its work (paged_sm100.cu).
//
// A context is a run of query tokens with one key sequence: sequence b
// (ragged), or the shared prefix with every sequence's token, and each
// sequence's own keys with its one token (prefix decode).  The query heads of
// one K/V head (in chunks of gt <= 128 of them) are packed with the tokens
// into row tiles of tpt tokens x gt heads <= 128 rows, so that every key and
// value is read once for all of them.  A unit is one head chunk with two row
// tiles, with one where no second is left, or with few rows (at most kFewRows
// in the whole context).  Its length is its number of 128-key blocks, weighted
// by the kind of unit.  The units' lengths, one after the other (context, then
// head chunk, then row tiles), form a line that is cut into pieces of `per`,
// one per CTA.  The lengths live in device memory, so every CTA works out the
// line itself, in closed form per context.  A piece that covers a whole ragged
// unit writes the result; all others write partials for a second kernel.
//
// Plain integer code, host and device.

#include <cuda_runtime.h>

#include "paged.cuh"

namespace cuflash {
namespace detail {

constexpr int kTileRows = 128;
constexpr int kBlockKeys = 128;

enum UnitMode { kOneTile = 0, kTwoTiles = 1, kFew = 2 };

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

// A ragged unit whose blocks several CTAs share: written by the first.
struct Split {
    int last;  // last CTA of the unit, -1: none
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
    int few_rows;         // contexts of at most this many rows are "few"
    int page_shift, max_prefix_pages, max_pages;
    int w_two, w_one, w_few;  // line length of a block
    int min_per;              // shortest piece, at least the largest weight
    int own_part_row;         // first partial row of the own-keys units
    int* per;                 // piece length, for the second kernel
    int* unit_start;          // prefix decode: line position of own-keys unit u
    Split* split;             // ragged: one per CTA
};

// sum over i in [0, n) of floor((a i + b) / m): the usual Euclid-like
// reduction (a, b >= 0, m > 0; n, m and b mod m small enough for 32 bits).
__host__ __device__ __forceinline__ int floor_sum(int n, int m, int a, int b) {
    int s = 0;
    while (n > 0) {
        s += static_cast<int>(static_cast<long long>(n) * (n - 1) / 2) * (a / m) + n * (b / m);
        a %= m;
        b %= m;
        const int top = a * n + b;
        n = top / m;
        b = top % m;
        const int t = m;
        m = a;
        a = t;
        if (m == 0) break;  // then top < the old m, so n == 0
    }
    return s;
}

struct Ctx {
    int tok, ntok, len;
    int pairs;      // units per head chunk
    int last_mode;  // of the last one; the others have two tiles
    int head_cost;  // line length of a head chunk
};

__host__ __device__ __forceinline__ int unit_blocks(const PagedLine& p, const Ctx& c, int pair) {
    int vis = c.len;
    if (p.causal && pair < c.pairs - 1)
        vis = c.len - c.ntok + (pair + 1) * 2 * p.tpt;  // what its last token sees
    const int nb = (vis + kBlockKeys - 1) / kBlockKeys;
    // ragged: a unit that sees no key takes one masked block, which writes its rows
    return p.prefix_mode ? nb : (vis > 0 ? nb : 1);
}

__host__ __device__ __forceinline__ int unit_mode(const Ctx& c, int pair) {
    return pair < c.pairs - 1 ? static_cast<int>(kTwoTiles) : c.last_mode;
}

__host__ __device__ __forceinline__ int mode_weight(const PagedLine& p, int mode) {
    return mode == kTwoTiles ? p.w_two : (mode == kOneTile ? p.w_one : p.w_few);
}

// Line length of the first `pairs` (two-tile) units of a head chunk.
__host__ __device__ __forceinline__ int pairs_cost(const PagedLine& p, const Ctx& c, int pairs) {
    if (pairs == 0) return 0;
    if (!p.causal) return pairs * unit_blocks(p, c, 0) * p.w_two;
    const int s = 2 * p.tpt;
    const int off = c.len - c.ntok;
    // units whose last token sees at most 128 keys take one block
    int ones = 128 - off >= 0 ? (128 - off) / s : 0;
    if (ones > pairs) ones = pairs;
    return (ones + floor_sum(pairs - ones, 128, s, off + (ones + 1) * s + 127)) * p.w_two;
}

// Context c: -1 is the shared prefix.
__host__ __device__ __forceinline__ Ctx load_ctx(const PagedLine& p, int c) {
    Ctx x;
    if (p.prefix_mode) {
        x.tok = c < 0 ? 0 : c;
        x.ntok = c < 0 ? p.B : 1;
        x.len = c < 0 ? clamp_len(*p.prefix_len, p.max_prefix_pages << p.page_shift)
                      : clamp_len(p.seq_lens[c], p.max_pages << p.page_shift);
    } else {
        x.tok = clamp_len(p.cu_seqlens[c], p.num_tokens);
        x.ntok = clamp_len(p.cu_seqlens[c + 1] - x.tok, p.num_tokens - x.tok);
        x.len = clamp_len(p.seq_lens[c], p.max_pages << p.page_shift);
    }
    const int tiles = (x.ntok + p.tpt - 1) / p.tpt;
    x.pairs = (tiles + 1) / 2;
    x.last_mode = (tiles & 1) == 0 ? kTwoTiles : (x.ntok * p.gt <= p.few_rows ? kFew : kOneTile);
    x.head_cost = 0;
    if (x.pairs > 0 && (x.len > 0 || !p.prefix_mode))
        x.head_cost = pairs_cost(p, x, x.pairs - 1) +
                      unit_blocks(p, x, x.pairs - 1) * mode_weight(p, x.last_mode);
    return x;
}

// The piece [x0, x1) of the line that belongs to CTA `cta`, unit by unit.
struct Walk {
    Ctx ctx;
    int c, hc, pair, cta;   // context, head chunk, unit of it
    int ub, x, x1, per;     // line position of the unit, of the walk, its end
};

// Context c holds position x0 and starts at ctx_base.
__host__ __device__ __forceinline__ void walk_start(const PagedLine& p, Walk& w, const Ctx& ctx,
                                                    int c, int ctx_base, int x0, int x1, int per,
                                                    int cta) {
    w.ctx = ctx;
    w.c = c;
    w.cta = cta;
    w.x = x0;
    w.x1 = x1;
    w.per = per;
    const int y = x0 - ctx_base;
    w.hc = y / ctx.head_cost;
    const int z = y - w.hc * ctx.head_cost;
    int lo = 0, hi = ctx.pairs;  // the unit of the head chunk that z falls into
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (pairs_cost(p, ctx, mid) <= z)
            lo = mid;
        else
            hi = mid;
    }
    w.pair = lo;
    w.ub = ctx_base + w.hc * ctx.head_cost + pairs_cost(p, ctx, lo);
}

// The next segment; false at the end.  Records where own-keys units start and
// which ragged units several CTAs share, for the second kernel.
__host__ __device__ __forceinline__ bool walk_next(const PagedLine& p, Walk& w, Seg& sg) {
    const int heads = p.hkv * p.chunks;
    while (w.x < w.x1) {
        const int nb = unit_blocks(p, w.ctx, w.pair);
        const int mode = unit_mode(w.ctx, w.pair);
        const int wt = mode_weight(p, mode);
        const int blk0 = (w.x - w.ub + wt - 1) / wt;
        const int end = (w.x1 - w.ub + wt - 1) / wt;
        const int blk1 = end < nb ? end : nb;
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
            if (p.prefix_mode) {
                if (w.c < 0) {
                    sg.part_row = (w.hc * w.ctx.pairs + w.pair + w.cta) * (2 * kTileRows);
                } else {
                    const int u = w.c * heads + w.hc;
                    if (blk0 == 0) p.unit_start[u] = w.ub;
                    sg.part_row = p.own_part_row + (u + w.cta) * p.gt;
                    sg.part_rows = p.gt;
                }
            } else if (blk0 == 0 && blk1 == nb) {
                sg.part_row = -1;
            } else {
                sg.part_row = (2 * w.cta + (blk0 == 0 ? 1 : 0)) * (2 * kTileRows);
                if (blk0 == 0) {
                    Split sp;
                    sp.last = (w.ub + (nb - 1) * wt) / w.per;
                    sp.tok0 = sg.tok0;
                    sp.tok_end = sg.tok_end;
                    sp.head0 = sg.head0;
                    sp.nh = sg.nh;
                    sp.mode = mode;
                    p.split[w.cta] = sp;
                }
            }
        }
        w.ub += nb * wt;
        w.x = w.ub;
        if (++w.pair == w.ctx.pairs) {
            w.pair = 0;
            if (++w.hc == heads) {
                w.hc = 0;
                while (w.x < w.x1 && w.c < p.B - 1) {
                    w.ctx = load_ctx(p, ++w.c);
                    if (w.ctx.head_cost != 0) break;
                }
            }
        }
        if (some) return true;
    }
    return false;
}

// Where the partials of the output row (sequence b, query head h) are: row r1
// of n1 tiles of kTileRows rows, 2 kTileRows apart from row1 on (the prefix),
// and row r2 of n2 tiles of gt rows from row2 on (own keys).
struct PrefixParts {
    int n1, row1, r1;
    int n2, row2, r2;
};

__host__ __device__ __forceinline__ PrefixParts prefix_parts(const PagedLine& p, int per,
                                                             const Ctx& pre, const Ctx& own, int b,
                                                             int hc, int hr) {
    PrefixParts q = {0, 0, 0, 0, 0, 0};
    if (pre.len > 0) {
        const int tile = b / p.tpt;
        const int pair = tile >> 1;
        const int nb = unit_blocks(p, pre, pair);
        const int ub = hc * pre.head_cost + pairs_cost(p, pre, pair);
        const int i0 = ub / per;
        q.n1 = (ub + (nb - 1) * mode_weight(p, unit_mode(pre, pair))) / per - i0 + 1;
        q.row1 = (hc * pre.pairs + pair + i0) * (2 * kTileRows) + (tile & 1) * kTileRows;
        q.r1 = (b - tile * p.tpt) * p.gt + hr;
    }
    if (own.len > 0) {
        const int u = b * p.hkv * p.chunks + hc;
        const int nb = unit_blocks(p, own, 0);
        const int ub = p.unit_start[u];
        const int i0 = ub / per;
        q.n2 = (ub + (nb - 1) * mode_weight(p, own.last_mode)) / per - i0 + 1;
        q.row2 = p.own_part_row + (u + i0) * p.gt;
        q.r2 = hr;
    }
    return q;
}

// Row tiles of the query heads and tokens.
inline void set_tiles(PagedLine& p, int few_rows) {
    p.group = p.hq / p.hkv;
    p.chunks = (p.group + kTileRows - 1) / kTileRows;
    p.gt = (p.group + p.chunks - 1) / p.chunks;
    p.tpt = kTileRows / p.gt;
    p.few_rows = few_rows;
    p.w_two = 2;
    p.w_one = 1;
    p.w_few = 1;
    p.min_per = 2;
}

// Partial rows and record bytes of a launch of `grid` CTAs; false if the line
// or the rows could pass 32 bits.  Going along the line, each piece starts a
// new unit, a new CTA or both, so unit + CTA numbers the pieces; ragged, only
// a CTA's first and last piece are partial.
inline bool set_parts(PagedLine& p, int grid, long long& rows, long long& records) {
    const long long heads = static_cast<long long>(p.hkv) * p.chunks;
    const long long nb =
        ((static_cast<long long>(p.max_pages) << p.page_shift) + kBlockKeys - 1) / kBlockKeys;
    const long long pairs = (static_cast<long long>(p.num_tokens) + 2 * p.tpt - 1) / (2 * p.tpt);
    long long line, own = 0;
    if (p.prefix_mode) {
        const long long nbp =
            ((static_cast<long long>(p.max_prefix_pages) << p.page_shift) + kBlockKeys - 1) / kBlockKeys;
        line = heads * (pairs * nbp + p.B * nb) * p.w_two;
        own = (heads * pairs + grid) * 2 * kTileRows;
        rows = own + (heads * p.B + grid) * p.gt;
        records = heads * p.B * static_cast<long long>(sizeof(int));
    } else {
        line = heads * (pairs + p.B) * nb * p.w_two;
        rows = 2LL * grid * 2 * kTileRows;
        records = grid * static_cast<long long>(sizeof(Split));
    }
    if (line > 0x7fffffffLL - 4096 || rows > 0x7fffffffLL) return false;
    p.own_part_row = static_cast<int>(own);
    return true;
}

}  // namespace detail
}  // namespace cuflash
