// Attention over a paged KV cache for serving (no reference counterpart: the
// reference has no KV cache):
//   * ragged attention of several new tokens per sequence (prompts, chunks of
//     prompts, single tokens) against the sequence's pages;
//   * decode of one token per sequence for a batch whose sequences share a
//     long prefix, whose scores are computed for all of them at once.

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "paged.cuh"

namespace cuflash {
namespace detail {

namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------------------
// CUDA-core kernel for pages of fewer than 8 rows, which a swizzled TMA box
// cannot place (its rows repeat every 8): one block per (token, query head).  Lane
// groups of D/8 lanes read one cache row each (16 bytes per lane), the dot
// product is reduced over the group with shuffles, and every group keeps its
// own running maximum, sum and output (fp32), merged once at the end.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 128;

template <typename T>
struct PagedParams {
    const T* Q;  // [tokens, hq, D]
    const T* K;  // [num_pages, page_size, hkv, D]
    const T* V;
    T* O;
    float* L;
    const int* prefix_table;  // shared prefix (nullptr: none)
    const int* prefix_len;
    const int* block_table;   // [B, max_pages]
    const int* seq_lens;      // [B]
    const int* cu_seqlens;    // [B + 1]; nullptr: token t is sequence t's only one
    int num_tokens, B, hq, hkv;
    int page_shift, max_prefix_pages, max_pages, num_pages;
    int causal;
    float scale_log2;
};

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads)
    paged_row_kernel(const PagedParams<T> p) {
    constexpr int LPR = D / 8;
    constexpr int RPW = 32 / LPR;
    constexpr int G = (kRowThreads / 32) * RPW;
    constexpr int U = 4;
    __shared__ float s_m[G];
    __shared__ float s_l[G];
    __shared__ float s_acc[G][D];
    const int t = blockIdx.x / p.hq;
    const int h = blockIdx.x - t * p.hq;
    const int hk = h / (p.hq / p.hkv);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int li = lane % LPR;
    const int grp = warp * RPW + lane / LPR;

    int b = t, from_end = 1;
    if (p.cu_seqlens != nullptr) {
        b = sequence_of_token(p.cu_seqlens, p.B, t);
        if (b < 0) return;  // behind the last sequence: left as it was
        from_end = p.cu_seqlens[b + 1] - t;
    }
    const long long qrow = static_cast<long long>(t) * p.hq + h;
    float q[8];
    {
        const uint4 v = *reinterpret_cast<const uint4*>(p.Q + qrow * D + li * 8);
        const uint32_t vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = DType<T>::unpack2(vs[e]);
            q[2 * e] = f.x * p.scale_log2;
            q[2 * e + 1] = f.y * p.scale_log2;
        }
    }
    float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;

    // one pass over the `n` keys of a page table
    auto attend = [&](const int* table, int n) {
        for (int r0 = warp * RPW; r0 < n; r0 += G * U) {  // warp-uniform bound
            uint4 kv[U], vv[U];
            float s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int row = r0 + u * G + lane / LPR;
                kv[u] = make_uint4(0, 0, 0, 0);
                vv[u] = make_uint4(0, 0, 0, 0);
                if (row < n) {
                    int page = table[row >> p.page_shift];
                    page = min(max(page, 0), p.num_pages - 1);
                    const long long slot = (static_cast<long long>(page) << p.page_shift) +
                                           (row & ((1 << p.page_shift) - 1));
                    const long long off = (slot * p.hkv + hk) * D + li * 8;
                    kv[u] = *reinterpret_cast<const uint4*>(p.K + off);
                    vv[u] = *reinterpret_cast<const uint4*>(p.V + off);
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t ks[4] = {kv[u].x, kv[u].y, kv[u].z, kv[u].w};
                float dot = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = DType<T>::unpack2(ks[e]);
                    dot = fmaf(q[2 * e], f.x, fmaf(q[2 * e + 1], f.y, dot));
                }
#pragma unroll
                for (int off = LPR / 2; off > 0; off >>= 1)
                    dot += __shfl_xor_sync(0xffffffffu, dot, off);
                s[u] = r0 + u * G + lane / LPR < n ? dot : -INFINITY;
                mx = fmaxf(mx, s[u]);
            }
            const float m_new = fmaxf(m, mx);
            if (m_new == -INFINITY) continue;
            const float alpha = sm100::ex2_approx(m - m_new);
            l *= alpha;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] *= alpha;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float pr = sm100::ex2_approx(s[u] - m_new);
                l += pr;
                const uint32_t vs[4] = {vv[u].x, vv[u].y, vv[u].z, vv[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = DType<T>::unpack2(vs[e]);
                    acc[2 * e] = fmaf(pr, f.x, acc[2 * e]);
                    acc[2 * e + 1] = fmaf(pr, f.y, acc[2 * e + 1]);
                }
            }
            m = m_new;
        }
    };
    if (p.prefix_table != nullptr)
        attend(p.prefix_table, clamp_len(*p.prefix_len, p.max_prefix_pages << p.page_shift));
    int n = min(max(p.seq_lens[b], 0), p.max_pages << p.page_shift);
    if (p.causal) n -= from_end - 1;
    attend(p.block_table + static_cast<long long>(b) * p.max_pages, n);

    if (li == 0) {
        s_m[grp] = m;
        s_l[grp] = l;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s_acc[grp][li * 8 + e] = acc[e];
    __syncthreads();
    const int d = threadIdx.x;
    if (d < D) {
        float M = -INFINITY;
        for (int g = 0; g < G; ++g) M = fmaxf(M, s_m[g]);
        float lt = 0.f, o = 0.f;
        if (M != -INFINITY)
            for (int g = 0; g < G; ++g) {
                const float w = sm100::ex2_approx(s_m[g] - M);
                lt = fmaf(w, s_l[g], lt);
                o = fmaf(w, s_acc[g][d], o);
            }
        p.O[qrow * D + d] = DType<T>::from_float(lt > 0.f ? o / lt : 0.f);
        if (d == 0) p.L[qrow] = lt > 0.f ? (M + log2f(lt)) * kLn2 : -INFINITY;
    }
}

template <typename T, int D>
FlashAttentionError paged_row(const PagedParams<T>& p, cudaStream_t stream) {
    paged_row_kernel<T, D><<<static_cast<unsigned>(p.num_tokens * p.hq), kRowThreads, 0, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? FlashAttentionError::SUCCESS
                                             : FlashAttentionError::CUDA_ERROR;
}

// ---------------------------------------------------------------------------
// Tensor-core kernel (pages of 8 rows and more).
//
// Work.  A context is a run of query tokens with one key sequence: sequence b
// (ragged), or the shared prefix with every sequence's token, and each
// sequence's own keys with its one token (prefix decode).  The query heads of
// one K/V head are packed with the tokens into row tiles of M = 128 (tpt tokens
// x gt heads), so K/V rows are read once for all of them.  A unit is one K/V
// head (and chunk of gt <= 128 query heads) with two row tiles, or one where
// no second is left; its length is its number of 128-key blocks.  All units'
// blocks, one after the other, form a line that is cut into equal pieces, one
// per CTA: lengths live in device memory, so every CTA sums the contexts'
// lengths itself and finds its piece.  A piece that covers a unit writes the
// result; other pieces write normalised fp32 partials with their
// log2-sum-exp, joined by a second kernel in a fixed order.
//
// CTA.  Two streams of 128 softmax threads (one per row) take the steps
// (row tile x key block) in turn, so one stream's softmax runs under the
// other's products:
//   two tiles:  tile 0 and tile 1 of the same block (K/V staged once);
//   one tile:   alternate blocks of the same tile, each stream with its own
//               maximum, sum and output; the stream that had the first block
//               joins both from TMEM at the end of the piece.
//   warp 0      TMA producer (query tiles, K/V blocks through a ring of
//               slots, one box per page and 64 columns, one lane each)
//   warp 1      tcgen05.mma issuer: S(n+2) behind O(n)
//   warp 2      walks the units and hands out segment descriptors
//   warps 4-11  softmax and epilogue
// S_t = Q K^T (M = N = 128) in TMEM columns [128 t, +128), P_t in 16 bits over
// its first half, O_t += P V in [256 + 128 t, +D).  Arithmetic as in the dense
// forward: fp32 statistics in the log2 domain, O rescaled only where a row's
// maximum grows by more than 2^8, P rounded to the input type for its product.
// ---------------------------------------------------------------------------
__device__ sm100::StatusWord g_paged_status;

constexpr int kTcThreads = 384;
constexpr int kSegRing = 4;
constexpr int kTileRows = 128;
constexpr int kBlockKeys = 128;
constexpr float kRescale = 8.0f;  // log2 units

template <int D>
struct PagedGeom {
    static constexpr int kRowBytes = D * 2;
    static constexpr int kSwz = kRowBytes >= 128 ? 128 : kRowBytes;
    static constexpr int kCbElems = kSwz / 2;
    static constexpr int kNumCb = D / kCbElems;
    static constexpr int kCbBytes = kTileRows * kSwz;
    static constexpr int kTileBytes = kTileRows * kRowBytes;
    // K and V blocks share one ring; at D = 128 five slots of 32 KB fill what
    // the two query tiles leave
    static constexpr int kSlots = D == 128 ? 5 : (D == 64 ? 10 : 12);
    static constexpr uint32_t kLayout = kSwz == 128 ? sm100::kLayoutSw128 : sm100::kLayoutSw64;
    static constexpr int kOffRing = 2 * kTileBytes;
    static constexpr int kOffMl = kOffRing + kSlots * kTileBytes;  // 128 x (maximum, sum)
    static constexpr int kOffSeg = kOffMl + kTileRows * 8;
    static constexpr int kOffScan = kOffSeg + kSegRing * 48;  // 12 warp sums, context, its start
    static constexpr int kOffBar = kOffScan + 12 * 8 + 16;
    static constexpr int kNumBars = 2 + 2 + 2 * kSlots + 4 * 2 + 2 + 2 * kSegRing + 1;
    static constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16 + 1024;
    static_assert(kOffBar % 8 == 0 && kSmemBytes <= 232448, "shared memory layout");
};

// What the roles need to know about one CTA's part of one unit.
struct Seg {
    int n_blk;     // key blocks; 0 ends the CTA's work
    int blk0;      // first key block
    int len;       // keys of the context
    int lim0;      // causal: last key the first token of tile 0 sees
    int tok0;      // first token of tile 0
    int tok_end;   // end of the context's tokens
    int head0;     // first query head
    int nh;        // query heads
    int hk;        // K/V head
    int ctx;       // sequence, or -1 for the shared prefix
    int two;       // two row tiles
    int part_row;  // first partial row, -1: the whole unit, write the result
};
static_assert(sizeof(Seg) == 48, "Seg layout");

// A unit whose blocks several CTAs share (ragged): written by the first.
struct Split {
    int last;  // last CTA of the unit, -1: none
    int tok0, tok_end, head0, nh, two;
    int pad[2];
};

struct TcParams {
    void* O;
    float* L;
    float* O_part;
    float* L_part;          // log2-sum-exp of each partial row
    long long* per;         // blocks per CTA, for the second kernel
    long long* unit_start;  // prefix decode: line position of each own-keys unit
    Split* split;           // ragged: per CTA
    const int* prefix_table;
    const int* prefix_len;
    const int* block_table;
    const int* seq_lens;
    const int* cu_seqlens;
    int prefix_mode;
    int num_tokens, B, hq, hkv, group;
    int gt, chunks, tpt;  // heads per tile, chunks of the group, tokens per tile
    int page_shift, max_prefix_pages, max_pages, num_pages;
    int causal;
    int w_two, w_one;  // line length of a block of a two-tile and of a one-tile unit
    int min_per;
    long long own_part_row;  // first partial row of the own-keys units
    float scale_log2;
};

// sum over i in [0, n) of floor((a i + b) / m): the usual Euclid-like
// reduction (a, b >= 0, m > 0).
__host__ __device__ __forceinline__ long long floor_sum(long long n, long long m, long long a, long long b) {
    long long s = 0;
    while (n > 0) {
        s += (n * (n - 1) / 2) * (a / m) + n * (b / m);
        a %= m;
        b %= m;
        const long long top = a * n + b;
        n = top / m;
        b = top % m;
        const long long t = m;
        m = a;
        a = t;
        if (m == 0) break;  // then top < the old m and n == 0
    }
    return s;
}

struct Ctx {
    int tok, ntok, len;
    int pairs;       // units per head chunk
    int last_two;    // the last unit has two tiles
    long long head_cost;
};

__host__ __device__ __forceinline__ int unit_blocks(const TcParams& p, const Ctx& c, int pair) {
    int vis = c.len;
    if (p.causal && pair < c.pairs - 1)
        vis = c.len - c.ntok + (pair + 1) * 2 * p.tpt;  // what its last token sees
    const int nb = (vis + kBlockKeys - 1) / kBlockKeys;
    // ragged: a unit that sees no key takes one masked block, which writes its rows
    return p.prefix_mode ? nb : (vis > 0 ? nb : 1);
}

__host__ __device__ __forceinline__ int unit_weight(const TcParams& p, const Ctx& c, int pair) {
    return pair < c.pairs - 1 || c.last_two ? p.w_two : p.w_one;
}

// Line length of the first `pairs` units (of two tiles each) of a head chunk.
__host__ __device__ __forceinline__ long long pairs_cost(const TcParams& p, const Ctx& c, int pairs) {
    if (!p.causal) return static_cast<long long>(pairs) * unit_blocks(p, c, 0) * p.w_two;
    const int s = 2 * p.tpt;
    const int off = c.len - c.ntok;
    // units whose last token sees at most 128 keys take one block
    int ones = 128 - off >= 0 ? (128 - off) / s : 0;
    if (ones > pairs) ones = pairs;
    return (ones + floor_sum(pairs - ones, 128, s,
                             static_cast<long long>(off) + static_cast<long long>(ones + 1) * s + 127)) *
           p.w_two;
}

// Context c: -1 is the shared prefix.
__host__ __device__ __forceinline__ Ctx load_ctx(const TcParams& p, int c) {
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
    x.last_two = (tiles & 1) == 0;
    x.head_cost = 0;
    if (x.pairs > 0 && (x.len > 0 || !p.prefix_mode))
        x.head_cost = pairs_cost(p, x, x.pairs - 1) +
                      static_cast<long long>(unit_blocks(p, x, x.pairs - 1)) *
                          unit_weight(p, x, x.pairs - 1);
    return x;
}

// The piece [x0, x1) of the line that belongs to CTA `cta`, unit by unit.
struct Walk {
    Ctx ctx;
    int c, hc, pair, cta;  // context, head chunk, unit of it
    long long ub, x, x1, per;  // line position of the unit, of the walk, its end
};

// Context c holds position x0 and starts at ctx_base.
__host__ __device__ __forceinline__ void walk_start(const TcParams& p, Walk& w, int c,
                                                    long long ctx_base, long long x0, long long x1,
                                                    long long per, int cta) {
    w.ctx = load_ctx(p, c);
    w.c = c;
    w.cta = cta;
    w.x = x0;
    w.x1 = x1;
    w.per = per;
    long long y = x0 - ctx_base;
    w.hc = static_cast<int>(y / w.ctx.head_cost);
    y -= w.hc * w.ctx.head_cost;
    int lo = 0, hi = w.ctx.pairs;  // the unit of the head chunk that y falls into
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (pairs_cost(p, w.ctx, mid) <= y)
            lo = mid;
        else
            hi = mid;
    }
    w.pair = lo;
    w.ub = ctx_base + w.hc * w.ctx.head_cost + pairs_cost(p, w.ctx, lo);
}

// The next segment; false at the end.  Records where units start (own keys)
// and which units several CTAs share (ragged) for the second kernel.
__host__ __device__ __forceinline__ bool walk_next(const TcParams& p, Walk& w, Seg& sg) {
    const int heads = p.hkv * p.chunks;
    while (w.x < w.x1) {
        const int nb = unit_blocks(p, w.ctx, w.pair);
        const int wt = unit_weight(p, w.ctx, w.pair);
        const int blk0 = static_cast<int>((w.x - w.ub + wt - 1) / wt);
        const long long end = (w.x1 - w.ub + wt - 1) / wt;
        const int blk1 = end < nb ? static_cast<int>(end) : nb;
        const bool some = blk1 > blk0;
        if (some) {
            sg.n_blk = blk1 - blk0;
            sg.blk0 = blk0;
            sg.len = w.ctx.len;
            sg.lim0 = w.ctx.len - w.ctx.ntok + w.pair * 2 * p.tpt;
            sg.tok0 = w.ctx.tok + w.pair * 2 * p.tpt;
            sg.tok_end = w.ctx.tok + w.ctx.ntok;
            sg.hk = w.hc / p.chunks;
            const int ch = w.hc - sg.hk * p.chunks;
            sg.head0 = sg.hk * p.group + ch * p.gt;
            sg.nh = p.group - ch * p.gt < p.gt ? p.group - ch * p.gt : p.gt;
            sg.ctx = w.c;
            sg.two = w.pair < w.ctx.pairs - 1 || w.ctx.last_two;
            if (p.prefix_mode) {
                if (w.c < 0) {
                    sg.part_row = (w.hc * w.ctx.pairs + w.pair + w.cta) * (2 * kTileRows);
                } else {
                    const long long u = static_cast<long long>(w.c) * heads + w.hc;
                    if (blk0 == 0) p.unit_start[u] = w.ub;
                    sg.part_row = static_cast<int>(p.own_part_row + (u + w.cta) * p.gt);
                }
            } else if (blk0 == 0 && blk1 == nb) {
                sg.part_row = -1;
            } else {
                sg.part_row = (2 * w.cta + (blk0 == 0 ? 1 : 0)) * (2 * kTileRows);
                if (blk0 == 0) {
                    Split sp;
                    sp.last = static_cast<int>((w.ub + static_cast<long long>(nb - 1) * wt) / w.per);
                    sp.tok0 = sg.tok0;
                    sp.tok_end = sg.tok_end;
                    sp.head0 = sg.head0;
                    sp.nh = sg.nh;
                    sp.two = sg.two;
                    p.split[w.cta] = sp;
                }
            }
        }
        w.ub += static_cast<long long>(nb) * wt;
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

// Partials of the output row (sequence b, query head h): n1 rows from row1 on,
// 2 kTileRows apart (the prefix), and n2 rows from row2 on, gt apart (own keys).
struct PrefixParts {
    int n1, n2;
    long long row1, row2;
};

__host__ __device__ __forceinline__ PrefixParts prefix_parts(const TcParams& p, const Ctx& pre,
                                                             const Ctx& own, int b, int h) {
    PrefixParts q = {0, 0, 0, 0};
    const long long per = *p.per;
    const int hk = h / p.group, hg = h - hk * p.group;
    const int ch = hg / p.gt, hr = hg - ch * p.gt;
    const int hc = hk * p.chunks + ch;
    if (pre.len > 0) {
        const int tile = b / p.tpt;
        const int pair = tile >> 1;
        const long long nb = unit_blocks(p, pre, pair);
        const long long ub = hc * pre.head_cost + pairs_cost(p, pre, pair);
        const long long i0 = ub / per;
        q.n1 = static_cast<int>((ub + (nb - 1) * unit_weight(p, pre, pair)) / per - i0) + 1;
        q.row1 = (static_cast<long long>(hc) * pre.pairs + pair + i0) * (2 * kTileRows) +
                 (tile & 1) * kTileRows + (b - tile * p.tpt) * p.gt + hr;
    }
    if (own.len > 0) {
        const long long u = static_cast<long long>(b) * p.hkv * p.chunks + hc;
        const long long nb = unit_blocks(p, own, 0);
        const long long ub = p.unit_start[u];
        const long long i0 = ub / per;
        q.n2 = static_cast<int>((ub + (nb - 1) * p.w_one) / per - i0) + 1;
        q.row2 = p.own_part_row + (u + i0) * p.gt + hr;
    }
    return q;
}

template <int D>
__device__ __forceinline__ uint64_t pg_kdesc(uint32_t base) {  // K-major, k-step 0
    using G = PagedGeom<D>;
    return sm100::make_smem_desc(base, 16, 8 * G::kSwz, G::kLayout);
}
template <int D>
__host__ __device__ constexpr uint32_t pg_kdelta(int kk) {
    using G = PagedGeom<D>;
    return ((static_cast<uint32_t>(kk) * 32u / G::kSwz) * G::kCbBytes +
            (static_cast<uint32_t>(kk) * 32u % G::kSwz)) >> 4;
}
template <int D>
__device__ __forceinline__ uint64_t pg_vdesc(uint32_t base) {  // MN-major, k-step 0
    using G = PagedGeom<D>;
    return sm100::make_smem_desc(base, G::kCbBytes, 8 * G::kSwz, G::kLayout);
}
template <int D>
__host__ __device__ constexpr uint32_t pg_vdelta(int kk) {
    return (static_cast<uint32_t>(kk) * 16u * PagedGeom<D>::kSwz) >> 4;
}

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQ1,
                      const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const TcParams p) {
    using G = PagedGeom<D>;
    using namespace sm100;
    constexpr int R = G::kSlots;
    extern __shared__ uint8_t smem_raw[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (cta_skip(&g_paged_status)) return;

    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t sbase = (raw + 1023u) & ~1023u;
    uint8_t* sptr = smem_raw + (sbase - raw);
    uint64_t* bar_q = reinterpret_cast<uint64_t*>(sptr + G::kOffBar);  // [2] query tile landed
    uint64_t* bar_qfree = bar_q + 2;      // [2] its last product retired
    uint64_t* full = bar_qfree + 2;       // [R]
    uint64_t* empty = full + R;           // [R]
    uint64_t* bar_s = empty + R;          // [2] S_t in TMEM
    uint64_t* bar_p = bar_s + 2;          // [2] first half of P_t stored
    uint64_t* bar_p2 = bar_p + 2;         // [2] second half
    uint64_t* bar_o = bar_p2 + 2;         // [2] O_t final for the segment
    uint64_t* bar_x = bar_o + 2;          // one tile: second stream's state is there
    uint64_t* bar_y = bar_x + 1;          // one tile: it has been read
    uint64_t* seg_full = bar_y + 1;       // [kSegRing]
    uint64_t* seg_free = seg_full + kSegRing;  // [kSegRing]
    uint64_t* bar_done = seg_free + kSegRing;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    Seg* segs = reinterpret_cast<Seg*>(sptr + G::kOffSeg);
    long long* scan = reinterpret_cast<long long*>(sptr + G::kOffScan);  // [12]
    long long* first_base = scan + 12;  // line position of the context the CTA starts in
    int* first_ctx = reinterpret_cast<int*>(scan + 13);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(bar_q + t, 1);
            mbar_init(bar_qfree + t, 1);
            mbar_init(bar_s + t, 1);
            mbar_init(bar_p + t, 128);
            mbar_init(bar_p2 + t, 128);
            mbar_init(bar_o + t, 1);
        }
        for (int s = 0; s < R; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        mbar_init(bar_x, 128);
        mbar_init(bar_y, 128);
        for (int s = 0; s < kSegRing; ++s) {
            mbar_init(seg_full + s, 1);
            mbar_init(seg_free + s, 10);  // producer, MMA, 8 softmax warps
        }
        mbar_init(bar_done, 1);
        *abort_flag = 0;
        *first_ctx = -2;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }

    // ---- the line: contexts' lengths summed over the block
    const int c_lo = p.prefix_mode ? -1 : 0;
    const int n_ctx = p.B - c_lo;
    const long long heads = static_cast<long long>(p.hkv) * p.chunks;
    const int run = (n_ctx + kTcThreads - 1) / kTcThreads;  // contexts per thread
    const int c_first = c_lo + static_cast<int>(min(static_cast<long long>(threadIdx.x) * run,
                                                    static_cast<long long>(n_ctx)));
    const int c_last = min(c_first + run, p.B);
    long long mine = 0;
    for (int c = c_first; c < c_last; ++c) mine += load_ctx(p, c).head_cost * heads;
    long long incl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kTcThreads / 32; ++w) {
        const long long v = scan[w];
        if (w < warp) before += v;
        total += v;
    }
    long long per = (total + gridDim.x - 1) / gridDim.x;
    if (per < p.min_per) per = p.min_per;
    const long long x0 = static_cast<long long>(blockIdx.x) * per;
    const long long x1 = min(x0 + per, total);
    {
        long long base = before + incl - mine;
        if (x0 >= base && x0 < base + mine) {
            for (int c = c_first; c < c_last; ++c) {
                const long long cost = load_ctx(p, c).head_cost * heads;
                if (x0 < base + cost) {
                    *first_ctx = c;
                    *first_base = base;
                    break;
                }
                base += cost;
            }
        }
    }
    if (threadIdx.x == 0) {
        if (blockIdx.x == 0) *p.per = per;
        if (!p.prefix_mode) p.split[blockIdx.x].last = -1;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Registers: launched with 168 per thread (384 x 168 = 64512); the first
    // warpgroup gives back down to 72 and the two softmax warpgroups take 216:
    // 128 * 72 + 256 * 216 = 64512.
    if (warp < 4) {
        setmaxnreg_dec<72>();
        if (warp == 0) {
            // ------------------------------------------------ TMA producer
            uint32_t q_cnt[2] = {0u, 0u};
            uint32_t kv = 0;  // ring fills
            int qs = 0;       // query slot of the next one-tile segment
            const int box_rows = min(1 << p.page_shift, kBlockKeys);
            const int boxes = kBlockKeys / box_rows;  // per block and column block, <= 16
            const int my_box = lane & 15;
            const int my_cb = lane >> 4;
            bool ok = true;
            if (lane == 0) {
                prefetch_tmap(&tmQ);
                prefetch_tmap(&tmQ1);
                prefetch_tmap(&tmK);
                prefetch_tmap(&tmV);
            }
            for (int k = 0;; ++k) {
                ok = mbar_wait(seg_full + k % kSegRing, (k / kSegRing) & 1, abort_flag, &g_paged_status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const Seg sg = segs[k % kSegRing];
                __syncwarp();
                if (lane == 0) mbar_arrive(seg_free + k % kSegRing);
                if (sg.n_blk == 0) break;
                const int* table = sg.ctx < 0 ? p.prefix_table
                                              : p.block_table + static_cast<long long>(sg.ctx) * p.max_pages;
                const int max_pages = sg.ctx < 0 ? p.max_prefix_pages : p.max_pages;
                auto load_page = [&](int blk) -> int {
                    const int row = blk * kBlockKeys + my_box * box_rows;
                    if (my_box >= boxes || row >= sg.len) return 0;
                    const int pg = table[min(row >> p.page_shift, max_pages - 1)];
                    return min(max(pg, 0), p.num_pages - 1);
                };
                int page = load_page(sg.blk0);
                // query tiles
                if (lane == 0) {
                    const bool single = sg.tok_end - sg.tok0 == 1;
                    const uint32_t bytes = static_cast<uint32_t>(p.gt * (single ? 1 : p.tpt)) * G::kRowBytes;
                    for (int u = 0; u < (sg.two ? 2 : 1) && ok; ++u) {
                        const int slot = sg.two ? u : qs;
                        if (q_cnt[slot] > 0)
                            ok = mbar_wait(bar_qfree + slot, (q_cnt[slot] - 1) & 1, abort_flag, &g_paged_status);
                        if (!ok) break;
                        mbar_arrive_expect_tx(bar_q + slot, bytes);
                        for (int cb = 0; cb < G::kNumCb; ++cb)
                            tma_load_3d(sptr + slot * G::kTileBytes + cb * G::kCbBytes,
                                        single ? &tmQ1 : &tmQ, bar_q + slot, cb * G::kCbElems,
                                        sg.head0, sg.tok0 + u * p.tpt);
                        ++q_cnt[slot];
                    }
                }
                if (!sg.two) qs ^= 1;
                ok = __shfl_sync(0xffffffffu, ok, 0);
                for (int j = 0; ok && j < sg.n_blk; ++j) {
                    const int r0 = (sg.blk0 + j) * kBlockKeys;
                    const int live = min(max(sg.len - r0, 0), kBlockKeys);
                    const int nbox = (live + box_rows - 1) / box_rows;
                    const int page_now = page;
                    if (j + 1 < sg.n_blk) page = load_page(sg.blk0 + j + 1);
                    const int row0 = (page_now << p.page_shift) +
                                     ((r0 + my_box * box_rows) & ((1 << p.page_shift) - 1));
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int s = kv % R;
                        if (lane == 0) {
                            if (kv >= static_cast<uint32_t>(R))
                                ok = mbar_wait(empty + s, (kv / R - 1) & 1, abort_flag, &g_paged_status);
                            if (ok)
                                mbar_arrive_expect_tx(full + s, static_cast<uint32_t>(nbox * box_rows) *
                                                                    G::kRowBytes);
                        }
                        ok = __shfl_sync(0xffffffffu, ok, 0);
                        if (!ok) break;
                        if (my_box < nbox && my_cb < G::kNumCb)
                            tma_load_3d(sptr + G::kOffRing + s * G::kTileBytes + my_cb * G::kCbBytes +
                                            my_box * box_rows * G::kSwz,
                                        v == 0 ? &tmK : &tmV, full + s, my_cb * G::kCbElems, sg.hk,
                                        row0);
                        ++kv;
                    }
                }
                if (!ok) break;
            }
            // every issued load lands before the CTA can exit
            if (lane == 0) {
                volatile int never = 0;
                for (int t = 0; t < 2; ++t)
                    if (q_cnt[t] > 0) mbar_wait(bar_q + t, (q_cnt[t] - 1) & 1, &never, &g_paged_status);
                for (uint32_t g = kv > R ? kv - R : 0; g < kv; ++g)
                    mbar_wait(full + g % R, (g / R) & 1, &never, &g_paged_status);
            }
            __syncwarp();
        } else if (warp == 1) {
            // ------------------------------------------------ MMA issuer
            // The whole warp walks the steps (the zeroing of a block's dead V
            // rows takes all lanes); lane 0 issues.
            constexpr uint32_t idesc_qk = make_idesc(DType<T>::kMmaFmt, 128, 128, false, false);
            constexpr uint32_t idesc_pv = make_idesc(DType<T>::kMmaFmt, 128, D, false, true);
            struct Step {
                uint32_t v;  // ring fill of its V block
                int live;    // live keys of the block; -1: already looked after
                int flags;   // 1: accumulate, 2: last of its stream, 4: releases V
            };
            uint32_t q_cnt[2] = {0u, 0u};
            uint32_t p_cnt[2] = {0u, 0u};
            uint32_t n_s = 0, n_o = 0;  // steps issued
            uint32_t g0 = 0;            // blocks before the current segment
            int k = 0, qs = 0, cur_q = 0;
            int i = 0, steps = 0, n_blk = 0, two = 0, len = 0, blk0 = 0;
            bool ok = true;
            auto next_s = [&](Step& st) -> bool {
                if (i == steps) {
                    g0 += n_blk;
                    ok = mbar_wait(seg_full + k % kSegRing, (k / kSegRing) & 1, abort_flag, &g_paged_status);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) return false;
                    const Seg& sg = segs[k % kSegRing];
                    n_blk = sg.n_blk;
                    two = sg.two;
                    len = sg.len;
                    blk0 = sg.blk0;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(seg_free + k % kSegRing);
                    ++k;
                    if (n_blk == 0) return false;
                    i = 0;
                    steps = two ? 2 * n_blk : n_blk;
                    if (two) {
                        ok = mbar_wait(bar_q, q_cnt[0] & 1, abort_flag, &g_paged_status) &&
                             mbar_wait(bar_q + 1, q_cnt[1] & 1, abort_flag, &g_paged_status);
                        ++q_cnt[0];
                        ++q_cnt[1];
                    } else {
                        cur_q = qs;
                        ok = mbar_wait(bar_q + qs, (qs ? q_cnt[1] : q_cnt[0]) & 1, abort_flag,
                                       &g_paged_status);
                        if (qs) ++q_cnt[1]; else ++q_cnt[0];
                        qs ^= 1;
                    }
                }
                const int j = two ? i >> 1 : i;
                const int u = two ? i & 1 : 0;
                const uint32_t kf = 2 * (g0 + j);
                const int s = kf % R;
                const int t = n_s & 1;
                if (ok && u == 0) ok = mbar_wait(full + s, (kf / R) & 1, abort_flag, &g_paged_status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return false;
                const int qslot = two ? u : cur_q;
                if (lane == 0) {
                    tc_fence_after();
                    uint64_t a0 = pg_kdesc<D>(sbase + qslot * G::kTileBytes);
                    uint64_t b0 = pg_kdesc<D>(sbase + G::kOffRing + s * G::kTileBytes);
                    asm volatile("" : "+l"(a0), "+l"(b0));
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        mma_f16_ss(tmem + t * 128, a0 + pg_kdelta<D>(kk), b0 + pg_kdelta<D>(kk), idesc_qk,
                                   kk > 0 ? 1u : 0u);
                    tc_commit(bar_s + t);
                    if (!two || u == 1) tc_commit(empty + s);
                    if (two ? j == n_blk - 1 : i == steps - 1) tc_commit(bar_qfree + qslot);
                }
                __syncwarp();
                st.v = kf + 1;
                st.live = u == 0 ? len - (blk0 + j) * kBlockKeys : -1;
                if (st.live < 0 && u == 0) st.live = 0;
                st.flags = ((two ? j > 0 : i >= 2) ? 1 : 0) |
                           ((two ? j == n_blk - 1 : i + 2 >= steps) ? 2 : 0) |
                           ((!two || u == 1) ? 4 : 0);
                ++i;
                ++n_s;
                return true;
            };
            auto do_o = [&](const Step& st) -> bool {
                const int t = n_o & 1;
                const int s = st.v % R;
                const uint32_t vbase = sbase + G::kOffRing + s * G::kTileBytes;
                ok = mbar_wait(full + s, (st.v / R) & 1, abort_flag, &g_paged_status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return false;
                if (st.live >= 0 && st.live < kBlockKeys) {
                    // rows behind the context's end hold whatever the page (or the
                    // ring) had; zero them so that P = 0 meets no NaN
                    constexpr int kChunks = G::kSwz / 16;
                    const int n = (kBlockKeys - st.live) * kChunks;
                    for (int e = lane; e < n * G::kNumCb; e += 32) {
                        const int cb = e / n;
                        const uint32_t a = vbase + cb * G::kCbBytes + st.live * G::kSwz + (e - cb * n) * 16;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0u) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                uint64_t v0 = pg_vdesc<D>(vbase);
                asm volatile("" : "+l"(v0));
                const uint32_t par = (t ? p_cnt[1] : p_cnt[0]) & 1;
                ok = mbar_wait(bar_p + t, par, abort_flag, &g_paged_status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return false;
                if (lane == 0) {
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, v0 + pg_vdelta<D>(kk),
                                   idesc_pv, ((st.flags & 1) || kk > 0) ? 1u : 0u);
                }
                __syncwarp();
                ok = mbar_wait(bar_p2 + t, par, abort_flag, &g_paged_status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return false;
                if (lane == 0) {
                    tc_fence_after();
#pragma unroll
                    for (int kk = 4; kk < 8; ++kk)
                        mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, v0 + pg_vdelta<D>(kk),
                                   idesc_pv, 1u);
                    if (st.flags & 2) tc_commit(bar_o + t);
                    if (st.flags & 4) tc_commit(empty + s);
                }
                __syncwarp();
                if (t) ++p_cnt[1]; else ++p_cnt[0];
                ++n_o;
                return true;
            };
            Step a, b, c;
            bool more_a = next_s(a);
            bool more_b = more_a && next_s(b);
            while (more_a && ok) {
                if (!do_o(a)) break;
                const bool more_c = more_b && next_s(c);
                if (!ok) break;
                a = b;
                more_a = more_b;
                b = c;
                more_b = more_c;
            }
            // all products (and their commits) retire before teardown
            if (lane == 0) {
                tc_commit(bar_done);
                volatile int never = 0;
                mbar_wait(bar_done, 0, &never, &g_paged_status);
            }
            __syncwarp();
        } else if (warp == 2) {
            // ------------------------------------------------ units and segments
            if (lane == 0) {
                int k = 0;
                bool ok = true;
                auto emit = [&](const Seg& sg) {
                    if (k >= kSegRing)
                        ok = mbar_wait(seg_free + k % kSegRing, (k / kSegRing - 1) & 1, abort_flag,
                                       &g_paged_status);
                    if (!ok) return;
                    segs[k % kSegRing] = sg;
                    mbar_arrive(seg_full + k % kSegRing);
                    ++k;
                };
                if (x0 < x1 && *first_ctx >= c_lo) {
                    Walk w;
                    walk_start(p, w, *first_ctx, *first_base, x0, x1, per, blockIdx.x);
                    Seg sg;
                    while (ok && walk_next(p, w, sg)) emit(sg);
                }
                Seg last = {};
                if (ok) emit(last);
            }
            __syncwarp();
        }
    } else {
        setmaxnreg_inc<216>();
        // ------------------------------------------------ softmax / epilogue
        const int t = (warp - 4) >> 2;
        const int wq = warp & 3;
        const int r = wq * 32 + lane;
        const int tok_r = r / p.gt;
        const int head_r = r - tok_r * p.gt;
        const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;
        const uint32_t s_tmem = tmem + lane_addr + t * 128;
        const uint32_t o_tmem = tmem + lane_addr + 256 + t * 128;
        const uint32_t o_other = tmem + lane_addr + 256 + (t ^ 1) * 128;
        float2* ml = reinterpret_cast<float2*>(sptr + G::kOffMl);
        const float c = p.scale_log2;
        uint32_t s_cnt = 0, o_cnt = 0, x_cnt = 0;
        uint32_t n0 = 0;  // steps before the segment, mod 2 matters
        bool y_pending = false;
        bool ok = true;
        for (int k = 0; ok; ++k) {
            ok = mbar_wait(seg_full + k % kSegRing, (k / kSegRing) & 1, abort_flag, &g_paged_status);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const Seg sg = segs[k % kSegRing];
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_free + k % kSegRing);
            if (sg.n_blk == 0) break;
            const int first = (t ^ n0) & 1;  // two tiles: this stream's tile; one: its first block
            const int tile = sg.two ? first : 0;
            const int n = sg.two ? sg.n_blk : (sg.n_blk - first + 1) / 2;
            n0 += sg.two ? 2 * sg.n_blk : sg.n_blk;
            const int token = sg.tok0 + tile * p.tpt + tok_r;
            const bool valid = tok_r < p.tpt && head_r < sg.nh && token < sg.tok_end;
            const bool active = __any_sync(0xffffffffu, valid);
            const int tile_lim = sg.lim0 + tile * p.tpt;  // first row's limit
            // last key this row sees
            const int row_end = p.causal ? min(sg.len - 1, tile_lim + tok_r) : sg.len - 1;

            float m_run = -INFINITY, l_run = 0.f;
            for (int j = 0; j < n; ++j) {
                ok = mbar_wait(bar_s + t, s_cnt & 1, abort_flag, &g_paged_status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ++s_cnt;
                if (y_pending) {  // the other stream has read the last segment's O_t
                    ok = mbar_wait(bar_y, (x_cnt - 1) & 1, abort_flag, &g_paged_status);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    y_pending = false;
                }
                if (!active) {
                    mbar_arrive(bar_p + t);
                    mbar_arrive(bar_p2 + t);
                    continue;
                }
                tc_fence_after();
                uint32_t sr[128];
                tmem_ld_x128(s_tmem, sr);
                const int blk = sg.blk0 + (sg.two ? j : first + 2 * j);
                const int col0 = blk * kBlockKeys;
                if (col0 + kBlockKeys > sg.len || (p.causal && col0 + kBlockKeys - 1 > tile_lim)) {
                    const int vis = row_end - col0;  // column i is visible iff i <= vis
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (i > vis) sr[i] = __float_as_uint(-INFINITY);
                }
                float mx;
                {
                    float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 128; i += 8) {
                        m0 = fmax3(m0, __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
                        m1 = fmax3(m1, __uint_as_float(sr[i + 2]), __uint_as_float(sr[i + 3]));
                        m2 = fmax3(m2, __uint_as_float(sr[i + 4]), __uint_as_float(sr[i + 5]));
                        m3 = fmax3(m3, __uint_as_float(sr[i + 6]), __uint_as_float(sr[i + 7]));
                    }
                    mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * c;  // c > 0
                }
                float alpha = 1.f;
                bool need = false;
                if (j == 0) {
                    m_run = mx;
                } else {
                    need = mx > m_run + kRescale;
                    if (need) {
                        alpha = ex2_approx(m_run - mx);
                        m_run = mx;
                    }
                }
                // S_t of this step was issued behind O_t of the last one, so O_t is at rest
                if (__any_sync(0xffffffffu, need)) {
#pragma unroll
                    for (int cb = 0; cb < D / 16; ++cb) {
                        uint32_t o[16];
                        tmem_ld_x16(o_tmem + cb * 16, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st_x16(o_tmem + cb * 16, o);
                    }
                }
                const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
                const uint64_t c2 = f2_pack(c, c);
                const uint64_t nm2 = f2_pack(-m_use, -m_use);
                uint64_t acc0 = 0, acc1 = 0, acc2 = 0, acc3 = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int c0 = h * 64 + 2 * i;
                        const float2 x = f2_unpack(
                            f2_fma(f2_pack(__uint_as_float(sr[c0]), __uint_as_float(sr[c0 + 1])), c2, nm2));
                        const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
                        const uint64_t pp = f2_pack(p0, p1);
                        switch (i & 3) {
                            case 0: acc0 = f2_add(acc0, pp); break;
                            case 1: acc1 = f2_add(acc1, pp); break;
                            case 2: acc2 = f2_add(acc2, pp); break;
                            default: acc3 = f2_add(acc3, pp); break;
                        }
                        pk[i] = DType<T>::pack2(p0, p1);
                    }
                    tmem_st_x32(s_tmem + h * 32, pk);
                    tc_fence_before();
                    mbar_arrive((h == 0 ? bar_p : bar_p2) + t);
                }
                const float2 sum = f2_unpack(f2_add(f2_add(acc0, acc1), f2_add(acc2, acc3)));
                l_run = l_run * alpha + (sum.x + sum.y);
            }
            if (!ok) break;

            // ---- the segment's result
            const bool join = !sg.two && sg.n_blk > 1;  // both streams have a part
            if (n > 0) {
                ok = mbar_wait(bar_o + t, o_cnt & 1, abort_flag, &g_paged_status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ++o_cnt;
                tc_fence_after();
            }
            if (join) ++x_cnt;
            if (!sg.two && first == 1) {  // second stream: hand over, or had no block
                if (join) {
                    ml[r] = make_float2(m_run, l_run);
                    tc_fence_before();
                    mbar_arrive(bar_x);
                    y_pending = true;
                }
                continue;
            }
            float w0 = 1.f, w1 = 0.f;  // O = w0 O_t + w1 O_other, unnormalised sums alike
            if (join) {
                ok = mbar_wait(bar_x, (x_cnt - 1) & 1, abort_flag, &g_paged_status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const float2 o2 = ml[r];
                const float M = fmaxf(m_run, o2.x);
                if (M != -INFINITY) {
                    w0 = ex2_approx(m_run - M);
                    w1 = ex2_approx(o2.x - M);
                }
                l_run = w0 * l_run + w1 * o2.y;
                m_run = M;
            }
            const float inv_l = l_run > 0.f ? 1.f / l_run : 0.f;
            w0 *= inv_l;
            w1 *= inv_l;
            const float lse2 = l_run > 0.f ? m_run + log2f(l_run) : -INFINITY;
            const int head = sg.head0 + head_r;
            if (active) {
                const long long prow = static_cast<long long>(sg.part_row) + tile * kTileRows + r;
                const long long orow = static_cast<long long>(token) * p.hq + head;
#pragma unroll
                for (int cb = 0; cb < D / 32; ++cb) {
                    uint32_t o[32];
                    tmem_ld_x32(o_tmem + cb * 32, o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w0);
                    if (join) {
                        uint32_t o2[32];
                        tmem_ld_x32(o_other + cb * 32, o2);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            o[i] = __float_as_uint(fmaf(__uint_as_float(o2[i]), w1, __uint_as_float(o[i])));
                    }
                    if (valid) {
                        if (sg.part_row >= 0) {
                            float4* dst = reinterpret_cast<float4*>(p.O_part + prow * D + cb * 32);
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                dst[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                     __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                        } else {
                            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.O) + orow * D + cb * 32);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint4 v;
                                v.x = DType<T>::pack2(__uint_as_float(o[8 * i]), __uint_as_float(o[8 * i + 1]));
                                v.y = DType<T>::pack2(__uint_as_float(o[8 * i + 2]), __uint_as_float(o[8 * i + 3]));
                                v.z = DType<T>::pack2(__uint_as_float(o[8 * i + 4]), __uint_as_float(o[8 * i + 5]));
                                v.w = DType<T>::pack2(__uint_as_float(o[8 * i + 6]), __uint_as_float(o[8 * i + 7]));
                                dst[i] = v;
                            }
                        }
                    }
                }
                if (valid) {
                    if (sg.part_row >= 0)
                        p.L_part[prow] = lse2;
                    else
                        p.L[orow] = lse2 * kLn2;
                }
            }
            if (join) {
                tc_fence_before();
                mbar_arrive(bar_y);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins normalised partial rows by their log2-sum-exp: one warp per row, a
// lane holds D/32 columns.  `row_of(k)` is the k-th partial's row.
template <typename T, int D, typename RowOf>
__device__ __forceinline__ void join_rows(const TcParams& p, int n, RowOf row_of, long long out_row) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    float M = -INFINITY;
    for (int k = lane; k < n; k += 32) M = fmaxf(M, p.L_part[row_of(k)]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    float acc[V], tot = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    if (M != -INFINITY) {
        for (int k0 = 0; k0 < n; k0 += 32) {
            const float w = k0 + lane < n ? sm100::ex2_approx(p.L_part[row_of(k0 + lane)] - M) : 0.f;
            tot += w;
            const int m = min(32, n - k0);
#pragma unroll 4
            for (int k = 0; k < m; ++k) {
                const float wk = __shfl_sync(0xffffffffu, w, k);
                const float* src = p.O_part + row_of(k0 + k) * D + lane * V;
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = fmaf(wk, src[e], acc[e]);
            }
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, off);
    }
    const float inv = tot > 0.f ? 1.f / tot : 0.f;
    T* dst = static_cast<T*>(p.O) + out_row * D + lane * V;
#pragma unroll
    for (int e = 0; e < V; ++e) dst[e] = DType<T>::from_float(acc[e] * inv);
    if (lane == 0) p.L[out_row] = tot > 0.f ? (M + log2f(tot)) * kLn2 : -INFINITY;
}

__device__ __forceinline__ bool partials_ready() {
    // the first kernel's writes are visible behind this; nothing is read if it failed
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return *reinterpret_cast<const volatile int*>(&g_paged_status.code) == 0;
}

// One warp per (sequence, query head): the prefix's partials, then its own.
template <typename T, int D>
__global__ void __launch_bounds__(128)
    paged_join_prefix_kernel(const TcParams p) {
    const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (row >= static_cast<long long>(p.B) * p.hq) return;
    const int b = static_cast<int>(row / p.hq);
    const int h = static_cast<int>(row - static_cast<long long>(b) * p.hq);
    const Ctx pre = load_ctx(p, -1), own = load_ctx(p, b);
    if (!partials_ready()) return;
    const PrefixParts q = prefix_parts(p, pre, own, b, h);
    join_rows<T, D>(
        p, q.n1 + q.n2,
        [&](int k) -> long long {
            return k < q.n1 ? q.row1 + static_cast<long long>(k) * (2 * kTileRows)
                            : q.row2 + static_cast<long long>(k - q.n1) * p.gt;
        },
        row);
}

// Block (i, y): rows [32 y, 32 y + 32) of the unit whose first blocks CTA i
// had and whose last CTA split[i].last had.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    paged_join_split_kernel(const TcParams p) {
    if (!partials_ready()) return;
    const Split sp = p.split[blockIdx.x];
    const int i = static_cast<int>(blockIdx.x);
    if (sp.last <= i) return;
    for (int q = 0; q < 4; ++q) {
        const int rr = blockIdx.y * 32 + (threadIdx.x >> 5) * 4 + q;
        const int tile = rr / kTileRows;
        const int r = rr - tile * kTileRows;
        const int tok_r = r / p.gt;
        const int head_r = r - tok_r * p.gt;
        const int token = sp.tok0 + tile * p.tpt + tok_r;
        if ((tile == 1 && !sp.two) || tok_r >= p.tpt || head_r >= sp.nh || token >= sp.tok_end) continue;
        join_rows<T, D>(
            p, sp.last - i + 1,
            [&](int k) -> long long {
                return static_cast<long long>(2 * (i + k) + (k == 0 ? 1 : 0)) * (2 * kTileRows) + rr;
            },
            static_cast<long long>(token) * p.hq + sp.head0 + head_r);
    }
}

// Launches `kern` so that its blocks may be scheduled while the kernel before
// it on the stream still runs (they wait for it inside).
template <typename... Args>
cudaError_t launch_behind(void (*kern)(Args...), dim3 grid, int threads, cudaStream_t stream,
                          const TcParams& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// Row tiles of the query heads and tokens, and the line's scale.
void set_tiles(TcParams& p) {
    p.group = p.hq / p.hkv;
    p.chunks = (p.group + kTileRows - 1) / kTileRows;
    p.gt = (p.group + p.chunks - 1) / p.chunks;
    p.tpt = kTileRows / p.gt;
    p.w_two = 2;
    p.w_one = 1;
    p.min_per = 2;  // at least the larger weight: every CTA of a unit has a block of it
}

// Partial rows and record bytes of a launch of `grid` CTAs.  Going along the
// line, each piece starts a new unit, a new CTA or both, so unit + CTA numbers
// the pieces; in ragged mode only a CTA's first and last piece are partial.
void set_parts(TcParams& p, int grid, long long& rows, long long& records) {
    const long long heads = static_cast<long long>(p.hkv) * p.chunks;
    if (p.prefix_mode) {
        const long long tiles = (p.B + p.tpt - 1) / p.tpt;
        p.own_part_row = (heads * ((tiles + 1) / 2) + grid) * 2 * kTileRows;
        rows = p.own_part_row + (heads * p.B + grid) * p.gt;
        records = heads * p.B * static_cast<long long>(sizeof(long long));
    } else {
        rows = 2LL * grid * 2 * kTileRows;
        records = grid * static_cast<long long>(sizeof(Split));
    }
}

template <typename T, int D>
FlashAttentionError paged_tc(const PagedParams<T>& a, cudaStream_t stream) {
    using G = PagedGeom<D>;
    TcParams p{};
    p.O = a.O;
    p.L = a.L;
    p.prefix_table = a.prefix_table;
    p.prefix_len = a.prefix_len;
    p.block_table = a.block_table;
    p.seq_lens = a.seq_lens;
    p.cu_seqlens = a.cu_seqlens;
    p.prefix_mode = a.prefix_table != nullptr;
    p.num_tokens = a.num_tokens;
    p.B = a.B;
    p.hq = a.hq;
    p.hkv = a.hkv;
    set_tiles(p);
    p.page_shift = a.page_shift;
    p.max_prefix_pages = a.max_prefix_pages;
    p.max_pages = a.max_pages;
    p.num_pages = a.num_pages;
    p.causal = a.causal;
    // a zero scale becomes a tiny positive one so that masked scores stay -inf
    p.scale_log2 = fmaxf(a.scale_log2, 1e-30f);

    const CUtensorMapDataType dt = DType<T>::kTmaType;
    const CUtensorMapSwizzle swz = G::kSwz == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    CUtensorMap mq, mq1, mk, mv;
    {
        const uint64_t dims[3] = {D, static_cast<uint64_t>(a.hq), static_cast<uint64_t>(a.num_tokens)};
        const uint64_t strides[2] = {D * 2, static_cast<uint64_t>(a.hq) * D * 2};
        const uint32_t box[3] = {G::kCbElems, static_cast<uint32_t>(p.gt), static_cast<uint32_t>(p.tpt)};
        const uint32_t box1[3] = {G::kCbElems, static_cast<uint32_t>(p.gt), 1};
        if (!encode_tmap_3d_strided(&mq, a.Q, dt, dims, strides, box, swz) ||
            !encode_tmap_3d_strided(&mq1, a.Q, dt, dims, strides, box1, swz))
            return FlashAttentionError::CUDA_ERROR;
    }
    {
        const int ps = 1 << a.page_shift;
        const uint64_t dims[3] = {D, static_cast<uint64_t>(a.hkv),
                                  static_cast<uint64_t>(a.num_pages) << a.page_shift};
        const uint64_t strides[2] = {D * 2, static_cast<uint64_t>(a.hkv) * D * 2};
        const uint32_t box[3] = {G::kCbElems, 1, static_cast<uint32_t>(std::min(ps, kBlockKeys))};
        if (!encode_tmap_3d_strided(&mk, a.K, dt, dims, strides, box, swz) ||
            !encode_tmap_3d_strided(&mv, a.V, dt, dims, strides, box, swz))
            return FlashAttentionError::CUDA_ERROR;
    }
    auto kern = paged_attn_kernel<T, D>;
    if (!ensure_smem_attr(reinterpret_cast<const void*>(kern), G::kSmemBytes))
        return FlashAttentionError::CUDA_ERROR;
    const int grid = persistent_grid(0x7fffffffLL, 1);

    // workspace: line scale, unit starts or split records, partial rows
    long long rows, records;
    set_parts(p, grid, rows, records);
    if (rows > 0x7fffffffLL) return FlashAttentionError::INVALID_DIMENSION;
    const size_t off_rec = 256;
    const size_t off_l = off_rec + align256(static_cast<size_t>(records));
    const size_t off_o = off_l + align256(static_cast<size_t>(rows) * sizeof(float));
    const size_t bytes = off_o + static_cast<size_t>(rows) * D * sizeof(float);
    void* ws = nullptr;
    const FlashAttentionError werr = workspace_alloc(&ws, bytes, stream);
    if (werr != FlashAttentionError::SUCCESS) return werr;
    char* base = static_cast<char*>(ws);
    p.per = reinterpret_cast<long long*>(base);
    p.unit_start = reinterpret_cast<long long*>(base + off_rec);
    p.split = reinterpret_cast<Split*>(base + off_rec);
    p.L_part = reinterpret_cast<float*>(base + off_l);
    p.O_part = reinterpret_cast<float*>(base + off_o);

    bind_status_word(reinterpret_cast<const void*>(&g_paged_status), stream);
    kern<<<grid, kTcThreads, G::kSmemBytes, stream>>>(mq, mq1, mk, mv, p);
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess) {
        if (p.prefix_mode)
            err = launch_behind(paged_join_prefix_kernel<T, D>,
                                dim3(static_cast<unsigned>((static_cast<long long>(p.B) * p.hq + 3) / 4)),
                                128, stream, p);
        else
            err = launch_behind(paged_join_split_kernel<T, D>, dim3(grid, 8), 256, stream, p);
        if (err != cudaSuccess) cudaGetLastError();
    }
    workspace_free(ws, stream);
    return err == cudaSuccess ? FlashAttentionError::SUCCESS : FlashAttentionError::CUDA_ERROR;
}

template <typename T, int D>
FlashAttentionError paged_typed(const PagedParams<T>& p, cudaStream_t stream) {
    return p.page_shift >= 3 ? paged_tc<T, D>(p, stream) : paged_row<T, D>(p, stream);
}

}  // namespace

template <typename T>
FlashAttentionError launch_paged_attention(const T* Q, const T* K_cache, const T* V_cache,
                                           const int* prefix_table, const int* prefix_len,
                                           const int* block_table, const int* seq_lens,
                                           const int* cu_seqlens, T* O, float* L, int num_tokens,
                                           int B, int Hq, int Hkv, int D, int page_size,
                                           int max_prefix_pages, int max_pages, int num_pages,
                                           float scale, bool causal, cudaStream_t stream) {
    for (const void* ptr : {static_cast<const void*>(Q), static_cast<const void*>(K_cache),
                            static_cast<const void*>(V_cache), static_cast<const void*>(O)})
        if ((reinterpret_cast<uintptr_t>(ptr) & 15u) != 0) return FlashAttentionError::CUDA_ERROR;
    PagedParams<T> p;
    p.Q = Q;
    p.K = K_cache;
    p.V = V_cache;
    p.O = O;
    p.L = L;
    p.prefix_table = prefix_table;
    p.prefix_len = prefix_len;
    p.block_table = block_table;
    p.seq_lens = seq_lens;
    p.cu_seqlens = cu_seqlens;
    p.num_tokens = num_tokens;
    p.B = B;
    p.hq = Hq;
    p.hkv = Hkv;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.max_prefix_pages = max_prefix_pages;
    p.max_pages = max_pages;
    p.num_pages = num_pages;
    p.causal = causal ? 1 : 0;
    p.scale_log2 = scale * kLog2e;
    switch (D) {
        case 32:
            return paged_typed<T, 32>(p, stream);
        case 64:
            return paged_typed<T, 64>(p, stream);
        case 128:
            return paged_typed<T, 128>(p, stream);
        default:
            return FlashAttentionError::UNSUPPORTED_HEAD_DIM;
    }
}

int paged_sm100_status() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(int));
    }
    return v;
}

#define CUFLASH_PAGED_INST(T)                                                                     \
    template FlashAttentionError launch_paged_attention<T>(                                       \
        const T*, const T*, const T*, const int*, const int*, const int*, const int*, const int*, \
        T*, float*, int, int, int, int, int, int, int, int, int, float, bool, cudaStream_t);
CUFLASH_PAGED_INST(__nv_bfloat16)
CUFLASH_PAGED_INST(half)
#undef CUFLASH_PAGED_INST

}  // namespace detail
}  // namespace cuflash
