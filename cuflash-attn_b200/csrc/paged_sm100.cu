// Attention over a paged KV cache for serving (no reference counterpart: the
// reference has no KV cache):
//   * ragged attention of several new tokens per sequence (prompts, chunks of
//     prompts, single tokens) against the sequence's pages;
//   * decode of one token per sequence for a batch whose sequences share a
//     long prefix, whose scores are computed for all of them at once.

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"
#include "paged_line.cuh"

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
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = sm100::ex2_approx(m - m_use);
            l *= alpha;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] *= alpha;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float pr = sm100::ex2_approx(s[u] - m_use);
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
    attend(p.block_table + static_cast<long long>(b) * p.max_pages,
           visible_keys(clamp_len(p.seq_lens[b], p.max_pages << p.page_shift), from_end, p.causal));

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
        const float M0 = M == -INFINITY ? 0.f : M;
        float lt = 0.f, o = 0.f;
        for (int g = 0; g < G; ++g) {
            const float w = sm100::ex2_approx(s_m[g] - M0);
            lt = fmaf(w, s_l[g], lt);
            o = fmaf(w, s_acc[g][d], o);
        }
        // a sum of zero is a row that sees no key; one that sees a NaN stays NaN
        p.O[qrow * D + d] = DType<T>::from_float(lt == 0.f ? 0.f : o / lt);
        if (d == 0) p.L[qrow] = lt == 0.f ? -INFINITY : (M + log2f(lt)) * kLn2;
    }
}

template <typename T, int D>
FlashAttentionError paged_row(const PagedParams<T>& p, cudaStream_t stream) {
    paged_row_kernel<T, D><<<static_cast<unsigned>(p.num_tokens * p.hq), kRowThreads, 0, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? FlashAttentionError::SUCCESS
                                             : FlashAttentionError::CUDA_ERROR;
}

// ---------------------------------------------------------------------------
// Tensor-core kernel (pages of 8 rows and more); paged_line.cuh says how the
// work is divided.  One CTA per SM walks its segments (its parts of units).
// Two streams of 128 softmax threads take the steps in turn, so that one
// stream's softmax runs under the other's products:
//   two tiles:  row tile 0 and row tile 1 of the same key block, a thread per
//               row: S = Q K^T (M = N = 128), P over S in TMEM, O += P V;
//   one tile:   the same with alternate blocks of the one tile, each stream
//               with its own maximum, sum and output; the stream that had the
//               first block joins both from TMEM at the segment's end;
//   few rows:   alternate blocks too, but transposed, a thread per key:
//               S^T = K Q^T (M = 128 keys, N = 16 rows), P^T through shared
//               memory, O^T += V^T P^T (M = head_dim).  A thread of the tile
//               forms evaluates 128 exponentials per block however few rows
//               are live (8 cycles each on the MUFU pipe of its quarter);
//               here 128 threads on four quarters share them, and the result's
//               rows lie across the lanes, so they are stored coalesced.
//   warps 0, 3  TMA producers (query tiles and keys; values): blocks through
//               a ring of slots, one box per page and 64 columns, a lane each
//   warp 1      tcgen05.mma issuer: S(n+2) behind O(n)
//   warp 2      walks the line and hands out segments
//   warps 4-11  softmax and epilogue
// TMEM: S_t in columns [128 t, +128), O_t in [256 + 128 t, +D).  Arithmetic as
// in the dense forward: fp32 statistics in the log2 domain, O rescaled only
// where a row's maximum grows by more than 2^8, P rounded to the input type
// for its product, O accumulated in fp32.
//
// Bounds.  Row tiles: a block of two tiles takes 4 x 128 x 128 x D multiply-adds on
// the tensor pipe and 2 x 128 x 128 exponentials (1024 cycles each tile on the MUFU
// pipe), but neither is full: what a step costs is its chain (S, maximum,
// exponentials, P, O, the next S) shared by two streams.  Measured, from 256 tokens
// of 148 heads over 6144 and 12288 keys: 1.11 us a tile and block at D = 128 (1119
// TFLOP/s, 0.69 of cuBLAS' burst rate), 0.90 at D = 64, 0.79 at D = 32; pages of 128
// rows, 1.08 at D = 128.  The dense forward at the same sizes: 1.02, 0.83, 0.80.
// Few rows: the bytes of keys and values; 128 sequences of 4096 keys (8 K/V heads of
// 128, group 4) take 320 us, 6.7 TB/s.
// Times here and below, unless they say otherwise, are per call in a CUDA graph of 8
// to 12 calls, which keeps short runs at the burst clock and leaves the host out.
//
// Partials (normalised fp32 rows with their log2-sum-exp) are kept as
// [D/4][rows][4], so that a warp of row-per-lane threads stores and loads 512
// contiguous bytes (a 128-row tile of D = 128 is stored in 1.35 us this way,
// in 3.3 us row-major, where a warp's 16-byte pieces lie 4 D bytes apart).
// ---------------------------------------------------------------------------
__device__ sm100::StatusWord g_paged_status;

constexpr int kTcThreads = 384;
constexpr int kSegRing = 4;
constexpr float kRescale = 8.0f;  // log2 units
constexpr int kFewRows = kFewTile;  // N of the transposed products

// Where a CTA's piece of a line starts.
struct Start {
    Ctx ctx;
    long long base, x0, x1, per;  // line position of the context; the piece; its length
    int c;                        // the context, -2: no piece
};

template <int D>
struct PagedGeom {
    static constexpr int kRowBytes = D * 2;
    static constexpr int kSwz = kRowBytes >= 128 ? 128 : kRowBytes;
    static constexpr int kCbElems = kSwz / 2;
    static constexpr int kNumCb = D / kCbElems;
    static constexpr int kCbBytes = kTileRows * kSwz;
    static constexpr int kTileBytes = kTileRows * kRowBytes;
    // the transposed form is not built for 64-byte rows (head_dim 32)
    static constexpr bool kHasFew = D >= 64;
    // K and V blocks share one ring; at D = 128 five slots of 32 KB fill what
    // the two query tiles leave
    static constexpr int kSlots = D == 128 ? 5 : (D == 64 ? 9 : 12);
    static constexpr uint32_t kLayout = kSwz == 128 ? sm100::kLayoutSw128 : sm100::kLayoutSw64;
    // Few rows: a query slot holds the 16 query rows at the start of each
    // column block, and in between, from 4 KB on, each stream's P^T (two
    // 64-key column blocks of 16 rows) and the exchange of block maxima; it is
    // released when the segment's last product has read P^T.
    static constexpr int kQSlotBytes = kTileBytes < 16384 ? 16384 : kTileBytes;
    static constexpr int kOffPt = 4096;
    static constexpr int kPtBytes = 2 * kFewRows * 128;
    static constexpr int kOffMax = kOffPt + 2 * kPtBytes;  // [2 streams][2][4 warps][16]
    static constexpr int kOffRing = 2 * kQSlotBytes;
    // the transposed value product reads 128 columns from every slot; at D = 64
    // the upper 64 are the next slot's (rows of O^T nobody reads), so the last
    // slot is followed by as many bytes
    static constexpr int kPad = kHasFew ? 128 * 256 - kTileBytes : 0;
    static constexpr int kOffMl = kOffRing + kSlots * kTileBytes + kPad;
    static constexpr int kOffSeg = kOffMl + kTileRows * 8;
    static constexpr int kOffScan = kOffSeg + kSegRing * static_cast<int>(sizeof(Seg));
    static constexpr int kOffBar = kOffScan + 192 + 2 * static_cast<int>(sizeof(Start));
    static constexpr int kNumBars = 2 + 2 + 2 * kSlots + 5 * 2 + 2 + 2 * kSegRing + 1;
    static constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16 + 1024;
    static_assert(kOffBar % 8 == 0 && kSmemBytes <= 232448, "shared memory layout");
};

struct TcParams {
    PagedLine ln;
    void* O;
    float* L;
    float* O_part;
    float* L_part;  // log2-sum-exp of each partial row
    const int* prefix_table;
    const int* block_table;
    int few_tok;  // tokens of the few-rows query box
    int num_pages;
    float scale_log2;
    uint32_t wait_ticks;  // limit of a wait, in ticks of 1024 ns
    int hold_keys;        // tests: the first CTA's first keys never count as landed
};

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
// P^T, K-major: [2 blocks of 64 keys][16 rows][128 bytes]
__host__ __device__ constexpr uint32_t pt_delta(int kk) {
    return (static_cast<uint32_t>(kk >> 2) * (kFewRows * 128) + static_cast<uint32_t>(kk & 3) * 32u) >> 4;
}

// A box with an L2 priority.
__device__ __forceinline__ void tma_load_3d_hint(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y,
                                                 int z, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4, %5}], [%2], %6;\n" ::"r"(sm100::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(sm100::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "l"(policy)
        : "memory");
}

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(sm100::smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// For a converged warp of which one lane issues (`leader`, elected once per
// role): the products stand under one branch, their operands are computed by
// all lanes before it and stay in uniform registers.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(p));
    return p;
}
template <typename V>
__device__ __forceinline__ V uniform(V v) {
    return __shfl_sync(0xffffffffu, v, 0);
}
__device__ __forceinline__ void commit(uint32_t leader, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "setp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(
            sm100::smem_u32(bar)),
        "r"(leader)
        : "memory");
}

__device__ __forceinline__ float warp_max(float v) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}

// NC: columns of the few-rows form (contexts of more rows take row tiles).
template <typename T, int D, int NC>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQf,
                      const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ TcParams p) {
    using G = PagedGeom<D>;
    using namespace sm100;
    constexpr int R = G::kSlots;
    extern __shared__ uint8_t smem_raw[];
    const PagedLine& ln = p.ln;
    const int c_lo = ln.prefix_mode ? -1 : 0;
    const int run = (ln.B - c_lo + kTcThreads - 1) / kTcThreads;  // contexts per thread
    const int c_first = c_lo + static_cast<int>(threadIdx.x) * run;
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t sbase = (raw + 1023u) & ~1023u;
    uint8_t* sptr = smem_raw + (sbase - raw);
    uint64_t* bar_q = reinterpret_cast<uint64_t*>(sptr + G::kOffBar);  // [2] query tile landed
    uint64_t* bar_qfree = bar_q + 2;      // [2] its slot is free
    uint64_t* full = bar_qfree + 2;       // [R]
    uint64_t* empty = full + R;           // [R]
    uint64_t* bar_s = empty + R;          // [2] S_t in TMEM
    uint64_t* bar_p = bar_s + 2;          // [2] first half of P_t (few rows: P_t) stored
    uint64_t* bar_p2 = bar_p + 2;         // [2] second half
    uint64_t* bar_o = bar_p2 + 2;         // [2] O_t final for the segment
    uint64_t* bar_m = bar_o + 2;          // [2] few rows: the stream's warps have exchanged
    uint64_t* bar_x = bar_m + 2;          // second stream's state is there
    uint64_t* bar_y = bar_x + 1;          // it has been read
    uint64_t* seg_full = bar_y + 1;       // [kSegRing]
    uint64_t* seg_free = seg_full + kSegRing;  // [kSegRing]
    uint64_t* bar_done = seg_free + kSegRing;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    Seg* segs = reinterpret_cast<Seg*>(sptr + G::kOffSeg);
    long long* scan = reinterpret_cast<long long*>(sptr + G::kOffScan);  // [2 lines][12 warps]
    Start* start = reinterpret_cast<Start*>(scan + 24);                   // [2 lines]

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
            mbar_init(bar_m + t, 4);
        }
        for (int s = 0; s < R; ++s) {
            mbar_init(full + s, s == 0 && blockIdx.x == 0 && p.hold_keys ? 2 : 1);
            mbar_init(empty + s, 1);
        }
        mbar_init(bar_x, 128);
        mbar_init(bar_y, 128);
        for (int s = 0; s < kSegRing; ++s) {
            mbar_init(seg_full + s, 1);
            mbar_init(seg_free + s, 11);  // producers, MMA, 8 softmax warps
        }
        mbar_init(bar_done, 1);
        *abort_flag = 0;
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
        prefetch_tmap(&tmQ);
        prefetch_tmap(&tmQf);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    stream_wait();
    // the joining kernel's blocks may wait on the SMs this one leaves
    stream_release();
    int failed = 0;  // an earlier launch's failure
    if (threadIdx.x == 0) {
        failed = *reinterpret_cast<const volatile int*>(&g_paged_status.code);
        if (!ln.prefix_mode) reset_records(ln, static_cast<int>(blockIdx.x));
    }

    // ---- the lines: contexts' lengths summed over the block, then the context
    // each of this CTA's pieces starts in
        long long mine[2] = {0, 0};  // pass 0: lengths; pass 1: position behind the contexts so far
    Ctx ctx = {};
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
        for (int c = c_first; c < min(c_first + run, ln.B); ++c) {
            if (pass == 0 || run > 1) ctx = load_ctx(ln, c);
            const int l = line_of(ctx);
            const long long cost = ctx.head_cost * ln.heads;
            long long& at = l == kTiles ? mine[0] : mine[1];
            if (pass == 1) {
                Start& st = start[l];
                if (st.x0 < st.x1 && st.x0 >= at && st.x0 < at + cost) {
                    st.ctx = ctx;
                    st.base = at;
                    st.c = c;
                }
            }
            at += cost;
        }
        if (pass == 1) break;
#pragma unroll
        for (int l = 0; l < 2; ++l) {
            long long incl = mine[l];
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += v;
            }
            if (lane == 31) scan[l * 12 + warp] = incl;
            mine[l] = incl - mine[l];
        }
        if (__syncthreads_or(failed)) {
            if (warp == 1) tmem_dealloc(*tmem_slot, 512);
            return;
        }
        long long sum[2] = {0, 0};
#pragma unroll 1
        for (int w = 0; w < kTcThreads / 32; ++w) {
            if (w == warp) {
                mine[0] += sum[0];
                mine[1] += sum[1];
            }
            sum[0] += scan[w];
            sum[1] += scan[12 + w];
        }
        if (threadIdx.x < 2) {
            const long long line = threadIdx.x == kTiles ? sum[0] : sum[1];
            const int piece = piece_index(ln, static_cast<int>(threadIdx.x), static_cast<int>(blockIdx.x));
            Start& st = start[threadIdx.x];
            st.c = -2;
            st.per = piece_length(line, ln.pieces);
            st.x0 = min(piece * st.per, line);
            st.x1 = min(st.x0 + st.per, line);
        }
        __syncthreads();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Bounded waits, short enough to be inlined everywhere: a wait gives up when
    // it has lasted the limit or another role has given up; the role that ran out
    // records it on its way out.  All but one are for a block or so of another
    // role; warp 2's is for a whole segment.  (A limit on the time since a segment's
    // start failed at segments of some 200 million keys, and its clock, alive over
    // the whole segment, cost spills: long chunks 1688 us a call in a graph, 1643
    // so.)
    bool ok = true;
    auto tick = [] { return static_cast<uint32_t>(globaltimer_ns() >> 10); };  // about 1 us
    auto poll = [&](uint64_t* bar, uint32_t parity) -> bool {
        const uint32_t addr = smem_u32(bar);
        if (mbar_try_wait(addr, parity)) return true;
        const uint32_t since = tick();
#pragma unroll 1
        do {
            if (*abort_flag || tick() - since > p.wait_ticks) return false;
        } while (!mbar_try_wait(addr, parity));
        return true;
    };
    // The same for waits that are not urgent: a polling warp takes issue slots
    // from the softmax warps of its quarter.
    auto poll_idle = [&](uint64_t* bar, uint32_t parity, unsigned ns, uint32_t ticks) -> bool {
        const uint32_t addr = smem_u32(bar);
        if (mbar_try_wait(addr, parity)) return true;
        const uint32_t since = tick();
#pragma unroll 1
        do {
            if (*abort_flag || tick() - since > ticks) return false;
            __nanosleep(ns);
        } while (!mbar_try_wait(addr, parity));
        return true;
    };

    // Registers: launched with 168 per thread (384 x 168 = 64512); the first
    // warpgroup gives back down to 72 and the two softmax warpgroups take 216:
    // 128 * 72 + 256 * 216 = 64512.
    if (warp < 4) {
        setmaxnreg_dec<72>();
        if (warp == 0 || warp == 3) {
            // ------------------------------------------------ TMA producers
            // Warp 0 loads query tiles and keys, warp 3 values: with 16-row pages
            // one warp needs 0.7 us to issue the 16 boxes of a tile.
            const int v = warp == 0 ? 0 : 1;
            const CUtensorMap* map = v == 0 ? &tmK : &tmV;
            uint32_t q_cnt[2] = {0u, 0u};
            // this warp's fills are every other one of the ring: fill `fills` + v in
            // slot slot_kv; `phase`: parity of the slot's release before it
            int slot_kv = v, fills = 0;
            uint32_t phase = 1;
            int qs = 0;  // query slot of the next segment of one tile
            const int box_rows = min(1 << ln.page_shift, kBlockKeys);
            const int box_shift = min(ln.page_shift, 7);
            const int chunk_shift = box_shift - 2;      // log2 of key blocks per 32 boxes
            const int my_box = lane & 15;
            const int my_cb = lane >> 4;
            uint8_t* const my_dst = sptr + G::kOffRing + my_cb * G::kCbBytes + my_box * box_rows * G::kSwz;
            // Table entries come 32 boxes at a time, one per lane, a chunk ahead
            // (and the first of the next segment with this one's last block), so
            // that no copy waits for its page's index.
            auto load_entry = [&](const Seg& sg, int chunk) -> int {
                const int* table = sg.ctx < 0 ? p.prefix_table
                                              : p.block_table + static_cast<long long>(sg.ctx) * ln.max_pages;
                const long long row = (static_cast<long long>(chunk) * 32 + lane) << box_shift;
                return row < sg.len ? table[row >> ln.page_shift] : 0;
            };
            // Units of few rows read a key and its value once for all of the
            // sequence's rows, the row tiles of a prompt or prefix read theirs again,
            // so the former leave L2 first: 32 sequences behind 4096 keys 30.1 us
            // without priorities, 28.7 with, single tokens of 128 sequences of 512 keys
            // 59 and 56.  Tables may name a page in several rows, and then few rows do
            // read it again; that costs less than it gains elsewhere (single tokens of
            // 32 sequences over the same 4096 keys 75.2 us without, 76.9 with, of 128
            // over the same 8192 keys 481 and 496), and only a look at all tables
            // could tell the two apart.
            uint64_t once, again;
            asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
            asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(again));
            int entry_next_seg = 0;
            bool have_next = false;
#pragma unroll 1
            for (int k = 0;; ++k) {
                ok = poll(seg_full + k % kSegRing, (k / kSegRing) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const Seg sg = segs[k % kSegRing];
                __syncwarp();
                if (lane == 0) mbar_arrive(seg_free + k % kSegRing);
                if (sg.n_blk == 0) break;
                int chunk = sg.blk0 >> chunk_shift;
                int entry = entry_next_seg;
                if (!have_next) entry = load_entry(sg, chunk);
                int entry_after = load_entry(sg, chunk + 1);
                have_next = false;
                // query tiles
                if (lane == 0 && v == 0) {
                    const bool few = sg.mode == kFew;
                    const uint32_t bytes =
                        static_cast<uint32_t>(ln.gt * (few ? p.few_tok : ln.tpt)) * G::kRowBytes;
#pragma unroll 1
                    for (int u = 0; u < (sg.mode == kTwoTiles ? 2 : 1) && ok; ++u) {
                        const int slot = sg.mode == kTwoTiles ? u : qs;
                        if (q_cnt[slot] > 0) ok = poll_idle(bar_qfree + slot, (q_cnt[slot] - 1) & 1, 20, p.wait_ticks);
                        if (!ok) break;
                        mbar_arrive_expect_tx(bar_q + slot, bytes);
                        for (int cb = 0; cb < G::kNumCb; ++cb)
                            tma_load_3d(sptr + slot * G::kQSlotBytes + cb * G::kCbBytes, few ? &tmQf : &tmQ,
                                        bar_q + slot, cb * G::kCbElems, sg.head0, sg.tok0 + u * ln.tpt);
                        ++q_cnt[slot];
                    }
                }
                if (sg.mode != kTwoTiles) qs ^= 1;
                ok = __shfl_sync(0xffffffffu, ok, 0);
#pragma unroll 1
                for (int j = 0; ok && j < sg.n_blk; ++j) {
                    const int blk = sg.blk0 + j;
                    if (blk >> chunk_shift != chunk) {
                        ++chunk;
                        entry = entry_after;
                        entry_after = load_entry(sg, chunk + 1);
                    }
                    if (j + 1 == sg.n_blk &&
                        __all_sync(0xffffffffu, mbar_test(seg_full + (k + 1) % kSegRing,
                                                          ((k + 1) / kSegRing) & 1))) {
                        const Seg& nx = segs[(k + 1) % kSegRing];
                        if (nx.n_blk > 0) {
                            entry_next_seg = load_entry(nx, nx.blk0 >> chunk_shift);
                            have_next = true;
                        }
                    }
                    const int r0 = blk * kBlockKeys;
                    const int live = min(max(sg.len - r0, 0), kBlockKeys);
                    const int nbox = (live + box_rows - 1) >> box_shift;
                    const int row = r0 + (my_box << box_shift);
                    // a page index outside the pool reads a wrong page instead of faulting
                    const int page = min(max(__shfl_sync(0xffffffffu, entry, (row >> box_shift) & 31), 0),
                                         p.num_pages - 1);
                    const int row0 = (page << ln.page_shift) + (row & ((1 << ln.page_shift) - 1));
                    if (lane == 0) {
                        // the first lap's waits pass: no fill has used the slot
                        if (fills + v >= R) ok = poll_idle(empty + slot_kv, phase, 20, p.wait_ticks);
                        if (ok)
                            mbar_arrive_expect_tx(full + slot_kv,
                                                  static_cast<uint32_t>(nbox << box_shift) * G::kRowBytes);
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    if (!ok) break;
                    if (my_box < nbox && my_cb < G::kNumCb)
                        tma_load_3d_hint(my_dst + slot_kv * G::kTileBytes, map, full + slot_kv,
                                         my_cb * G::kCbElems, sg.hk, row0, sg.mode == kFew ? once : again);
                    slot_kv += 2;
                    if (slot_kv >= R) {
                        slot_kv -= R;
                        phase ^= 1;
                    }
                    fills += 2;
                }
                if (!ok) break;
            }
            // Every issued load lands before the CTA can exit: those of this warp's
            // fills that are the newest of their slots (older ones were consumed).
            if (lane == 0) {
                volatile int never = 0;
                const unsigned long long ns = static_cast<unsigned long long>(p.wait_ticks) << 10;
                for (int t = 0; t < 2; ++t)
                    if (q_cnt[t] > 0) mbar_wait(bar_q + t, (q_cnt[t] - 1) & 1, &never, &g_paged_status, ns);
                const int old = max(fills - R - v, 0);
                for (int g = old + (old & 1) + v; g < fills; g += 2)
                    mbar_wait(full + g % R, (g / R) & 1, &never, &g_paged_status, ns);
            }
            __syncwarp();
        } else if (warp == 1) {
            // ------------------------------------------------ MMA issuer
            // The warp stays converged and one elected lane issues: every value a
            // product takes is then warp-uniform for the compiler (registers of
            // the uniform datapath, no per-thread copies before each instruction).
            // What it spends between products is on every step's critical path,
            // so ring positions are counted up and a step waiting for its O is a
            // word of flags.
            {
                const uint32_t leader = elect_lane();
                const uint32_t tm = uniform(tmem);
                const uint32_t sb = uniform(sbase);
                auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                    ok = __all_sync(0xffffffffu, poll(bar, parity));
                    return ok;
                };
                // two at once: their first tries, usually successful, overlap
                auto wait2 = [&](uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) -> bool {
                    const bool ra = mbar_try_wait(smem_u32(a), pa), rb = mbar_try_wait(smem_u32(b), pb);
                    ok = __all_sync(0xffffffffu, (ra || poll(a, pa)) && (rb || poll(b, pb)));
                    return ok;
                };
                constexpr uint32_t idesc_qk = make_idesc(DType<T>::kMmaFmt, 128, 128, false, false);
                constexpr uint32_t idesc_pv = make_idesc(DType<T>::kMmaFmt, 128, D, false, true);
                constexpr uint32_t idesc_kq = make_idesc(DType<T>::kMmaFmt, 128, kFewRows, false, false);
                constexpr uint32_t idesc_vp = make_idesc(DType<T>::kMmaFmt, 128, kFewRows, true, false);
                constexpr uint32_t kDue = 1, kAcc = 2, kLast = 4, kWaitV = 8, kFreeV = 16, kIsFew = 32,
                                   kFreeQ = 64, kQSlot1 = 128;
                uint32_t ks = 0, kph = 0;  // ring slot and phase of the next block's K
                uint32_t vs = 1, vph = 0;  // of the V of the step whose O is next
                uint32_t due = 0;  // 16 bits per stream: its step that has its S but not its O
                uint32_t par = 0;  // bit t: phase of bar_p[t]
                uint32_t qph = 0;             // bit u: phase of bar_q[u]
                int k = 0, qs = 0, cur_q = 0;
                int i = 0, steps = 0, mode = kTwoTiles;
                bool end = false;
                bool k_ready = false;  // the next K fill is known to have landed
                auto next_slot = [](uint32_t& s, uint32_t& ph) {
                    s += 2;
                    if (s >= R) {
                        s -= R;
                        ph ^= 1;
                    }
                };
                // S of the next step, a row tile's
                auto rows_s = [&](int t) {
                    const int qslot = mode == kTwoTiles ? i & 1 : cur_q;
                    const uint64_t a0 = pg_kdesc<D>(sb + qslot * G::kQSlotBytes);
                    const uint64_t b0 = pg_kdesc<D>(sb + G::kOffRing + ks * G::kTileBytes);
                    if (leader)
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        mma_f16_ss(tm + t * 128, a0 + pg_kdelta<D>(kk), b0 + pg_kdelta<D>(kk), idesc_qk,
                                   kk > 0 ? 1u : 0u);
                };
                // behind an S: what waits for it, the step's flags, the next step
                auto s_issued = [&](int t) -> uint32_t {
                    commit(leader, bar_s + t);
                    uint32_t flags = kDue | (i >= 2 ? kAcc : 0) | (i + 2 >= steps ? kLast : 0);
                    if (mode == kTwoTiles) {
                        if (i + 2 >= steps) commit(leader, bar_qfree + (i & 1));
                        flags |= i & 1 ? kFreeV : kWaitV;
                    } else {
                        if (G::kHasFew && mode == kFew)
                            flags |= kIsFew | (cur_q ? kQSlot1 : 0) | (i + 1 == steps ? kFreeQ : 0);
                        else if (i + 1 == steps)
                            commit(leader, bar_qfree + cur_q);
                        flags |= kFreeV | kWaitV;
                    }
                    if (flags & kFreeV) {
                        commit(leader, empty + ks);
                        next_slot(ks, kph);
                    }
                    ++i;
                    return flags;
                };
                // S of the next step (stream t); its flags, 0 at the end
                auto issue_s = [&](int t) -> uint32_t {
                    if (i == steps) {
                        if (!wait(seg_full + k % kSegRing, (k / kSegRing) & 1)) return 0;
                        const Seg& sg = segs[k % kSegRing];
                        steps = uniform(sg.n_blk);
                        mode = uniform(sg.mode);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(seg_free + k % kSegRing);
                        ++k;
                        i = 0;
                        end = steps == 0;
                        if (end) return 0;
                        if (mode == kTwoTiles) {
                            steps *= 2;
                            if (!wait(bar_q, qph & 1) || !wait(bar_q + 1, qph >> 1)) return 0;
                            qph ^= 3;
                        } else {
                            cur_q = qs;
                            if (!wait(bar_q + qs, (qph >> qs) & 1)) return 0;
                            qph ^= 1u << qs;
                            qs ^= 1;
                        }
                    }
                    if (!(mode == kTwoTiles && (i & 1)) && !k_ready && !wait(full + ks, kph)) return 0;
                    k_ready = false;
                    tc_fence_after();
                    if (G::kHasFew && mode == kFew) {
                        const uint64_t a0 = pg_kdesc<D>(sb + cur_q * G::kQSlotBytes);
                        const uint64_t b0 = pg_kdesc<D>(sb + G::kOffRing + ks * G::kTileBytes);
                        if (leader)
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            mma_f16_ss(tm + t * 128, b0 + pg_kdelta<D>(kk), a0 + pg_kdelta<D>(kk), idesc_kq,
                                       kk > 0 ? 1u : 0u);
                    } else {
                        rows_s(t);
                    }
                    return s_issued(t);
                };
                // O of stream t's step, in step order; with `next`, the stream's next S
                // right behind it if that is in the segment and its keys have landed
                auto issue_o = [&](int t, uint32_t flags, uint32_t* next) -> bool {
                    bool with_s = false;
                    const uint32_t phase = (par >> t) & 1;
                    if (flags & kWaitV) {
                        if (!wait2(full + vs, vph, bar_p + t, phase)) return false;
                    } else if (!wait(bar_p + t, phase)) {
                        return false;
                    }
                    const uint64_t v0 = pg_vdesc<D>(sb + G::kOffRing + vs * G::kTileBytes);
                    const uint32_t o_tm = tm + 256 + t * 128;
                    const uint32_t acc = (flags & kAcc) ? 1u : 0u;
                    tc_fence_after();
                    if (G::kHasFew && (flags & kIsFew)) {
                        const uint32_t q_off = (flags & kQSlot1) ? G::kQSlotBytes : 0;
                        const uint64_t p0 = make_smem_desc(sb + q_off + G::kOffPt + t * G::kPtBytes, 16, 1024,
                                                     kLayoutSw128);
                        if (leader)
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            mma_f16_ss(o_tm, v0 + pg_vdelta<D>(kk), p0 + pt_delta(kk), idesc_vp,
                                       kk > 0 ? 1u : acc);
                        if (flags & kFreeQ) commit(leader, bar_qfree + ((flags & kQSlot1) ? 1 : 0));
                    } else {
                        if (leader)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_f16_ts(o_tm, tm + t * 128 + kk * 8, v0 + pg_vdelta<D>(kk), idesc_pv,
                                       kk > 0 ? 1u : acc);
                        const bool kr = (mode == kTwoTiles && (i & 1)) || mbar_test(full + ks, kph);
                        if (!wait(bar_p2 + t, phase)) return false;
                        k_ready = __all_sync(0xffffffffu, kr);
                        with_s = next != nullptr && k_ready && i != steps && mode != kFew;
                        tc_fence_after();
                        if (leader)
#pragma unroll
                        for (int kk = 4; kk < 8; ++kk)
                            mma_f16_ts(o_tm, tm + t * 128 + kk * 8, v0 + pg_vdelta<D>(kk), idesc_pv, 1u);
                    }
                    if (with_s) {
                        rows_s(t);
                        *next = s_issued(t);
                        k_ready = false;
                    }
                    if (flags & kLast) commit(leader, bar_o + t);
                    if (flags & kFreeV) {
                        commit(leader, empty + vs);
                        next_slot(vs, vph);
                    }
                    par ^= 1u << t;
                    return true;
                };
                // The streams' turns: O of one, then its next S behind it (in order,
                // so that S may overwrite P).  Issuing S earlier where TMEM has room for
                // P beside it (D = 64) only made the streams' softmax collide: 1.4 us a
                // step instead of 1.05.
#pragma unroll 1
                for (int t = 0;; t ^= 1) {
                    const uint32_t mine = (due >> (16 * t)) & 0xffffu;
                    uint32_t next = 0;
                    if (mine != 0 && !issue_o(t, mine, &next)) break;
                    // The other stream's O does not wait behind an S whose keys have
                    // not landed; and a segment of few rows ends with all its
                    // products, as the next one may need the query slot that holds P^T.
                    // (Two tiles take twice the products per key: their loads are ahead.)
                    uint32_t other = (due >> (16 * (t ^ 1))) & 0xffffu;
                    if (mode != kTwoTiles && other != 0 && next == 0) {
                        bool now = G::kHasFew && mode == kFew && i == steps;
                        uint32_t since = 0;  // of the second round
#pragma unroll 1
                        while (!now && i != steps && !__any_sync(0xffffffffu, mbar_test(full + ks, kph))) {
                            now = __any_sync(0xffffffffu, mbar_test(bar_p + (t ^ 1), (par >> (t ^ 1)) & 1));
                            if (since == 0) since = tick() | 1;
                            if (__any_sync(0xffffffffu, *abort_flag != 0 || static_cast<int>(tick() - since) >
                                                                                static_cast<int>(p.wait_ticks)))
                                break;
                        }
                        if (now) {
                            if (!issue_o(t ^ 1, other, nullptr)) break;
                            other = 0;
                        }
                    }
                    if (next == 0 && !end) next = issue_s(t);
                    due = (next << (16 * t)) | (other << (16 * (t ^ 1)));
                    if (!ok || due == 0) break;
                }
                // all products (and their commits) retire before teardown
                commit(leader, bar_done);
                volatile int never = 0;
                mbar_wait(bar_done, 0, &never, &g_paged_status);
            }
            __syncwarp();
        } else if (warp == 2) {
            // ------------------------------------------------ units and segments
            // The warp walks converged; lane 0 writes.  CTAs that share a TPC's
            // instruction cache go through the lines in the same order, their
            // neighbours in the other one.
            unsigned smid;
            asm volatile("mov.u32 %0, %%smid;" : "=r"(smid));
            int k = 0, longest = 0;  // segments; blocks of the longest, which a wait may be for
            auto emit = [&](const Seg& sg) {
                if (k >= kSegRing)
                    ok = __all_sync(0xffffffffu, poll_idle(seg_free + k % kSegRing, (k / kSegRing - 1) & 1, 500,
                                                           wait_ticks(p.wait_ticks, longest)));
                if (!ok) return;
                longest = max(longest, sg.n_blk);
                if (lane == 0) {
                    segs[k % kSegRing] = sg;
                    mbar_arrive(seg_full + k % kSegRing);
                }
                ++k;
            };
            // 32 contexts at a time: a batch may have many between two of a line
            auto next_ctx = [&](int c, int line, Ctx& out) -> int {
#pragma unroll 1
                for (int base = c + 1; base < ln.B; base += 32) {
                    Ctx x = {};
                    if (base + lane < ln.B) x = load_ctx(ln, base + lane);
                    const unsigned hit = __ballot_sync(0xffffffffu, x.head_cost != 0 && line_of(x) == line);
                    if (hit == 0) continue;
                    const int src = __ffs(hit) - 1;
                    out.tok = __shfl_sync(0xffffffffu, x.tok, src);
                    out.ntok = __shfl_sync(0xffffffffu, x.ntok, src);
                    out.len = __shfl_sync(0xffffffffu, x.len, src);
                    out.pairs = __shfl_sync(0xffffffffu, x.pairs, src);
                    out.last_mode = __shfl_sync(0xffffffffu, x.last_mode, src);
                    out.head_cost = __shfl_sync(0xffffffffu, x.head_cost, src);
                    return base + src;
                }
                return c;  // not reached while the walk is inside the line
            };
            Seg sg = {};
#pragma unroll 1
            for (int turn = 0; turn < 2 && ok; ++turn) {
                const int l = (turn ^ static_cast<int>(smid >> 1)) & 1;
                if (start[l].c < c_lo) continue;
                Walk w;
                walk_start(ln, w, start[l].ctx, start[l].c, start[l].base, start[l].x0, start[l].x1, start[l].per, l,
                           piece_index(ln, l, static_cast<int>(blockIdx.x)), lane == 0);
#pragma unroll 1
                while (ok && walk_next(ln, w, sg, next_ctx)) emit(sg);
            }
            sg.n_blk = 0;
            if (ok) emit(sg);
            __syncwarp();
        }
    } else {
        setmaxnreg_inc<216>();
        // ------------------------------------------------ softmax / epilogue
        const int t = (warp - 4) >> 2;
        const int wq = warp & 3;
        const int r = wq * 32 + lane;
        const int tok_r = r / ln.gt;
        const int head_r = r - tok_r * ln.gt;
        const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;
        const uint32_t s_tmem = tmem + lane_addr + t * 128;
        const uint32_t o_tmem = tmem + lane_addr + 256 + t * 128;
        const uint32_t o_other = tmem + lane_addr + 256 + (t ^ 1) * 128;
        float2* ml = reinterpret_cast<float2*>(sptr + G::kOffMl);
        const float c = p.scale_log2;
        uint32_t s_cnt = 0, o_cnt = 0, x_cnt = 0, m_cnt = 0;
        uint32_t n0 = 0;  // steps before the segment (its parity matters)
        int qs = 0;       // query slot of the next segment of one tile
        bool y_pending = false;
        uint32_t g0 = 0;  // key blocks before the segment
        // Rows behind the context's end hold whatever the page (or the ring)
        // had: this thread's V row is zeroed so that P = 0 meets no NaN.  The
        // block's V fill is waited for here; its slot's fill before that one was
        // read by a step at least two back, so the parity is not ambiguous.
        auto clean_v = [&](uint32_t fill, int live) -> bool {
            ok = __all_sync(0xffffffffu, poll(full + fill % R, (fill / R) & 1));
            if (ok && r >= live) {
                const uint32_t row = sbase + G::kOffRing + (fill % R) * G::kTileBytes + r * G::kSwz;
#pragma unroll
                for (int e = 0; e < G::kRowBytes / 16; ++e)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                                     row + (e * 16 / G::kSwz) * G::kCbBytes + e * 16 % G::kSwz),
                                 "r"(0u)
                                 : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            return ok;
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
            ok = __all_sync(0xffffffffu, poll(bar, parity));
            return ok;
        };
        // ======================================== few rows, transposed
        // Straight-line code for the kernel's 4, 8 or 16 columns: with one body
        // for 16 and a test per column, instruction fetches took most of a step.
        // Columns from ncol on hold garbage that stays in its column.
        auto few_rows = [&](const Seg& sg, int ncol, int first, int n) {
            const bool join = sg.n_blk > 1;
            const bool follower = first == 1;
            uint8_t* slot = sptr + qs * G::kQSlotBytes;
            const uint32_t pt = sbase + qs * G::kQSlotBytes + G::kOffPt + t * G::kPtBytes +
                                (r >> 6) * (kFewRows * 128) + (r & 7) * 2;
            float* rmax = reinterpret_cast<float*>(slot + G::kOffMax) + t * (2 * 4 * kFewRows);
            float* sums = reinterpret_cast<float*>(ml);  // [2 streams][4 warps][16]
            float* maxs = sums + 2 * 4 * kFewRows;       // [16], the second stream's
            float m_run[NC], neg_m[NC], l_part[NC];
#pragma unroll
            for (int g = 0; g < NC; ++g) {
                m_run[g] = -INFINITY;
                neg_m[g] = 0.f;
                l_part[g] = 0.f;
            }
#pragma unroll 1
            for (int j = 0; j < n; ++j) {
                if (!wait(bar_s + t, s_cnt & 1)) return;
                ++s_cnt;
                if (y_pending) {
                    if (!wait(bar_y, (x_cnt - 1) & 1)) return;
                    y_pending = false;
                }
                tc_fence_after();
                uint32_t sv[kFewRows];
                tmem_ld_x16(s_tmem, sv);
                const int key0 = (sg.blk0 + first + 2 * j) * kBlockKeys;
                if (key0 + kBlockKeys > sg.len || (ln.causal && key0 + kBlockKeys - 1 > sg.lim0)) {
                    int lim = ln.causal ? sg.lim0 : sg.len - 1, h = 0;
#pragma unroll
                    for (int g = 0; g < NC; ++g) {
                        if (key0 + r > min(lim, sg.len - 1)) sv[g] = __float_as_uint(-INFINITY);
                        if (++h == ln.gt) {  // the next token
                            h = 0;
                            lim += ln.causal;
                        }
                    }
                }
                if (key0 + kBlockKeys > sg.len &&
                    !clean_v(2 * (g0 + first + 2 * j) + 1, sg.len - key0))
                    return;
                float* rm = rmax + (j & 1) * (4 * kFewRows);
                float mx[NC];
#pragma unroll
                for (int g = 0; g < NC; ++g) mx[g] = warp_max(__uint_as_float(sv[g]));
                if (lane == 0) {
#pragma unroll
                    for (int g = 0; g < NC; g += 4)
                        *reinterpret_cast<float4*>(rm + wq * kFewRows + g) =
                            make_float4(mx[g], mx[g + 1], mx[g + 2], mx[g + 3]);
                    mbar_arrive(bar_m + t);
                }
                __syncwarp();
                if (!wait(bar_m + t, m_cnt & 1)) return;
                ++m_cnt;
                bool grow = false;
#pragma unroll
                for (int g = 0; g < NC; g += 4) {
                    const float4 a = *reinterpret_cast<const float4*>(rm + g);
                    const float4 b = *reinterpret_cast<const float4*>(rm + kFewRows + g);
                    const float4 d = *reinterpret_cast<const float4*>(rm + 2 * kFewRows + g);
                    const float4 e = *reinterpret_cast<const float4*>(rm + 3 * kFewRows + g);
                    mx[g] = fmaxf(fmax3(a.x, b.x, d.x), e.x) * c;
                    mx[g + 1] = fmaxf(fmax3(a.y, b.y, d.y), e.y) * c;
                    mx[g + 2] = fmaxf(fmax3(a.z, b.z, d.z), e.z) * c;
                    mx[g + 3] = fmaxf(fmax3(a.w, b.w, d.w), e.w) * c;
                }
#pragma unroll
                for (int g = 0; g < NC; ++g) grow = grow || mx[g] > m_run[g] + kRescale;
                if (grow) {  // uniform: every thread saw the same maxima
                    float alpha[NC];
#pragma unroll
                    for (int g = 0; g < NC; ++g) {
                        alpha[g] = 1.f;
                        if (mx[g] > m_run[g] + kRescale) {
                            alpha[g] = ex2_approx(m_run[g] - mx[g]);
                            m_run[g] = mx[g];
                            neg_m[g] = -mx[g];
                        }
                        l_part[g] *= alpha[g];
                    }
                    if (j > 0) {
                        uint32_t ov[kFewRows];
                        tmem_ld_x16(o_tmem, ov);
#pragma unroll
                        for (int g = 0; g < NC; ++g)
                            ov[g] = __float_as_uint(__uint_as_float(ov[g]) * alpha[g]);
                        tmem_st_x16(o_tmem, ov);
                    }
                }
#pragma unroll
                for (int g = 0; g < NC; ++g) {
                    const float pv = ex2_approx(fmaf(__uint_as_float(sv[g]), c, neg_m[g]));
                    l_part[g] += pv;
                    const T hv = DType<T>::from_float(pv);
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(pt + g * 128 +
                                                                 ((((r & 63) >> 3) ^ (g & 7)) << 4)),
                                 "h"(*reinterpret_cast<const uint16_t*>(&hv))
                                 : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_before();
                mbar_arrive(bar_p + t);
                mbar_arrive(bar_p2 + t);
            }
            if (join) ++x_cnt;
            if (n == 0) return;
#pragma unroll
            for (int g = 0; g < NC; ++g) {
                float v = l_part[g];
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
                l_part[g] = v;
            }
            if (!wait(bar_o + t, o_cnt & 1)) return;
            ++o_cnt;
            tc_fence_after();
            if (lane == 0) {
#pragma unroll
                for (int g = 0; g < NC; ++g) {
                    sums[(t * 4 + wq) * kFewRows + g] = l_part[g];
                    if (follower && wq == 0) maxs[g] = m_run[g];
                }
            }
            __syncwarp();
            if (follower) {
                tc_fence_before();
                mbar_arrive(bar_x);
                y_pending = true;
                return;
            }
            if (lane == 0) mbar_arrive(bar_m + t);
            if (!wait(bar_m + t, m_cnt & 1)) return;
            ++m_cnt;
            uint32_t ov[kFewRows], ov2[kFewRows];
            tmem_ld_x16(o_tmem, ov);
            if (join) {
                if (!wait(bar_x, (x_cnt - 1) & 1)) return;
                tc_fence_after();
                tmem_ld_x16(o_other, ov2);
            }
            int tok = 0, h = 0;
#pragma unroll
            for (int g = 0; g < NC; ++g) {
                const float* s0 = sums + t * 4 * kFewRows + g;
                float l = (s0[0] + s0[kFewRows]) + (s0[2 * kFewRows] + s0[3 * kFewRows]);
                float M = m_run[g], o = __uint_as_float(ov[g]);
                if (join) {
                    const float* s1 = sums + (t ^ 1) * 4 * kFewRows + g;
                    const float l1 = (s1[0] + s1[kFewRows]) + (s1[2 * kFewRows] + s1[3 * kFewRows]);
                    const float m1 = maxs[g];
                    M = fmaxf(M, m1);
                    const float w0 = M == -INFINITY ? 1.f : ex2_approx(m_run[g] - M);
                    const float w1 = M == -INFINITY ? 0.f : ex2_approx(m1 - M);
                    l = w0 * l + w1 * l1;
                    o = w0 * o + w1 * __uint_as_float(ov2[g]);
                }
                o *= l > 0.f ? __fdividef(1.f, l) : 0.f;
                const float lse2 = l == 0.f ? -INFINITY : M + __log2f(l);
                if (g < ncol && h < sg.nh && r < D) {  // lane r holds column r of the head
                    if (sg.part_row >= 0) {
                        p.O_part[static_cast<long long>(sg.part_row) * D + ((r >> 2) * sg.part_rows + g) * 4 +
                                 (r & 3)] = o;
                        if (r == 0) p.L_part[sg.part_row + g] = lse2;
                    } else {
                        const long long orow = static_cast<long long>(sg.tok0 + tok) * ln.hq + sg.head0 + h;
                        static_cast<T*>(p.O)[orow * D + r] = DType<T>::from_float(o);
                        if (r == 0) p.L[orow] = lse2 * kLn2;
                    }
                }
                if (++h == ln.gt) {
                    h = 0;
                    ++tok;
                }
            }
            if (join) {
                tc_fence_before();
                mbar_arrive(bar_y);
            }
        };
        int blocks = 0;  // of the last segment
#pragma unroll 1
        for (int k = 0; ok; ++k) {
            if (!wait(seg_full + k % kSegRing, (k / kSegRing) & 1)) break;
            const Seg sg = segs[k % kSegRing];
            g0 += blocks;
            blocks = sg.n_blk;
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_free + k % kSegRing);
            if (sg.n_blk == 0) break;
            const bool two = sg.mode == kTwoTiles;
            const int first = (t ^ n0) & 1;  // two tiles: this stream's tile; else: its first block
            const int n = two ? sg.n_blk : (sg.n_blk - first + 1) / 2;
            n0 += two ? 2 * sg.n_blk : sg.n_blk;
            const bool join = !two && sg.n_blk > 1;  // both streams have a part
            const bool follower = !two && first == 1;

            if (G::kHasFew && sg.mode == kFew) {
                few_rows(sg, min((sg.tok_end - sg.tok0) * ln.gt, NC), first, n);
                qs ^= 1;
                if (!ok) break;
                continue;
            }

            // ============================================ row tiles
            if (!two) qs ^= 1;
            const int tile = two ? first : 0;
            const int token = sg.tok0 + tile * ln.tpt + tok_r;
            const bool valid = tok_r < ln.tpt && head_r < sg.nh && token < sg.tok_end;
            const bool active = __any_sync(0xffffffffu, valid);
            const int tile_lim = sg.lim0 + tile * ln.tpt;  // first row's limit
            // last key this row sees
            const int row_end = ln.causal ? min(sg.len - 1, tile_lim + tok_r) : sg.len - 1;

            float m_run = -INFINITY, l_run = 0.f;
#pragma unroll 1
            for (int j = 0; j < n; ++j) {
                if (!wait(bar_s + t, s_cnt & 1)) break;
                ++s_cnt;
                if (y_pending) {  // the other stream has read the last segment's O_t
                    if (!wait(bar_y, (x_cnt - 1) & 1)) break;
                    y_pending = false;
                }
                const int in_seg = two ? j : first + 2 * j;  // key block
                const int col0 = (sg.blk0 + in_seg) * kBlockKeys;
                // (two tiles: tile 0's product is issued before tile 1's)
                if (col0 + kBlockKeys > sg.len && tile == 0 &&
                    !clean_v(2 * (g0 + in_seg) + 1, sg.len - col0))
                    break;
                if (!active) {
                    mbar_arrive(bar_p + t);
                    mbar_arrive(bar_p2 + t);
                    continue;
                }
                tc_fence_after();
                uint32_t sr[128];
                tmem_ld_x128(s_tmem, sr);
                if (col0 + kBlockKeys > sg.len || (ln.causal && col0 + kBlockKeys - 1 > tile_lim)) {
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
#pragma unroll 1
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
            if (join) ++x_cnt;
            if (n == 0) continue;
            if (!wait(bar_o + t, o_cnt & 1)) break;
            ++o_cnt;
            tc_fence_after();
            if (follower) {
                ml[r] = make_float2(m_run, l_run);
                tc_fence_before();
                mbar_arrive(bar_x);
                y_pending = true;
                continue;
            }
            float w0 = 1.f, w1 = 0.f;  // O = w0 O_t + w1 O_other, and the sums alike
            if (join) {
                if (!wait(bar_x, (x_cnt - 1) & 1)) break;
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
            const float inv_l = l_run > 0.f ? __fdividef(1.f, l_run) : 0.f;
            w0 *= inv_l;
            w1 *= inv_l;
            const float lse2 = l_run == 0.f ? -INFINITY : m_run + __log2f(l_run);  // NaN stays NaN
            if (active) {
                const long long prow = static_cast<long long>(sg.part_row) + tile * kTileRows;
                const long long orow = static_cast<long long>(token) * ln.hq + sg.head0 + head_r;
#pragma unroll 1
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
                            float4* dst = reinterpret_cast<float4*>(p.O_part + prow * D) + r;
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                dst[(cb * 8 + i) * sg.part_rows] =
                                    make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
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
                        p.L_part[prow + r] = lse2;
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

    if (!ok && lane == 0 && !*abort_flag) {
        *abort_flag = 1;
        record_status(&g_paged_status, kStatusWaitTimeout);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// The second kernel: joins partial rows by their log2-sum-exp.  A block takes 32
// rows (one per lane, so that loads of the partials' layout are contiguous) and
// 8 or 32 columns; its 8 warps share the partials (warp w those at w, w + 8, ...),
// and their sums are joined through shared memory in warp order, so a result
// depends on the lengths alone.  Bound by latency: with the maxima, weights and
// products of all partials in one warp after the other, 37 partials took 26 us,
// this way one round of loads and one exchange.  Measured: about 4 us behind the
// first kernel's end in a small call, of which 1.5 are that end.
// ---------------------------------------------------------------------------
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
// Columns of a block: the prefix join's blocks each know their rows, and fewer
// columns make more of them (32, 16 or 8 columns: 19 sequences behind 5003 keys 25.6,
// 23.7, 23.3 us, 4 behind 512 14.2, 13.5, 13.0, and the largest alike, 128 behind
// 32768 152.1, 150.4, 150.8); the ragged one's have to find them, and more columns
// make fewer searches (32 or 16: one chunk of 33 tokens 16.9, 21.2, 16 mixed sequences
// 110.7, 116.3).
constexpr int kPrefixCols = 8;
constexpr int kSplitCols = 32;

// A lane's partials: n of them, tiles of `rows` rows `step` rows apart from
// `base` on, row r of each.
struct Parts {
    int n, base, step, rows, r;
};

template <typename T, int C>
struct JoinSmem {
    float4 acc[kJoinWarps][C / 4][32];
    float top[kJoinWarps][32];
    float tot[kJoinWarps][32];
    int row[32];
    __align__(16) T tile[32][C + 8];
};

// A lane's running maximum, sum and output, and two partials into it (their
// loads in flight together; the second may be absent).
template <int C>
struct JoinState {
    float top, tot;
    float4 acc[C / 4];
};

template <int C>
__device__ __forceinline__ void join_init(JoinState<C>& st) {
    st.top = -INFINITY;
    st.tot = 0.f;
#pragma unroll
    for (int q = 0; q < C / 4; ++q) st.acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
}

struct PartRow {
    int tile_row, rows, r;
};

template <int D, int C>
__device__ __forceinline__ void join_two(const TcParams& p, JoinState<C>& st, const PartRow& a, const PartRow& b,
                                         bool has_b, int col0) {
    constexpr int Q = C / 4;
    const float4* src0 = reinterpret_cast<const float4*>(p.O_part + static_cast<long long>(a.tile_row) * D) +
                         (col0 / 4) * a.rows + a.r;
    const float4* src1 = reinterpret_cast<const float4*>(p.O_part + static_cast<long long>(b.tile_row) * D) +
                         (col0 / 4) * b.rows + b.r;
    float4 v0[Q], v1[Q];
    const float l0 = p.L_part[a.tile_row + a.r];
    const float l1 = has_b ? p.L_part[b.tile_row + b.r] : -INFINITY;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        v0[q] = src0[q * a.rows];
        v1[q] = has_b ? src1[q * b.rows] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float m = fmaxf(fmaxf(st.top, l0), l1);
    const float m0 = m == -INFINITY ? 0.f : m;
    const float w = sm100::ex2_approx(st.top - m0);
    const float w0 = sm100::ex2_approx(l0 - m0), w1 = sm100::ex2_approx(l1 - m0);
    st.top = m;
    st.tot = st.tot * w + (w0 + w1);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        st.acc[q].x = fmaf(w1, v1[q].x, fmaf(w0, v0[q].x, st.acc[q].x * w));
        st.acc[q].y = fmaf(w1, v1[q].y, fmaf(w0, v0[q].y, st.acc[q].y * w));
        st.acc[q].z = fmaf(w1, v1[q].z, fmaf(w0, v0[q].z, st.acc[q].z * w));
        st.acc[q].w = fmaf(w1, v1[q].w, fmaf(w0, v0[q].w, st.acc[q].w * w));
    }
}

// Partial k of two lists, one behind the other.
__device__ __forceinline__ PartRow part_row(const Parts& a, const Parts& b, int k) {
    return k < a.n ? PartRow{a.base + k * a.step, a.rows, a.r}
                   : PartRow{b.base + (k - a.n) * b.step, b.rows, b.r};
}

// Joins the partials of both lists, a lane's row going to out_row (-1: none),
// columns [col0, col0 + C).
template <typename T, int D, int C>
__device__ __forceinline__ void join_rows(const TcParams& p, JoinSmem<T, C>& sm, const Parts& a, const Parts& b,
                                          int out_row, int col0) {
    constexpr int Q = C / 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = a.n + b.n;
    JoinState<C> st;
    join_init(st);
#pragma unroll 1
    for (int k = warp; k < n; k += 2 * kJoinWarps)
        join_two<D>(p, st, part_row(a, b, k), part_row(a, b, min(k + kJoinWarps, n - 1)), k + kJoinWarps < n, col0);
    __syncthreads();  // the last use of the shared memory is over
#pragma unroll
    for (int q = 0; q < Q; ++q) sm.acc[warp][q][lane] = st.acc[q];
    sm.top[warp][lane] = st.top;
    sm.tot[warp][lane] = st.tot;
    if (warp == 0) sm.row[lane] = out_row;
    __syncthreads();
    if (warp < Q) {  // columns 4 warp .. 4 warp + 3
        float M = -INFINITY;
#pragma unroll
        for (int u = 0; u < kJoinWarps; ++u) M = fmaxf(M, sm.top[u][lane]);
        const float M0 = M == -INFINITY ? 0.f : M;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float tot = 0.f;
#pragma unroll
        for (int u = 0; u < kJoinWarps; ++u) {
            const float w = sm100::ex2_approx(sm.top[u][lane] - M0);
            const float4 v = sm.acc[u][warp][lane];
            tot = fmaf(w, sm.tot[u][lane], tot);
            o.x = fmaf(w, v.x, o.x);
            o.y = fmaf(w, v.y, o.y);
            o.z = fmaf(w, v.z, o.z);
            o.w = fmaf(w, v.w, o.w);
        }
        const float inv = tot > 0.f ? __fdividef(1.f, tot) : 0.f;
        uint2 packed;
        packed.x = DType<T>::pack2(o.x * inv, o.y * inv);
        packed.y = DType<T>::pack2(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>(&sm.tile[lane][warp * 4]) = packed;
        if (warp == 0 && col0 == 0 && out_row >= 0)
            p.L[out_row] = tot == 0.f ? -INFINITY : (M + __log2f(tot)) * kLn2;
    }
    __syncthreads();
    const int r = threadIdx.x / (C / 8), c = threadIdx.x % (C / 8) * 8;
    if (r < 32 && sm.row[r] >= 0)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.O) + static_cast<long long>(sm.row[r]) * D + col0 + c) =
            *reinterpret_cast<const uint4*>(&sm.tile[r][c]);
}

// The first kernel's writes are visible behind this; nonzero: it failed (asked
// for together with the records, which are only used if it did not).
__device__ __forceinline__ int partials_wait() {
    stream_wait();
    return *reinterpret_cast<const volatile int*>(&g_paged_status.code);
}

// Block (32 rows of the batch's row tiles, head chunk, columns): the prefix's
// partials, then the sequence's own.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
    paged_join_prefix_kernel(const __grid_constant__ TcParams p) {
    __shared__ JoinSmem<T, kPrefixCols> sm;
    const PagedLine& ln = p.ln;
    const int hc = blockIdx.y;
    const int row = blockIdx.x * 32 + (threadIdx.x & 31);  // of the head chunk
    const int tile = row / kTileRows;
    const int r = row % kTileRows;
    const int tok_r = r / ln.gt;
    const int hr = r - tok_r * ln.gt;
    const int b = tile * ln.tpt + tok_r;
    const int hk = ln.chunks == 1 ? hc : hc / ln.chunks;
    const int head = hk * ln.group + (hc - hk * ln.chunks) * ln.gt + hr;
    const bool valid = tok_r < ln.tpt && b < ln.B && head < (hk + 1) * ln.group;
    stream_release();
    const int u0 = hc * ln.prefix_pairs + (tile >> 1), u1 = b * ln.heads + hc;
    const int failed = partials_wait();
    // lengths and spans are asked for together: a unit without keys has no span, and
    // what stands in its place is not used
    const Span none = {0, -1};
    Span sp0 = none, sp1 = none;
    if (valid) {
        const int own_len = ln.seq_lens[b], prefix_len = *ln.prefix_len;
        sp0 = ln.span[u0];
        sp1 = ln.span[ln.heads * ln.prefix_pairs + u1];
        if (prefix_len <= 0) sp0 = none;
        if (own_len <= 0) sp1 = none;
    }
    if (__syncthreads_or(failed)) return;
    const Parts pre = {sp0.last - sp0.first + 1, (u0 + sp0.first) * (2 * kTileRows) + (tile & 1) * kTileRows,
                       2 * kTileRows, kTileRows, r};
    const Parts own = {sp1.last - sp1.first + 1, ln.own_part_row + (u1 + sp1.first) * ln.gt, ln.gt, ln.gt, hr};
    join_rows<T, D>(p, sm, pre, own, valid ? b * ln.hq + head : -1, blockIdx.z * kPrefixCols);
}

// The ragged units that several pieces share, 32 rows and 32 columns at a time.
// Every block lists their records.  Units of few partials, the usual kind, are
// joined by single warps, a lane per row, without any exchange; the others by
// whole blocks as above.  Little code: in a small call most of it is fetched cold
// (an exact count of every unit's items, 20 us instead of 17 for a chunk of 33
// tokens).  With 2, 4 or 8 partials as few: the chunk of 33 tokens 17.7, 17.7, 23.7 us,
// 16 mixed sequences 109.2, 111.1, 114.3, 7 scored without a mask 35.5, 34.8, 34.9.
constexpr int kLightParts = 4;
struct Record {
    int tok0, head0, parts;
    int nh_tokens;  // heads << 16 | tokens (256 at most)
};
constexpr int kMaxRecords = 2 * kJoinThreads;  // two per thread; two per SM

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
    paged_join_split_kernel(const __grid_constant__ TcParams p) {
    constexpr int kColGroups = D / kSplitCols;
    constexpr int kItems = 2 * kTileRows / 32 * kColGroups;  // of a record
    __shared__ JoinSmem<T, kSplitCols> sm;
    __shared__ short list[2][kMaxRecords];  // [light, heavy]: their records
    __shared__ int counts[2][kJoinWarps];
    __shared__ Record recs[kMaxRecords];
    const PagedLine& ln = p.ln;
    stream_release();
    const int failed = partials_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n_rec = 2 * ln.pieces;
    const int run = (n_rec + kJoinThreads - 1) / kJoinThreads;
    auto piece_of = [&](int i) -> int { return i < ln.pieces ? i : i - ln.pieces; };
    auto record = [&](int i) -> Record {
        const Split sp = ln.split[i];
        return Record{sp.tok0, sp.head0, sp.last - piece_of(i) + 1,
                      sp.nh << 16 | min(sp.tok_end - sp.tok0, sp.mode == kTwoTiles ? 2 * ln.tpt : ln.tpt)};
    };
    // a thread's two loads are in flight together
    const int i0 = threadIdx.x * run, i1 = min(i0 + run, n_rec) - 1;
    int parts[2] = {0, 0};
    if (i0 < n_rec) {
        const Record a = record(i0), b = record(i1);
        recs[i0] = a;
        recs[i1] = b;
        parts[0] = a.parts;
        if (i1 > i0) parts[1] = b.parts;
    }
    int rank[2];
    bool is[2][2];
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            is[kind][k] = kind ? parts[k] > kLightParts : parts[k] > 1 && parts[k] <= kLightParts;
        const unsigned a = __ballot_sync(0xffffffffu, is[kind][0]), b = __ballot_sync(0xffffffffu, is[kind][1]);
        const unsigned before = (1u << lane) - 1;
        rank[kind] = __popc(a & before) + __popc(b & before);
        if (lane == 0) counts[kind][warp] = __popc(a) + __popc(b);
    }
    if (__syncthreads_or(failed)) return;
    int total[2] = {0, 0};
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            if (w == warp) rank[kind] += total[kind];
            total[kind] += counts[kind][w];
        }
        if (is[kind][0]) list[kind][rank[kind]++] = static_cast<short>(i0);
        if (is[kind][1]) list[kind][rank[kind]] = static_cast<short>(i1);
    }
    __syncthreads();
    struct Item {
        Parts head, rest;
        int out_row, col0;
    };
    // item `at` of a kind, for this lane's row.  Every record has the items of 256
    // rows; where the unit has fewer, no lane has one.  A record's are turned by
    // its number, so that a warp does not meet the same rows of one on every lap
    // (16 mixed sequences 110.0 us, 113.1 unturned).
    auto find = [&](int at, int kind) -> Item {
        const int nth = at / kItems, rec = list[kind][nth], left = (at + 5 * nth) % kItems;
        const Record u = recs[rec];
        const bool few = rec >= ln.pieces;
        const int i = piece_of(rec);
        const int row = left / kColGroups * 32 + lane;
        const int tile = row / kTileRows;
        const int r = row % kTileRows;
        const int tok_r = r / ln.gt;
        const int hr = r - tok_r * ln.gt;
        const int token = tile * ln.tpt + tok_r;  // of the unit
        const bool valid = tok_r < ln.tpt && hr < (u.nh_tokens >> 16) && token < (u.nh_tokens & 0xffff);
        // piece i's last segment, then the first ones of the pieces behind it
        const int rows = few ? kFewTile : kTileRows;      // of a tile
        const int slot = few ? kFewTile : 2 * kTileRows;  // of a segment
        const int base = (few ? ln.few_part_row : tile * kTileRows) + 2 * i * slot;
        return Item{Parts{valid ? 1 : 0, base + slot, 0, rows, r},
                    Parts{valid ? u.parts - 1 : 0, base + 2 * slot, 2 * slot, rows, r},
                    valid ? (u.tok0 + token) * ln.hq + u.head0 + hr : -1, left % kColGroups * kSplitCols};
    };
    const int light = total[0] * kItems, heavy = total[1] * kItems;
#pragma unroll 1
    for (int at = blockIdx.x; at < heavy; at += gridDim.x) {
        const Item it = find(at, 1);
        if (!__any_sync(0xffffffffu, it.out_row >= 0)) continue;  // the same in every warp
        join_rows<T, D>(p, sm, it.head, it.rest, it.out_row, it.col0);
    }
#pragma unroll 1
    for (int at = (gridDim.x - 1 - blockIdx.x) * kJoinWarps + warp; at < light; at += gridDim.x * kJoinWarps) {
        const Item it = find(at, 0);
        if (it.out_row < 0) continue;
        constexpr int Q = kSplitCols / 4;
        JoinState<kSplitCols> st;
        join_init(st);
        const int n = it.rest.n + 1;
#pragma unroll 1
        for (int k = 0; k < n; k += 2)
            join_two<D>(p, st, part_row(it.head, it.rest, k), part_row(it.head, it.rest, min(k + 1, n - 1)),
                        k + 1 < n, it.col0);
        const float inv = st.tot > 0.f ? __fdividef(1.f, st.tot) : 0.f;
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.O) + static_cast<long long>(it.out_row) * D + it.col0);
#pragma unroll
        for (int q = 0; q < Q; q += 2) {
            uint4 v;
            v.x = DType<T>::pack2(st.acc[q].x * inv, st.acc[q].y * inv);
            v.y = DType<T>::pack2(st.acc[q].z * inv, st.acc[q].w * inv);
            v.z = DType<T>::pack2(st.acc[q + 1].x * inv, st.acc[q + 1].y * inv);
            v.w = DType<T>::pack2(st.acc[q + 1].z * inv, st.acc[q + 1].w * inv);
            dst[q / 2] = v;
        }
        if (it.col0 == 0) p.L[it.out_row] = st.tot == 0.f ? -INFINITY : (st.top + __log2f(st.tot)) * kLn2;
    }
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

template <typename T, int D, int NC>
FlashAttentionError paged_tc(const PagedParams<T>& a, cudaStream_t stream) {
    using G = PagedGeom<D>;
    TcParams p{};
    PagedLine& ln = p.ln;
    p.O = a.O;
    p.L = a.L;
    p.prefix_table = a.prefix_table;
    p.block_table = a.block_table;
    p.num_pages = a.num_pages;
    // a zero scale becomes a tiny positive one so that masked scores stay -inf
    p.scale_log2 = fmaxf(a.scale_log2, 1e-30f);
    const int limit_ms = std::min(env_int("CUFLASH_TEST_WAIT_LIMIT_MS", 0), 100000);
    const unsigned long long limit_ns = limit_ms > 0 ? limit_ms * 1000000ull : sm100::kWaitTimeoutNs;
    p.wait_ticks = static_cast<uint32_t>(limit_ns >> 10);
    p.hold_keys = env_int("CUFLASH_TEST_SKIP_K_LOAD", 0) != 0;
    ln.prefix_len = a.prefix_len;
    ln.seq_lens = a.seq_lens;
    ln.cu_seqlens = a.cu_seqlens;
    ln.prefix_mode = a.prefix_table != nullptr;
    ln.causal = a.causal;
    ln.num_tokens = a.num_tokens;
    ln.B = a.B;
    ln.hq = a.hq;
    ln.hkv = a.hkv;
    ln.page_shift = a.page_shift;
    ln.max_prefix_pages = a.max_prefix_pages;
    ln.max_pages = a.max_pages;
    set_tiles(ln, G::kHasFew ? NC : 0);
    p.few_tok = std::max(1, kFewRows / ln.gt);
    const int grid = persistent_grid(0x7fffffffLL, 1);
    long long rows, records;
    if (!set_parts(ln, grid, rows, records) || ln.heads > 65535 || 2 * grid > kMaxRecords) return FlashAttentionError::INVALID_DIMENSION;

    const CUtensorMapDataType dt = DType<T>::kTmaType;
    const CUtensorMapSwizzle swz = G::kSwz == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    CUtensorMap mq, mqf, mk, mv;
    {
        const uint64_t dims[3] = {D, static_cast<uint64_t>(a.hq), static_cast<uint64_t>(a.num_tokens)};
        const uint64_t strides[2] = {D * 2, static_cast<uint64_t>(a.hq) * D * 2};
        const uint32_t gt = static_cast<uint32_t>(ln.gt);
        const uint32_t box[3] = {G::kCbElems, gt, static_cast<uint32_t>(ln.tpt)};
        const uint32_t boxf[3] = {G::kCbElems, gt, static_cast<uint32_t>(p.few_tok)};
        if (!encode_tmap_3d_strided(&mq, a.Q, dt, dims, strides, box, swz) ||
            !encode_tmap_3d_strided(&mqf, a.Q, dt, dims, strides, boxf, swz))
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
    auto kern = paged_attn_kernel<T, D, NC>;
    if (!ensure_smem_attr(reinterpret_cast<const void*>(kern), G::kSmemBytes))
        return FlashAttentionError::CUDA_ERROR;

    // workspace: records of the units' pieces, partial rows
    const size_t off_rec = 0;
    const size_t off_l = off_rec + align256(static_cast<size_t>(records));
    const size_t off_o = off_l + align256(static_cast<size_t>(rows) * sizeof(float));
    const size_t bytes = off_o + static_cast<size_t>(rows) * D * sizeof(float);
    void* ws = nullptr;
    const FlashAttentionError werr = workspace_alloc(&ws, bytes, stream);
    if (werr != FlashAttentionError::SUCCESS) return werr;
    char* base = static_cast<char*>(ws);
    ln.span = reinterpret_cast<Span*>(base + off_rec);
    ln.split = reinterpret_cast<Split*>(base + off_rec);
    p.L_part = reinterpret_cast<float*>(base + off_l);
    p.O_part = reinterpret_cast<float*>(base + off_o);

    bind_status_word(reinterpret_cast<const void*>(&g_paged_status), stream);
    cudaError_t err = launch_behind(kern, dim3(grid), kTcThreads, G::kSmemBytes, stream, mq, mqf, mk, mv, p);
    if (err == cudaSuccess) {
        if (ln.prefix_mode) {
            const int tiles = (ln.B + ln.tpt - 1) / ln.tpt;
            const int last = (ln.B - (tiles - 1) * ln.tpt) * ln.gt;  // rows of the last tile
            const int groups = (tiles - 1) * (kTileRows / 32) + (last + 31) / 32;
            err = launch_behind(paged_join_prefix_kernel<T, D>, dim3(groups, ln.heads, D / kPrefixCols), kJoinThreads, 0,
                                stream, p);
        } else {
            // As many blocks as are resident at once, two per SM (three, with fewer
            // registers: 16 mixed sequences 110.0 us against 112.6, but a chunk of 33
            // tokens 18.2 against 16.9).
            err = launch_behind(paged_join_split_kernel<T, D>, dim3(2 * grid), kJoinThreads, 0, stream, p);
        }
    }
    if (err != cudaSuccess) cudaGetLastError();
    workspace_free(ws, stream);
    return err == cudaSuccess ? FlashAttentionError::SUCCESS : FlashAttentionError::CUDA_ERROR;
}

template <typename T, int D>
FlashAttentionError paged_typed(const PagedParams<T>& p, cudaStream_t stream) {
    if (p.page_shift < 3) return paged_row<T, D>(p, stream);
    if constexpr (PagedGeom<D>::kHasFew) {
        // one token's heads fit the few-rows form up to groups of 16
        const int group = p.hq / p.hkv;
        if (group > 4 && group <= 8) return paged_tc<T, D, 8>(p, stream);
        if (group > 8 && group <= 16) return paged_tc<T, D, 16>(p, stream);
    }
    return paged_tc<T, D, 4>(p, stream);
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
