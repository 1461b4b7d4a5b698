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
// CUDA-core kernel: one block per (token, query head), any page size.  Lane
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
        attend(p.prefix_table, min(max(*p.prefix_len, 0), p.max_prefix_pages << p.page_shift));
    int n = min(max(p.seq_lens[b], 0), p.max_pages << p.page_shift);
    if (p.causal) n = min(n, p.seq_lens[b] - from_end + 1);
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
FlashAttentionError paged_typed(const PagedParams<T>& p, cudaStream_t stream) {
    paged_row_kernel<T, D><<<static_cast<unsigned>(p.num_tokens * p.hq), kRowThreads, 0, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? FlashAttentionError::SUCCESS
                                             : FlashAttentionError::CUDA_ERROR;
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

#define CUFLASH_PAGED_INST(T)                                                                     \
    template FlashAttentionError launch_paged_attention<T>(                                       \
        const T*, const T*, const T*, const int*, const int*, const int*, const int*, const int*, \
        T*, float*, int, int, int, int, int, int, int, int, int, float, bool, cudaStream_t);
CUFLASH_PAGED_INST(__nv_bfloat16)
CUFLASH_PAGED_INST(half)
#undef CUFLASH_PAGED_INST

}  // namespace detail
}  // namespace cuflash
