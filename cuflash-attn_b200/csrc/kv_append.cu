// Appending keys and values to a paged cache, with the rotary position
// rotation applied on the way (no reference counterpart: the reference has
// no KV cache).
//
// For token t of sequence b, at index p of the sequence (its last new token
// sits at seq_lens[b] - 1): every pair (x0, x1) of a query or key head's
// first rotary_dim elements becomes
//     x0 cos a - x1 sin a,   x1 cos a + x0 sin a
// with cos a, sin a from row `position` of a table the caller lays out once;
// pairs are (i, i + rotary_dim/2), or (2i, 2i + 1) when interleaved.  The key
// and value rows go to page block_table[b][p / page_size], slot
// p % page_size; the queries to Q_out.
//
// Bound by bytes: each 16-bit element is read once and written once (24.6 kB
// per token of 32 query heads and 8 key/value heads of 128), the angles' row
// (512 B in fp32) serves every head of the token.  A block of 128 threads takes
// one token; a thread owns the same 16 bytes (8 elements) of every head it
// visits, so the angles it needs stay in registers, and it issues the loads of
// all its heads before it looks up the token's sequence, so that the dependent
// look-ups (sequence, length, page) overlap them.  The partner of an element
// is half a rotation away in the same head and is fetched from the owning lane
// by a shuffle.  Measured, at those sizes: 26915 tokens in 103 us (6.5 TB/s of
// elements, the rate of a plain copy); 256 tokens every 3.0 us inside a graph,
// which is the launch and the chain of look-ups.

#include "common.cuh"
#include "paged.cuh"

namespace cuflash {
namespace detail {

namespace {

constexpr int kAppendThreads = 128;
constexpr int kAppendHeads = 6;  // heads in flight per thread

template <typename T>
struct AppendParams {
    const T* Q;  // nullptr: keys and values only
    const T* K;
    const T* V;
    T* Q_out;
    T* K_cache;
    T* V_cache;
    const float* rope;  // [max_position, rotary_dim], nullptr: no rotation
    const int* positions;
    const int* block_table;
    const int* seq_lens;
    const int* cu_seqlens;  // nullptr: token t is sequence t's only one
    long long q_stride, k_stride, v_stride;
    int B, hq, hkv;
    int page_shift, max_pages, num_pages;
    int rotary_dim, max_position;
};

// 8 packed 16-bit elements, read once and written once: both pass L2 by as far as
// they can (116.7 us with plain accesses, 103.0 so; the attention behind it takes
// as long either way).  Not the read-only path: queries may be rotated in place.
__device__ __forceinline__ uint4 load16(const void* p) {
    return __ldcs(reinterpret_cast<const uint4*>(p));
}

template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads)
    kv_append_kernel(const AppendParams<T> p) {
    constexpr int kChunks = D / 8;                        // threads per head
    constexpr int kSlots = kAppendThreads / kChunks;      // heads per pass of the block
    const int lane = threadIdx.x & 31;
    const int c = threadIdx.x % kChunks;
    const int slot = threadIdx.x / kChunks;
    const int t = blockIdx.x;
    const int heads = p.hq + 2 * p.hkv;  // query heads, then key heads, then value heads

    auto src = [&](int h) -> const T* {
        if (h < p.hq) return p.Q + t * p.q_stride + h * D + c * 8;
        if (h < p.hq + p.hkv) return p.K + t * p.k_stride + (h - p.hq) * D + c * 8;
        return p.V + t * p.v_stride + (h - p.hq - p.hkv) * D + c * 8;
    };
    stream_release();
    stream_wait();
    uint4 x[kAppendHeads];
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i) {
        const int h = slot + i * kSlots;
        x[i] = h < heads ? load16(src(h)) : make_uint4(0, 0, 0, 0);
    }

    int b = t, first_from_end = 1;  // the token is that many from its sequence's end
    if (p.cu_seqlens != nullptr) {
        b = sequence_of_token(p.cu_seqlens, p.B, t);
        if (b < 0) return;  // behind the last sequence
        first_from_end = p.cu_seqlens[b + 1] - t;
    }
    const int idx = p.seq_lens[b] - first_from_end;
    // where the token's key and value go; tokens without a place in the cache
    // (an index outside the table, a page outside the pool) are not stored
    const int page_idx = idx >> p.page_shift;
    const bool in_table = idx >= 0 && page_idx < p.max_pages;
    const int page =
        in_table ? p.block_table[static_cast<long long>(b) * p.max_pages + page_idx] : -1;
    const bool stored = page >= 0 && page < p.num_pages;
    const long long row = (static_cast<long long>(page) << p.page_shift) +
                          (idx & ((1 << p.page_shift) - 1));

    const int half = p.rotary_dim / 2;
    const bool rotated = p.rope != nullptr && c * 8 < p.rotary_dim;
    float cs[8], sn[8];  // element e of the chunk: y = x * cs + partner * sn
    if (rotated) {
        int pos = p.positions != nullptr ? p.positions[t] : idx;
        pos = min(max(pos, 0), p.max_position - 1);
        const float* row_cos = p.rope + static_cast<long long>(pos) * p.rotary_dim;
        const float* row_sin = row_cos + half;
        if constexpr (kInterleaved) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(row_cos + c * 4));
            const float4 s = __ldg(reinterpret_cast<const float4*>(row_sin + c * 4));
            const float av[4] = {a.x, a.y, a.z, a.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                cs[e] = av[e / 2];
                sn[e] = (e & 1) ? sv[e / 2] : -sv[e / 2];
            }
        } else {
            const bool low = c * 8 < half;
            const int i0 = low ? c * 8 : c * 8 - half;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float4 a = __ldg(reinterpret_cast<const float4*>(row_cos + i0) + q);
                const float4 s = __ldg(reinterpret_cast<const float4*>(row_sin + i0) + q);
                cs[4 * q] = a.x; cs[4 * q + 1] = a.y; cs[4 * q + 2] = a.z; cs[4 * q + 3] = a.w;
                sn[4 * q] = low ? -s.x : s.x;
                sn[4 * q + 1] = low ? -s.y : s.y;
                sn[4 * q + 2] = low ? -s.z : s.z;
                sn[4 * q + 3] = low ? -s.w : s.w;
            }
        }
    }
    // lane that owns the partner elements (non-interleaved; multiples of 8 apart)
    const int partner = rotated ? (c * 8 < half ? lane + half / 8 : lane - half / 8) : lane;

    for (int h0 = slot;; h0 += kAppendHeads * kSlots) {
#pragma unroll
        for (int i = 0; i < kAppendHeads; ++i) {
            const int h = h0 + i * kSlots;
            uint4 y = x[i];
            if (p.rope != nullptr) {  // uniform: every lane reaches the shuffles
                uint4 o = x[i];
                if constexpr (!kInterleaved) {
                    o.x = __shfl_sync(0xffffffffu, x[i].x, partner);
                    o.y = __shfl_sync(0xffffffffu, x[i].y, partner);
                    o.z = __shfl_sync(0xffffffffu, x[i].z, partner);
                    o.w = __shfl_sync(0xffffffffu, x[i].w, partner);
                }
                if (rotated && h < p.hq + p.hkv) {
                    const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                    const uint32_t os[4] = {o.x, o.y, o.z, o.w};
                    uint32_t ys[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float2 a = DType<T>::unpack2(xs[q]);
                        float2 w = DType<T>::unpack2(os[q]);
                        if constexpr (kInterleaved) w = make_float2(a.y, a.x);
                        // products and sum in fp32, rounded once to the cache's type
                        ys[q] = DType<T>::pack2(fmaf(a.x, cs[2 * q], w.x * sn[2 * q]),
                                                fmaf(a.y, cs[2 * q + 1], w.y * sn[2 * q + 1]));
                    }
                    y = make_uint4(ys[0], ys[1], ys[2], ys[3]);
                }
            }
            if (h < heads) {
                T* dst = nullptr;
                if (h < p.hq)
                    dst = p.Q_out + (static_cast<long long>(t) * p.hq + h) * D + c * 8;
                else if (stored)
                    dst = (h < p.hq + p.hkv ? p.K_cache + (row * p.hkv + (h - p.hq)) * D
                                            : p.V_cache + (row * p.hkv + (h - p.hq - p.hkv)) * D) +
                          c * 8;
                if (dst != nullptr) __stcs(reinterpret_cast<uint4*>(dst), y);
            }
        }
        // the block's head ranges are the same for every slot up to one head,
        // so this bound is uniform over the block
        const int next = h0 - slot + kAppendHeads * kSlots;
        if (next >= heads) break;
#pragma unroll
        for (int i = 0; i < kAppendHeads; ++i) {
            const int h = next + slot + i * kSlots;
            x[i] = h < heads ? load16(src(h)) : make_uint4(0, 0, 0, 0);
        }
    }
}

template <typename T, int D>
FlashAttentionError append_typed(const AppendParams<T>& p, int num_tokens, bool interleaved,
                                 cudaStream_t stream) {
    const cudaError_t err = launch_behind(interleaved ? kv_append_kernel<T, D, true>
                                                      : kv_append_kernel<T, D, false>,
                                          dim3(num_tokens), kAppendThreads, 0, stream, p);
    if (err != cudaSuccess) cudaGetLastError();
    return err == cudaSuccess ? FlashAttentionError::SUCCESS : FlashAttentionError::CUDA_ERROR;
}

}  // namespace

template <typename T>
FlashAttentionError launch_kv_append(const T* Q, const T* K, const T* V, T* Q_out, T* K_cache,
                                     T* V_cache, const float* rope, const int* positions,
                                     const int* block_table, const int* seq_lens,
                                     const int* cu_seqlens, int num_tokens, int B, int Hq, int Hkv,
                                     int D, int page_size, int max_pages, int num_pages,
                                     long long q_stride, long long k_stride, long long v_stride,
                                     int rotary_dim, int max_position, bool interleaved,
                                     cudaStream_t stream) {
    for (const void* ptr : {static_cast<const void*>(Q), static_cast<const void*>(K),
                            static_cast<const void*>(V), static_cast<const void*>(Q_out),
                            static_cast<const void*>(K_cache), static_cast<const void*>(V_cache),
                            static_cast<const void*>(rope)})
        if ((reinterpret_cast<uintptr_t>(ptr) & 15u) != 0) return FlashAttentionError::CUDA_ERROR;
    AppendParams<T> p;
    p.Q = Q;
    p.K = K;
    p.V = V;
    p.Q_out = Q_out;
    p.K_cache = K_cache;
    p.V_cache = V_cache;
    p.rope = rope;
    p.positions = positions;
    p.block_table = block_table;
    p.seq_lens = seq_lens;
    p.cu_seqlens = cu_seqlens;
    p.hq = Q != nullptr ? Hq : 0;
    p.hkv = Hkv;
    p.B = B;
    p.q_stride = q_stride != 0 ? q_stride : static_cast<long long>(Hq) * D;
    p.k_stride = k_stride != 0 ? k_stride : static_cast<long long>(Hkv) * D;
    p.v_stride = v_stride != 0 ? v_stride : static_cast<long long>(Hkv) * D;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.max_pages = max_pages;
    p.num_pages = num_pages;
    p.rotary_dim = rotary_dim;
    p.max_position = max_position;
    switch (D) {
        case 32:
            return append_typed<T, 32>(p, num_tokens, interleaved, stream);
        case 64:
            return append_typed<T, 64>(p, num_tokens, interleaved, stream);
        case 128:
            return append_typed<T, 128>(p, num_tokens, interleaved, stream);
        default:
            return FlashAttentionError::UNSUPPORTED_HEAD_DIM;
    }
}

#define CUFLASH_APPEND_INST(T)                                                                     \
    template FlashAttentionError launch_kv_append<T>(                                              \
        const T*, const T*, const T*, T*, T*, T*, const float*, const int*, const int*,            \
        const int*, const int*, int, int, int, int, int, int, int, int, long long, long long,      \
        long long, int, int, bool, cudaStream_t);
CUFLASH_APPEND_INST(__nv_bfloat16)
CUFLASH_APPEND_INST(half)
#undef CUFLASH_APPEND_INST

}  // namespace detail
}  // namespace cuflash
