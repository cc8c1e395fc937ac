// Attention of new tokens over a paged cache.
#include <math_constants.h>

#include "common.cuh"

namespace qb {

struct AttentionParams {
    __nv_bfloat16* out;
    const __nv_bfloat16 *q, *k, *v;
    const int *page_table, *kv_lens, *cu;
    long long o_token, o_head, q_token, q_head, k_page, k_token, k_head, v_page, v_token, v_head;
    float scale;
    int rows, batch, width, hq, hkv, num_pages, page;
};

// One warp per row and head, the running maximum and sum of the softmax over the keys one by one; a lane owns D / 32 columns.
template <int D>
__global__ void __launch_bounds__(128) paged_attention_simple_kernel(const AttentionParams p) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long long item = blockIdx.x * 4ll + (threadIdx.x >> 5);
    const int row = (int)(item / p.hq), h = (int)(item % p.hq);
    if (row >= p.rows) return;
    int lo = 0, hi = p.batch;  // the request of the row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid + 1] > row) hi = mid; else lo = mid + 1;
    }
    if (lo == p.batch || row < p.cu[0]) return;
    const int n = p.cu[lo + 1] - p.cu[lo], kv = min(max(p.kv_lens[lo], 0), p.width * p.page);
    const int seen = kv - n + (row - p.cu[lo]) + 1, kvh = h / (p.hq / p.hkv);
    float q[E], o[E], m = -CUDART_INF_F, l = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = __bfloat162float(p.q[row * p.q_token + h * p.q_head + lane * E + e]) * p.scale;
        o[e] = 0;
    }
    for (int j = 0; j < seen; ++j) {
        const int page = p.page_table[(long long)lo * p.width + j / p.page];
        const bool there = page >= 0 && page < p.num_pages;
        const __nv_bfloat16* k = p.k + (there ? page : 0) * p.k_page + (j % p.page) * p.k_token + kvh * p.k_head + lane * E;
        const __nv_bfloat16* v = p.v + (there ? page : 0) * p.v_page + (j % p.page) * p.v_token + kvh * p.v_head + lane * E;
        float s = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) s += there ? q[e] * __bfloat162float(k[e]) : 0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
        const float top = fmaxf(m, s), c = __expf(m - top), x = __expf(s - top);
        m = top;
        l = l * c + x;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + (there ? x * __bfloat162float(v[e]) : 0);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) p.out[row * p.o_token + h * p.o_head + lane * E + e] = __float2bfloat16(seen > 0 ? o[e] / l : 0);
}

}  // namespace qb

using namespace qb;

extern "C" int paged_attention_workspace(int rows, int batch, int n_head, int n_kv_head, int head_dim) {
    return 0;
}

extern "C" int paged_attention_cuda_bf16(void* out, const long long* out_strides, const void* q, const long long* q_strides,
                                         const void* k_cache, const long long* k_strides, const void* v_cache,
                                         const long long* v_strides, const int* page_table, const int* kv_lens, const int* cu_new,
                                         void* workspace, float scale, int rows, int batch, int width, int n_head, int n_kv_head,
                                         int head_dim, int num_pages, int page_size, cudaStream_t stream) {
    if (rows < 0 || batch < 0 || width < 0 || n_head <= 0 || n_kv_head <= 0 || num_pages < 0 || page_size <= 0) return QB200_ERR_INVALID_ARGUMENT;
    if (rows == 0 || batch == 0) return QB200_OK;
    if (!out || !out_strides || !q || !q_strides || !k_strides || !v_strides || !kv_lens || !cu_new || (width && !page_table) ||
        (num_pages && (!k_cache || !v_cache)))
        return QB200_ERR_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || n_head % n_kv_head != 0 || (page_size != 16 && page_size != 32 && page_size != 64 && page_size % 128 != 0) ||
        (long long)width * page_size > 0x7fffffffll || !aligned16(out) || !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache))
        return QB200_ERR_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (k_strides[i] % 8 || v_strides[i] % 8 || (i < 2 && (q_strides[i] % 8 || out_strides[i] % 8))) return QB200_ERR_UNSUPPORTED;
    AttentionParams p{static_cast<__nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(k_cache),
                      static_cast<const __nv_bfloat16*>(v_cache), page_table, kv_lens, cu_new, out_strides[0], out_strides[1],
                      q_strides[0], q_strides[1], k_strides[0], k_strides[1], k_strides[2], v_strides[0], v_strides[1], v_strides[2],
                      scale, rows, batch, width, n_head, n_kv_head, num_pages, page_size};
    const long long blocks = ((long long)rows * n_head + 3) / 4;
    if (head_dim == 64) paged_attention_simple_kernel<64><<<(unsigned)blocks, 128, 0, stream>>>(p);
    else paged_attention_simple_kernel<128><<<(unsigned)blocks, 128, 0, stream>>>(p);
    return launch_status();
}
