// Attention of one new token per sequence over a paged KV cache.
//
//   out = sum_j exp(scale q . k_j - m) v_j / sum_j exp(scale q . k_j - m),  j < len,  m = max_j scale q . k_j
//
// One pass over the keys with a running maximum and sum, in fp32. A block takes one query head of one
// sequence; its warps take the keys in turn and join at the end.
#include <cfloat>

#include "paged.cuh"
#include "../runtime/internal.h"

namespace vkb
{
namespace
{

constexpr uint32_t kAttThreads = 256;

struct PagedAttArgs
{
    vkllm_b200_paged_kv kv;
    vkllm_b200_paged_table t;
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;
    const uint32_t *lens;
    uint32_t heads;
    float scale;
    uint32_t *status;
};

template <typename T> __global__ void __launch_bounds__(kAttThreads) k_paged_attention(const PagedAttArgs a)
{
    __shared__ float acc_sm[kAttThreads / 32][256], m_sm[kAttThreads / 32], l_sm[kAttThreads / 32];
    const uint32_t h = blockIdx.x, s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t hd = a.kv.head_dim, R = a.kv.page_rows, kh = h / (a.heads / a.kv.kv_heads);
    const uint64_t cap = table_rows(a.t);
    uint32_t len = a.lens[s], e = 0;
    if (len > cap)
        len = (uint32_t)cap, e = VKLLM_B200_PAGED_TOO_LONG;
    float q[8], acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const uint32_t d = lane + 32 * i;
        q[i] = d < hd ? to_f32<T>(((const T *)a.q)[s * a.q_stride + (uint64_t)h * hd + d]) : 0.f;
        acc[i] = 0.f;
    }
    for (uint32_t j = warp; j < len; j += kAttThreads / 32)
    {
        const uint32_t page = a.t.table[s * a.t.stride + j / R];
        if (page >= a.t.n_pages)
        {
            e |= VKLLM_B200_PAGED_BAD_PAGE;
            continue;
        }
        const uint64_t at = page * a.kv.page_stride + kh * a.kv.head_stride + (j % R) * a.kv.row_stride;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd)
                dot = fmaf(q[i], to_f32<T>(((const T *)a.kv.k)[at + lane + 32 * i]), dot);
        dot = warp_sum(dot) * a.scale;
        const float mn = fmaxf(m, dot), base = mn == -INFINITY ? 0.f : mn;
        const float p = expf(dot - base), f = expf(m - base);
        m = mn;
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd)
                acc[i] = fmaf(p, to_f32<T>(((const T *)a.kv.v)[at + lane + 32 * i]), acc[i] * f);
    }
    if (e && lane == 0)
        atomicOr(a.status, e);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        acc_sm[warp][lane + 32 * i] = acc[i];
    if (lane == 0)
        m_sm[warp] = m, l_sm[warp] = l;
    __syncthreads();
    float mx = -INFINITY;
    for (uint32_t w = 0; w < kAttThreads / 32; ++w)
        mx = fmaxf(mx, m_sm[w]);
    if (mx == -INFINITY)
        mx = 0.f;
    for (uint32_t d = threadIdx.x; d < hd; d += kAttThreads)
    {
        float o = 0.f, sum = 0.f;
        for (uint32_t w = 0; w < kAttThreads / 32; ++w)
        {
            const float f = expf(m_sm[w] - mx);
            o = fmaf(f, acc_sm[w][d], o);
            sum = fmaf(f, l_sm[w], sum);
        }
        ((T *)a.out)[s * a.out_stride + (uint64_t)h * hd + d] = from_f32<T>(sum == 0.f ? 0.f : o / sum);
    }
}

} // namespace
} // namespace vkb

extern "C" vkllm_err_t vkllm_b200_paged_attention(const struct vkllm_b200_paged_kv *kv,
                                                  const struct vkllm_b200_paged_table *t, const void *q,
                                                  uint64_t q_stride, uint32_t heads, const uint32_t *lens, float scale,
                                                  void *out, uint64_t out_stride, void *workspace,
                                                  uint64_t workspace_bytes, uint32_t *status, void *stream)
{
    using namespace vkb;
    _CHECK_ARGS(kv_fits(kv) && table_fits(t));
    _CHECK_ARGS(t->page_rows == kv->page_rows && t->n_pages == kv->n_pages);
    _CHECK_ARGS(heads > 0 && heads <= 65535 && heads % kv->kv_heads == 0 && t->n_seqs <= 65535);
    const uint32_t es = paged_elem_bytes(kv->dtype);
    const uint64_t width = (uint64_t)heads * kv->head_dim;
    _CHECK_ARGS(rows_fit(q, q_stride, width, es) && rows_fit(out, out_stride, width, es) && q != out);
    _CHECK_ARGS(words(lens) && words(status));
    _CHECK_ARGS(workspace && aligned_to(workspace, 16) && workspace_bytes >= VKLLM_B200_PAGED_WORKSPACE_BYTES);
    int sms = 0, dev = 0;
    _CHECK(check_device(kv->k, &sms, &dev));
    const PagedAttArgs a{*kv, *t, q, out, q_stride, out_stride, lens, heads, scale, status};
    const dim3 grid(heads, t->n_seqs);
    if (kv->dtype == vkllm_dtype_float16)
        k_paged_attention<__half><<<grid, kAttThreads, 0, (cudaStream_t)stream>>>(a);
    else
        k_paged_attention<float><<<grid, kAttThreads, 0, (cudaStream_t)stream>>>(a);
    VKB_CUDA(cudaGetLastError());
    return VKLLM_ERR_OK;
}
