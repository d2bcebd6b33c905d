// What the paged serving kernels (paged_tables.cu, paged_rope.cu, paged_attention.cu, logits_rules.cu)
// share: checks of arguments on the host and of values on the device.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>
#include <initializer_list>

#include "../runtime/internal.h"
#include "common.cuh"
#include "vkllm_b200_paged.h"
#include "vkllm_common.h"
#include "vkllm_log.h"

namespace vkb
{

// Pages that hold `rows` rows.
__host__ __device__ __forceinline__ uint32_t pages_of(uint64_t rows, uint32_t page_rows)
{
    return (uint32_t)((rows + page_rows - 1) / page_rows);
}

// Rows that a sequence's row of the table has room for.
__host__ __device__ __forceinline__ uint64_t table_rows(const vkllm_b200_paged_table &t)
{
    return (uint64_t)t.cols * t.page_rows;
}

// The status bits of `len` cached rows and of one page id, shared by the kernels and the host check.
__host__ __device__ __forceinline__ uint32_t length_status(const vkllm_b200_paged_table &t, uint64_t len)
{
    return len > table_rows(t) || len > 0xffffffffull ? (uint32_t)VKLLM_B200_PAGED_TOO_LONG : 0u;
}
__host__ __device__ __forceinline__ uint32_t page_status(uint32_t page, uint32_t n_pages)
{
    return page >= n_pages ? (uint32_t)VKLLM_B200_PAGED_BAD_PAGE : 0u;
}

// Largest i < n with start[i] <= x, for ascending start and start[0] <= x.
__device__ __forceinline__ uint32_t last_at_most(const uint32_t *start, uint32_t n, uint32_t x)
{
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1)
    {
        const uint32_t mid = (lo + hi) >> 1;
        if (start[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

inline bool aligned_to(const void *p, uintptr_t bytes)
{
    return ((uintptr_t)p & (bytes - 1)) == 0;
}

// A non-null pointer to 32-bit words.
inline bool words(const void *p)
{
    return p && aligned_to(p, 4);
}

// Refuses arrays that the current device does not own: a launch on them would fault or read across the bus
// (null pointers are passed over). *sms receives the SM count of the current device. Looking at a pointer
// takes the host 50 ns.
vkllm_err_t check_device(std::initializer_list<const void *> arrays, int *sms, int *device);

// Launches a kernel without attributes and returns its own status: cudaGetLastError after <<<>>> would also tell of
// errors of earlier calls.
template <typename Args>
vkllm_err_t launch_plain(void (*kernel)(const Args), const Args &args, dim3 grid, uint32_t threads, size_t smem,
                         cudaStream_t s)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    VKB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    return VKLLM_ERR_OK;
}

// A table whose shape fits (the pointers' targets are not looked at).
inline bool table_fits(const vkllm_b200_paged_table *t)
{
    return t && words(t->table) && t->n_seqs > 0 && t->cols > 0 && t->page_rows > 0 && t->n_pages > 0 &&
           t->stride >= t->cols && t->stride < (1ull << 40) && (uint64_t)t->n_pages * t->page_rows <= 0xffffffffull;
}

inline uint32_t paged_elem_bytes(uint32_t dtype)
{
    return dtype == vkllm_dtype_float16 ? 2u : dtype == vkllm_dtype_float32 ? 4u : 0u;
}

// Rows of `width` elements read and written 16 bytes at a time.
inline bool rows_fit(const void *p, uint64_t stride, uint64_t width, uint32_t elem)
{
    return p && aligned_to(p, 16) && stride >= width && stride < (1ull << 40) && stride * elem % 16 == 0;
}

inline bool kv_fits(const vkllm_b200_paged_kv *kv)
{
    const uint32_t es = kv ? paged_elem_bytes(kv->dtype) : 0;
    if (!es || kv->reserved != 0)
        return false;
    return kv->k && kv->v && aligned_to(kv->k, 16) && aligned_to(kv->v, 16) && kv->n_pages > 0 && kv->page_rows > 0 &&
           (uint64_t)kv->n_pages * kv->page_rows <= 0xffffffffull && kv->kv_heads > 0 && kv->kv_heads <= 65535 &&
           kv->head_dim > 0 && kv->head_dim <= 256 && kv->head_dim * es % 16 == 0 && kv->page_stride * es % 16 == 0 &&
           kv->head_stride * es % 16 == 0 && kv->row_stride * es % 16 == 0 && kv->page_stride < (1ull << 40) &&
           kv->head_stride < (1ull << 40) && kv->row_stride < (1ull << 40) &&
           (kv->page_rows == 1 || kv->row_stride >= kv->head_dim) &&
           (kv->kv_heads == 1 || kv->head_stride >= kv->head_dim);
}

} // namespace vkb
