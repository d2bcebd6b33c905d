// Page tables and slot maps of a paged KV cache, built on the GPU from the sequences' lengths.
//
//   want[s]   = ceil((len[s] + new[s]) / R) - ceil(len[s] / R)      pages of R rows each
//   starts    = exclusive sum of new, first = exclusive sum of want
//   page j of all new pages (first[s] <= j < first[s + 1]) is free[n_free - 1 - j] and goes to
//   table[s][ceil(len[s] / R) + j - first[s]]
//   token t (starts[s] <= t < starts[s + 1]): position p = len[s] + t - starts[s],
//   slot = table[s][p / R] * R + p % R
//
// The floor is the words in and out (8 bytes a token and 20 a sequence), microseconds at most: the calls
// are bound by the latency of one launch and of a few dependent loads.
//
// One thread-block cluster does a call (but for the slots of many tokens, which a second kernel spreads
// over the GPU). Every CTA sums all sequences itself (they are few; a scan split over CTAs would need an
// exchange more) into shared memory, then takes its share of the tokens, pages and sequences, found by
// binary search in the sums, so one long prompt among many short ones spreads evenly. The cluster barrier
// between the last read and the first write is what makes all-or-nothing and new_lens == lens possible. The
// CTAs say at their start that they run: only then may another one write their shared memory.
#include <atomic>
#include <cooperative_groups.h>
#include <vector>

#include "paged.cuh"
#include "../runtime/internal.h"

namespace vkb
{

vkllm_err_t check_device(std::initializer_list<const void *> arrays, int *sms, int *device)
{
    int dev = 0;
    VKB_CUDA(cudaGetDevice(&dev));
    for (const void *p : arrays)
    {
        cudaPointerAttributes a;
        if (!p)
            continue;
        VKB_CUDA(cudaPointerGetAttributes(&a, p));
        if ((a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) || a.device != dev)
        {
            log_error("an array is not memory of the current device (%d)", dev);
            return VKLLM_ERR_ARGS;
        }
    }
    if (device)
        *device = dev;
    if (sms)
        VKB_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    return VKLLM_ERR_OK;
}

namespace
{

constexpr uint32_t kMaxSeqs = 16384; // three words a sequence in shared memory
constexpr uint32_t kTabThreads = 512;
constexpr uint32_t kMaxCluster = 8;
// Most tokens whose slots the cluster writes itself. More go to a second kernel over the whole GPU: a
// release and an append of 131072 tokens in 512 sequences took 23.9 us with one cluster for all, and take
// 13.5 this way.
constexpr uint32_t kTokensHere = kMaxCluster * kTabThreads;
constexpr uint32_t kSlotThreads = 256;

struct AppendArgs
{
    vkllm_b200_paged_table t;
    const uint32_t *lens, *n_new, *n_free;
    uint32_t *new_lens, *n_free_out, *starts, *slots, *positions;
    uint32_t max_tokens;
    uint32_t *status;
};

struct ReleaseArgs
{
    vkllm_b200_paged_table t;
    const uint32_t *lens, *done, *n_free;
    uint32_t *new_lens, *n_free_out;
    uint32_t *status;
};

// Exclusive sum over the block's threads of a pair of 64-bit counts; *ta, *tb receive the totals.
__device__ void block_sums(uint64_t &a, uint64_t &b, uint64_t *ta, uint64_t *tb)
{
    __shared__ uint64_t wa[kTabThreads / 32], wb[kTabThreads / 32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t sa = a, sb = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const uint64_t xa = __shfl_up_sync(0xffffffffu, sa, o), xb = __shfl_up_sync(0xffffffffu, sb, o);
        if (lane >= o)
            sa += xa, sb += xb;
    }
    if (lane == 31)
        wa[warp] = sa, wb[warp] = sb;
    __syncthreads();
    uint64_t pa = 0, pb = 0, qa = 0, qb = 0;
#pragma unroll
    for (uint32_t w = 0; w < kTabThreads / 32; ++w)
    {
        if (w < warp)
            pa += wa[w], pb += wb[w];
        qa += wa[w], qb += wb[w];
    }
    a = pa + sa - a, b = pb + sb - b;
    *ta = qa, *tb = qb;
}

// The OR of every CTA's `err` (shared memory) over the cluster, and a barrier between the reads before
// and the writes after it. Every thread of the cluster has to have arrived at the cluster's barrier once
// before (cluster_started): a CTA's shared memory may be written by others from its start on only, and the
// wait here, which the sums have mostly hidden, is what says that all have started.
__device__ __forceinline__ void cluster_started()
{
    cooperative_groups::this_cluster().barrier_arrive();
}
__device__ uint32_t cluster_or(uint32_t *err)
{
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    __shared__ uint32_t all[kMaxCluster];
    __syncthreads(); // err is final in this CTA
    cl.barrier_wait();
    if (threadIdx.x < cl.num_blocks())
        *cl.map_shared_rank(&all[cl.block_rank()], threadIdx.x) = *err;
    cl.sync();
    uint32_t e = 0;
    for (uint32_t i = 0; i < cl.num_blocks(); ++i)
        e |= all[i];
    return e;
}

__global__ void __launch_bounds__(kTabThreads) k_paged_append(const AppendArgs a)
{
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t sm[];
    __shared__ uint32_t err;
    const uint32_t n = a.t.n_seqs, R = a.t.page_rows, tid = threadIdx.x;
    const uint32_t rank = cg::this_cluster().block_rank(), size = cg::this_cluster().num_blocks();
    cluster_started();
    uint32_t *starts = sm, *first = sm + n + 1, *len = first + n + 1; // [n + 1], [n + 1], [n]
    const uint32_t nf = *a.n_free;
    if (tid == 0)
        err = 0;
    __syncthreads();
    const uint32_t per = (n + kTabThreads - 1) / kTabThreads, s0 = min(tid * per, n), s1 = min(s0 + per, n);
    uint64_t tok = 0, pg = 0;
    uint32_t e = 0;
    for (uint32_t s = s0; s < s1; ++s)
    {
        const uint64_t l = a.lens[s], m = l + a.n_new[s];
        e |= length_status(a.t, m);
        len[s] = (uint32_t)l;
        tok += m - l;
        pg += pages_of(m, R) - pages_of(l, R);
    }
    uint64_t tokens, pages;
    block_sums(tok, pg, &tokens, &pages);
    if (nf > a.t.n_pages || pages > nf)
        e |= VKLLM_B200_PAGED_NO_PAGES;
    if (tokens > a.max_tokens)
        e |= VKLLM_B200_PAGED_TOO_MANY;
    if (e)
        atomicOr(&err, e);
    __syncthreads();
    bool ok = err == 0;
    if (ok)
    {
        for (uint32_t s = s0; s < s1; ++s)
        {
            const uint64_t l = len[s], m = l + a.n_new[s];
            starts[s] = (uint32_t)tok, first[s] = (uint32_t)pg;
            tok += m - l;
            pg += pages_of(m, R) - pages_of(l, R);
        }
        if (tid == 0)
            starts[n] = (uint32_t)tokens, first[n] = (uint32_t)pages;
        // the ids that the call would use: pages off the list and partly filled pages that get more rows
#pragma unroll 4
        for (uint32_t j = rank * kTabThreads + tid; j < pages; j += size * kTabThreads)
            e |= page_status(a.t.free_pages[nf - 1 - j], a.t.n_pages);
        __syncthreads();
        for (uint32_t s = rank * kTabThreads + tid; s < n; s += size * kTabThreads)
            if (starts[s + 1] != starts[s] && len[s] % R != 0)
                e |= page_status(a.t.table[s * a.t.stride + len[s] / R], a.t.n_pages);
        if (e)
            atomicOr(&err, e);
    }
    e = cluster_or(&err);
    if (e && rank == 0 && tid == 0)
        atomicOr(a.status, e);
    ok = e == 0;
    if (!ok) // as with nothing new
    {
        for (uint32_t s = tid; s <= n; s += kTabThreads)
            starts[s] = first[s] = 0;
        tokens = pages = 0;
        __syncthreads();
    }
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t g0 = rank * kTabThreads + tid, step = size * kTabThreads;
    if (g0 == 0)
    {
        *a.n_free_out = nf - (uint32_t)pages;
        a.starts[n] = (uint32_t)tokens;
    }
    for (uint32_t s = g0; s < n; s += step)
    {
        a.starts[s] = starts[s];
        a.new_lens[s] = len[s] + (starts[s + 1] - starts[s]);
    }
#pragma unroll 4
    for (uint32_t j = g0; j < pages; j += step)
    {
        const uint32_t page = a.t.free_pages[nf - 1 - j], s = last_at_most(first, n, j);
        a.t.table[s * a.t.stride + pages_of(len[s], R) + (j - first[s])] = page;
    }
    if (a.max_tokens > kTokensHere) // k_paged_slots
        return;
    for (uint32_t t = g0; t < a.max_tokens; t += step)
    {
        uint32_t slot = VKLLM_B200_NO_SLOT, pos = 0;
        if (t < tokens)
        {
            const uint32_t s = last_at_most(starts, n, t), held = pages_of(len[s], R);
            pos = len[s] + (t - starts[s]);
            const uint32_t c = pos / R;
            const uint32_t page = c < held ? a.t.table[s * a.t.stride + c] : a.t.free_pages[nf - 1 - (first[s] + (c - held))];
            slot = page * R + pos % R;
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
}

// Slots and positions of many tokens, from what k_paged_append left: runs of four per thread, which mostly
// share their sequence, its search and its page.
__global__ void __launch_bounds__(kSlotThreads) k_paged_slots(const AppendArgs a)
{
    extern __shared__ uint32_t starts[];
    const uint32_t n = a.t.n_seqs, R = a.t.page_rows;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint32_t s = threadIdx.x; s <= n; s += kSlotThreads)
        starts[s] = a.starts[s];
    __syncthreads();
    const uint32_t tokens = starts[n];
    const uint64_t t0 = ((uint64_t)blockIdx.x * kSlotThreads + threadIdx.x) * 4;
    if (t0 >= a.max_tokens)
        return;
    const uint32_t t = (uint32_t)t0;
    uint32_t slot[4], pos[4];
    uint32_t s = 0, p = 0, row = 0, c = 0, page = 0; // of the token: its sequence, position, row, column and page
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
    {
        slot[i] = VKLLM_B200_NO_SLOT, pos[i] = 0;
        if (t0 + i >= tokens)
            continue;
        bool fresh = i == 0 || t + i == starts[s + 1]; // another sequence, or another page
        if (fresh)
        {
            if (i == 0)
                s = last_at_most(starts, n, t);
            else
                do
                    ++s;
                while (t + i == starts[s + 1]);
            p = a.new_lens[s] - (starts[s + 1] - (t + i)); // tokens end at the sequence's new end
            c = p / R, row = p - c * R;
        }
        else
        {
            ++p, ++row;
            if (row == R)
                row = 0, ++c, fresh = true;
        }
        if (fresh)
            page = a.t.table[s * a.t.stride + c];
        slot[i] = page * R + row;
        pos[i] = p;
    }
    if (t0 + 4 <= a.max_tokens && (((uintptr_t)a.slots | (uintptr_t)a.positions) & 15) == 0)
    {
        *reinterpret_cast<uint4 *>(a.slots + t) = make_uint4(slot[0], slot[1], slot[2], slot[3]);
        *reinterpret_cast<uint4 *>(a.positions + t) = make_uint4(pos[0], pos[1], pos[2], pos[3]);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (t0 + i < a.max_tokens)
            a.slots[t + i] = slot[i], a.positions[t + i] = pos[i];
}

__global__ void __launch_bounds__(kTabThreads) k_paged_release(const ReleaseArgs a)
{
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t sm[];
    __shared__ uint32_t err;
    const uint32_t n = a.t.n_seqs, R = a.t.page_rows, tid = threadIdx.x;
    const uint32_t rank = cg::this_cluster().block_rank(), size = cg::this_cluster().num_blocks();
    cluster_started();
    uint32_t *first = sm, *len = sm + n + 1; // [n + 1], [n]
    const uint32_t nf = *a.n_free;
    if (tid == 0)
        err = 0;
    __syncthreads();
    const uint32_t per = (n + kTabThreads - 1) / kTabThreads, s0 = min(tid * per, n), s1 = min(s0 + per, n);
    uint64_t pg = 0, unused = 0;
    uint32_t e = 0;
    for (uint32_t s = s0; s < s1; ++s)
    {
        const uint32_t l = a.lens[s];
        len[s] = l;
        if (a.done[s])
        {
            e |= length_status(a.t, l);
            pg += pages_of(l, R);
        }
    }
    uint64_t pages, total;
    block_sums(pg, unused, &pages, &total);
    if ((uint64_t)nf + pages > a.t.n_pages)
        e |= VKLLM_B200_PAGED_TOO_MANY;
    if (e)
        atomicOr(&err, e);
    __syncthreads();
    if (err == 0)
    {
        for (uint32_t s = s0; s < s1; ++s)
        {
            first[s] = (uint32_t)pg;
            if (a.done[s])
                pg += pages_of(len[s], R);
        }
        if (tid == 0)
            first[n] = (uint32_t)pages;
        __syncthreads();
#pragma unroll 4
        for (uint32_t j = rank * kTabThreads + tid; j < pages; j += size * kTabThreads)
        {
            const uint32_t s = last_at_most(first, n, j);
            e |= page_status(a.t.table[s * a.t.stride + (j - first[s])], a.t.n_pages);
        }
        if (e)
            atomicOr(&err, e);
    }
    e = cluster_or(&err);
    if (e && rank == 0 && tid == 0)
        atomicOr(a.status, e);
    const bool ok = e == 0;
    if (!ok)
        pages = 0;
    const uint32_t g0 = rank * kTabThreads + tid, step = size * kTabThreads;
    if (g0 == 0)
        *a.n_free_out = nf + (uint32_t)pages;
    for (uint32_t s = g0; s < n; s += step)
        a.new_lens[s] = ok && a.done[s] ? 0 : len[s];
#pragma unroll 4
    for (uint32_t j = g0; j < pages; j += step)
    {
        const uint32_t s = last_at_most(first, n, j);
        a.t.free_pages[nf + j] = a.t.table[s * a.t.stride + (j - first[s])];
    }
}

template <typename Args>
vkllm_err_t launch_cluster(void (*kernel)(const Args), const Args &args, uint32_t ctas, size_t smem, int device,
                           cudaStream_t s)
{
    static std::atomic<bool> done[64]; // the attribute of this kernel, set once a device (twice does no harm)
    if (device >= 64 || !done[device].load(std::memory_order_relaxed))
    {
        VKB_CUDA(cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)((3 * (size_t)kMaxSeqs + 2) * 4)));
        if (device < 64)
            done[device].store(true, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kTabThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    VKB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    return VKLLM_ERR_OK;
}

// CTAs for `items` tokens, pages or sequences.
uint32_t cluster_for(uint64_t items)
{
    uint32_t c = 1;
    while (c < kMaxCluster && (uint64_t)c * kTabThreads * 2 < items)
        c *= 2;
    return c;
}

} // namespace
} // namespace vkb

extern "C" vkllm_err_t vkllm_b200_paged_append(const struct vkllm_b200_paged_table *t, const uint32_t *lens,
                                               const uint32_t *n_new, const uint32_t *n_free, uint32_t *new_lens,
                                               uint32_t *n_free_out, uint32_t *starts, uint32_t *slots,
                                               uint32_t *positions, uint32_t max_tokens, uint32_t *status, void *stream)
{
    using namespace vkb;
    _CHECK_ARGS(table_fits(t) && words(t->free_pages) && t->n_seqs <= kMaxSeqs);
    _CHECK_ARGS(words(lens) && words(n_new) && words(n_free) && words(new_lens) && words(n_free_out) && words(starts) &&
                words(status));
    _CHECK_ARGS(max_tokens == 0 || (words(slots) && words(positions)));
    int dev = 0;
    _CHECK(check_device({t->table, t->free_pages, lens, n_new, n_free, new_lens, n_free_out, starts,
                         max_tokens ? slots : nullptr, max_tokens ? positions : nullptr, status},
                        nullptr, &dev));
    const AppendArgs a{*t, lens, n_new, n_free, new_lens, n_free_out, starts, slots, positions, max_tokens, status};
    const uint32_t here = max_tokens <= kTokensHere ? max_tokens : 0, items = here > t->n_seqs ? here : t->n_seqs;
    cudaStream_t s = (cudaStream_t)stream;
    _CHECK(launch_cluster(k_paged_append, a, here == max_tokens ? cluster_for(items) : kMaxCluster,
                          (3 * (size_t)t->n_seqs + 2) * 4, dev, s));
    if (here == max_tokens)
        return VKLLM_ERR_OK;
    const uint32_t smem = (t->n_seqs + 1) * 4;
    if (smem > 48 * 1024)
        VKB_CUDA(cudaFuncSetAttribute((const void *)k_paged_slots, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)((kMaxSeqs + 1) * 4)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((uint64_t)max_tokens + 4 * kSlotThreads - 1) / (4 * kSlotThreads)));
    cfg.blockDim = dim3(kSlotThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; // its launch overlaps the first kernel
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    VKB_CUDA(cudaLaunchKernelEx(&cfg, k_paged_slots, a));
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_b200_paged_release(const struct vkllm_b200_paged_table *t, const uint32_t *lens,
                                                const uint32_t *done, const uint32_t *n_free, uint32_t *new_lens,
                                                uint32_t *n_free_out, uint32_t *status, void *stream)
{
    using namespace vkb;
    _CHECK_ARGS(table_fits(t) && words(t->free_pages) && t->n_seqs <= kMaxSeqs);
    _CHECK_ARGS(words(lens) && words(done) && words(n_free) && words(new_lens) && words(n_free_out) && words(status));
    int dev = 0;
    _CHECK(check_device({t->table, t->free_pages, lens, done, n_free, new_lens, n_free_out, status}, nullptr, &dev));
    const ReleaseArgs a{*t, lens, done, n_free, new_lens, n_free_out, status};
    return launch_cluster(k_paged_release, a, cluster_for((uint64_t)t->n_seqs * 16), // the pages are not known here
                           (2 * (size_t)t->n_seqs + 1) * 4, dev,
                          (cudaStream_t)stream);
}

extern "C" vkllm_err_t vkllm_b200_paged_check(const struct vkllm_b200_paged_table *t, const uint32_t *lens,
                                              uint32_t n_free, uint32_t *status, uint32_t *bad_seq)
{
    using namespace vkb;
    _CHECK_ARGS(table_fits(t) && words(lens) && (n_free == 0 || words(t->free_pages)));
    uint32_t e = 0, at = t->n_seqs;
    try
    {
        std::vector<bool> held(t->n_pages, false);
        auto take = [&](uint32_t page) {
            if (const uint32_t bad = page_status(page, t->n_pages))
                return bad;
            const bool twice = held[page];
            held[page] = true;
            return twice ? (uint32_t)VKLLM_B200_PAGED_BAD_PAGE : 0u;
        };
        for (uint32_t s = 0; s < t->n_seqs && !e; ++s)
        {
            at = s;
            e = length_status(*t, lens[s]);
            for (uint32_t c = 0; !e && c < pages_of(lens[s], t->page_rows); ++c)
                e = take(t->table[s * t->stride + c]);
        }
        if (!e)
        {
            at = t->n_seqs;
            if (n_free > t->n_pages)
                e = VKLLM_B200_PAGED_NO_PAGES;
            for (uint32_t j = 0; !e && j < n_free; ++j)
                e = take(t->free_pages[j]);
        }
    }
    catch (...)
    {
        return VKLLM_ERR_ALLOC;
    }
    if (status)
        *status = e;
    if (bad_seq)
        *bad_seq = at;
    return e ? VKLLM_ERR_ARGS : VKLLM_ERR_OK;
}
