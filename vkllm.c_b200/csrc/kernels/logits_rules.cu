// Rules on logits before the token choice: penalties for tokens of the history, biases, grammar masks.
//
//   x = id in the history ? (x > 0 ? x / r : x * r) : x
//   x = x - frequency * (times generated) - (generated ? presence : 0)
//   x = x + the id's biases;  x = mask bit ? x : -infinity
//
// Every logit is read and written once (HBM bounds a large batch, latency a few rows), but the penalties
// and biases touch at most as many ids as the history and the lists are long. So there are two steps:
//   k_logits_copy   streams the rows through, with the mask: out = mask bit ? x : -infinity. In place it writes masked
//                   logits only, and without a mask it is not launched.
//   k_logits_touch  one block per row: the touched ids with their counts and bias sums in a hash table in
//                   shared memory, then x read, ruled, rounded once and written at those ids.
// The second is the first one's programmatic dependent: it builds its tables while the first streams and
// waits for it only before it touches the rows. The first's grid is resident at once for that reason. Few
// rows take one kernel, k_logits_touch<T, true>, whose blocks do both steps for a piece of a row. Counts
// are integer atomics, and biases are added by one warp in the order of the list: the result does not
// depend on the order of arrival. 256 rows of 100003 fp16 logits with 1024 to 2048 ids of history, all
// rules (107 MB): 30.9 us, of which the first kernel alone takes 23 and a plain copy of as much 19. What is
// left is the second one's scattered reads and writes, 1000 ids a row. (All in one kernel of pieces: 62.9
// us with counts in arrays over the piece, 44 with hash tables.)
#include <atomic>
#include <cmath>

#include "paged.cuh"
#include "../runtime/internal.h"

namespace vkb
{
namespace
{

// 16-byte vectors that a thread has in flight, and CTAs per SM: 40 KB of loads, and registers left for two
// blocks of the other kernel. (256 rows of 100003 fp16 logits, all rules: 30.9 us; with 6 CTAs, which leave
// it fewer registers, 31.1 to 34.4, with 4 31.7; 4 vectors x 4 CTAs 33.8; two items in flight a thread 34.1.)
constexpr uint32_t kCopyThreads = 256, kCopyVecs = 2, kCopyCtas = 5;
constexpr uint32_t kTouchThreads = 512; // of a row, or half as many where rows share an SM (see launch)
// Slots of the hash table, 16 bytes each; it takes lists of up to 3/4 as many ids (with repeats), longer ones
// go over ranges of the vocabulary instead. The small table lets more rows share an SM.
constexpr uint32_t kSlotsSmall = 4096, kSlotsLarge = 8192, kLeastSlots = 512;
constexpr uint32_t kNoId = 0xffffffffu; // not an id: vocab < 2^31
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u; // in the prompt; in the biases; the bits below: times generated
// Ids of a history are fewer: an id's count stays below kBiased, and places in a history do not wrap in 32 bits
// where a thread looks a few thousand ahead.
constexpr uint64_t kMostHistory = kBiased;

struct RuleArgs
{
    vkllm_b200_logit_rules r;
    const void *x;
    void *y;
    uint64_t x_stride, y_stride;
    uint32_t vocab, rows;
    uint32_t slots; // of the hash table, a power of two
    uint32_t chunk, chunks; // places of a chunk and chunks of a row (the first kernel's)
};

template <typename T> union Vec // 16 bytes of logits
{
    uint4 raw;
    T e[16 / sizeof(T)];
};

// 4 bits as 4 bytes of 0x00 or 0xff.
__device__ __forceinline__ uint32_t bytes_of(uint32_t bits)
{
    return ((bits & 15u) * 0x00204081u & 0x01010101u) * 0xffu;
}

// The elements whose bit is set, -infinity for the others.
template <typename T> __device__ __forceinline__ uint4 masked(uint4 v, uint32_t bits);
template <> __device__ __forceinline__ uint4 masked<__half>(uint4 v, uint32_t bits)
{
    const uint32_t inf = 0xfc00fc00u, lo = bytes_of(bits), hi = bytes_of(bits >> 4);
    const uint32_t m0 = __byte_perm(lo, 0, 0x1100), m1 = __byte_perm(lo, 0, 0x3322), m2 = __byte_perm(hi, 0, 0x1100),
                   m3 = __byte_perm(hi, 0, 0x3322);
    return make_uint4((v.x & m0) | (inf & ~m0), (v.y & m1) | (inf & ~m1), (v.z & m2) | (inf & ~m2), (v.w & m3) | (inf & ~m3));
}
template <> __device__ __forceinline__ uint4 masked<float>(uint4 v, uint32_t bits)
{
    const uint32_t inf = 0xff800000u;
    return make_uint4(bits & 1 ? v.x : inf, bits & 2 ? v.y : inf, bits & 4 ? v.z : inf, bits & 8 ? v.w : inf);
}

// One thread's vectors of a chunk of a row. A row is cut at the 128-byte boundaries of the input, into
// chunks of equal size: place e of a row is id e - lead, where `lead` elements lie between the boundary at
// or before the row's start and the row. (Chunks that began at any 16-byte boundary, where warps meet in
// the middle of lines, copied 51 MB in 24.3 us instead of 21.8.)
template <typename T> struct CopyItem
{
    static constexpr uint32_t E = 16 / sizeof(T), kAll = (1u << E) - 1;
    const T *x;
    T *y;
    const uint32_t *mask;
    uint32_t lead, end, stop, e0;
    uint4 v[kCopyVecs];
    uint32_t allowed[kCopyVecs];

    __device__ __forceinline__ void load(const RuleArgs &a, uint32_t row, uint32_t chunk)
    {
        x = (const T *)a.x + row * a.x_stride;
        y = (T *)a.y + row * a.y_stride;
        mask = a.r.mask ? a.r.mask + row * a.r.mask_stride : nullptr;
        lead = (uint32_t)((uintptr_t)x & 127) / sizeof(T);
        end = a.vocab + lead;
        stop = min(end, (chunk + 1) * a.chunk);
        e0 = chunk * a.chunk + threadIdx.x * E;
#pragma unroll
        for (uint32_t k = 0; k < kCopyVecs; ++k)
        {
            const uint32_t e = e0 + k * kCopyThreads * E;
            allowed[k] = kAll;
            if (e < lead || e >= stop || e + E > end)
                continue;
            const uint32_t id = e - lead;
            v[k] = *reinterpret_cast<const uint4 *>(x + id);
            if (mask)
            {
                const uint32_t w = id >> 5, last = (id + E - 1) >> 5;
                const uint32_t lo = __ldg(mask + w), hi = last != w ? __ldg(mask + last) : 0u;
                allowed[k] &= __funnelshift_r(lo, hi, id & 31);
            }
        }
    }

    __device__ __forceinline__ void store() const
    {
        const bool together = (((uintptr_t)x ^ (uintptr_t)y) & 15) == 0; // the output's 16-byte boundaries are the input's
#pragma unroll
        for (uint32_t k = 0; k < kCopyVecs; ++k)
        {
            const uint32_t e = e0 + k * kCopyThreads * E;
            if (e >= stop || e + E <= lead)
                continue;
            if (e >= lead && e + E <= end)
            {
                if (x == y && allowed[k] == kAll)
                    continue;
                Vec<T> o;
                o.raw = mask ? masked<T>(v[k], allowed[k]) : v[k];
                if (together)
                    *reinterpret_cast<uint4 *>(y + (e - lead)) = o.raw;
                else
#pragma unroll
                    for (uint32_t i = 0; i < E; ++i)
                        y[e - lead + i] = o.e[i];
                continue;
            }
            for (uint32_t i = 0; i < E; ++i) // the row begins or ends inside these 16 bytes
            {
                if (e + i < lead || e + i >= end)
                    continue;
                const uint32_t id = e + i - lead;
                y[id] = !mask || ((mask[id >> 5] >> (id & 31)) & 1u) ? x[id] : from_f32<T>(-INFINITY);
            }
        }
    }
};

template <typename T> __global__ void __launch_bounds__(kCopyThreads) k_logits_copy(const RuleArgs a)
{
    asm volatile("griddepcontrol.launch_dependents;");
    uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const uint32_t rows = gridDim.x / a.chunks, chunks = gridDim.x % a.chunks;
    while (row < a.rows)
    {
        CopyItem<T> item;
        item.load(a, row, chunk);
        item.store();
        row += rows, chunk += chunks;
        if (chunk >= a.chunks)
            chunk -= a.chunks, ++row;
    }
}

// The touched ids: of a row (one block each), or with PIECE of one chunk of a row, which the block streams
// through itself before.
template <typename T, bool PIECE> __global__ void __launch_bounds__(PIECE ? kCopyThreads : kTouchThreads, PIECE ? 4 : 3) k_logits_touch(const RuleArgs a)
{
    extern __shared__ __align__(16) uint32_t sm[];
    uint32_t *key = sm, *count = sm + a.slots;
    float *bias = reinterpret_cast<float *>(sm + 2 * a.slots);
    uint32_t *list = sm + 3 * a.slots;
    __shared__ uint32_t listed;
    const uint32_t row = PIECE ? blockIdx.y : blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const uint32_t threads = blockDim.x, historians = threads - 32; // the last warp sums the biases
    const uint32_t have = a.r.history ? (uint32_t)min((uint64_t)a.r.history_lens[row], a.r.history_stride) : 0;
    const uint32_t prompt = a.r.history && a.r.prompt_lens ? a.r.prompt_lens[row] : 0;
    const uint32_t *h = a.r.history + row * a.r.history_stride;
    const uint32_t b0 = a.r.bias_starts ? a.r.bias_starts[row] : 0, b1 = a.r.bias_starts ? a.r.bias_starts[row + 1] : 0;
    const uint32_t biases = b1 > b0 ? b1 - b0 : 0;
    const float rep = a.r.repetition ? a.r.repetition[row] : 1.f, freq = a.r.frequency ? a.r.frequency[row] : 0.f,
                pres = a.r.presence ? a.r.presence[row] : 0.f;
    uint32_t id0 = 0, id1 = a.vocab; // the block's ids
    if constexpr (PIECE)
    {
        CopyItem<T> item;
        item.load(a, row, blockIdx.x);
        if (a.x != a.y || a.r.mask)
            item.store();
        id0 = blockIdx.x * a.chunk > item.lead ? blockIdx.x * a.chunk - item.lead : 0;
        id1 = item.stop > item.lead ? item.stop - item.lead : 0;
    }
    // Few enough entries: hashed, in a table of four times their number where that is smaller than all. Else
    // ranges of ids one after the other, each id at its place.
    const uint64_t entries = (uint64_t)have + biases;
    const bool hashed = entries <= a.slots / 4 * 3;
    uint32_t slots = a.slots;
    if (hashed)
        while (slots > kLeastSlots && slots / 2 >= 4 * entries)
            slots /= 2;
    bool waited = PIECE;
    for (uint32_t base = id0, width; base < id1; base += width)
    {
        width = hashed ? id1 - base : min(slots, id1 - base); // ids of this round: base .. base + width - 1
        for (uint32_t i = 4 * tid; i < slots; i += 4 * threads)
        {
            *reinterpret_cast<uint4 *>(key + i) = make_uint4(kNoId, kNoId, kNoId, kNoId);
            *reinterpret_cast<uint4 *>(count + i) = *reinterpret_cast<uint4 *>(bias + i) = make_uint4(0, 0, 0, 0);
        }
        if (tid == 0)
            listed = 0;
        __syncthreads();
        // the slot of an id, or kNoId where it has none
        auto place = [&](uint32_t id) {
            if (id - base >= width)
                return kNoId;
            if (!hashed)
                return id - base;
            uint32_t s = (id * 0x9E3779B1u) >> 8 & (slots - 1);
            for (;; s = (s + 1) & (slots - 1)) // ends: the table has more slots than ids
            {
                uint32_t k = *(volatile uint32_t *)&key[s]; // mostly there already: common ids come often
                if (k == kNoId)
                    k = atomicCAS(&key[s], kNoId, id);
                if (k == kNoId || k == id)
                    return s;
            }
        };
        auto enlist = [&](uint32_t s, bool fresh) { // one count per warp: all lanes together
            const uint32_t who = __ballot_sync(0xffffffffu, fresh);
            uint32_t at = 0;
            if (who && lane == 0)
                at = atomicAdd(&listed, (uint32_t)__popc(who));
            at = __shfl_sync(0xffffffffu, at, 0);
            if (fresh)
                list[at + __popc(who & ((1u << lane) - 1))] = s;
        };
        if (tid < historians)
        {
            for (uint32_t i0 = tid - lane; i0 < have; i0 += 4 * historians) // (the whole warp together)
            {
                uint32_t id[4];
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u)
                    id[u] = i0 + lane + u * historians < have ? h[i0 + lane + u * historians] : kNoId;
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u)
                {
                    const uint32_t s = place(id[u]);
                    bool fresh = false; // the first to touch it
                    if (s != kNoId)
                        fresh = (i0 + lane + u * historians < prompt ? atomicOr(&count[s], kSeen) : atomicAdd(&count[s], 1u)) == 0;
                    enlist(s, fresh);
                }
            }
        }
        else
            // the last warp, 32 entries at a time: lanes with the same id add one after another, as listed
            for (uint32_t b = 0; b < biases; b += 32)
            {
                const bool in = biases - b > lane;
                const uint32_t id = in ? a.r.bias_ids[b0 + b + lane] : kNoId;
                const float value = in ? a.r.bias_values[b0 + b + lane] : 0.f;
                const uint32_t s = place(id), peers = __match_any_sync(0xffffffffu, s);
                const uint32_t turn = __popc(peers & ((1u << lane) - 1));
                const uint32_t turns = __reduce_max_sync(0xffffffffu, s == kNoId ? 0u : turn);
                enlist(s, s != kNoId && turn == 0 && atomicOr(&count[s], kBiased) == 0);
                for (uint32_t k = 0; k <= turns; ++k)
                {
                    if (turn == k && s != kNoId)
                        bias[s] += value;
                    __syncwarp();
                }
                if (biases - b <= 32)
                    break;
            }
        __syncthreads();
        // ids that the mask forbids leave the list
        const uint32_t *mask = a.r.mask ? a.r.mask + row * a.r.mask_stride : nullptr;
        const uint32_t n = listed;
        if (mask)
            for (uint32_t i0 = tid; i0 < n; i0 += 4 * threads)
            {
                uint32_t word[4];
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u)
                    if (i0 + u * threads < n)
                    {
                        const uint32_t s = list[i0 + u * threads];
                        word[u] = __ldg(mask + ((hashed ? key[s] : base + s) >> 5));
                    }
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u)
                    if (i0 + u * threads < n)
                    {
                        const uint32_t s = list[i0 + u * threads];
                        if (!((word[u] >> ((hashed ? key[s] : base + s) & 31)) & 1u))
                            list[i0 + u * threads] = kNoId;
                    }
            }
        if (!waited) // the rows are the first kernel's until it is done
            asm volatile("griddepcontrol.wait;" ::: "memory");
        waited = true;
        // A row's logits are read back from the output, where the first kernel just put them: they are in
        // L2, while the input's lines would be fetched from memory once more. A piece's are still there
        // from its own loads (in place as well: what the mask allows is as it was).
        T *y = (T *)a.y + row * a.y_stride;
        const T *in = PIECE ? (const T *)a.x + row * a.x_stride : y;
        for (uint32_t i0 = tid; i0 < n; i0 += 4 * threads)
        {
            uint32_t id[4], s[4];
            T x[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u)
            {
                s[u] = i0 + u * threads < n ? list[i0 + u * threads] : kNoId;
                if (s[u] != kNoId)
                {
                    id[u] = hashed ? key[s[u]] : base + s[u];
                    x[u] = in[id[u]];
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u)
                if (s[u] != kNoId)
                {
                    const uint32_t c = count[s[u]];
                    float v = to_f32<T>(x[u]);
                    if (c != kBiased)
                    {
                        v = v > 0.f ? v / rep : v * rep;
                        const uint32_t times = c & ~(kSeen | kBiased);
                        if (times)
                            v = v - freq * (float)times - pres;
                    }
                    y[id[u]] = from_f32<T>(v + bias[s[u]]);
                }
        }
        __syncthreads();
    }
}

template <typename T> vkllm_err_t launch_rules(RuleArgs &a, int sms, int device, cudaStream_t s)
{
    // 16-byte vectors of a row at the worst lead, cut into equal chunks of whole 128-byte lines
    const uint32_t vecs = (a.vocab + 128 / sizeof(T) - 1 + 16 / sizeof(T) - 1) / (16 / sizeof(T));
    a.chunks = (vecs + kCopyThreads * kCopyVecs - 1) / (kCopyThreads * kCopyVecs);
    a.chunk = ((vecs + a.chunks - 1) / a.chunks + 7) / 8 * 8 * (16 / sizeof(T));
    const bool copy = a.x != a.y || a.r.mask, touch = a.r.history || a.r.bias_starts;
    static std::atomic<bool> done[64]; // the kernels' attributes, set once a device (twice does no harm)
    if (device >= 64 || !done[device].load(std::memory_order_relaxed))
    {
        VKB_CUDA(cudaFuncSetAttribute((const void *)k_logits_touch<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)(kSlotsLarge * 16)));
        VKB_CUDA(cudaFuncSetAttribute((const void *)k_logits_touch<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)(kSlotsLarge * 16)));
        // an SM changes its split of L1 and shared memory only when it is idle: with the same split for both,
        // the second kernel's blocks can join the first one's
        VKB_CUDA(cudaFuncSetAttribute((const void *)k_logits_touch<T, false>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                      cudaSharedmemCarveoutMaxShared));
        VKB_CUDA(cudaFuncSetAttribute((const void *)k_logits_copy<T>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                      cudaSharedmemCarveoutMaxShared));
        if (device < 64)
            done[device].store(true, std::memory_order_relaxed);
    }
    // One kernel while its blocks run at once: each reads the whole history, but nothing waits for a second
    // kernel. Of 32000 fp16 logits with up to 768 ids of history, 4 / 32 / 64 / 128 rows take 4.8 / 5.4 / 9.0 /
    // 13.3 us in one kernel and 6.4 / 7.0 / 7.2 / 8.2 in two; 16 / 32 rows of 100003 with up to 2048 ids 8.1 /
    // 13.2 and 10.1 / 10.2; 16 rows of 32000 fp32 ones with up to 5000 ids, where the large table leaves an SM
    // one block, 19.3 and 16.3.
    if (copy && touch && (uint64_t)a.rows * a.chunks <= (a.slots == kSlotsSmall ? 3 : 1) * (uint64_t)sms)
        return launch_plain(k_logits_touch<T, true>, a, dim3(a.chunks, a.rows), kCopyThreads, a.slots * 16, s);
    if (copy)
    {
        const uint64_t items = (uint64_t)a.rows * a.chunks, most = (uint64_t)sms * kCopyCtas;
        _CHECK(launch_plain(k_logits_copy<T>, a, dim3((unsigned)(items < most ? items : most)), kCopyThreads, 0, s));
    }
    if (!touch)
        return VKLLM_ERR_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows);
    cfg.blockDim = dim3(a.rows <= (uint32_t)sms ? kTouchThreads : kTouchThreads / 2);
    cfg.dynamicSmemBytes = a.slots * 16;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = copy ? 1 : 0; // alone it follows whatever is in the stream
    VKB_CUDA(cudaLaunchKernelEx(&cfg, k_logits_touch<T, false>, a));
    return VKLLM_ERR_OK;
}

} // namespace
} // namespace vkb

extern "C" vkllm_err_t vkllm_b200_logits_apply(const struct vkllm_b200_logit_rules *rules, const void *logits,
                                               uint64_t logits_stride, uint32_t rows, uint32_t vocab, uint32_t dtype,
                                               void *out, uint64_t out_stride, void *stream)
{
    using namespace vkb;
    const uint32_t es = paged_elem_bytes(dtype);
    _CHECK_ARGS(rules && es != 0);
    _CHECK_ARGS(rows > 0 && rows <= 65535 && vocab > 0 && vocab <= 0x7fff0000u);
    _CHECK_ARGS(logits && aligned_to(logits, es) && logits_stride >= vocab && logits_stride < (1ull << 40));
    _CHECK_ARGS(out && aligned_to(out, es) && out_stride >= vocab && out_stride < (1ull << 40));
    _CHECK_ARGS(logits != out || logits_stride == out_stride);
    _CHECK_ARGS(!rules->history || (words(rules->history) && words(rules->history_lens)));
    _CHECK_ARGS(rules->history || (!rules->repetition && !rules->frequency && !rules->presence));
    _CHECK_ARGS(aligned_to(rules->prompt_lens, 4) && aligned_to(rules->repetition, 4) && aligned_to(rules->frequency, 4) &&
                aligned_to(rules->presence, 4));
    _CHECK_ARGS(!rules->bias_starts || (words(rules->bias_starts) && words(rules->bias_ids) && words(rules->bias_values)));
    _CHECK_ARGS(!rules->mask || (words(rules->mask) && rules->mask_stride >= ((uint64_t)vocab + 31) / 32));
    _CHECK_ARGS((!rules->history || rules->history_stride < kMostHistory) && rules->mask_stride < (1ull << 40));
    int sms = 0, dev = 0;
    const vkllm_b200_logit_rules &r = *rules;
    _CHECK(check_device({logits, out, r.history, r.history ? r.prompt_lens : nullptr, r.history ? r.history_lens : nullptr, r.repetition,
                         r.frequency, r.presence, r.bias_starts, r.bias_starts ? r.bias_ids : nullptr,
                         r.bias_starts ? r.bias_values : nullptr, r.mask},
                        &sms, &dev));
    // the longest history that fits the small table with 512 biases
    const uint32_t slots = !rules->history || rules->history_stride <= kSlotsSmall / 4 * 3 - 512 ? kSlotsSmall : kSlotsLarge;
    RuleArgs a{*rules, logits, out, logits_stride, out_stride, vocab, rows, slots, 0, 0};
    return dtype == vkllm_dtype_float16 ? launch_rules<__half>(a, sms, dev, (cudaStream_t)stream)
                                        : launch_rules<float>(a, sms, dev, (cudaStream_t)stream);
}
