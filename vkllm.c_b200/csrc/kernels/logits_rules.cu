// Rules on logits before the token choice: penalties for tokens of the history, biases, grammar masks.
//
//   x = id in the history ? (x > 0 ? x / r : x * r) : x
//   x = x - frequency * (times generated) - (generated ? presence : 0)
//   x = x + the id's biases;  x = mask bit ? x : -infinity
//
// Every logit is read and written once: HBM bounds a large batch, latency a single row. A block takes a
// piece of the vocabulary of one row, counts the row's history ids that fall into it in shared memory
// (integer atomics: the order of the additions does not matter) and adds up its biases there, then
// passes over its logits once. The history (a few KB, in L2) is read once per piece; no table of
// counts is kept in memory or between calls.
#include "paged.cuh"
#include "../runtime/internal.h"

namespace vkb
{
namespace
{

constexpr uint32_t kRuleThreads = 256;
constexpr uint32_t kPiece = 4096; // ids per block: 16 KB of counts and 16 KB of biases
constexpr uint32_t kSeen = 0x80000000u; // in the history at all; the bits below count the times generated

struct RuleArgs
{
    vkllm_b200_logit_rules r;
    const void *x;
    void *y;
    uint64_t x_stride, y_stride;
    uint32_t vocab;
};

template <typename T> __global__ void __launch_bounds__(kRuleThreads) k_logits_rules(const RuleArgs a)
{
    __shared__ uint32_t count[kPiece];
    __shared__ float bias[kPiece];
    const uint32_t row = blockIdx.y, v0 = blockIdx.x * kPiece, n = min(kPiece, a.vocab - v0), tid = threadIdx.x;
    for (uint32_t i = tid; i < n; i += kRuleThreads)
        count[i] = 0, bias[i] = 0.f;
    __syncthreads();
    if (a.r.history)
    {
        const uint32_t have = (uint32_t)min((uint64_t)a.r.history_lens[row], a.r.history_stride);
        const uint32_t prompt = a.r.prompt_lens ? a.r.prompt_lens[row] : 0;
        const uint32_t *h = a.r.history + row * a.r.history_stride;
        for (uint32_t i = tid; i < have; i += kRuleThreads)
        {
            const uint32_t id = h[i] - v0;
            if (id >= n)
                continue;
            if (i >= prompt)
                atomicAdd(&count[id], 1u);
            atomicOr(&count[id], kSeen);
        }
    }
    if (a.r.bias_starts && tid < 32)
    {
        // one warp, 32 entries at a time: lanes with the same id add one after another, as listed
        const uint32_t b0 = a.r.bias_starts[row], b1 = a.r.bias_starts[row + 1];
        for (uint32_t b = b0; b < b1; b += 32)
        {
            const bool in = b + tid < b1;
            const uint32_t id = in ? a.r.bias_ids[b + tid] - v0 : 0xffffffffu;
            const float value = in ? a.r.bias_values[b + tid] : 0.f;
            const uint32_t peers = __match_any_sync(0xffffffffu, id);
            const uint32_t turn = __popc(peers & ((1u << tid) - 1)), turns = __reduce_max_sync(0xffffffffu, turn);
            for (uint32_t k = 0; k <= turns; ++k)
            {
                if (turn == k && id < n)
                    bias[id] += value;
                __syncwarp();
            }
        }
    }
    __syncthreads();
    const float rep = a.r.repetition ? a.r.repetition[row] : 1.f, freq = a.r.frequency ? a.r.frequency[row] : 0.f,
                pres = a.r.presence ? a.r.presence[row] : 0.f;
    const T *x = (const T *)a.x + row * a.x_stride + v0;
    T *y = (T *)a.y + row * a.y_stride + v0;
    const uint32_t *mask = a.r.mask ? a.r.mask + row * a.r.mask_stride : nullptr;
    for (uint32_t i = tid; i < n; i += kRuleThreads)
    {
        float v = to_f32<T>(x[i]);
        const uint32_t c = count[i];
        if (c)
        {
            v = v > 0.f ? v / rep : v * rep;
            if (c != kSeen)
                v = v - freq * (float)(c & ~kSeen) - pres;
        }
        v += bias[i];
        if (mask && !((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u))
            v = __int_as_float(0xff800000);
        y[i] = from_f32<T>(v);
    }
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
    _CHECK_ARGS(rows > 0 && rows <= 65535 && vocab > 0 && vocab <= 0x7fffffffu);
    _CHECK_ARGS(logits && aligned_to(logits, es) && logits_stride >= vocab && logits_stride < (1ull << 40));
    _CHECK_ARGS(out && aligned_to(out, es) && out_stride >= vocab && out_stride < (1ull << 40));
    _CHECK_ARGS(logits != out || logits_stride == out_stride);
    _CHECK_ARGS(!rules->history || (words(rules->history) && words(rules->history_lens)));
    _CHECK_ARGS(rules->history || (!rules->repetition && !rules->frequency && !rules->presence));
    _CHECK_ARGS(aligned_to(rules->prompt_lens, 4) && aligned_to(rules->repetition, 4) && aligned_to(rules->frequency, 4) &&
                aligned_to(rules->presence, 4));
    _CHECK_ARGS(!rules->bias_starts || (words(rules->bias_starts) && words(rules->bias_ids) && words(rules->bias_values)));
    _CHECK_ARGS(!rules->mask || (words(rules->mask) && rules->mask_stride >= ((uint64_t)vocab + 31) / 32));
    _CHECK_ARGS(rules->history_stride < (1ull << 40) && rules->mask_stride < (1ull << 40));
    _CHECK(check_device(logits, nullptr, nullptr));
    const RuleArgs a{*rules, logits, out, logits_stride, out_stride, vocab};
    const dim3 grid((vocab + kPiece - 1) / kPiece, rows);
    if (dtype == vkllm_dtype_float16)
        k_logits_rules<__half><<<grid, kRuleThreads, 0, (cudaStream_t)stream>>>(a);
    else
        k_logits_rules<float><<<grid, kRuleThreads, 0, (cudaStream_t)stream>>>(a);
    VKB_CUDA(cudaGetLastError());
    return VKLLM_ERR_OK;
}
