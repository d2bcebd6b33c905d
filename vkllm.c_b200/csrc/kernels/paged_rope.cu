// RoPE of new tokens with their key and value rows written into a paged cache.
//
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * base^(-2w / hd),  pairs (2w, 2w + 1)
//
// on q (to q_out) and k (to the slot's key row); v is copied to the slot's value row. The pairs are those
// of VKLLM_OP_ROPE. Every element is read and written once, so a long call is bound by HBM and a short one
// by latency.
//
// Angles: fp32 loses the angle of far positions (at position 200000 the rounding of position * frequency
// alone is 8e-3 radians). The frequency is kept as a fraction of a turn in 64-bit fixed point, f =
// base^(-2w / hd) / (2 pi) < 2^-2, so position * f modulo 2^64 is the exact fraction of the last turn for
// the rounded f: an error of at most position * 2^-64 turns, and no range reduction. Rounded to fp32 as a
// number of half turns it is off by up to 2^-25 of one, which moves a sine by up to 9.4e-8, at near positions
// as at far ones. With fp32 rows that shows (5.5e-8 of the outputs' size from 64 bits, where a sine of a 64-bit
// angle gives 4.2e-8), with fp16 rows it does not.
//
// A block works out a token's sines and cosines once, into shared memory; each thread owns one 16-byte
// piece of a head (4 or 2 pairs), keeps those of its pairs, and walks over its share of the token's heads,
// kAhead loads in flight, the first of them on their way before the position and the sines are known. 2048
// tokens of 40 + 80 heads of 128 (126 MB, fp16): 21.6 us, 5.8 TB/s (24.6 with the loads after the sines, 27.5
// with sines worked out by every thread), where a plain copy of 102 MB reaches 5.5.
//
// The loads wait for the slot: a step that is launched for the most tokens it may have is mostly padding, whose
// rows are not read. 64 tokens among 8192, 32 + 16 heads of 128: 5.5 us; 20.6 where the loads go out first, which
// gives 64 tokens without padding 2.65 us instead of 2.80, 2048 of 32 + 16 heads 10.2 instead of 10.5 and longer
// calls nothing.
#include <cmath>

#include "paged.cuh"
#include "../runtime/internal.h"

namespace vkb
{
namespace
{

constexpr uint32_t kRopeThreads = 256;

struct RopeArgs
{
    vkllm_b200_paged_kv kv;
    const void *q, *k, *v;
    void *q_out;
    uint64_t q_stride, k_stride, v_stride, q_out_stride; // elements
    const uint32_t *positions, *slots;
    uint32_t n_tokens, heads;
    uint32_t *status;
    uint64_t turns[128]; // base^(-2w / hd) / (2 pi) * 2^64
};

// 16 bytes as fp32 pairs. kAhead: rows of a thread in flight; kCtas: blocks of an SM that the registers are kept
// to. fp16, 2048 tokens of 40 + 80 heads, three sets of rows into one pool: 20.4 us with 4 x 6 blocks, 21.5 with
// 4 x 5, 21.8 with 3 x 8, 23.1 with 4 x 8 (registers spill); fp32, 1500 tokens of 32 + 16 heads: 12.5 with 3 x 8,
// 13.4 with 4 x 6.
template <typename T> struct Piece;
template <> struct Piece<__half>
{
    static constexpr int kPairs = 4;
    static constexpr uint32_t kAhead = 4, kCtas = 6;
    __device__ static void load(const uint4 &r, float2 (&p)[4])
    {
        const __half2 *h = reinterpret_cast<const __half2 *>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            p[i] = __half22float2(h[i]);
    }
    __device__ static uint4 store(const float2 (&p)[4])
    {
        uint4 r;
        __half2 *h = reinterpret_cast<__half2 *>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            h[i] = __floats2half2_rn(p[i].x, p[i].y);
        return r;
    }
};
template <> struct Piece<float>
{
    static constexpr int kPairs = 2;
    static constexpr uint32_t kAhead = 3, kCtas = 8;
    __device__ static void load(const uint4 &r, float2 (&p)[2])
    {
        p[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
        p[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
    }
    __device__ static uint4 store(const float2 (&p)[2])
    {
        return make_uint4(__float_as_uint(p[0].x), __float_as_uint(p[0].y), __float_as_uint(p[1].x),
                          __float_as_uint(p[1].y));
    }
};

// Block: a multiple of the pieces of a head; grid.x: tokens, grid.y: shares of the token's rows (q heads,
// then key heads, then value heads).
template <typename T>
__global__ void __launch_bounds__(kRopeThreads, Piece<T>::kCtas) k_paged_rope_write(const RopeArgs a)
{
    constexpr int P = Piece<T>::kPairs, E = 2 * P;
    constexpr uint32_t kAhead = Piece<T>::kAhead;
    __shared__ __align__(16) float2 table[128]; // (cos, sin) of every pair of a head at the token's position
    const uint32_t t = blockIdx.x, slot = a.slots[t];
    const uint32_t hd = a.kv.head_dim, pieces = hd / E, piece = threadIdx.x % pieces, lanes = blockDim.x / pieces;
    const uint32_t H = a.heads, K = a.kv.kv_heads, rows = H + 2 * K, off = piece * E;
    const uint32_t step = gridDim.y * lanes;
    uint32_t r0 = blockIdx.y * lanes + threadIdx.x / pieces;
    uint4 x[kAhead];
    auto load = [&] {
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
        {
            const uint32_t r = r0 + u * step;
            if (r >= rows)
                break;
            const T *src = r < H       ? (const T *)a.q + t * a.q_stride + (uint64_t)r * hd
                           : r < H + K ? (const T *)a.k + t * a.k_stride + (uint64_t)(r - H) * hd
                                       : (const T *)a.v + t * a.v_stride + (uint64_t)(r - H - K) * hd;
            x[u] = *reinterpret_cast<const uint4 *>(src + off);
        }
    };
    if (slot == VKLLM_B200_NO_SLOT)
        return;
    load();
    const uint32_t position = a.positions[t]; // (read with the slot, it would be waited for with it)
    const uint32_t page = slot / a.kv.page_rows, row = slot % a.kv.page_rows;
    if (page >= a.kv.n_pages)
    {
        if (threadIdx.x == 0 && blockIdx.y == 0)
            atomicOr(a.status, (uint32_t)VKLLM_B200_PAGED_BAD_SLOT);
        return;
    }
    for (uint32_t w = threadIdx.x; w < hd / 2; w += blockDim.x)
    {
        // half turns in [-1, 1)
        const float half_turns = __ll2float_rn((long long)(position * a.turns[w])) * 0x1p-63f;
        float s, c;
        sincospif(half_turns, &s, &c);
        table[w] = make_float2(c, s);
    }
    __syncthreads();
    float cs[P], sn[P];
#pragma unroll
    for (int i = 0; i < P; ++i)
        cs[i] = table[piece * P + i].x, sn[i] = table[piece * P + i].y;
    const uint64_t cache = page * a.kv.page_stride + row * a.kv.row_stride + off;
    while (r0 < rows)
    {
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
        {
            const uint32_t r = r0 + u * step;
            if (r >= rows)
                break;
            if (r < H + K)
            {
                float2 p[P];
                Piece<T>::load(x[u], p);
#pragma unroll
                for (int i = 0; i < P; ++i)
                    p[i] = make_float2(cs[i] * p[i].x - sn[i] * p[i].y, sn[i] * p[i].x + cs[i] * p[i].y);
                x[u] = Piece<T>::store(p);
            }
            T *dst = r < H       ? (T *)a.q_out + t * a.q_out_stride + (uint64_t)r * hd + off
                     : r < H + K ? (T *)a.kv.k + cache + (r - H) * a.kv.head_stride
                                 : (T *)a.kv.v + cache + (r - H - K) * a.kv.head_stride;
            *reinterpret_cast<uint4 *>(dst) = x[u];
        }
        r0 += kAhead * step;
        load();
    }
}

} // namespace
} // namespace vkb

extern "C" vkllm_err_t vkllm_b200_paged_rope_write(const struct vkllm_b200_paged_kv *kv, const void *q,
                                                   uint64_t q_stride, const void *k, uint64_t k_stride, const void *v,
                                                   uint64_t v_stride, const uint32_t *positions, const uint32_t *slots,
                                                   uint32_t n_tokens, uint32_t heads, float rope_base, void *q_out,
                                                   uint64_t q_out_stride, uint32_t *status, void *stream)
{
    using namespace vkb;
    _CHECK_ARGS(kv_fits(kv));
    _CHECK_ARGS(heads > 0 && heads <= 65535 && heads % kv->kv_heads == 0);
    const uint32_t es = paged_elem_bytes(kv->dtype), hd = kv->head_dim;
    _CHECK_ARGS(rope_base <= 0.f || (rope_base > 1.f && std::isfinite(rope_base)));
    if (n_tokens == 0)
        return VKLLM_ERR_OK;
    _CHECK_ARGS(n_tokens <= 0x7fffffffu);
    _CHECK_ARGS(rows_fit(q, q_stride, (uint64_t)heads * hd, es) && rows_fit(q_out, q_out_stride, (uint64_t)heads * hd, es));
    _CHECK_ARGS(rows_fit(k, k_stride, (uint64_t)kv->kv_heads * hd, es) &&
                rows_fit(v, v_stride, (uint64_t)kv->kv_heads * hd, es));
    _CHECK_ARGS(q != q_out || q_stride == q_out_stride);
    _CHECK_ARGS(words(positions) && words(slots) && words(status));
    int sms = 0;
    _CHECK(check_device({kv->k, kv->v, q, k, v, positions, slots, q_out, status}, &sms, nullptr));
    RopeArgs a;
    a.kv = *kv;
    a.q = q, a.k = k, a.v = v, a.q_out = q_out;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride, a.q_out_stride = q_out_stride;
    a.positions = positions, a.slots = slots, a.n_tokens = n_tokens, a.heads = heads, a.status = status;
    // one power, then products: each costs half a unit in the 64th bit, 2^-57 of a frequency at the last
    const long double base = rope_base <= 0.f ? 10000.0L : (long double)rope_base;
    const long double ratio = powl(base, -2.0L / hd);
    long double f = 0x1p64L / (2.0L * 3.14159265358979323846264338327950288L);
    for (uint32_t w = 0; w < hd / 2; ++w, f *= ratio)
        a.turns[w] = (uint64_t)f;
    const uint32_t pieces = hd * es / 16, threads = kRopeThreads / pieces * pieces, lanes = threads / pieces;
    // Blocks of a token: so many that a thread has one batch of rows in flight (2048 tokens of 120 heads: 2
    // blocks a token 24.6 us, one 25.9, when that was measured), and of few tokens more, until the call
    // reaches about two blocks an SM.
    const uint32_t ahead = es == 2 ? Piece<__half>::kAhead : Piece<float>::kAhead;
    const uint32_t passes = (heads + 2 * kv->kv_heads + lanes - 1) / lanes;
    uint32_t shares = (passes + ahead - 1) / ahead;
    while (shares < passes && (uint64_t)n_tokens * shares < 2u * (uint32_t)sms)
        ++shares;
    const dim3 grid(n_tokens, shares);
    return launch_plain(kv->dtype == vkllm_dtype_float16 ? k_paged_rope_write<__half> : k_paged_rope_write<float>, a, grid,
                        threads, 0, (cudaStream_t)stream);
}
