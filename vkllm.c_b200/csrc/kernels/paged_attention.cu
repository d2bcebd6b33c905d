// Attention of one query row per row of a page table (a sequence, or a token of one) over a paged KV cache.
//
//   out = sum_j exp(scale q . k_j - m) v_j / sum_j exp(scale q . k_j - m),  j < len,  m = max_j scale q . k_j
//
// Every cached row is read once for all the query heads that share its key head: 2 to 32 flops a byte, so
// HBM bounds the call, and what matters is that every SM keeps enough loads in flight from the first
// microsecond to the last.
//
// Work. Lengths are known on the device only, so the kernel divides the work itself. An item is one
// (sequence, key head, tile of up to 8 or 16 of its queries); its keys are cut into tiles of 4 slices, one
// slice per warp (16 keys in fp16, 8 in fp32). All tiles of all items form one line, in which an item's end
// counts too, and every CTA of a grid that fills the GPU takes an equal part of it: a long sequence spreads
// over all SMs and short ones share a CTA. A CTA that holds only a part of an item leaves (m, l, O) in the
// workspace and counts itself at the item; the last one to arrive joins the parts in the order of the line,
// so the result does not depend on who was last. (Handing the last quarter of the line out in small chunks
// off a ticket counter was slower: 98 us for 64 sequences of 128 to 640 keys, where equal parts took 78 then and
// take 67 now, since every chunk refills the rings.)
//
// Loads. Each warp streams its own slices through a private ring of cp.async stages, also across the
// borders of items: no barrier of the CTA stands between a load and its use. Page ids are read one tile
// ahead of the rows that they lead to. Rows past the end, and rows of bad pages, are filled with zeros
// without being read and masked out of the scores.
//
// fp16: S^T = K Q^T on the tensor cores (mma.sync m16n8k16: 16 keys x 8 queries), so that the 8 columns
// take up to 8 queries that share the keys and each lane keeps the statistics of two of them; then O^T +=
// V^T P with P^T moved into operand order by movmatrix. The weights are kept as the sum of two fp16 parts,
// scaled by 2^15: one part alone would double the error of the rounded output, and unscaled ones would lose
// their bits below fp16's range where one key outweighs very many small ones (the tensor cores have the
// time: they idle behind the loads). fp32: plain FMAs; 4 lanes share a key's dot product, and every lane
// owns head_dim / 32 of the output.
#include <atomic>
#include <type_traits>

#include "paged.cuh"
#include "../runtime/internal.h"

namespace vkb
{
namespace
{

constexpr uint32_t kWarps = 4, kThreads = kWarps * 32;
constexpr uint32_t kCounters = 1024;      // words at the start of the workspace, one per CTA of the grid
// Lengths on the line: a tile, and what an item costs beside its tiles (its queries read, its warps joined).
constexpr uint32_t kTileUnits = 4, kItemUnits = 6;
constexpr uint32_t kMinUnits = 2 * kTileUnits + kItemUnits; // least part of a CTA: an item of two tiles
constexpr uint32_t kNoPage = 0xffffffffu;
constexpr float kWeightShift = 15.f;      // weights are at most 2^15, below fp16's 65504

struct PagedAttArgs
{
    vkllm_b200_paged_kv kv;
    const uint32_t *table;
    uint64_t table_stride;
    uint32_t n_seqs;
    uint32_t cap; // most rows of a sequence (cols * page_rows)
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;
    uint64_t page_bytes, head_bytes, row_bytes; // strides of the pools
    uint64_t page_magic; // ceil(2^64 / page_rows), to divide a key's number by page_rows; 0: page_rows is 1
    const uint32_t *lens;
    uint32_t group;  // queries that share a key head
    uint32_t qtiles; // tiles of these queries
    uint32_t gq;     // queries of a tile (the last tile may have fewer)
    float scale_log2; // scale * log2(e): the softmax runs in powers of two
    uint32_t *status;
    uint32_t *counters;
    float *parts; // [2 * grid] parts of items: [gq][KD] O, then [gq] m, [gq] l
    uint32_t part_stride;
};

// Shared memory for a head size. KD: dimensions that are computed, head_dim rounded up. Rows must not meet in the same banks
// where 8 of them are read at once: a power of two of 16-byte pieces is swizzled, other rows get a piece more.
template <typename T, int KD> struct Shape
{
    static constexpr bool kPow2 = (KD & (KD - 1)) == 0;
    static constexpr uint32_t kKeys = sizeof(T) == 2 ? 16 : 8;                  // keys of a slice
    static constexpr uint32_t kRow = KD * sizeof(T) + (kPow2 ? 0 : 16);         // bytes of a row
    static constexpr uint32_t kStage = 2 * kKeys * kRow;                        // K and V of a slice
    static constexpr uint32_t kQBytes = sizeof(T) == 4 ? 8 * KD * 4 : 0;        // the queries (fp32 only)
    // Stages of a warp's ring, CTAs of an SM and queries that a join buffer takes. Small heads need more warps for
    // the same bytes: 8 x 16 heads of 64 with 4096 keys take 31.7 us with 3 CTAs of 4 stages, 35.9 with 2 of 6; 28
    // heads of 80 over 4 take 72 with 3 of 2 and 80 with 2 of 3. Of 128, 3 CTAs of 2 stages (kRound 2) are better
    // where items are short (200 sequences of up to 120 keys: 48 instead of 57 us) and worse where they are long or
    // 16 queries share a head (65 instead of 59), so it stays at 2 of 3. With 3 CTAs a thread has 168 registers, which
    // costs most kernels of up to 96 dimensions 8 to 60 bytes of spills; the times above include them.
    static constexpr uint32_t kStages = KD <= 64 ? (sizeof(T) == 4 ? 3 : 4) : sizeof(T) == 4 || KD == 96 ? 2 : 3;
    static constexpr uint32_t kCtas = KD > 128 ? 1 : KD <= 96 ? 3 : 2;
    static constexpr uint32_t kRound = 4;
    static constexpr uint32_t kPitch = KD + 4;                                  // floats of a row of a join buffer
    static constexpr uint32_t kRing = kWarps * kStages * kStage;
    static constexpr uint32_t kJoin = kWarps * kRound * (kPitch + 2); // floats of a join buffer: O, then m and l
    static constexpr uint32_t kSmem = kRing + kQBytes + 2 * kJoin * 4 + kWarps * kStages * 4;
    static_assert(kSmem <= 227 * 1024 && kCtas * (kSmem + 1200) <= 228 * 1024, "shared memory of an SM");

    // Byte of 16-byte piece p of row r.
    static __device__ __forceinline__ uint32_t at(uint32_t r, uint32_t p)
    {
        return r * kRow + (kPow2 ? p ^ (r & 7) : p) * 16;
    }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes, uint64_t policy)
{
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
                 "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void cp_commit()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N> __device__ __forceinline__ void cp_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Two fp32 FMAs in one instruction: c + a * b, element by element.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(d)
        : "l"(*reinterpret_cast<const uint64_t *>(&a)), "l"(*reinterpret_cast<const uint64_t *>(&b)),
          "l"(*reinterpret_cast<const uint64_t *>(&c)));
    return *reinterpret_cast<const float2 *>(&d);
}
__device__ __forceinline__ float pow2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t v)
{
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
// exp2's base for a maximum: any finite number does where no key counts yet.
__device__ __forceinline__ float finite_base(float m)
{
    return m == -INFINITY ? 0.f : m;
}

__host__ __device__ __forceinline__ uint32_t item_units(uint32_t tiles)
{
    return tiles ? tiles * kTileUnits + kItemUnits : 0;
}

// a / b; places on the line mostly fit 32 bits, whose division takes a tenth of the time.
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b)
{
    return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b;
}

// A place in the line of tiles: tile `tile` of `tiles` of item (seq, hq), hq = key head * qtiles + query
// tile, `unit` units behind the start of the CTA's part.
struct Cursor
{
    uint32_t seq, hq, tile, tiles, len, unit;

    __device__ __forceinline__ void set_len(const PagedAttArgs &a, uint32_t tile_keys)
    {
        len = min(a.lens[seq], a.cap);
        tiles = (len + tile_keys - 1) / tile_keys;
    }
    // One tile on; behind the last one seq is n_seqs.
    __device__ __forceinline__ void next(const PagedAttArgs &a, uint32_t items, uint32_t tile_keys)
    {
        unit += kTileUnits;
        if (++tile >= tiles)
            next_item(a, items, tile_keys);
    }
    // From behind the last tile to the first of the next item.
    __device__ __forceinline__ void next_item(const PagedAttArgs &a, uint32_t items, uint32_t tile_keys)
    {
        unit += kItemUnits;
        tile = 0;
        if (++hq < items)
            return;
        hq = 0;
        do
            ++seq;
        while (seq < a.n_seqs && (set_len(a, tile_keys), tiles == 0));
    }
};

// The stream of one warp's slices: page ids one tile ahead, rows kStages - 1 tiles ahead. A warp issues a
// few hundred instructions for a tile, with no other warp to hide their latency behind in a short call, so
// what can be worked out before is.
template <typename T, int KD, bool EXACT> struct Loader
{
    using S = Shape<T, KD>;
    static constexpr uint32_t kPieces = KD * sizeof(T) / 16;
    // a lane copies the same piece of every row that it copies
    static constexpr bool kFixed = EXACT && S::kPow2 && kPieces <= 32;
    Cursor c;
    uint32_t end;       // units of the CTA's part
    uint32_t page, row; // of key `lane % kKeys` of the slice at c, and its row in the page
    uint64_t head;      // bytes from a page's start to the item's key head
    uint32_t ring;      // shared address of the warp's ring
    uint32_t *valid;    // [kStages] masks of the slice's keys that count
    uint32_t stage = 0, status = 0;
    uint32_t pieces, row0, p0, drow, dp; // the copies of a lane: pieces of a row, its first one, from one to the next
    const char *k, *v;                   // the pools (at the lane's piece where that is fixed)
    // rows are read once: they leave L2 first, and what others have there stays (one sequence of 131072 92.4 -> 91.1 us,
    // 64 of 128 to 640 74.3 -> 72.5, when that was measured)
    uint64_t policy;

    __device__ __forceinline__ void begin(const PagedAttArgs &a, uint32_t warp, uint32_t lane)
    {
        pieces = EXACT ? kPieces : a.kv.head_dim * (uint32_t)sizeof(T) / 16;
        row0 = lane / pieces, p0 = lane % pieces;
        drow = 32 / pieces, dp = 32 % pieces;
        k = (const char *)a.kv.k + (kFixed ? p0 * 16 : 0), v = (const char *)a.kv.v + (kFixed ? p0 * 16 : 0);
        asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        lookup(a, warp, lane);
        new_item(a, lane);
    }
    __device__ __forceinline__ bool more(const PagedAttArgs &a) const
    {
        return c.unit < end && c.seq < a.n_seqs;
    }
    __device__ __forceinline__ void lookup(const PagedAttArgs &a, uint32_t warp, uint32_t lane)
    {
        const uint32_t key = (c.tile * kWarps + warp) * S::kKeys + lane % S::kKeys;
        const uint32_t col = a.page_magic ? (uint32_t)__umul64hi(key, a.page_magic) : key;
        row = key - col * a.kv.page_rows;
        page = kNoPage; // behind the end
        if (more(a) && key < c.len)
        {
            page = __ldg(a.table + c.seq * a.table_stride + col);
            if (page == kNoPage) // an id past every pool, however many pages that has
                status |= VKLLM_B200_PAGED_BAD_PAGE;
        }
    }
    // At an item's first tile: where its keys lie, and its queries, which will be wanted, on their way to L1.
    __device__ __forceinline__ void new_item(const PagedAttArgs &a, uint32_t lane)
    {
        uint32_t kh = c.hq, qt = 0;
        if (a.qtiles > 1)
            kh = c.hq / a.qtiles, qt = c.hq - kh * a.qtiles;
        head = kh * a.head_bytes;
        const uint32_t nq = min(a.gq, a.group - qt * a.gq);
        const char *q = (const char *)((const T *)a.q + c.seq * a.q_stride + (uint64_t)(kh * a.group + qt * a.gq) * a.kv.head_dim);
        for (uint32_t b = lane * 128; more(a) && b < nq * a.kv.head_dim * (uint32_t)sizeof(T); b += 32 * 128)
            asm volatile("prefetch.global.L1 [%0];" ::"l"(q + b));
    }
    // Issues the slice at c as one group of copies (an empty one behind the end) and moves on.
    __device__ __forceinline__ void issue(const PagedAttArgs &a, uint32_t items, uint32_t warp, uint32_t lane)
    {
        if (more(a))
        {
            const bool ok = page < a.kv.n_pages;
            if (!ok && page != kNoPage)
                status |= VKLLM_B200_PAGED_BAD_PAGE;
            const uint64_t at = ok ? page * a.page_bytes + head + row * a.row_bytes : 0;
            const uint32_t mask = __ballot_sync(0xffffffffu, ok) & ((1u << S::kKeys) - 1);
            if (lane == 0)
                valid[stage] = mask;
            if (mask)
            {
                const uint32_t base = ring + stage * S::kStage;
                constexpr uint32_t kMost = S::kKeys * kPieces / 32; // (a whole number for every KD)
                if constexpr (kFixed)
                {
                    // row r = row0 + i * drow with row0 < drow, both powers of two: the swizzle splits in two
                    constexpr uint32_t kRows = 32 / kPieces;
                    const uint32_t lane_dst = base + row0 * S::kRow + (p0 ^ row0) * 16;
#pragma unroll
                    for (uint32_t i = 0; i < kMost; ++i)
                    {
                        const uint32_t r = row0 + i * kRows;
                        const uint64_t off = __shfl_sync(0xffffffffu, at, r);
                        const uint32_t bytes = (mask >> r) & 1u ? 16u : 0u;
                        const uint32_t dst = (lane_dst ^ ((i * kRows & 7) * 16)) + i * kRows * S::kRow;
                        cp_async16(dst, k + off, bytes, policy);
                        cp_async16(dst + S::kKeys * S::kRow, v + off, bytes, policy);
                    }
                }
                else
                {
                    uint32_t r0 = row0, p = p0;
#pragma unroll
                    for (uint32_t i = 0; i < kMost; ++i)
                    {
                        if (!EXACT && i * 32 >= S::kKeys * pieces)
                            break;
                        const uint32_t r = r0 % S::kKeys; // r0 < kKeys for every copy that is made
                        const uint64_t off = __shfl_sync(0xffffffffu, at, r) + p * 16;
                        const uint32_t bytes = (mask >> r) & 1u ? 16u : 0u;
                        if (EXACT || r0 < S::kKeys)
                        {
                            const uint32_t dst = base + S::at(r, p);
                            cp_async16(dst, k + off, bytes, policy);
                            cp_async16(dst + S::kKeys * S::kRow, v + off, bytes, policy);
                        }
                        r0 += drow, p += dp;
                        if (p >= pieces)
                            p -= pieces, ++r0;
                    }
                }
            }
            c.next(a, items, kWarps * S::kKeys);
            lookup(a, warp, lane);
            if (c.tile == 0)
                new_item(a, lane);
        }
        cp_commit();
        stage = stage + 1 == S::kStages ? 0 : stage + 1;
    }
};

// What a warp keeps of an item: statistics and outputs of its keys, for 8 NQ queries.
template <int KD, int NQ, bool EXACT> struct HalfCore
{
    using T = __half;
    using S = Shape<T, KD>;
    static constexpr int kQueries = 8 * NQ;
    static constexpr int kK = KD / 16;
    uint32_t qf[NQ][kK][2]; // Q^T as the B operand
    float o[NQ][kK][4], m[NQ][2], l[NQ][2];

    __device__ __forceinline__ void start(const PagedAttArgs &a, uint32_t seq, uint32_t head0, uint32_t nq, uint32_t lane,
                                          float *)
    {
        const uint32_t hd = a.kv.head_dim;
#pragma unroll
        for (int n = 0; n < NQ; ++n)
        {
            const uint32_t qi = n * 8 + (lane >> 2);
            const T *row = (const T *)a.q + seq * a.q_stride + (uint64_t)(head0 + qi) * hd;
#pragma unroll
            for (int k = 0; k < kK; ++k)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                {
                    const uint32_t d = k * 16 + b * 8 + (lane & 3) * 2;
                    qf[n][k][b] = qi < nq && (EXACT || d < hd) ? __ldg(reinterpret_cast<const uint32_t *>(row + d)) : 0u;
                }
#pragma unroll
            for (int k = 0; k < kK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[n][k][i] = 0.f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
    }

    __device__ __forceinline__ void slice(const PagedAttArgs &a, uint32_t base, uint32_t mask, uint32_t lane,
                                          const float *)
    {
        float s[NQ][2][4]; // two chains of products
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[n][0][i] = s[n][1][i] = 0.f;
        const uint32_t kr = lane & 15;
#pragma unroll
        for (int k = 0; k < kK; ++k)
        {
            uint32_t f[4];
            ldsm4(f, base + S::at(kr, 2 * k + (lane >> 4)));
#pragma unroll
            for (int n = 0; n < NQ; ++n)
                mma16816(s[n][k & 1], f, qf[n][k][0], qf[n][k][1]);
        }
        const bool in0 = (mask >> (lane >> 2)) & 1u, in1 = (mask >> ((lane >> 2) + 8)) & 1u;
        uint32_t hi[NQ][2], lo[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
        {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = (i < 2 ? in0 : in1) ? (s[n][0][i] + s[n][1][i]) * a.scale_log2 : -INFINITY;
            float f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
            {
                float mx = fmaxf(x[i], x[i + 2]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                mx = fmaxf(mx, m[n][i]);
                const float b = finite_base(mx);
                f[i] = pow2(m[n][i] - b);
                m[n][i] = mx;
                x[i] = pow2(x[i] - b + kWeightShift);
                x[i + 2] = pow2(x[i + 2] - b + kWeightShift);
                l[n][i] = fmaf(l[n][i], f[i], x[i] + x[i + 2]);
            }
            if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f))
#pragma unroll
                for (int k = 0; k < kK; ++k)
                {
                    o[n][k][0] *= f[0], o[n][k][1] *= f[1];
                    o[n][k][2] *= f[0], o[n][k][3] *= f[1];
                }
#pragma unroll
            for (int b = 0; b < 2; ++b)
            {
                const uint32_t h = pack2(x[2 * b], x[2 * b + 1]);
                const float2 hf = unpack2(h);
                hi[n][b] = transpose8x8(h);
                lo[n][b] = transpose8x8(pack2(x[2 * b] - hf.x, x[2 * b + 1] - hf.y));
            }
        }
        const uint32_t vr = (lane & 7) + ((lane >> 4) & 1) * 8, vbase = base + S::kKeys * S::kRow;
#pragma unroll
        for (int k = 0; k < kK; ++k)
        {
            uint32_t f[4];
            ldsm4_t(f, vbase + S::at(vr, 2 * k + ((lane >> 3) & 1)));
#pragma unroll
            for (int n = 0; n < NQ; ++n)
            {
                mma16816(o[n][k], f, hi[n][0], hi[n][1]);
                mma16816(o[n][k], f, lo[n][0], lo[n][1]);
            }
        }
    }

    // Queries kRound r .. of the item, those below nq, into the warp's join buffer: os [kRound][kPitch], ml [kRound][2].
    __device__ __forceinline__ void deposit(int r, uint32_t nq, float *os, float *ml, uint32_t lane)
    {
        constexpr uint32_t kPairs = S::kRound / 2, kPer = 8 / S::kRound; // pairs of queries of a round; rounds of 8
#pragma unroll
        for (int n = 0; n < NQ; ++n)
            if (n == r / (int)kPer)
            {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                {
                    float t = l[n][i];
                    t += __shfl_xor_sync(0xffffffffu, t, 4);
                    t += __shfl_xor_sync(0xffffffffu, t, 8);
                    t += __shfl_xor_sync(0xffffffffu, t, 16);
                    // this lane's query is 8 n + 2 pair + i
                    const uint32_t pair = lane & 3, q = pair % kPairs * 2 + i;
                    if (pair / kPairs != r % kPer || r * S::kRound + q >= nq)
                        continue;
                    if (lane < 4)
                        ml[q * 2] = m[n][i], ml[q * 2 + 1] = t;
#pragma unroll
                    for (int k = 0; k < kK; ++k)
                    {
                        os[q * S::kPitch + k * 16 + (lane >> 2)] = o[n][k][i];
                        os[q * S::kPitch + k * 16 + (lane >> 2) + 8] = o[n][k][i + 2];
                    }
                }
            }
    }
};

// fp32: 8 keys of a slice; lane = (part << 3) | key computes a quarter of that key's dot products (the
// 16-byte pieces p with p % 4 == part); for the outputs a lane owns the pieces lane % kP, lane % kP + 32 ...
template <int KD, int NQ, bool EXACT> struct FloatCore
{
    using T = float;
    using S = Shape<T, KD>;
    static constexpr int kQueries = NQ;
    static constexpr int kP = KD / 4;                       // pieces of a row
    static constexpr int kRowP = S::kRow / 16;              // and from row to row
    static constexpr int kOwn = (kP + 31) / 32;             // pieces that a lane owns
    static constexpr int kHalves = kP == 16 ? 2 : 1;      // lane groups that share the keys (KD = 64: 2)
    float4 o[NQ][kOwn];
    float m[NQ], l[NQ];

    __device__ __forceinline__ void start(const PagedAttArgs &a, uint32_t seq, uint32_t head0, uint32_t nq, uint32_t lane,
                                          float *qs)
    {
        // the CTA's warps are at the same item here: each loads every fourth query, 16 bytes a lane, all in flight
        // (element by element 118 sequences of up to 13 keys, 64 heads of 128 over 32, took 36.7 us instead of 27.4)
        const uint32_t hd = a.kv.head_dim, warp = threadIdx.x >> 5;
        const T *q = (const T *)a.q + seq * a.q_stride + (uint64_t)head0 * hd;
#pragma unroll
        for (uint32_t j = 0; j < (NQ + kWarps - 1) / kWarps; ++j)
#pragma unroll
            for (uint32_t k = 0; k < kOwn; ++k)
            {
                const uint32_t i = warp + kWarps * j, d = 4 * (lane + 32 * k);
                if (i < NQ && d < KD)
                    reinterpret_cast<float4 *>(qs)[(i * KD + d) / 4] =
                        i < nq && (EXACT || d < hd) ? __ldg(reinterpret_cast<const float4 *>(q + i * hd + d))
                                                    : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NQ; ++i)
        {
#pragma unroll
            for (int k = 0; k < kOwn; ++k)
                o[i][k] = make_float4(0.f, 0.f, 0.f, 0.f);
            m[i] = -INFINITY, l[i] = 0.f;
        }
    }

    __device__ __forceinline__ void slice(const PagedAttArgs &a, uint32_t base, uint32_t mask, uint32_t lane,
                                          const float *qs)
    {
        extern __shared__ __align__(128) unsigned char sm[];
        const uint32_t off = base - (uint32_t)__cvta_generic_to_shared(sm);
        const float4 *K = reinterpret_cast<const float4 *>(sm + off);
        const float4 *V = K + S::kKeys * kRowP;
        const uint32_t key = lane & 7, part = lane >> 3;
        // every query's dot product in two chains (even and odd elements), all queries side by side
        float2 d[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            d[i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < KD / 16; ++j)
        {
            const float4 k = K[S::at(key, 4 * j + part) / 16];
#pragma unroll
            for (int i = 0; i < NQ; ++i)
            {
                const float4 q = reinterpret_cast<const float4 *>(qs + i * KD)[4 * j + part];
                d[i] = fma2(make_float2(q.x, q.y), make_float2(k.x, k.y), d[i]);
                d[i] = fma2(make_float2(q.z, q.w), make_float2(k.z, k.w), d[i]);
            }
        }
        const bool in = (mask >> key) & 1u;
        float p[NQ], mx[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            p[i] = d[i].x + d[i].y;
#pragma unroll
        for (int x = 8; x < 32; x <<= 1)
#pragma unroll
            for (int i = 0; i < NQ; ++i)
                p[i] += __shfl_xor_sync(0xffffffffu, p[i], x);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            mx[i] = p[i] = in ? p[i] * a.scale_log2 : -INFINITY;
#pragma unroll
        for (int x = 1; x < 8; x <<= 1)
#pragma unroll
            for (int i = 0; i < NQ; ++i)
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], x));
        bool moved = false;
        float f[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i)
        {
            const float mn = fmaxf(mx[i], m[i]), b = finite_base(mn);
            f[i] = pow2(m[i] - b);
            moved |= f[i] != 1.f;
            m[i] = mn;
            p[i] = pow2(p[i] - b);
            l[i] = fmaf(l[i], f[i], p[i]);
        }
        if (__any_sync(0xffffffffu, moved))
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int k = 0; k < kOwn; ++k)
                    o[i][k].x *= f[i], o[i][k].y *= f[i], o[i][k].z *= f[i], o[i][k].w *= f[i];
        const uint32_t first = kHalves > 1 ? lane / kP : 0;
#pragma unroll
        for (uint32_t j = 0; j < S::kKeys / kHalves; ++j)
        {
            const uint32_t r = j * kHalves + first;
            float4 v[kOwn];
#pragma unroll
            for (int k = 0; k < kOwn; ++k)
                v[k] = V[S::at(r, (lane + 32 * k) % kP) / 16]; // (a lane without a piece takes another's)
#pragma unroll
            for (int i = 0; i < NQ; ++i)
            {
                const float w = __shfl_sync(0xffffffffu, p[i], r);
#pragma unroll
                for (int k = 0; k < kOwn; ++k)
                {
                    const float2 lo = fma2(make_float2(w, w), make_float2(v[k].x, v[k].y), make_float2(o[i][k].x, o[i][k].y));
                    const float2 hi = fma2(make_float2(w, w), make_float2(v[k].z, v[k].w), make_float2(o[i][k].z, o[i][k].w));
                    o[i][k] = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
            }
        }
    }

    __device__ __forceinline__ void deposit(int r, uint32_t nq, float *os, float *ml, uint32_t lane)
    {
#pragma unroll
        for (int i = 0; i < NQ; ++i)
        {
            if (i / (int)S::kRound != r || i >= nq)
                continue;
            const uint32_t q = i % S::kRound;
            float t = l[i];
            t += __shfl_xor_sync(0xffffffffu, t, 1);
            t += __shfl_xor_sync(0xffffffffu, t, 2);
            t += __shfl_xor_sync(0xffffffffu, t, 4);
            if (lane == 0)
                ml[q * 2] = m[i], ml[q * 2 + 1] = t;
#pragma unroll
            for (int k = 0; k < kOwn; ++k)
            {
                float4 v = o[i][k];
                if (kHalves > 1)
                {
                    v.x += __shfl_xor_sync(0xffffffffu, v.x, 16), v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
                    v.z += __shfl_xor_sync(0xffffffffu, v.z, 16), v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
                }
                if (lane + 32 * k < kP)
                    *reinterpret_cast<float4 *>(os + q * S::kPitch + 4 * (lane + 32 * k)) = v;
            }
        }
    }
};

template <typename T>
__device__ __forceinline__ void store_out(const PagedAttArgs &a, uint32_t seq, uint32_t head, uint32_t d, float4 o, float l)
{
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *dst = (T *)a.out + seq * a.out_stride + (uint64_t)head * a.kv.head_dim + d;
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
    else
        *reinterpret_cast<float4 *>(dst) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

__device__ __forceinline__ void add_scaled(float4 &o, float f, const float4 &v)
{
    o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
}

// A join buffer, joined over the warps: queries q0 .. q0 + n - 1 of the item (at most S::kRound), to the
// output or to a part.
template <typename T, int KD>
__device__ __forceinline__ void join_warps(const PagedAttArgs &a, const float *os, const float *ml, uint32_t n,
                                           uint32_t q0, uint32_t seq, uint32_t head0, float *part)
{
    using S = Shape<T, KD>;
    for (uint32_t i = threadIdx.x; i < n * (KD / 4); i += kThreads)
    {
        const uint32_t q = i / (KD / 4), d = i % (KD / 4) * 4;
        float mx = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w)
            mx = fmaxf(mx, ml[(w * S::kRound + q) * 2]);
        const float b = finite_base(mx);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w)
        {
            const float f = pow2(ml[(w * S::kRound + q) * 2] - b);
            l = fmaf(f, ml[(w * S::kRound + q) * 2 + 1], l);
            add_scaled(o, f, *reinterpret_cast<const float4 *>(os + (w * S::kRound + q) * S::kPitch + d));
        }
        if (part)
        {
            *reinterpret_cast<float4 *>(part + (q0 + q) * KD + d) = o;
            if (d == 0)
                part[a.gq * KD + q0 + q] = mx, part[a.gq * (KD + 1) + q0 + q] = l;
        }
        else if (d < a.kv.head_dim)
            store_out<T>(a, seq, head0 + q0 + q, d, o, l);
    }
}

// The part of CTA c of an item that begins in CTA c0: a CTA's second place is for the item that begins in
// it and goes on.
__device__ __forceinline__ float *part_of(const PagedAttArgs &a, uint32_t c, bool begins)
{
    return a.parts + (2 * (uint64_t)c + begins) * a.part_stride;
}

// An item joined over its parts in CTAs c0 .. c1, in their order, to the output. What it costs is the
// latency of its loads, at the end of a CTA's work: so every thread takes 4 elements of a query with the
// statistics of their parts on its own, 16 parts in flight, and where the item has too few elements to fill
// the CTA, and parts enough, groups of threads take every `groups`-th part and meet in shared memory.
template <typename T, int KD>
__device__ __noinline__ void join_parts(const PagedAttArgs &a, uint32_t c0, uint32_t c1, float *sm, uint32_t nq,
                                        uint32_t seq, uint32_t head0)
{
    constexpr uint32_t kCols = KD / 4, kAhead = 16;
    const uint32_t cols = nq * kCols, np = c1 - c0 + 1;
    const uint32_t groups = np > kAhead && cols < kThreads ? kThreads / cols : 1;
    const uint32_t group = groups > 1 ? threadIdx.x / cols : 0;
    for (uint32_t c = threadIdx.x - group * cols; c < cols && group < groups; c += groups > 1 ? cols : kThreads)
    {
        const uint32_t q = c / kCols, d = c % kCols * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float mx = -INFINITY, l = 0.f;
        for (uint32_t p0 = c0 + group; p0 <= c1; p0 += groups * kAhead)
        {
            float m[kAhead], pl[kAhead], top = mx;
            float4 v[kAhead];
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u)
            {
                const uint32_t p = p0 + u * groups;
                m[u] = -INFINITY, pl[u] = 0.f, v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p > c1)
                    continue;
                const float *src = part_of(a, p, p == c0);
                m[u] = __ldcg(src + a.gq * KD + q), pl[u] = __ldcg(src + a.gq * (KD + 1) + q);
                v[u] = __ldcg(reinterpret_cast<const float4 *>(src + q * KD + d));
            }
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u)
                top = fmaxf(top, m[u]);
            const float b = finite_base(top), f = pow2(mx - b);
            mx = top;
            l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u)
            {
                const float g = pow2(m[u] - b);
                l = fmaf(g, pl[u], l);
                add_scaled(o, g, v[u]);
            }
        }
        if (groups > 1)
        {
            float *row = sm + (group * cols + c) * 8;
            *reinterpret_cast<float4 *>(row) = o;
            row[4] = mx, row[5] = l;
        }
        else if (d < a.kv.head_dim)
            store_out<T>(a, seq, head0 + q, d, o, l);
    }
    if (groups == 1)
        return;
    __syncthreads();
    if (threadIdx.x < cols)
    {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float mx = -INFINITY, l = 0.f;
        for (uint32_t g = 0; g < groups; ++g)
            mx = fmaxf(mx, sm[(g * cols + threadIdx.x) * 8 + 4]);
        const float b = finite_base(mx);
        for (uint32_t g = 0; g < groups; ++g)
        {
            const float *row = sm + (g * cols + threadIdx.x) * 8;
            const float f = pow2(row[4] - b);
            l = fmaf(f, row[5], l);
            add_scaled(o, f, *reinterpret_cast<const float4 *>(row));
        }
        if (threadIdx.x % kCols * 4 < a.kv.head_dim)
            store_out<T>(a, seq, head0 + threadIdx.x / kCols, threadIdx.x % kCols * 4, o, l);
    }
    __syncthreads();
}

template <template <int, int, bool> class Kind, typename T, int KD, int NQ, bool EXACT>
__global__ void __launch_bounds__(kThreads, Shape<T, KD>::kCtas) k_paged_attention(const __grid_constant__ PagedAttArgs a)
{
    using S = Shape<T, KD>;
    using Core = Kind<KD, NQ, EXACT>;
    constexpr uint32_t kTile = kWarps * S::kKeys;
    constexpr int kRounds = (Core::kQueries + S::kRound - 1) / S::kRound;
    extern __shared__ __align__(128) unsigned char sm[];
    float *qs = reinterpret_cast<float *>(sm + S::kRing);
    // two join buffers: one is joined while the other fills
    float *join = reinterpret_cast<float *>(sm + S::kRing + S::kQBytes);
    uint32_t *valid = reinterpret_cast<uint32_t *>(join + 2 * S::kJoin); // [kWarps][kStages]
    __shared__ uint64_t sums[kWarps];
    __shared__ Cursor first;
    __shared__ uint32_t last_one;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t items = a.kv.kv_heads * a.qtiles; // of a sequence
    if (!EXACT)
    {
        // the pieces of a key behind head_dim are never loaded: they have to be zeros, not whatever was there
        const uint32_t have = a.kv.head_dim * (uint32_t)sizeof(T) / 16, gap = KD * (uint32_t)sizeof(T) / 16 - have;
        for (uint32_t i = tid; i < kWarps * S::kStages * S::kKeys * gap; i += kThreads)
        {
            const uint32_t row = i / gap, r = row % S::kKeys, p = have + i % gap;
            *reinterpret_cast<uint4 *>(sm + row / S::kKeys * S::kStage + S::at(r, p)) = make_uint4(0, 0, 0, 0);
        }
    }

    // This CTA's part of the line: every thread sums a run of sequences, the one in whose run the part
    // begins finds its place. On the way, sequences without keys get their zeros (each from one CTA).
    const uint32_t per_thread = (a.n_seqs + kThreads - 1) / kThreads;
    uint64_t mine = 0;
    uint32_t status = 0;
    for (uint32_t i = 0; i < per_thread; ++i)
    {
        const uint32_t s = tid * per_thread + i;
        const uint32_t len = s < a.n_seqs ? a.lens[s] : 1;
        if (s < a.n_seqs)
        {
            if (len > a.cap)
                status = VKLLM_B200_PAGED_TOO_LONG;
            mine += item_units((min(len, a.cap) + kTile - 1) / kTile);
        }
        uint32_t empty = __ballot_sync(0xffffffffu, len == 0 && s % gridDim.x == blockIdx.x);
        while (empty)
        {
            const uint32_t z = __shfl_sync(0xffffffffu, s, __ffs(empty) - 1);
            empty &= empty - 1;
            uint4 *row = reinterpret_cast<uint4 *>((T *)a.out + z * a.out_stride);
            for (uint32_t d = lane; d < a.kv.kv_heads * a.group * a.kv.head_dim * (uint32_t)sizeof(T) / 16; d += 32)
                row[d] = make_uint4(0, 0, 0, 0);
        }
    }
    if (status)
        atomicOr(a.status, status);
    mine *= items;
    uint64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const uint64_t t = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o)
            before += t;
    }
    if (lane == 31)
        sums[warp] = before;
    __syncthreads();
    uint64_t total = 0;
    before -= mine;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w)
    {
        if (w < warp)
            before += sums[w];
        total += sums[w];
    }
    const uint64_t per = max(quotient(total + gridDim.x - 1, gridDim.x), (uint64_t)kMinUnits);
    const uint64_t begin = blockIdx.x * per;
    if (begin >= total)
        return;
    const uint32_t end = (uint32_t)min(per, total - begin);
    if (before <= begin && begin < before + mine)
    {
        Cursor c;
        c.seq = tid * per_thread;
        uint64_t at = before;
        uint32_t units = 0;
        for (; c.seq < a.n_seqs; ++c.seq)
        {
            c.set_len(a, kTile);
            units = item_units(c.tiles);
            if (begin < at + (uint64_t)units * items)
                break;
            at += (uint64_t)units * items;
        }
        units = max(units, 1u);
        c.hq = (uint32_t)quotient(begin - at, units);
        // a tile is the CTA's in whose part its first unit lies
        const uint32_t x = (uint32_t)(begin - at - (uint64_t)c.hq * units);
        c.tile = (x + kTileUnits - 1) / kTileUnits;
        c.unit = c.tile * kTileUnits - x;
        if (c.tile >= c.tiles)
        {
            c.unit = units - x - kItemUnits; // modulo 2^32: next_item adds them again
            c.next_item(a, items, kTile);
        }
        first = c;
    }
    __syncthreads();

    Cursor c = first;
    Loader<T, KD, EXACT> ld;
    ld.c = c;
    ld.end = end;
    ld.ring = (uint32_t)__cvta_generic_to_shared(sm) + warp * S::kStages * S::kStage;
    ld.valid = valid + warp * S::kStages;
    ld.begin(a, warp, lane);
#pragma unroll 1 // (a copy of the code for every round would only be fetched from memory once more)
    for (uint32_t i = 0; i + 1 < S::kStages; ++i)
        ld.issue(a, items, warp, lane);

    Core core;
    uint32_t stage = 0, buffer = 0;
    while (c.unit < end && c.seq < a.n_seqs)
    {
        // one item, or this CTA's part of it
        const uint32_t from = c.tile, n = min(c.tiles - from, (end - c.unit + kTileUnits - 1) / kTileUnits);
        const uint32_t kh = a.qtiles > 1 ? c.hq / a.qtiles : c.hq, qt = c.hq - kh * a.qtiles;
        const uint32_t head0 = kh * a.group + qt * a.gq;
        const uint32_t nq = min(a.gq, a.group - qt * a.gq);
        core.start(a, c.seq, head0, nq, lane, qs);
        for (uint32_t i = 0; i < n; ++i)
        {
            cp_wait<S::kStages - 2>();
            __syncwarp();
            ld.issue(a, items, warp, lane); // into the stage that the warp read before
            const uint32_t mask = ld.valid[stage];
            if (mask)
                core.slice(a, ld.ring + stage * S::kStage, mask, lane, qs);
            stage = stage + 1 == S::kStages ? 0 : stage + 1;
        }
        const bool whole = n == c.tiles;
        float *part = whole ? nullptr : part_of(a, blockIdx.x, from == 0);
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
        {
            if (r * S::kRound >= nq)
                break;
            // the barrier also says that every warp is done with the other buffer
            float *os = join + buffer * S::kJoin, *ml = os + kWarps * S::kRound * S::kPitch;
            core.deposit(r, nq, os + warp * S::kRound * S::kPitch, ml + warp * S::kRound * 2, lane);
            __syncthreads();
            join_warps<T, KD>(a, os, ml, min(nq - r * S::kRound, S::kRound), r * S::kRound, c.seq, head0, part);
            buffer ^= 1;
        }
        if (!whole)
        {
            // CTAs c0 .. c1 hold the item's parts
            const uint64_t item = begin + c.unit - from * kTileUnits;
            const uint32_t c0 = (uint32_t)quotient(item, per),
                           c1 = (uint32_t)quotient(item + (c.tiles - 1) * (uint64_t)kTileUnits, per);
            __syncthreads();
            if (tid == 0)
            {
                __threadfence(); // the part, which the barrier made this thread's to publish, before the count
                const uint32_t came = atomicAdd(a.counters + c0, 1u);
                last_one = came == c1 - c0;
                if (came > c1 - c0)
                    atomicOr(a.status, (uint32_t)VKLLM_B200_PAGED_BAD_WORKSPACE);
                __threadfence();
            }
            __syncthreads();
            if (last_one)
            {
                if (tid == 0)
                    a.counters[c0] = 0; // ready for the next call
                join_parts<T, KD>(a, c0, c1, join, nq, c.seq, head0);
            }
        }
        c.tile = from + n - 1;
        c.unit += (n - 1) * kTileUnits;
        c.next(a, items, kTile);
    }
    if (ld.status)
        atomicOr(a.status, ld.status);
}

template <template <int, int, bool> class Kind, typename T, int KD, int NQ, bool EXACT>
vkllm_err_t launch(PagedAttArgs &a, int sms, int device, cudaStream_t s)
{
    using S = Shape<T, KD>;
    auto kernel = k_paged_attention<Kind, T, KD, NQ, EXACT>;
    static std::atomic<bool> done[64]; // the attribute of this kernel, set once a device (twice does no harm)
    if (device >= 64 || !done[device].load(std::memory_order_relaxed))
    {
        VKB_CUDA(cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
        if (device < 64)
            done[device].store(true, std::memory_order_relaxed);
    }
    a.part_stride = a.gq * (KD + 2);
    a.part_stride = (a.part_stride + 3) / 4 * 4;
    // most CTAs that can have work, that the counters and the workspace serve, and that the GPU holds at once
    const uint32_t tiles = (uint32_t)((a.cap + (uint64_t)kWarps * S::kKeys - 1) / (kWarps * S::kKeys));
    const uint64_t units = (uint64_t)tiles * kTileUnits + kItemUnits;
    const uint64_t work = (units * a.n_seqs * a.kv.kv_heads * a.qtiles + kMinUnits - 1) / kMinUnits;
    const uint64_t room = (VKLLM_B200_PAGED_WORKSPACE_BYTES - kCounters * 4) / (2 * (uint64_t)a.part_stride * 4);
    uint64_t grid = (uint64_t)sms * S::kCtas;
    grid = grid < work ? grid : work;
    grid = grid < room ? grid : room;
    grid = grid < kCounters ? grid : kCounters;
    return launch_plain(kernel, a, dim3((unsigned)grid), kThreads, S::kSmem, s);
}

template <template <int, int, bool> class Kind, typename T, int KD, int NQ>
vkllm_err_t launch_exact(PagedAttArgs &a, int sms, int device, cudaStream_t s)
{
    return a.kv.head_dim == KD ? launch<Kind, T, KD, NQ, true>(a, sms, device, s)
                               : launch<Kind, T, KD, NQ, false>(a, sms, device, s);
}

template <int KD> vkllm_err_t launch_head(PagedAttArgs &a, int sms, int device, cudaStream_t s)
{
    if (a.kv.dtype == vkllm_dtype_float16)
        return a.gq <= 8 ? launch_exact<HalfCore, __half, KD, 1>(a, sms, device, s)
                         : launch_exact<HalfCore, __half, KD, 2>(a, sms, device, s);
    return a.gq == 1   ? launch_exact<FloatCore, float, KD, 1>(a, sms, device, s)
           : a.gq <= 4 ? launch_exact<FloatCore, float, KD, 4>(a, sms, device, s)
                       : launch_exact<FloatCore, float, KD, 8>(a, sms, device, s);
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
    _CHECK(check_device({kv->k, kv->v, t->table, q, lens, out, workspace, status}, &sms, &dev));
    PagedAttArgs a;
    a.kv = *kv;
    a.table = t->table, a.table_stride = t->stride, a.n_seqs = t->n_seqs;
    a.cap = (uint32_t)(table_rows(*t) < 0xffffff00ull ? table_rows(*t) : 0xffffff00ull);
    a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.lens = lens;
    a.page_bytes = kv->page_stride * es, a.head_bytes = kv->head_stride * es, a.row_bytes = kv->row_stride * es;
    a.page_magic = kv->page_rows > 1 ? ~0ull / kv->page_rows + 1 : 0;
    a.group = heads / kv->kv_heads;
    const uint32_t most = kv->dtype == vkllm_dtype_float16 ? 16 : 8; // queries that a CTA takes through one pass
    a.qtiles = (a.group + most - 1) / most;
    a.gq = (a.group + a.qtiles - 1) / a.qtiles;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.status = status;
    a.counters = (uint32_t *)workspace;
    a.parts = (float *)((char *)workspace + kCounters * 4);
    cudaStream_t s = (cudaStream_t)stream;
    return kv->head_dim <= 64    ? launch_head<64>(a, sms, dev, s)
           : kv->head_dim <= 96  ? launch_head<96>(a, sms, dev, s)
           : kv->head_dim <= 128 ? launch_head<128>(a, sms, dev, s)
           : kv->head_dim <= 192 ? launch_head<192>(a, sms, dev, s)
                                 : launch_head<256>(a, sms, dev, s);
}
