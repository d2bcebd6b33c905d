"""The paged serving operators on the GPU against their definitions in 64 bits: page tables and slot maps
(whole numbers: equal), RoPE with rows written into the pages, attention of one new token per sequence
over the pages, and the run of them as a decoding server makes it.

Tolerances (u = 2^-24, half a step of fp32; an fp16 output is off by half a step, 2^-11 |value|, or by
2^-25 below its normal range):
  rope   a result is c x - s y with |c|, |s| <= 1: sincospif is off by at most 2 units in the last place
         (2^-22), each product and the sum round once: 2^-20 (|x| + |y|) covers them, plus the output's.
  attention  a score is a sum of head_dim products; in any order, with sums that may cut instead of round (tensor cores),
         it is off by ds = scale * (head_dim + 8) 2u * sum |q_d k_d|. The factor exp(ds) on each weight
         and on their sum changes the result by at most 2 ds * sum p |v|; exp2 of a rounded argument is off by (|s - m| + 4) 2u
         of the weight, weights kept as two fp16 parts by 2^-21, and the sums over n keys by (n + 64) 2u.
"""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def i32(torch, x):
    """uint32 values as an int32 tensor with the same bits."""
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x, dtype=np.uint32).view(np.int32))).cuda()


def u32(t):
    return t.cpu().numpy().view(np.uint32)


# ---- page tables ---------------------------------------------------------------------------------

class Book:
    """A table with its free list on the GPU, and the same on the CPU."""

    def __init__(self, vk, torch, lens, cols, page_rows, spare, seed=0, pad=0):
        rng = np.random.default_rng(seed)
        n = len(lens)
        held = [-(-l // page_rows) for l in lens]
        self.n_pages = sum(held) + spare
        order = rng.permutation(self.n_pages).astype(np.uint32)
        self.table = np.full((n, cols + pad), 0xffffffff, dtype=np.uint32)
        at = 0
        for s, h in enumerate(held):
            self.table[s, :h] = order[at:at + h]
            at += h
        self.free = np.concatenate([order[at:], np.full(at, 0xeeeeeeee, dtype=np.uint32)])
        self.count, self.lens = spare, np.asarray(lens, dtype=np.uint32)
        self.cols, self.page_rows, self.torch, self.vk = cols, page_rows, torch, vk
        self.d_table, self.d_free = i32(torch, self.table), i32(torch, self.free)
        self.d_lens, self.d_count = i32(torch, self.lens), i32(torch, [self.count])
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def c_table(self):
        return self.vk.PagedTable(self.d_table.data_ptr(), self.d_free.data_ptr(), self.table.shape[1], len(self.lens),
                                  self.cols, self.page_rows, self.n_pages)

    def append(self, new, max_tokens, in_place=True):
        """The device call; returns (new_lens, n_free_out, starts, slots, positions) as uint32 arrays."""
        torch, n = self.torch, len(self.lens)
        d_new = i32(torch, new)
        guard = 7  # words behind each output that have to stay
        out = {"starts": n + 1, "slots": max_tokens, "positions": max_tokens, "lens": n, "count": 1}
        buf = {k: torch.full((m + guard,), 0x55555555, dtype=torch.int32, device="cuda") for k, m in out.items()}
        lens = self.d_lens if in_place else buf["lens"]
        count = self.d_count if in_place else buf["count"]
        err = self.vk.lib().vkllm_b200_paged_append(
            C.byref(self.c_table()), self.d_lens.data_ptr(), d_new.data_ptr(), self.d_count.data_ptr(), lens.data_ptr(),
            count.data_ptr(), buf["starts"].data_ptr(), buf["slots"].data_ptr(), buf["positions"].data_ptr(), max_tokens,
            self.status.data_ptr(), stream(torch))
        assert err == self.vk.OK
        torch.cuda.synchronize()
        for k, m in out.items():
            assert (u32(buf[k])[m:] == 0x55555555).all(), k
        return (u32(lens)[:n].copy(), int(u32(count)[0]), u32(buf["starts"])[:n + 1], u32(buf["slots"])[:max_tokens],
                u32(buf["positions"])[:max_tokens])

    def want_append(self, new, max_tokens):
        """The same by loops over sequences and tokens, on the CPU arrays; returns the outputs and the status."""
        R, st = self.page_rows, 0
        new = [int(x) for x in new]
        want = [-(-(int(l) + m) // R) - -(-int(l) // R) for l, m in zip(self.lens, new)]
        if any(int(l) + m > self.cols * R for l, m in zip(self.lens, new)):
            st |= 2
        if sum(want) > self.count:
            st |= 4
        if sum(new) > max_tokens:
            st |= 8
        if st:
            new = [0] * len(new)
        starts, slots, pos = [0], [], []
        for s, m in enumerate(new):
            for p in range(int(self.lens[s]), int(self.lens[s]) + m):
                if p % R == 0:
                    self.count -= 1
                    self.table[s, p // R] = self.free[self.count]
                slots.append(int(self.table[s, p // R]) * R + p % R)
                pos.append(p)
            starts.append(starts[-1] + m)
        gap = max_tokens - len(slots)
        self.lens = (self.lens + np.asarray(new, dtype=np.uint32)).astype(np.uint32)
        return (self.lens, self.count, np.asarray(starts), np.asarray(slots + [0xffffffff] * gap),
                np.asarray(pos + [0] * gap)), st

    def release(self, done, in_place=True):
        torch, n = self.torch, len(self.lens)
        lens = self.d_lens if in_place else torch.full((n,), 0x5a5a5a5a, dtype=torch.int32, device="cuda")
        count = self.d_count if in_place else torch.full((1,), 0x5a5a5a5a, dtype=torch.int32, device="cuda")
        d_done = i32(torch, done)
        err = self.vk.lib().vkllm_b200_paged_release(C.byref(self.c_table()), self.d_lens.data_ptr(), d_done.data_ptr(),
                                                     self.d_count.data_ptr(), lens.data_ptr(), count.data_ptr(),
                                                     self.status.data_ptr(), stream(torch))
        assert err == self.vk.OK
        torch.cuda.synchronize()
        return u32(lens).copy(), int(u32(count)[0])

    def want_release(self, done):
        for s, d in enumerate(done):
            if d:
                for c in range(-(-int(self.lens[s]) // self.page_rows)):
                    self.free[self.count] = self.table[s, c]
                    self.count += 1
                self.lens[s] = 0
        return self.lens, self.count

    def same(self, got, want):
        for g, w, what in zip(got, want, ("lens", "count", "starts", "slots", "positions")):
            assert np.array_equal(np.asarray(g, dtype=np.uint32), np.asarray(w, dtype=np.uint32)), what
        assert np.array_equal(u32(self.d_table), self.table)
        assert np.array_equal(u32(self.d_free), self.free)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n,page_rows,cols,hi,max_tokens", [
    (1, 16, 4, 1, 1), (1, 1, 9, 5, 9), (3, 16, 8, 20, 64), (64, 16, 256, 1, 64), (65, 7, 40, 30, 2000),
    (513, 32, 12, 90, 60000), (5, 24, 2000, 9000, 50000), (2100, 3, 9, 4, 9001), (16384, 16, 3, 2, 40000)])
def test_append(vk, torch, n, page_rows, cols, hi, max_tokens, in_place):
    """Lengths from none to as long as the new rows allow; slots beside page ends; more outputs than tokens."""
    rng = np.random.default_rng(n * 7 + page_rows)
    new = rng.integers(0, hi + 1, n)
    new[0] = hi
    lens = [int(rng.choice([0, page_rows, page_rows - 1, rng.integers(0, cols * page_rows - m + 1),
                            cols * page_rows - m])) for m in new]
    lens = [min(l, cols * page_rows - int(m)) for l, m in zip(lens, new)]
    b = Book(vk, torch, lens, cols, page_rows, spare=int(sum(new)) + 3, seed=n, pad=n % 3)
    got = b.append(new, max_tokens, in_place)
    want, st = b.want_append(new, max_tokens)
    assert st == 0 and int(u32(b.status)[0]) == 0
    b.same(got, want)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_append_of_many_tokens_to_any_alignment(vk, torch, shift):
    """The slot map's outputs on no 16-byte boundary, both of them or one."""
    b = Book(vk, torch, [30, 0, 9], 1000, 7, spare=1500, seed=6)
    new, most = [3000, 1, 2500], 5502 + shift
    slots, pos = (torch.full((most + 8,), 0x55, dtype=torch.int32, device="cuda") for _ in range(2))
    starts = torch.zeros(4, dtype=torch.int32, device="cuda")
    ps, pp = slots.data_ptr() + 4 * shift, pos.data_ptr() + 4 * (shift if shift != 2 else 0)
    err = vk.lib().vkllm_b200_paged_append(C.byref(b.c_table()), b.d_lens.data_ptr(), i32(torch, new).data_ptr(),
                                           b.d_count.data_ptr(), b.d_lens.data_ptr(), b.d_count.data_ptr(),
                                           starts.data_ptr(), ps, pp, most, b.status.data_ptr(), stream(torch))
    assert err == vk.OK
    torch.cuda.synchronize()
    want, st = b.want_append(new, most)
    at = shift if shift != 2 else 0
    assert st == 0 and int(b.status) == 0
    assert np.array_equal(u32(slots)[shift:shift + most], want[3]) and np.array_equal(u32(pos)[at:at + most], want[4])
    assert (u32(slots)[shift + most:] == 0x55).all() and (u32(slots)[:shift] == 0x55).all()
    assert (u32(pos)[at + most:] == 0x55).all()


def test_append_with_slots_past_31_bits(vk, torch):
    """Pages of 2^24 rows: lengths, positions and slots beyond 2^31, and a capacity beyond 2^32."""
    R = 1 << 24
    b = Book(vk, torch, [100 * R + R - 3, 30 * R, 0, 77 * R + 5], 400, R, spare=20, seed=8)
    new = [6, 2, 1, 4]
    got = b.append(new, 15)
    slots = []
    for s, (l, m) in enumerate(zip([100 * R + R - 3, 30 * R, 0, 77 * R + 5], new)):
        for p in range(l, l + m):
            if p % R == 0:
                b.count -= 1
                b.table[s, p // R] = b.free[b.count]
            slots.append(int(b.table[s, p // R]) * R + p % R)
    b.lens = (b.lens + np.asarray(new, dtype=np.uint32)).astype(np.uint32)
    assert int(b.status) == 0 and max(slots) >= 1 << 31
    want = (b.lens, b.count, [0, 6, 8, 9, 13], slots + [0xffffffff] * 2,
            [p for l, m in zip([100 * R + R - 3, 30 * R, 0, 77 * R + 5], new) for p in range(l, l + m)] + [0, 0])
    b.same(got, want)


def test_append_exactly_what_is_free_and_nothing(vk, torch):
    b = Book(vk, torch, [4, 0, 3], 4, 4, spare=3)
    b.same(b.append([1, 4, 5], 10), b.want_append([1, 4, 5], 10)[0])  # 1 + 1 + 1 pages: the list is empty now
    assert int(u32(b.status)[0]) == 0 and b.count == 0
    b.same(b.append([3, 0, 0], 3), b.want_append([3, 0, 0], 3)[0])  # rows of a page that is already held
    b.same(b.append([0, 0, 0], 0), b.want_append([0, 0, 0], 0)[0])  # no token and no slot
    assert int(u32(b.status)[0]) == 0


@pytest.mark.parametrize("n", [3, 5000])
@pytest.mark.parametrize("what,bit", [("pages", 4), ("long", 2), ("tokens", 8), ("bad free id", 1), ("bad held id", 1),
                                      ("count past the pool", 4)])
def test_append_is_all_or_nothing(vk, torch, what, bit, n):
    """A call that cannot be done sets its bit, and does what it would do for nothing new."""
    new = [5] + [1] * (n - 1)
    b = Book(vk, torch, [6] * n, 4, 4, spare=0 if what == "pages" else 2 * n + 5, seed=4)
    max_tokens = sum(new)
    if what == "long":
        new[n - 1] = 11
        max_tokens += 10
    if what == "tokens":
        max_tokens -= 1
    if what == "bad free id":
        b.free[b.count - 1] = b.n_pages
        b.d_free = i32(torch, b.free)
    if what == "bad held id":
        b.table[n - 1, 1] = b.n_pages + 5
        b.d_table = i32(torch, b.table)
    if what == "count past the pool":
        b.count = b.n_pages + 1
        b.d_count = i32(torch, [b.count])
    got = b.append(new, max_tokens)
    assert int(u32(b.status)[0]) & bit
    count = b.count
    want, _ = b.want_append([0] * n, max_tokens)
    assert b.count == count
    b.same(got, want)


@pytest.mark.parametrize("n,page_rows,cols,in_place", [(1, 4, 5, True), (7, 16, 9, False), (700, 5, 30, True),
                                                       (16384, 8, 3, True)])
def test_release_and_append_again(vk, torch, n, page_rows, cols, in_place):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, cols * page_rows + 1, n)
    b = Book(vk, torch, list(lens), cols, page_rows, spare=5, seed=3, pad=1)
    done = (rng.random(n) < 0.4).astype(np.uint32) * 7
    done[0] = 1
    got = b.release(done, in_place)
    b.same(got, b.want_release(done))
    if in_place:
        new = np.where(done != 0, np.minimum(lens, 3), 0)
        got = b.append(new, int(sum(new)) + 2)
        b.same(got, b.want_append(new, int(sum(new)) + 2)[0])
    assert int(u32(b.status)[0]) == 0


@pytest.mark.parametrize("what,bit", [("bad id", 1), ("long", 2), ("twice", 8)])
def test_release_is_all_or_nothing(vk, torch, what, bit):
    b = Book(vk, torch, [6, 9, 4], 3, 4, spare=1, seed=2)
    if what == "bad id":
        b.table[1, 2] = b.n_pages
        b.d_table = i32(torch, b.table)
    if what == "long":
        b.lens[1] = 13
        b.d_lens = i32(torch, b.lens)
    if what == "twice":  # more pages than the pool has left to give
        b.count = b.n_pages - 2
        b.d_count = i32(torch, [b.count])
    got = b.release([0, 1, 0])
    assert int(u32(b.status)[0]) == bit
    b.same(got, (b.lens, b.count))


@pytest.mark.parametrize("n", [65, 129, 1100, 2100])
def test_tables_beside_other_work(vk, torch, n):
    """Clusters of 2 to 8 CTAs (release: 65, 129 and more slots; append: 1100 and 2100) while products on another
    stream leave SMs free a few at a time, so that a cluster's CTAs start when they can. Their words about bad
    values have to reach every one of them: each round has one call that has to be refused by all."""
    b = Book(vk, torch, [4] * n, 6, 4, spare=2 * n, seed=n)
    other, x = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda").half()
    torch.cuda.synchronize()
    done = np.zeros(n, dtype=np.uint32)
    done[::3] = 1
    for i in range(12):
        with torch.cuda.stream(other):
            for _ in range(4):
                x @ x
        b.same(b.append([1] * n, n + 5), b.want_append([1] * n, n + 5)[0])
        assert int(u32(b.status)[0]) == 0
        # a bad page of one sequence, found by one CTA alone
        s = int(np.flatnonzero(done)[-1 - i % 3])
        keep, b.table[s, 1] = b.table[s, 1], b.n_pages
        b.d_table.copy_(i32(torch, b.table))
        with torch.cuda.stream(other):
            x @ x
        for call in (lambda: b.release(done), lambda: b.append([1] * n, n)):
            got = call()
            assert int(u32(b.status)[0]) == vk.PAGED_BAD_PAGE
            assert np.array_equal(got[0], b.lens) and got[1] == b.count
            b.status.zero_()
        assert np.array_equal(u32(b.d_table), b.table) and np.array_equal(u32(b.d_free), b.free)
        b.table[s, 1] = keep
        b.d_table.copy_(i32(torch, b.table))
        b.same(b.release(done), b.want_release(done))
        new = np.where(done != 0, 4, 0)
        b.same(b.append(new, 4 * n), b.want_append(new, 4 * n)[0])
        b.lens[:] = np.where(done != 0, b.lens, 4)  # the others' second pages go back to the list by hand
        held = b.table[done == 0, 1]
        b.free[b.count:b.count + len(held)], b.count = held, b.count + len(held)
        b.d_lens.copy_(i32(torch, b.lens))
        b.d_free.copy_(i32(torch, b.free))
        b.d_count.copy_(i32(torch, [b.count]))
        assert int(u32(b.status)[0]) == 0
    torch.cuda.synchronize()


# ---- pools ---------------------------------------------------------------------------------------

LAYOUTS = ["heads first", "rows first", "joined"]


def make_pools(vk, torch, layout, n_pages, page_rows, kv_heads, hd, dtype, g):
    """K and V with the logical shape [page, head, row, d]; joined: K and V of a page lie side by side in a
    page that is longer still."""
    dt = torch.float16 if dtype == "f16" else torch.float32
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)  # noqa: E731
    if layout == "heads first":
        k, v = (r(n_pages, kv_heads, page_rows, hd) for _ in range(2))
    elif layout == "rows first":
        k, v = (r(n_pages, page_rows, kv_heads, hd).transpose(1, 2) for _ in range(2))
    else:
        both = r(n_pages, 2 * kv_heads + 1, page_rows, hd + 8)
        k, v = both[:, :kv_heads, :, :hd], both[:, kv_heads:2 * kv_heads, :, :hd]
    c = vk.PagedKV(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), n_pages, page_rows, kv_heads, hd,
                   vk.F16 if dtype == "f16" else vk.F32, 0)
    return k, v, c


def out_tol(ref, dtype):
    """Half a step of the output's type."""
    return ref.abs() * 2.0 ** -11 + 2.0 ** -25 if dtype == "f16" else ref.abs() * U + 2.0 ** -149


def within(got, ref, tol, what=""):
    d = (got.double() - ref).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol).max()):.3g} x tol"


# ---- rope ----------------------------------------------------------------------------------------

def rope_call(vk, torch, kv, qkv, H, HK, hd, positions, slots, n, base, q_out, status, in_place=False):
    es = qkv.element_size()
    st = qkv.stride(0)
    q = qkv.data_ptr()
    out, out_st = (q, st) if in_place else (q_out.data_ptr(), q_out.stride(0))
    return vk.lib().vkllm_b200_paged_rope_write(
        C.byref(kv), q, st, q + H * hd * es, st, q + (H + HK) * hd * es, st, positions.data_ptr(), slots.data_ptr(), n, H,
        base, out, out_st, status.data_ptr(), stream(torch))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("H,HK,hd,n,page_rows,base", [
    (1, 1, 8, 1, 1, 0.0), (6, 6, 48, 5, 16, 10000.0), (32, 32, 128, 64, 16, 10000.0), (8, 1, 64, 33, 7, 500000.0),
    (12, 4, 80, 300, 24, 10000.0), (4, 2, 256, 17, 64, 1000000.0), (16, 2, 96, 700, 32, 2.0)])
def test_rope_write(vk, torch, dtype, layout, H, HK, hd, n, page_rows, base):
    """Queries, keys and values as parts of one longer row; far and near positions; every fourth token and
    the last without a slot; the rest of the pools, of q_out and of the row stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(n + hd)
    n_pages = n // page_rows + 3
    k, v, kv = make_pools(vk, torch, layout, n_pages, page_rows, HK, hd, dtype, g)
    dt = k.dtype
    qkv = torch.randn((n, (H + 2 * HK) * hd + 8), generator=g, device="cuda").to(dt)
    q_out = torch.full((n, H * hd + 16), 3.25, dtype=dt, device="cuda")
    slots = torch.randperm(n_pages * page_rows, generator=g, device="cuda")[:n].to(torch.int32)
    if n > 1:
        slots[3::4] = -1
        slots[n - 1] = -1
    positions = torch.randint(0, 200000, (n,), generator=g, device="cuda", dtype=torch.int32)
    positions[0] = 0 if n > 1 else 2 ** 31 - 1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    k0, v0, q0, qkv0 = k.double(), v.double(), q_out.double(), qkv.clone()
    assert rope_call(vk, torch, kv, qkv, H, HK, hd, positions, slots, n, base, q_out, status) == vk.OK
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(qkv, qkv0)
    w = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    th = positions.double()[:, None] * torch.pow(torch.tensor(base or 10000.0, dtype=torch.float64, device="cuda"),
                                                 -2 * w / hd)
    cos, sin = th.cos()[:, None], th.sin()[:, None]

    def turn(x):
        x = x.double().reshape(n, -1, hd // 2, 2)
        a, b = x[..., 0], x[..., 1]
        mag = (a.abs() + b.abs())[..., None].expand(-1, -1, -1, 2).reshape(n, -1, hd)
        return torch.stack([cos * a - sin * b, sin * a + cos * b], -1).reshape(n, -1, hd), mag

    here = slots >= 0
    qr, qm = turn(qkv[:, :H * hd])
    kr, km = turn(qkv[:, H * hd:(H + HK) * hd])
    ref = q0.clone()
    ref[:, :H * hd][here] = qr.reshape(n, -1)[here]
    tol = torch.zeros_like(ref)
    # the angle in the reference, position * frequency in 64 bits, is itself off by 2^-52 of up to 2^31
    tol[:, :H * hd][here] = ((2.0 ** -20 + 2.0 ** -20 * (n == 1)) * qm + out_tol(qr, dtype)).reshape(n, -1)[here]
    within(q_out, ref, tol, "q")
    page, row = (slots[here] // page_rows).long(), (slots[here] % page_rows).long()
    refk, refv, tolk = k0, v0.clone(), torch.zeros_like(k0)
    refk[page, :, row] = kr[here]
    tolk[page, :, row] = ((2.0 ** -20 + 2.0 ** -20 * (n == 1)) * km + out_tol(kr, dtype))[here]
    refv[page, :, row] = qkv[:, (H + HK) * hd:(H + 2 * HK) * hd].double().reshape(n, HK, hd)[here]
    within(k, refk, tolk, "k")
    assert torch.equal(v.double(), refv)


@pytest.mark.parametrize("hd,base", [(128, 10000.0), (256, 1000000.0), (8, 1.5)])
def test_rope_sines_at_far_positions(vk, torch, hd, base):
    """Queries of (1, 0) pairs in fp32 come out as the cosines and sines themselves. Tolerance 2^-22: the angle as a
    number of half turns in fp32 is off by 2^-25 of one, a sine by pi times that (9.4e-8), and sincospif by 2 units in the
    last place of values below 1 (1.2e-7). The reference's angle, with 64 bits of mantissa, is off by 2^-33."""
    assert np.finfo(np.longdouble).nmant >= 63
    n = 4096
    g = torch.Generator(device="cuda").manual_seed(hd)
    k, v, kv = make_pools(vk, torch, "heads first", 1, n, 1, hd, "f32", g)
    qkv = torch.zeros((n, 3 * hd), device="cuda")
    qkv[:, 0:hd:2] = 1
    positions = np.random.default_rng(hd).integers(0, 2 ** 31, n)
    positions[:3] = 0, 1, 2 ** 31 - 1
    q_out, status = torch.zeros((n, hd), device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.arange(n, device="cuda", dtype=torch.int32)
    assert rope_call(vk, torch, kv, qkv, 1, 1, hd, i32(torch, positions), slots, n, base, q_out, status) == vk.OK
    got = q_out.cpu().numpy().astype(np.longdouble)
    w = np.arange(hd // 2, dtype=np.longdouble)
    th = positions.astype(np.longdouble)[:, None] * np.longdouble(np.float32(base)) ** (-2 * w / hd)
    assert int(status) == 0
    assert float(np.abs(got[:, 0::2] - np.cos(th)).max()) <= 2.0 ** -22
    assert float(np.abs(got[:, 1::2] - np.sin(th)).max()) <= 2.0 ** -22


def test_rope_write_in_place_equals_out_of_place(vk, torch):
    g = torch.Generator(device="cuda").manual_seed(5)
    H, HK, hd, n = 8, 2, 64, 40
    k, v, kv = make_pools(vk, torch, "heads first", 4, 16, HK, hd, "f16", g)
    qkv = torch.randn((n, (H + 2 * HK) * hd), generator=g, device="cuda").half()
    q_out = torch.zeros((n, H * hd), dtype=torch.float16, device="cuda")
    pos, slots = (torch.arange(n, device="cuda", dtype=torch.int32) for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert rope_call(vk, torch, kv, qkv, H, HK, hd, pos, slots, n, 0.0, q_out, status) == vk.OK
    k1 = k.clone()
    assert rope_call(vk, torch, kv, qkv, H, HK, hd, pos, slots, n, 0.0, None, status, in_place=True) == vk.OK
    assert torch.equal(qkv[:, :H * hd], q_out) and torch.equal(k, k1) and int(status) == 0


def test_rope_write_flags_a_slot_outside_the_pool(vk, torch):
    g = torch.Generator(device="cuda").manual_seed(6)
    H, HK, hd, n = 4, 4, 64, 6
    k, v, kv = make_pools(vk, torch, "rows first", 3, 8, HK, hd, "f16", g)
    qkv = torch.randn((n, 3 * H * hd), generator=g, device="cuda").half()
    q_out = torch.full((n, H * hd), 2.0, dtype=torch.float16, device="cuda")
    slots = i32(torch, [1, 24, 5, 0xfffffffe, 23, 0xffffffff])
    status, k0 = torch.zeros(1, dtype=torch.int32, device="cuda"), k.clone()
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    assert rope_call(vk, torch, kv, qkv, H, HK, hd, pos, slots, n, 0.0, q_out, status) == vk.OK
    torch.cuda.synchronize()
    assert int(status) == vk.PAGED_BAD_SLOT
    assert bool((q_out[[1, 3, 5]] == 2.0).all()) and not bool((q_out[[0, 2, 4]] == 2.0).all(1).any())
    changed = (k != k0).any(-1).any(1)  # [page, row]
    assert sorted((p * 8 + r) for p, r in changed.nonzero().tolist()) == [1, 5, 23]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_rope_write_of_padding_does_not_read_its_rows(vk, torch, dtype):
    """64 tokens in a launch for 16384, as a captured step for the most tokens has it: it costs what the slots and
    the launch cost, not the traffic of rows that no slot wants. Rows read for nothing would take 14 us (fp16; 100 MB
    at 7 TB/s) beyond that, so a third of the full call's time is a bound that only reading them passes."""
    g = torch.Generator(device="cuda").manual_seed(8)
    H, HK, hd, n, R = 16, 4, 128, 16384, 64
    if dtype == "f16":
        H, HK = 32, 8
    k, v, kv = make_pools(vk, torch, "heads first", n // R, R, HK, hd, dtype, g)
    qkv = torch.randn((n, (H + 2 * HK) * hd), generator=g, device="cuda").to(k.dtype)
    q_out = torch.zeros((n, H * hd), dtype=k.dtype, device="cuda")
    full = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    few = full.clone()
    few[64:] = -1
    pos, status = torch.arange(n, device="cuda", dtype=torch.int32), torch.zeros(1, dtype=torch.int32, device="cuda")

    def best(slots):
        graph, times = torch.cuda.CUDAGraph(), []
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):  # the GPU's time, whatever the host is doing
            for _ in range(5):
                assert rope_call(vk, torch, kv, qkv, H, HK, hd, pos, slots, n, 0.0, q_out, status) == vk.OK
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times[2:])

    q_out.zero_()
    padded = best(few)
    assert bool((q_out[64:] == 0).all()) and bool((q_out[:64] != 0).any())
    assert padded < best(full) / 3 and int(status) == 0


# ---- attention -----------------------------------------------------------------------------------

class Attend:
    def __init__(self, vk, torch, lens, H, HK, hd, page_rows, dtype, layout="heads first", seed=0, sharp=1.0, cols=None,
                 poison=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.vk, self.torch, self.H, self.HK, self.hd, self.R, self.dtype = vk, torch, H, HK, hd, page_rows, dtype
        self.lens = list(lens)
        n = len(lens)
        cols = cols or max(1, max(-(-l // page_rows) for l in lens))
        held = [-(-l // page_rows) for l in lens]
        self.n_pages = sum(held) + 2
        self.k, self.v, self.kv = make_pools(vk, torch, layout, self.n_pages, page_rows, HK, hd, dtype, g)
        order = torch.randperm(self.n_pages, generator=g, device="cuda").to(torch.int32).cpu().numpy()
        tab = np.full((n, cols + 1), 0xffffffff, dtype=np.uint32)  # entries that hold no page are no page ids
        at = 0
        for s, h in enumerate(held):
            tab[s, :h] = order[at:at + h]
            at += h
            if poison and h and lens[s] % page_rows:  # behind the end: no numbers, infinities
                self.k[int(tab[s, h - 1]), :, lens[s] % page_rows:] = float("nan")
                self.v[int(tab[s, h - 1]), :, lens[s] % page_rows:] = float("inf")
        for p in order[at:]:
            self.k[int(p)] = float("nan")
            self.v[int(p)] = float("nan")
        self.tab, self.d_tab = tab, i32(torch, tab)
        self.d_lens = i32(torch, lens)
        self.q = (torch.randn((n, H * hd + 8), generator=g, device="cuda") * sharp).to(self.k.dtype)
        self.out = torch.full((n + 2, H * hd + 16), 7.5, dtype=self.k.dtype, device="cuda")
        self.ws = torch.zeros(vk.PAGED_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.scale = hd ** -0.5
        self.table = vk.PagedTable(self.d_tab.data_ptr(), None, tab.shape[1], n, cols, page_rows, self.n_pages)

    def call(self, ws=None):
        ws = self.ws if ws is None else ws
        return self.vk.lib().vkllm_b200_paged_attention(
            C.byref(self.kv), C.byref(self.table), self.q.data_ptr(), self.q.stride(0), self.H, self.d_lens.data_ptr(),
            self.scale, self.out.data_ptr(), self.out.stride(0), ws.data_ptr(), ws.numel(), self.status.data_ptr(),
            stream(self.torch))

    def reference(self):
        """Outputs [n, H, hd] in 64 bits and the tolerance of each."""
        torch, H, HK, hd = self.torch, self.H, self.HK, self.hd
        ref = torch.zeros((len(self.lens), H, hd), dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(ref)
        for s, n in enumerate(self.lens):
            if n == 0:
                continue
            ids = torch.from_numpy(self.tab[s, :-(-n // self.R)].astype(np.int64)).cuda()
            k = self.k[ids].transpose(0, 1).reshape(HK, -1, hd)[:, :n].double()
            v = self.v[ids].transpose(0, 1).reshape(HK, -1, hd)[:, :n].double()
            q = self.q[s, :H * hd].double().view(HK, H // HK, hd)
            sc = q @ k.transpose(1, 2) * self.scale
            mag = (q.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * self.scale
            p = sc.softmax(-1)
            ds = (hd + 8) * 2 * U * mag
            far = (sc.amax(-1, keepdim=True) - sc)  # |s - m| of each key weighs with its own p
            off = ((2 * ds + (far * 1.4427 + 4) * 2 * U + 2.0 ** -21 + (n + 64) * 2 * U) * p) @ v.abs()
            o = p @ v
            ref[s], tol[s] = o.reshape(H, hd), off.reshape(H, hd) + out_tol(o, self.dtype).reshape(H, hd)
        return ref, tol

    def check(self, what=""):
        n, w = len(self.lens), self.H * self.hd
        self.torch.cuda.synchronize()
        assert int(self.status) == 0, what
        ref, tol = self.reference()
        within(self.out[:n, :w].reshape(n, self.H, self.hd), ref, tol, what)
        assert bool((self.out[n:] == 7.5).all()) and bool((self.out[:, w:] == 7.5).all()), what  # left as they were


LENS = {"none": [0], "one": [1], "few": [0, 1, 2, 15, 16, 17, 31, 0, 33, 63, 64, 65],
        "ragged": [700, 0, 1, 129, 255, 256, 257, 3, 511, 40, 1000, 64], "long": [5000, 3]}


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("H,HK,hd,page_rows,layout", [
    (1, 1, 8, 16, "heads first"), (6, 6, 48, 16, "heads first"), (32, 32, 128, 16, "heads first"),
    (8, 2, 64, 7, "rows first"), (16, 4, 80, 24, "joined"), (14, 2, 128, 64, "rows first"),
    (16, 1, 128, 1, "heads first"), (40, 2, 96, 32, "joined"), (9, 1, 256, 16, "heads first"),
    (34, 2, 256, 128, "rows first"), (12, 4, 192, 5, "heads first")])
def test_attention(vk, torch, lens, dtype, H, HK, hd, page_rows, layout):
    a = Attend(vk, torch, LENS[lens], H, HK, hd, page_rows, dtype, layout, seed=H + hd)
    assert a.call() == vk.OK
    a.check("first")
    first = a.out.clone()
    a.out.fill_(7.5)
    assert a.call() == vk.OK  # again with the same workspace: the same bits
    a.check("again")
    assert torch.equal(a.out, first)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n,H,HK,hd,hi", [(150, 8, 8, 64, 90), (700, 4, 1, 128, 40), (40, 32, 8, 128, 1500),
                                          (1, 32, 8, 128, 40000), (2, 2, 1, 64, 100001), (3000, 1, 1, 64, 5)])
def test_attention_many_and_long(vk, torch, dtype, n, H, HK, hd, hi):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, hi + 1, n)
    lens[0] = hi
    a = Attend(vk, torch, [int(x) for x in lens], H, HK, hd, 16, dtype, seed=n, poison=n < 200)
    assert a.call() == vk.OK
    a.check()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_shapes_share_a_workspace(vk, torch, dtype):
    """Calls of different shapes one after the other on one workspace."""
    ws = torch.zeros(vk.PAGED_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    for seed, (lens, H, HK, hd) in enumerate([([3000], 32, 1, 256), ([70] * 33, 8, 8, 64), ([0, 0], 4, 4, 128),
                                              ([9000, 1, 9000], 16, 8, 128), ([12000], 2, 2, 48)]):
        a = Attend(vk, torch, lens, H, HK, hd, 16, dtype, seed=seed)
        assert a.call(ws) == vk.OK
        a.check(str(lens))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("sharp", [30.0, 0.0])
def test_attention_of_peaked_and_of_equal_scores(vk, torch, dtype, sharp):
    """One key takes nearly everything (the far keys' weights lie below fp16's range), or all weigh the same."""
    a = Attend(vk, torch, [4000, 33], 8, 2, 128, 16, dtype, seed=9, sharp=sharp)
    assert a.call() == vk.OK
    a.check()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_to_one_strong_first_key_and_many_weak_ones(vk, torch, dtype):
    """The first key scores 11 above the others, whose sum still counts: their weights must not lose bits."""
    a = Attend(vk, torch, [60000], 4, 1, 64, 16, dtype, seed=12)
    a.k.mul_(0.01)
    a.q[:, :256] = 1.0
    a.k[int(a.tab[0, 0]), :, 0] = 11.0 / 8
    a.v[int(a.tab[0, 0])] *= 0.0
    a.v += 1.0
    assert a.call() == vk.OK
    a.check()


def test_attention_offsets_past_32_bits(vk, torch):
    """Pages that lie more than 2^32 elements apart."""
    H, HK, hd, R = 4, 2, 64, 16
    stride = 2 ** 31 + 4096
    big = torch.empty(3 * stride, dtype=torch.float16, device="cuda")
    a = Attend(vk, torch, [37, 9], H, HK, hd, R, "f16", seed=3, poison=False)
    n_pages = 3
    view = big.as_strided((n_pages, 2 * HK, R, hd), (stride, R * hd, hd, 1))
    view.copy_(torch.randn(view.shape, device="cuda"))
    a.k, a.v, a.n_pages = view[:, :HK], view[:, HK:], n_pages
    a.kv = vk.PagedKV(a.k.data_ptr(), a.v.data_ptr(), stride, R * hd, hd, n_pages, R, HK, hd, vk.F16, 0)
    a.tab = np.array([[2, 0, 1], [1, 0xffffffff, 0xffffffff]], dtype=np.uint32)
    a.d_tab = i32(torch, a.tab)
    a.table = vk.PagedTable(a.d_tab.data_ptr(), None, 3, 2, 3, R, n_pages)
    assert a.call() == vk.OK
    a.check()
    q_out = torch.zeros((3, H * hd), dtype=torch.float16, device="cuda")
    qkv = torch.randn((3, (H + 2 * HK) * hd), device="cuda").half()
    slots = i32(torch, [2 * R + 3, 1, R + 15])
    assert rope_call(vk, torch, a.kv, qkv, H, HK, hd, i32(torch, [0, 0, 0]), slots, 3, 0.0, q_out, a.status) == vk.OK
    torch.cuda.synchronize()
    assert torch.equal(a.k[2, :, 3].reshape(-1), qkv[0, H * hd:(H + HK) * hd])
    assert torch.equal(a.v[1, :, 15].reshape(-1), qkv[2, (H + HK) * hd:])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_flags_bad_pages_and_lengths(vk, torch, dtype):
    """A bad page id has no keys and a long length is cut; the other sequences are right."""
    a = Attend(vk, torch, [100, 40, 64, 200], 8, 2, 64, 16, dtype, seed=4)
    tab = a.tab.copy()
    tab[0, 2], tab[2, :] = a.n_pages, 0xfffffff0  # rows 32 .. 47 of the first, everything of the third
    lens = [100, 40, 64, a.table.cols * 16 + 50]  # the last one's rows run past its row of the table
    a.d_tab, a.d_lens = i32(torch, tab), i32(torch, lens)
    a.table.table = a.d_tab.data_ptr()
    assert a.call() == vk.OK
    torch.cuda.synchronize()
    assert int(a.status) == vk.PAGED_BAD_PAGE | vk.PAGED_TOO_LONG
    ref, tol = a.reference()
    got = a.out[:4, :8 * 64].reshape(4, 8, 64)
    within(got[1], ref[1], tol[1])
    assert bool((got[2] == 0).all())
    # the first without the rows of its bad page
    ids = torch.from_numpy(a.tab[0, :7].astype(np.int64)).cuda()
    keep = torch.tensor([j for j in range(100) if not 32 <= j < 48], device="cuda")
    k = a.k[ids].transpose(0, 1).reshape(2, -1, 64)[:, keep].double()
    v = a.v[ids].transpose(0, 1).reshape(2, -1, 64)[:, keep].double()
    p = (a.q[0, :512].double().view(2, 4, 64) @ k.transpose(1, 2) * a.scale).softmax(-1)
    within(got[0], (p @ v).reshape(8, 64), 2 * tol[0] + 2.0 ** -18)
    assert bool((a.out[4:] == 7.5).all())


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_flags_the_last_id_beside_the_largest_pool(vk, torch, dtype):
    """2^32 - 1 pages (one above the other: their stride is 0), whose last id is 2^32 - 2: the id 2^32 - 1 is bad, and
    has no key."""
    dt = torch.float16 if dtype == "f16" else torch.float32
    k, v, q = (torch.randn((1, 64), device="cuda").to(dt) for _ in range(3))
    out, status = torch.zeros_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    kv = vk.PagedKV(k.data_ptr(), v.data_ptr(), 0, 64, 64, 0xffffffff, 1, 1, 64, vk.F16 if dtype == "f16" else vk.F32, 0)
    table, lens = i32(torch, [5, 0xfffffffe, 7]), i32(torch, [3])
    ws = torch.zeros(vk.PAGED_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    t = vk.PagedTable(table.data_ptr(), None, 3, 1, 3, 1, 0xffffffff)

    def call():
        out.zero_()
        status.zero_()
        assert vk.lib().vkllm_b200_paged_attention(C.byref(kv), C.byref(t), q.data_ptr(), 64, 1, lens.data_ptr(), 0.125,
                                                   out.data_ptr(), 64, ws.data_ptr(), ws.numel(), status.data_ptr(),
                                                   stream(torch)) == vk.OK
        torch.cuda.synchronize()
        return int(status)

    tol = (3 + 64 + 8) * 2 * U + 2.0 ** -21
    assert call() == 0
    within(out, v.double(), tol * v.double().abs() + out_tol(v.double(), dtype))
    table[1] = -1
    assert call() == vk.PAGED_BAD_PAGE
    within(out, v.double(), tol * v.double().abs() + out_tol(v.double(), dtype))
    table.fill_(-1)
    assert call() == vk.PAGED_BAD_PAGE and bool((out == 0).all())


def test_memory_that_is_not_the_devices_is_refused(vk, torch):
    """Every array of every call in turn as pinned host memory: refused, and nothing runs."""
    a = Attend(vk, torch, [20], 2, 2, 64, 16, "f16")
    host = torch.zeros(1 << 16, dtype=torch.float16).pin_memory().data_ptr()
    out0 = a.out.clone()
    for name in ("k", "v"):
        keep = getattr(a.kv, name)
        setattr(a.kv, name, host)
        assert a.call() == vk.ARGS, name
        setattr(a.kv, name, keep)
    s, kv, t, lib = stream(torch), C.byref(a.kv), C.byref(a.table), vk.lib()
    dev, n = a.q.data_ptr(), 8
    at = lambda i, k: host if i == k else dev  # noqa: E731
    for k in range(5):
        assert lib.vkllm_b200_paged_attention(kv, t, at(0, k), a.q.stride(0), 2, at(1, k), 0.1,
                                              host if k == 2 else a.out.data_ptr(), a.out.stride(0),
                                              host if k == 3 else a.ws.data_ptr(), a.ws.numel(), at(4, k), s) == vk.ARGS, k
    for k in range(7):
        assert lib.vkllm_b200_paged_rope_write(kv, at(0, k), 128, at(1, k), 128, at(2, k), 128, at(3, k), at(4, k), n, 2, 0.0,
                                               host if k == 5 else a.out.data_ptr(), 128, at(6, k), s) == vk.ARGS, k
    t2 = vk.PagedTable(a.d_tab.data_ptr(), a.d_tab.data_ptr(), 4, 1, 2, 16, 4)
    for k in range(9):
        assert lib.vkllm_b200_paged_append(C.byref(t2), *(at(i, k) for i in range(8)), 4, at(8, k), s) == vk.ARGS, k
    for k in range(6):
        assert lib.vkllm_b200_paged_release(C.byref(t2), *(at(i, k) for i in range(6)), s) == vk.ARGS, k
    t2.free_pages = host
    assert lib.vkllm_b200_paged_append(C.byref(t2), *[dev] * 8, 4, dev, s) == vk.ARGS
    torch.cuda.synchronize()
    assert torch.equal(a.out, out0)


@pytest.mark.parametrize("seed", range(24))
def test_attention_of_random_shapes(vk, torch, seed):
    rng = np.random.default_rng(900 + seed)
    HK, group = int(rng.integers(1, 9)), int(rng.choice([1, 2, 3, 5, 8, 12, 16, 20]))
    hd = int(rng.integers(1, 33)) * 8
    n, hi = int(rng.integers(1, 40)), int(2 ** rng.uniform(0, 11))
    lens = [int(x) for x in rng.integers(0, hi + 1, n)]
    a = Attend(vk, torch, lens, HK * group, HK, hd, int(rng.choice([1, 3, 16, 32, 100])), ["f16", "f32"][seed % 2],
               LAYOUTS[int(rng.integers(0, 3))], seed=seed)
    assert a.call() == vk.OK
    a.check(f"{HK} x {group} heads of {hd}, {n} up to {hi}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_keeps_infinities_where_they_are(vk, torch, dtype):
    """An infinite value among the rows that count shows in its element of its heads and sequence alone; a key
    that scores -infinity counts for nothing."""
    a = Attend(vk, torch, [50, 50], 8, 2, 64, 16, dtype, seed=14)
    page = int(a.tab[0, 1])
    a.v[page, 1, 3, 5] = float("inf")
    a.q[:, :512] = a.q[:, :512].abs() + 0.1
    a.k[int(a.tab[1, 2]), 0, 7] = -float("inf")  # key 39 of the second sequence, first key head
    assert a.call() == vk.OK
    torch.cuda.synchronize()
    got = a.out[:2, :512].reshape(2, 8, 64)
    fin = torch.isfinite(got)
    want = torch.ones_like(fin)
    want[0, 4:, 5] = False
    assert torch.equal(fin, want)
    keep = torch.tensor([j for j in range(50) if j != 39], device="cuda")
    ids = torch.from_numpy(a.tab[1, :4].astype(np.int64)).cuda()
    k = a.k[ids].transpose(0, 1).reshape(2, -1, 64)[0, keep].double()
    v = a.v[ids].transpose(0, 1).reshape(2, -1, 64)[0, keep].double()
    p = (a.q[1, :256].double().view(4, 64) @ k.T * a.scale).softmax(-1)
    within(got[1, :4], p @ v, 2.0 ** -11 * (p @ v).abs() + 2.0 ** -16 * (p @ v.abs()) + 2.0 ** -25)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("hd", [4, 12, 36, 68, 100, 196, 252])
def test_fp32_heads_of_an_odd_number_of_pieces(vk, torch, layout, hd):
    """fp32 head sizes that are multiples of 4 and not of 8, through RoPE and attention."""
    test_rope_write(vk, torch, "f32", layout, 6, 3, hd, 37, 7, 10000.0)
    for lens in (LENS["few"], LENS["long"]):
        a = Attend(vk, torch, lens, 10, 2, hd, 7, "f32", layout, seed=hd)
        assert a.call() == vk.OK
        a.check(f"heads of {hd}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_whose_every_score_is_minus_infinity(vk, torch, dtype):
    """Rows of zeros for the heads of a key head that scores so throughout, in one part of a CTA and in parts of
    many; the other key head's are as ever."""
    a = Attend(vk, torch, [50, 40000, 1, 0, 300], 8, 2, 64, 16, dtype, seed=15)
    a.q[:, :512] = a.q[:, :512].abs() + 0.1
    a.k[:, 0, :, 7] = -float("inf")
    assert a.call() == vk.OK
    torch.cuda.synchronize()
    ref, tol = a.reference()
    got = a.out[:5, :512].reshape(5, 8, 64)
    assert int(a.status) == 0 and bool((got[:, :4] == 0).all())
    within(got[:, 4:], ref[:, 4:], tol[:, 4:])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_of_the_most_sequences(vk, torch, dtype):
    """65535 slots of none to three rows, a page each: many sequences for every thread of the division, and
    slots without rows in every CTA's share."""
    n, hd, R = 65535, 64, 3
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v, kv = make_pools(vk, torch, "heads first", n, R, 1, hd, dtype, g)
    table = torch.randperm(n, generator=g, device="cuda").to(torch.int32).view(n, 1)
    lens = torch.randint(0, R + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn((n, hd), generator=g, device="cuda").to(k.dtype)
    out = torch.full_like(q, 7.5)
    ws, status = torch.zeros(vk.PAGED_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    t = vk.PagedTable(table.data_ptr(), None, 1, n, 1, R, n)
    assert vk.lib().vkllm_b200_paged_attention(C.byref(kv), C.byref(t), q.data_ptr(), hd, 1, lens.data_ptr(), hd ** -0.5,
                                               out.data_ptr(), hd, ws.data_ptr(), ws.numel(), status.data_ptr(),
                                               stream(torch)) == vk.OK
    torch.cuda.synchronize()
    assert int(status) == 0
    K, V = k[table[:, 0].long(), 0].double(), v[table[:, 0].long(), 0].double()
    sc = (q.double()[:, None] * K).sum(-1) * hd ** -0.5
    here = torch.arange(R, device="cuda") < lens[:, None]
    p = torch.where(here, sc, -torch.inf).softmax(-1).nan_to_num(0.0)
    ref = (p[..., None] * V).sum(1)
    ds = (hd + 8) * 2 * U * ((q.double()[:, None] * K).abs().sum(-1) * hd ** -0.5).amax(-1)
    far = (sc.amax(-1) - sc.amin(-1)) * 1.4427
    tol = (2 * ds + (far + 4 + R + 64) * 2 * U + 2.0 ** -21)[:, None] * (p[..., None] * V.abs()).sum(1) + out_tol(ref, dtype)
    within(out, ref, tol)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_of_sequences_that_share_pages(vk, torch, dtype):
    """A common beginning held once: both tables name its pages."""
    a = Attend(vk, torch, [100, 90, 70], 8, 2, 64, 16, dtype, seed=31, poison=False)
    a.tab[1, :4], a.tab[2, :4] = a.tab[0, :4], a.tab[0, :4]
    a.d_tab.copy_(i32(torch, a.tab))
    assert a.call() == vk.OK
    a.check()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_shared_beginning_outlives_release_and_append(vk, torch, dtype):
    """A common beginning of three pages is held by one slot; the others hold what is their own, and a table of the
    attention's own names the beginning's pages before theirs. Readers end, others come: nothing of the beginning
    is handed out, and the slots' table stays consistent. The joint table itself is refused by the check."""
    H, HK, hd, R, n, cols = 8, 2, 64, 16, 4, 5
    a = Attend(vk, torch, [48, 20, 33, 7], H, HK, hd, R, dtype, seed=41, poison=False, cols=cols)
    lens, own = [48, 20, 33, 7], a.tab[:, :cols].copy()
    spare = sorted(set(range(a.n_pages)) - {int(p) for s in range(n) for p in own[s, :-(-lens[s] // R)]})
    a.k.copy_(torch.randn(a.k.shape, device="cuda"))
    a.v.copy_(torch.randn(a.v.shape, device="cuda"))
    beginning = own[0, :3].copy()
    d_own, d_lens, count = i32(torch, own), i32(torch, lens), i32(torch, [len(spare)])
    free = i32(torch, spare + [0xeeeeeeee] * (a.n_pages - len(spare)))
    t = vk.PagedTable(d_own.data_ptr(), free.data_ptr(), cols, n, cols, R, a.n_pages)
    z = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
    starts, slots, pos = z(n + 1), z(16), z(16)
    p = lambda x: x.data_ptr()  # noqa: E731

    def check(table, ln, some):
        ht = vk.PagedTable(table.ctypes.data, some.ctypes.data, table.shape[1], n, cols + 3, R, a.n_pages)
        return vk.lib().vkllm_b200_paged_check(C.byref(ht), ln.ctypes.data, len(some), None, None)

    for done, new in (([0] * n, [0, 1, 1, 1]), ([0, 1, 0, 0], [0, 9, 0, 1]), ([0, 0, 1, 1], [0, 1, 5, 2])):
        assert vk.lib().vkllm_b200_paged_release(C.byref(t), p(d_lens), p(i32(torch, done)), p(count), p(d_lens), p(count),
                                                 p(a.status), stream(torch)) == vk.OK
        assert vk.lib().vkllm_b200_paged_append(C.byref(t), p(d_lens), p(i32(torch, new)), p(count), p(d_lens), p(count), p(starts),
                                                p(slots), p(pos), 16, p(a.status), stream(torch)) == vk.OK
        torch.cuda.synchronize()
        lens = [0 if d else l for l, d in zip(lens, done)]
        lens = [l + m for l, m in zip(lens, new)]
        own = u32(d_own).copy()
        assert int(a.status) == 0 and u32(d_lens).tolist() == lens and (own[0, :3] == beginning).all()
        left = u32(free)[:int(count)].copy()
        assert not set(beginning.tolist()) & set(left.tolist())
        wide = np.full((n, cols + 3), 0xffffffff, dtype=np.uint32)
        wide[:, :cols] = own
        assert check(wide, np.asarray(lens, dtype=np.uint32), left) == vk.OK
        a.tab = np.full((n, cols + 3), 0xffffffff, dtype=np.uint32)
        a.tab[0, :cols], a.tab[1:, :3], a.tab[1:, 3:] = own[0], beginning, own[1:]
        a.lens = [lens[0]] + [48 + l for l in lens[1:]]
        assert check(a.tab, np.asarray(a.lens, dtype=np.uint32), left) == vk.ARGS
        a.d_tab, a.d_lens = i32(torch, a.tab), i32(torch, a.lens)
        a.table = vk.PagedTable(p(a.d_tab), None, cols + 3, n, cols + 3, R, a.n_pages)
        a.out.fill_(7.5)
        assert a.call() == vk.OK
        a.check()


def test_attention_says_when_its_workspace_was_not_zero(vk, torch):
    a = Attend(vk, torch, [40000], 8, 2, 64, 16, "f16")
    a.ws.fill_(255)
    assert a.call() == vk.OK
    torch.cuda.synchronize()
    assert int(a.status) == vk.PAGED_BAD_WORKSPACE
    a.ws.zero_()
    a.status.zero_()
    assert a.call() == vk.OK
    a.check()


def test_an_error_of_one_call_is_not_told_again_by_the_next(vk, torch, ctx):
    """A call on the legacy stream while another, blocking stream is being captured is an error of CUDA's (and ends
    that capture). The calls after it are right and say so, the graph ops among them."""
    a = Attend(vk, torch, [20, 3], 2, 2, 64, 16, "f16")
    b = Book(vk, torch, [3], 4, 4, spare=3)
    qkv, q_out = torch.ones((2, 6 * 64), dtype=torch.float16, device="cuda"), a.out.clone()
    pos = i32(torch, [0, 1])
    slots = i32(torch, [0xffffffff, 0xffffffff])
    x = torch.randn((2, 64), device="cuda").half()
    y, rule = torch.zeros_like(x), vk.LogitRules()
    t = vk.tensor_new(ctx, "x", (1, 1, 2, 64), vk.F16)
    vk.put(ctx, t, np.arange(128, dtype=np.float16).reshape(1, 1, 2, 64))
    torch.cuda.synchronize()
    cuda = C.CDLL("libcuda.so.1")

    def fail():
        s, g = C.c_void_p(), C.c_void_p()
        assert cuda.cuStreamCreate(C.byref(s), 0) == 0  # blocking: ordered with the legacy stream
        assert cuda.cuStreamBeginCapture_v2(s, 2) == 0
        err = vk.lib().vkllm_b200_paged_release(C.byref(b.c_table()), b.d_lens.data_ptr(), b.d_lens.data_ptr(),
                                                b.d_count.data_ptr(), b.d_lens.data_ptr(), b.d_count.data_ptr(),
                                                b.status.data_ptr(), None)
        cuda.cuStreamEndCapture(s, C.byref(g))
        assert cuda.cuStreamDestroy_v2(s) == 0
        return err

    own = torch.cuda.Stream()
    with torch.cuda.stream(own):
        for call in (lambda: rope_call(vk, torch, a.kv, qkv, 2, 2, 64, pos, slots, 2, 0.0, q_out, a.status), a.call,
                     lambda: vk.lib().vkllm_b200_logits_apply(C.byref(rule), x.data_ptr(), 64, 2, 64, vk.F16, y.data_ptr(), 64,
                                                              own.cuda_stream)):
            assert fail() == vk.VULKAN
            assert call() == vk.OK
    assert fail() == vk.VULKAN
    node = vk.tensor_new(ctx, "token", (1, 1, 2, 1), vk.U32, op=vk.OP_ARG_MAX, srcs=[t], mapped=True)
    vk.run_op(ctx, node, "vkllm_op_arg_max_init", "vkllm_op_arg_max_run")
    assert vk.fetch(ctx, node).reshape(-1).tolist() == [63, 63]
    torch.cuda.synchronize()
    a.check()
    assert torch.equal(y, x) and int(b.d_lens) == 3
    vk.tensor_free(ctx, node)
    vk.tensor_free(ctx, t)


FIRST_CALLS = """
import ctypes as C, sys
sys.path[:0] = [{pkg!r}]
import torch, vkllm_b200 as vk
z = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device="cuda")
lib, R, n = vk.lib(), 16, 2
table, free, lens, count, new, starts, slots, pos, st, done = (z(n, 4), torch.arange(8, device="cuda", dtype=torch.int32),
    z(n), z(1) + 8, z(n) + 20, z(n + 1), z(5000), z(5000), z(1), z(n))
k, v = z(8, 2, R, 64, t=torch.float16), z(8, 2, R, 64, t=torch.float16)
qkv = torch.randn(5000, 512, device="cuda").half()
q, out = torch.zeros(5000, 256, device="cuda").half(), z(n, 256, t=torch.float16)
ws = z(vk.PAGED_WORKSPACE_BYTES, t=torch.uint8)
x, hist, hl = torch.randn(70, 32000, device="cuda").half(), z(70, 8), z(70) + 8
y = torch.zeros_like(x)
t = vk.PagedTable(table.data_ptr(), free.data_ptr(), 4, n, 4, R, 8)
kv = vk.PagedKV(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), 64, 8, R, 2, 64, vk.F16, 0)
rep = torch.ones(70, device="cuda") * 2
rules = vk.LogitRules(history=hist.data_ptr(), history_lens=hl.data_ptr(), repetition=rep.data_ptr(), history_stride=8)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    p = lambda a: a.data_ptr()
    assert lib.vkllm_b200_paged_release(C.byref(t), p(lens), p(done), p(count), p(lens), p(count), p(st), s) == vk.OK
    assert lib.vkllm_b200_paged_append(C.byref(t), p(lens), p(new), p(count), p(lens), p(count), p(starts), p(slots), p(pos),
                                       5000, p(st), s) == vk.OK
    assert lib.vkllm_b200_paged_rope_write(C.byref(kv), p(qkv), 512, p(qkv) + 512, 512, p(qkv) + 768, 512, p(pos), p(slots), 5000,
                                           4, 0.0, p(q), 256, p(st), s) == vk.OK
    assert lib.vkllm_b200_paged_attention(C.byref(kv), C.byref(t), p(q), 256, 4, p(lens), 0.125, p(out), 256, p(ws), ws.numel(),
                                          p(st), s) == vk.OK
    assert lib.vkllm_b200_logits_apply(C.byref(rules), p(x), 32000, 70, 32000, vk.F16, p(y), 32000, s) == vk.OK
g.replay()
torch.cuda.synchronize()
assert int(st) == 0 and lens.tolist() == [20, 20] and int(count) == 4 and slots[39:41].tolist()[1] == -1
assert bool((y[:, 1:] == x[:, 1:]).all()) and bool((out != 0).any())
w = torch.where(x[:, 0] > 0, x[:, 0] / 2, x[:, 0] * 2)
assert bool((y[:, 0] == w).all())
print("first calls ok")
"""


def test_first_calls_of_a_process_may_be_captured(vk, torch):
    """Nothing has to run before the capture: no allocation, no lazy set-up that a capture forbids."""
    import os
    import subprocess
    import sys

    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vkllm.c_b200")
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(pkg=pkg)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "first calls ok" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_captured_and_replayed_on_two_streams(vk, torch, dtype):
    """Two captured calls with a workspace each, replayed at the same time many times over, give the bits of
    calls made alone; new lengths and queries are read at each replay."""
    calls = [Attend(vk, torch, lens, 16, 4, 128, 16, dtype, seed=i, cols=300) for i, lens in
             enumerate(([4000, 7, 0, 900], [2000] * 6))]
    alone = []
    for a in calls:
        assert a.call() == vk.OK
        torch.cuda.synchronize()
        alone.append(a.out.clone())
    streams = [torch.cuda.Stream() for _ in calls]
    graphs = []
    for a, s in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            assert a.call() == vk.OK
        graphs.append(g)
    for _ in range(20):
        for a in calls:
            a.out.fill_(7.5)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, ref in zip(calls, alone):
            assert torch.equal(a.out, ref)
    a = calls[0]
    a.lens[0], a.lens[3] = 2500, 1  # shorter: what is behind stays where it was
    a.d_lens.copy_(i32(torch, a.lens))
    a.q.copy_(torch.randn_like(a.q))
    a.out.fill_(7.5)
    graphs[0].replay()
    a.check()


# ---- a server's run ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_serving_steps_match_contiguous_attention(vk, torch, dtype):
    """Prompts, decode steps, an ended sequence whose slot takes a new prompt: tables, slots, rotated rows and
    attention over the pages against the same tokens' keys kept contiguously in 64 bits. The decode steps are one captured graph, advanced in place."""
    H, HK, hd, R, n, cols, n_pages, base = 8, 2, 64, 16, 5, 12, 40, 10000.0
    g = torch.Generator(device="cuda").manual_seed(21)
    k, v, kv = make_pools(vk, torch, "heads first", n_pages, R, HK, hd, dtype, g)
    k.fill_(float("nan"))
    v.fill_(float("nan"))
    dt = k.dtype
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    table, free, lens, count, status = z(n, cols) - 1, torch.randperm(n_pages, device="cuda").to(torch.int32), z(n), z(1), z(1)
    count.fill_(n_pages)
    t = vk.PagedTable(table.data_ptr(), free.data_ptr(), cols, n, cols, R, n_pages)
    ws = torch.zeros(vk.PAGED_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    lib = vk.lib()
    kept = [[] for _ in range(n)]  # per sequence: the unrotated (k, v) rows of its tokens
    most = 96
    qkv = torch.zeros((most, (H + 2 * HK) * hd), dtype=dt, device="cuda")
    q_out = torch.zeros((most, H * hd), dtype=dt, device="cuda")
    starts, slots, pos, new, done = z(n + 1), z(most), z(most), z(n), z(n)
    out, last = torch.zeros((n, H * hd), dtype=dt, device="cuda"), torch.zeros((n, H * hd), dtype=dt, device="cuda")

    def step(tokens):
        assert lib.vkllm_b200_paged_release(C.byref(t), lens.data_ptr(), done.data_ptr(), count.data_ptr(), lens.data_ptr(),
                                            count.data_ptr(), status.data_ptr(), stream(torch)) == vk.OK
        assert lib.vkllm_b200_paged_append(C.byref(t), lens.data_ptr(), new.data_ptr(), count.data_ptr(), lens.data_ptr(),
                                           count.data_ptr(), starts.data_ptr(), slots.data_ptr(), pos.data_ptr(), tokens,
                                           status.data_ptr(), stream(torch)) == vk.OK
        assert rope_call(vk, torch, kv, qkv, H, HK, hd, pos, slots, tokens, base, q_out, status) == vk.OK

    def attend(q):
        assert lib.vkllm_b200_paged_attention(C.byref(kv), C.byref(t), q.data_ptr(), q.stride(0), H, lens.data_ptr(),
                                              hd ** -0.5, out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(),
                                              status.data_ptr(), stream(torch)) == vk.OK

    def feed(counts, ended=()):
        """New rows for the step's tokens, and the same kept on the side."""
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda").to(dt))
        new.copy_(i32(torch, counts))
        done.copy_(i32(torch, [int(s in ended) for s in range(n)]))
        at = 0
        for s, m in enumerate(counts):
            if s in ended:
                kept[s] = []
            for _ in range(m):
                kept[s].append(qkv[at, H * hd:].double().view(2, HK, hd).clone())
                at += 1

    w = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    freq = base ** (-2 * w / hd)

    def turn(x, p):  # [..., hd] at position p
        a, b = x[..., 0::2], x[..., 1::2]
        c, s = torch.cos(p * freq), torch.sin(p * freq)
        return torch.stack([c * a - s * b, s * a + c * b], -1).flatten(-2)

    def compare(rows):
        torch.cuda.synchronize()
        assert int(status) == 0
        assert u32(lens).tolist() == [len(x) for x in kept]
        for s in range(n):
            if not kept[s]:
                assert bool((out[s] == 0).all())
                continue
            K = torch.stack([turn(x[0], float(i)) for i, x in enumerate(kept[s])], 1)
            V = torch.stack([x[1] for x in kept[s]], 1)
            q = turn(rows[s].double().view(H, hd), float(len(kept[s]) - 1)).view(HK, H // HK, hd)
            sc = q @ K.transpose(1, 2) * hd ** -0.5
            p = sc.softmax(-1)
            # rotated rows are off by 2^-20 (|x| + |y|) of a pair, 2^-19 of its length, and by half a step of their type
            e = 2.0 ** -11 if dtype == "f16" else U
            ds = ((q.abs() @ K.abs().transpose(1, 2)).amax(-1, keepdim=True) * hd ** -0.5) * (2 * e + (hd + 8) * 2 * U)
            ds = ds + 2.0 ** -18 * hd ** -0.5 * q.norm(dim=-1, keepdim=True) * K.norm(dim=-1).amax()
            ref = p @ V
            tol = (2 * ds + 2.0 ** -16) * 1.1 * (p @ V.abs()) + out_tol(ref, dtype)
            within(out[s].view(HK, H // HK, hd), ref, tol, f"sequence {s}")

    def last_rows(m):  # the row of each sequence's last token in the packed step
        return [max(0, int(x) - 1) for x in u32(starts)[1:]]

    feed([20, 1, 0, 33, 16])
    step(most)
    torch.cuda.synchronize()
    idx = last_rows(n)
    last.copy_(q_out[idx])
    attend(last)
    rows = qkv[idx, :H * hd].clone()
    compare(rows)
    assert u32(slots)[70:].tolist() == [vk.NO_SLOT] * (most - 70)
    feed([0, 3, 40, 10, 0], ended=(3,))
    step(most)
    torch.cuda.synchronize()
    idx = last_rows(n)
    torch.cuda.synchronize()
    assert u32(lens).tolist() == [20, 4, 40, 10, 16]
    # decode steps: one token each, one graph
    feed([1] * n)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(n)
        attend(q_out)
    for i in range(20):
        if i:
            feed([1] * n)
        graph.replay()
        compare(qkv[:n, :H * hd])
    assert int(u32(count)[0]) == n_pages - sum(-(-len(x) // R) for x in kept)
    # what the tables say at the end is consistent, page by page
    tab, ln, fr = u32(table).copy(), u32(lens).copy(), u32(free).copy()
    ht = vk.PagedTable(tab.ctypes.data, fr.ctypes.data, cols, n, cols, R, n_pages)
    assert lib.vkllm_b200_paged_check(C.byref(ht), ln.ctypes.data, int(u32(count)[0]), None, None) == vk.OK
