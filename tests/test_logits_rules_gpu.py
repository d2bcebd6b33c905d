"""vkllm_b200_logits_apply on the GPU against its definition in 64 bits (loops over rows and ids).

Tolerance: the rules are at most 4 + b fp32 operations on values of magnitude M = |x| max(r, 1/r) +
|frequency count| + |presence| + sum |biases| (b biases of the id), each off by half a step, 2^-24 M;
then half a step of the output's type (fp16: 2^-11 of the value, 2^-25 below its normal range)."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def case(rows, vocab, past, seed, dtype, bias=5, pad=0):
    rng = np.random.default_rng(seed)
    dt = np.float16 if dtype == "f16" else np.float32
    c = {"x": (rng.standard_normal((rows, vocab + pad)) * 5).astype(dt), "vocab": vocab}
    # repeated ids, ids at the ends, ids past the vocabulary
    pick = np.concatenate([rng.integers(0, vocab, max(1, past // 2)), [0, vocab - 1, vocab, vocab + 7, 0xffffffff]])
    c["history"] = rng.choice(pick, (rows, past + 3)).astype(np.uint32)
    c["prompt_lens"] = rng.integers(0, past + 1, rows).astype(np.uint32)
    c["history_lens"] = rng.integers(0, past + 1, rows).astype(np.uint32)  # some shorter than the prompt
    c["history_lens"][0] = past
    c["prompt_lens"][0] = past // 3
    for name in ("repetition", "frequency", "presence"):
        c[name] = (rng.random(rows) + (0.5 if name == "repetition" else -0.3)).astype(np.float32)
    each = rng.integers(0, bias + 1, rows)
    each[-1] = bias
    c["bias_starts"] = np.concatenate([[2], 2 + np.cumsum(each)]).astype(np.uint32)  # the list need not begin at 0
    c["bias_ids"] = rng.choice(pick, 2 + each.sum()).astype(np.uint32)
    c["bias_values"] = (rng.standard_normal(2 + each.sum()) * 3).astype(np.float32)
    words = -(-vocab // 32) + 1
    c["mask"] = rng.integers(0, 2 ** 32, (rows, words), dtype=np.uint64).astype(np.uint32)
    c["mask"][rows // 2] = 0  # nothing is allowed in this row
    if rows > 2:
        c["mask"][1] = 0xffffffff
    return c


def reference(c, on):
    x = c["x"].astype(np.float64)[:, :c["vocab"]]
    tol_m, nb = np.abs(x), np.zeros_like(x)
    for r in range(len(x)):
        V = c["vocab"]
        if "history" in on:
            n = min(int(c["history_lens"][r]), c["history"].shape[1])
            prompt = int(c["prompt_lens"][r]) if "prompt_lens" in on else 0
            ids = c["history"][r, :n]
            out, count = np.unique(ids[prompt:], return_counts=True)
            count = dict(zip(out.tolist(), count.tolist()))
            for i in set(ids.tolist()):
                if i >= V:
                    continue
                if "repetition" in on:
                    f = float(c["repetition"][r])
                    x[r, i] = x[r, i] / f if x[r, i] > 0 else x[r, i] * f
                    tol_m[r, i] *= max(f, 1 / f)
                if i in count:
                    fc = float(c["frequency"][r]) * count[i] if "frequency" in on else 0.0
                    pr = float(c["presence"][r]) if "presence" in on else 0.0
                    x[r, i] -= fc + pr
                    tol_m[r, i] += abs(fc) + abs(pr)
        if "bias_starts" in on:
            for e in range(c["bias_starts"][r], c["bias_starts"][r + 1]):
                i = int(c["bias_ids"][e])
                if i < V:
                    x[r, i] += float(c["bias_values"][e])
                    tol_m[r, i] += abs(float(c["bias_values"][e]))
                    nb[r, i] += 1
        if "mask" in on:
            bits = (c["mask"][r][:, None] >> np.arange(32, dtype=np.uint32)) & 1
            x[r, bits.reshape(-1)[:V] == 0] = -np.inf
    return x, (4 + nb) * U * tol_m


ALL = ["history", "prompt_lens", "history_lens", "repetition", "frequency", "presence", "bias_starts", "bias_ids",
       "bias_values", "mask"]
RULES = {"all": ALL, "nothing": [], "mask": ["mask"], "bias": ["bias_starts", "bias_ids", "bias_values"],
         "repetition": ["history", "history_lens", "repetition"],
         "counts": ["history", "history_lens", "prompt_lens", "frequency", "presence"]}


def run(vk, torch, c, on, dtype, x, out, vocab=None):
    dev = {k: torch.from_numpy(c[k].view(np.int32) if c[k].dtype == np.uint32 else c[k]).cuda() for k in on}
    r = vk.LogitRules(**{k: t.data_ptr() for k, t in dev.items()}, history_stride=c["history"].shape[1],
                      mask_stride=c["mask"].shape[1])
    s = torch.cuda.current_stream().cuda_stream
    err = vk.lib().vkllm_b200_logits_apply(C.byref(r), x.data_ptr(), x.stride(0), x.shape[0], c["vocab"],
                                           vk.F16 if dtype == "f16" else vk.F32, out.data_ptr(), out.stride(0), s)
    torch.cuda.synchronize()
    return err


def close(got, ref, tol, dtype):
    fin = np.isfinite(ref)
    assert np.array_equal(fin, np.isfinite(got)) and (got[~fin] == ref[~fin]).all()
    half = np.abs(ref[fin]) * 2.0 ** -11 + 2.0 ** -25 if dtype == "f16" else np.abs(ref[fin]) * U
    d = np.abs(got[fin] - ref[fin])
    bad = d > tol[fin] + half
    assert not bad.any(), (int(bad.sum()), float((d / (tol[fin] + half)).max()))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("on", list(RULES))
@pytest.mark.parametrize("rows,vocab,past,bias,pad", [(1, 1, 1, 1, 0), (1, 32000, 700, 8, 0), (3, 31, 40, 3, 2),
                                                      (5, 4097, 300, 40, 1), (2, 8192, 5000, 300, 8),
                                                      (64, 1003, 20, 2, 0), (7, 100003, 900, 33, 3),
                                                      (3, 20011, 9000, 40, 1), (2, 40, 6144, 0, 0), (2, 9000, 6100, 70, 0),
                                                      (200, 5000, 60, 4, 0), (160, 4099, 4000, 3, 1)])
def test_rules(vk, dtype, on, rows, vocab, past, bias, pad):
    import torch

    c = case(rows, vocab, past, rows + vocab, dtype, bias, pad)
    x = torch.from_numpy(c["x"]).cuda()
    out = torch.full((rows + 1, vocab + pad + 5), 9.0, dtype=x.dtype, device="cuda")
    assert run(vk, torch, c, RULES[on], dtype, x, out) == vk.OK
    ref, tol = reference(c, RULES[on])
    close(out[:rows, :vocab].cpu().numpy().astype(np.float64), ref, tol, dtype)
    assert bool((out[rows:] == 9.0).all()) and bool((out[:, vocab:] == 9.0).all())  # left as they were
    if on == "nothing":
        assert torch.equal(out[:rows, :vocab], x[:, :vocab])
    # in place: the same bits, and nothing behind the vocabulary
    y = x.clone()
    assert run(vk, torch, c, RULES[on], dtype, y, y) == vk.OK
    assert torch.equal(y[:, :vocab], out[:rows, :vocab])
    assert torch.equal(y[:, vocab:], x[:, vocab:])


@pytest.mark.parametrize("on", ["all", "mask", "nothing"])
def test_the_most_rows(vk, on):
    import torch

    c = case(65535, 23, 5, 6, "f16", 2, 1)
    x = torch.from_numpy(c["x"]).cuda()
    out = torch.full((65535, 24), 9.0, dtype=x.dtype, device="cuda")
    assert run(vk, torch, c, RULES[on], "f16", x, out) == vk.OK
    ref, tol = reference(c, RULES[on])
    close(out[:, :23].cpu().numpy().astype(np.float64), ref, tol, "f16")
    assert bool((out[:, 23:] == 9.0).all())


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("shift_in,shift_out", [(0, 0), (1, 1), (3, 3), (1, 2), (5, 0)])
def test_rows_at_every_alignment(vk, dtype, shift_in, shift_out):
    """Rows whose first element is on no vector's boundary, the same for both or not."""
    import torch

    c = case(4, 2501, 200, 77, dtype)
    buf = torch.zeros(4 * 2600 + 64, dtype=torch.float16 if dtype == "f16" else torch.float32, device="cuda")
    x = buf[shift_in:shift_in + 4 * 2507].view(4, 2507)[:, :2501]
    x.copy_(torch.from_numpy(c["x"]))
    out = torch.full((4 * 2600 + 64,), 9.0, dtype=x.dtype, device="cuda")
    o = out[shift_out:shift_out + 4 * 2509].view(4, 2509)
    assert run(vk, torch, c, ALL, dtype, x, o) == vk.OK
    ref, tol = reference(c, ALL)
    close(o[:, :2501].cpu().numpy().astype(np.float64), ref, tol, dtype)
    assert bool((o[:, 2501:] == 9.0).all()) and bool((out[:shift_out] == 9.0).all())


def test_biases_of_one_id_add_in_the_order_of_the_list(vk):
    """1e8, 1, -1e8 in fp32: the order shows. 70 entries of one id, beyond one warp's load."""
    import torch

    rng = np.random.default_rng(3)
    values = (rng.standard_normal(70) * 10.0 ** rng.integers(-3, 8, 70)).astype(np.float32)
    c = case(1, 50, 4, 1, "f32")
    c["x"][:] = 0
    c["bias_starts"] = np.array([0, 70], dtype=np.uint32)
    c["bias_ids"], c["bias_values"] = np.full(70, 13, dtype=np.uint32), values
    x = torch.from_numpy(c["x"]).cuda()
    out = torch.zeros_like(x)
    assert run(vk, torch, c, RULES["bias"], "f32", x, out) == vk.OK
    want = np.float32(0)
    for v in values:
        want = np.float32(want + v)
    assert float(out[0, 13]) == float(want)


def test_a_row_whose_biases_end_before_they_start_has_none(vk):
    """Starts that fall, all of them within the lists: rows 1 and 3 have no biases, the others theirs."""
    import torch

    c = case(5, 300, 4, 2, "f32")
    c["bias_starts"] = np.array([6, 9, 2, 8, 0, 4], dtype=np.uint32)
    c["bias_ids"] = np.arange(12, dtype=np.uint32) * 7
    c["bias_values"] = np.arange(1, 13).astype(np.float32)
    x = torch.from_numpy(c["x"]).cuda()
    out = torch.zeros_like(x)
    assert run(vk, torch, c, RULES["bias"], "f32", x, out) == vk.OK
    ref, tol = reference(c, RULES["bias"])
    assert (ref[[1, 3]] == c["x"][[1, 3]]).all() and (ref[[0, 2, 4]] != c["x"][[0, 2, 4]]).any(1).all()
    close(out.cpu().numpy().astype(np.float64), ref, tol, "f32")


def test_one_id_over_and_over(vk):
    """A history of one repeated id, in the prompt and after it, that is also biased."""
    import torch

    c = case(3, 40000, 3000, 8, "f32")
    c["history"][:], c["history_lens"][:] = 123, [3000, 2999, 1]
    c["prompt_lens"][:] = [1000, 2999, 0]
    c["bias_ids"][:] = 123
    c["mask"][:] = 0xffffffff
    x = torch.from_numpy(c["x"]).cuda()
    out = torch.zeros_like(x)
    assert run(vk, torch, c, ALL, "f32", x, out) == vk.OK
    ref, tol = reference(c, ALL)
    close(out.cpu().numpy().astype(np.float64), ref, tol, "f32")


@pytest.mark.parametrize("rows", [2, 70])
@pytest.mark.parametrize("in_place", [False, True])
def test_captured_and_replayed_with_new_tokens(vk, rows, in_place):
    """One captured call (few rows: one kernel; more: two, the second launched early) replayed while the
    history, its lengths and the logits change, as a decoding server's do."""
    import torch

    c = case(rows, 32000, 400, 21, "f16")
    dev = {k: torch.from_numpy(c[k].view(np.int32) if c[k].dtype == np.uint32 else c[k]).cuda() for k in ALL}
    r = vk.LogitRules(**{k: t.data_ptr() for k, t in dev.items()}, history_stride=c["history"].shape[1],
                      mask_stride=c["mask"].shape[1])
    x = torch.from_numpy(c["x"]).cuda()
    out = x if in_place else torch.zeros_like(x)
    fresh = x.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.copy_(fresh)
        assert vk.lib().vkllm_b200_logits_apply(C.byref(r), x.data_ptr(), 32000, rows, 32000, vk.F16, out.data_ptr(), 32000,
                                                torch.cuda.current_stream().cuda_stream) == vk.OK
    rng = np.random.default_rng(4)
    for _ in range(4):
        c["x"] = (rng.standard_normal((rows, 32000)) * 5).astype(np.float16)
        c["history_lens"] = np.minimum(c["history_lens"] + 1, 400).astype(np.uint32)
        c["history"][np.arange(rows), c["history_lens"] - 1] = rng.integers(0, 32000, rows)
        fresh.copy_(torch.from_numpy(c["x"]))
        dev["history"].copy_(torch.from_numpy(c["history"].view(np.int32)))
        dev["history_lens"].copy_(torch.from_numpy(c["history_lens"].view(np.int32)))
        g.replay()
        torch.cuda.synchronize()
        ref, tol = reference(c, ALL)
        close(out.cpu().numpy().astype(np.float64), ref, tol, "f16")


def test_memory_that_is_not_the_devices_is_refused(vk):
    import torch

    c = case(1, 64, 4, 1, "f16")
    dev = {k: torch.from_numpy(c[k].view(np.int32) if c[k].dtype == np.uint32 else c[k]).cuda() for k in ALL}
    x = torch.from_numpy(c["x"]).cuda()
    host = torch.zeros(4096, dtype=torch.float16).pin_memory().data_ptr()
    for bad in ALL + ["logits", "out"]:
        r = vk.LogitRules(**{k: host if k == bad else t.data_ptr() for k, t in dev.items()}, history_stride=7, mask_stride=3)
        assert vk.lib().vkllm_b200_logits_apply(C.byref(r), host if bad == "logits" else x.data_ptr(), 64, 1, 64, vk.F16,
                                                host if bad == "out" else x.data_ptr(), 64, None) == vk.ARGS, bad


def test_infinities_and_no_numbers(vk):
    """-infinity stays, no number stays one where it is allowed, the mask wins over both."""
    import torch

    c = case(2, 64, 4, 1, "f16")
    c["x"][:] = 1
    c["x"][:, 3], c["x"][:, 4], c["x"][:, 5] = -np.inf, np.nan, np.inf
    c["history"][:, :4], c["history_lens"][:], c["prompt_lens"][:] = [3, 4, 5, 5], 4, 0
    c["mask"][0], c["mask"][1] = 0xffffffff, 0xffffffff ^ (1 << 4) ^ (1 << 5)
    c["bias_starts"][:] = 0
    x = torch.from_numpy(c["x"]).cuda()
    out = torch.zeros_like(x)
    assert run(vk, torch, c, ALL, "f16", x, out) == vk.OK
    got = out.cpu().numpy()
    assert got[0, 3] == -np.inf and np.isnan(got[0, 4]) and got[0, 5] == np.inf
    assert got[1, 3] == -np.inf and got[1, 4] == -np.inf and got[1, 5] == -np.inf


def test_rules_then_arg_max_gives_the_allowed_token(vk, ctx):
    """As a server uses it: the rules, in place on the logits tensor of a graph node, before VKLLM_OP_ARG_MAX."""
    import torch

    rows, vocab = 6, 32000
    c = case(rows, vocab, 300, 5, "f16")
    c["mask"][rows // 2] = 0
    c["mask"][rows // 2, 700] = 1 << 9  # one id is allowed in this row
    t = vk.tensor_new(ctx, "logits", (1, 1, rows, vocab), vk.F16)
    vk.put(ctx, t, c["x"].reshape(1, 1, rows, vocab))
    dev = {k: torch.from_numpy(c[k].view(np.int32) if c[k].dtype == np.uint32 else c[k]).cuda() for k in ALL}
    torch.cuda.synchronize()
    r = vk.LogitRules(**{k: v.data_ptr() for k, v in dev.items()}, history_stride=c["history"].shape[1],
                      mask_stride=c["mask"].shape[1])
    p = t.contents.data.dev
    assert vk.lib().vkllm_b200_logits_apply(C.byref(r), p, vocab, rows, vocab, vk.F16, p, vocab, ctx.stream) == vk.OK
    node = vk.tensor_new(ctx, "token", (1, 1, rows, 1), vk.U32, op=vk.OP_ARG_MAX, srcs=[t], mapped=True)
    vk.run_op(ctx, node, "vkllm_op_arg_max_init", "vkllm_op_arg_max_run")
    got = vk.fetch(ctx, node).reshape(-1)
    ref, tol = reference(c, ALL)
    for i in range(rows):
        best = ref[i].max()
        assert ref[i][got[i]] >= best - 2 * (abs(best) * 2.0 ** -11 + tol[i].max()), i
    assert got[rows // 2] == 700 * 32 + 9
    vk.tensor_free(ctx, node)
    vk.tensor_free(ctx, t)
