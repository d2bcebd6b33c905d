"""The documented serving loop, compiled as it stands in the integration notes: on the CPU that it compiles, on the
GPU what it computes for steps in which slots wait, decode, get prompts, end and start again, called and replayed."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def loop(vk, tmp_path_factory):
    import build

    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    at = text.index('#include "vkllm_b200_paged.h"')
    d = tmp_path_factory.mktemp("loop")
    src, so = str(d / "loop.cu"), str(d / "loop.so")
    with open(src, "w") as f:
        f.write(text[at:text.index("```", at)])
    r = subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                        "-o", so, src, vk.LIB_PATH, "-Xlinker", "-rpath," + os.path.dirname(vk.LIB_PATH)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(so)
    lib.server_step.argtypes = [C.c_void_p, C.c_void_p]
    lib.server_rules.argtypes = [C.c_void_p, C.c_void_p, C.c_uint32, C.c_uint32, C.c_void_p]
    return lib


def test_the_documented_loop_compiles(loop):
    assert loop.server_step and loop.server_rules


def server(vk):
    class Server(C.Structure):
        _fields_ = [("slots", vk.PagedTable), ("rows", vk.PagedTable), ("kv", C.c_void_p), ("layers", C.c_uint32),
                    ("heads", C.c_uint32), ("max_tokens", C.c_uint32)] + [
                        (n, C.c_void_p) for n in ("lens", "n_free", "n_new", "done", "starts", "token_slots", "positions",
                                                  "row_lens", "qkv", "q_rot", "out", "workspace", "status")] + [("scale", C.c_float)]
    return Server()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("captured", [False, True])
def test_the_documented_loop_with_waiting_slots(vk, loop, dtype, captured):
    """Every token's attention, prompts' tokens included, against the rows of its own sequence in 64 bits. Tolerance: a
    rotated element is off by 2^-20 (|a| + |b|) of its pair and by half a step e of its type (fp16 2^-11, fp32 2^-24), so
    a score by (2 e + 2^-18 + (head_dim + 8) 2^-23) * scale * |q| |k|, which changes the weights by at most twice that; the
    rest as for the attention alone, and half a step of the output."""
    import torch

    H, HK, hd, R, n, cols, n_pages, most = 8, 2, 64, 16, 6, 9, 48, 64
    dt = torch.float16 if dtype == "f16" else torch.float32
    g = torch.Generator(device="cuda").manual_seed(3)
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    pools = [torch.full((n_pages, HK, R, hd), float("nan"), dtype=dt, device="cuda") for _ in range(4)]
    kv = (vk.PagedKV * 2)(*[vk.PagedKV(k.data_ptr(), v.data_ptr(), HK * R * hd, R * hd, hd, n_pages, R, HK, hd,
                                       vk.F16 if dtype == "f16" else vk.F32, 0) for k, v in (pools[:2], pools[2:])])
    t = {k: z(m) for k, m in dict(lens=n, n_free=1, n_new=n, done=n, starts=n + 1, token_slots=most, positions=most,
                                  row_lens=most, status=1).items()}
    t["n_free"].fill_(n_pages)
    table, rows, free = z(n, cols) - 1, z(most, cols) - 1, torch.randperm(n_pages, device="cuda").to(torch.int32)
    t["qkv"] = torch.zeros((most, (H + 2 * HK) * hd), dtype=dt, device="cuda")
    t["q_rot"], t["out"] = (torch.zeros((most, H * hd), dtype=dt, device="cuda") for _ in range(2))
    t["workspace"] = torch.zeros(vk.PAGED_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    s = server(vk)
    s.slots = vk.PagedTable(table.data_ptr(), free.data_ptr(), cols, n, cols, R, n_pages)
    s.rows = vk.PagedTable(rows.data_ptr(), None, cols, most, cols, R, n_pages)
    s.kv, s.layers, s.heads, s.max_tokens, s.scale = C.addressof(kv), 2, H, most, hd ** -0.5
    for k, v in t.items():
        setattr(s, k, v.data_ptr())

    def step():
        assert loop.server_step(C.byref(s), torch.cuda.current_stream().cuda_stream) == vk.OK

    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    w = torch.arange(hd // 2, device="cuda", dtype=torch.float64)

    def turn(x, p):  # [tokens, heads, hd] at positions p
        th = p[:, None, None] * 10000.0 ** (-2 * w / hd)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([th.cos() * a - th.sin() * b, th.sin() * a + th.cos() * b], -1).flatten(-2)

    e = 2.0 ** -11 if dtype == "f16" else 2.0 ** -24
    kept = [torch.zeros((0, (H + 2 * HK) * hd), dtype=torch.float64, device="cuda") for _ in range(n)]
    steps = [([5, 0, 1, 20, 0, 0], []), ([1, 0, 1, 1, 0, 0], []), ([0, 7, 0, 1, 0, 1], []), ([1, 1, 0, 0, 3, 0], [3]),
             ([1, 0, 1, 7, 0, 1], []), ([0] * 6, [0]), ([40, 1, 1, 1, 1, 1], []), ([1] * 6, []), ([0, 0, 0, 0, 0, 1], []),
             ([17, 0, 0, 2, 16, 0], [1, 2])]
    for counts, ended in steps:
        t["qkv"].copy_(torch.randn(t["qkv"].shape, generator=g, device="cuda").to(dt))
        t["n_new"].copy_(torch.tensor(counts, dtype=torch.int32))
        t["done"].copy_(torch.tensor([int(i in ended) for i in range(n)], dtype=torch.int32))
        t["out"].fill_(7.5)
        graph.replay() if captured else step()
        torch.cuda.synchronize()
        assert int(t["status"]) == 0
        at, got = 0, t["out"].double()
        for i, m in enumerate(counts):
            if i in ended:
                kept[i] = kept[i][:0]
            kept[i] = torch.cat([kept[i], t["qkv"][at:at + m].double()])
            have = len(kept[i])
            if m:
                p = torch.arange(have, device="cuda", dtype=torch.float64)
                q = turn(kept[i][-m:, :H * hd].view(m, H, hd), p[-m:])
                k = turn(kept[i][:, H * hd:(H + HK) * hd].view(have, HK, hd), p).repeat_interleave(H // HK, 1)
                v = kept[i][:, (H + HK) * hd:].view(have, HK, hd).repeat_interleave(H // HK, 1)
                sc = torch.einsum("mhd,jhd->hmj", q, k) * s.scale
                later = p[None, None, :] > p[-m:, None]
                pr = sc.masked_fill(later, -torch.inf).softmax(-1)
                ref = torch.einsum("hmj,jhd->mhd", pr, v)
                ds = (2 * e + 2.0 ** -18 + (hd + 8) * 2.0 ** -23) * s.scale * q.norm(dim=-1).amax() * k.norm(dim=-1).amax()
                tol = (2 * ds + 2.0 ** -16) * 1.1 * torch.einsum("hmj,jhd->mhd", pr, v.abs()) + e * ref.abs() + 2.0 ** -25
                d = (got[at:at + m].view(m, H, hd) - ref).abs()
                assert bool((d <= tol).all()), (counts, i, float((d / tol).max()))
            at += m
        assert bool((got[at:] == 0).all())  # rows without a token
        assert t["lens"].tolist() == [len(x) for x in kept]
        assert t["row_lens"][at:].tolist() == [0] * (most - at)


@pytest.mark.gpu
def test_the_documented_rules(vk, loop):
    import torch

    x = torch.randn((3, 100), device="cuda").half()
    mask = torch.tensor([[-1, 0, 1 << 5, 0]] * 3, dtype=torch.int32, device="cuda")
    r, y = vk.LogitRules(mask=mask.data_ptr(), mask_stride=4), x.clone()
    assert loop.server_rules(C.byref(r), y.data_ptr(), 3, 100, torch.cuda.current_stream().cuda_stream) == vk.OK
    torch.cuda.synchronize()
    keep = np.isin(np.arange(100), list(range(32)) + [69])
    assert torch.equal(y[:, keep], x[:, keep]) and bool((y[:, ~keep] == -torch.inf).all())
