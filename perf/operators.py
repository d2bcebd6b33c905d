"""Measured cases of the paged serving operators: page tables and slot maps built on the GPU, RoPE with
the key and value rows written into a paged cache, attention of one new token a sequence over that
cache, and penalties, biases and grammar masks on logits.

`run` computes each operator in a plain form (elementary torch operations in 32 bits, rounded once at
the end) or, with `own` set, through the library's entry points. `exact` restates the definitions in
64 bits. Sequence slots, pages, cache slots and token ids are 32-bit unsigned in the library; int32
tensors hold the same bits here (0xffffffff, "no slot", reads as -1).
"""
import ctypes
import functools
import math
import struct

import torch

own = False

DTYPES = {"f16": torch.float16, "f32": torch.float32}
CODES = {"f16": 2, "f32": 1}  # vkllm_dtype_float16, vkllm_dtype_float32
WORKSPACE_BYTES = 16 << 20  # VKLLM_B200_PAGED_WORKSPACE_BYTES


# ---- cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of 64 sequences (the batched decode's size): three ended, each other one adds a token
        tables("tables decode 64", seqs=64, page_rows=16, cols=256, max_len=4095, new_hi=1, max_tokens=64, done=3),
        # a step that mixes long prompts with decoding over many slots: the slot map is what takes the time
        tables("tables prefill 512", seqs=512, page_rows=32, cols=256, max_len=4000, new_hi=450, max_tokens=131072,
               done=40),
        # decode step of the batched workload: 64 tokens, 32 heads of 128, fused Q/K/V rows
        rope("rope write decode", "f16", tokens=64, heads=32, kv_heads=32, head_dim=128, page_rows=16, pages=256,
             rows_first=False, skip=0, far=4096),
        # prefill of one 2048-token prompt at 40 heads, the widest model of the benchmark
        rope("rope write prefill", "f16", tokens=2048, heads=40, kv_heads=40, head_dim=128, page_rows=64, pages=64,
             rows_first=False, skip=0, far=2048),
        # the tiny model's head size in 32 bits: odd count, pages that are no power of two, padded tokens at
        # the end, far positions, row-major pages
        rope("rope write f32 odd", "f32", tokens=777, heads=12, kv_heads=6, head_dim=48, page_rows=24, pages=80,
             rows_first=True, skip=9, far=200000),
        # one short sequence of the tiny model: latency alone
        attention("attention one short", "f16", seqs=1, heads=6, kv_heads=6, head_dim=48, page_rows=16, min_len=96,
                  max_len=96, rows_first=False),
        # the batched decode workload: 64 sequences of 32 heads, each head with its own keys
        attention("attention batch 64", "f16", seqs=64, heads=32, kv_heads=32, head_dim=128, page_rows=16, min_len=128,
                  max_len=640, rows_first=False),
        # shared key heads, ragged lengths from none to 8192, pages of 64 rows in row-major order
        attention("attention shared ragged", "f16", seqs=48, heads=64, kv_heads=8, head_dim=128, page_rows=64,
                  min_len=0, max_len=8192, rows_first=True),
        # one very long sequence: the work has to be split over its length
        attention("attention one long", "f16", seqs=1, heads=32, kv_heads=8, head_dim=128, page_rows=16,
                  min_len=131072, max_len=131072, rows_first=False),
        # a 32-bit cache with an odd head size and pages that are no power of two
        attention("attention f32 odd", "f32", seqs=24, heads=16, kv_heads=4, head_dim=80, page_rows=24, min_len=1,
                  max_len=2000, rows_first=False),
        # one sequence's logits over the benchmark's vocabulary, with its 512-token prompt and 256 new tokens
        logits("logits one", "f16", rows=1, vocab=32000, prompt=512, output=256, biases=8, masked=0),
        # a large batch over a large odd vocabulary: penalties, biases and a grammar mask in every row
        logits("logits batch", "f16", rows=256, vocab=100003, prompt=1024, output=1024, biases=64, masked=1),
    ]


def tables(name, **k):
    return {"name": name, "op": "tables", **k}


def rope(name, dtype, **k):
    return {"name": name, "op": "rope", "dtype": dtype, "base": 10000.0, **k}


def attention(name, dtype, **k):
    return {"name": name, "op": "attention", "dtype": dtype, **k}


def logits(name, dtype, **k):
    return {"name": name, "op": "logits", "dtype": dtype, **k}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "rope", "attention", "attention", "logits"])
    page_rows = rng.choice([16, 16, 32, 64, 128, 24, 7])
    dtype = rng.choice(["f16", "f16", "f32"])
    if op == "tables":
        seqs, new_hi = _log(rng, 1, 2000), _log(rng, 1, 500)
        new_hi = min(new_hi, 131072 // seqs)
        cols = rng.randint(-(-(new_hi + 1) // page_rows) + 1, max(200, new_hi))
        c = tables("", seqs=seqs, page_rows=page_rows, cols=cols, max_len=cols * page_rows - new_hi, new_hi=new_hi,
                   max_tokens=seqs * new_hi + rng.randint(0, 40), done=rng.randint(0, seqs // 4))
    else:
        kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 16, 32])
        group = rng.choice([1, 1, 2, 4, 7, 8, 16] if kv_heads < 8 else [1, 2, 4])
        head_dim = rng.choice([64, 128, 128, 128, 48, 80, 96, 192, 256])
        row = kv_heads * head_dim
        if op == "rope":
            most = max(4, min(8192, (2048 * 40 * 384) // ((kv_heads * group + 2 * kv_heads) * head_dim)))
            tokens = _log(rng, 1, most // (1 if dtype == "f16" else 2))
            c = rope("", dtype, tokens=tokens, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                     page_rows=page_rows, pages=tokens // page_rows + rng.randint(2, 40),
                     rows_first=rng.random() < 0.5, skip=rng.randint(0, tokens // 3), far=_log(rng, 512, 200000))
        elif op == "attention":
            seqs = _log(rng, 1, 200)
            most = 150_000_000 // (1 if dtype == "f16" else 2) // (seqs * row)
            hi = _log(rng, 1, max(1, min(131072, most)))
            c = attention("", dtype, seqs=seqs, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                          page_rows=page_rows, min_len=rng.choice([0, 1, hi // 2, hi]), max_len=hi,
                          rows_first=rng.random() < 0.5)
        else:
            vocab = _log(rng, 300, 160000)
            rows = _log(rng, 1, min(400, 20_000_000 // vocab))
            c = logits("", dtype, rows=rows, vocab=vocab, prompt=_log(rng, 1, 3000), output=_log(rng, 1, 2000),
                       biases=_log(rng, 1, min(200, vocab // 2)), masked=rng.choice([0, 1]))
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(g, lo, hi, shape):
    """Uniform 32-bit integers of lo .. hi inclusive."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _lengths(g, n, lo, hi):
    """Sequence lengths of lo .. hi; the ends of the range are among them."""
    x = _ints(g, lo, hi, (n,))
    x[0] = hi
    if n > 1:
        x[n // 2] = lo
    return x


def _pool(c, g, pages):
    """A key and a value pool with the logical shape [page, key head, row, head_dim]; in memory the rows of
    a head are together, or (rows_first) the heads of a row."""
    order = (pages, c["page_rows"], c["kv_heads"], c["head_dim"])
    if not c["rows_first"]:
        order = (pages, c["kv_heads"], c["page_rows"], c["head_dim"])
    made = [torch.randn(order, generator=g, device="cuda", dtype=torch.float32).to(DTYPES[c["dtype"]]) for _ in range(2)]
    return [x.transpose(1, 2) if c["rows_first"] else x for x in made]


def _kv_struct(c, k, v, pages):
    """struct vkllm_b200_paged_kv: what a program keeps for each layer's pools."""
    return ctypes.create_string_buffer(struct.pack(
        "=QQQQQIIIIII", k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), pages, c["page_rows"],
        c["kv_heads"], c["head_dim"], CODES[c["dtype"]], 0))


def _table_struct(table, free, pages, page_rows):
    """struct vkllm_b200_paged_table."""
    return ctypes.create_string_buffer(struct.pack("=QQQIIII", table.data_ptr(), 0 if free is None else free.data_ptr(),
                                                   table.stride(0), table.shape[0], table.shape[1], page_rows, pages))


def prepare(case, seed):
    return {"tables": _prepare_tables, "rope": _prepare_rope, "attention": _prepare_attention,
            "logits": _prepare_logits}[case["op"]](case, _gen(seed))


def _prepare_tables(c, g):
    n, pr, cols = c["seqs"], c["page_rows"], c["cols"]
    # some slots are empty, some hold whole pages, most end inside one
    lens = _lengths(g, n, 0, c["max_len"])
    new = _ints(g, 1 if c["new_hi"] == 1 else 0, c["new_hi"], (n,))
    done = torch.zeros(n, dtype=torch.int32, device="cuda")
    done[torch.randperm(n, generator=g, device="cuda")[:c["done"]]] = 1
    held = (lens + pr - 1) // pr
    pages = n * cols + 17
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(cols, device="cuda")
    table = torch.where(col < held[:, None], order[:n * cols].view(n, cols), -1).to(torch.int32)
    # the pages that no sequence holds, in a random order, are the free list
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(table < 0, pages, table).long()] = True
    free = torch.cat([order[~used[:pages][order.long()]], order[used[:pages][order.long()]]]).contiguous()
    count = (~used[:pages]).sum().to(torch.int32).view(1)
    z = functools.partial(torch.zeros, dtype=torch.int32, device="cuda")
    s = {"case": c, "lens": lens, "new": new, "done": done, "table": table, "free": free, "count": count,
         "pages": pages, "lens1": z(n), "count1": z(1), "lens2": z(n), "count2": z(1), "starts": z(n + 1),
         "slots": z(c["max_tokens"]), "positions": z(c["max_tokens"]), "status": z(1)}
    s["tab"] = _table_struct(table, free, pages, pr)
    return s


def _prepare_rope(c, g):
    t, h, hk, hd, pr = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"], c["page_rows"]
    dt = DTYPES[c["dtype"]]
    # the output of one Q/K/V product: a row holds a token's queries, keys and values
    qkv = torch.randn((t, (h + 2 * hk) * hd), generator=g, device="cuda", dtype=torch.float32).to(dt)
    k, v = _pool(c, g, c["pages"] + 1)  # the last page takes what the plain form has to put nowhere
    slots = torch.randperm(c["pages"] * pr, generator=g, device="cuda")[:t].to(torch.int32)
    if c["skip"]:
        slots[t - c["skip"]:] = -1
    return {"case": c, "qkv": qkv, "q": qkv[:, :h * hd], "k_new": qkv[:, h * hd:(h + hk) * hd],
            "v_new": qkv[:, (h + hk) * hd:], "k": k, "v": v, "slots": slots,
            "positions": _ints(g, 0, c["far"], (t,)), "q_out": torch.zeros((t, h * hd), dtype=dt, device="cuda"),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda"), "kv": _kv_struct(c, k, v, c["pages"])}


def _prepare_attention(c, g):
    n, h, hd, pr = c["seqs"], c["heads"], c["head_dim"], c["page_rows"]
    lens = _lengths(g, n, c["min_len"], c["max_len"])
    cols = -(-c["max_len"] // pr) + 1
    pages = n * cols + 3
    k, v = _pool(c, g, pages)
    table = torch.randperm(pages, generator=g, device="cuda")[:n * cols].to(torch.int32).view(n, cols)
    # the last page's rows behind the end hold whatever was there: here no number
    at = lens[:, None] + torch.arange(8, device="cuda")
    page, row = table.gather(1, (at // pr).clamp(max=cols - 1)).long(), (at % pr).long()
    k[page, :, row] = float("nan")
    v[page, :, row] = float("nan")
    q = torch.randn((n, h * hd), generator=g, device="cuda", dtype=torch.float32).mul_(1.5).to(DTYPES[c["dtype"]])
    return {"case": c, "q": q, "k": k, "v": v, "table": table, "lens": lens, "out": torch.zeros_like(q),
            "scale": 1.0 / math.sqrt(hd), "workspace": torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda"),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda"), "kv": _kv_struct(c, k, v, pages),
            "tab": _table_struct(table, None, pages, pr)}


def _prepare_logits(c, g):
    n, vocab = c["rows"], c["vocab"]
    x = torch.randn((n, vocab), generator=g, device="cuda", dtype=torch.float32).mul_(4).to(DTYPES[c["dtype"]])
    prompt = _lengths(g, n, c["prompt"] // 2, c["prompt"])
    total = prompt + _lengths(g, n, 0, c["output"])
    # text repeats its common tokens: the id falls off with its rank, and ranks lie all over the vocabulary
    u = torch.rand((n, c["prompt"] + c["output"]), generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab)) - 1).long().clamp(max=vocab - 1)
    history = (rank * 7919 % vocab).to(torch.int32)
    f = functools.partial(torch.rand, n, generator=g, device="cuda")
    each = _ints(g, 0, c["biases"], (n,))
    each[0] = c["biases"]
    starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    starts[1:] = each.cumsum(0)
    at = torch.arange(n * c["biases"], device="cuda")
    ids = ((at % c["biases"]) * (vocab // c["biases"]) + at // c["biases"]) % vocab
    ids = ids.to(torch.int32).contiguous()
    values = torch.randn(len(ids), generator=g, device="cuda").mul_(10)
    words = -(-vocab // 32)
    s = {"case": c, "x": x, "history": history, "prompt_lens": prompt, "history_lens": total.to(torch.int32),
         "repetition": 1.0 + f() * 0.5, "frequency": f(), "presence": f(), "bias_starts": starts, "bias_ids": ids,
         "bias_values": values, "mask": _ints(g, -2**31, 2**31 - 1, (n, words)) if c["masked"] else None,
         "out": torch.zeros_like(x)}
    keys = ("history", "prompt_lens", "history_lens", "repetition", "frequency", "presence", "bias_starts", "bias_ids",
            "bias_values", "mask")
    s["rules"] = ctypes.create_string_buffer(struct.pack(
        "=10QQQ", *(0 if s[k] is None else s[k].data_ptr() for k in keys), history.stride(0), words))
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "rope": _own_rope, "attention": _own_attention, "logits": _own_logits}[op](state)
    return {"tables": _plain_tables, "rope": _plain_rope, "attention": _plain_attention,
            "logits": _plain_logits}[op](state)


@functools.lru_cache(maxsize=None)
def _library():
    import os
    import sys
    sys.path.insert(0, os.path.join(os.getcwd(), "vkllm.c_b200"))
    import vkllm_b200
    return vkllm_b200


def _check(err, what):
    if err != 1:
        _library().check(err, what)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _tables_outputs(s):
    return {k: s[k] for k in ("table", "free", "lens2", "count2", "starts", "slots", "positions")}


def _own_tables(s):
    lib, stream = _library().lib(), _stream()
    _check(lib.vkllm_b200_paged_release(s["tab"], s["lens"].data_ptr(), s["done"].data_ptr(), s["count"].data_ptr(),
                                        s["lens1"].data_ptr(), s["count1"].data_ptr(), s["status"].data_ptr(), stream),
           "paged_release")
    _check(lib.vkllm_b200_paged_append(s["tab"], s["lens1"].data_ptr(), s["new"].data_ptr(), s["count1"].data_ptr(),
                                       s["lens2"].data_ptr(), s["count2"].data_ptr(), s["starts"].data_ptr(),
                                       s["slots"].data_ptr(), s["positions"].data_ptr(), s["case"]["max_tokens"],
                                       s["status"].data_ptr(), stream), "paged_append")
    return _tables_outputs(s)


def _own_rope(s):
    c = s["case"]
    row = s["qkv"].stride(0)
    _check(_library().lib().vkllm_b200_paged_rope_write(
        s["kv"], s["q"].data_ptr(), row, s["k_new"].data_ptr(), row, s["v_new"].data_ptr(), row,
        s["positions"].data_ptr(), s["slots"].data_ptr(), c["tokens"], c["heads"], c["base"], s["q_out"].data_ptr(),
        s["q_out"].stride(0), s["status"].data_ptr(), _stream()), "paged_rope_write")
    return {"q": s["q_out"], "k": s["k"][:c["pages"]], "v": s["v"][:c["pages"]]}


def _own_attention(s):
    q, out = s["q"], s["out"]
    _check(_library().lib().vkllm_b200_paged_attention(
        s["kv"], s["tab"], q.data_ptr(), q.stride(0), s["case"]["heads"], s["lens"].data_ptr(), s["scale"],
        out.data_ptr(), out.stride(0), s["workspace"].data_ptr(), WORKSPACE_BYTES, s["status"].data_ptr(), _stream()),
        "paged_attention")
    return out


def _own_logits(s):
    c, x, out = s["case"], s["x"], s["out"]
    _check(_library().lib().vkllm_b200_logits_apply(s["rules"], x.data_ptr(), x.stride(0), c["rows"], c["vocab"],
                                                    CODES[c["dtype"]], out.data_ptr(), out.stride(0), _stream()),
           "logits_apply")
    return out


def _plain_tables(s):
    c = s["case"]
    pr, cols, pages, most = c["page_rows"], c["cols"], s["pages"], c["max_tokens"]
    lens, table, col = s["lens"].long(), s["table"].long(), torch.arange(cols, device="cuda")
    # ended sequences give their pages back, in the order of the slots and of their pages
    held = (lens + pr - 1) // pr
    gone = (col < held[:, None]) & (s["done"] != 0)[:, None]
    at = s["count"] + gone.view(-1).cumsum(0) - 1
    free = torch.cat([s["free"].long(), s["free"].new_zeros(1).long()])
    free = free.scatter(0, torch.where(gone.view(-1), at, pages), table.view(-1))[:pages]
    count = s["count"].long() + gone.sum()
    lens = torch.where(s["done"] != 0, 0, lens)
    # new pages from the top of the list, first slot first
    held, new = (lens + pr - 1) // pr, s["new"].long()
    want = (lens + new + pr - 1) // pr - held
    fits = (want.sum() <= count) & (lens + new <= cols * pr).all() & (new.sum() <= most)
    want, new = torch.where(fits, want, 0), torch.where(fits, new, 0)
    rank = (want.cumsum(0) - want)[:, None] + col - held[:, None]
    taken = (col >= held[:, None]) & (col < (held + want)[:, None])
    table = torch.where(taken, free[(count - 1 - rank).clamp(0, pages - 1)], table)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    token = torch.arange(most, device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True).clamp(max=c["seqs"] - 1)
    here = token < starts[-1]
    position = torch.where(here, lens[seq] + token - starts[seq], 0)
    slot = table[seq, (position // pr).clamp(max=cols - 1)] * pr + position % pr
    s["table"].copy_(table)
    s["free"].copy_(free)
    s["lens2"].copy_(lens + new)
    s["count2"].copy_(count - want.sum())
    s["starts"].copy_(starts)
    s["slots"].copy_(torch.where(here, slot, -1))
    s["positions"].copy_(position)
    return _tables_outputs(s)


def _plain_rope(s):
    c = s["case"]
    t, hd, pr = c["tokens"], c["head_dim"], c["page_rows"]
    angle = s["positions"].double()[:, None] * c["base"] ** (-torch.arange(0, hd, 2, device="cuda").double() / hd)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x):
        x = x.float().reshape(t, -1, hd // 2, 2)
        a, b = x[..., 0], x[..., 1]
        return torch.stack([cos * a - sin * b, sin * a + cos * b], -1).view(t, -1, hd).to(s["q"].dtype)

    here = s["slots"] >= 0
    page = torch.where(here, s["slots"] // pr, c["pages"]).long()
    row = torch.where(here, s["slots"] % pr, 0).long()
    s["k"][page, :, row] = turned(s["k_new"])
    s["v"][page, :, row] = s["v_new"].reshape(t, -1, hd)
    s["q_out"].copy_(torch.where(here[:, None], turned(s["q"]).view(t, -1), s["q_out"]))
    return {"q": s["q_out"], "k": s["k"][:c["pages"]], "v": s["v"][:c["pages"]]}


def _plain_attention(s):
    c, lens = s["case"], s["lens"]
    n, hk, hd, pr = c["seqs"], c["kv_heads"], c["head_dim"], c["page_rows"]
    at = torch.arange(max(1, c["max_len"]), device="cuda")
    there = at < lens[:, None]
    page, row = s["table"][:, at // pr].long(), (at % pr).expand(n, -1)
    keys = s["k"][page, :, row].float().masked_fill_(~there[:, :, None, None], 0).permute(0, 2, 3, 1)
    q = s["q"].float().view(n, hk, -1, hd)
    score = (q @ keys * s["scale"]).masked_fill_(~there[:, None, None], -math.inf)
    del keys
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0, top)).exp()
    values = s["v"][page, :, row].float().masked_fill_(~there[:, :, None, None], 0).permute(0, 2, 1, 3)
    out = (p @ values) / p.sum(-1, keepdim=True)
    out = torch.where((lens > 0)[:, None, None, None], out, 0)
    return out.view(n, -1).to(s["q"].dtype)


def _plain_logits(s):
    c, x = s["case"], s["x"].float()
    n, vocab = x.shape
    at = torch.arange(s["history"].shape[1], device="cuda")
    ids = s["history"].long()
    said = at < s["history_lens"][:, None]
    output = said & (at >= s["prompt_lens"][:, None])
    seen = torch.zeros((n, vocab), dtype=torch.int32, device="cuda").scatter_add_(1, ids, said.int())
    count = torch.zeros((n, vocab), dtype=torch.int32, device="cuda").scatter_add_(1, ids, output.int()).float()
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    entry = torch.arange(len(s["bias_ids"]), device="cuda")
    row = torch.searchsorted(s["bias_starts"][1:], entry, right=True)
    value = torch.where(entry < s["bias_starts"][-1], s["bias_values"], 0.0)
    x.index_put_((row.clamp(max=n - 1), s["bias_ids"].long()), value, accumulate=True)
    if s["mask"] is not None:
        v = torch.arange(vocab, device="cuda")
        x = torch.where((s["mask"][:, v >> 5] >> (v & 31)) & 1 != 0, x, -math.inf)
    return x.to(s["x"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "tables":
        n, most = c["seqs"], c["max_tokens"]
        # lengths, new tokens and ended marks in, lengths and starts out, a slot and a position for each token;
        # every new token's share of a page taken from the list and put into the table
        return {"bytes": 4 * (5 * n + 2 * most + 2 * (n * c["new_hi"] // 2) // c["page_rows"]), "flops": 4 * most}
    size = 2 if c["dtype"] == "f16" else 4
    if c["op"] == "rope":
        t, row = c["tokens"] - c["skip"], (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]
        return {"bytes": 2 * t * row * size + 8 * c["tokens"], "flops": 3 * t * (c["heads"] + c["kv_heads"]) * c["head_dim"]}
    if c["op"] == "attention":
        keys = c["seqs"] * (c["min_len"] + c["max_len"]) // 2 + (c["max_len"] - c["min_len"]) // 2
        row = c["kv_heads"] * c["head_dim"] * size
        pages = keys // c["page_rows"] + c["seqs"]
        return {"bytes": 2 * keys * row + 2 * c["seqs"] * c["heads"] * c["head_dim"] * size + 4 * pages,
                "flops": 4 * keys * c["heads"] * c["head_dim"]}
    n, vocab = c["rows"], c["vocab"]
    past = c["prompt"] * 3 // 4 + c["output"] // 2
    return {"bytes": n * (2 * vocab * size + 4 * past + 4 * c["biases"] + c["masked"] * vocab // 8),
            "flops": n * (2 * vocab + 4 * past)}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return None  # whole numbers
    return {"rope": _exact_rope, "attention": _exact_attention, "logits": _exact_logits}[case["op"]](case, s)


def _exact_rope(c, s):
    hd, pr = c["head_dim"], c["page_rows"]
    w = torch.arange(hd // 2, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones((c["tokens"], hd // 2), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] / torch.pow(c["base"], 2 * w / hd))
    kept = torch.arange(c["tokens"] - c["skip"], device="cuda")

    def spun(x):
        z = torch.view_as_complex(x[kept].double().reshape(len(kept), -1, hd // 2, 2).contiguous())
        return torch.view_as_real(z * turn[kept][:, None]).reshape(len(kept), -1, hd)

    q, k, v = s["q_out"].double(), s["k"][:c["pages"]].double(), s["v"][:c["pages"]].double()
    q[kept] = spun(s["q"]).flatten(1)
    slot = s["slots"][kept].long()
    k[slot // pr, :, slot % pr] = spun(s["k_new"])
    v[slot // pr, :, slot % pr] = s["v_new"][kept].double().reshape(len(kept), -1, hd)
    return {"q": q, "k": k, "v": v}


def _exact_attention(c, s):
    out = torch.zeros((c["seqs"], c["heads"], c["head_dim"]), dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv_heads"]
    for i, keys in enumerate(s["lens"].tolist()):
        if keys == 0:
            continue
        used = s["table"][i, :-(-keys // c["page_rows"])].long()
        k = s["k"][used].transpose(0, 1).flatten(1, 2)[:, :keys].double()
        v = s["v"][used].transpose(0, 1).flatten(1, 2)[:, :keys].double()
        q = s["q"][i].double().view(c["kv_heads"], group, -1)
        weight = torch.einsum("hgd,hld->hgl", q, k).mul_(s["scale"]).softmax(-1)
        out[i] = torch.einsum("hgl,hld->hgd", weight, v).reshape(c["heads"], -1)
    return out.view(c["seqs"], -1)


def _exact_logits(c, s):
    out = s["x"].double()
    for i in range(c["rows"]):
        ids = s["history"][i, :int(s["history_lens"][i])].long()
        said = torch.unique(ids)
        x, r = out[i], s["repetition"][i].double()
        x[said] = torch.where(x[said] > 0, x[said] / r, x[said] * r)
        again, count = torch.unique(ids[int(s["prompt_lens"][i]):], return_counts=True)
        x[again] -= count.double() * s["frequency"][i].double() + s["presence"][i].double()
        lo, hi = int(s["bias_starts"][i]), int(s["bias_starts"][i + 1])
        x[s["bias_ids"][lo:hi].long()] += s["bias_values"][lo:hi].double()
        if s["mask"] is not None:
            bits = (s["mask"][i][:, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
            x[bits.flatten()[:c["vocab"]] == 0] = -math.inf
    return out
