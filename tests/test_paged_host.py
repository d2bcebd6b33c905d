"""Host side of the paged serving operators, without a GPU: every argument that does not fit is refused
before CUDA is touched, and vkllm_b200_paged_check finds what the kernels would flag."""
import ctypes as C

import numpy as np
import pytest

P = 0x10000  # a 16-byte aligned address that nothing reads: the calls are refused first


def table(vk, **k):
    d = dict(table=P, free_pages=P, stride=8, n_seqs=4, cols=8, page_rows=16, n_pages=64)
    d.update(k)
    return vk.PagedTable(*(d[f] for f, _ in vk.PagedTable._fields_))


def pools(vk, **k):
    d = dict(k=P, v=P, page_stride=16 * 2 * 64, head_stride=16 * 64, row_stride=64, n_pages=64, page_rows=16,
             kv_heads=2, head_dim=64, dtype=vk.F16, reserved=0)
    d.update(k)
    return vk.PagedKV(*(d[f] for f, _ in vk.PagedKV._fields_))


def by(s):
    return None if s is None else C.byref(s)


def append(vk, t, **k):
    d = dict(lens=P, n_new=P, n_free=P, new_lens=P, n_free_out=P, starts=P, slots=P, positions=P, max_tokens=4, status=P,
             stream=None)
    d.update(k)
    return vk.lib().vkllm_b200_paged_append(by(t), *d.values())


def release(vk, t, **k):
    d = dict(lens=P, done=P, n_free=P, new_lens=P, n_free_out=P, status=P, stream=None)
    d.update(k)
    return vk.lib().vkllm_b200_paged_release(by(t), *d.values())


def rope(vk, kv, **k):
    d = dict(q=P, q_stride=512, k=P, k_stride=512, v=P, v_stride=512, positions=P, slots=P, n_tokens=3, heads=4, base=0.0,
             q_out=P + 4096, q_out_stride=512, status=P, stream=None)
    d.update(k)
    return vk.lib().vkllm_b200_paged_rope_write(by(kv), *d.values())


def attend(vk, kv, t, **k):
    d = dict(q=P, q_stride=256, heads=4, lens=P, scale=0.1, out=P + 4096, out_stride=256, workspace=P,
             workspace_bytes=vk.PAGED_WORKSPACE_BYTES, status=P, stream=None)
    d.update(k)
    return vk.lib().vkllm_b200_paged_attention(by(kv), by(t), *d.values())


def rules(vk, **k):
    d = {f: None for f, _ in vk.LogitRules._fields_}
    d.update(history_stride=16, mask_stride=4)
    d.update(k)
    return vk.LogitRules(*d.values())


def apply(vk, r, **k):
    d = dict(logits=P, logits_stride=100, rows=2, vocab=100, dtype=vk.F16, out=P, out_stride=100, stream=None)
    d.update(k)
    return vk.lib().vkllm_b200_logits_apply(by(r), *d.values())


@pytest.mark.parametrize("bad", [dict(table=None), dict(table=P + 2), dict(stride=7), dict(n_seqs=0), dict(cols=0),
                                 dict(page_rows=0), dict(n_pages=0), dict(n_pages=1 << 28, page_rows=32),
                                 dict(free_pages=None), dict(n_seqs=16385), dict(stride=1 << 40)])
def test_tables_refuse_a_table(vk, bad):
    assert append(vk, table(vk, **bad)) == vk.ARGS
    assert release(vk, table(vk, **bad)) == vk.ARGS


def test_tables_refuse_arrays(vk):
    assert append(vk, None) == vk.ARGS and release(vk, None) == vk.ARGS
    for name in ("lens", "n_new", "n_free", "new_lens", "n_free_out", "starts", "slots", "positions", "status"):
        for p in (None, P + 1):
            assert append(vk, table(vk), **{name: p}) == vk.ARGS, name
    for name in ("lens", "done", "n_free", "new_lens", "n_free_out", "status"):
        for p in (None, P + 2):
            assert release(vk, table(vk), **{name: p}) == vk.ARGS, name


BAD_POOLS = [dict(k=None), dict(v=P + 8), dict(page_stride=1028), dict(head_stride=1020), dict(row_stride=68),
             dict(row_stride=56), dict(head_stride=56), dict(n_pages=0), dict(page_rows=0), dict(kv_heads=0),
             dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(dtype=3), dict(dtype=0), dict(reserved=1),
             dict(page_stride=1 << 41), dict(n_pages=1 << 29)]


@pytest.mark.parametrize("bad", BAD_POOLS)
def test_pools_refused(vk, bad):
    assert rope(vk, pools(vk, **bad)) == vk.ARGS
    t = table(vk, page_rows=pools(vk, **bad).page_rows or 16, n_pages=min(pools(vk, **bad).n_pages or 64, 1 << 20))
    assert attend(vk, pools(vk, **bad), t) == vk.ARGS


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=P + 8), dict(k=P + 2), dict(v=None), dict(q_out=P + 4),
                                 dict(q_stride=255), dict(q_stride=260), dict(k_stride=120), dict(v_stride=129),
                                 dict(q_out_stride=248), dict(positions=None), dict(slots=P + 1), dict(status=None),
                                 dict(heads=0), dict(heads=3), dict(heads=65536), dict(base=1.0), dict(base=0.5),
                                 dict(base=float("nan")), dict(base=float("inf")), dict(n_tokens=1 << 31),
                                 dict(q_out=P, q_out_stride=256)])
def test_rope_write_refused(vk, bad):
    assert rope(vk, pools(vk), **bad) == vk.ARGS
    assert rope(vk, None) == vk.ARGS


def test_rope_write_of_no_tokens_does_nothing(vk):
    assert rope(vk, pools(vk), n_tokens=0, q=None, k=None, v=None, q_out=None) == vk.OK


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=P + 8), dict(out=None), dict(out=P), dict(q_stride=252),
                                 dict(q_stride=248), dict(out_stride=250), dict(heads=0), dict(heads=5), dict(lens=None),
                                 dict(status=P + 3), dict(workspace=None), dict(workspace=P + 8),
                                 dict(workspace_bytes=(16 << 20) - 1)])
def test_attention_refused(vk, bad):
    assert attend(vk, pools(vk), table(vk), **bad) == vk.ARGS


def test_attention_refuses_a_table_of_other_pools(vk):
    assert attend(vk, pools(vk), None) == vk.ARGS and attend(vk, None, table(vk)) == vk.ARGS
    assert attend(vk, pools(vk), table(vk, page_rows=8)) == vk.ARGS
    assert attend(vk, pools(vk), table(vk, n_pages=63)) == vk.ARGS


@pytest.mark.parametrize("bad", [dict(logits=None), dict(logits=P + 1), dict(out=None), dict(out=P + 3),
                                 dict(logits_stride=99), dict(out_stride=99), dict(rows=0), dict(rows=65536),
                                 dict(vocab=0), dict(dtype=3), dict(dtype=4), dict(out_stride=101)])
def test_logits_refused(vk, bad):
    assert apply(vk, rules(vk), **bad) == vk.ARGS


@pytest.mark.parametrize("bad", [dict(history=P), dict(history=P + 2, history_lens=P), dict(repetition=P),
                                 dict(frequency=P), dict(presence=P), dict(bias_starts=P, bias_ids=P),
                                 dict(bias_starts=P, bias_values=P), dict(mask=P, mask_stride=3), dict(mask=P + 1),
                                 dict(history=P, history_lens=P, repetition=P + 2)])
def test_logit_rules_refused(vk, bad):
    assert apply(vk, rules(vk, **bad)) == vk.ARGS
    assert apply(vk, None) == vk.ARGS


@pytest.mark.parametrize("stride", [1 << 30, (1 << 32) - 1, 1 << 39])
def test_logit_rules_refuse_histories_past_30_bits(vk, stride):
    """An id's count has 30 bits beside two marks, and a history of nearly 2^32 ids would wrap the 32-bit places."""
    assert apply(vk, rules(vk, history=P, history_lens=P, history_stride=stride)) == vk.ARGS


# ---- vkllm_b200_paged_check ----------------------------------------------------------------------

def check(vk, tab, lens, free=(), page_rows=4, n_pages=10, n_free=None):
    tab = np.ascontiguousarray(tab, dtype=np.uint32)
    lens, free = np.asarray(lens, dtype=np.uint32), np.asarray(free, dtype=np.uint32)
    t = vk.PagedTable(tab.ctypes.data, free.ctypes.data if len(free) else None, tab.shape[1], tab.shape[0], tab.shape[1],
                      page_rows, n_pages)
    status, bad = C.c_uint32(77), C.c_uint32(77)
    err = vk.lib().vkllm_b200_paged_check(C.byref(t), lens.ctypes.data, len(free) if n_free is None else n_free,
                                          C.byref(status), C.byref(bad))
    return err, status.value, bad.value


def test_check_accepts_and_ignores_what_is_not_held(vk):
    x = vk.NO_SLOT  # entries behind the held pages are never looked at
    assert check(vk, [[3, 1, x], [x, x, x], [9, x, x]], [8, 0, 4], [0, 2, 5])[:2] == (vk.OK, 0)


@pytest.mark.parametrize("tab,lens,free,status,seq", [
    ([[3, 10], [1, 2]], [5, 8], [], 1, 0),        # an id past the pool
    ([[3, 10], [1, 2]], [4, 9], [], 2, 1),        # a length past the row (the bad id is not held)
    ([[3, 4], [4, 2]], [8, 1], [], 1, 1),         # a page of two sequences
    ([[3, 4], [5, 2]], [8, 1], [0, 3], 1, 2),     # a held page on the free list
    ([[3, 4], [5, 2]], [8, 1], [0, 11], 1, 2),    # an id past the pool on the free list
    ([[3, 4], [5, 2]], [8, 1], [0, 0], 1, 2),     # a page twice on the free list
])
def test_check_finds(vk, tab, lens, free, status, seq):
    assert check(vk, tab, lens, free) == (vk.ARGS, status, seq)


def test_check_finds_a_free_list_past_the_pool(vk):
    assert check(vk, [[3, 4]], [8], [0] * 11, n_pages=10)[:2] == (vk.ARGS, 4)
    assert vk.lib().vkllm_b200_paged_check(None, None, 0, None, None) == vk.ARGS


def test_struct_layouts(vk):
    for name, mirror in (("vkllm_b200_paged_table", vk.PagedTable), ("vkllm_b200_paged_kv", vk.PagedKV),
                         ("vkllm_b200_logit_rules", vk.LogitRules)):
        assert vk.lib().vkllm_b200_sizeof(name.encode()) == C.sizeof(mirror), name
