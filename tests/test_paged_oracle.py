"""The paged oracle against closed forms, and what the host refuses before
any launch: descriptors of the C ABI and arguments of the Python layer."""
import ctypes
import json
import subprocess

import numpy as np
import pytest
import torch

from conftest import ROOT
from oracle import paged as P

HEADER = ROOT / "include" / "dforktree_amd.h"


def plan(prefix, new, held, free, **kw):
    B, cols, ps = len(prefix), kw.pop("cols", 16), kw.pop("page_size", 4)
    table = np.full((B, cols), -1, np.int32)
    page = 100
    for b, h in enumerate(held):
        table[b, :h] = np.arange(page, page + h)
        page += h
    ring = np.array(list(free) + [-1] * kw.pop("room", 40), np.int32)
    return P.page_plan(prefix, new, table, held, ring, [0, len(free)], page_size=ps, rows=kw.pop("rows", sum(new)), **kw)


def test_plan_takes_pages_in_request_order():
    r = plan([3, 0, 8], [2, 5, 4], [1, 0, 2], [7, 8, 9, 10])
    assert r["block_table"][0, :2].tolist() == [100, 7]
    assert r["block_table"][1, :2].tolist() == [8, 9]
    assert r["block_table"][2, :3].tolist() == [101, 102, 10]
    assert r["slots"].tolist() == [100 * 4 + 3, 7 * 4, 32, 33, 34, 35, 36, 40, 41, 42, 43]
    assert r["positions"].tolist() == [3, 4, 0, 1, 2, 3, 4, 8, 9, 10, 11]
    assert r["held"].tolist() == [2, 2, 3] and r["free_pos"].tolist() == [4, 4]
    assert r["seq_len"].tolist() == [5, 5, 12] and not r["status"].any()


def test_plan_refuses_what_does_not_fit():
    r = plan([3, 0, 8], [2, 5, 0], [1, 0, 2], [7, 8])
    assert r["status"].tolist() == [0, P.STATUS_PAGES, 0]
    assert r["free_pos"].tolist() == [1, 2] and r["held"].tolist() == [2, 0, 2]
    assert r["slots"].tolist() == [403, 28, -1, -1, -1, -1, -1] and r["seq_len"].tolist() == [5, 0, 8]
    r = plan([0], [17], [0], [1, 2, 3, 4, 5, 6], cols=4)
    assert r["status"].tolist() == [P.STATUS_TABLE] and (r["slots"] == -1).all()
    r = plan([0, 0], [4, 6], [0, 0], [1, 2], rows=7)
    assert r["cu_seqlens"].tolist() == [0, 4, 7] and r["status"].tolist() == [0, P.STATUS_SPAN]


def test_plan_returns_pages_in_order():
    r = plan([0, 5], [0, 1], [2, 4], [7], trim=True)
    assert r["held"].tolist() == [0, 2] and r["free_pos"].tolist() == [0, 5]
    assert r["free_pages"][:5].tolist() == [7, 100, 101, 104, 105]


def test_attend_matches_a_dense_softmax():
    rng = np.random.default_rng(0)
    q, k, v = rng.normal(size=(5, 4, 8)), rng.normal(size=(9, 2, 8)), rng.normal(size=(9, 2, 8))
    sees = P.sees_causal(5, 9)
    assert sees.sum(1).tolist() == [5, 6, 7, 8, 9]
    o, lse, _, _ = P.attend(q, k, v, sees, 0.3)
    for h in range(4):
        s = np.where(sees, 0.3 * q[:, h] @ k[:, h // 2].T, -np.inf)
        e = np.exp(s)
        assert np.allclose(o[:, h], e @ v[:, h // 2] / e.sum(1, keepdims=True)) and np.allclose(lse[:, h], np.log(e.sum(1)))


def test_attend_leaves_out_what_a_row_does_not_see():
    q, k, v = np.ones((2, 1, 4)), np.ones((3, 1, 4)), np.ones((3, 1, 4))
    k[2], v[1] = np.nan, np.inf
    sees = np.array([[True, False, False], [False, False, False]])
    o, lse, _, _ = P.attend(q, k, v, sees, 1.0)
    assert (o[0] == 1).all() and lse[0, 0] == 4 and (o[1] == 0).all() and lse[1, 0] == -np.inf


def test_tree_rows_see_their_ancestors():
    sees = P.sees_tree(np.array([1, 3, 5, 1 << 63], np.uint64), 6)
    assert sees.tolist() == [[True, True, True, False, False, False], [True, True, True, True, False, False],
                             [True, True, True, False, True, False], [True, True, False, False, False, False]]
    assert P.sees_causal(3, 2).sum(1).tolist() == [0, 1, 2]


def test_bad_pages_hold_no_keys():
    cache = np.arange(2 * 3 * 1 * 1).reshape(2, 3, 1, 1)
    k, there = P.paged_keys(cache, np.array([1, 2, -1, 0]), 14)
    assert there.tolist() == [True] * 3 + [False] * 6 + [True] * 3 + [False] * 2
    assert k[:3, 0, 0].tolist() == [3, 4, 5] and k[9:12, 0, 0].tolist() == [0, 1, 2]


# ---- the C ABI --------------------------------------------------------------
def test_descriptors_match_the_header(tmp_path):
    from dforktree_amd import _lib
    structs = {"dft_page_plan_args": _lib.PagePlanArgs, "dft_kv_append_args": _lib.KvAppendArgs,
               "dft_paged_attention_args": _lib.PagedAttentionArgs,
               "dft_prompt_attention_args": _lib.PromptAttentionArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {", 'printf("{\\"\\": 0");']
    for c, py in structs.items():
        for f, _ in py._fields_:
            lines.append(f'printf(",\\"{c}.{f}\\": %zu", offsetof({c}, {f}));')
        lines.append(f'printf(",\\"{c}\\": %zu", sizeof({c}));')
    lines += ['printf("}");', f"return !(DFT_STATUS_PAGES == {_lib.DFT_STATUS_PAGES} && "
              f"DFT_STATUS_TABLE == {_lib.DFT_STATUS_TABLE} && DFT_ATTN_CAUSAL == {_lib.DFT_ATTN_CAUSAL});", "}"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    layout = json.loads(subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout)
    for c, py in structs.items():
        assert ctypes.sizeof(py) == layout[c], c
        for f, _ in py._fields_:
            assert getattr(py, f).offset == layout[f"{c}.{f}"], f"{c}.{f}"


def call(name, args, **changes):
    from dforktree_amd import _lib
    old = {k: getattr(args, k) for k in changes}
    for k, v in changes.items():
        setattr(args, k, v)
    r = getattr(_lib.load(), name)(ctypes.byref(args), None)
    for k, v in old.items():
        setattr(args, k, v)
    return r


def test_page_plan_descriptors():
    from dforktree_amd import _lib
    OK, INVALID, UNSUPPORTED = _lib.DFT_OK, _lib.DFT_ERR_INVALID, _lib.DFT_ERR_UNSUPPORTED
    assert _lib.load().dft_page_plan(None, None) == INVALID
    a = _lib.PagePlanArgs()
    a.batch, a.columns, a.page_size, a.rows, a.capacity = 2, 4, 16, 8, 9
    for f in ("prefix_len", "new_len", "block_table", "held", "free_pages", "free_pos", "slots", "positions",
              "cu_seqlens", "seq_len", "status"):
        setattr(a, f, 16)
    a.held_out, a.free_pos_out = 32, 32
    a.prefix_len_dtype = a.new_len_dtype = a.index_dtype = _lib.DFT_I32
    for bad in (dict(batch=-1), dict(columns=-1), dict(page_size=0), dict(rows=-1), dict(capacity=0), dict(held=None),
                dict(held_out=16), dict(free_pos_out=16), dict(free_pages=None), dict(free_pos=None), dict(slots=None),
                dict(positions=None), dict(cu_seqlens=None), dict(seq_len=None), dict(status=None),
                dict(block_table=None), dict(prefix_len=None), dict(new_len_dtype=1), dict(index_dtype=0),
                dict(depth=16, depth_dtype=2)):
        assert call("dft_page_plan", a, **bad) == INVALID, bad
    for bad in (dict(batch=8193), dict(rows=1 << 31), dict(capacity=1 << 31)):
        assert call("dft_page_plan", a, **bad) == UNSUPPORTED, bad


def test_kv_append_descriptors():
    from dforktree_amd import _lib
    OK, INVALID = _lib.DFT_OK, _lib.DFT_ERR_INVALID
    a = _lib.KvAppendArgs()
    a.heads, a.head_dim, a.page_size, a.n, a.src_rows, a.num_pages = 2, 64, 16, 4, 4, 3
    a.k = a.v = a.key_cache = a.value_cache = a.slots = 16
    a.src_dtype = a.cache_dtype = _lib.DFT_BF16
    a.slots_dtype = _lib.DFT_I64
    for bad in (dict(heads=0), dict(head_dim=0), dict(page_size=0), dict(n=-1), dict(src_rows=-1), dict(num_pages=-1),
                dict(src_dtype=3), dict(cache_dtype=9), dict(slots_dtype=0), dict(rows=16, rows_dtype=1),
                dict(slots=None), dict(k=None), dict(v=None), dict(key_cache=None), dict(value_cache=None)):
        assert call("dft_kv_append", a, **bad) == INVALID, bad
    assert call("dft_kv_append", a, n=0) == OK
    assert _lib.load().dft_kv_append(None, None) == INVALID


def attention_args(cls):
    from dforktree_amd import _lib
    a = cls()
    a.batch, a.hq, a.hkv, a.head_dim, a.rows, a.scale, a.dtype, a.o_dtype = 1, 8, 2, 128, 4, 1.0, _lib.DFT_BF16, _lib.DFT_BF16
    a.q = a.o = 16
    return a


def test_attention_descriptors():
    from dforktree_amd import _lib
    OK, INVALID, UNSUPPORTED = _lib.DFT_OK, _lib.DFT_ERR_INVALID, _lib.DFT_ERR_UNSUPPORTED
    shared = [(INVALID, b) for b in (dict(batch=-1), dict(rows=-1), dict(hq=0), dict(hkv=0), dict(hkv=3), dict(q=None),
                                     dict(o=None), dict(q=8), dict(q_row_stride=4), dict(q_h_stride=12), dict(o_dtype=4))]
    shared += [(UNSUPPORTED, b) for b in (dict(head_dim=80), dict(dtype=_lib.DFT_F32), dict(batch=65536), dict(hq=65536))]
    a = attention_args(_lib.PagedAttentionArgs)
    a.n_new, a.page_size, a.columns, a.num_pages = 4, 16, 4, 8
    a.key_cache = a.value_cache = a.block_table = a.seq_len = a.workspace = 16
    a.seq_len_dtype, a.workspace_bytes = _lib.DFT_I32, 0
    for want, bad in shared + [(INVALID, b) for b in (
            dict(n_new=-1), dict(page_size=0), dict(columns=-1), dict(num_pages=-1), dict(seq_len=None),
            dict(seq_len_dtype=1), dict(block_table=None), dict(key_cache=None), dict(value_cache=24),
            dict(kc_page_stride=4), dict(vc_token_stride=2), dict(vc_h_stride=1),
            dict(anc_bits=16, flags=_lib.DFT_ATTN_CAUSAL))] + [(UNSUPPORTED, dict(anc_bits=16, n_new=65)),
                                                               (UNSUPPORTED, dict(num_pages=1 << 31))]:
        assert call("dft_paged_attention", a, **bad) == want, bad
    for empty in (dict(batch=0), dict(n_new=0), dict(rows=0)):
        assert call("dft_paged_attention", a, **empty) == OK, empty
    n = ctypes.c_int64(-1)
    assert _lib.load().dft_paged_attention_workspace(ctypes.byref(a), None) == INVALID
    assert _lib.load().dft_paged_attention_workspace(None, ctypes.byref(n)) == INVALID
    assert _lib.load().dft_paged_attention_workspace(ctypes.byref(a), ctypes.byref(n)) == OK and n.value >= 0
    if n.value:  # a workspace that is missing, misaligned or too small
        for bad in (dict(workspace=None, workspace_bytes=n.value), dict(workspace=8, workspace_bytes=n.value),
                    dict(workspace_bytes=n.value - 1)):
            assert call("dft_paged_attention", a, **bad) == INVALID, bad
    a = attention_args(_lib.PromptAttentionArgs)
    a.max_len, a.k, a.v = 4, 16, 16
    for want, bad in shared + [(INVALID, b) for b in (dict(max_len=-1), dict(k=None), dict(v=None), dict(k=8),
                                                      dict(v_row_stride=4), dict(k_h_stride=2))]:
        assert call("dft_prompt_attention", a, **bad) == want, bad
    for empty in (dict(batch=0), dict(max_len=0), dict(rows=0)):
        assert call("dft_prompt_attention", a, **empty) == OK, empty
    for name in ("dft_paged_attention", "dft_prompt_attention"):
        assert getattr(_lib.load(), name)(None, None) == INVALID


def test_python_layer_takes_gpu_tensors_only():
    from dforktree_amd import ops
    x, i = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    cache = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16)
    for f in (lambda: ops.prompt_attention(x, x, x), lambda: ops.kv_append(x, x, cache, cache, i),
              lambda: ops.paged_attention(x, cache, cache, i.view(4, 1), i),
              lambda: ops.page_plan(i, i, i.view(4, 1), i, i, i.long()[:2], page_size=4, rows=4)):
        with pytest.raises(ValueError, match="GPU tensors"):
            f()


def test_attention_sizes_past_the_kernels_counters():
    """Rows times the heads of a group are counted in 31 bits, a tile's rows reached by 32-bit offsets."""
    from dforktree_amd import _lib
    INVALID, UNSUPPORTED = _lib.DFT_ERR_INVALID, _lib.DFT_ERR_UNSUPPORTED
    a = attention_args(_lib.PromptAttentionArgs)
    a.max_len, a.k, a.v = 4, 16, 16
    for want, bad in ((UNSUPPORTED, dict(max_len=1 << 30)), (UNSUPPORTED, dict(k_row_stride=1 << 24)),
                      (UNSUPPORTED, dict(v_row_stride=1 << 24)), (INVALID, dict(k_row_stride=-8)),
                      (INVALID, dict(v_row_stride=-8))):
        assert call("dft_prompt_attention", a, **bad) == want, bad
    p = attention_args(_lib.PagedAttentionArgs)
    p.n_new, p.page_size, p.columns, p.num_pages = 1 << 30, 16, 4, 8
    p.key_cache = p.value_cache = p.block_table = p.seq_len = 16
    p.seq_len_dtype = _lib.DFT_I32
    assert call("dft_paged_attention", p) == UNSUPPORTED


def test_workspace_goes_with_the_sizes_alone():
    """None where the block table is short; else a bound that the lengths do not move."""
    from dforktree_amd import _lib
    a = attention_args(_lib.PagedAttentionArgs)
    a.page_size, a.num_pages = 16, 8
    n = ctypes.c_int64(-1)
    need = {}
    for new, columns in ((1, 32), (1, 33), (1, 9000), (4, 33), (40, 33), (1000, 33)):
        a.n_new, a.columns = new, columns
        assert _lib.load().dft_paged_attention_workspace(ctypes.byref(a), ctypes.byref(n)) == _lib.DFT_OK
        need[new, columns] = n.value
    assert need[1, 32] == 0 < need[1, 33] == need[1, 9000] <= need[4, 33] < need[40, 33] == need[1000, 33]
