"""What the attentions' C entry points answer before any launch: without rows, and for the size of a workspace."""
import ctypes

import pytest

from test_paged_oracle import attention_args, call


@pytest.mark.parametrize("empty", [dict(n_new=0), dict(rows=0)])
def test_status_without_rows(empty):
    from dforktree_amd import _lib
    a = attention_args(_lib.PagedAttentionArgs)
    a.n_new, a.page_size, a.columns, a.num_pages = 4, 16, 4, 8
    a.key_cache = a.value_cache = a.block_table = a.seq_len = 16
    a.seq_len_dtype = _lib.DFT_I32
    assert call("dft_paged_attention", a, **empty, batch=0, status=16) == _lib.DFT_OK
    assert call("dft_paged_attention", a, **empty, status=16, seq_len=None) == _lib.DFT_ERR_INVALID
    assert call("dft_paged_attention", a, **empty, status=16, seq_len_dtype=1) == _lib.DFT_ERR_INVALID
    assert call("dft_paged_attention", a, **empty, status=16, batch=65536) == _lib.DFT_ERR_UNSUPPORTED
    p = attention_args(_lib.PromptAttentionArgs)
    p.max_len = 4
    empty = {"max_len" if k == "n_new" else k: v for k, v in empty.items()}
    assert call("dft_prompt_attention", p, **empty, batch=0, status=16) == _lib.DFT_OK
    assert call("dft_prompt_attention", p, **empty, status=16, batch=65536) == _lib.DFT_ERR_UNSUPPORTED


def test_workspace_before_there_are_buffers():
    """Its size is asked for to allocate it, when no pointer of the launch need be known."""
    from dforktree_amd import _lib
    n = ctypes.c_int64(-1)
    a = attention_args(_lib.PagedAttentionArgs)
    a.n_new, a.page_size, a.columns, a.num_pages, a.seq_len_dtype = 4, 16, 400, 8, _lib.DFT_I32
    assert _lib.load().dft_paged_attention_workspace(ctypes.byref(a), ctypes.byref(n)) == _lib.DFT_OK
    want = n.value
    assert want > 0
    a.q = a.o = None
    assert _lib.load().dft_paged_attention_workspace(ctypes.byref(a), ctypes.byref(n)) == _lib.DFT_OK and n.value == want
    for bad in (dict(head_dim=80), dict(hkv=3), dict(n_new=-1)):
        old = {k: getattr(a, k) for k in bad}
        for k, v in bad.items():
            setattr(a, k, v)
        assert _lib.load().dft_paged_attention_workspace(ctypes.byref(a), ctypes.byref(n)) != _lib.DFT_OK and n.value == 0
        for k, v in old.items():
            setattr(a, k, v)
