"""The C boundary of the packed GDN entry points and the accepted path, on the CPU: the structs' layouts, and what is
refused before any launch."""
import ctypes
import json
import subprocess

import pytest

from conftest import ROOT


def structs():
    from dforktree_amd import _lib
    return {"dft_prompt_conv_args": _lib.PromptConvArgs, "dft_prompt_gdn_args": _lib.PromptGdnArgs,
            "dft_tree_accept_args": _lib.TreeAcceptArgs}


def test_ctypes_structs_match_c_layout(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "dforktree_amd.h"}"',
             'int main(void) { const char* s = "{";']
    for name, py in structs().items():
        for f, _ in py._fields_:
            lines.append(f'printf("%s\\"{name}.{f}\\": %zu", s, offsetof({name}, {f})); s = ",";')
        lines.append(f'printf(",\\"{name}\\": %zu", sizeof({name}));')
    lines.append('printf("}"); return 0; }')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-o", str(exe), str(src)], check=True)
    layout = json.loads(subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout)
    for name, py in structs().items():
        assert ctypes.sizeof(py) == layout[name], name
        for f, _ in py._fields_:
            assert getattr(py, f).offset == layout[f"{name}.{f}"], f"{name}.{f}"


def conv_args():
    from dforktree_amd import _lib
    a = _lib.PromptConvArgs()
    a.batch, a.max_len, a.channels, a.width, a.rows, a.slots = 2, 4, 8, 4, 8, 2
    a.x = a.y = a.weight = a.conv_state = 16
    a.x_dtype = a.y_dtype = a.w_dtype = a.cs_dtype = _lib.DFT_BF16
    return a


def gdn_args():
    from dforktree_amd import _lib
    a = _lib.PromptGdnArgs()
    a.batch, a.max_len, a.hk, a.hv, a.dk, a.dv, a.rows, a.slots = 2, 4, 1, 2, 128, 128, 8, 2
    a.y = a.a = a.b = a.o = a.A_log = a.dt_bias = a.state = a.workspace = 16
    a.y_row_stride, a.workspace_bytes = 512, 1 << 40
    a.a_dtype = a.b_dtype = a.o_dtype = a.A_log_dtype = a.dt_bias_dtype = _lib.DFT_BF16
    return a


def accept_args():
    from dforktree_amd import _lib
    a = _lib.TreeAcceptArgs()
    a.batch, a.n_nodes, a.vocab, a.path_cols, a.rows = 2, 4, 100, 16, 8
    a.tokens = a.parent = a.probs = a.uniform = a.last = 16
    a.path = a.path_len = a.path_rows = a.token = a.workspace = 16
    a.workspace_bytes = 1 << 40
    a.tokens_dtype = a.parent_dtype = _lib.DFT_I32
    return a


INVALID, UNSUPPORTED = 1, 2
REFUSED = [
    ("dft_prompt_conv", conv_args, INVALID, [
        dict(batch=-1), dict(max_len=-1), dict(channels=-1), dict(rows=-1), dict(slots=-1), dict(x=None), dict(y=None),
        dict(weight=None), dict(conv_state=None), dict(x_dtype=3), dict(y_dtype=9), dict(w_dtype=4), dict(cs_dtype=3),
        dict(bias=16, bias_dtype=3), dict(cs_indices=16, cs_indices_dtype=0)]),
    ("dft_prompt_conv", conv_args, UNSUPPORTED, [
        dict(width=0), dict(width=9), dict(rows=1 << 31), dict(rows=(1 << 31) - 1, channels=1 << 30)]),
    ("dft_prompt_gdn", gdn_args, INVALID, [
        dict(batch=-1), dict(max_len=-1), dict(rows=-1), dict(slots=-1), dict(hk=0), dict(hv=0), dict(hk=2, hv=3),
        dict(y=None), dict(a=None), dict(b=None), dict(o=None), dict(A_log=None), dict(dt_bias=None), dict(state=None),
        dict(a_dtype=3), dict(b_dtype=4), dict(o_dtype=3), dict(A_log_dtype=3), dict(dt_bias_dtype=4),
        dict(state_indices=16, state_indices_dtype=1), dict(y=24), dict(y_row_stride=516)]),
    ("dft_prompt_gdn", gdn_args, UNSUPPORTED, [
        dict(dk=64), dict(dv=256), dict(rows=1 << 31), dict(batch=1 << 30)]),
    ("dft_tree_accept", accept_args, INVALID, [
        dict(batch=-1), dict(n_nodes=-1), dict(vocab=-1), dict(rows=-1), dict(path_cols=0), dict(tokens=None),
        dict(parent=None), dict(probs=None), dict(uniform=None), dict(last=None), dict(path=None), dict(path_len=None),
        dict(path_rows=None), dict(token=None), dict(tokens_dtype=0), dict(parent_dtype=2), dict(probs_dtype=3),
        dict(draft_probs=16, draft_dtype=4)]),
    ("dft_tree_accept", accept_args, UNSUPPORTED, [
        dict(n_nodes=65), dict(path_cols=65), dict(batch=65536), dict(rows=1 << 31), dict(vocab=(1 << 30) + 1)]),
]


@pytest.mark.parametrize("name,make,status,cases", REFUSED)
def test_refused_before_any_launch(name, make, status, cases):
    from dforktree_amd import _lib
    fn = getattr(_lib.load(), name)
    assert fn(None, None) == _lib.DFT_ERR_INVALID
    for case in cases:
        a = make()
        for k, v in case.items():
            setattr(a, k, v)
        assert fn(ctypes.byref(a), None) == status, case
    a = make()
    a.batch = 0  # nothing to do
    assert fn(ctypes.byref(a), None) == _lib.DFT_OK


@pytest.mark.parametrize("name,make,bad", [("dft_prompt_gdn", gdn_args, dict(hv=3, hk=2)),
                                           ("dft_tree_accept", accept_args, dict(path_cols=0))])
def test_workspace_is_asked_for_and_checked(name, make, bad):
    """Its size is known before there are buffers; a launch with less of it, or an unaligned one, is refused."""
    from dforktree_amd import _lib
    lib = _lib.load()
    n, a = ctypes.c_int64(-1), make()
    if name == "dft_prompt_gdn":
        a.max_len, a.rows = 300, 600
    size = getattr(lib, name + "_workspace")
    assert size(ctypes.byref(a), None) == _lib.DFT_ERR_INVALID
    blank = type(a)()
    for f, t in a._fields_:
        if t is not ctypes.c_void_p:
            setattr(blank, f, getattr(a, f))
    assert size(ctypes.byref(blank), ctypes.byref(n)) == _lib.DFT_OK and n.value > 0
    for k, v in bad.items():
        setattr(blank, k, v)
    want = n.value
    assert size(ctypes.byref(blank), ctypes.byref(n)) == _lib.DFT_ERR_INVALID and n.value == 0
    for change in (dict(workspace=None), dict(workspace=24), dict(workspace_bytes=want - 1)):
        b = make()
        b.rows = a.rows
        if name == "dft_prompt_gdn":
            b.max_len = a.max_len
        for k, v in change.items():
            setattr(b, k, v)
        assert getattr(lib, name)(ctypes.byref(b), None) == _lib.DFT_ERR_INVALID, change


def test_operators_take_gpu_tensors():
    import torch
    from dforktree_amd import ops
    f, i = torch.zeros, torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.prompt_conv(f(4, 8), f(1, 8, 3), f(8, 4))
    y, g = f(4, 512, dtype=torch.bfloat16), f(4, 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.prompt_gdn(y, g, g, f(2), f(2), f(1, 2, 128, 128), hk=1, hv=2)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_gdn(y, g, g, f(2), f(2), f(4, 2, 128, 128), hk=1, hv=2)
    with pytest.raises(ValueError, match="GPU"):
        ops.tree_accept(i, i, f(4, 10), f(4), f(1))


@pytest.mark.parametrize("current", [0, 1])
def test_launched_with_the_tensors_device_current(monkeypatch, current):
    """The default stream's handle is 0 on every device: it names the current one's."""
    import contextlib
    from types import SimpleNamespace

    import torch
    from dforktree_amd import _lib, ops
    seen, at = [], [current]

    @contextlib.contextmanager
    def device(dev):
        was, at[0] = at[0], dev.index
        yield
        at[0] = was

    def entry(args, stream):
        seen.append((at[0], stream))
        return _lib.DFT_OK

    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "load", lambda: SimpleNamespace(dft_prompt_conv=entry))
    ops._launch("dft_prompt_conv", _lib.PromptConvArgs(), torch.device("cuda", 1))
    assert seen == [(1, 0)] and at == [current]
