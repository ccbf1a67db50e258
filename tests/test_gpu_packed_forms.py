"""The forms that the packed operators take by their types, layouts and the work there is: tests of each beside the
oracle, where tests of their sizes keep to few heads, few requests and one type."""
import numpy as np
import pytest
import torch

import test_gpu_accept as A
from conftest import announce, rel_l2
from test_gpu_gdn import BF16, F16, F32, Case, cu_of
from test_gpu_gdn_precision import OUT, STATE

pytestmark = pytest.mark.gpu


# ---- accepted paths: probabilities of every type, over short rows and in slices --------------------------------------
@pytest.mark.parametrize("V", [777, 20001])
@pytest.mark.parametrize("probs,draft", [(F32, BF16), (BF16, F32), (BF16, F16), (F16, BF16), (F16, F32)])
def test_accept_of_unlike_types(cuda, V, probs, draft):
    for kind, seed in (("tree", 60), ("star", 61)):
        c = A.Case([7, 30, 2, 12], V, kind, True, seed, dtype=probs)
        c.draft = c.draft.float().to(draft)
        if kind == "star":
            c.u.mul_(0.5).add_(0.5)
        c.check(cuda, label=f"{kind} {probs} {draft}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [20001, 131072])
def test_accept_of_16_bits_over_long_rows(cuda, dtype, drawn, V):
    for kind, seed in (("tree", 62), ("star", 63)):
        c = A.Case([9, 1, 20], V, kind, drawn, seed, dtype=dtype)
        if kind == "star":
            c.u.mul_(0.5).add_(0.5)
        c.check(cuda, label=f"{kind} {dtype}")


@pytest.mark.parametrize("dtype,draft", [(BF16, BF16), (F16, F16), (BF16, F32)])
def test_accept_of_16_bits_at_odd_places(cuda, dtype, draft):
    for V in (779, 20003):
        c = A.Case([9, 30, 4], V, "star", True, 64, dtype=dtype)
        c.u.mul_(0.5).add_(0.5)
        for name, at, t in (("probs", 3, dtype), ("draft", 5, draft)):
            wide = torch.full((43, V + 10), float("nan"), dtype=t, device=cuda)
            wide[:, at:at + V] = getattr(c, name)
            setattr(c, name, wide[:, at:at + V])
        c.check(cuda, label=f"odd places {dtype} {draft}")


# ---- GDN ------------------------------------------------------------------------------------------------------------
def recurrence(c, sizes):
    """Outputs and states in 64 bits on the GPU, the requests side by side, each from its slot."""
    rows, D = len(c.y), 128
    q, k, v = (t.unflatten(1, (-1, D)) for t in c.y.double().split([c.hk * D, c.hk * D, c.hv * D], 1))
    q, k = (t / torch.sqrt((t * t).sum(2, keepdim=True) + 1e-6) for t in (q, k))
    q, k = (t.repeat_interleave(c.hv // c.hk, 1) for t in (q * D ** -0.5, k))
    x = c.a.double() + c.dt_bias.double()
    decay = torch.exp(-torch.exp(c.A_log).double() * torch.logaddexp(x, torch.zeros_like(x)))  # (the rate in 32 bits)
    beta = 1 / (1 + torch.exp(-c.b.double()))
    S = c.pool.double()[:len(sizes)]  # [request, head, v, k]
    o = torch.empty(rows, c.hv, D, dtype=torch.float64, device=c.y.device)
    first = torch.tensor(np.cumsum([0, *sizes[:-1]]), device=c.y.device)
    n = torch.tensor(sizes, device=c.y.device)
    for t in range(max(sizes)):
        at = (n > t).nonzero()[:, 0]
        r = first[at] + t
        s = S[at] * decay[r][:, :, None, None]
        u = beta[r][:, :, None] * (v[r] - (s * k[r][:, :, None]).sum(3))
        s = s + u[:, :, :, None] * k[r][:, :, None]
        o[r] = (s * q[r][:, :, None]).sum(3)
        S[at] = s
    return o, S


def check(c, sizes, cuda, layout, o, label):
    from dforktree_amd import ops
    host, cu = cu_of(sizes, cuda)
    announce(f"prompt_gdn {label} {layout} {len(sizes)} requests, {host[-1]} rows, {c.hk} and {c.hv} heads")
    want, want_state = recurrence(c, sizes)
    state = c.pool.transpose(-1, -2)
    state = state.contiguous() if layout == "k first" else state
    ops.prompt_gdn(c.y, c.a, c.b, None, c.dt_bias, state, cu, hk=c.hk, hv=c.hv, max_len=max(sizes), o=o,
                   neg_exp_A=-torch.exp(c.A_log))
    for b in range(len(sizes)):
        assert rel_l2(state[b].cpu(), want_state[b].transpose(-1, -2).cpu()) <= STATE, (label, b)
    half = torch.finfo(o.dtype).eps / 2 if o.dtype != F32 else 0
    err = (o.double() - want).abs()
    least = 2.0 ** -25 if o.dtype == F16 else 0  # half of fp16's smallest step
    assert (err <= half * want.abs() + 2.0 ** -19 * want.abs().max() + least).all(), label
    if o.dtype == F32:
        assert rel_l2(o.cpu(), want.cpu()) <= OUT, (label, rel_l2(o.cpu(), want.cpu()))


# (requests, heads): few heads each of 32 columns a workgroup and whole ones, row by row; 16 and 32 columns in chunks
FORMS = {"rows, few": ([1, 5, 7, 3], 1, 2), "rows": ([1] * 70, 4, 8), "rows of 16": ([16, 1, 9] * 30, 2, 8),
         "one column tile": ([200, 70], 1, 2), "two column tiles": ([100] * 40, 2, 8),
         "two column tiles, long": ([1300, 1290, 1100], 8, 32), "rows beside chunks": ([1, 16, 17, 100] * 18, 2, 8)}


@pytest.mark.parametrize("layout", ["k first", "k last"])
@pytest.mark.parametrize("o_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("form", FORMS)
def test_gdn_forms(cuda, form, o_dtype, layout):
    sizes, hk, hv = FORMS[form]
    c = Case(sum(sizes), hk, hv, len(sizes), cuda, seed=70, gates=F32)
    check(c, sizes, cuda, layout, torch.empty(sum(sizes), hv, 128, dtype=o_dtype, device=cuda), form)


@pytest.mark.parametrize("o_dtype", [BF16, F32])
@pytest.mark.parametrize("form", ["rows", "one column tile", "two column tiles"])
def test_gdn_outputs_at_odd_places(cuda, form, o_dtype):
    sizes, hk, hv = FORMS[form]
    c = Case(sum(sizes), hk, hv, len(sizes), cuda, seed=71, gates=F32)
    wide = torch.zeros(sum(sizes), hv, 131, dtype=o_dtype, device=cuda)
    check(c, sizes, cuda, "k last", wide[:, :, 1:129], form)
    assert not wide[:, :, 0].any() and not wide[:, :, 129:].any()


@pytest.mark.parametrize("n,beside", [(100, [64, 1, 300]), (100, [100] * 39), (100, [3, 90] * 70), (1, [1] * 300),
                                      (5, [7, 1, 2]), (12, [16, 9] * 70)])
def test_gdn_alone_as_beside_others(cuda, n, beside):
    """What a request gets does not depend on those beside it, where they leave it in the same form: 32 value columns a
    workgroup are 16 twice, and a head's columns over four workgroups the same sums as in one."""
    from dforktree_amd import ops
    sizes = [*beside, n]
    host, cu = cu_of(sizes, cuda)
    announce(f"prompt_gdn {n} rows alone and beside {len(beside)} requests")
    c = Case(sum(sizes), 2, 8, len(sizes), cuda, seed=72)
    pool, alone = c.pool.clone(), c.pool[-1:].clone()
    o = ops.prompt_gdn(c.y, c.a, c.b, c.A_log, c.dt_bias, pool.transpose(-1, -2), cu, hk=2, hv=8, max_len=max(sizes), o_dtype=F32)
    r = slice(host[-2], None)
    repeat = 70 if n == 12 else 1  # (up to 16 rows are taken row by row where there are 512 heads)
    own = torch.cat([alone] * repeat).transpose(-1, -2)
    again = ops.prompt_gdn(*(t[r].repeat(repeat, 1) for t in (c.y, c.a, c.b)), c.A_log, c.dt_bias, own, hk=2, hv=8, max_len=n,
                           batch=repeat, o_dtype=F32)
    assert torch.equal(o[r], again[:n]) and torch.equal(pool[-1], own[0].transpose(-1, -2))
