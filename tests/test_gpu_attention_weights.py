"""Many keys of small weights beside one of a large weight, in fp16.

Weights below 2^-14 of fp16 lose their relative precision.  They are taken against a reference that leaves the row's
largest at 2^7 or more, so a key's error stays at half of fp16's last step, 2^-25, over 2^7 of the row's sum.  With u
the half step, eps the error of a 32-bit score and fp32 outputs,

    |o - exact| <= (u + 2 eps + (L + 64) 2^-24) sum_j p_j |v_j| + L 2^-32 max |v|
"""
import numpy as np
import pytest
import torch

from conftest import announce
from test_gpu_attention import dense

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def inputs(L, d, hkv, seed):
    """Scores (of a query (1, 0, ..)) of 18.7 for key 3, of -2 to 2 for the others, whose values are near 1."""
    g = torch.Generator().manual_seed(seed)
    k = torch.zeros(L, hkv, d)
    k[..., 0] = 4 * torch.rand(L, hkv, generator=g) - 2
    k[3, :, 0] = 18.71875
    v = 1 + torch.rand(L, hkv, d, generator=g)
    v[3] = 0
    return k.to(F16), v.to(F16)


def check(o, q, k, v, sees, what):
    L, d = k.shape[0], k.shape[2]
    exact, _, weight, reach = dense(q.double(), k.double(), v.double(), sees, 1.0)
    eps = (d + 8) * 2.0 ** -24 * reach
    tol = (2.0 ** -11 + 2 * eps + (L + 64) * 2.0 ** -24)[..., None] * weight + L * 2.0 ** -32 * float(v.abs().max())
    off = (o.double().cpu() - exact).abs()
    assert (off <= tol).all(), f"{what}: off by {(off / tol).max():.2f} of the bound, {off.max():.2e} of {exact.max():.2e}"


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,hq,hkv", [(1, 1, 1), (1, 24, 1), (40, 4, 1)])
@pytest.mark.parametrize("L", [500, 40000])
def test_paged(cuda, d, rows, hq, hkv, L):
    """Every kernel, cut over workgroups and, with a short table, not."""
    from dforktree_amd import ops
    announce(f"small weights d={d} rows={rows} hq={hq} keys={L}")
    k, v = inputs(L, d, hkv, d)
    ps = 500
    q = torch.zeros(rows, hq, d, dtype=F16)
    q[..., 0] = 1
    o = torch.empty(rows, hq, d, dtype=F32, device=cuda)
    table = torch.arange(L // ps, dtype=torch.int32, device=cuda)[None]
    ops.paged_attention(q.to(cuda), k.view(-1, ps, hkv, d).to(cuda), v.view(-1, ps, hkv, d).to(cuda), table,
                        torch.tensor([L], device=cuda), causal=False, scale=1.0, o=o)
    torch.cuda.synchronize()
    check(o, q, k, v, np.ones((rows, L), bool), f"d={d} rows={rows}")


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt(cuda, d):
    from dforktree_amd import ops
    L = 3000
    announce(f"small weights of a prompt d={d}")
    k, v = inputs(L, d, 1, d)
    q = torch.zeros(L, 2, d, dtype=F16)
    q[..., 0] = 1
    o = torch.empty(L, 2, d, dtype=F32, device=cuda)
    ops.prompt_attention(q.to(cuda), k.to(cuda), v.to(cuda), scale=1.0, o=o)
    torch.cuda.synchronize()
    check(o, q, k, v, np.tril(np.ones((L, L), bool)), f"prompt d={d}")


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,hq", [(1, 1), (40, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, F16])
def test_huge_scores(cuda, d, rows, hq, dtype):
    """Scores of up to 2^26 in log2 units, whose own rounding is some of them: outputs stay finite, as an average of the
    values does."""
    from dforktree_amd import ops
    announce(f"huge scores d={d} rows={rows} {dtype}")
    L, ps = 1000, 20
    g = torch.Generator().manual_seed(d)
    k = (torch.rand(L, 1, d, generator=g) * 2 - 1) * 2.0 ** 12
    k[:, 0, 0] = torch.linspace(0, 2.0 ** 13, L)
    q = torch.full((rows, hq, d), 0.0)
    q[..., 0] = 2.0 ** 12
    q[..., 1] = 2.0
    v = torch.rand(L, 1, d, generator=g)
    table = torch.arange(L // ps, dtype=torch.int32, device=cuda)[None]
    o = ops.paged_attention(q.to(cuda, dtype), k.to(cuda, dtype).view(-1, ps, 1, d), v.to(cuda, dtype).view(-1, ps, 1, d), table,
                            torch.tensor([L], device=cuda), causal=False, scale=1.0)
    p = ops.prompt_attention(q.to(cuda, dtype)[:1].expand(L, hq, d), k.to(cuda, dtype), v.to(cuda, dtype), scale=1.0)
    torch.cuda.synchronize()
    for x in (o, p):
        assert torch.isfinite(x).all() and (x >= 0).all() and (x <= 1.01).all()
