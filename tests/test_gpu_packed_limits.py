"""The ends of what the packed operators take: sizes of nothing, and outputs that must not be laid over other memory."""
import pytest
import torch

from conftest import announce
from oracle import packed as P

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("W", [1, 4])
def test_conv_without_channels(cuda, W):
    """There is nothing to compute, but the requests' status is told as ever."""
    from dforktree_amd import ops
    announce(f"prompt_conv without channels W={W}")
    x = torch.zeros(6, 0, dtype=BF16, device=cuda)
    state, weight = torch.zeros(2, 0, W - 1, dtype=BF16, device=cuda), torch.zeros(0, W, dtype=BF16, device=cuda)
    cu = torch.tensor([0, 3, 3, 6], dtype=torch.int32, device=cuda)
    status = torch.full((3,), -1, dtype=torch.int32, device=cuda)
    at = torch.tensor([1, -1, 2], device=cuda)
    y = ops.prompt_conv(x, state, weight, None, cu, max_len=2, cs_indices=at, status=status)
    assert y.shape == (6, 0) and status.tolist() == [P.STATUS_SPAN, 0, P.STATUS_SPAN | P.STATUS_SLOT]
    assert ops.prompt_conv(x, state, weight, batch=2).shape == (6, 0)


def conv(cuda, rows=6, C=8):
    x = torch.randn(rows, C, device=cuda).to(BF16)
    return x, torch.zeros(1, C, 3, dtype=BF16, device=cuda), torch.randn(C, 4, device=cuda).to(BF16)


def test_conv_outputs_have_memory_of_their_own(cuda):
    from dforktree_amd import ops
    x, state, w = conv(cuda)
    wide = torch.zeros(8, 40, dtype=BF16, device=cuda)
    inside = wide[:6, 4:12]
    for x_, y in ((x, x), (x, x.new_empty(1, 8).expand(6, 8)), (x, x.new_empty(48).as_strided((6, 8), (7, 1))),
                  (inside, wide[:6, 8:16]), (inside, wide[2:, 4:12]), (inside, wide[1:7, :8]),
                  (inside[:1], wide[:1, 11:19]), (x, x.view(-1)[4:].as_strided((5, 8), (8, 1)))):
        with pytest.raises(ValueError, match="must not lie over"):
            ops.prompt_conv(x_[:y.shape[0]], state, w, y=y)


def test_conv_beside_its_input(cuda):
    """Rows side by side in one buffer, or behind each other, share no memory."""
    from dforktree_amd import ops
    announce("prompt_conv beside its input")
    x, state, w = conv(cuda)
    want = ops.prompt_conv(x, state.clone(), w)
    for a, b in ((0, 8), (8, 0), (3, 11), (30, 2)):
        wide = torch.zeros(6, 40, dtype=BF16, device=cuda)
        wide[:, a:a + 8] = x
        ops.prompt_conv(wide[:, a:a + 8], state.clone(), w, y=wide[:, b:b + 8])
        assert torch.equal(wide[:, b:b + 8], want) and torch.equal(wide[:, a:a + 8], x)
    both = torch.cat([x, x])
    ops.prompt_conv(both[:6], state.clone(), w, y=both[6:])
    assert torch.equal(both[6:], want)


def gdn(cuda, rows, wider=0):
    g = torch.Generator().manual_seed(rows)
    y = torch.randn(rows, 512 + wider, generator=g).to(BF16).to(cuda)
    a, b = (torch.randn(rows, 2, generator=g).to(cuda) for _ in range(2))
    rest = torch.zeros(2, device=cuda), torch.zeros(2, device=cuda), torch.zeros(1, 2, 128, 128, device=cuda)
    return y, (a, b, *rest)


def test_gdn_outputs_have_memory_of_their_own(cuda):
    from dforktree_amd import ops
    y, rest = gdn(cuda, 6)
    empty = lambda *s: torch.empty(*s, dtype=BF16, device=cuda)  # noqa: E731
    for o in (empty(1, 2, 128).expand(6, 2, 128), empty(6, 1, 128).expand(6, 2, 128), y[:, :256].unflatten(1, (2, 128)),
              y[:, 256:].unflatten(1, (2, 128)), empty(2000).as_strided((6, 2, 128), (256, 64, 1)),
              y.view(-1)[:1536].view(6, 2, 128)):
        with pytest.raises(ValueError, match="must not lie over"):
            ops.prompt_gdn(y, *rest, hk=1, hv=2, o=o)


@pytest.mark.parametrize("rows", [5, 70])
def test_gdn_beside_its_input(cuda, rows):
    from dforktree_amd import ops
    announce(f"prompt_gdn beside its input, {rows} rows")
    y, rest = gdn(cuda, rows, 256)
    run = lambda y, **kw: ops.prompt_gdn(y, *rest[:4], rest[4].clone(), hk=1, hv=2, **kw)  # noqa: E731
    want = run(y[:, :512].contiguous())
    o = y[:, 512:].unflatten(1, (2, 128))
    assert torch.equal(run(y[:, :512], o=o), want) and torch.equal(o, want)
    assert torch.equal(run(y, o=o), want)  # columns past the values are not read
    apart = torch.zeros(2, rows, 128, dtype=BF16, device=cuda)  # heads behind each other
    assert torch.equal(run(y, o=apart.transpose(0, 1)), want)
