"""PagedKV's own bookkeeping on the CPU, its four operators replaced by the oracle's."""
from types import SimpleNamespace

import pytest
import torch

from oracle import paged as P

NAMES = ("slots", "positions", "cu_seqlens", "seq_len", "held", "free_pos", "status")


def page_plan(prefix_len, new_len, block_table, held, free_pages, free_pos, *, page_size, rows, trim=False, depth=None):
    r = P.page_plan(*(x.numpy() for x in (prefix_len, new_len, block_table, held, free_pages, free_pos)), page_size=page_size,
                    rows=rows, trim=trim, depth=None if depth is None else depth.numpy())
    block_table.copy_(torch.from_numpy(r["block_table"]))
    free_pages.copy_(torch.from_numpy(r["free_pages"]))
    return {name: torch.from_numpy(r[name]) for name in NAMES}


def kv_append(k, v, key_cache, value_cache, slots, rows=None):
    kc, vc, status = P.kv_append(k.numpy(), v.numpy(), key_cache.numpy(), value_cache.numpy(), slots.reshape(-1).tolist(),
                                 None if rows is None else rows.reshape(-1).tolist())
    assert status == 0
    key_cache.copy_(torch.from_numpy(kc))
    value_cache.copy_(torch.from_numpy(vc))


@pytest.fixture
def make(monkeypatch):
    from dforktree_amd import paged
    monkeypatch.setattr(paged, "ops", SimpleNamespace(page_plan=page_plan, kv_append=kv_append))
    return lambda *a: paged.PagedKV(*a, 1, 1, dtype=torch.float32, device="cpu")


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def marks(*x):
    """Rows [n, 1, 1] whose key and value say whose they are."""
    return torch.tensor(x, dtype=torch.float32).view(-1, 1, 1)


def tokens(kv, b):
    """The keys that request b's next attention takes as committed."""
    return P.paged_keys(kv.keys[0].numpy(), kv.block_table[b].numpy(), int(kv.prefix[b]))[0].reshape(-1).tolist()


def test_a_refused_request_does_not_grow(make):
    """Two pages of four tokens: request 0 finds none for its fifth token until request 1 has ended."""
    kv = make(1, 2, 4, 2, 4)
    plan = kv.plan(ints(4, 3), rows=7, n_new=4)
    x = marks(10, 11, 12, 13, 20, 21, 22)
    kv.append(0, x, x, plan)
    kv.commit(ints(4, 3))
    plan = kv.plan(ints(1, 1), rows=2, n_new=1)
    assert plan["status"].tolist() == [P.STATUS_PAGES, 0]
    x = marks(14, 23)
    kv.append(0, x, x, plan)
    kv.commit(ints(1, 1))
    assert kv.prefix.tolist() == [4, 4]
    kv.prefix[1] = 0  # request 1 ends
    plan = kv.plan(ints(0, 0), rows=0, n_new=0, trim=True)
    kv.commit(ints(0, 0))
    plan = kv.plan(ints(1, 0), rows=1, n_new=1)
    assert not plan["status"].any()
    x = marks(14)
    kv.append(0, x, x, plan)
    kv.commit(ints(1, 0))
    assert tokens(kv, 0) == [10, 11, 12, 13, 14]


def test_a_full_table_and_cut_lengths_do_not_grow(make):
    kv = make(1, 3, 2, 9, 2)
    plan = kv.plan(ints(3, 5, 2), rows=9, n_new=5)  # two pages of two are too few for request 1; a row for request 2's two
    assert plan["status"].tolist() == [0, P.STATUS_TABLE, P.STATUS_SPAN]
    kv.commit(ints(3, 5, 2))
    assert kv.prefix.tolist() == [3, 0, 1]


def test_a_plan_commits_no_more_than_it_placed(make):
    """In pieces, and not again without a plan; an int64 length of an accepted path."""
    kv = make(1, 1, 4, 4, 4)
    kv.plan(ints(5), rows=5, n_new=5)
    for length, prefix in ((ints(2), 2), (torch.tensor([2]), 4), (ints(2), 5), (ints(1), 5)):
        kv.commit(length)
        assert kv.prefix.tolist() == [prefix] and kv.prefix.dtype == torch.int32


def test_a_cut_request_keeps_to_its_own_places(make):
    """The rows end inside request 1's tree and before request 2's: what of their paths has no place is left out."""
    kv = make(1, 3, 4, 9, 4)
    plan = kv.plan(ints(2, 4, 3), rows=4, n_new=4)
    assert plan["status"].tolist() == [0, P.STATUS_SPAN, P.STATUS_SPAN]
    x = marks(10, 11, 20, 21, 22, 23, 30, 31, 32)
    kv.accept(0, x, x, plan, torch.tensor([[0, 1, -1], [2, 3, 5], [6, 7, 8]]))
    kv.commit(ints(2, 3, 3))
    assert kv.prefix.tolist() == [2, 2, 0]
    assert tokens(kv, 0) == [10, 11] and tokens(kv, 1) == [20, 21]
    assert sorted(kv.keys[kv.keys != 0].tolist()) == [10, 11, 20, 21]
    kv.prefix.zero_()
    plan = kv.plan(ints(0, 4, 3), rows=4, n_new=4)  # request 2 follows a whole one
    kv.keys.zero_()
    kv.accept(0, x, x, plan, torch.tensor([[0, 1, -1], [2, 3, 5], [6, 7, 8]]))
    assert sorted(kv.keys[kv.keys != 0].tolist()) == [20, 21, 23]


def test_a_step_without_rows(make):
    """Every request waits: nothing is written, and no slot of none is looked up."""
    kv = make(1, 2, 4, 9, 4)
    plan = kv.plan(ints(0, 0), rows=0, n_new=0)
    kv.accept(0, marks(), marks(), plan, torch.full((2, 3), -1))
    kv.commit(ints(0, 0))
    assert not kv.keys.any() and kv.prefix.tolist() == [0, 0]


def test_two_plans_of_one_step(make):
    """A prompt and a single token planned apart: each plan says what is to be committed of it."""
    kv = make(1, 2, 4, 9, 4)
    prompt = kv.plan(ints(6, 0), rows=6, n_new=6)
    token = kv.plan(ints(0, 1), rows=1, n_new=1)
    kv.append(0, *[marks(10, 11, 12, 13, 14, 15)] * 2, prompt)
    kv.append(0, *[marks(20)] * 2, token)
    kv.commit(ints(6, 0), prompt)
    kv.commit(ints(0, 1), token)
    assert tokens(kv, 0) == [10, 11, 12, 13, 14, 15] and tokens(kv, 1) == [20]
    kv.commit(ints(6, 0), prompt)
    assert kv.prefix.tolist() == [6, 1]
