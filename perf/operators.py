"""The operators of the hybrid model's full-attention layers, as measurable cases.

The GDN layers of a speculative decoding step have their own kernels; the
full-attention layers beside them keep a paged KV cache.  A case is one pass
through one operator of that half:

plan     page tables, slot maps and positions of a batch, built on the GPU
         from the request lengths (``ops.page_plan``)
append   new K/V rows into their pages, or the rows of an accepted path
         (``ops.kv_append``)
paged    attention of each request's new tokens over its pages: one token, a
         draft tree, a chunk of a long prompt (``ops.paged_attention``)
prompt   attention over whole prompts, packed (``ops.prompt_attention``)

``own`` false: the operators in elementary torch operations, in 32 bits,
rounded once at the end.  ``own`` true: the package's kernels.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_PATH = 16  # columns of an accepted path (-1 padded)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a decode step of a full server: one token per request
        dict(name="plan_decode", op="plan", batch=64, new_lo=1, new_hi=1, pre_lo=17, pre_hi=4096, page=16, trim=False,
             depth=False),
        # draft trees of every size after a step that accepted part of the last one: pages come and go
        dict(name="plan_trees", op="plan", batch=128, new_lo=8, new_hi=64, pre_lo=100, pre_hi=9000, page=1, trim=True,
             depth=True),
        # chunks of many long prompts at once
        dict(name="plan_chunks", op="plan", batch=1000, new_lo=1, new_hi=511, pre_lo=0, pre_hi=16384, page=16, trim=True,
             depth=False),
        # the accepted paths of 64 draft trees, gathered to their final places
        dict(name="append_paths", op="append", batch=64, rows=32, path=True, hkv=2, d=256, page=16, type="bf16",
             heads_first=False),
        # a step's worth of prompt chunks, K and V as slices of one projection
        dict(name="append_chunk", op="append", batch=7, rows=2341, path=False, hkv=8, d=128, page=64, type="bf16",
             heads_first=True),
        # decode of a full, ragged batch
        dict(name="paged_decode", op="paged", batch=64, new_lo=1, new_hi=1, pre_lo=300, pre_hi=8191, hq=32, hkv=8, d=128,
             page=16, type="bf16", mask="causal", lse=False),
        # one request at a long context
        dict(name="paged_long", op="paged", batch=1, new_lo=1, new_hi=1, pre_lo=131000, pre_hi=131000, hq=16, hkv=2,
             d=256, page=64, type="f16", mask="causal", lse=True),
        # the verify step: a 32-node draft tree per request
        dict(name="paged_trees", op="paged", batch=64, new_lo=32, new_hi=32, pre_lo=500, pre_hi=4000, hq=32, hkv=8,
             d=128, page=1, type="bf16", mask="tree", lse=False),
        # chunked prefill: a chunk of new tokens over a long prefix, two requests
        dict(name="paged_chunk", op="paged", batch=2, new_lo=777, new_hi=1024, pre_lo=9000, pre_hi=15001, hq=16, hkv=2,
             d=256, page=16, type="bf16", mask="causal", lse=True),
        # short prompts, few of them: latency
        dict(name="prompt_short", op="prompt", batch=3, lo=1, hi=130, hq=12, hkv=12, d=64, type="f16", causal=True,
             lse=False),
        # a packed batch of ordinary prompts
        dict(name="prompt_packed", op="prompt", batch=6, lo=257, hi=2999, hq=32, hkv=8, d=128, type="bf16", causal=True,
             lse=False),
        # one long prompt
        dict(name="prompt_long", op="prompt", batch=1, lo=8192, hi=8192, hq=32, hkv=8, d=128, type="bf16", causal=True,
             lse=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("plan", "append", "paged", "paged", "prompt", "prompt"))
    page = rng.choice((1, 8, 16, 24, 64, 256))
    d = rng.choice((64, 128, 256))
    hkv = rng.choice((1, 2, 4, 8))
    hq = hkv * rng.choice((1, 2, 4, 7, 8))
    kind = rng.choice(("bf16", "bf16", "f16"))
    if op == "plan":
        batch = _log(rng, 1, 1000)
        new = _log(rng, 1, 511)
        return dict(op=op, batch=batch, new_lo=_log(rng, 1, new), new_hi=new, pre_lo=0, pre_hi=_log(rng, 16, 16384),
                    page=page, trim=rng.random() < 0.5, depth=new <= 64)
    if op == "append":
        batch = _log(rng, 1, 64)
        path = rng.random() < 0.5
        return dict(op=op, batch=batch, rows=rng.randint(_PATH, 64) if path else _log(rng, 1, 16384 // batch), path=path,
                    hkv=hkv, d=d, page=page, type=kind, heads_first=rng.random() < 0.5)
    if op == "paged":
        mask = rng.choice(("causal", "tree", "all"))
        batch = _log(rng, 1, 64)
        new = rng.randint(1, 64) if mask == "tree" else 1 if rng.random() < 0.4 else _log(rng, 2, 1024)
        pre = _log(rng, 64, 131000)
        # the keys' and the scores' share of the largest listed case
        pre = max(1, min(pre, int(1.5e8 / (batch * hkv * d)), int(3.5e8 / (batch * new * hq))))
        new = min(new, max(1, int(5e7 / (batch * hq * d))), max(1, int(3.5e8 / (batch * hq * (pre + new)))))
        return dict(op=op, batch=batch, new_lo=_log(rng, 1, new), new_hi=new, pre_lo=rng.randint(0, pre), pre_hi=pre,
                    hq=hq, hkv=hkv, d=d, page=page, type=kind, mask=mask, lse=rng.random() < 0.5)
    batch = _log(rng, 1, 32)
    hi = _log(rng, 1, 8192)
    hi = max(1, min(hi, int(math.sqrt(1.3e11 / (batch * hq * d))), int(6e7 / (batch * hq * d))))
    return dict(op=op, batch=batch, lo=_log(rng, 1, hi), hi=hi, hq=hq, hkv=hkv, d=d, type=kind,
                causal=rng.random() < 0.8, lse=rng.random() < 0.5)


def _spread(n, lo, hi):
    """n lengths from lo to hi in a mixed order, the same for every seed."""
    at = np.argsort(np.argsort([(i * 0.6180339887498949) % 1.0 for i in range(n)]))
    return [hi] if n == 1 else [int(lo + (hi - lo) * int(a) // (n - 1)) for a in at]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(sizes):
    return [0, *np.cumsum(sizes).tolist()]


def _tables(held, columns, pages, gen):
    """Each request's pages, scattered over the cache; -1 past them."""
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    held = _ints(held, torch.int64)
    col = torch.arange(columns, device="cuda")
    at = (held.cumsum(0) - held)[:, None] + col
    return torch.where(col < held[:, None], order[at.clamp_max(pages - 1)], -1).contiguous(), order


def _rows(n, heads, d, dtype, gen, scale=1.0):
    return (torch.randn(n, heads, d, generator=gen, device="cuda") * scale).to(dtype)


def _parents(n, rng):
    """A draft tree in topological order: depth first favoured, as a drafter's best-first growth gives."""
    return [-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]


def _ancestry(parent):
    """Each node's ancestor-or-self bits, as int64."""
    bits = []
    for i, p in enumerate(parent):
        bits.append((bits[p] if p >= 0 else 0) | (1 << i))
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": case}
    if case["op"] == "plan":
        B, ps = case["batch"], case["page"]
        prefix, new = _spread(B, case["pre_lo"], case["pre_hi"]), _spread(B, case["new_lo"], case["new_hi"])[::-1]
        # what a request holds: its prefix's pages, and with trim what a rejected draft left it
        most = 1 + 80 // ps if case["trim"] else 0
        spare = rng.integers(0, most + 1, B)
        held = [-(-p // ps) + int(x) for p, x in zip(prefix, spare)]
        want = [-(-(p + n) // ps) for p, n in zip(prefix, new)]
        room = [max(-(-p // ps) + most, w) for p, w in zip(prefix, want)]
        pages, columns = sum(room) + 7, max(room) + 3
        s["block_table"], order = _tables(held, columns, pages, gen)
        free = order[sum(held):]
        head = int(rng.integers(0, 1 << 20))
        ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(free.numel(), device="cuda")) % pages] = free
        s |= {"prefix": _ints(prefix), "new": _ints(new), "held": _ints(held), "free": ring, "rows": sum(new),
              "pos": _ints([head, head + free.numel()], torch.int64), "depth": None}
        if case["depth"]:
            depth = []
            for n in new:
                level = []
                for p in _parents(n, rng):
                    level.append(level[p] + 1 if p >= 0 else 0)
                depth += level
            s["depth"] = _ints(depth)
        return s
    dtype = _TYPE[case["type"]]
    if case["op"] == "append":
        B, n, ps, hkv, d = case["batch"], case["rows"], case["page"], case["hkv"], case["d"]
        T = B * n
        s["k"], s["v"] = (torch.randn(T, 2 * hkv * d, generator=gen, device="cuda").to(dtype).view(T, 2, hkv, d)
                          .unbind(1))
        count = B * _PATH if case["path"] else T
        pages = -(-count // ps) + B + 5
        shape = (pages, hkv, ps, d) if case["heads_first"] else (pages, ps, hkv, d)
        for name in ("key_cache", "value_cache"):
            c = torch.randn(shape, generator=gen, device="cuda").to(dtype)
            s[name] = c.transpose(1, 2) if case["heads_first"] else c
        s["slots"] = torch.randperm(pages * ps, generator=gen, device="cuda")[:count]
        s["rows"] = None
        if case["path"]:  # increasing nodes of each tree, -1 past the accepted ones
            rows = np.full((B, _PATH), -1, np.int64)
            for b in range(B):
                m = int(rng.integers(1, _PATH + 1))
                rows[b, :m] = b * n + np.sort(rng.choice(n, m, replace=False))
            s["rows"] = _ints(rows.reshape(-1))
        return s
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "paged":
        B, ps = case["batch"], case["page"]
        prefix, new = _spread(B, case["pre_lo"], case["pre_hi"]), _spread(B, case["new_lo"], case["new_hi"])[::-1]
        total = [p + n for p, n in zip(prefix, new)]
        held = [-(-t // ps) for t in total]
        pages = sum(held) + 9
        s["block_table"], _ = _tables(held, max(held) + 1, pages, gen)
        s["key_cache"], s["value_cache"] = (
            torch.randn(pages, ps, hkv, d, generator=gen, device="cuda").to(dtype) for _ in range(2))
        s["q"] = _rows(sum(new), hq, d, dtype, gen, 1.5)
        s |= {"seq_len": _ints(total), "cu": _ints(_starts(new)), "n_new": max(new), "longest": max(total),
              "anc_bits": None}
        if case["mask"] == "tree":
            s["anc_bits"] = _ints([b for n in new for b in _ancestry(_parents(n, rng))], torch.int64)
        return s
    sizes = _spread(case["batch"], case["lo"], case["hi"])
    T = sum(sizes)
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=gen, device="cuda").to(dtype).view(T, hq + 2 * hkv, d)
    s |= {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hkv], "v": qkv[:, hq + hkv:], "cu": _ints(_starts(sizes)),
          "longest": max(sizes)}
    return s


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "append": _append, "paged": _paged, "prompt": _prompt}[state["case"]["op"]](state)


def _own(s):
    from dforktree_amd import ops
    case = s["case"]
    if case["op"] == "plan":
        r = ops.page_plan(s["prefix"], s["new"], s["block_table"], s["held"], s["free"], s["pos"], page_size=case["page"],
                          rows=s["rows"], trim=case["trim"], depth=s["depth"])
        return r | {"block_table": s["block_table"], "free_pages": s["free"]}
    if case["op"] == "append":
        ops.kv_append(s["k"], s["v"], s["key_cache"], s["value_cache"], s["slots"], rows=s["rows"])
        return {"key_cache": s["key_cache"], "value_cache": s["value_cache"]}
    lse = torch.empty(s["q"].shape[:2], device="cuda") if case["lse"] else None
    if case["op"] == "paged":
        o = ops.paged_attention(s["q"], s["key_cache"], s["value_cache"], s["block_table"], s["seq_len"],
                                cu_seqlens=s["cu"], n_new=s["n_new"], causal=case["mask"] == "causal",
                                anc_bits=s["anc_bits"], lse=lse)
    else:
        o = ops.prompt_attention(s["q"], s["k"], s["v"], s["cu"], max_len=s["longest"], causal=case["causal"], lse=lse)
    return {"o": o, "lse": lse} if case["lse"] else {"o": o}


def _plan(s):
    """Requests' page counts by cumulative sums; every row's page by a search for its request."""
    case = s["case"]
    ps, rows = case["page"], s["rows"]
    table, held, ring, pos = s["block_table"], s["held"].long(), s["free"], s["pos"]
    columns, cap = table.shape[1], ring.numel()
    prefix = s["prefix"].long().clamp_min(0)
    end = s["new"].long().clamp_min(0).cumsum(0).clamp_max(rows)
    start = torch.cat([end.new_zeros(1), end[:-1]])
    new = end - start
    want = (prefix + new + ps - 1) // ps
    fits = want <= columns
    need = torch.where(fits, (want - held).clamp_min(0), 0)
    need_end = need.cumsum(0)
    room = pos[1] - pos[0]
    served = fits & ((need == 0) | (need_end <= room))
    give = torch.where(served, held - want, 0).clamp_min(0) if case["trim"] else torch.zeros_like(held)
    give_start = give.cumsum(0) - give
    col = torch.arange(columns, device=table.device)
    first = pos[0] + need_end - need
    fresh = ring[(first[:, None] + col - held[:, None]) % cap]
    grown = served[:, None] & (col >= held[:, None]) & (col < want[:, None])
    back = (give > 0)[:, None] & (col >= want[:, None]) & (col < held[:, None])
    to = torch.where(back, (pos[1] + give_start[:, None] + col - want[:, None]) % cap, cap)
    table.copy_(torch.where(grown, fresh, table))
    more = torch.cat([ring, ring.new_zeros(1)]).scatter(0, to.reshape(-1), table.reshape(-1))
    ring.copy_(more[:cap])
    row = torch.arange(rows, device=table.device)
    of = torch.searchsorted(end, row, right=True)
    place = prefix[of] + row - start[of]
    slot = table[of, (place // ps).clamp_max(columns - 1)].long() * ps + place % ps
    at = prefix[of] + s["depth"].long() if case["depth"] else place
    taken = torch.where(served, need, 0).sum()
    held = torch.where(served, torch.where(give > 0, want, torch.maximum(held, want)), held)
    return {"slots": torch.where(served[of], slot, -1), "positions": at,
            "cu_seqlens": torch.cat([start[:1], end]).int(), "seq_len": torch.where(served, prefix + new, 0).int(),
            "held": held.int(), "free_pos": torch.stack([pos[0] + taken, pos[1] + give.sum()]),
            "status": torch.where(fits, torch.where(served, 0, 8), 16).int(), "block_table": table, "free_pages": ring}


def _append(s):
    k, v, slots = s["k"], s["v"], s["slots"]
    page, at = slots // s["case"]["page"], slots % s["case"]["page"]
    rows = s["rows"] if s["rows"] is not None else torch.arange(slots.numel(), device=slots.device)
    kept = (rows >= 0)[:, None, None]
    rows = rows.clamp_min(0)
    for name, new in (("key_cache", k), ("value_cache", v)):
        cache = s[name]
        cache[page, at] = torch.where(kept, new[rows].to(cache.dtype), cache[page, at])
    return {"key_cache": s["key_cache"], "value_cache": s["value_cache"]}


def _softmax_sum(q, k, v, sees, scale):
    """q [B, hkv, rows, d], k / v [B, hkv, keys, d], sees [B, 1, rows, keys]: the outputs and the scores' log-sum-exp."""
    x = torch.matmul(q, k.transpose(2, 3)).mul_(scale).masked_fill_(~sees, -math.inf)
    top = x.amax(3, keepdim=True).clamp_min(-3e38)
    x = x.sub_(top).exp_()
    total = x.sum(3, keepdim=True)
    o = torch.matmul(x, v) / torch.where(total > 0, total, 1)
    return o, (top + total.log())[..., 0]


def _grouped(x, at, hkv):
    """Packed rows [T, hq, d] as [B, hkv, rows * group, d] in 32 bits, by each request's row numbers `at` [B, rows]."""
    B, n = at.shape
    d = x.shape[2]
    return x[at].float().view(B, n, hkv, -1, d).permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, d)


def _packed(o, lse, at, inside, T, hq):
    """_grouped undone: [B, hkv, rows * group, d] to the packed rows [T, hq, d]."""
    B, n = at.shape
    hkv, d = o.shape[1], o.shape[3]
    o = o.view(B, hkv, n, -1, d).permute(0, 2, 1, 3, 4).reshape(B * n, hq, d)
    lse = lse.view(B, hkv, n, -1).permute(0, 2, 1, 3).reshape(B * n, hq)
    to = torch.where(inside, at, T).reshape(-1)
    out, out_lse = o.new_zeros(T + 1, hq, d), lse.new_zeros(T + 1, hq)
    return out.index_copy_(0, to, o)[:T], out_lse.index_copy_(0, to, lse)[:T]


def _paged(s):
    case = s["case"]
    q, hkv, ps = s["q"], case["hkv"], case["page"]
    T, hq, d = q.shape
    n, L = s["n_new"], s["longest"]
    cu, total = s["cu"].long(), s["seq_len"].long()
    start, new = cu[:-1], cu[1:] - cu[:-1]
    i, j = torch.arange(n, device=q.device), torch.arange(L, device=q.device)
    inside = i < new[:, None]
    at = (start[:, None] + i).clamp_max(T - 1)
    page = s["block_table"][:, j // ps].clamp_min(0).long()
    k, v = (s[c][page, j % ps].float().transpose(1, 2) for c in ("key_cache", "value_cache"))
    kept = j < total[:, None]
    v = torch.where(kept[:, None, :, None], v, 0)
    before = total - new
    if case["mask"] == "tree":
        node = j - before[:, None]
        bit = (s["anc_bits"][at][:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1
        sees = (node < 0)[:, None, :] | (bit == 1)
    elif case["mask"] == "causal":
        sees = j <= (before[:, None] + i)[:, :, None]
    else:
        sees = torch.ones(1, n, L, dtype=torch.bool, device=q.device)
    sees = (sees & kept[:, None, :]).repeat_interleave(hq // hkv, 1)[:, None]
    o, lse = _softmax_sum(_grouped(q, at, hkv), k, v, sees, d ** -0.5)
    o, lse = _packed(o, lse, at, inside, T, hq)
    return {"o": o.to(q.dtype), "lse": lse} if case["lse"] else {"o": o.to(q.dtype)}


def _prompt(s):
    case = s["case"]
    q, hkv, n = s["q"], case["hkv"], s["longest"]
    T, hq, d = q.shape
    cu = s["cu"].long()
    i = torch.arange(n, device=q.device)
    inside = i < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + i).clamp_max(T - 1)
    k, v = (s[c][at].float().transpose(1, 2) for c in ("k", "v"))
    sees = inside[:, None, :] & (i <= i[:, None] if case["causal"] else torch.ones(n, n, dtype=torch.bool,
                                                                                    device=q.device))
    sees = sees.repeat_interleave(hq // hkv, 1)[:, None]
    o, lse = _softmax_sum(_grouped(q, at, hkv), k, v, sees, d ** -0.5)
    o, lse = _packed(o, lse, at, inside, T, hq)
    return {"o": o.to(q.dtype), "lse": lse} if case["lse"] else {"o": o.to(q.dtype)}


# ---------------------------------------------------------------------------
# the floor and the 64-bit values
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "plan":
        B, ps = case["batch"], case["page"]
        prefix, new = _spread(B, case["pre_lo"], case["pre_hi"]), _spread(B, case["new_lo"], case["new_hi"])[::-1]
        rows = sum(new)
        # every touched page's id: the new rows' pages read or popped, the new ones also written
        read = sum(-(-(p + n) // ps) - p // ps for p, n in zip(prefix, new))
        fresh = sum(-(-(p + n) // ps) - -(-p // ps) for p, n in zip(prefix, new))
        return {"bytes": 4 * (6 * B + read + fresh) + rows * (16 + (4 if case["depth"] else 0)), "flops": 0}
    size = 2
    if case["op"] == "append":
        n = case["batch"] * (_PATH if case["path"] else case["rows"])
        moved = n * (9 / 16 if case["path"] else 1)  # half of a path's columns are empty on average
        return {"bytes": int(moved * 4 * case["hkv"] * case["d"] * size + n * (16 if case["path"] else 8)), "flops": 0}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "paged":
        B, ps = case["batch"], case["page"]
        prefix, new = _spread(B, case["pre_lo"], case["pre_hi"]), _spread(B, case["new_lo"], case["new_hi"])[::-1]
        keys, rows = sum(prefix) + sum(new), sum(new)
        pairs = sum(n * p + (n * (n + 1) // 2 if case["mask"] == "causal" else 4 * n if case["mask"] == "tree" else n * n)
                    for p, n in zip(prefix, new))
        tables = 4 * sum(-(-(p + n) // ps) for p, n in zip(prefix, new))
    else:
        sizes = _spread(case["batch"], case["lo"], case["hi"])
        keys = rows = sum(sizes)
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in sizes)
        tables = 0
    return {"bytes": 2 * keys * hkv * d * size + 2 * rows * hq * d * size + tables + (4 * rows * hq if case["lse"] else 0),
            "flops": 4 * pairs * hq * d}


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        out = {}
        slots = s["slots"].tolist()
        rows = s["rows"].tolist() if s["rows"] is not None else range(len(slots))
        pairs = _ints([(t, r) for t, r in zip(slots, rows) if r >= 0], torch.int64)
        for name, new in (("key_cache", "k"), ("value_cache", "v")):
            flat = s[name].double().reshape(-1, case["hkv"], case["d"])  # slot by slot
            flat[pairs[:, 0]] = s[new].double()[pairs[:, 1]]
            out[name] = flat.view(s[name].shape)
        return out
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q = s["q"].double()
    o, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    cu = s["cu"].tolist()
    for b in range(len(cu) - 1):
        r0, n = cu[b], cu[b + 1] - cu[b]
        if n == 0:
            continue
        if case["op"] == "paged":
            L, ps = int(s["seq_len"][b]), case["page"]
            pages = s["block_table"][b, :-(-L // ps)].long()
            k, v = (s[c][pages].flatten(0, 1)[:L].double() for c in ("key_cache", "value_cache"))
            sees = torch.ones(n, L, dtype=torch.bool, device=q.device)
            if case["mask"] == "causal":
                sees = sees.tril(L - n)
            elif case["mask"] == "tree":
                words = [w % (1 << 64) for w in s["anc_bits"][r0:r0 + n].tolist()]
                sees[:, L - n:] = _ints([[w >> c & 1 for c in range(n)] for w in words]).bool()
        else:
            k, v = s["k"][r0:r0 + n].double(), s["v"][r0:r0 + n].double()
            sees = torch.ones(n, n, dtype=torch.bool, device=q.device)
            sees = sees.tril() if case["causal"] else sees
        for h in range(hq):
            g = h * hkv // hq
            x = torch.where(sees, torch.mm(q[r0:r0 + n, h], k[:, g].t()) / math.sqrt(d), -math.inf)
            lse[r0:r0 + n, h] = torch.logsumexp(x, 1)
            o[r0:r0 + n, h] = torch.mm(torch.softmax(x, 1), v[:, g])
    return {"o": o, "lse": lse} if case["lse"] else {"o": o}
