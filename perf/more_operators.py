"""What a request of the hybrid model passes through around its tree steps, as measurable cases.

The tree kernels verify and commit drafts over a GDN state that is there.  A
case is one pass through an operator that brings it there or goes on from it:

conv     the causal convolution in front of a GDN layer, over whole packed
         prompts or one token a request, with the requests' windows kept
         (``ops.prompt_conv``)
prompt   the gated delta rule over whole packed prompts, from and into the
         requests' states (``ops.prompt_gdn``)
token    the same for one token a request (``ops.token_gdn``)
accept   which drafted tokens stand, by the target's probabilities and given
         random numbers, and the token behind them (``ops.tree_accept``)

``own`` false: the operators in elementary torch operations, in 32 bits,
rounded once at the end (``accept``: in 64, where a border decides).  ``own``
true: the package's kernels.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_D = 128     # both head dims of a GDN layer
_TAPS = 4    # of the convolution
_CHUNK = 64  # rows that the plain prompt form takes at once
_COLS = 16   # of an accepted path (-1 padded)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    layer = dict(hk=16, hv=32)  # a whole layer; 8192 channels of q, k and v
    return [
        # a full server without drafts: one token per request
        dict(name="conv_tokens", op="conv", batch=64, lo=1, hi=1, channels=8192, bias=False, resume="all"),
        # a packed batch of ordinary prompts, some of them going on from an earlier chunk
        dict(name="conv_packed", op="conv", batch=6, lo=257, hi=2999, channels=8192, bias=True, resume="some"),
        # a single request decoding
        dict(name="token_one", op="token", batch=1, **layer),
        # a full server decoding
        dict(name="token_full", op="token", batch=64, **layer),
        # a few short prompts: latency
        dict(name="prompt_short", op="prompt", batch=3, lo=1, hi=130, resume="none", **layer),
        # a packed batch of ordinary prompts
        dict(name="prompt_packed", op="prompt", batch=6, lo=257, hi=2999, resume="some", **layer),
        # one long prompt
        dict(name="prompt_long", op="prompt", batch=1, lo=8192, hi=8192, resume="none", **layer),
        # a rank's share of a layer (a quarter of the heads) over two long prompts, further chunks of longer ones
        dict(name="prompt_share", op="prompt", batch=2, lo=9001, hi=16384, resume="all", hk=4, hv=8),
        # a single request's draft tree, drawn from the drafter's probabilities
        dict(name="accept_one", op="accept", batch=1, lo=16, hi=16, vocab=131072, shape="tree", drawn=True),
        # the chains of a drafter without trees
        dict(name="accept_chains", op="accept", batch=64, lo=3, hi=9, vocab=131072, shape="chain", drawn=True),
        # trees of the drafter's likeliest tokens
        dict(name="accept_likeliest", op="accept", batch=64, lo=32, hi=32, vocab=131072, shape="tree", drawn=False),
        # ragged trees, drawn
        dict(name="accept_trees", op="accept", batch=48, lo=8, hi=40, vocab=100003, shape="tree", drawn=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("conv", "token", "prompt", "prompt", "accept", "accept"))
    hk = rng.choice((1, 2, 4, 8, 16))
    hv = hk * rng.choice((1, 2, 2, 4))
    resume = rng.choice(("all", "some", "none"))
    if op == "conv":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, 8192 // batch)
        return dict(op=op, batch=batch, lo=_log(rng, 1, hi), hi=hi, channels=(2 * hk + min(hv, 32)) * _D,
                    bias=rng.random() < 0.5, resume=resume)
    if op == "token":
        return dict(op=op, batch=_log(rng, 1, 64 * 32 // max(hv, 8)), hk=hk, hv=hv)
    if op == "prompt":
        batch = _log(rng, 1, 32)
        hi = _log(rng, 1, min(16384, 8192 * 32 // (batch * max(hv, 8))))
        return dict(op=op, batch=batch, lo=_log(rng, 1, hi), hi=hi, resume=resume, hk=hk, hv=hv)
    batch = _log(rng, 1, 64)
    hi = rng.randint(1, 64)
    vocab = min(_log(rng, 2, 131072), 64 * 32 * 131072 // (2 * batch * hi))
    return dict(op=op, batch=batch, lo=rng.randint(1, hi), hi=hi, vocab=vocab, shape=rng.choice(("chain", "tree", "tree")),
                drawn=rng.random() < 0.5)


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


def _resumes(batch, resume):
    """Which requests go on from their slot; None: all."""
    return None if resume == "all" else torch.tensor([resume == "some" and b % 2 == 1 for b in range(batch)], device="cuda")


def _parents(n, shape, rng):
    """A draft tree in topological order: depth first favoured, as a drafter's best-first growth gives."""
    return [-1] + [i - 1 if shape == "chain" else int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": case}

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "accept":
        return _prepare_accept(case, rng, gen, randn, s)
    B = case["batch"]
    s["slots"] = _ints(rng.permutation(B + 3)[:B].tolist())
    if case["op"] == "conv":
        sizes, C = _spread(B, case["lo"], case["hi"]), case["channels"]
        s |= {"x": randn(sum(sizes), C).bfloat16(), "conv_state": randn(B + 3, C, _TAPS - 1).bfloat16(),
              "weight": (randn(C, _TAPS) * 0.5).bfloat16(), "bias": randn(C).bfloat16() if case["bias"] else None,
              "cu": _ints(_starts(sizes)), "longest": max(sizes), "initial": _resumes(B, case["resume"])}
        return s
    hk, hv = case["hk"], case["hv"]
    sizes = [1] * B if case["op"] == "token" else _spread(B, case["lo"], case["hi"])
    T = sum(sizes)
    y = torch.nn.functional.silu(randn(T, (2 * hk + hv) * _D))  # what the convolution in front leaves
    # decay rates from 1 to 16 and steps from 0.001 to 0.1, as trained layers start from
    step = torch.exp(torch.rand(hv, generator=gen, device="cuda") * math.log(100) + math.log(1e-3))
    s |= {"y": y.bfloat16(), "a": randn(T, hv).bfloat16(), "b": randn(T, hv).bfloat16(),
          "A_log": torch.log(1 + 15 * torch.rand(hv, generator=gen, device="cuda")),
          "dt_bias": step + torch.log(-torch.expm1(-step)), "pool": randn(B + 3, hv, _D, _D) * 0.05}  # [slot, head, v, k]
    if case["op"] == "prompt":
        s |= {"cu": _ints(_starts(sizes)), "longest": max(sizes), "initial": _resumes(B, case["resume"])}
    return s


def _prepare_accept(case, rng, gen, randn, s):
    B, V = case["batch"], case["vocab"]
    sizes = _spread(B, case["lo"], case["hi"])
    T = sum(sizes)
    parents = [_parents(n, case["shape"], rng) for n in sizes]
    logits = randn(T, V) * 2.5
    s["probs"] = torch.softmax(logits, 1)
    # the drafter knows the target's distribution roughly
    logits += randn(T, V) * 0.7
    s["draft"] = torch.softmax(logits, 1) if case["drawn"] else None
    if case["drawn"]:  # children drawn one after the other without replacement: the largest of perturbed logits
        logits -= torch.log(-torch.log(torch.rand(T, V, generator=gen, device="cuda").clamp_(1e-20, 1 - 2.0 ** -24)))
    place = []  # which of its siblings a node is
    for p in parents:
        place += [0] + [p[1:i].count(p[i]) for i in range(1, len(p))]
    top = torch.topk(logits, min(V, max(place) + 1), dim=1)[1]
    cu = _starts(sizes)
    above = _ints([c + max(p, 0) for c, ps in zip(cu, parents) for p in ps], torch.int64)
    s["tokens"] = top[above, _ints(place, torch.int64) % top.shape[1]].contiguous()
    s |= {"parent": _ints(sum(parents, [])), "cu": _ints(cu), "longest": max(sizes),
          "u": torch.rand(T, generator=gen, device="cuda"), "last": torch.rand(B, generator=gen, device="cuda")}
    return s


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    return {"conv": _conv, "prompt": _prompt, "token": _token, "accept": _accept}[state["case"]["op"]](state)


def _own(s):
    from dforktree_amd import ops
    case = s["case"]
    if case["op"] == "conv":
        y = ops.prompt_conv(s["x"], s["conv_state"], s["weight"], s["bias"], s["cu"], max_len=s["longest"],
                            cs_indices=s["slots"], initial=s["initial"])
        return {"y": y, "conv_state": s["conv_state"]}
    if case["op"] == "accept":
        return ops.tree_accept(s["tokens"], s["parent"], s["probs"], s["u"], s["last"], draft_probs=s["draft"],
                               cu_seqlens=s["cu"], n_nodes=s["longest"], path_cols=_COLS)
    state = s["pool"].transpose(-1, -2)
    if case["op"] == "token":
        o = ops.token_gdn(s["y"], s["a"], s["b"], s["A_log"], s["dt_bias"], state, hk=case["hk"], hv=case["hv"],
                          state_indices=s["slots"])
    else:
        o = ops.prompt_gdn(s["y"], s["a"], s["b"], s["A_log"], s["dt_bias"], state, s["cu"], hk=case["hk"], hv=case["hv"],
                           max_len=s["longest"], state_indices=s["slots"], initial=s["initial"])
    return {"o": o, "state": s["pool"]}


def _start(s, x):
    """The requests' slots of x [slots, ...] in 32 bits, zero for those that start anew."""
    x = x[s["slots"].long()].float()
    return x if s.get("initial") is None else x * s["initial"].view(-1, *[1] * (x.dim() - 1))


def _conv(s):
    """Every row with the rows before it, or the columns of its request's window."""
    x, W = s["x"].float(), s["weight"].float()
    T = x.shape[0]
    cu = s["cu"].long()
    window = _start(s, s["conv_state"]).transpose(1, 2)  # [batch, taps - 1, channels]
    row = torch.arange(T, device=x.device)
    of = torch.searchsorted(cu[1:], row, right=True)

    def back(row, of, r):
        """The input r places in front of a row."""
        place = row - r - cu[of]
        return torch.where((place >= 0)[:, None], x[(row - r).clamp(0, T - 1)], window[of, (place + _TAPS - 1).clamp(0, _TAPS - 2)])

    y = sum(back(row, of, r) * W[:, _TAPS - 1 - r] for r in range(_TAPS))
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = y / (1 + torch.exp(-y))
    every = torch.arange(cu.numel() - 1, device=x.device)
    left = torch.stack([back(cu[1:], every, r) for r in range(_TAPS - 1, 0, -1)], 2)
    s["conv_state"][s["slots"].long()] = left.to(s["conv_state"].dtype)
    return {"y": y.to(s["x"].dtype), "conv_state": s["conv_state"]}


def _gates(s):
    """Log decays and write strengths [rows, hv]."""
    g = -torch.exp(s["A_log"].float()) * torch.nn.functional.softplus(s["a"].float() + s["dt_bias"].float())
    return g, torch.sigmoid(s["b"].float())


def _heads(s, dtype=torch.float32):
    """q, k (normalised, q scaled, repeated for their value heads) and v, [rows, hv, 128]."""
    hk, hv = s["case"]["hk"], s["case"]["hv"]
    y = s["y"].to(dtype)
    q, k, v = (t.unflatten(1, (-1, _D)) for t in y.split([hk * _D, hk * _D, hv * _D], 1))
    q, k = (t * torch.rsqrt((t * t).sum(2, keepdim=True) + 1e-6) for t in (q, k))
    return (q * _D ** -0.5).repeat_interleave(hv // hk, 1), k.repeat_interleave(hv // hk, 1), v


def _token(s):
    q, k, v = _heads(s)
    g, beta = _gates(s)
    slots = s["slots"].long()
    S = _start(s, s["pool"]) * torch.exp(g)[:, :, None, None]  # [batch, head, v, k]
    u = beta[:, :, None] * (v - (S * k[:, :, None]).sum(3))
    S = S + u[:, :, :, None] * k[:, :, None]
    o = (S * q[:, :, None]).sum(3)
    s["pool"][slots] = S
    return {"o": o.to(s["y"].dtype), "state": s["pool"]}


def _inverse(A):
    """(I + A)^-1 of the strictly lower parts, from 1 x 1 diagonal blocks to ones of twice the size: the block below
    two inverted ones X and Y is -Y A X."""
    n = A.shape[-1]
    inv = torch.eye(n, device=A.device).expand(A.shape).contiguous()
    size = 1
    while size < n:
        block = torch.arange(0, n, 2 * size, device=A.device)[:, None]
        one = block + torch.arange(size, device=A.device)
        two = one + size
        x, y, a = (m[..., r[:, :, None], c[:, None, :]] for m, r, c in ((inv, one, one), (inv, two, two), (A, two, one)))
        inv[..., two[:, :, None], one[:, None, :]] = -torch.matmul(torch.matmul(y, a), x)
        size *= 2
    return inv


def _prompt(s):
    """Chunks of 64 rows: what needs no state for all chunks at once, the states chunk after chunk."""
    case = s["case"]
    hv, T = case["hv"], s["y"].shape[0]
    cu = s["cu"].long()
    B = cu.numel() - 1
    chunks = -(-s["longest"] // _CHUNK)
    i = torch.arange(chunks * _CHUNK, device=cu.device)
    at = (cu[:-1, None] + i).clamp_max(T - 1)
    inside = i < (cu[1:] - cu[:-1])[:, None]

    def chunked(x):
        """Packed rows [T, hv, ...] as [batch, chunk, hv, 64, ...], zero past a request's last."""
        x = torch.where(inside.view(B, -1, *[1] * (x.dim() - 1)), x[at], 0)
        return x.unflatten(1, (chunks, _CHUNK)).transpose(2, 3).contiguous()

    q, k, v = (chunked(t) for t in _heads(s))
    g, beta = (chunked(t) for t in _gates(s))
    G = g.cumsum(3)
    lower = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=cu.device).tril()
    decay = torch.where(lower, torch.exp(torch.where(lower, G[..., :, None] - G[..., None, :], 0)), 0)
    kt = k.transpose(-1, -2).contiguous()
    X = _inverse(torch.matmul(k * beta[..., None], kt) * decay)
    U = torch.matmul(X, v * beta[..., None])
    W = torch.matmul(X, k * (beta * torch.exp(G))[..., None])
    P = torch.matmul(q, kt) * decay
    q = q * torch.exp(G)[..., None]
    out = kt * torch.exp(G[..., -1:] - G)[..., None, :]
    S = _start(s, s["pool"]).transpose(-1, -2).contiguous()  # [batch, head, k, v]
    o = torch.empty_like(v)
    for c in range(chunks):
        u = U[:, c] - torch.matmul(W[:, c], S)
        o[:, c] = torch.matmul(q[:, c], S) + torch.matmul(P[:, c], u)
        S = S * torch.exp(G[:, c, :, -1])[..., None, None] + torch.matmul(out[:, c], u)
    s["pool"][s["slots"].long()] = S.transpose(-1, -2)
    o = o.transpose(2, 3).reshape(-1, hv, _D)
    to = torch.where(inside, at, T).reshape(-1)
    return {"o": o.new_zeros(T + 1, hv, _D).index_copy_(0, to, o)[:T].to(s["y"].dtype), "state": s["pool"]}


def _accept(s):
    """Node after node of all trees at once: each is examined where its parent is the last node that stands."""
    probs, draft, tokens = s["probs"], s["draft"], s["tokens"].long()
    V = probs.shape[1]
    cu = s["cu"].long()
    start, n = cu[:-1], cu[1:] - cu[:-1]
    B = n.numel()
    each = torch.arange(B, device=cu.device)

    def row(p, at):
        p = p[at].double()
        return torch.where(p > 0, p, 0)

    node = torch.zeros_like(n)
    r = row(probs, start)  # the distribution to draw from at `node`, given what was refused there
    q0 = row(draft, start) if draft is not None else None  # what its children were drawn from
    gone = torch.zeros_like(r, dtype=torch.bool)  # tokens refused at `node`
    off = torch.zeros(B, dtype=torch.float64, device=cu.device)  # their mass: of q0, without a drafter's probabilities of r
    path = torch.full((B, _COLS), -1, dtype=torch.int32, device=cu.device)
    path[:, 0] = torch.where(n > 0, 0, -1)
    length = torch.where(n > 0, 1, 0)
    for i in range(1, s["longest"]):
        at = (start + i).clamp_max(tokens.numel() - 1)
        here = (i < n) & (s["parent"][at].clamp_min(0) == node) & (length < _COLS)
        t = tokens[at]
        u = s["u"][at].double()
        if draft is None:
            weight = torch.where(gone[each, t], 0, r[each, t])
            stands = here & (u * (1 - off) < weight)
        else:
            q = torch.where(gone | (off >= 1)[:, None], 0, q0) / (1 - off)[:, None].clamp_min(1e-300)
            stands = here & (u * q[each, t] < r[each, t])
        falls = here & ~stands
        if draft is not None:
            rest = (r - q).clamp_min(0)
            mass = rest.sum(1, keepdim=True)
            r = torch.where(falls[:, None] & (mass > 0), rest / mass, r)
        off = off + torch.where(falls & ~gone[each, t], (r if draft is None else q0)[each, t], 0)
        gone[each, t] |= falls
        node = torch.where(stands, i, node)
        path[each, length.clamp_max(_COLS - 1)] = torch.where(stands, i, path[each, length.clamp_max(_COLS - 1)])
        length = length + stands
        move = stands[:, None]
        r = torch.where(move, row(probs, at), r)
        if draft is not None:
            q0 = torch.where(move, row(draft, at), q0)
        gone &= ~move
        off = torch.where(stands, 0, off)
    if draft is None:
        rest = torch.where(gone, 0, r)
        r = torch.where(rest.sum(1, keepdim=True) > 0, rest, r)
    cum = r.cumsum(1)
    total = cum[:, -1:]
    some = torch.where(r > 0, torch.arange(V, device=cu.device), -1).amax(1)  # the last token of any weight
    token = torch.minimum((cum <= s["last"].double()[:, None] * total).sum(1), some)
    rows = torch.where(path >= 0, start[:, None] + path, -1)
    return {"path": path, "path_len": length.int(), "rows": rows, "token": token}


# ---------------------------------------------------------------------------
# the floor and the 64-bit values
# ---------------------------------------------------------------------------
def work(case):
    B = case["batch"]
    if case["op"] == "conv":
        T, C = sum(_spread(B, case["lo"], case["hi"])), case["channels"]
        kept = {"all": B, "some": B // 2, "none": 0}[case["resume"]]
        return {"bytes": 2 * C * (2 * T + (kept + B) * (_TAPS - 1) + _TAPS + case["bias"]), "flops": 2 * _TAPS * T * C}
    if case["op"] == "accept":
        # one row of the target's probabilities a request, one of the drafter's where its last node was drawn
        return {"bytes": B * case["vocab"] * 4 * (2 if case["drawn"] else 1) + B * case["hi"] * 24, "flops": 0}
    hk, hv = case["hk"], case["hv"]
    T = B if case["op"] == "token" else sum(_spread(B, case["lo"], case["hi"]))
    kept = B if case["op"] == "token" else {"all": B, "some": B // 2, "none": 0}[case["resume"]]
    rows = T * (2 * (2 * hk + 2 * hv) * _D + 4 * hv)
    # a row and head: the state times k and q, and the product of k and u onto it
    return {"bytes": rows + (kept + B) * hv * _D * _D * 4, "flops": T * hv * 6 * _D * _D}


def exact(case, seed):
    if case["op"] == "accept":
        return None  # whole numbers
    s = prepare(case, seed)
    slots = s["slots"].tolist()
    cu = s["cu"].tolist() if "cu" in s else list(range(case["batch"] + 1))
    fresh = [False] * case["batch"] if s.get("initial") is None else (~s["initial"]).tolist()
    if case["op"] == "conv":
        y, left = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda"), s["conv_state"].double()
        for b, slot in enumerate(slots):
            x = s["x"][cu[b]:cu[b + 1]].double().t()  # [channels, rows]
            x = torch.cat([left[slot] * (not fresh[b]), x], 1)
            z = torch.stack([x[:, j:x.shape[1] - _TAPS + 1 + j] for j in range(_TAPS)], 2)
            z = (z * s["weight"].double()[:, None]).sum(2).t()
            z = z if s["bias"] is None else z + s["bias"].double()
            y[cu[b]:cu[b + 1]] = z * torch.sigmoid(z)
            left[slot] = x[:, x.shape[1] - _TAPS + 1:]
        return {"y": y, "conv_state": left}
    # the recurrence token by token, all requests side by side
    q, k, v = _heads(s, torch.float64)
    x = s["a"].double() + s["dt_bias"].double()
    decay = torch.exp(-torch.exp(s["A_log"].double()) * torch.log1p(torch.exp(x)))
    beta = 1 / (1 + torch.exp(-s["b"].double()))
    pool, o = s["pool"].double(), torch.empty(v.shape, dtype=torch.float64, device="cuda")
    S = pool[s["slots"].long()] * (1 - torch.tensor(fresh, dtype=torch.float64, device="cuda")).view(-1, 1, 1, 1)
    first = torch.tensor(cu[:-1], device="cuda")
    order = sorted(range(len(slots)), key=lambda b: cu[b] - cu[b + 1])  # the longest first: those that go on are a prefix
    S, first = S[order], first[order]
    sizes = [cu[b + 1] - cu[b] for b in order]
    for t in range(sizes[0]):
        m = sum(n > t for n in sizes)
        r = first[:m] + t
        kt = k[r]
        Sm = S[:m]
        Sm *= decay[r][:, :, None, None]
        u = beta[r][:, :, None] * (v[r] - (Sm @ kt[..., None])[..., 0])
        Sm += u[..., None] * kt[:, :, None]
        o[r] = (Sm @ q[r][..., None])[..., 0]
    pool[s["slots"].long()[order]] = S
    return {"o": o, "state": pool}
