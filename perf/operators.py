"""Measured operators of tree drafting over a KV cache and of the training that goes with it.

A decoding program drafts a tree of tokens from the top logits of its draft rows, verifies the tree in one forward
over its caches, keeps the accepted path, and copies prompts and sequences between cache slots. A training program
distils the drafter from the top logits of a teacher. The kinds below are those operators:

* ``tree``     attention of a tree of drafted tokens: node t sees the committed cache rows, its ancestors and itself;
* ``keep``     the accepted path of a tree kept in the caches of all layers: rows ``length + node`` move to ``length + i``;
* ``copy``     sequences copied between cache slots of all layers (a prompt forked to several slots);
* ``topk``     the k largest logits of each row, ties to the lowest index, with the row's log-sum-exp;
* ``distill``  the distillation loss from a teacher's top logits and its gradient.

Head layouts are those of the framework's own configurations (``HEADS``); vocabularies 151936, 32000 and 4096.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# (q heads, K/V heads, head dim)
HEADS = {"8b": (32, 8, 128), "1b": (16, 8, 128), "mha7b": (32, 32, 128), "tiny": (4, 2, 64)}
VOCABS = (151936, 32000, 4096)


def listed():
    return [
        # One token over a short cache: plain decoding, where only latency counts.
        dict(name="tree 1b 1x1 ctx130", kind="tree", heads="1b", dtype="bf16", batch=1, nodes=1, ctx=130, room=60, pad=0),
        # Verification of a 16-node tree per sequence, eight sequences: the ordinary serving step.
        dict(name="tree 8b 8x16 ctx4096", kind="tree", heads="8b", dtype="bf16", batch=8, nodes=16, ctx=4096, room=64,
             pad=3),
        # The fp32 parity configuration with odd sizes and padded trees.
        dict(name="tree tiny fp32 3x37 ctx901", kind="tree", heads="tiny", dtype="fp32", batch=3, nodes=37, ctx=901,
             room=41, pad=9),
        # Wide trees over long caches.
        dict(name="tree 8b 16x64 ctx16384", kind="tree", heads="8b", dtype="bf16", batch=16, nodes=64, ctx=16384, room=64,
             pad=5),
        # Three accepted tokens of one sequence, 24 layers.
        dict(name="keep 1b 1x3 of 8", kind="keep", heads="1b", dtype="bf16", layers=24, batch=1, nodes=8, path=3, ctx=200,
             max_len=256),
        # The accepted paths of eight 16-node trees, 36 layers.
        dict(name="keep 8b 8x6 of 16", kind="keep", heads="8b", dtype="bf16", layers=36, batch=8, nodes=16, path=6, ctx=480,
             max_len=512),
        # A sequence of the fp32 configuration into another cache.
        dict(name="copy tiny fp32 2 of 2 ctx77", kind="copy", heads="tiny", dtype="fp32", layers=2, src_batch=3, batch=5,
             copies=2, fan=1, ctx=77, max_len=128),
        # A 2048-token prompt prefilled once and forked to eight slots, 36 layers.
        dict(name="copy 8b 1 to 8 ctx2048", kind="copy", heads="8b", dtype="bf16", layers=36, src_batch=1, batch=8, copies=1,
             fan=8, ctx=2048, max_len=2304),
        # Candidates of a draft tree: the top logits of one 16-row draft block.
        dict(name="topk 16x151936 k10", kind="topk", dtype="bf16", rows=16, vocab=151936, k=10, extra=0),
        # A teacher's top logits for one micro-batch row of training.
        dict(name="topk 4096x151936 k64", kind="topk", dtype="bf16", rows=4096, vocab=151936, k=64, extra=0),
        # The fp32 parity configuration: few rows, a small vocabulary, rows with a stride of their own.
        dict(name="distill fp32 511x4096 k17", kind="distill", dtype="fp32", rows=511, vocab=4096, k=17, extra=5,
             temperature=1.0),
        # Distillation of one 4096-token row at the large vocabulary.
        dict(name="distill 4096x151936 k64", kind="distill", dtype="bf16", rows=4096, vocab=151936, k=64, extra=0,
             temperature=2.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "keep", "copy", "topk", "distill"])
    heads = rng.choice(list(HEADS))
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "tree":
        while True:
            c = dict(kind=kind, heads=heads, dtype=dtype, batch=_log_int(rng, 1, 16), nodes=_log_int(rng, 1, 64),
                     ctx=_log_int(rng, 1, 16384), room=rng.randint(0, 70))
            c["pad"] = rng.randint(0, c["nodes"] // 2)
            w = work(c)
            if w["bytes"] <= 1.1e9 and w["flops"] <= 2.8e11:
                return c
    if kind in ("keep", "copy"):
        while True:
            c = dict(kind=kind, heads=heads, dtype=dtype, layers=rng.randint(1, 36), batch=_log_int(rng, 1, 16),
                     ctx=_log_int(rng, 1, 2048))
            if kind == "keep":
                c["nodes"] = _log_int(rng, 1, 64)
                c["path"] = rng.randint(1, min(c["nodes"], 24))
                c["max_len"] = c["ctx"] + c["nodes"] + rng.randint(0, 33)
                total = c["batch"]
            else:
                c["src_batch"] = rng.randint(1, 4)
                c["copies"] = rng.randint(1, min(c["src_batch"], c["batch"]))
                c["fan"] = rng.randint(1, c["batch"] // c["copies"])
                c["max_len"] = c["ctx"] + rng.randint(0, 150)
                total = c["src_batch"] + c["batch"]
            nq, nk, d = HEADS[heads]
            if total * c["layers"] * 2 * nk * c["max_len"] * d * DTYPES[dtype].itemsize <= 2.6e9:
                return c
    while True:
        vocab = rng.choice([*VOCABS, _log_int(rng, 40, 152000)])
        c = dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, 4096), vocab=vocab, k=_log_int(rng, 1, min(128, vocab)),
                 extra=rng.choice([0, 0, 1, 8, 13]))
        if kind == "distill":
            c["temperature"] = rng.choice([1.0, 1.0, 2.0, 0.7])
        if c["rows"] * vocab * DTYPES[dtype].itemsize <= 1.25e9:
            return c


def _lengths(case):
    """Committed rows per sequence: the first holds ``ctx``, the others fewer, down to about half."""
    ctx, B = case["ctx"], case.get("src_batch", case["batch"])
    return [ctx - (b * ctx) // (2 * B) for b in range(B)]


def _counts(case):
    """Accepted nodes per sequence: the first keeps ``path``, the others fewer."""
    return [case["path"] - b % max(1, (case["path"] + 1) // 2) for b in range(case["batch"])]


def _pairs(case):
    """(source, destination) slots: source i goes to ``fan`` slots, from the last slot down."""
    return [(i, case["batch"] - 1 - (i * case["fan"] + j)) for i in range(case["copies"]) for j in range(case["fan"])]


def work(case):
    es = DTYPES[case["dtype"]].itemsize
    if case["kind"] in ("topk", "distill"):
        R, V, k = case["rows"], case["vocab"], case["k"]
        if case["kind"] == "topk":
            return dict(bytes=R * V * es + R * (k * 12 + 4), flops=4 * R * V)
        # forward: logits read; backward: logits read, gradient written
        return dict(bytes=3 * R * V * es + 2 * R * k * 12 + 4, flops=10 * R * V)
    nq, nk, d = HEADS[case["heads"]]
    n = _lengths(case)
    if case["kind"] == "tree":
        B, T = case["batch"], case["nodes"]
        keys = sum(n) + B * T
        return dict(bytes=keys * nk * d * 2 * es + 2 * B * T * nq * d * es + B * T * 4, flops=4 * d * nq * T * keys)
    row = nk * d * es * 2 * case["layers"]
    if case["kind"] == "keep":
        return dict(bytes=2 * sum(_counts(case)) * row, flops=0)
    pairs = _pairs(case)
    return dict(bytes=(sum(n[s] for s in {s for s, _ in pairs}) + sum(n[s] for s, _ in pairs)) * row, flops=0)


# ---- inputs ------------------------------------------------------------------------------------
def _tree(B, T, pad, g):
    """Parents of B trees of T nodes: node 0 is a root, a later node hangs on an earlier one (a few more roots among
    them); the last ``pad`` nodes of every second tree are padding (-2)."""
    t = torch.arange(T, device=DEV)
    p = (torch.rand((B, T), device=DEV, generator=g) * (t + 0.2)).floor().long() - (t == 0).long()
    p = torch.where(torch.rand((B, T), device=DEV, generator=g) < 0.05, -1, torch.minimum(p, t - 1))
    if pad:
        p[::2, T - pad:] = -2
    return p.int().contiguous()


def _logits(rows, vocab, extra, dtype, g):
    """Logits as an LM head gives them: most within a few units of zero, a handful per row well above; rows with
    ``extra`` elements between them."""
    z = torch.empty((rows, vocab + extra), device=DEV, dtype=dtype)
    for r in range(0, rows, 512):
        part = torch.randn((min(512, rows - r), vocab + extra), device=DEV, generator=g)
        peak = torch.rand(part.shape, device=DEV, generator=g) < 8.0 / vocab
        z[r:r + 512] = torch.where(peak, part.abs() * 4 + 6, part * 2).to(dtype)
    return z[:, :vocab]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    kind = case["kind"]
    s = dict(kind=kind)
    if kind in ("topk", "distill"):
        s["z"], s["k"] = _logits(case["rows"], case["vocab"], case["extra"], dt, g), case["k"]
        if kind == "distill":
            # the teacher agrees with the student on most of its top: its logits are the student's with noise
            R, k = case["rows"], case["k"]
            values, indices = [], []
            for r in range(0, R, 512):
                t = s["z"][r:r + 512].float()
                t = t + torch.randn(t.shape, device=DEV, generator=g)
                v, i = torch.topk(t, k, dim=1)
                values.append(v)
                indices.append(i)
            s["values"], s["indices"] = torch.cat(values), torch.cat(indices)
            if R > 2:                                   # a ragged row and a row without a teacher
                s["values"][1, k // 2 + 1:] = -math.inf
                s["values"][2] = -math.inf
            s["tokens"], s["temperature"] = R + 7, case["temperature"]
        return s
    nq, nk, d = HEADS[case["heads"]]
    n = _lengths(case)
    s["lengths"] = torch.tensor(n, device=DEV)

    def cache(batch, max_len, tensors=1):
        """``tensors`` caches of ``batch`` slots, one behind the other in memory."""
        c = torch.empty((tensors, batch, nk, max_len, d), device=DEV, dtype=dt)
        for t in c:
            t.copy_(torch.randn(t.shape, device=DEV, generator=g))
        return c

    if kind == "tree":
        B, T = case["batch"], case["nodes"]
        s["parents"] = _tree(B, T, case["pad"], g)
        s["q"] = torch.randn((B * T, nq * d), device=DEV, generator=g).to(dt)
        s["k"], s["v"] = (cache(B, case["ctx"] + T + case["room"])[0] for _ in "kv")
    elif kind == "keep":
        counts = _counts(case)
        s["counts"] = torch.tensor(counts, device=DEV)
        order = torch.rand((case["batch"], case["nodes"]), device=DEV, generator=g).argsort(1)[:, :case["path"]]
        s["nodes"] = order.sort(1).values.contiguous()
        s["caches"] = cache(case["batch"], case["max_len"], 2 * case["layers"])
    else:
        s["pairs"] = _pairs(case)
        s["src"] = cache(case["src_batch"], case["ctx"], 2 * case["layers"])
        s["dst"] = cache(case["batch"], case["max_len"], 2 * case["layers"])
        s["dst_lengths"] = torch.zeros(case["batch"], device=DEV, dtype=torch.int64)
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)[state["kind"]](state)


def _own_tree(s):
    from uno_amd import kernels as K

    return K.tree_attn(s["q"], s["k"], s["v"], s["lengths"], s["parents"])


def _own_keep(s):
    from uno_amd import kernels as K

    K.cache_keep(s["caches"].unbind(), s["lengths"], s["nodes"], s["counts"])
    return s["caches"]


def _own_copy(s):
    from uno_amd import kernels as K

    K.cache_copy(s["src"].unbind(), s["dst"].unbind(), s["lengths"], s["dst_lengths"], s["pairs"])
    return s["dst"], s["dst_lengths"]


def _own_topk(s):
    from uno_amd import kernels as K

    return K.row_top_k(s["z"], s["k"])


def _own_distill(s):
    from uno_amd.training.losses import token_normalized_top_k_distillation

    z = s["z"].detach().requires_grad_(True)
    loss = token_normalized_top_k_distillation(z, s["values"], s["indices"], s["tokens"], temperature=s["temperature"])
    (grad,) = torch.autograd.grad(loss, z)
    return loss.detach(), grad


def _plain_tree(s):
    q, k, v, n, parents = s["q"], s["k"], s["v"], s["lengths"], s["parents"]
    B, nk, max_len, d = k.shape
    T = parents.shape[1]
    rep = q.shape[1] // (nk * d)
    # ancestors by repeated squaring of "is me or my parent"
    t = torch.arange(T, device=q.device)
    real = parents >= -1
    step = ((parents[:, :, None] == t) & (t < t[:, None]) & real[:, None, :]).float()
    anc = step + torch.eye(T, device=q.device)
    for _ in range((T - 1).bit_length()):
        anc = ((anc @ anc) > 0).float()
    anc = (anc > 0) & real[:, :, None]
    j = torch.arange(max_len, device=q.device)
    node = (j - n[:, None]).clamp(0, T - 1)                                    # [B, max_len]
    in_tree = (j >= n[:, None]) & (j < n[:, None] + T)
    seen = anc.gather(2, node[:, None, :].expand(B, T, max_len)) & in_tree[:, None, :]
    seen |= (j < n[:, None])[:, None, :] & real[:, :, None]
    qs = q.view(B, T, nk, rep, d).permute(0, 2, 3, 1, 4).reshape(B, nk, rep * T, d).float()
    z = (qs @ k.float().transpose(2, 3)).view(B, nk, rep, T, max_len) * d ** -0.5
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p.view(B, nk, rep * T, max_len) @ v.float()
    return o.view(B, nk, rep, T, d).permute(0, 3, 1, 2, 4).reshape(B * T, nk * rep * d).to(q.dtype)


def _plain_keep(s):
    nodes, counts, n = s["nodes"], s["counts"], s["lengths"]
    B, P = nodes.shape
    i = torch.arange(P, device=nodes.device)
    # entries past the count move their own destination row onto itself
    src = n[:, None] + torch.where(i < counts[:, None], nodes, i)
    dst = (n[:, None] + i)[:, None, :, None]
    for c in s["caches"]:
        shape = (B, c.shape[1], P, c.shape[3])
        c.scatter_(2, dst.expand(shape), c.gather(2, src[:, None, :, None].expand(shape)))
    return s["caches"]


def _plain_copy(s):
    src = torch.tensor([a for a, _ in s["pairs"]], device=DEV)
    dst = torch.tensor([b for _, b in s["pairs"]], device=DEV)
    rows = s["src"].shape[3]
    n = s["lengths"][src]
    live = (torch.arange(rows, device=DEV) < n[:, None])[:, None, :, None]
    for a, b in zip(s["src"], s["dst"]):
        b[dst, :, :rows] = torch.where(live, a[src], b[dst, :, :rows])
    s["dst_lengths"][dst] = n
    return s["dst"], s["dst_lengths"]


def _plain_topk(s):
    z, k = s["z"].float() + 0.0, s["k"]                  # + 0.0: -0 and 0 are the same value
    V = z.shape[1]
    top = z.amax(1)
    lse = top + torch.exp(z - top[:, None]).sum(1).log()
    # larger value first, then lower index: one 64-bit key per entry
    bits = z.view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    key = (order << 32) | (V - 1 - torch.arange(V, device=z.device))
    picked = torch.topk(key, k, dim=1).values
    indices = V - 1 - (picked & 0xFFFFFFFF)
    return z.gather(1, indices), indices, lse


def _plain_distill(s):
    z, tau = s["z"].float() / s["temperature"], s["temperature"]
    t, idx = s["values"].float() / tau, s["indices"]
    inv_n = 1.0 / s["tokens"]
    t_top = t.amax(1, keepdim=True)
    live = t_top > -math.inf
    e = torch.exp(t - torch.where(live, t_top, 0.0))
    total = e.sum(1, keepdim=True)
    p = e / torch.where(live, total, 1.0)
    log_p = t - torch.where(live, t_top + total.log(), 0.0)
    top = z.amax(1, keepdim=True)
    ez = torch.exp(z - top)
    zsum = ez.sum(1, keepdim=True)
    log_q = z.gather(1, idx) - (top + zsum.log())
    loss = torch.where(p > 0, p * (log_p - log_q), 0.0).sum() * (tau * tau * inv_n)
    grad = ez / zsum * live
    grad.scatter_add_(1, idx, -p)
    return loss, (grad * (tau * inv_n)).to(s["z"].dtype)


_own = dict(tree=_own_tree, keep=_own_keep, copy=_own_copy, topk=_own_topk, distill=_own_distill)
_plain = dict(tree=_plain_tree, keep=_plain_keep, copy=_plain_copy, topk=_plain_topk, distill=_plain_distill)


# ---- the definitions in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    if case["kind"] in ("keep", "copy"):
        return None                                       # moved rows, not computed ones
    s = prepare(case, seed)
    if case["kind"] == "tree":
        return _exact_tree(s)
    z = s["z"]
    R, V = z.shape
    if case["kind"] == "topk":
        values, indices, lse = [], [], []
        for r in range(0, R, 256):
            zr = z[r:r + 256].double() + 0.0
            v, i = torch.sort(zr, dim=1, descending=True, stable=True)
            values.append(v[:, :s["k"]].clone())
            indices.append(i[:, :s["k"]].clone())
            lse.append(torch.logsumexp(zr, 1))
        return torch.cat(values), torch.cat(indices), torch.cat(lse)
    tau = s["temperature"]
    loss = torch.zeros((), device=DEV, dtype=torch.float64)
    grad = torch.zeros((R, V), device=DEV, dtype=torch.float64)
    t, idx = s["values"].double(), s["indices"]
    for r in range(0, R, 512):
        rows = slice(r, r + 512)
        has = (t[rows] > -math.inf).any(1)
        p = torch.softmax(t[rows][has] / tau, 1)
        logq = torch.log_softmax(z[rows][has].double() / tau, 1)
        part = p * (p.log() - logq.gather(1, idx[rows][has]))
        loss += torch.where(p > 0, part, torch.zeros_like(part)).sum()
        gr = logq.exp()
        gr.scatter_add_(1, idx[rows][has], -p)
        grad[rows][has] = gr
    return loss * tau * tau / s["tokens"], grad * (tau / s["tokens"])


def _exact_tree(s):
    q, k, v, n, parents = s["q"], s["k"], s["v"], s["lengths"].tolist(), s["parents"].tolist()
    B, nk, _, d = k.shape
    T = len(parents[0])
    rep = q.shape[1] // (nk * d)
    out = torch.zeros((B, T, nk, rep, d), device=DEV, dtype=torch.float64)
    for b in range(B):
        keep = torch.zeros((T, n[b] + T), dtype=torch.bool)
        for t in range(T):
            if parents[b][t] < -1:
                continue
            keep[t, :n[b]] = True
            a = t
            while a >= 0:
                keep[t, n[b] + a] = True
                p = parents[b][a]
                a = p if p < a and (p < 0 or parents[b][p] >= -1) else -1
        bias = torch.zeros(keep.shape, dtype=torch.float64).masked_fill(~keep, -math.inf).to(DEV)
        some = keep.any(1).to(DEV)
        for h in range(nk):
            kd, vd = k[b, h, :n[b] + T].double(), v[b, h, :n[b] + T].double()
            for r in range(rep):
                qd = q.view(B, T, nk, rep, d)[b, :, h, r].double()
                a = torch.softmax(qd @ kd.T * d ** -0.5 + bias, 1)
                out[b, some, h, r] = (a @ vd)[some]
    return out.view(B * T, nk * rep * d)
