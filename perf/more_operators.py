"""Measured operators of decoding with a KV cache held in 4 bits, and of the verification of what was drafted.

A decoding program that is bound by its caches' size keeps them in 4 bits: it stores the rows of a prompt or of a drafted block
there, attends over them, and samples what is accepted from the target's logits and given random numbers. The kinds below are
those operators:

* ``store``  K and V rows of all sequences put into 4-bit caches, and read back as the numbers that they then are;
* ``attn``   attention of a tree of drafted tokens over 4-bit caches: node t sees the committed rows, its ancestors and itself;
* ``draft``  a drafted block verified against the target's logits: tokens accepted with probability min(1, p / q), the next one
             drawn from the rest of p, or from p itself behind the last;
* ``walk``   a drafted tree verified: from node 0 on, the token drawn at a node leads to the child that holds it.

The 4-bit format: 32 consecutive elements share a scale 2^(byte - 127), the least for which the largest magnitude is below 7
scales; an element is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 scales (ties to the even code 0 .. 7, bit 3 the sign); the
element of an even index is a byte's low half. Byte 2 is the least scale, 252 the largest.

Sampling is by the inverse distribution function: the lowest index at which the running sum of the weights exp((z - max z) / T)
exceeds u times their sum (weights below e^-700 are 0). Temperature 0 takes the largest logit, the lowest index of equal ones.
The next token behind a refused draft has the weights max(p - q, 0), or p's where these sum to less than 2^-40.

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
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LEAST = 2.0 ** -40                      # of the probability left to a refused token's place


def listed():
    return [
        # One decoded token of one sequence: only latency counts.
        dict(name="store 1b 1x1", kind="store", heads="1b", dtype="bf16", batch=1, rows=1, ctx=130, room=60),
        # The prompts of four sequences, one layer.
        dict(name="store 8b 4x2048", kind="store", heads="8b", dtype="bf16", batch=4, rows=2048, ctx=0, room=256),
        # Plain decoding of one sequence over a short cache.
        dict(name="attn 1b 1x1 ctx130", kind="attn", heads="1b", dtype="bf16", batch=1, nodes=1, ctx=130, room=60, pad=0),
        # Verification of a 16-node tree per sequence, eight sequences: the ordinary serving step.
        dict(name="attn 8b 8x16 ctx4096", kind="attn", heads="8b", dtype="bf16", batch=8, nodes=16, ctx=4096, room=64, pad=3),
        # The fp32 parity configuration with odd sizes and padded trees.
        dict(name="attn tiny fp32 3x37 ctx901", kind="attn", heads="tiny", dtype="fp32", batch=3, nodes=37, ctx=901, room=41,
             pad=9),
        # Single tokens over long caches, what such a cache is for.
        dict(name="attn 8b 4x1 ctx65536", kind="attn", heads="8b", dtype="bf16", batch=4, nodes=1, ctx=65536, room=64, pad=0),
        # Wide trees over long caches.
        dict(name="attn 8b 16x64 ctx16384", kind="attn", heads="8b", dtype="bf16", batch=16, nodes=64, ctx=16384, room=64,
             pad=5),
        # A short block of one sequence at a small vocabulary, its draft by the largest logits (no distribution of its own).
        dict(name="draft fp32 1x3 4096 point", kind="draft", dtype="fp32", batch=1, drafted=3, vocab=4096, extra=5, point=True,
             temperature=1.0),
        # The framework's draft blocks: eight sequences of 15 drafted tokens, drawn from the drafter's own logits.
        dict(name="draft 8x15 151936", kind="draft", dtype="bf16", batch=8, drafted=15, vocab=151936, extra=0, point=False,
             temperature=0.8),
        # One sequence, one node: the next token of plain decoding.
        dict(name="walk 1x1 32000", kind="walk", dtype="bf16", batch=1, nodes=1, vocab=32000, extra=0, pad=0, temperature=0.7),
        # Trees of an ordinary serving step, requests of different temperatures, greedy ones among them.
        dict(name="walk 8x16 151936", kind="walk", dtype="bf16", batch=8, nodes=16, vocab=151936, extra=0, pad=3,
             temperature=-1.0),
        # Wide trees of many sequences.
        dict(name="walk 16x64 151936", kind="walk", dtype="bf16", batch=16, nodes=64, vocab=151936, extra=0, pad=5,
             temperature=1.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "attn", "attn", "draft", "walk"])
    heads = rng.choice(list(HEADS))
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    while True:
        if kind == "store":
            c = dict(kind=kind, heads=heads, dtype=dtype, batch=_log_int(rng, 1, 16), rows=_log_int(rng, 1, 4096),
                     ctx=rng.choice([0, 0, _log_int(rng, 1, 4096)]), room=rng.randint(0, 70))
        elif kind == "attn":
            c = dict(kind=kind, heads=heads, dtype=dtype, batch=_log_int(rng, 1, 16), nodes=_log_int(rng, 1, 64),
                     ctx=_log_int(rng, 1, 65536), room=rng.randint(0, 70))
            c["pad"] = rng.randint(0, c["nodes"] // 2)
        else:
            c = dict(kind=kind, dtype=dtype, batch=_log_int(rng, 1, 16), vocab=rng.choice([*VOCABS, _log_int(rng, 40, 152000)]),
                     extra=rng.choice([0, 0, 1, 8, 13]), temperature=rng.choice([1.0, 0.7, 0.0, -1.0]))
            if kind == "draft":
                c["drafted"], c["point"] = _log_int(rng, 1, 31), rng.random() < 0.3
            else:
                c["nodes"] = _log_int(rng, 1, 64)
                c["pad"] = rng.randint(0, c["nodes"] // 2)
        w = work(c)
        if w["bytes"] <= 3.2e8 and w["flops"] <= 2e11:
            return c


def _lengths(case):
    """Committed rows per sequence: the first holds ``ctx``, the others fewer, down to about half."""
    ctx, B = case["ctx"], case["batch"]
    return [ctx - (b * ctx) // (2 * B) for b in range(B)]


def _drafted(case):
    """Drafted tokens per sequence: ragged blocks."""
    return [max(0, case["drafted"] - b % 3) for b in range(case["batch"])]


def work(case):
    es = DTYPES[case["dtype"]].itemsize
    B = case["batch"]
    if case["kind"] in ("draft", "walk"):
        V = case["vocab"]
        if case["kind"] == "walk":
            R = B * case["nodes"] - case["pad"] * ((B + 1) // 2)
            return dict(bytes=R * V * es + 32 * B * case["nodes"], flops=4 * R * V)
        n = sum(_drafted(case))
        R = n + B + (0 if case["point"] else n)
        return dict(bytes=R * V * es + 12 * B * (case["drafted"] + 1), flops=4 * R * V)
    nq, nk, d = HEADS[case["heads"]]
    row4 = d // 2 + d // 32
    if case["kind"] == "store":
        rows = 2 * B * case["rows"] * nk
        # rows read, 4-bit rows written; those read, and their numbers written
        return dict(bytes=rows * (2 * d * es + 2 * row4), flops=4 * rows * d)
    T = case["nodes"]
    keys = sum(_lengths(case)) + B * T
    return dict(bytes=keys * nk * row4 * 2 + 2 * B * T * nq * d * es + B * T * 4, flops=4 * d * nq * T * keys)


# ---- the 4-bit format --------------------------------------------------------------------------
def _quantise(x):
    """Codes (0 .. 7, 8 the sign) and scale bytes of rows of x [..., D] fp32."""
    g = x.unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)                                       # top = m 2^e, m in [0.5, 1): below 7 scales of 2^(e - 3), or the next
    e = torch.where(m >= 0.875, e - 2, e - 3)
    byte = torch.where(top > 0, e + 127, 2).clamp(2, 252)
    y = torch.ldexp(g.abs(), 127 - byte)
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int() + (y >= 3.5).int()
            + (y > 5).int())
    return (code + 8 * torch.signbit(g).int()).flatten(-2), byte.squeeze(-1)


def _values(code, byte):
    """The numbers that codes and scale bytes stand for, fp32."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=code.device)
    return torch.ldexp(grid[code.long()].unflatten(-1, (-1, 32)), (byte.int() - 127)[..., None]).flatten(-2)


def _pack(code, byte):
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), byte.to(torch.uint8)


def _unpack(codes, scales):
    c = codes.int()
    return _values(torch.stack((c & 15, c >> 4), -1).flatten(-2), scales)


# ---- inputs ------------------------------------------------------------------------------------
def _tree(B, T, pad, g):
    """Parents of B trees of T nodes: node 0 is the root, a later node hangs on an earlier one; the last ``pad`` nodes of
    every second tree are padding (-2)."""
    t = torch.arange(T, device=DEV)
    p = (torch.rand((B, T), device=DEV, generator=g) * t).floor().long()
    p = torch.minimum(p, (t - 1).clamp(min=0))
    p[:, 0] = -1
    if pad:
        p[::2, T - pad:] = -2
    return p.int().contiguous()


def _logits(rows, vocab, extra, dtype, g):
    """Logits as an LM head gives them: most within a few units of zero, a handful per row well above, some tokens that may
    not come (-inf); rows with ``extra`` elements between them."""
    z = torch.empty((rows, vocab + extra), device=DEV, dtype=dtype)
    for r in range(0, rows, 256):
        part = torch.randn((min(256, rows - r), vocab + extra), device=DEV, generator=g)
        chance = torch.rand(part.shape, device=DEV, generator=g)
        part = torch.where(chance < 8.0 / vocab, part.abs() * 2 + 9, part * 2)
        z[r:r + 256] = part.masked_fill(chance > 1 - 1e-3, -math.inf).to(dtype)
    return z[:, :vocab]


def _temperature(case, g):
    """The case's temperature; -1: another one for each sequence, some of them 0."""
    if case["temperature"] >= 0:
        return case["temperature"]
    t = 0.5 + torch.rand(case["batch"], device=DEV, generator=g)
    t[::3] = 0.0
    return t


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    kind, B = case["kind"], case["batch"]
    s = dict(kind=kind)

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=g)

    if kind == "draft":
        L, V = case["drafted"], case["vocab"]
        s["z"] = _logits(B * (L + 1), V, case["extra"], dt, g)
        t = s["temperature"] = _temperature(case, g)
        t_row = torch.as_tensor(t, device=DEV, dtype=torch.float32).expand(B)[:, None]
        tokens = torch.empty((B, L), device=DEV, dtype=torch.int64)
        s["draft"] = None if case["point"] else torch.empty((B * L, V), device=DEV, dtype=dt)
        for b in range(B):
            # the drafter's logits: the target's with noise; its tokens drawn from them (largest of logits with Gumbel noise)
            y = s["z"][b * (L + 1):(b + 1) * (L + 1) - 1].float()
            y = y + 0.5 * randn(L, V)
            if s["draft"] is not None:
                s["draft"][b * L:(b + 1) * L] = y.to(dt)
                y = s["draft"][b * L:(b + 1) * L].float()
                noise = -torch.log(-torch.log(torch.rand((L, V), device=DEV, generator=g).clamp(1e-7, 1 - 1e-7)))
                y = y + t_row[b] * noise
            tokens[b] = y.argmax(1)
        s["tokens"] = tokens
        s["u"] = torch.rand((B, L + 1), device=DEV, generator=g)
        s["counts"] = torch.tensor(_drafted(case), device=DEV)
        return s
    if kind == "walk":
        T, V = case["nodes"], case["vocab"]
        s["z"] = _logits(B * T, V, case["extra"], dt, g)
        s["temperature"] = _temperature(case, g)
        s["parents"] = _tree(B, T, case["pad"], g)
        # a node's token: one of the largest few of its parent's logits, the first children the likelier ones
        k = min(8, V)
        top = torch.cat([torch.topk(s["z"][r:r + 256].float(), k, dim=1).indices for r in range(0, B * T, 256)]).view(B, T, k)
        p = s["parents"].long()
        rank = torch.stack([(p[:, :t] == p[:, t:t + 1]).sum(1) for t in range(T)], 1).clamp(max=k - 1)
        s["tokens"] = top.gather(1, p.clamp(min=0)[..., None].expand(B, T, k)).gather(2, rank[..., None])[..., 0].contiguous()
        s["u"] = torch.rand((B, T), device=DEV, generator=g)
        return s
    nq, nk, d = HEADS[case["heads"]]
    n = _lengths(case)
    s["lengths"] = torch.tensor(n, device=DEV)
    if kind == "store":
        T = case["rows"]
        max_len = case["ctx"] + T + case["room"]
        # keys as the norm and the rotation leave them, values as columns of the projection's output
        s["rows"] = [randn(B * T, nk * d).to(dt), randn(B * T, (nq + 2 * nk) * d).to(dt)[:, (nq + nk) * d:]]
        s["caches"] = [(torch.zeros((B, nk, max_len, d // 2), device=DEV, dtype=torch.uint8),
                        torch.zeros((B, nk, max_len, d // 32), device=DEV, dtype=torch.uint8)) for _ in "kv"]
        s["T"], s["d"], s["dtype"] = T, d, dt
        return s
    T = case["nodes"]
    max_len = case["ctx"] + T + case["room"]
    s["parents"] = _tree(B, T, case["pad"], g)
    s["q"] = randn(B * T, nq * d).to(dt)
    for name in "kv":
        codes = torch.empty((B, nk, max_len, d // 2), device=DEV, dtype=torch.uint8)
        scales = torch.empty((B, nk, max_len, d // 32), device=DEV, dtype=torch.uint8)
        for b in range(B):
            codes[b], scales[b] = _pack(*_quantise(randn(nk, max_len, d)))
        s[name] = (codes, scales)
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)[state["kind"]](state)


def _own_store(s):
    from uno_amd import kernels as K

    caches = [K.Rows4(*c) for c in s["caches"]]
    K.cache4_store(s["rows"], caches, s["lengths"])
    return K.cache4_load(caches, s["lengths"], s["T"], dtype=s["dtype"])


def _own_attn(s):
    from uno_amd import kernels as K

    return K.tree_attn4(s["q"], K.Rows4(*s["k"]), K.Rows4(*s["v"]), s["lengths"], s["parents"])


def _own_draft(s):
    from uno_amd import kernels as K

    return K.verify_draft(s["z"], s["draft"], s["tokens"], s["u"], counts=s["counts"], temperature=s["temperature"])


def _own_walk(s):
    from uno_amd import kernels as K

    return K.verify_tree(s["z"], s["tokens"], s["parents"], s["u"], temperature=s["temperature"])


def _plain_store(s):
    return [_values(*_quantise(x.float().unflatten(1, (-1, s["d"])))).flatten(1).to(x.dtype) for x in s["rows"]]


def _plain_attn(s):
    q, n, parents = s["q"], s["lengths"], s["parents"]
    k, v = _unpack(*s["k"]), _unpack(*s["v"])
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
    z = (qs @ k.transpose(2, 3).contiguous()).view(B, nk, rep, T, max_len) * d ** -0.5
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p.view(B, nk, rep * T, max_len) @ v
    return o.view(B, nk, rep, T, d).permute(0, 3, 1, 2, 4).reshape(B * T, nk * rep * d).to(q.dtype)


def _weights(z, temperature):
    """Sampling weights [R, V] fp64 of logits [R, V] at a temperature (a device scalar)."""
    z = z.double()
    top = z.amax(1, keepdim=True)
    x = (z - top) / torch.where(temperature > 0, temperature, 1.0).double()
    w = torch.where(x >= -700, torch.exp(x), 0.0)
    j = torch.arange(z.shape[1], device=z.device)
    first = torch.where(z == top, j, z.shape[1]).amin(1, keepdim=True)
    return torch.where(temperature > 0, w, (j == first).double())


def _sample(w, u):
    """For each row of the weights w [R, V] the token at u [R]."""
    total = w.cumsum(1)
    at = (total <= u.double()[:, None] * total[:, -1:]).sum(1)
    last = torch.where(w > 0, torch.arange(w.shape[1], device=w.device), -1).amax(1)
    return torch.minimum(at, last)


def _plain_draft(s):
    z, y, tokens, u, counts = s["z"], s["draft"], s["tokens"], s["u"], s["counts"]
    B, L = tokens.shape
    V = z.shape[1]
    temperature = torch.as_tensor(s["temperature"], device=z.device, dtype=torch.float32).expand(B)
    j = torch.arange(L, device=z.device)
    accepted, nexts = [], []
    for b in range(B):
        w = _weights(z[b * (L + 1):(b + 1) * (L + 1)], temperature[b])
        p = w / w.sum(1, keepdim=True)
        if y is None:
            q = (torch.arange(V, device=z.device) == tokens[b, :, None]).double()
        else:
            q = _weights(y[b * L:(b + 1) * L], temperature[b])
            q = q / q.sum(1, keepdim=True)
        px, qx = (a[:L].gather(1, tokens[b, :, None])[:, 0] for a in (p, q))
        ok = (u[b, :L].double() * qx < px) & (j < counts[b])
        n = ok.long().cumprod(0).sum()
        here = p.index_select(0, n[None])
        left = (here - q.index_select(0, n.clamp(max=L - 1)[None])).clamp(min=0)
        left = torch.where((n < counts[b]) & (left.sum() >= LEAST), left, here)
        accepted.append(n)
        nexts.append(_sample(left, u[b, L:])[0])
    return torch.stack(accepted), torch.stack(nexts)


def _plain_walk(s):
    z, tokens, parents, u = s["z"], s["tokens"], s["parents"], s["u"]
    B, T = tokens.shape
    temperature = torch.as_tensor(s["temperature"], device=z.device, dtype=torch.float32).expand(B)
    drawn = torch.stack([_sample(_weights(z[b * T:(b + 1) * T], temperature[b]), u[b]) for b in range(B)])
    t = torch.arange(T, device=z.device)
    b = torch.arange(B, device=z.device)
    nodes = torch.full((B, T), -1, device=z.device)
    nodes[:, 0] = 0
    at, counts, live = torch.zeros_like(b), torch.ones_like(b), torch.ones_like(b, dtype=torch.bool)
    for i in range(1, T):
        child = (parents == at[:, None]) & (tokens == drawn[b, at][:, None]) & (t > at[:, None])
        live = live & child.any(1)
        at = torch.where(live, torch.where(child, t, T).amin(1).clamp(max=T - 1), at)
        nodes[:, i] = torch.where(live, at, -1)
        counts = counts + live
    return nodes, counts, drawn[b, at]


_own = dict(store=_own_store, attn=_own_attn, draft=_own_draft, walk=_own_walk)
_plain = dict(store=_plain_store, attn=_plain_attn, draft=_plain_draft, walk=_plain_walk)


# ---- the definitions in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return [_exact_values(x.double(), s["d"]) for x in s["rows"]]
    if case["kind"] == "attn":
        return _exact_attn(s)
    return _exact_draft(s) if case["kind"] == "draft" else _exact_walk(s)


def _exact_values(x, d):
    """Each element's nearest number of its group's grid."""
    out = []
    for part in x.reshape(-1, 32).split(1 << 16):
        top = part.abs().amax(1, keepdim=True)
        step = torch.full_like(top, 2.0 ** -125)
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 7))
        for de in (-1, 0, 1):                                     # the least power of two with top < 7 step
            s = torch.exp2((e + de).clamp(-125, 125))
            step = torch.where((top < 7 * s) & ((top >= 3.5 * s) | (e + de <= -125)) | ((e + de >= 125) & (top >= 7 * s)), s, step)
        grid = torch.tensor(GRID, device=x.device, dtype=torch.float64)
        far = (part.abs()[..., None] / step[..., None] - grid).abs()
        near = far.amin(-1, keepdim=True) == far                  # one, or two neighbours: the even code
        even = torch.arange(8, device=x.device) % 2 == 0
        pick = near & (even | (near.sum(-1, keepdim=True) == 1))
        out.append((pick * grid).sum(-1) * step * torch.sign(part))
    return torch.cat(out).view(x.shape)


def _exact_attn(s):
    q, n, parents = s["q"], s["lengths"].tolist(), s["parents"].tolist()
    B, nk, _, half = s["k"][0].shape
    d, T = 2 * half, len(parents[0])
    rep = q.shape[1] // (nk * d)
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=DEV, dtype=torch.float64)
    j = torch.arange(d, device=DEV)

    def rows(cache, b, h, end):
        codes, scales = (c[b, h, :end].long() for c in cache)
        return grid[codes[:, j // 2] >> 4 * (j % 2) & 15] * torch.exp2(scales[:, j // 32] - 127.0)

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
            kd, vd = (rows(c, b, h, n[b] + T) for c in (s["k"], s["v"]))
            for r in range(rep):
                qd = q.view(B, T, nk, rep, d)[b, :, h, r].double()
                a = torch.softmax(qd @ kd.T.contiguous() * d ** -0.5 + bias, 1)
                out[b, some, h, r] = (a @ vd)[some]
    return out.view(B * T, nk * rep * d)


def _probabilities(z, temperature):
    """The distribution [V] that one row of logits gives at a temperature."""
    z = z.double()
    if temperature == 0:
        p = torch.zeros_like(z)
        p[int((z == z.max()).nonzero()[0])] = 1.0
        return p
    x = (z - z.max()) / temperature
    p = torch.where(x < -700, torch.zeros_like(x), x.exp())
    return p / p.sum()


def _drawn(p, u):
    total = torch.cumsum(p, 0)
    over = (total > u * total[-1]).nonzero()
    return int(over[0]) if len(over) else int((p > 0).nonzero()[-1])


def _per_sequence(s, B):
    t = s["temperature"]
    return t.tolist() if torch.is_tensor(t) else torch.full((B,), t).tolist()     # as fp32 holds it


def _exact_draft(s):
    tokens, u, counts = s["tokens"].tolist(), s["u"].tolist(), s["counts"].tolist()
    B, L = len(tokens), len(tokens[0])
    accepted, nexts = [], []
    for b, temperature in enumerate(_per_sequence(s, B)):
        for i in range(L + 1):
            p = _probabilities(s["z"][b * (L + 1) + i], temperature)
            if i == counts[b]:
                break
            x = tokens[b][i]
            if s["draft"] is None:
                q = torch.zeros_like(p)
                q[x] = 1.0
            else:
                q = _probabilities(s["draft"][b * L + i], temperature)
            if not u[b][i] * float(q[x]) < float(p[x]):
                left = torch.where(p > q, p - q, torch.zeros_like(p))
                p = left if float(left.sum()) >= LEAST else p
                break
        accepted.append(i)
        nexts.append(_drawn(p, u[b][L]))
    return torch.tensor(accepted, device=DEV), torch.tensor(nexts, device=DEV)


def _exact_walk(s):
    tokens, u, parents = s["tokens"].tolist(), s["u"].tolist(), s["parents"].tolist()
    B, T = len(tokens), len(tokens[0])
    nodes, counts, nexts = [], [], []
    for b, temperature in enumerate(_per_sequence(s, B)):
        path = [0]
        while True:
            at = path[-1]
            token = _drawn(_probabilities(s["z"][b * T + at], temperature), u[b][at])
            children = [t for t in range(at + 1, T) if parents[b][t] == at and tokens[b][t] == token]
            if not children:
                break
            path.append(children[0])
        nodes.append(path + [-1] * (T - len(path)))
        counts.append(len(path))
        nexts.append(token)
    return torch.tensor(nodes, device=DEV), torch.tensor(counts, device=DEV), torch.tensor(nexts, device=DEV)
