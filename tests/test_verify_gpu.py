"""Verification of drafted tokens (K.verify_draft, K.verify_tree) against the definition in 64 bits, on the host. Results are whole
numbers: they are compared for equality. (A result could differ where u lies within the sums' errors, some 1e-13, of a border between
tokens; with fp32 random numbers and 1e5 columns that has a chance of 1e-8 for a drawn token.)"""
import math

import pytest
import torch

from uno_amd import kernels as K

pytestmark = pytest.mark.gpu

BF, F32, I64 = torch.bfloat16, torch.float32, torch.int64


def _distribution(z, t):
    """The distribution of one row of logits at temperature t, fp64 on the CPU (None: none)."""
    z = z.double().cpu()
    top = z.max()
    if bool(z.isnan().any()) or not bool(torch.isfinite(top)):
        return None
    if not t > 0:
        return (torch.arange(len(z)) == int((z == top).nonzero()[0])).double()
    x = torch.where(z == -math.inf, -math.inf, (z - top) / t)
    w = torch.where(x >= -700, x.exp(), 0.0)
    return w / w.sum()


def _draw(p, u):
    u = max(u, 0.0)                                     # below 0: as 0
    run = p.cumsum(0)
    over = (run > u * run[-1]).nonzero()
    return int(over[0]) if len(over) else int((p > 0).nonzero()[-1])


def _temps(temperature, B):
    return temperature.tolist() if torch.is_tensor(temperature) else torch.full((B,), temperature).tolist()


def _draft(z, y, tokens, u, counts, temperature):
    B, L = tokens.shape
    accepted, nexts = [], []
    for b, t in enumerate(_temps(temperature, B)):
        n = L if counts is None else min(max(int(counts[b]), 0), L)
        for i in range(n + 1):
            p = _distribution(z[b * (L + 1) + i], t)
            if p is None or i == n:
                break
            x = int(tokens[b, i])
            inside = 0 <= x < len(p)
            if y is None or not t > 0:
                q = (torch.arange(len(p)) == x).double()
            else:
                q = _distribution(y[b * L + i], t)
                if q is None:
                    p = None
                    break
            if not t > 0:
                ok = inside and p[x] == 1
            else:
                ok = inside and max(float(u[b, i]), 0.0) * float(q[x]) < float(p[x])
            if not ok:
                left = (p - q).clamp(min=0) if t > 0 else p
                p = left if left.sum() >= 2.0 ** -40 else p
                break
        accepted.append(i)
        nexts.append(-1 if p is None else _draw(p, float(u[b, L])))
    return torch.tensor(accepted), torch.tensor(nexts)


def _tree(z, tokens, parents, u, temperature):
    B, T = tokens.shape
    nodes, counts, nexts = torch.full((B, T), -1), torch.zeros(B, dtype=I64), torch.full((B,), -1)
    for b, t in enumerate(_temps(temperature, B)):
        par = parents[b] if parents.dim() == 2 else parents
        at = 0 if par[0] >= -1 else None
        while at is not None:
            nodes[b, counts[b]] = at
            counts[b] += 1
            p = _distribution(z[b * T + at], t)
            nexts[b] = -1 if p is None else _draw(p, float(u[b, at]))
            at = next((c for c in range(at + 1, T) if p is not None and par[c] == at and tokens[b, c] == nexts[b]), None)
    return nodes, counts, nexts


def _logits(dev, rows, V, dtype, seed, extra=0):
    """As an LM head gives them: a few large ones, some -inf."""
    g = torch.Generator(device=dev).manual_seed(seed)
    z = torch.randn(rows, V + extra, device=dev, generator=g) * 2
    z = torch.where(torch.rand(z.shape, device=dev, generator=g) < 6.0 / V, z.abs() + 8, z)
    if V > 8:
        z = z.masked_fill(torch.rand(z.shape, device=dev, generator=g) < 0.01, -math.inf)
    return z.to(dtype)[:, :V]


def _drafted(dev, B, L, V, dtype, seed, extra=0, point=False, temperature=1.0):
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    z = _logits(dev, B * (L + 1), V, dtype, seed, extra)
    own = torch.arange(B * (L + 1), device=dev).view(B, L + 1)[:, :L].reshape(-1)
    y = z[own].float() + 0.5 * torch.randn(B * L, V, device=dev, generator=g)
    if extra:
        y = torch.cat([y, y[:, :extra]], 1).to(dtype)[:, :V]
    else:
        y = y.to(dtype)
    t = temperature if not torch.is_tensor(temperature) else 1.0
    noise = -torch.log(-torch.log(torch.rand(B * L, V, device=dev, generator=g).clamp(1e-7, 1 - 1e-7)))
    x = (y.float() + (0 if point else t) * noise).argmax(1).view(B, L)
    u = torch.rand(B, L + 1, device=dev, generator=g)
    return z, None if point else y, x, u


def _check_draft(z, y, x, u, counts=None, temperature=1.0):
    got = K.verify_draft(z, y, x, u, counts=counts, temperature=temperature)
    want = _draft(z, y, x.cpu(), u.cpu(), counts, temperature)
    assert torch.equal(got[0].cpu(), want[0]), (got[0].tolist(), want[0].tolist())
    assert torch.equal(got[1].cpu(), want[1]), (got[1].tolist(), want[1].tolist())
    return want


def _check_tree(z, tokens, parents, u, temperature=1.0):
    got = K.verify_tree(z, tokens, parents, u, temperature=temperature)
    want = _tree(z, tokens.cpu(), parents.cpu(), u.cpu(), temperature)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b), (a.tolist(), b.tolist())
    return want


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("point", [False, True])
@pytest.mark.parametrize("B,L,V,extra", [(1, 1, 1, 0), (2, 3, 2, 1), (3, 5, 7, 0), (4, 15, 1000, 3), (3, 4, 2047, 0), (3, 4, 2048, 8),
                                         (3, 4, 2049, 1), (2, 31, 4096, 5), (5, 7, 32000, 0), (2, 4, 151936, 13)])
def test_drafted_blocks(dev, dtype, point, B, L, V, extra):
    print(f"[draft] {dtype} B={B} L={L} V={V} point={point}", flush=True)
    for seed in range(2):
        _check_draft(*_drafted(dev, B, L, V, dtype, seed, extra, point))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("temperature", [0.0, 1e-38, 0.3, 2.5, 1e30])
def test_temperatures(dev, dtype, temperature):
    z, y, x, u = _drafted(dev, 6, 5, 3001, dtype, 4, temperature=min(temperature, 2.5))
    _check_draft(z, y, x, u, temperature=temperature)
    _check_draft(z, None, x, u, temperature=temperature)


def test_temperatures_of_each_sequence(dev):
    """Greedy ones, warm ones, and what is no temperature (taken as 0; infinity as every finite logit alike)."""
    temps = torch.tensor([0.0, 0.7, 1.0, -1.0, math.nan, 3.0, math.inf], device=dev)
    z, y, x, u = _drafted(dev, 7, 6, 5000, BF, 5)
    want = [0.0, 0.7, 1.0, 0.0, 0.0, 3.0, 1e30]
    got = K.verify_draft(z, y, x, u, temperature=temps)
    ref = _draft(z, y, x.cpu(), u.cpu(), None, torch.tensor(want))
    assert torch.equal(got[0].cpu(), ref[0]) and torch.equal(got[1].cpu(), ref[1])
    T = 7
    tokens, parents = x.repeat(1, 2)[:, :T].contiguous(), (torch.arange(T, dtype=torch.int32, device=dev) - 1)
    got = K.verify_tree(z[:7 * T], tokens, parents, torch.rand(7, T, device=dev), temperature=temps * 0)
    ref = _tree(z[:7 * T], tokens.cpu(), parents.cpu(), torch.zeros(7, T), 0.0)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, ref))


def test_counts(dev):
    """Blocks of different lengths; the rows behind them may hold anything."""
    B, L, V = 7, 6, 700
    z, y, x, u = _drafted(dev, B, L, V, F32, 7)
    counts = torch.tensor([0, 1, 3, 6, 99, -5, 5], device=dev)
    for b, n in enumerate(counts.clamp(0, L).tolist()):
        z[b * (L + 1) + n + 1:(b + 1) * (L + 1)] = math.nan
        y[b * L + n:(b + 1) * L] = math.nan
        x[b, n:] = -1
    want = _check_draft(z, y, x, u, counts)
    assert bool((want[1] >= 0).all())
    _check_draft(z, None, x, u, counts)


def test_no_drafted_tokens(dev):
    z, _, x, u = _drafted(dev, 4, 1, 900, BF, 8)
    z, u, x = z[:4], u[:, :1].contiguous(), x[:, :0].contiguous()
    _check_draft(z, None, x, u)
    _check_draft(z, z[:0], x, u)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_extreme_random_numbers(dev, dtype):
    """u = 0 (and below) takes the first token with a weight, u = 1 (and above) the last; nothing is accepted at u = 1 where p < q, all
    is at u = 0 where p > 0."""
    B, L, V = 4, 3, 5000
    z, y, x, u = _drafted(dev, B, L, V, dtype, 9)
    z[:, :70], z[:, -70:] = -math.inf, -math.inf
    z[0, 0] = z[0].max() - 750                          # a weight that counts as 0
    for value in (0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -3.0):
        u.fill_(value)
        _check_draft(z, y, x, u)
        _check_draft(z, None, x, u)
        _check_tree(z, x.new_zeros(B, L + 1), torch.tensor([-1, 0, 0, 2], device=dev, dtype=torch.int32), u)


@pytest.mark.parametrize("scale,temperature", [(1e9, 1.0), (50.0, 1e-7), (50.0, 1e-12), (1e4, 1e-3), (1e30, 1e30), (3e38, 1e36), (1e-30, 1e-32),
                                               (1.0, 3e38), (1.0, 1e-38), (700.0, 1.0), (3e38, 1e-30)])
def test_logits_and_temperatures_of_any_size(dev, scale, temperature):
    """Logits around +- scale that differ by multiples of an fp32 step, of the temperature, and by infinities."""
    B, L, V = 3, 4, 4100
    temperature = float(torch.tensor(temperature))       # as fp32 has it
    g = torch.Generator("cpu").manual_seed(17)
    near = max(temperature, scale * 2.0 ** -22)
    z = (scale * (1 - 2.0 ** -10) - near * 2 * torch.rand(B * (L + 1), V, generator=g).double()).float()
    z[:, ::5] = -math.inf
    z[:, 1::7] = -scale
    z[2::3] = (-scale + near * torch.rand(V, generator=g).double()).float()
    z[0, 2100:] = -math.inf
    z = z.to(dev)
    u = torch.rand(B, L + 1, generator=g).to(dev)
    x = torch.zeros(B, L, device=dev, dtype=I64)
    _check_draft(z, None, x, u, temperature=temperature)
    _check_tree(z, x.new_zeros(B, L + 1), torch.tensor([-1, 0, 0, 2, 3], device=dev, dtype=torch.int32), u, temperature=temperature)


def test_equal_logits(dev):
    """Flat rows: every border is a multiple of 1 / V, and u on a border belongs to the token behind it."""
    V = 4096
    z = torch.full((8, V), 3.0, device=dev)
    u = torch.tensor([[0.0], [1 / V], [5 / V], [2047 / V], [2048 / V], [0.5 - 2.0 ** -13], [4095 / V], [1 - 2.0 ** -24]], device=dev)
    parents = torch.tensor([[-1]] * 8, device=dev, dtype=torch.int32)
    nodes, counts, token = K.verify_tree(z, torch.zeros(8, 1, device=dev, dtype=I64), parents, u)
    assert token.tolist() == [0, 1, 5, 2047, 2048, 2047, 4095, 4095] and counts.tolist() == [1] * 8 and not nodes.any()
    accepted, token = K.verify_draft(z, None, torch.zeros(4, 1, device=dev, dtype=I64), torch.rand(4, 2, device=dev), temperature=0.0)
    assert accepted.tolist() == [1] * 4 and token.tolist() == [0] * 4      # the lowest of equal ones
    z[:, 100] = 4.0
    z[:, 90] = 4.0
    accepted, token = K.verify_draft(z, None, torch.full((4, 1), 100, device=dev), torch.rand(4, 2, device=dev), temperature=0.0)
    assert accepted.tolist() == [0] * 4 and token.tolist() == [90] * 4


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_rows_without_a_distribution(dev, dtype, temperature):
    """NaN, +inf or -inf alone end a sequence where they are met, and nowhere else."""
    B, L, V = 9, 4, 2100
    z, y, x, u = _drafted(dev, B, L, V, dtype, 11)
    u[:, :L] = 0.0                                      # accepted while p > 0
    z[z == -math.inf] = -20.0
    if temperature == 0:
        x = z.view(B, L + 1, V)[:, :L].float().argmax(2)
    z[0 * (L + 1) + 2, V - 1] = math.nan
    z[1 * (L + 1) + 0, 0] = math.inf
    z[2 * (L + 1) + 4] = -math.inf                      # behind the last
    y[3 * L + 1, 5] = math.nan
    y[4 * L + 3] = -math.inf
    y[5 * L, V // 2] = math.inf
    z[6 * (L + 1), 1:] = -math.inf                      # one token alone
    z[7 * (L + 1), 33] = 3e38 if dtype == F32 else 3.3e38
    want = _check_draft(z, y, x, u, temperature=temperature)
    assert want[1][0] == want[1][1] == want[1][2] == -1
    _check_draft(z, None, x, u, temperature=temperature)
    tokens = torch.cat([x[:, :1], x], 1).contiguous()   # a chain of the same tokens
    _check_tree(z, tokens, torch.arange(-1, L, device=dev, dtype=torch.int32), torch.rand(B, L + 1, device=dev), temperature)


def test_tokens_outside_the_vocabulary(dev):
    """Are refused, and take nothing from the target's distribution."""
    z, y, x, u = _drafted(dev, 5, 2, 300, F32, 12)
    x[0, 0], x[1, 1], x[2, 0], x[3, 0], x[4, 0] = -1, 300, 2 ** 40, -2 ** 63, 2 ** 32 + 5
    _check_draft(z, y, x, u)
    _check_draft(z, None, x, u)
    _check_tree(z, torch.cat([x, x[:, :1]], 1).contiguous(), torch.tensor([-1, 0, 1], device=dev, dtype=torch.int32),
                torch.rand(5, 3, device=dev))


def test_a_draft_like_the_target_is_accepted(dev):
    z, _, x, u = _drafted(dev, 4, 8, 6000, BF, 13)
    y = z.view(4, 9, -1)[:, :8].reshape(32, -1).contiguous()
    x = torch.multinomial(torch.softmax(y.float(), 1), 1).view(4, 8)
    assert _check_draft(z, y, x, u)[0].tolist() == [8] * 4


def test_tokens_are_distributed_as_the_target_says(dev):
    """60000 blocks of one token over six columns: the first token that comes out (the drafted one or the next) has the
    target's frequencies, whatever drafted; counts of a binomial distribution, within six of its deviations. So have a tree's."""
    B, V = 60000, 6
    g = torch.Generator(device=dev).manual_seed(5)
    p, q = torch.tensor([0.3, 0.25, 0.2, 0.15, 0.08, 0.02]), torch.tensor([0.05, 0.1, 0.5, 0.3, 0.03, 0.02])
    z, y = p.log().to(dev).repeat(2 * B, 1), q.log().to(dev).repeat(B, 1)
    x = torch.multinomial(q.to(dev), B, replacement=True, generator=g)[:, None].contiguous()
    u = torch.rand(B, 2, device=dev, generator=g)
    for draft, tokens in ((y, x), (None, torch.full_like(x, 2))):
        accepted, token = K.verify_draft(z, draft, tokens, u)
        first = torch.where(accepted > 0, tokens[:, 0], token)
        for a, b in ((first, p), (token[accepted > 0], p)):
            n = a.numel()
            off = (torch.bincount(a, minlength=V).cpu().double() - n * b).abs()
            assert bool((off <= 6 * (n * b * (1 - b)).sqrt()).all())
        share = float(torch.minimum(p, q).sum()) if draft is not None else float(p[2])
        assert abs(float(accepted.sum()) - B * share) <= 6 * math.sqrt(B * share * (1 - share))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,V,extra", [(1, 1, 1, 0), (3, 1, 32000, 0), (2, 3, 2, 1), (4, 16, 1000, 3), (3, 37, 2049, 1), (2, 256, 300, 0),
                                         (2, 64, 4096, 8), (2, 16, 151936, 13)])
def test_trees(dev, dtype, B, T, V, extra):
    """Random trees whose nodes hold likely tokens of their parents, several of them the same; padding; another root."""
    print(f"[walk] {dtype} B={B} T={T} V={V}", flush=True)
    g = torch.Generator().manual_seed(T)
    for seed in range(2):
        z = _logits(dev, B * T, V, dtype, seed, extra)
        parents = torch.full((B, T), -1, dtype=torch.int32)
        for b in range(B):
            for t in range(1, T):
                parents[b, t] = int(torch.randint(max(-1, t - 6), t, (1,), generator=g))
            if T > 9 and b % 2:
                parents[b, T - 4:] = -2
                z[b * T + T - 4:(b + 1) * T] = math.nan
        k = min(3, V)
        top = torch.topk(z.float(), k, dim=1).indices.view(B, T, k).cpu()
        pick = torch.randint(0, k, (B, T), generator=g)
        tokens = torch.stack([top[b, parents[b].long().clamp(min=0), pick[b]] for b in range(B)])
        u = torch.rand(B, T, generator=g)
        _check_tree(z, tokens.to(dev), parents.to(dev), u.to(dev), 0.5)
        _check_tree(z, tokens.to(dev), parents[0].to(dev), u.to(dev), 0.5)


def test_odd_parents(dev):
    """Parents that are no earlier node have no way to them; a tree whose node 0 is padding has no path."""
    B, T, V = 3, 6, 50
    z = torch.full((B * T, V), -math.inf, device=dev)
    z[:, 7] = 0.0                                       # every node draws token 7
    tokens = torch.full((B, T), 7, device=dev)
    parents = torch.tensor([[0, 5, 1, 0, 9, 3], [-2, 0, 1, 2, 3, 4], [-1, -1, 1, -2, 3, 0]], device=dev, dtype=torch.int32)
    nodes, counts, token = K.verify_tree(z, tokens, parents, torch.rand(B, T, device=dev))
    assert nodes.tolist() == [[0, 3, 5, -1, -1, -1], [-1] * 6, [0, 5, -1, -1, -1, -1]]
    assert counts.tolist() == [3, 0, 2] and token.tolist() == [7, -1, 7]


def test_a_chain_of_256(dev):
    B, T, V = 2, 256, 400
    z = _logits(dev, B * T, V, BF, 3)
    greedy = z.float().argmax(1).view(B, T)
    tokens = torch.cat([greedy[:, :1], greedy[:, :-1]], 1).contiguous()
    tokens[1, 200] += 1
    parents = torch.arange(-1, T - 1, device=dev, dtype=torch.int32)
    want = _check_tree(z, tokens, parents, torch.rand(B, T, device=dev), 0.0)
    assert want[1].tolist() == [256, 200]
    x = tokens[:, 1:].contiguous()
    assert _check_draft(z, None, x, torch.rand(B, T, device=dev), temperature=0.0)[0].tolist() == [255, 199]


def test_large_rows_and_row_offsets(dev):
    """Rows past every 32-bit offset, and a vocabulary of many chunks."""
    V, R = 1_000_003, 2200
    z = torch.full((R, V), -30.0, device=dev, dtype=BF)
    assert z.numel() * 2 > 2 ** 32
    z[-3:] = _logits(dev, 3, V, BF, 1)
    tokens, u = torch.zeros(R, 1, device=dev, dtype=I64), torch.rand(R, 1, device=dev)
    parents = torch.full((1,), -1, device=dev, dtype=torch.int32)
    token = K.verify_tree(z, tokens, parents, u)[2].cpu()
    for r in (0, 1, R - 3, R - 2, R - 1):
        assert int(token[r]) == _draw(_distribution(z[r], 1.0), float(u[r, 0])), r
    x = torch.zeros(R // 2, 1, device=dev, dtype=I64)
    uu = u.view(R // 2, 2)
    accepted, token = K.verify_draft(z, None, x, uu)
    b = R // 2 - 1
    want = _draft(z[2 * b:], None, x[b:].cpu(), uu[b:].cpu(), None, 1.0)
    assert int(accepted[b]) == int(want[0][0]) and int(token[b]) == int(want[1][0])


def test_many_sequences(dev):
    """More sequences than CUs, a few columns."""
    B, L, V = 3000, 2, 40
    z, y, x, u = _drafted(dev, B, L, V, F32, 21)
    got = K.verify_draft(z, y, x, u)
    pick = list(range(0, B, 97))
    rows = torch.cat([torch.arange(b * 3, b * 3 + 3) for b in pick])
    drafts = torch.cat([torch.arange(b * 2, b * 2 + 2) for b in pick])
    want = _draft(z[rows.to(dev)], y[drafts.to(dev)], x[pick].cpu(), u[pick].cpu(), None, 1.0)
    assert torch.equal(got[0][pick].cpu(), want[0]) and torch.equal(got[1][pick].cpu(), want[1])


def test_nothing_to_do(dev):
    z = torch.zeros(0, 50, device=dev)
    a, t = K.verify_draft(z, None, torch.zeros(0, 3, device=dev, dtype=I64), torch.zeros(0, 4, device=dev))
    n, c, s = K.verify_tree(z, torch.zeros(0, 3, device=dev, dtype=I64), torch.zeros(0, 3, device=dev, dtype=torch.int32),
                            torch.zeros(0, 3, device=dev))
    assert a.shape == t.shape == c.shape == s.shape == (0,) and n.shape == (0, 3)


def test_captured_and_replayed(dev):
    """Both in one graph, replayed over new logits, tokens, random numbers and temperatures, eager work between the replays, each
    replay against the eager calls on another stream."""
    B, L, V = 3, 6, 9001
    z, y, x, u = _drafted(dev, B, L, V, BF, 30)
    parents = torch.arange(-1, L, device=dev, dtype=torch.int32)
    temps, counts = torch.ones(B, device=dev), torch.tensor([6, 2, 5], device=dev)
    tokens = torch.cat([x[:, :1], x], 1).contiguous()

    def work():
        return [*K.verify_draft(z, y, x, u, counts=counts, temperature=temps), *K.verify_tree(z, tokens, parents, u, temperature=temps)]

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    stream = torch.cuda.Stream()
    for i in range(4):
        new = _drafted(dev, B, L, V, BF, 31 + i)
        for t, s in zip((z, y, x, u), new):
            t.copy_(s)
        tokens.copy_(torch.cat([x[:, :1], x], 1))
        temps.copy_(torch.tensor([1.0, 0.4 * i, 0.0]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            eager = work()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        want = [*_draft(z, y, x.cpu(), u.cpu(), counts, temps), *_tree(z, tokens.cpu(), parents.cpu(), u.cpu(), temps)]
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
        torch.randn(4096, device=dev).sum().item()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,skip", [(1, 3), (9, 1), (511, 0), (513, 3), (1100, 5), (2047, 7), (2050, 1), (2560, 2), (5003, 1)])
def test_every_token_of_flat_rows(dev, dtype, V, skip):
    """Rows of equal logits at any alignment: u in the middle of token j's share draws j, from p and from what a refused token leaves."""
    B = min(V, 1300)
    z = torch.full((B, V + 9), 2.0, device=dev).to(dtype)[:, skip:skip + V]
    j = (torch.arange(B, device=dev) * V) // B
    u = ((j + 0.5) / V).float()[:, None]
    parents = torch.full((B, 1), -1, device=dev, dtype=torch.int32)
    assert torch.equal(K.verify_tree(z, torch.zeros(B, 1, device=dev, dtype=I64), parents, u)[2], j)
    assert torch.equal(K.verify_draft(z, None, torch.zeros(B, 0, device=dev, dtype=I64), u)[1], j)
    if V == 1:
        return
    x = (j * 7 + 3) % V                                  # refused (u = 1 > p), then token i of the V - 1 others
    i = (torch.arange(B, device=dev) * (V - 1)) // B
    both = torch.stack([torch.ones(B, device=dev), (i + 0.5) / (V - 1)], 1).float()
    z2 = torch.full((2 * B, V + 9), 2.0, device=dev).to(dtype)[:, skip:skip + V]
    accepted, token = K.verify_draft(z2, None, x[:, None], both)
    assert not accepted.any() and torch.equal(token, i + (i >= x))
    y = torch.where(torch.arange(V, device=dev) == x[:, None], 2.0, -math.inf).to(dtype)   # the same by a drafter that was certain
    accepted, token = K.verify_draft(z2, y, x[:, None], both)
    assert not accepted.any() and torch.equal(token, i + (i >= x))


def test_two_streams_at_once(dev):
    z, y, x, u = _drafted(dev, 4, 15, 40000, BF, 3)
    parents = torch.arange(-1, 15, device=dev, dtype=torch.int32)
    nodes = torch.cat([x.new_zeros(4, 1), x], 1)
    want = (*K.verify_draft(z, y, x, u), *K.verify_tree(z, nodes, parents, u))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((*K.verify_draft(z, y, x, u), *K.verify_tree(z, nodes, parents, u)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_outputs_depend_on_the_operands_alone(dev):
    """A sequence's tokens do not change with the sequences beside it, nor with the number of rows."""
    z, y, x, u = _drafted(dev, 6, 20, 3000, F32, 5)
    accepted, token = K.verify_draft(z, y, x, u)
    parents = torch.arange(-1, 20, device=dev, dtype=torch.int32)
    nodes = torch.cat([x.new_zeros(6, 1), x], 1)
    tree = K.verify_tree(z, nodes, parents, u)
    for b in range(6):
        own = slice(b * 21, (b + 1) * 21)
        one = K.verify_draft(z[own], y[b * 20:(b + 1) * 20], x[b:b + 1], u[b:b + 1])
        assert one[0] == accepted[b] and one[1] == token[b]
        assert all(torch.equal(a[0], t[b]) for a, t in zip(K.verify_tree(z[own], nodes[b:b + 1], parents, u[b:b + 1]), tree))


def test_single_nodes_that_are_padding(dev):
    z, _, x, u = _drafted(dev, 4, 1, 700, BF, 31)
    parents = torch.tensor([[-1], [-2], [-1], [-5]], device=dev, dtype=torch.int32)
    nodes, counts, _ = _check_tree(z[:4], x, parents, u[:, :1].contiguous())
    assert counts.tolist() == [1, 0, 1, 0] and nodes.tolist() == [[0], [-1], [0], [-1]]


def test_a_tree_s_tokens_are_distributed_as_the_target_says(dev):
    """60000 trees of a root and one child over six columns: the token drawn at the root, whether the child holds it or not, and the
    token drawn at the child where it does, have the target's frequencies; counts within six deviations."""
    B, V, held = 60000, 6, 2
    g = torch.Generator(device=dev).manual_seed(6)
    p, r = torch.tensor([0.3, 0.25, 0.2, 0.15, 0.08, 0.02]), torch.tensor([0.05, 0.1, 0.5, 0.3, 0.03, 0.02])
    z = torch.stack([p.log(), r.log()]).to(dev).repeat(B, 1)
    tokens = torch.full((B, 2), held, device=dev)
    parents = torch.tensor([-1, 0], device=dev, dtype=torch.int32)
    nodes, counts, token = K.verify_tree(z, tokens, parents, torch.rand(B, 2, device=dev, generator=g))
    down = counts == 2
    assert bool((counts >= 1).all()) and not nodes[:, 0].any() and torch.equal(nodes[:, 1], torch.where(down, 1, -1))
    for a, b in ((torch.where(down, held, token), p), (token[down], r)):
        n = a.numel()
        off = (torch.bincount(a, minlength=V).cpu().double() - n * b).abs()
        assert bool((off <= 6 * (n * b * (1 - b)).sqrt()).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 16, 17, 37, 130])
def test_trees_at_temperatures_of_each_sequence(dev, dtype, T):
    """Greedy, warm and hot sequences side by side, rows drawn alone and in workgroups of eight; infinity as every finite logit alike."""
    print(f"[walk temperatures] {dtype} T={T}", flush=True)
    temps = torch.tensor([0.0, 0.7, 1.0, 3.0, -1.0, math.inf, 0.05])
    B, V = len(temps), 3001
    g = torch.Generator().manual_seed(100 + T)
    z = _logits(dev, B * T, V, dtype, 40 + T, 3)
    parents = torch.full((B, T), -1, dtype=torch.int32)
    for t in range(1, T):
        parents[:, t] = torch.randint(max(0, t - 4), t, (B,), generator=g).int()
    top = torch.topk(z.float(), 3, dim=1).indices.view(B, T, 3).cpu()
    pick = torch.randint(0, 3, (B, T), generator=g)
    tokens = torch.stack([top[b, parents[b].long().clamp(min=0), pick[b]] for b in range(B)]).to(dev)
    u = torch.rand(B, T, generator=g)
    got = K.verify_tree(z, tokens, parents.to(dev), u.to(dev), temperature=temps.to(dev))
    want = _tree(z, tokens.cpu(), parents, u, torch.where(temps.isinf(), 1e30, temps))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b), (a.tolist(), b.tolist())
