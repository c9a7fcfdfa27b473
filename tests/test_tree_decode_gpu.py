"""Trees of drafted tokens through the decoder (BlockDecoder.tree_block, capture_tree), accepted paths and copied sequences
(BlockKVCache.accept, copy_from), against the oracle decoder: one pass over [committed tokens, nodes] with each node's
position and ancestors as its mask.

Bounds on the relative L2 error of a sequence's logits, 2 layers: bf16 rounds about 9 times a layer (norms, q|k|v, RoPE,
probabilities, attention, o, SwiGLU, down, residuals) and 2 times at the head, each by at most half a step, 2^-8, with a
root mean square of 2^-8 / sqrt 3 independent of each other: sqrt(20) 2^-8 / sqrt 3 = 1.0e-2, doubled for what the layers
pass on. fp32: sums of at most 1024 terms, 2^-24 sqrt(1024) sqrt(20) = 8.5e-6, and the fast exp and sincos; 1e-4."""
import pytest
import torch

from oracle.model import Cfg, decoder, init_lora, init_params
from uno_amd import kernels as K
from uno_amd.inference import BlockDecoder
from uno_amd.model import UnoQwen3Config, UnoQwen3ForCausalLM
from uno_amd.training.config import LoraSettings
from uno_amd.training.lora import create_lora_model

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
TOL = {F32: 1e-4, BF: 2e-2}
CFGS = {
    "gqa2": Cfg(4096, 256, 768, 2, 4, 2, 64, lora_rank=8, lora_alpha=16),
    "gqa4_d128": Cfg(4096, 512, 1024, 2, 4, 1, 128, lora_rank=32, lora_alpha=64),
}


def _build(dev, name, dtype):
    cfg = CFGS[name]
    params = init_params(cfg, seed=0)
    if dtype == BF:
        params = {k: v.bfloat16().float() for k, v in params.items()}
    lora = init_lora(cfg, seed=1)
    ucfg = UnoQwen3Config(vocab_size=cfg.vocab_size, hidden_size=cfg.hidden_size, intermediate_size=cfg.intermediate_size,
                          num_hidden_layers=cfg.num_hidden_layers, num_attention_heads=cfg.num_attention_heads,
                          num_key_value_heads=cfg.num_key_value_heads, head_dim=cfg.head_dim, block_size=16)
    model = UnoQwen3ForCausalLM(ucfg, device=dev, dtype=dtype)
    model.load_weights(params)
    lm, _ = create_lora_model(model, LoraSettings("all", cfg.lora_rank, cfg.lora_alpha, 0.0))
    lm.load_lora(lora)
    return cfg, params, lora, BlockDecoder(lm)


def _trees(B, T, g, padding=True):
    """Random trees: node 0 a root, every other below an earlier node; a few padding nodes."""
    p = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        for t in range(1, T):
            p[b, t] = int(torch.randint(0, t, (1,), generator=g))
            if padding and t > 2 and int(torch.randint(0, 9, (1,), generator=g)) == 0:
                p[b, t] = -2
    for b in range(B):                                   # no node below padding
        for t in range(1, T):
            if p[b, t] >= 0 and p[b, p[b, t]] == -2:
                p[b, t] = 0
    return p


def _chain(parents, t):
    path = []
    while t >= 0:
        path.append(t)
        t = int(parents[t])
    return path[::-1]


def _oracle(params, lora, cfg, history, nodes, parents, gate):
    n, T = history.numel(), nodes.numel()
    ids = torch.cat([history, nodes])[None]
    mask = torch.tril(torch.ones(n + T, n + T)).bool()
    mask[n:, n:] = False
    pos = torch.arange(n + T)
    for t in range(T):
        if parents[t] < -1:
            mask[n + t, n + t] = True
            continue
        path = _chain(parents, t)
        mask[n + t, [n + i for i in path]] = True
        pos[n + t] = n + len(path) - 1
    h = decoder(params, lora, cfg, ids, pos[None], mask[None], torch.cat([torch.zeros(n), gate])[None])
    return (h[0] @ params["lm_head.weight"].T)[n:]


def _check(got, params, lora, cfg, history, nodes, parents, gate, tol):
    ref = _oracle(params, lora, cfg, history, nodes, parents, gate)
    live = parents >= -1
    rel = ((got.float().cpu() - ref)[live].norm() / ref[live].norm()).item()
    assert rel < tol, rel


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("T", [1, 13, 60, 200])
def test_tree_block_accept_and_next(dev, name, dtype, T):
    print(f"[tree block] {name} {dtype} T={T}", flush=True)
    cfg, params, lora, dec = _build(dev, name, dtype)
    g = torch.Generator().manual_seed(T)
    B, P, cap = 3, 40, 320
    prompt = torch.randint(0, cfg.vocab_size - 1, (B, P), generator=g)
    cache = dec.new_cache(B, cap)
    dec.prefill(cache, prompt.to(dev))
    kept = [P, 17, 31]
    cache.lengths.copy_(torch.tensor(kept))
    history = [prompt[b, :n] for b, n in enumerate(kept)]
    for step in range(2):
        nodes = torch.randint(0, cfg.vocab_size - 1, (B, T), generator=g)
        parents = _trees(B, T, g)
        gate = (torch.rand(B, T, generator=g) < 0.5) if step else None
        got = dec.tree_block(cache, nodes.to(dev), parents.to(dev), None if gate is None else gate.to(dev))
        assert cache.lengths.tolist() == [h.numel() for h in history]
        for b in range(B):
            row = torch.zeros(T) if gate is None else gate[b].float()
            _check(got[b], params, lora, cfg, history[b], nodes[b], parents[b], row, TOL[dtype])
        if step:
            break
        # sequence 0 keeps its deepest path, 1 nothing, 2 the path to the last node that is no padding
        live = [t for t in range(T) if parents[2, t] >= -1]
        paths = [max((_chain(parents[0], t) for t in range(T) if parents[0, t] >= -1), key=len), [], _chain(parents[2], live[-1])]
        width = max(len(p) for p in paths) + 2
        table = torch.zeros(B, width, dtype=torch.int64)
        for b, p in enumerate(paths):
            table[b, :len(p)] = torch.tensor(p, dtype=torch.int64)
            history[b] = torch.cat([history[b], nodes[b, p]])
        cache.accept(table.to(dev), torch.tensor([len(p) for p in paths], device=dev))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_chain_is_a_draft_block(dev, dtype):
    """A tree that is a chain, gated as a draft block is: the draft block's logits up to rounding, and one tree [T] for all."""
    cfg, params, lora, dec = _build(dev, "gqa4_d128", dtype)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, cfg.vocab_size - 1, (2, 30), generator=g).to(dev)
    blk = torch.randint(0, cfg.vocab_size - 1, (2, 16), generator=g).to(dev)
    gate = torch.ones(2, 16, device=dev, dtype=torch.bool)
    gate[:, 0] = False
    caches = [dec.new_cache(2, 64) for _ in range(2)]
    for c in caches:
        dec.prefill(c, prompt)
    parents = torch.arange(-1, 15, device=dev, dtype=torch.int32)
    a = dec.tree_block(caches[0], blk, parents, gate)
    b = dec.draft_block(caches[1], blk, commit=0)
    assert ((a - b).float().norm() / b.float().norm()).item() < TOL[dtype]
    assert torch.equal(a, dec.tree_block(caches[0], blk, parents.expand(2, 16), gate))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_copied_sequences(dev, dtype):
    """A prompt prefilled once and copied into the slots of another cache, and within a cache; then trees over the copies."""
    cfg, params, lora, dec = _build(dev, "gqa2", dtype)
    g = torch.Generator().manual_seed(4)
    prompt = torch.randint(0, cfg.vocab_size - 1, (2, 33), generator=g)
    one, many = dec.new_cache(2, 50), dec.new_cache(4, 64)
    dec.prefill(one, prompt.to(dev))
    one.lengths[1] = 20
    many.lengths.fill_(7)
    many.copy_from(one, [(0, 2), (1, 0), (0, 3)])
    assert many.lengths.tolist() == [20, 7, 33, 33]
    many.copy_from(many, [(0, 1)])
    assert many.lengths.tolist() == [20, 20, 33, 33]
    for a, b in zip(one.k + one.v, many.k + many.v):
        for s, d, n in ((0, 2, 33), (1, 0, 20), (0, 3, 33), (1, 1, 20)):
            assert torch.equal(a[s, :, :n], b[d, :, :n])
            assert not b[d, :, n:].any()
    nodes = torch.randint(0, cfg.vocab_size - 1, (4, 9), generator=g)
    parents = _trees(4, 9, g)
    got = dec.tree_block(many, nodes.to(dev), parents.to(dev))
    for b, (s, n) in enumerate(((1, 20), (1, 20), (0, 33), (0, 33))):
        _check(got[b], params, lora, cfg, prompt[s, :n], nodes[b], parents[b], torch.zeros(9), TOL[dtype])
    small = dec.new_cache(3, 32)
    with pytest.raises(RuntimeError, match="do not fit"):
        small.copy_from(one, [(0, 1)])
    small.copy_from(one, [(1, 1)])
    assert small.lengths.tolist() == [0, 20, 0]
    for bad in ([(2, 0)], [(0, 3)], [(0, 1), (1, 1)], [(-1, 0)]):
        with pytest.raises((RuntimeError, ValueError)):
            small.copy_from(one, bad)
    with pytest.raises((RuntimeError, ValueError)):
        many.copy_from(many, [(0, 1), (1, 2)])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T", [4, 40])
def test_captured_trees(dev, dtype, T):
    """Replays of a captured tree block, with accepts, eager work and synchronizations between them: bit for bit the eager
    logits, lengths and committed rows."""
    cfg, params, lora, dec = _build(dev, "gqa4_d128", dtype)
    g = torch.Generator().manual_seed(T)
    B, P, cap = 2, 21, 21 + 3 * 2 + T + 1
    prompt = torch.randint(0, cfg.vocab_size - 1, (B, P), generator=g).to(dev)
    eager, graphed = dec.new_cache(B, cap), dec.new_cache(B, cap)
    for c in (eager, graphed):
        dec.prefill(c, prompt)
        c.lengths[1] = 9
    tg = dec.capture_tree(graphed, T)
    for step in range(3):
        nodes = torch.randint(0, cfg.vocab_size - 1, (B, T), generator=g).to(dev)
        parents = _trees(B, T, g).to(dev)
        ref = dec.tree_block(eager, nodes, parents)
        torch.cuda.synchronize()
        got = tg.replay(nodes, parents)
        live = parents >= -1
        assert torch.equal(got[live], ref[live]), step
        last = torch.stack([torch.zeros(B, dtype=torch.int64, device=dev),
                            torch.tensor([int(live[b].nonzero()[-1]) for b in range(B)], device=dev)], 1)
        counts = torch.tensor([2 if T > 1 else 1, step % 2], device=dev)
        for c in (eager, graphed):
            c.accept(last, counts)
        torch.randn(4096, device=dev).sum().item()
    assert torch.equal(graphed.lengths, eager.lengths) and graphed.lengths.tolist() == [P + 6, 10]
    for a, b in zip(eager.k + eager.v, graphed.k + graphed.v):
        for i, n in enumerate(eager.lengths.tolist()):
            assert torch.equal(a[i, :, :n], b[i, :, :n])
    eager.lengths[0] = graphed.lengths[0] = cap - T + 1
    for call in (lambda: tg.replay(nodes, parents), lambda: dec.tree_block(eager, nodes, parents)):
        with pytest.raises(RuntimeError, match="does not fit"):
            call()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_draft_graph_follows_accepts_and_copies(dev, dtype):
    """A captured draft block between accepts and copies: the eager block's logits, and a refusal once the cache is full."""
    cfg, params, lora, dec = _build(dev, "gqa2", dtype)
    g = torch.Generator().manual_seed(6)
    B, P, L = 2, 10, 8
    prompt = torch.randint(0, cfg.vocab_size - 1, (B, P), generator=g).to(dev)
    cache = dec.new_cache(B, P + 3 * 4 + L)
    dec.prefill(cache, prompt)
    graph = dec.capture_draft(cache, L, commit=0)
    parents = torch.arange(-1, 3, device=dev, dtype=torch.int32)
    path, counts = torch.arange(4, device=dev).repeat(B, 1), torch.tensor([4, 0], device=dev)
    for step in range(4):
        blk = torch.randint(0, cfg.vocab_size - 1, (B, L), generator=g).to(dev)
        assert torch.equal(graph.replay(blk).clone(), dec.draft_block(cache, blk, commit=0)), step
        if step == 3:
            break
        dec.tree_block(cache, blk[:, :4], parents)
        cache.accept(path, counts)
    assert cache.lengths.tolist() == [P + 12, P]
    longer = dec.new_cache(1, 2 * cache.max_len)
    dec.prefill(longer, torch.randint(0, cfg.vocab_size - 1, (1, P + 13), generator=g).to(dev))
    cache.copy_from(longer, [(0, 1)])
    with pytest.raises(RuntimeError, match="does not fit"):
        graph.replay(blk)


def test_drafting_with_trees_is_greedy_decoding(dev):
    """The operators as they are used together: the top logits of the last pass become the children of the next tree, one
    pass verifies it, the longest path of the model's own choices is kept. Every token it gives is the oracle's choice
    up to the bound on the logits."""
    cfg, params, lora, dec = _build(dev, "gqa4_d128", F32)
    g = torch.Generator().manual_seed(9)
    P, width = 24, 4
    prompt = torch.randint(0, cfg.vocab_size - 1, (1, P), generator=g)
    cache, start = dec.new_cache(2, 128), dec.new_cache(1, 64)
    z = dec.prefill(start, prompt.to(dev))
    cache.copy_from(start, [(0, 0), (0, 1)])
    values, cols, _ = K.row_top_k(z[0, -1:].contiguous(), width)
    seed = cols[:, 0].repeat(2)
    guess = cols.repeat(2, 1)                            # children of the next seed: whatever was likely before
    text = [prompt[0].tolist() for _ in range(2)]
    text[0].append(int(seed[0]))
    text[1].append(int(seed[1]))
    # root, its `width` children and one child below each
    parents = torch.tensor([-1] + [0] * width + list(range(1, width + 1)), dtype=torch.int32, device=dev)
    for _ in range(6):
        nodes = torch.cat([seed[:, None], guess, guess], 1)
        z = dec.tree_block(cache, nodes, parents)
        T = nodes.shape[1]
        values, cols, _ = K.row_top_k(z.reshape(2 * T, -1), width)
        best = cols[:, 0].view(2, T).tolist()
        ids = nodes.tolist()
        table, counts = torch.zeros(2, 3, dtype=torch.int64), []
        for b in range(2):
            path = [0]
            while True:
                t = path[-1]
                child = [i for i in range(T) if int(parents[i]) == t and ids[b][i] == best[b][t]]
                if not child:
                    break
                path.append(child[0])
            table[b, :len(path)] = torch.tensor(path)
            counts.append(len(path))
            text[b] += [ids[b][i] for i in path[1:]] + [best[b][path[-1]]]
            seed[b] = best[b][path[-1]]
            guess[b] = cols.view(2, T, width)[b, path[-1]]
        cache.accept(table.to(dev), torch.tensor(counts, device=dev))
        assert cache.lengths.tolist() == [len(t) - 1 for t in text]
    assert text[0] == text[1]                            # copies of one sequence
    full = torch.tensor(text[0])
    parents_of = torch.arange(-1, len(full) - P - 1, dtype=torch.int32)
    ref = _oracle(params, lora, cfg, full[:P - 1], full[P - 1:], torch.cat([parents_of, parents_of[-1:] + 1]),
                  torch.zeros(len(full) - P + 1))
    for i, tok in enumerate(full[P:].tolist()):
        slack = 2 * TOL[F32] * ref[i].norm().item()
        assert ref[i, tok] >= ref[i].max() - slack, i


@pytest.mark.parametrize("dtype", [F32, BF])
def test_draft_graph_follows_replayed_accepts(dev, dtype):
    """Tree blocks and accepts replayed from graphs, and a captured draft block between them: the eager block's logits, and a
    refusal once the cache is full."""
    cfg, params, lora, dec = _build(dev, "gqa2", dtype)
    g = torch.Generator().manual_seed(7)
    B, P, L = 2, 10, 8
    prompt = torch.randint(0, cfg.vocab_size - 1, (B, P), generator=g).to(dev)
    cache = dec.new_cache(B, P + 3 * 4 + L)
    dec.prefill(cache, prompt)
    draft, tree = dec.capture_draft(cache, L, commit=0), dec.capture_tree(cache, 4)
    parents = torch.arange(-1, 3, device=dev, dtype=torch.int32)
    path, counts = torch.arange(4, device=dev).repeat(B, 1), torch.tensor([4, 1], device=dev)
    lengths, rows = cache.lengths.clone(), [c.clone() for c in cache.k + cache.v]
    cache.accept(path, counts)                           # once before the capture, and undone
    cache.lengths.copy_(lengths)
    for c, r in zip(cache.k + cache.v, rows):
        c.copy_(r)
    accept = torch.cuda.CUDAGraph()
    with torch.cuda.graph(accept):
        cache.accept(path, counts)
    assert cache.lengths.tolist() == [P, P]
    for step in range(4):
        blk = torch.randint(0, cfg.vocab_size - 1, (B, L), generator=g).to(dev)
        assert torch.equal(draft.replay(blk).clone(), dec.draft_block(cache, blk, commit=0)), step
        if step == 3:
            break
        tree.replay(blk[:, :4], parents)
        accept.replay()
    assert cache.lengths.tolist() == [P + 12, P + 3]
    accept.replay()
    with pytest.raises(RuntimeError, match="does not fit"):
        draft.replay(blk)
