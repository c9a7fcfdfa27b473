"""Decoding over KV caches in 4 bits (BlockDecoder.new_cache(bits=4)) and with drawn tokens (verify_tree, verify_draft), as they are
used together.

The decoder's passes are checked layer by layer against plain ones on the CPU (the oracle's norms, rotation and gated linears) that
attend over the numbers the cache holds, so that a code that rounds to its other neighbour (the layers' inputs differ by their
roundings) is no difference; the numbers of the new rows are checked against the plain pass's own keys and values: within half a step
of their groups, a seventh of the largest magnitude (2/7 at the top of the range), and the bound on the rows.
Bounds on the relative L2 error of logits as in the tests of trees over 16-bit caches: 2e-2 for bf16, 1e-4 for fp32."""
import pytest
import torch
import torch.nn.functional as F

from oracle.model import Cfg, init_lora, init_params, lora_linear, module_path, rms_norm, rope_cos_sin, rotate_half
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


def _trees(B, T, g):
    """Random trees: node 0 a root, every other below an earlier node; the last node of sequence 1 is padding."""
    p = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        for t in range(1, T):
            p[b, t] = int(torch.randint(0, t, (1,), generator=g))
    if B > 1 and T > 3:
        p[1, T - 1] = -2
    return p


def _rows(cache4, n):
    """The numbers of the first n rows of each slot, [B, nk, n, D] on the CPU."""
    B, nk, _, half = cache4.codes.shape
    zero = torch.zeros(B, device=cache4.codes.device, dtype=torch.int64)
    return K.cache4_load([cache4], zero, n, dtype=F32)[0].view(B, n, nk, 2 * half).transpose(1, 2).cpu()


def _near(numbers, rows, tol):
    """4-bit numbers of rows known up to a relative error of their size."""
    step = rows.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(*rows.shape[:-1], -1, 32).flatten(-2) * (2 / 7)
    assert bool(((numbers - rows).abs() <= step * 1.01 + 4 * tol * rows.abs().amax() + 1e-6).all())
    assert ((numbers - rows).norm() / rows.norm()).item() < 0.25


def _plain(params, lora, cfg, cache, b, n, ids, parents, gate, tol):
    """Logits [T, V] of the nodes ids [T] of sequence b over the numbers that ``cache`` holds in its rows 0 .. n + T - 1."""
    T, Hq, Hkv, d = ids.numel(), cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    seen, depth = torch.zeros(T, n + T, dtype=torch.bool), torch.zeros(T, dtype=torch.int64)
    for t in range(T):
        if parents[t] < -1:
            seen[t, n + t] = True                       # (its logits are not looked at)
            continue
        seen[t, :n] = True
        a = t
        while a >= 0:
            seen[t, n + a] = True
            a = int(parents[a])
        depth[t] = seen[t, n:].sum() - 1
    cos, sin = (x[:, None] for x in rope_cos_sin(n + depth, d, cfg.rope_theta))
    h = params["model.embed_tokens.weight"][ids]
    live = parents >= -1
    for i in range(cfg.num_hidden_layers):
        def lin(name, x):
            p = module_path(i, name)
            return lora_linear(x, params[p + ".weight"], lora[p + ".lora_A.weight"], lora[p + ".lora_B.weight"], gate, cfg.lora_scale)
        pre = f"model.layers.{i}."
        x = rms_norm(h, params[pre + "input_layernorm.weight"], cfg.rms_norm_eps)
        q, k, v = lin("q_proj", x).view(T, Hq, d), lin("k_proj", x).view(T, Hkv, d), lin("v_proj", x).view(T, Hkv, d)
        q = rms_norm(q, params[pre + "self_attn.q_norm.weight"], cfg.rms_norm_eps)
        k = rms_norm(k, params[pre + "self_attn.k_norm.weight"], cfg.rms_norm_eps)
        q, k = (y * cos + rotate_half(y) * sin for y in (q, k))
        ck, cv = (_rows(c[i], n + T)[b] for c in (cache.k, cache.v))          # [Hkv, n + T, d]
        _near(ck[:, n:].transpose(0, 1)[live], k[live], tol)
        _near(cv[:, n:].transpose(0, 1)[live], v[live], tol)
        rep = Hq // Hkv
        scores = q.transpose(0, 1) @ ck.repeat_interleave(rep, 0).transpose(1, 2).contiguous() * d ** -0.5
        a = torch.softmax(scores.masked_fill(~seen, float("-inf")), -1) @ cv.repeat_interleave(rep, 0)
        h = h + lin("o_proj", a.transpose(0, 1).reshape(T, Hq * d))
        x = rms_norm(h, params[pre + "post_attention_layernorm.weight"], cfg.rms_norm_eps)
        h = h + lin("down_proj", F.silu(lin("gate_proj", x)) * lin("up_proj", x))
    return rms_norm(h, params["model.norm.weight"], cfg.rms_norm_eps) @ params["lm_head.weight"].T


def _check(got, params, lora, cfg, cache, lengths, ids, parents, gate, tol):
    for b, n in enumerate(lengths):
        ref = _plain(params, lora, cfg, cache, b, n, ids[b].cpu(), parents[b].cpu(), gate[b].cpu().float(), tol)
        live = parents[b].cpu() >= -1
        rel = ((got[b].float().cpu() - ref)[live].norm() / ref[live].norm()).item()
        assert rel < tol, (b, rel)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", list(CFGS))
def test_prefill(dev, name, dtype):
    """The logits of the 16-bit cache, and its rows quantised."""
    cfg, _, _, dec = _build(dev, name, dtype)
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, cfg.vocab_size - 1, (3, 45), generator=g).to(dev)
    wide, cache = dec.new_cache(3, 64), dec.new_cache(3, 64, bits=4)
    assert torch.equal(dec.prefill(wide, prompt), dec.prefill(cache, prompt))
    assert cache.lengths.tolist() == [45] * 3
    zero = torch.zeros(3, device=dev, dtype=torch.int64)
    for a, b in zip(wide.k + wide.v, cache.k + cache.v):
        own = K.Rows4(torch.zeros_like(b.codes), torch.zeros_like(b.scales))
        K.cache4_store([a[:, :, :45].transpose(1, 2).reshape(3 * 45, -1).contiguous()], [own], zero)
        assert torch.equal(own.codes, b.codes) and torch.equal(own.scales, b.scales)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("T", [1, 13, 60, 200])
def test_tree_blocks_and_accepts(dev, name, dtype, T):
    print(f"[tree4 block] {name} {dtype} T={T}", flush=True)
    cfg, params, lora, dec = _build(dev, name, dtype)
    g = torch.Generator().manual_seed(T)
    B, P, cap = 3, 40, 320
    cache = dec.new_cache(B, cap, bits=4)
    dec.prefill(cache, torch.randint(0, cfg.vocab_size - 1, (B, P), generator=g).to(dev))
    cache.lengths.copy_(torch.tensor([P, 17, 31]))
    for step in range(2):
        lengths = cache.lengths.tolist()
        nodes, parents = torch.randint(0, cfg.vocab_size - 1, (B, T), generator=g), _trees(B, T, g)
        gate = (torch.rand(B, T, generator=g) < 0.5) if step else torch.zeros(B, T, dtype=torch.bool)
        got = dec.tree_block(cache, nodes.to(dev), parents.to(dev), gate.to(dev) if step else None)
        assert cache.lengths.tolist() == lengths
        _check(got, params, lora, cfg, cache, lengths, nodes, parents, gate, TOL[dtype])
        path = [T - 1]
        while path[0] > 0:
            path.insert(0, max(0, int(parents[0, path[0]])))
        table = torch.zeros(B, len(path), dtype=torch.int64)
        table[0] = torch.tensor(path)
        before = [_rows(c, cap) for c in cache.k + cache.v]
        cache.accept(table.to(dev), torch.tensor([len(path), 1, 0], device=dev))
        assert cache.lengths.tolist() == [lengths[0] + len(path), lengths[1] + 1, lengths[2]]
        for c, was in zip(cache.k + cache.v, before):
            now = _rows(c, cap)
            for i, t in enumerate(path):
                assert torch.equal(now[0, :, lengths[0] + i], was[0, :, lengths[0] + t])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name,L", [("gqa2", 16), ("gqa4_d128", 60)])
def test_draft_blocks(dev, name, dtype, L):
    """A draft block over a 4-bit cache is the chain of its rows, gated; its first rows are committed. Captured, it gives the
    eager block's logits."""
    cfg, params, lora, dec = _build(dev, name, dtype)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, cfg.vocab_size - 1, (2, 30), generator=g).to(dev)
    cache, other = (dec.new_cache(2, 400, bits=4) for _ in range(2))
    for c in (cache, other):
        dec.prefill(c, prompt)
    graph = dec.capture_draft(other, L)
    gate = torch.ones(2, L, dtype=torch.bool)
    gate[:, 0] = False
    chain = torch.arange(-1, L - 1, dtype=torch.int32).expand(2, L)
    for step in range(3):
        blk = torch.randint(0, cfg.vocab_size - 1, (2, L), generator=g)
        got = dec.draft_block(cache, blk.to(dev))
        assert cache.lengths.tolist() == [31 + step] * 2
        _check(got, params, lora, cfg, cache, [30 + step] * 2, blk, chain, gate, TOL[dtype])
        torch.cuda.synchronize()
        assert torch.equal(graph.replay(blk.to(dev)), got)
        torch.randn(4096, device=dev).sum().item()
    assert torch.equal(other.lengths, cache.lengths)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_captured_trees(dev, dtype):
    """Replays with accepts, eager work and synchronizations between them: bit for bit the eager logits and rows."""
    cfg, params, lora, dec = _build(dev, "gqa4_d128", dtype)
    T, B, P = 40, 2, 21
    g = torch.Generator().manual_seed(T)
    prompt = torch.randint(0, cfg.vocab_size - 1, (B, P), generator=g).to(dev)
    eager, graphed = (dec.new_cache(B, P + 3 * 2 + T, bits=4) for _ in range(2))
    for c in (eager, graphed):
        dec.prefill(c, prompt)
        c.lengths[1] = 9
    tg = dec.capture_tree(graphed, T)
    for step in range(3):
        nodes, parents = torch.randint(0, cfg.vocab_size - 1, (B, T), generator=g).to(dev), _trees(B, T, g).to(dev)
        ref = dec.tree_block(eager, nodes, parents)
        torch.cuda.synchronize()
        got = tg.replay(nodes, parents)
        live = parents >= -1
        assert torch.equal(got[live], ref[live]), step
        for c in (eager, graphed):
            c.accept(torch.tensor([[0, T - 2]] * B, device=dev), torch.tensor([2, step % 2], device=dev))
        torch.randn(4096, device=dev).sum().item()
    assert torch.equal(graphed.lengths, eager.lengths)
    for a, b in zip(eager.k + eager.v, graphed.k + graphed.v):
        for i, n in enumerate(eager.lengths.tolist()):
            assert torch.equal(a.codes[i, :, :n], b.codes[i, :, :n]) and torch.equal(a.scales[i, :, :n], b.scales[i, :, :n])


def test_copied_sequences(dev):
    """Sequences between 4-bit caches and within one; not between a 4-bit and a 16-bit cache."""
    cfg, _, _, dec = _build(dev, "gqa2", BF)
    g = torch.Generator().manual_seed(4)
    one, many = dec.new_cache(2, 50, bits=4), dec.new_cache(4, 64, bits=4)
    dec.prefill(one, torch.randint(0, cfg.vocab_size - 1, (2, 33), generator=g).to(dev))
    one.lengths[1] = 20
    many.lengths.fill_(7)
    many.copy_from(one, [(0, 2), (1, 0), (0, 3)])
    assert many.lengths.tolist() == [20, 7, 33, 33]
    many.copy_from(many, [(0, 1)])
    assert many.lengths.tolist() == [20, 20, 33, 33]
    for a, b in zip(one.k + one.v, many.k + many.v):
        for x, y in zip(a, b):
            for s, d, n in ((0, 2, 33), (1, 0, 20), (0, 3, 33), (1, 1, 20)):
                assert torch.equal(x[s, :, :n], y[d, :, :n]) and not y[d, :, n:].any()
    with pytest.raises(RuntimeError, match="do not fit"):
        dec.new_cache(3, 32, bits=4).copy_from(one, [(0, 1)])
    for a, b in ((many, dec.new_cache(2, 50)), (dec.new_cache(2, 50), one)):
        with pytest.raises(RuntimeError, match="do not go into"):
            a.copy_from(b, [(0, 1)])


@pytest.mark.parametrize("bits", [None, 4])
def test_verified_trees_are_the_target_s_own_tokens(dev, bits):
    """Trees from the top logits, verified, kept, and drawn on, at once for greedy and warm sequences: every token is the one that
    the plain definition draws from the pass's own logits; greedy text is what plain greedy decoding writes."""
    cfg, params, lora, dec = _build(dev, "gqa4_d128", F32)
    g = torch.Generator().manual_seed(9)
    B, P, width, steps = 3, 24, 4, 6
    prompt = torch.randint(0, cfg.vocab_size - 1, (1, P), generator=g).to(dev)
    start, cache = dec.new_cache(1, 64, bits), dec.new_cache(B, 128, bits)
    z = dec.prefill(start, prompt)
    cache.copy_from(start, [(0, b) for b in range(B)])
    temps = torch.tensor([0.0, 0.05, 1.0], device=dev)
    parents = torch.tensor([-1] + [0] * width + list(range(1, width + 1)), dtype=torch.int32, device=dev)
    _, cols, _ = K.row_top_k(z[0, -1:].contiguous(), width)
    seed, guess = cols[:, 0].repeat(B), cols.repeat(B, 1)
    text, T = [[int(s)] for s in seed], 2 * width + 1
    for _ in range(steps):
        before = cache.lengths.clone()
        nodes = torch.cat([seed[:, None], guess, guess], 1)
        u = torch.rand(B, T, generator=g).to(dev)
        logits = []
        keep = dec.tree_block
        dec.tree_block = lambda *a, **k: logits.append(keep(*a, **k)) or logits[0]
        path, counts, token = dec.verify_tree(cache, nodes, parents, u, temps)
        dec.tree_block = keep
        assert torch.equal(cache.lengths, before + counts)
        for b in range(B):
            at = 0
            for i in range(int(counts[b])):
                assert int(path[b, i]) == at
                row = logits[0][b, at].double().cpu()
                if temps[b] == 0:
                    drawn = int(row.argmax())
                else:
                    run = torch.softmax(row / float(temps[b]), 0).cumsum(0)
                    drawn = int((run > float(u[b, at]) * run[-1]).nonzero()[0])
                text[b].append(drawn)
                child = [t for t in range(at + 1, T) if int(parents[t]) == at and int(nodes[b, t]) == drawn]
                at = child[0] if child else None
            assert at is None and text[b][-1] == int(token[b])
        seed = token
        last = path.gather(1, counts[:, None] - 1)
        _, cols, _ = K.row_top_k(torch.stack([logits[0][b, int(last[b])] for b in range(B)]), width)
        guess = cols
    if bits is None:                                    # (4-bit rows of a node are the same in whatever pass they are stored)
        greedy, plain = text[0], dec.new_cache(1, 128)
        full = torch.tensor(greedy, device=dev)
        z = dec.prefill(plain, torch.cat([prompt[0], full[:-1]])[None])[0, P:]
        for i, tok in enumerate(greedy[1:]):
            assert z[i, tok] >= z[i].max() - 2 * TOL[F32] * z[i].norm()


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_verified_drafts(dev, dtype, bits):
    """Blocks drafted with the LoRA and drawn from its logits, verified without it, kept, and drafted on, with ragged blocks: the
    outcome is K.verify_draft's on the pass's logits, and the rows that stay are those of the accepted tokens."""
    cfg, params, lora, dec = _build(dev, "gqa2", dtype)
    g = torch.Generator(device=dev).manual_seed(3)
    B, P, L = 3, 20, 5
    cache = dec.new_cache(B, 96, bits)
    z = dec.prefill(cache, torch.randint(0, cfg.vocab_size - 1, (B, P), generator=g, device=dev))
    seed = z[:, -1].float().argmax(1)
    counts = torch.tensor([L, 2, 0], device=dev)
    for step in range(5):
        before = cache.lengths.clone()
        noise = torch.randint(0, cfg.vocab_size - 1, (B, L - 1), generator=g, device=dev)
        draft = dec.draft_block(cache, torch.cat([seed[:, None], noise], 1), commit=0)
        tokens = torch.multinomial(torch.softmax(draft.float().flatten(0, 1), 1), 1, generator=g).view(B, L)
        u = torch.rand(B, L + 1, generator=g, device=dev)
        block = torch.cat([seed[:, None], tokens], 1)
        chain = torch.arange(-1, L, device=dev, dtype=torch.int32)
        target = dec.tree_block(cache, block, chain)
        want = K.verify_draft(target.flatten(0, 1), draft.flatten(0, 1), tokens, u, counts=counts)
        accepted, token = dec.verify_draft(cache, block, u, draft, counts=counts)
        assert torch.equal(accepted, want[0]) and torch.equal(token, want[1])
        assert bool((accepted <= counts).all()) and torch.equal(cache.lengths, before + 1 + accepted)
        again = dec.tree_block(cache, token[:, None].contiguous(), chain[:1])   # the next token over the rows kept
        if bits is None:
            for b in range(B):
                n = int(accepted[b])
                one = dec.new_cache(1, 96)
                one.copy_from(cache, [(b, 0)])
                one.lengths.copy_(before[b:b + 1])
                whole = torch.cat([block[b, :n + 1], token[b:b + 1]])[None]
                ref = dec.tree_block(one, whole, torch.arange(-1, n + 1, device=dev, dtype=torch.int32))[0, -1]
                assert ((again[b, 0] - ref).float().norm() / ref.float().norm()).item() < TOL[dtype]
        seed = token


def test_refusals(dev):
    cfg, _, _, dec = _build(dev, "gqa2", BF)
    with pytest.raises(ValueError, match="not in 8"):
        dec.new_cache(2, 64, bits=8)
    cache = dec.new_cache(2, 300, bits=4)
    dec.prefill(cache, torch.zeros(2, 8, device=dev, dtype=torch.int64))
    with pytest.raises(NotImplementedError, match="256"):
        dec.draft_block(cache, torch.zeros(2, 257, device=dev, dtype=torch.int64))
    for n in (0, 257):
        with pytest.raises(ValueError, match="1 to 256"):
            dec.verify_draft(cache, torch.zeros(2, n, device=dev, dtype=torch.int64), torch.rand(2, max(n, 1), device=dev))
    with pytest.raises(RuntimeError, match="u must be"):
        dec.verify_draft(cache, torch.zeros(2, 4, device=dev, dtype=torch.int64), torch.rand(2, 3, device=dev))
    with pytest.raises(RuntimeError, match="does not fit"):
        dec.draft_block(dec.new_cache(2, 8, bits=4), torch.zeros(2, 9, device=dev, dtype=torch.int64))
    assert cache.lengths.tolist() == [8, 8]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", list(CFGS))
def test_rows_of_verified_drafts(dev, name, dtype):
    """What verify_draft keeps of a block in a 4-bit cache: codes and scales of the rows of the last token and the accepted ones, as a pass
    over the same block stored them, behind rows that stay as they were; and the next pass attends over them."""
    cfg, params, lora, dec = _build(dev, name, dtype)
    g = torch.Generator(device=dev).manual_seed(13)
    B, P, L = 3, 20, 6
    cache = dec.new_cache(B, 96, bits=4)
    z = dec.prefill(cache, torch.randint(0, cfg.vocab_size - 1, (B, P), generator=g, device=dev))
    cache.lengths.copy_(torch.tensor([P, 11, 16]))
    seed = z[:, -1].float().argmax(1)
    counts = torch.tensor([L, 3, 0], device=dev)
    chain = torch.arange(-1, L, device=dev, dtype=torch.int32)
    tensors = [t for c in cache.k + cache.v for t in c]
    taken = 0
    for step in range(4):
        before = cache.lengths.tolist()
        block = torch.cat([seed[:, None], torch.zeros(B, L, device=dev, dtype=torch.int64)], 1)
        for i in range(L):                              # each token the likeliest behind those before it, but some
            x = dec.tree_block(cache, block, chain)[:, i]
            block[:, i + 1] = torch.where(x == x.amax(1, keepdim=True), torch.arange(x.shape[1], device=dev), x.shape[1]).amin(1)
        block[0, 2 + step] = (block[0, 2 + step] + 1) % cfg.vocab_size
        dec.tree_block(cache, block, chain)
        want = [t.clone() for t in tensors]
        accepted, token = dec.verify_draft(cache, block, torch.rand(B, L + 1, generator=g, device=dev), None, counts, 0.0)
        assert accepted.tolist() == [1 + step, 3, 0]
        after = cache.lengths.tolist()
        assert after == [n + 1 + a for n, a in zip(before, accepted.tolist())]
        for t, w in zip(tensors, want):
            for b, n in enumerate(after):
                assert torch.equal(t[b, :, :n], w[b, :, :n])
        taken += int(accepted.sum())
        again = dec.tree_block(cache, token[:, None].contiguous(), chain[:1])
        _check(again, params, lora, cfg, cache, after, token[:, None], torch.full((B, 1), -1, dtype=torch.int32), torch.zeros(B, 1),
               TOL[dtype])
        seed = token
    assert taken == 1 + 2 + 3 + 4 + 4 * 3
