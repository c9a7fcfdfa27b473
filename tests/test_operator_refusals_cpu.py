"""That the tree, cache, top-k and distillation operators refuse an operand for its own reason: with operands that pass for device
tensors, so that no later check of the device hides a missing one, and by the message. (No GPU: every call ends in the
checks, or where it should pass them, at the launch.)"""
import re

import pytest
import torch

from uno_amd import _native as N
from uno_amd import kernels as K
from uno_amd.adapter import LoraState
from uno_amd.inference import BlockDecoder
from uno_amd.model import UnoQwen3Config, UnoQwen3ForCausalLM
from uno_amd.objectives import top_k_distillation_loss
from uno_amd.training.losses import token_normalized_top_k_distillation

BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
B, T, NQ, NK, D, LEN = 2, 5, 4, 2, 64, 16


class Launched(Exception):
    pass


@pytest.fixture
def launches(monkeypatch):
    """Launches raise; the operands' device is checked as it is."""
    if not N.LIB_PATH.exists():
        pytest.skip("libunok.so not built")

    def call(name, *args):
        raise Launched(name)
    monkeypatch.setattr(N, "call", call)
    monkeypatch.setattr(N, "stream", lambda: 0)


@pytest.fixture
def device(launches, monkeypatch):
    """Every tensor passes for one of the current device."""
    monkeypatch.setattr(K, "_same_device", lambda *a: None)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))


def z(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


def i64(*shape):
    return z(*shape, dtype=I64)


def i32(*shape):
    return z(*shape, dtype=I32)


def bf(*shape):
    return z(*shape, dtype=BF)


def caches(n=2, batch=B, length=LEN, dtype=BF, heads=NK, d=D):
    return [z(batch, heads, length, d, dtype=dtype) for _ in range(n)]


def tree(**over):
    a = dict(q=bf(B * T, NQ * D), k=bf(B, NK, LEN, D), v=bf(B, NK, LEN, D), lengths=i64(B), parents=i32(B, T))
    out = over.pop("out", None)
    a.update(over)
    return K.tree_attn(*a.values(), out=out)


def prep(**over):
    a = dict(qkv=bf(B * T, (NQ + 2 * NK) * D), wq=bf(D), wk=bf(D), lengths=i64(B), depths=i32(B, T), inv=z(D // 2), eps=1e-6,
             kc=bf(B, NK, LEN, D), vc=bf(B, NK, LEN, D))
    a.update(over)
    return K.tree_prep(*a.values(), B, T, NQ, NK, D)


def keep(c=None, lengths=None, nodes=None, counts=None):
    K.cache_keep(caches() if c is None else c, i64(B) if lengths is None else lengths, i64(B, 3) if nodes is None else nodes,
                 i64(B) if counts is None else counts)


def copy(src=None, dst=None, sl=None, dl=None, pairs=((0, 1),)):
    K.cache_copy(caches() if src is None else src, caches() if dst is None else dst, i64(B) if sl is None else sl,
                 i64(B) if dl is None else dl, pairs)


def distill(s=None, v=None, i=None, **kw):
    return token_normalized_top_k_distillation(z(4, 8) if s is None else s, z(4, 2) if v is None else v,
                                               i64(4, 2) if i is None else i, 4, **kw)


def head(v=None, i=None, n=None, **kw):
    return top_k_distillation_loss(None, z(4, 8), z(4, 2) if v is None else v, i64(4, 2) if i is None else i,
                                   torch.ones(1) if n is None else n, **kw)


KV, Q, LENGTHS, PARENTS = "k and v must be [B, nk, max_len, D]", "q must be [", "must be contiguous int64", "parents must be int32"
MATCH = "top-k distillation: teacher values and indices"
CASES = {
    "tree q 3-d": (lambda: tree(q=bf(B, T, NQ * D)), "q must be 2-D"),
    "tree q rows": (lambda: tree(q=bf(B * T + 1, NQ * D)), Q),
    "tree q heads": (lambda: tree(q=bf(B * T, 3 * D)), Q),
    "tree q width": (lambda: tree(q=bf(B * T, NQ * D + 8)), Q),
    "tree q columns": (lambda: tree(q=bf(NQ * D, B * T).t()), "q must have unit stride"),
    "tree q type": (lambda: tree(q=z(B * T, NQ * D)), KV),
    "tree k 3-d": (lambda: tree(k=bf(B, NK, D)), KV),
    "tree v shape": (lambda: tree(v=bf(B, NK, LEN + 1, D)), KV),
    "tree v type": (lambda: tree(v=z(B, NK, LEN, D)), KV),
    "tree k layout": (lambda: tree(k=bf(B, NK, D, LEN).transpose(2, 3)), "unit stride along their last"),
    "tree lengths type": (lambda: tree(lengths=i32(B)), LENGTHS),
    "tree lengths shape": (lambda: tree(lengths=i64(B + 1)), LENGTHS),
    "tree lengths layout": (lambda: tree(lengths=i64(2 * B)[::2]), LENGTHS),
    "tree parents type": (lambda: tree(parents=i64(B, T)), PARENTS),
    "tree parents batch": (lambda: tree(parents=i32(B + 1, T)), PARENTS),
    "tree parents 3-d": (lambda: tree(parents=i32(1, B, T)), PARENTS),
    "tree parents layout": (lambda: tree(parents=i32(T, B).t()), PARENTS),
    "tree out shape": (lambda: tree(out=bf(B * T, NQ * D - D)), "out must have the shape and dtype"),
    "tree out type": (lambda: tree(out=z(B * T, NQ * D)), "out must have the shape and dtype"),
    "tree out columns": (lambda: tree(out=bf(NQ * D, B * T).t()), "out must have unit stride"),
    "depths type": (lambda: K.tree_depths(i64(B, T)), "contiguous int32 parents"),
    "depths shape": (lambda: K.tree_depths(i32(T)), "contiguous int32 parents"),
    "depths layout": (lambda: K.tree_depths(i32(T, B).t()), "contiguous int32 parents"),
    "prep type": (lambda: prep(qkv=z(B * T, (NQ + 2 * NK) * D)), "bf16 qkv"),
    "prep width": (lambda: prep(qkv=bf(B * T, NQ * D)), "bf16 qkv"),
    "prep rows": (lambda: prep(qkv=bf(B * T - 1, (NQ + 2 * NK) * D)), "bf16 qkv"),
    "prep lengths": (lambda: prep(lengths=i32(B)), LENGTHS),
    "prep depths type": (lambda: prep(depths=i64(B, T)), "contiguous int32 depths"),
    "prep depths shape": (lambda: prep(depths=i32(B, T + 1)), "contiguous int32 depths"),
    "prep depths layout": (lambda: prep(depths=i32(T, B).t()), "contiguous int32 depths"),
    "prep caches' shape": (lambda: prep(vc=bf(B, NK, LEN + 1, D)), "caches must be contiguous"),
    "prep caches' heads": (lambda: prep(kc=bf(B, 1, LEN, D), vc=bf(B, 1, LEN, D)), "bf16 caches"),
    "prep caches' type": (lambda: prep(kc=z(B, NK, LEN, D), vc=z(B, NK, LEN, D)), "bf16 caches"),
    "prep norm length": (lambda: prep(wq=bf(D // 2)), "norm weights"),
    "prep norm type": (lambda: prep(wk=z(D)), "norm weights"),
    "prep frequencies": (lambda: prep(inv=z(D)), "fp32 inv_freq"),
    "keep nothing": (lambda: keep([]), "no cache tensors"),
    "keep shapes": (lambda: keep(caches() + caches(length=LEN + 1)), "caches must be contiguous"),
    "keep types": (lambda: keep(caches() + caches(dtype=F32)), "caches must be contiguous"),
    "keep layout": (lambda: keep([c.transpose(1, 2) for c in caches()]), "caches must be contiguous"),
    "keep 3-d": (lambda: keep([c[0] for c in caches()]), "caches must be [B, nk, max_len, D]"),
    "keep lengths type": (lambda: keep(lengths=i32(B)), "lengths " + LENGTHS),
    "keep lengths shape": (lambda: keep(lengths=i64(B + 1)), "lengths " + LENGTHS),
    "keep nodes type": (lambda: keep(nodes=i32(B, 3)), "nodes " + LENGTHS),
    "keep nodes batch": (lambda: keep(nodes=i64(B + 1, 3)), "nodes " + LENGTHS),
    "keep nodes layout": (lambda: keep(nodes=i64(3, B).t()), "nodes " + LENGTHS),
    "keep counts shape": (lambda: keep(counts=i64(B + 1)), "counts " + LENGTHS),
    "keep counts type": (lambda: keep(counts=i32(B)), "counts " + LENGTHS),
    "copy numbers": (lambda: copy(dst=caches(3)), "do not match"),
    "copy heads": (lambda: copy(dst=caches(heads=1)), "do not match"),
    "copy widths": (lambda: copy(dst=caches(d=128)), "do not match"),
    "copy types": (lambda: copy(dst=caches(dtype=F32)), "do not match"),
    "copy layout": (lambda: copy(src=[c.transpose(1, 2) for c in caches()]), "caches must be contiguous"),
    "copy source lengths": (lambda: copy(sl=i64(B + 1)), "source lengths " + LENGTHS),
    "copy source lengths' type": (lambda: copy(sl=i32(B)), "source lengths " + LENGTHS),
    "copy destination lengths": (lambda: copy(dst=caches(batch=4)), "destination lengths " + LENGTHS),
    "copy destination lengths' type": (lambda: copy(dl=i32(B)), "destination lengths " + LENGTHS),
    "top k 1-d": (lambda: K.row_top_k(z(8), 1), "z must be 2-D"),
    "top k columns": (lambda: K.row_top_k(z(8, 4).t(), 1), "z must have unit stride"),
    "distill rows": (lambda: distill(v=z(3, 2), i=i64(3, 2)), MATCH),
    "distill shapes": (lambda: distill(i=i64(4, 3)), MATCH),
    "distill index type": (lambda: distill(i=i32(4, 2)), "teacher indices must be int64"),
    "distill value type": (lambda: distill(v=i64(4, 2)), "teacher values must be floating-point"),
    "distill devices": (lambda: distill(v=torch.empty(4, 2, device="meta")), "teacher on meta, student on cpu"),
    "distill head rows": (lambda: head(v=z(3, 2), i=i64(3, 2)), MATCH),
    "distill head index type": (lambda: head(i=i32(4, 2)), "teacher indices must be int64"),
    "distill head inv_n type": (lambda: head(n=torch.ones(1).double()), "inv_n must be one fp32 number"),
    "distill head inv_n size": (lambda: head(n=torch.ones(2)), "inv_n must be one fp32 number"),
}


@pytest.mark.parametrize("what", CASES)
def test_refused_for_its_reason(device, what):
    call, message = CASES[what]
    with pytest.raises(RuntimeError, match=re.escape(message)):
        call()


VALID = {"tree": (tree, "unok_tree_attn"), "tree out": (lambda: tree(out=bf(B * T, NQ * D)), "unok_tree_attn"),
         "one tree": (lambda: tree(parents=i32(T)), "unok_tree_attn"), "depths": (lambda: K.tree_depths(i32(B, T)), "unok_tree_depths"),
         "prep": (prep, "unok_tree_prep"), "prep plain": (lambda: prep(wq=None, wk=None), "unok_tree_prep"),
         "keep": (keep, "unok_cache_keep"), "copy": (copy, "unok_cache_copy"),
         "top k": (lambda: K.row_top_k(z(4, 8), 8), "unok_row_topk"), "distill": (distill, "unok_distill_fwd"),
         "distill temperature": (lambda: distill(temperature=0.3), "unok_distill_fwd")}


@pytest.mark.parametrize("what", VALID)
def test_valid_operands_reach_the_launch(device, what):
    """What the refusals above differ from in one thing."""
    call, entry = VALID[what]
    with pytest.raises(Launched, match=entry):
        call()


@pytest.mark.parametrize("what", VALID)
def test_operands_in_host_memory_are_refused(launches, what):
    with pytest.raises(RuntimeError, match="current device|device tensor"):
        VALID[what][0]()


def _decoder():
    cfg = UnoQwen3Config(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                         num_key_value_heads=1, head_dim=64, block_size=4)
    model = UnoQwen3ForCausalLM(cfg, device="cpu", dtype=BF)
    model.model._uno_lora = LoraState(cfg, 8, 16.0, "cpu", BF)
    return BlockDecoder(model)


def test_tree_blocks_are_refused_for_their_reason(device):
    dec = _decoder()
    cache = dec.new_cache(B, LEN)
    ids, par = i64(B, T), i32(B, T)
    for bad, message in ((lambda: dec.tree_block(cache, i64(B + 1, T), par), "tree batch"),
                         (lambda: dec.tree_block(cache, ids, par.long()), "parents must be int32"),
                         (lambda: dec.tree_block(cache, ids, par[:, :-1]), "parents must be int32"),
                         (lambda: dec.tree_block(cache, ids, i32(B)), "parents must be int32"),
                         (lambda: dec.tree_block(cache, ids, par, torch.ones(B, T + 1, dtype=torch.bool)), "LoRA row mask"),
                         (lambda: dec.tree_block(cache, i64(B, LEN + 1), i32(B, LEN + 1)), "does not fit"),
                         (lambda: cache.accept(i32(B, 3), i64(B)), "nodes must be contiguous int64"),
                         (lambda: cache.accept(i64(B, 3), i32(B)), "counts must be contiguous int64"),
                         (lambda: cache.accept(i64(B, 257), i64(B)), "at most 256 nodes")):
        with pytest.raises(RuntimeError, match=message):
            bad()
    assert cache.lengths.tolist() == [0, 0] and cache.moves == 0
    with pytest.raises(Launched, match="unok_tree_depths"):
        dec.tree_block(cache, ids, par)
