"""What the tree, cache, top-k and distillation operators refuse, and that they do so before any kernel is launched: the
Python entry points with tensors of the wrong type, shape, layout or device, and the C entry points with sizes, strides,
pointers and workspaces they do not take. (No GPU: every call ends in the checks.)"""
import ctypes

import pytest
import torch

from uno_amd import _native as N
from uno_amd import kernels as K
from uno_amd.inference import BlockDecoder
from uno_amd.adapter import LoraState
from uno_amd.model import UnoQwen3Config, UnoQwen3ForCausalLM
from uno_amd.objectives import top_k_distillation_loss
from uno_amd.training.losses import token_normalized_top_k_distillation

BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
B, T, NQ, NK, D, LEN = 2, 5, 4, 2, 64, 16


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    if not N.LIB_PATH.exists():
        pytest.skip("libunok.so not built")

    def call(name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(N, "call", call)


def _tree(**over):
    a = dict(q=torch.zeros(B * T, NQ * D, dtype=BF), k=torch.zeros(B, NK, LEN, D, dtype=BF),
             v=torch.zeros(B, NK, LEN, D, dtype=BF), lengths=torch.zeros(B, dtype=I64), parents=torch.zeros(B, T, dtype=I32))
    out = over.pop("out", None)
    a.update(over)
    return K.tree_attn(*a.values(), out=out)


TREE = {
    "q 3-d": dict(q=torch.zeros(B, T, NQ * D, dtype=BF)),
    "q rows": dict(q=torch.zeros(B * T + 1, NQ * D, dtype=BF)),
    "q heads": dict(q=torch.zeros(B * T, 3 * D, dtype=BF)),
    "q width": dict(q=torch.zeros(B * T, NQ * D + 8, dtype=BF)),
    "q columns": dict(q=torch.zeros(NQ * D, B * T, dtype=BF).t()),
    "q type": dict(q=torch.zeros(B * T, NQ * D)),
    "k 3-d": dict(k=torch.zeros(B, NK, D, dtype=BF)),
    "v shape": dict(v=torch.zeros(B, NK, LEN + 1, D, dtype=BF)),
    "v type": dict(v=torch.zeros(B, NK, LEN, D)),
    "k layout": dict(k=torch.zeros(B, NK, D, LEN, dtype=BF).transpose(2, 3)),
    "lengths type": dict(lengths=torch.zeros(B, dtype=I32)),
    "lengths shape": dict(lengths=torch.zeros(B + 1, dtype=I64)),
    "lengths layout": dict(lengths=torch.zeros(2 * B, dtype=I64)[::2]),
    "parents type": dict(parents=torch.zeros(B, T, dtype=I64)),
    "parents batch": dict(parents=torch.zeros(B + 1, T, dtype=I32)),
    "parents 3-d": dict(parents=torch.zeros(1, B, T, dtype=I32)),
    "parents layout": dict(parents=torch.zeros(T, B, dtype=I32).t()),
    "out shape": dict(out=torch.zeros(B * T, NQ * D - D, dtype=BF)),
    "out type": dict(out=torch.zeros(B * T, NQ * D)),
    "device": {},
}


@pytest.mark.parametrize("what", list(TREE))
def test_tree_attention_refuses(what):
    with pytest.raises(RuntimeError):
        _tree(**TREE[what])


def _cache(n=2, batch=B, length=LEN, dtype=BF, heads=NK, d=D):
    return [torch.zeros(batch, heads, length, d, dtype=dtype) for _ in range(n)]


def _nodes(*shape, dtype=I64):
    return torch.zeros(*shape, dtype=dtype)


OTHERS = {
    "depths type": lambda: K.tree_depths(_nodes(B, T)),
    "depths shape": lambda: K.tree_depths(_nodes(T, dtype=I32)),
    "depths layout": lambda: K.tree_depths(_nodes(T, B, dtype=I32).t()),
    "depths device": lambda: K.tree_depths(_nodes(B, T, dtype=I32)),
    "keep nothing": lambda: K.cache_keep([], _nodes(B), _nodes(B, 3), _nodes(B)),
    "keep shapes": lambda: K.cache_keep(_cache() + _cache(length=LEN + 1), _nodes(B), _nodes(B, 3), _nodes(B)),
    "keep types": lambda: K.cache_keep(_cache() + _cache(dtype=F32), _nodes(B), _nodes(B, 3), _nodes(B)),
    "keep layout": lambda: K.cache_keep([c.transpose(1, 2) for c in _cache()], _nodes(B), _nodes(B, 3), _nodes(B)),
    "keep 3-d": lambda: K.cache_keep([c[0] for c in _cache()], _nodes(B), _nodes(B, 3), _nodes(B)),
    "keep lengths": lambda: K.cache_keep(_cache(), _nodes(B, dtype=I32), _nodes(B, 3), _nodes(B)),
    "keep nodes type": lambda: K.cache_keep(_cache(), _nodes(B), _nodes(B, 3, dtype=I32), _nodes(B)),
    "keep nodes batch": lambda: K.cache_keep(_cache(), _nodes(B), _nodes(B + 1, 3), _nodes(B)),
    "keep nodes layout": lambda: K.cache_keep(_cache(), _nodes(B), _nodes(3, B).t(), _nodes(B)),
    "keep counts": lambda: K.cache_keep(_cache(), _nodes(B), _nodes(B, 3), _nodes(B + 1)),
    "keep device": lambda: K.cache_keep(_cache(), _nodes(B), _nodes(B, 3), _nodes(B)),
    "copy numbers": lambda: K.cache_copy(_cache(2), _cache(3), _nodes(B), _nodes(B), [(0, 1)]),
    "copy heads": lambda: K.cache_copy(_cache(), _cache(heads=1), _nodes(B), _nodes(B), [(0, 1)]),
    "copy widths": lambda: K.cache_copy(_cache(), _cache(d=128), _nodes(B), _nodes(B), [(0, 1)]),
    "copy types": lambda: K.cache_copy(_cache(), _cache(dtype=F32), _nodes(B), _nodes(B), [(0, 1)]),
    "copy source lengths": lambda: K.cache_copy(_cache(), _cache(), _nodes(B + 1), _nodes(B), [(0, 1)]),
    "copy destination lengths": lambda: K.cache_copy(_cache(), _cache(batch=4), _nodes(B), _nodes(B), [(0, 1)]),
    "copy device": lambda: K.cache_copy(_cache(), _cache(), _nodes(B), _nodes(B), [(0, 1)]),
    "top k 1-d": lambda: K.row_top_k(torch.zeros(8), 1),
    "top k columns": lambda: K.row_top_k(torch.zeros(8, 4).t(), 1),
    "top k device": lambda: K.row_top_k(torch.zeros(4, 8), 1),
    "distill rows": lambda: token_normalized_top_k_distillation(torch.zeros(4, 8), torch.zeros(3, 2), _nodes(3, 2), 4),
    "distill shapes": lambda: token_normalized_top_k_distillation(torch.zeros(4, 8), torch.zeros(4, 2), _nodes(4, 3), 4),
    "distill index type": lambda: token_normalized_top_k_distillation(torch.zeros(4, 8), torch.zeros(4, 2), _nodes(4, 2, dtype=I32), 4),
    "distill value type": lambda: token_normalized_top_k_distillation(torch.zeros(4, 8), _nodes(4, 2), _nodes(4, 2), 4),
    "distill device": lambda: token_normalized_top_k_distillation(torch.zeros(4, 8), torch.zeros(4, 2), _nodes(4, 2), 4),
    "distill inv_n": lambda: top_k_distillation_loss(None, torch.zeros(4, 8), torch.zeros(4, 2), _nodes(4, 2), torch.ones(1).double()),
    "distill hidden rows": lambda: top_k_distillation_loss(None, torch.zeros(4, 8), torch.zeros(3, 2), _nodes(3, 2), torch.ones(1)),
}


@pytest.mark.parametrize("what", list(OTHERS))
def test_operators_refuse(what):
    with pytest.raises(RuntimeError):
        OTHERS[what]()


@pytest.mark.parametrize("tau", [0.0, -1.0, float("inf"), float("nan")])
def test_distillation_refuses_temperatures(tau):
    with pytest.raises(ValueError):
        token_normalized_top_k_distillation(torch.zeros(4, 8), torch.zeros(4, 2), _nodes(4, 2), 4, temperature=tau)


def test_tree_blocks_refuse():
    cfg = UnoQwen3Config(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                         num_key_value_heads=1, head_dim=64, block_size=4)
    model = UnoQwen3ForCausalLM(cfg, device="cpu", dtype=BF)
    model.model._uno_lora = LoraState(cfg, 8, 16.0, "cpu", BF)
    dec = BlockDecoder(model)
    cache = dec.new_cache(B, LEN)
    ids, par = _nodes(B, T), _nodes(B, T, dtype=I32)
    for bad in (lambda: dec.tree_block(cache, _nodes(B + 1, T), par), lambda: dec.tree_block(cache, ids, par.long()),
                lambda: dec.tree_block(cache, ids, par[:, :-1]), lambda: dec.tree_block(cache, ids, _nodes(B, dtype=I32)),
                lambda: dec.tree_block(cache, ids, par, torch.ones(B, T + 1, dtype=torch.bool)),
                lambda: dec.tree_block(cache, _nodes(B, LEN + 1), _nodes(B, LEN + 1, dtype=I32))):
        with pytest.raises(RuntimeError):
            bad()
    for n in (0, 257):
        with pytest.raises(ValueError):
            dec.tree_block(dec.new_cache(B, 512), _nodes(B, n), _nodes(B, n, dtype=I32))
    cache.lengths[1] = LEN - T + 1
    with pytest.raises(RuntimeError, match="does not fit"):
        dec.tree_block(cache, ids, par)
    wide = dec.new_cache(B, 2 * LEN)
    wide.lengths[1] = LEN + 1
    with pytest.raises(RuntimeError, match="do not fit"):
        cache.copy_from(wide, [(1, 0)])
    cache.copy_from(wide, [])                            # nothing to do


# 64 KiB of host memory for pointers that are only ever compared
ROOM = ctypes.create_string_buffer(1 << 16)
BASE = (ctypes.addressof(ROOM) + 255) // 256 * 256


def _at(*offsets):
    return (ctypes.c_void_p * len(offsets))(*(BASE + o if o is not None else None for o in offsets))


def _ints(*v):
    return (ctypes.c_int * len(v))(*v)


def _tree_call(**over):
    a = dict(dtype=N.dtype_code(BF), B=1, T=4, nq=2, nk=1, D=64, q=BASE, ldq=128, k=BASE + 4096, kb=2048, kh=2048, kr=64,
             v=BASE + 8192, vb=2048, vh=2048, vr=64, max_len=32, lengths=BASE + 12288, parents=BASE + 12544, ldp=4, scale=1.0,
             o=BASE + 16384, ldo=128, ws=None, nws=0, stream=None)
    a.update(over)
    return a.values()


def _keep(ptrs=None, **over):
    a = dict(n=2, caches=ptrs if ptrs is not None else _at(0, 4096), row=128, B=1, nk=1, max_len=16, P=2, lengths=BASE + 16384,
             nodes=BASE + 16640, counts=BASE + 16896, stream=None)
    a.update(over)
    return a.values()


def _copy(**over):
    a = dict(n=1, src=_at(0), dst=_at(8192), row=128, nk=1, sb=2, sm=16, db=3, dm=16, sl=BASE + 16384, dl=BASE + 16640, np=1,
             pairs=_ints(0, 1), stream=None)
    a.update(over)
    return a.values()


def _topk(**over):
    a = dict(dtype=N.dtype_code(F32), R=2, V=64, k=4, z=BASE, ldz=64, values=BASE + 4096, cols=BASE + 8192, lse=BASE + 12288,
             ws=None, n=0, stream=None)
    a.update(over)
    return a.values()


def _dfwd(**over):
    a = dict(dtype=N.dtype_code(F32), R=2, V=64, k=4, z=BASE, ldz=64, t=BASE + 4096, idx=BASE + 4352, tau=1.0, inv_n=None, scale=1.0,
             stat=BASE + 8192, loss=BASE + 8448, ws=BASE + 12288, n=1 << 12, stream=None)
    a.update(over)
    return a.values()


def _dbwd(**over):
    a = dict(dtype=N.dtype_code(F32), R=2, V=64, k=4, z=BASE, ldz=64, t=BASE + 4096, idx=BASE + 4352, tau=1.0, stat=BASE + 8192,
             g=BASE + 8448, inv_n=None, scale=1.0, grad=BASE + 16384, ldg=64, stream=None)
    a.update(over)
    return a.values()


def _prep(**over):
    a = dict(B=1, T=2, nq=2, nk=1, D=64, qkv=BASE, ld=256, wq=None, wk=None, lengths=BASE + 4096, depth=BASE + 4352,
             inv=BASE + 4608, eps=1e-6, kc=BASE + 8192, vc=BASE + 12288, max_len=8, q=BASE + 16384, stream=None)
    a.update(over)
    return a.values()


C = ctypes.c_void_p
ENTRIES = [
    ("unok_tree_attn", _tree_call, [dict(dtype=7), dict(B=-1), dict(T=-1), dict(T=257), dict(nq=3, nk=2), dict(nk=0), dict(D=96),
                                    dict(max_len=0), dict(max_len=1 << 30), dict(B=1 << 20, T=256), dict(B=1 << 15, max_len=1 << 23), dict(q=None), dict(k=None),
                                    dict(lengths=None), dict(parents=None), dict(o=None), dict(kr=32), dict(vr=32),
                                    dict(kr=1 << 23), dict(ldp=3), dict(q=BASE + 2), dict(k=BASE + 8), dict(ldq=129),
                                    dict(kb=2047), dict(vh=2047), dict(kr=65), dict(ldo=130), dict(max_len=8192),
                                    dict(max_len=8192, ws=BASE, nws=64), dict(ldq=64), dict(ldo=64), dict(o=BASE),
                                    dict(o=BASE + 128), dict(ldq=256, o=BASE + 512), dict(B=2, ldo=192, o=BASE + 768)]),
    ("unok_tree_attn_workspace", lambda **o: [{**dict(dtype=1, B=1, T=4, nq=2, nk=1, D=64, max_len=8), **o}[n] for n in
                                              ("dtype", "B", "T", "nq", "nk", "D", "max_len")],
     [dict(T=257), dict(D=32), dict(nq=3, nk=2), dict(max_len=0)]),
    ("unok_tree_depths", lambda **o: [{**dict(B=1, T=4, p=BASE, d=BASE + 256, s=None), **o}[n] for n in "BTpds"],
     [dict(B=-1), dict(T=257), dict(p=None), dict(d=None)]),
    ("unok_tree_prep", _prep, [dict(B=-1), dict(nq=3, nk=2), dict(D=96), dict(qkv=None), dict(depth=None), dict(q=None),
                               dict(ld=255), dict(qkv=BASE + 2), dict(kc=BASE + 4), dict(wq=BASE + 2)]),
    ("unok_cache_keep", _keep, [dict(n=-1), dict(P=257), dict(row=24), dict(row=528), dict(row=0), dict(nk=0), dict(lengths=None),
                                dict(nodes=None), dict(counts=None), dict(caches=None), dict(ptrs=_at(0, None)),
                                dict(ptrs=_at(0, 8)), dict(ptrs=_at(0, 1024)), dict(ptrs=_at(0, 0))]),
    ("unok_cache_copy", _copy, [dict(n=-1), dict(row=24), dict(nk=0), dict(nk=1 << 16), dict(sl=None), dict(src=None), dict(dst=None),
                                dict(pairs=None), dict(src=_at(8)), dict(dst=_at(None)), dict(dst=_at(2048)),
                                dict(dst=_at(0)), dict(pairs=_ints(2, 0)), dict(pairs=_ints(0, 3)), dict(pairs=_ints(-1, 0)),
                                dict(np=2, pairs=_ints(0, 1, 1, 1)), dict(dst=_at(0), db=2, pairs=_ints(1, 1)),
                                dict(dst=_at(0), db=2, dl=BASE + 16384, np=2, pairs=_ints(0, 1, 1, 0)),
                                dict(dl=BASE + 16392), dict(n=2, src=_at(0, 4096), dst=_at(8192, 10240)),
                                dict(dl=BASE + 16384, np=2, pairs=_ints(0, 1, 1, 0))]),
    ("unok_row_topk", _topk, [dict(dtype=5), dict(R=-1), dict(ldz=63), dict(k=0), dict(k=257, V=300, ldz=300), dict(k=65), dict(z=None),
                              dict(values=None), dict(cols=None), dict(lse=None), dict(V=151936, ldz=151936),
                              dict(V=151936, ldz=151936, ws=BASE, n=8)]),
    ("unok_distill_fwd", _dfwd, [dict(dtype=5), dict(R=-1), dict(V=0), dict(ldz=63), dict(k=0), dict(k=257), dict(tau=0.0),
                                 dict(tau=float("inf")), dict(tau=float("nan")), dict(tau=1e-40), dict(z=None), dict(t=None), dict(idx=None),
                                 dict(stat=None), dict(loss=None), dict(ws=None), dict(n=4), dict(ws=BASE + 4)]),
    ("unok_distill_bwd", _dbwd, [dict(dtype=5), dict(R=-1), dict(V=0), dict(ldz=63), dict(k=0), dict(k=257), dict(tau=-1.0),
                                 dict(z=None), dict(t=None), dict(idx=None), dict(stat=None), dict(g=None), dict(grad=None),
                                 dict(ldg=63), dict(grad=BASE + 16), dict(ldg=128, grad=BASE)]),
]


@pytest.mark.parametrize("name,make,over", [(n, m, o) for n, m, os in ENTRIES for o in os],
                         ids=[f"{n[5:]}-{'-'.join(o)}-{i}" for n, _, os in ENTRIES for i, o in enumerate(os)])
def test_entry_points_refuse(name, make, over):
    lib = N.lib()
    rc = getattr(lib, name)(*make(**over))
    assert rc < 0 and rc != -100, (rc, lib.unok_last_error())
    assert name[5:].replace("_workspace", "") in lib.unok_last_error().decode()
    with pytest.raises((ValueError, RuntimeError)):
        N.check(int(rc), name)


def test_empty_calls_need_nothing():
    lib = N.lib()
    for name, args in (("unok_tree_attn", _tree_call(B=0)), ("unok_tree_attn", _tree_call(T=0)), ("unok_tree_prep", _prep(T=0)),
                       ("unok_cache_keep", _keep(P=0)), ("unok_cache_keep", _keep(n=0)), ("unok_cache_copy", _copy(np=0)),
                       ("unok_row_topk", _topk(R=0)), ("unok_distill_bwd", _dbwd(R=0))):
        assert getattr(lib, name)(*args) == 0, name


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan"), 3e38])
def test_tree_attention_refuses_scales(scale):
    lib = N.lib()
    assert lib.unok_tree_attn(*_tree_call(scale=scale)) == -1
    assert "must be finite" in lib.unok_last_error().decode()


@pytest.mark.parametrize("entry,make", [("unok_distill_fwd", _dfwd), ("unok_distill_bwd", _dbwd)])
@pytest.mark.parametrize("scale", [float("inf"), float("nan")])
def test_distillation_refuses_scales(entry, make, scale):
    """(A temperature whose square is no number of fp32 arrives as such a scale.)"""
    lib = N.lib()
    assert getattr(lib, entry)(*make(scale=scale)) == -1
    assert "must be finite" in lib.unok_last_error().decode()


@pytest.mark.parametrize("pairs", [[(2 ** 32, 1)], [(0, 2 ** 32 + 1)], [(-2 ** 32, 1)], [(0, 1, 1)], [(0,)], [(0, 1), (0,), (1, 1, 0)]])
def test_copies_refuse_pairs(monkeypatch, pairs):
    """Slots that are no 32-bit numbers (they would arrive as others), and lists that are no pairs."""
    monkeypatch.setattr(K, "_same_device", lambda *a: None)
    with pytest.raises((RuntimeError, ValueError), match="cache_copy: "):
        K.cache_copy(_cache(batch=4), _cache(batch=4), _nodes(4), _nodes(4), pairs)


@pytest.mark.parametrize("k", [0, -1, 9, 257, 2 ** 32 + 1])
def test_top_k_refuses_numbers(monkeypatch, k):
    """Before results of that size are allocated."""
    monkeypatch.setattr(K, "_same_device", lambda *a: None)
    monkeypatch.setattr(K, "_rowmajor", lambda *a: None)
    with pytest.raises(ValueError, match="row_top_k: k="):
        K.row_top_k(torch.zeros(2, 8 if k < 257 else 300), k)


META = dict(device="meta")


@pytest.mark.parametrize("call", [
    lambda: K.row_top_k(torch.empty(1, 2 ** 32 + 5, **META), 2), lambda: K.row_top_k(torch.empty(2 ** 32 + 5, 4, **META), 2),
    lambda: token_normalized_top_k_distillation(torch.empty(1, 2 ** 32 + 5, **META), torch.empty(1, 2, **META),
                                                torch.empty(1, 2, dtype=I64, **META), 4),
    lambda: token_normalized_top_k_distillation(torch.empty(2 ** 32 + 5, 4, **META), torch.empty(2 ** 32 + 5, 2, **META),
                                                torch.empty(2 ** 32 + 5, 2, dtype=I64, **META), 4),
    lambda: token_normalized_top_k_distillation(torch.empty(1, 4, **META), torch.empty(1, 2 ** 32 + 5, **META),
                                                torch.empty(1, 2 ** 32 + 5, dtype=I64, **META), 4),
    lambda: K.cache_keep(_cache(), _nodes(B), torch.empty(B, 2 ** 32 + 2, dtype=I64, **META), _nodes(B))],
    ids=["top k columns", "top k rows", "distill columns", "distill rows", "distill entries", "keep nodes"])
def test_sizes_beyond_32_bits_are_refused(monkeypatch, call):
    """(They would arrive as others.)"""
    monkeypatch.setattr(K, "_same_device", lambda *a: None)
    monkeypatch.setattr(K, "_rowmajor", lambda *a: None)
    with pytest.raises((RuntimeError, ValueError), match="at most|exceed"):
        call()
