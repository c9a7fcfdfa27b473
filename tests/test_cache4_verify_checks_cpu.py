"""What the 4-bit caches and the verification refuse: operands in Python, each for its own reason and before anything is launched, and
arguments at the C entries. (No GPU: operands pass for device tensors, and a launch raises.)"""
import ctypes

import pytest
import torch

from uno_amd import _native as N
from uno_amd import kernels as K

BF, F32, I32, I64, U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8
B, T, NQ, NK, D, LEN, V, L = 2, 5, 4, 2, 64, 16, 50, 3


class Launched(Exception):
    pass


@pytest.fixture
def device(monkeypatch):
    if not N.LIB_PATH.exists():
        pytest.skip("libunok.so not built")

    def call(name, *args):
        raise Launched(name)
    monkeypatch.setattr(N, "call", call)
    monkeypatch.setattr(N, "stream", lambda: 0)
    monkeypatch.setattr(K, "_same_device", lambda *a: None)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))


def z(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


def c4(batch=B, heads=NK, length=LEN, d=D, groups=None, dtype=U8, sdtype=U8):
    return K.Rows4(z(batch, heads, length, d // 2, dtype=dtype), z(batch, heads, length, d // 32 if groups is None else groups, dtype=sdtype))


def store(rows=None, caches=None, starts=None):
    K.cache4_store([z(B * T, NK * D)] * 2 if rows is None else rows, [c4(), c4()] if caches is None else caches,
                   z(B, dtype=I64) if starts is None else starts)


def load(caches=None, starts=None, n=T, dtype=BF):
    K.cache4_load([c4()] if caches is None else caches, z(B, dtype=I64) if starts is None else starts, n, dtype)


def attn(**over):
    a = dict(q=z(B * T, NQ * D, dtype=BF), k=c4(), v=c4(), lengths=z(B, dtype=I64), parents=z(B, T, dtype=I32))
    out = over.pop("out", None)
    a.update(over)
    K.tree_attn4(*a.values(), out=out)


def draft(**over):
    a = dict(z=z(B * (L + 1), V), y=z(B * L, V), tokens=z(B, L, dtype=I64), u=z(B, L + 1))
    kw = {k: over.pop(k) for k in ("counts", "temperature") if k in over}
    a.update(over)
    K.verify_draft(*a.values(), **kw)


def tree(**over):
    a = dict(z=z(B * T, V), tokens=z(B, T, dtype=I64), parents=z(B, T, dtype=I32), u=z(B, T))
    kw = {k: over.pop(k) for k in ("temperature",) if k in over}
    a.update(over)
    K.verify_tree(*a.values(), **kw)


CASES = {
    "store number": (lambda: store(caches=[c4()]), "2 tensors for 1 caches"),
    "store nothing": (lambda: store([], []), "no cache tensors"),
    "store shapes": (lambda: store(caches=[c4(), c4(length=LEN + 1)]), "caches must be contiguous"),
    "store code type": (lambda: store(caches=[c4(dtype=torch.int8)] * 2), "uint8 codes"),
    "store scale type": (lambda: store(caches=[c4(sdtype=torch.int8)] * 2), "uint8 codes"),
    "store groups": (lambda: store(caches=[c4(groups=1)] * 2), "uint8 codes"),
    "store head dim": (lambda: store([z(B * T, NK * 32)] * 2, [c4(d=32)] * 2), "uint8 codes"),
    "store scale rows": (lambda: store(caches=[K.Rows4(c4().codes, c4(length=LEN + 1).scales)] * 2), "uint8 codes"),
    "store layout": (lambda: store(caches=[K.Rows4(*(t.transpose(1, 2) for t in c4()))] * 2), "caches must be contiguous"),
    "store starts": (lambda: store(starts=z(B, dtype=I32)), "starts must be contiguous int64"),
    "store width": (lambda: store([z(B * T, NK * D + 1)] * 2), "rows must be"),
    "store rows": (lambda: store([z(B * T + 1, NK * D)] * 2), "rows must be"),
    "store types": (lambda: store([z(B * T, NK * D), z(B * T, NK * D, dtype=BF)]), "rows must be"),
    "store lengths": (lambda: store([z(B * T, NK * D), z(B * T + B, NK * D)]), "rows must be"),
    "store columns": (lambda: store([z(NK * D, B * T).t()] * 2), "unit stride"),
    "store half": (lambda: store([z(B * T, NK * D, dtype=torch.float16)] * 2), "unsupported dtype"),
    "load number": (lambda: load(n=-1), "-1 rows"),
    "load type": (lambda: load(dtype=torch.float16), "unsupported dtype"),
    "load starts": (lambda: load(starts=z(B + 1, dtype=I64)), "starts must be"),
    "load size": (lambda: load(n=1 << 31), "exceed"),
    "attn k": (lambda: attn(k=c4(length=LEN + 1)), "caches must be contiguous"),
    "attn scales": (lambda: attn(v=c4(groups=4)), "caches must be contiguous|uint8 codes"),
    "attn queries": (lambda: attn(q=z(B * T, NQ * D + 8, dtype=BF)), "q must be"),
    "attn heads": (lambda: attn(q=z(B * T, 3 * D, dtype=BF)), "q must be"),
    "attn rows": (lambda: attn(q=z(B * T + 1, NQ * D, dtype=BF)), "q must be"),
    "attn half": (lambda: attn(q=z(B * T, NQ * D, dtype=torch.float16)), "unsupported dtype"),
    "attn lengths": (lambda: attn(lengths=z(B, dtype=I32)), "lengths must be"),
    "attn parents": (lambda: attn(parents=z(B, T, dtype=I64)), "parents must be"),
    "attn parents batch": (lambda: attn(parents=z(B + 1, T, dtype=I32)), "parents must be"),
    "attn out": (lambda: attn(out=z(B * T, NQ * D)), "out must have"),
    "draft tokens": (lambda: draft(tokens=z(B, L, dtype=I32)), "tokens must be"),
    "draft tokens layout": (lambda: draft(tokens=z(L, B, dtype=I64).t()), "tokens must be"),
    "draft rows": (lambda: draft(z=z(B * L, V)), "logits must be"),
    "draft no columns": (lambda: draft(z=z(B * (L + 1), 0), y=z(B * L, 0)), "logits must be"),
    "draft columns": (lambda: draft(z=z(V, B * (L + 1)).t()), "unit stride"),
    "draft half": (lambda: draft(z=z(B * (L + 1), V, dtype=torch.float16)), "unsupported dtype"),
    "draft y rows": (lambda: draft(y=z(B * L + 1, V)), "draft_logits must be"),
    "draft y columns": (lambda: draft(y=z(B * L, V + 1)), "draft_logits must be"),
    "draft y type": (lambda: draft(y=z(B * L, V, dtype=BF)), "draft_logits must be"),
    "draft u": (lambda: draft(u=z(B, L)), "u must be"),
    "draft u type": (lambda: draft(u=z(B, L + 1, dtype=torch.float64)), "u must be"),
    "draft u layout": (lambda: draft(u=z(L + 1, B).t()), "u must be"),
    "draft counts": (lambda: draft(counts=z(B, dtype=I32)), "counts must be"),
    "draft temperature": (lambda: draft(temperature=-1.0), "temperature -1.0"),
    "draft temperature nan": (lambda: draft(temperature=float("nan")), "temperature nan"),
    "draft temperature inf": (lambda: draft(temperature=float("inf")), "temperature inf"),
    "draft temperatures": (lambda: draft(temperature=z(B + 1)), "temperatures must be"),
    "draft temperatures type": (lambda: draft(temperature=z(B, dtype=BF)), "temperatures must be"),
    "tree tokens": (lambda: tree(tokens=z(B, T, dtype=I32)), "tokens must be"),
    "tree no nodes": (lambda: tree(z=z(0, V), tokens=z(B, 0, dtype=I64), parents=z(B, 0, dtype=I32), u=z(B, 0)), "tokens must be"),
    "tree parents": (lambda: tree(parents=z(B, T + 1, dtype=I32)), "parents .* do not match"),
    "tree parents type": (lambda: tree(parents=z(B, T, dtype=I64)), "parents must be"),
    "tree parents batch": (lambda: tree(parents=z(B + 1, T, dtype=I32)), "parents must be"),
    "tree rows": (lambda: tree(z=z(B * T + 1, V)), "logits must be"),
    "tree u": (lambda: tree(u=z(B, T + 1)), "u must be"),
    "tree temperatures": (lambda: tree(temperature=z(B, 1)), "temperatures must be"),
}


@pytest.mark.parametrize("what", list(CASES))
def test_operands_are_refused(device, what):
    call, text = CASES[what]
    with pytest.raises((RuntimeError, ValueError), match=text):
        call()


@pytest.mark.parametrize("call,name", [(store, "unok_cache4_store"), (load, "unok_cache4_load"), (attn, "unok_tree_attn4"),
                                       (draft, "unok_verify_draft"), (tree, "unok_verify_tree")])
def test_operands_pass(device, call, name):
    with pytest.raises(Launched, match=name):
        call()


@pytest.mark.parametrize("call,name", [(store, "cache4_store"), (load, "cache4_load"), (attn, "tree_attn4"), (draft, "verify_draft"),
                                       (tree, "verify_tree")])
def test_operands_on_the_host_are_refused(call, name):
    with pytest.raises(RuntimeError, match="device"):
        call()


def test_more_than_256_drafted_tokens(device):
    for call in (lambda: draft(z=z(2 * 258, V), y=None, tokens=z(2, 257, dtype=I64), u=z(2, 258)),
                 lambda: tree(z=z(2 * 257, V), tokens=z(2, 257, dtype=I64), parents=z(2, 257, dtype=I32), u=z(2, 257))):
        with pytest.raises(Launched):                    # (the library refuses them)
            call()
    lib = N.lib()
    assert lib.unok_verify_draft(*_draft(L=257)) == -3 and b"at most 256" in lib.unok_last_error()
    assert lib.unok_verify_tree(*_tree(T=257)) == -3 and b"at most 256" in lib.unok_last_error()


# ---- C entries: 64 KiB of host memory for pointers that are only ever compared ---------------------
ROOM = ctypes.create_string_buffer(1 << 16)
BASE = (ctypes.addressof(ROOM) + 255) // 256 * 256


def _at(*offsets):
    return (ctypes.c_void_p * len(offsets))(*(BASE + o if o is not None else None for o in offsets))


def _lds(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _move(**over):
    a = dict(dtype=0, n=2, rows=_at(0, 4096), ld=_lds(64, 64), codes=_at(8192, 12288), scales=_at(16384, 20480), B=1, T=2, nk=1, D=64,
             max_len=16, starts=BASE + 24576, stream=None)
    a.update(over)
    return a.values()


def _attn(**over):
    a = dict(dtype=1, B=1, T=4, nq=2, nk=1, D=64, q=BASE, ldq=128, k=BASE + 4096, ks=BASE + 8192, v=BASE + 12288, vs=BASE + 16384,
             max_len=32, lengths=BASE + 20480, parents=BASE + 20736, ldp=4, scale=1.0, o=BASE + 24576, ldo=128, ws=None, nws=0,
             stream=None)
    a.update(over)
    return a.values()


def _draft(**over):
    a = dict(dtype=0, B=1, L=2, V=50, z=BASE, ldz=50, y=BASE + 4096, ldy=50, tokens=BASE + 8192, counts=None, u=BASE + 8448, temp=1.0,
             temps=None, accepted=BASE + 12288, token=BASE + 12544, ws=BASE + 16384, nws=1 << 12, stream=None)
    a.update(over)
    return a.values()


def _tree(**over):
    a = dict(dtype=0, B=1, T=3, V=50, z=BASE, ldz=50, tokens=BASE + 8192, parents=BASE + 8448, ldp=3, u=BASE + 8704, temp=1.0, temps=None,
             nodes=BASE + 12288, counts=BASE + 12544, token=BASE + 12800, ws=BASE + 16384, nws=1 << 12, stream=None)
    a.update(over)
    return a.values()


MOVES = [dict(dtype=5), dict(n=-1), dict(B=-1), dict(T=-1), dict(nk=0), dict(D=32), dict(max_len=-1), dict(B=1 << 16, T=1 << 16),
         dict(B=1 << 20, T=1 << 10, nk=1 << 4), dict(nk=1 << 20), dict(rows=None), dict(ld=None), dict(codes=None), dict(scales=None),
         dict(starts=None), dict(rows=_at(0, None)), dict(codes=_at(8192, None)), dict(rows=_at(0, 4100)), dict(codes=_at(8196, 12288)),
         dict(scales=_at(16384, 20481)), dict(ld=_lds(64, 63)), dict(ld=_lds(64, 66)), dict(rows=_at(0, 8192)), dict(rows=_at(0, 16384)),
         dict(codes=_at(8192, 16384)), dict(scales=_at(16384, 8192)), dict(rows=_at(12288, 0))]
ENTRIES = [
    ("unok_cache4_store", _move, [*MOVES, dict(codes=_at(8192, 8192)), dict(codes=_at(8192, 8448)), dict(scales=_at(16384, 16384))]),
    ("unok_cache4_load", _move, [*MOVES, dict(rows=_at(0, 0)), dict(rows=_at(0, 256))]),
    ("unok_tree_attn4", _attn, [dict(dtype=7), dict(B=-1), dict(T=257), dict(nq=3, nk=2), dict(nk=0), dict(D=96), dict(max_len=0),
                                dict(max_len=1 << 30), dict(max_len=(1 << 24) + 1, ws=BASE + 65536, nws=1 << 40), dict(B=1 << 20, T=256), dict(q=None), dict(k=None), dict(ks=None), dict(v=None),
                                dict(vs=None), dict(lengths=None), dict(parents=None), dict(o=None), dict(ldp=3), dict(q=BASE + 2),
                                dict(k=BASE + 4104), dict(ks=BASE + 8194), dict(ldq=129), dict(ldo=130), dict(ldq=64), dict(ldo=64),
                                dict(o=BASE), dict(o=BASE + 128), dict(max_len=8192), dict(max_len=8192, ws=BASE, nws=64),
                                dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=3e38)]),
    ("unok_tree_attn4_workspace", lambda **o: [{**dict(dtype=1, B=1, T=4, nq=2, nk=1, D=64, max_len=8), **o}[n] for n in
                                               ("dtype", "B", "T", "nq", "nk", "D", "max_len")],
     [dict(T=257), dict(D=32), dict(nq=3, nk=2), dict(max_len=0), dict(max_len=(1 << 24) + 1)]),
    ("unok_verify_draft", _draft, [dict(dtype=5), dict(B=-1), dict(L=-1), dict(L=257), dict(V=0), dict(V=(1 << 30) + 1), dict(B=1 << 16),
                                   dict(B=60000, L=200, V=1 << 24), dict(z=None), dict(tokens=None), dict(u=None), dict(accepted=None),
                                   dict(token=None), dict(ws=None), dict(nws=8), dict(ws=BASE + 16392), dict(ldz=49), dict(ldy=49),
                                   dict(z=BASE + 2), dict(y=BASE + 4097), dict(temp=-1.0), dict(temp=float("nan")),
                                   dict(temp=float("inf")), dict(accepted=BASE + 12544), dict(accepted=BASE + 8200),
                                   dict(counts=BASE + 12288), dict(token=BASE + 8448), dict(ws=BASE + 8192), dict(ws=BASE),
                                   dict(y=BASE + 16384), dict(temps=BASE + 12292), dict(accepted=BASE + 596)]),
    ("unok_verify_tree", _tree, [dict(dtype=5), dict(B=-1), dict(T=-1), dict(T=0), dict(T=257), dict(V=0), dict(z=None), dict(tokens=None),
                                 dict(parents=None), dict(u=None), dict(nodes=None), dict(counts=None), dict(token=None), dict(ws=None),
                                 dict(nws=8), dict(ldp=2), dict(ldz=49), dict(z=BASE + 1), dict(temp=-0.5), dict(temp=float("nan")),
                                 dict(nodes=BASE + 8200), dict(nodes=BASE + 8456), dict(counts=BASE + 12304), dict(token=BASE + 8712),
                                 dict(ws=BASE + 12288), dict(nodes=BASE), dict(temps=BASE + 16388)]),
    ("unok_verify_draft_workspace", lambda **o: [{**dict(dtype=1, B=1, L=2, V=50), **o}[n] for n in ("dtype", "B", "L", "V")],
     [dict(dtype=3), dict(B=-1), dict(L=257), dict(V=0)]),
    ("unok_verify_tree_workspace", lambda **o: [{**dict(dtype=1, B=1, T=2, V=50), **o}[n] for n in ("dtype", "B", "T", "V")],
     [dict(dtype=3), dict(B=-1), dict(T=257), dict(V=0)]),
]


@pytest.mark.parametrize("name,make,over", [(n, m, o) for n, m, os in ENTRIES for o in os],
                         ids=[f"{n[5:]}-{'-'.join(o)}-{i}" for n, _, os in ENTRIES for i, o in enumerate(os)])
def test_entry_points_refuse(name, make, over):
    lib = N.lib()
    rc = getattr(lib, name)(*make(**over))
    assert -100 < rc < 0, (rc, lib.unok_last_error())
    assert name[5:].replace("_workspace", "") in lib.unok_last_error().decode()
    with pytest.raises((ValueError, RuntimeError)):
        N.check(int(rc), name)


def test_empty_calls_need_nothing():
    lib = N.lib()
    for name, args in (("unok_cache4_store", _move(n=0)), ("unok_cache4_store", _move(T=0)), ("unok_cache4_store", _move(max_len=0)),
                       ("unok_cache4_load", _move(B=0)), ("unok_tree_attn4", _attn(B=0)), ("unok_tree_attn4", _attn(T=0)),
                       ("unok_verify_draft", _draft(B=0)), ("unok_verify_tree", _tree(B=0))):
        assert getattr(lib, name)(*args) == 0, name
