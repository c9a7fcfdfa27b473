"""Whether a captured draft block still fits the cache after the cache's lengths moved: by accepts and copies, eager or replayed
from a graph, by other blocks over the same cache. (No GPU: graphs and kernels are replaced by what they do to the lengths.)"""
import pytest
import torch

from uno_amd import inference
from uno_amd import kernels as K
from uno_amd.adapter import LoraState
from uno_amd.inference import BlockDecoder, DraftGraph
from uno_amd.model import UnoQwen3Config, UnoQwen3ForCausalLM

B, L, LEN = 2, 4, 32


def _decoder():
    cfg = UnoQwen3Config(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2,
                         num_key_value_heads=1, head_dim=64, block_size=L)
    model = UnoQwen3ForCausalLM(cfg, device="cpu", dtype=torch.float32)
    model.model._uno_lora = LoraState(cfg, 8, 16.0, "cpu", torch.float32)
    return BlockDecoder(model)


class _Graph:
    """What a captured draft block does to the lengths."""

    def __init__(self, cache, commit):
        self.cache, self.commit = cache, commit

    def replay(self):
        assert int(self.cache.lengths.max()) + L <= self.cache.max_len, "a block past the cache's end was replayed"
        self.cache.lengths += self.commit


def _draft(cache, commit):
    d = DraftGraph.__new__(DraftGraph)
    d.cache, d.block_size, d.commit = cache, L, commit
    d.ids, d.gate = torch.zeros(B, L, dtype=torch.int64), torch.ones(B, L, dtype=torch.bool)
    d._len_max, d._moves = int(cache.lengths.max()), cache.moves
    d.graph, d.logits = _Graph(cache, commit), None
    return d


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(K, "cache_keep", lambda *a: None)

    def copy(src, dst, src_lengths, dst_lengths, pairs):
        for a, b in pairs:
            dst_lengths[b] = src_lengths[a]
    monkeypatch.setattr(K, "cache_copy", copy)
    return _decoder().new_cache(B, LEN)


def _capture(monkeypatch, work, *caches):
    """Runs work() as if captured: the lengths stay as they were until the returned function replays it."""
    before = [c.lengths.clone() for c in caches]
    with monkeypatch.context() as m:
        m.setattr(inference, "_capturing", lambda: True, raising=False)
        work()
    moved = [c.lengths - b for c, b in zip(caches, before)]
    for c, b in zip(caches, before):
        c.lengths.copy_(b)

    def replay():
        for c, m in zip(caches, moved):
            c.lengths += m
    return replay


IDS = torch.zeros(B, L, dtype=torch.int64)
PATH, COUNTS = torch.arange(4).repeat(B, 1), torch.tensor([4, 2])


def test_replayed_accepts(cache, monkeypatch):
    replay = _capture(monkeypatch, lambda: cache.accept(PATH, COUNTS), cache)
    draft = _draft(cache, 0)
    for _ in range((LEN - L) // 4):
        draft.replay(IDS)
        replay()
    draft.replay(IDS)
    replay()
    with pytest.raises(RuntimeError, match="does not fit"):
        draft.replay(IDS)


def test_replayed_copies(cache, monkeypatch):
    other = _decoder().new_cache(B, LEN)
    replay = _capture(monkeypatch, lambda: cache.copy_from(other, [(1, 0)]), cache)
    del replay                                           # (its lengths are those at the replay)
    draft = _draft(cache, 0)
    draft.replay(IDS)
    other.lengths[1] = LEN - 1
    cache.lengths[0] = LEN - 1                           # what the replayed copy does
    with pytest.raises(RuntimeError, match="does not fit"):
        draft.replay(IDS)


def test_two_captured_blocks_over_one_cache(cache):
    a, b = _draft(cache, 2), _draft(cache, 2)
    for _ in range((LEN - L) // 4):
        a.replay(IDS)
        b.replay(IDS)
    a.replay(IDS)
    with pytest.raises(RuntimeError, match="does not fit"):
        b.replay(IDS)
    assert cache.lengths.tolist() == [LEN - L + 2] * 2


def test_blocks_that_commit_between_replays(cache, monkeypatch):
    """An eager draft block's commits count too."""
    dec = _decoder()
    monkeypatch.setattr(K, "embedding", lambda ids, table: torch.zeros(ids.numel(), 128))
    monkeypatch.setattr(dec, "_layer", lambda h, *a: h)
    monkeypatch.setattr(dec, "_head", lambda h, prefill: h)
    draft = _draft(cache, 0)
    for _ in range((LEN - L) // 4):
        draft.replay(IDS)
        dec.draft_block(cache, IDS, commit=4)
    draft.replay(IDS)
    dec.draft_block(cache, IDS, commit=1)
    with pytest.raises(RuntimeError, match="does not fit"):
        draft.replay(IDS)


def test_accepted_lengths_end_at_the_cache(cache):
    cache.lengths.copy_(torch.tensor([LEN - 3, LEN]))
    cache.accept(PATH, torch.tensor([99, 4]))
    assert cache.lengths.tolist() == [LEN, LEN]
    cache.accept(PATH, torch.tensor([-7, 0]))
    assert cache.lengths.tolist() == [LEN, LEN]


def test_maps_stay_in_the_cache(cache):
    """Key intervals and store rows of an fp32 block over lengths past the cache's end stay in the sequence's own slots."""
    dec = _decoder()
    cache.lengths.copy_(torch.tensor([LEN - 2, LEN + 40]))
    maps = dec._maps(cache, cache.lengths, B, L)
    iv, store = maps["iv"].view(B, 128, 8), maps["store"].view(B, L)
    for b in range(B):
        for m in (iv[b, :, 0], iv[b, :, 1] - 1, store[b]):
            assert bool(((m >= b * LEN) & (m < (b + 1) * LEN)).all())
