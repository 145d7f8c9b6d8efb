"""The paged cache's host side: pages, lengths and the batch description (CPU)."""
import pytest
import torch

from spruce_research_b200.paged import PagedKVCache, PagedSparseLayer


def cache(pages=6, page=16, layers=2):
    return PagedKVCache(layers, pages, page, 2, 64, torch.float32, "cpu")


def test_steps_allocate_pages_and_describe_the_batch():
    c = cache()
    s = c.step([("a", 17), ("b", 0), ("c", 16)])
    assert c.free_pages == 3 and s.seq_ids == ["a", "b", "c"] and s.tokens == 33
    assert s.cu_q.tolist() == [0, 17, 17, 33] and s.kv_lens.tolist() == [17, 0, 16]
    assert (s.max_q_len, s.max_kv_len) == (17, 17)
    assert s.block_table.shape == (3, 2) and s.block_table.dtype == s.cu_q.dtype == s.kv_lens.dtype == torch.int32
    a, cc = s.block_table[0].tolist(), s.block_table[2, 0].item()
    assert len({*a, cc}) == 3
    s = c.step([("c", 1), ("a", 15)])                      # c takes a new page, a fills its second
    assert s.block_table[0, 0].item() == cc and s.block_table[1].tolist() == a
    assert s.kv_lens.tolist() == [17, 32] and s.cu_q.tolist() == [0, 1, 16]
    assert c.free_pages == 2 and c.length("a") == 32 and c.length("nobody") == 0
    for t in (s.block_table, s.cu_q, s.kv_lens):
        assert t.stride(-1) == 1


def test_pages_return_and_nothing_changes_on_refusal():
    c = cache(pages=3)
    c.step([("a", 32)])
    with pytest.raises(RuntimeError, match="needs 2 more pages and has 1"):
        c.step([("a", 1), ("b", 1)])
    assert c.length("a") == 32 and c.length("b") == 0 and c.free_pages == 1
    c.drop("a")
    c.drop("nobody")
    assert c.free_pages == 3 and c.length("a") == 0
    s = c.step([("b", 48)])
    assert sorted(s.block_table[0].tolist()) == [0, 1, 2]
    e = c.step([])
    assert e.tokens == 0 and e.block_table.shape[0] == 0 and e.cu_q.tolist() == [0]


def test_refusals():
    for bad in (dict(page=8), dict(page=24), dict(pages=0), dict(layers=0)):
        with pytest.raises(ValueError):
            cache(**bad)
    c = cache()
    with pytest.raises(ValueError, match="twice"):
        c.step([("a", 1), ("a", 2)])
    with pytest.raises(ValueError, match="negative"):
        c.step([("a", -1)])
    with pytest.raises(ValueError, match="outside"):
        PagedSparseLayer(c, 2, torch.zeros(4, 64))
    layer = PagedSparseLayer(c, 1, torch.zeros(64, 64))
    x = torch.zeros(20, 2, 64)
    with pytest.raises(ValueError, match="without a SparsePrefillLayer"):
        layer.prefill(x, x, x, c.step([("a", 20)]))
    layer.sparse = object()
    with pytest.raises(ValueError, match="one whole prompt"):
        layer.prefill(x[:1], x[:1], x[:1], c.step([("a", 1)]))
