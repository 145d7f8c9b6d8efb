"""The operators on attention weight on the host (CPU): what they refuse, the current GPU, the cache's eviction, the C entries."""
import re

import pytest
import torch
from test_serving_host import _elsewhere, fake_gpus  # noqa: F401

from spruce_research_b200 import _lib, native
from spruce_research_b200.paged import PagedKVCache, PagedSparseLayer
from spruce_research_b200.selector.gate import FlatGate
from spruce_research_b200.selector.loss import teacher_top_blocks, topk_distill_loss
from spruce_research_b200.selector.train import gate_loss, gate_training_scores

I32 = torch.int32


def _mass_args(**change):
    """q, k_cache, mass, block_table, cu_q, kv_lens, lse on another GPU."""
    a = dict(q=_elsewhere(3, 4, 64), k=_elsewhere(4, 2, 16, 64), mass=_elsewhere(4, 2, 16),
             table=_elsewhere(1, 2, dtype=I32), cu=_elsewhere(2, dtype=I32), kv=_elsewhere(1, dtype=I32), lse=_elsewhere(3, 4))
    return tuple((a | change).values())


def _evict_args(**change):
    a = dict(k=_elsewhere(4, 2, 16, 64), v=_elsewhere(4, 2, 16, 64), mass=_elsewhere(4, 2, 16),
             table=_elsewhere(1, 2, dtype=I32), kv=_elsewhere(1, dtype=I32))
    return tuple((a | change).values())


def test_calls_run_on_the_gpu_of_their_tensors(fake_gpus):  # noqa: F811
    current, made = fake_gpus
    native.paged_key_mass(*_mass_args(), max_q_len=3, max_kv_len=32)
    native.paged_attention(_elsewhere(3, 4, 64), _elsewhere(4, 2, 16, 64), _elsewhere(4, 2, 16, 64),
                           _elsewhere(1, 2, dtype=I32), _elsewhere(2, dtype=I32), _elsewhere(1, dtype=I32), max_q_len=3,
                           max_kv_len=32, lse=_elsewhere(3, 4))
    native.paged_evict(*_evict_args(), 8, max_kv_len=32)
    native.block_mass(_elsewhere(1, 4, 70, 64), _elsewhere(1, 2, 70, 64), workspace=_elsewhere(1 << 20))
    native.topk_distill(_elsewhere(3, 9), _elsewhere(3, 2, dtype=I32), _elsewhere(3, 2), grad_weight=_elsewhere(3))
    assert made == [(f"spruce_{x}", 1) for x in ("paged_key_mass", "paged_attention_lse", "paged_evict", "block_mass",
                                                  "topk_distill")]
    assert current[0] == 0


@pytest.mark.parametrize("change, words", [
    (dict(lse=_elsewhere(3, 5)), "lse must be"), (dict(lse=_elsewhere(3, 4, dtype=torch.float16)), "lse must be"),
    (dict(mass=_elsewhere(4, 2, 8)), "mass must be"), (dict(mass=_elsewhere(4, 2, 16, dtype=torch.float16)), "mass must be"),
    (dict(q=_elsewhere(3, 4, 32)), "q must be"), (dict(table=_elsewhere(1, 2)), "must be int32"),
    (dict(cu=_elsewhere(3, dtype=I32)), r"cu_q \[S \+ 1\]"), (dict(q=_elsewhere(3, 4, 64, dtype=torch.float16)), "dtype")])
def test_key_mass_refuses(fake_gpus, change, words):  # noqa: F811
    with pytest.raises(ValueError, match=words):
        native.paged_key_mass(*_mass_args(**change), max_q_len=3, max_kv_len=32)
    assert not fake_gpus[1]


@pytest.mark.parametrize("change, kw, words", [
    (dict(v=_elsewhere(4, 2, 16, 32)), {}, "of one shape"), (dict(mass=_elsewhere(4, 2, 8)), {}, "mass must be"),
    (dict(table=_elsewhere(2, 2, dtype=I32)), {}, "block table must be"), (dict(kv=_elsewhere(1)), {}, "kv_lens must be"),
    (dict(v=_elsewhere(4, 2, 16, 64, dtype=torch.float16)), {}, "share a dtype"), ({}, dict(keep=-1), "not be negative"),
    ({}, dict(into=(_elsewhere(4, 2, 32, 64), _elsewhere(4, 2, 32, 64), _elsewhere(4, 2, 32), _elsewhere(1, 2, dtype=I32))),
     "caches of `into`"),
    ({}, dict(into=(_elsewhere(4, 2, 16, 64), _elsewhere(4, 2, 16, 64), _elsewhere(4, 2, 15), _elsewhere(1, 2, dtype=I32))),
     "mass of `into`")])
def test_evict_refuses(fake_gpus, change, kw, words):  # noqa: F811
    with pytest.raises(ValueError, match=words):
        native.paged_evict(*_evict_args(**change), **(dict(keep=8, max_kv_len=32) | kw))
    assert not fake_gpus[1]


@pytest.mark.parametrize("q, k, kw, words", [
    (_elsewhere(1, 4, 70), _elsewhere(1, 2, 70, 64), {}, "must be"), (_elsewhere(1, 4, 70, 64), _elsewhere(1, 2, 71, 64), {}, "k must be"),
    (_elsewhere(1, 4, 70, 64), _elsewhere(1, 2, 70, 64, dtype=torch.float16), {}, "share a dtype"),
    (_elsewhere(1, 4, 70, 64), _elsewhere(1, 2, 70, 64), dict(out=_elsewhere(1, 2, 2, 3)), "out must be"),
    (_elsewhere(1, 4, 70, 64, dtype=torch.float64), _elsewhere(1, 2, 70, 64, dtype=torch.float64), {}, "unsupported dtype"),
    (_elsewhere(1, 4, 70, 64), _elsewhere(1, 2, 70, 64), dict(workspace=_elsewhere(9, 9)[:, :4]), "contiguous")])
def test_block_mass_refuses(fake_gpus, q, k, kw, words):  # noqa: F811
    with pytest.raises(ValueError, match=words):
        native.block_mass(q, k, **kw)
    assert not fake_gpus[1]


@pytest.mark.parametrize("change, words", [
    (dict(ids=_elsewhere(3, 2)), "ids must be"), (dict(ids=_elsewhere(4, 2, dtype=I32)), "expected scores"),
    (dict(teacher=_elsewhere(3, 3)), "expected scores"), (dict(visible=_elsewhere(3, 1, dtype=I32)), "visible must be"),
    (dict(visible=_elsewhere(3, dtype=torch.int64)), "visible must be"), (dict(grad_weight=_elsewhere(2)), "weights must be"),
    (dict(teacher=_elsewhere(3, 2, dtype=torch.float64)), "unsupported dtype")])
def test_distill_refuses(fake_gpus, change, words):  # noqa: F811
    a = dict(scores=_elsewhere(3, 9), ids=_elsewhere(3, 2, dtype=I32), teacher=_elsewhere(3, 2)) | change
    with pytest.raises(ValueError, match=words):
        native.topk_distill(**a)
    assert not fake_gpus[1]
    with pytest.raises(ValueError, match="stats must be"):
        native.topk_distill_backward(_elsewhere(3, 9), _elsewhere(3, 2, dtype=I32), _elsewhere(3, 2), _elsewhere(2, 2), _elsewhere(3))


def test_tensors_of_the_host_and_of_two_gpus_are_refused():
    with pytest.raises(RuntimeError, match="require CUDA"):
        native.topk_distill(torch.zeros(2, 4), torch.zeros(2, 1, dtype=I32), torch.zeros(2, 1))
    with pytest.raises(RuntimeError, match="require CUDA"):
        native.block_mass(torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, 3, 64))
    with pytest.raises(RuntimeError, match="require CUDA"):
        topk_distill_loss(torch.zeros(2, 4, requires_grad=True), torch.zeros(2, 1, dtype=I32), torch.zeros(2, 1))
    with pytest.raises((RuntimeError, ValueError)):
        native.paged_evict(*_evict_args(kv=torch.zeros(1, dtype=I32)), 8, max_kv_len=32)


def _pack(struct, names, **values):
    assert len(names) * 8 == struct.size
    unknown = set(values) - set(names)
    assert not unknown, unknown
    return struct.pack(*[values.get(n, 0) for n in names])


def _fields(name):
    """Field names of an argument struct of the header, arrays numbered, in order."""
    import os

    from test_host import ROOT
    text = open(os.path.join(ROOT, "include", "spruce_b200.h")).read()
    body = re.search(r"typedef struct \{([^}]*)\} spruce_" + name + "_args;", text).group(1)
    out = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        decl = re.sub(r"^\s*(const\s+)?\w+\s", "", decl.strip())
        for item in filter(None, (x.strip().lstrip("*") for x in decl.split(","))):
            m = re.fullmatch(r"(\w+)(?:\[(\d+)\])?", item)
            out += [m[1]] if m[2] is None else [f"{m[1]}{i}" for i in range(int(m[2]))]
    return out


GOOD = {
    "paged_key_mass": (_lib.PAGED_KEY_MASS_ARGS, dict(
        q=256, k_cache=256, lse=256, mass=256, mass_out=256, block_table=256, cu_q=256, kv_lens=256, q_strides0=256,
        q_strides1=64, kc_strides0=2048, kc_strides1=1024, kc_strides2=64, dtype=1, N=3, S=1, Hq=4, Hkv=2, D=64, num_pages=4,
        page_size=16, table_stride=2, max_pages=2, max_q_len=3, max_kv_len=32, scale=1.0, decay=1.0)),
    "paged_evict": (_lib.PAGED_EVICT_ARGS, dict(
        k_cache=256, v_cache=512, mass=256, k_out=256, v_out=512, mass_out=256, block_table=256, out_table=256, kv_lens=256,
        kept=256, new_lens=512, kc_strides2=64, vc_strides2=64, k_out_strides2=64, v_out_strides2=64, dtype=1, S=1, Hkv=2, D=64,
        num_pages=4, page_size=16, table_stride=2, max_pages=2, out_pages=4, out_table_stride=2, out_max_pages=2,
        max_kv_len=32, width=8, keep=8)),
    "block_mass": (_lib.BLOCK_MASS_ARGS, dict(
        q=256, k=256, out=256, workspace=256, q_strides0=64, q_strides1=64, q_strides2=64, q_strides3=1, k_strides0=64,
        k_strides1=64, k_strides2=64, k_strides3=1, dtype=1, B=1, Hq=4, Hkv=2, T=70, D=64, workspace_bytes=1 << 30, scale=1.0)),
    "topk_distill": (_lib.TOPK_DISTILL_ARGS, dict(
        scores=256, ids=256, teacher=256, loss=256, score_stride=9, id_stride=2, teacher_stride=2, dtype=1, R=3, n=9, K=2, tau=1.0)),
}


@pytest.mark.parametrize("name, change, words", [
    ("paged_key_mass", dict(dtype=7), "dtype"), ("paged_key_mass", dict(Hq=3), "divisible"), ("paged_key_mass", dict(D=96), "head_dim"),
    ("paged_key_mass", dict(page_size=24), "page_size"), ("paged_key_mass", dict(decay=1.5), "decay"),
    ("paged_key_mass", dict(decay=float("nan")), "decay"), ("paged_key_mass", dict(scale=-1.0), "scale"),
    ("paged_key_mass", dict(lse=0), "null"), ("paged_key_mass", dict(q=264), "aligned"), ("paged_key_mass", dict(q_strides0=4), "aligned"),
    ("paged_key_mass", dict(q_strides1=0), "positive strides"), ("paged_key_mass", dict(kc_strides1=-1024), "positive strides"),
    ("paged_key_mass", dict(num_pages=0), "no pages"), ("paged_key_mass", dict(max_q_len=1 << 40), "too long"),
    ("paged_evict", dict(dtype=-1), "dtype"), ("paged_evict", dict(D=60), "16 bytes"), ("paged_evict", dict(D=1024), "512"),
    ("paged_evict", dict(keep=-1), "negative"), ("paged_evict", dict(width=7), "wide"), ("paged_evict", dict(new_lens=256), "may not be"),
    ("paged_evict", dict(page_size=8), "page_size"), ("paged_evict", dict(mass=0), "null"), ("paged_evict", dict(out_max_pages=0), "stay"),
    ("paged_evict", dict(k_cache=264, k_out=264), "aligned"), ("paged_evict", dict(v_out=1024), "in place"),
    ("paged_evict", dict(mass_out=1024), "in place"), ("paged_evict", dict(k_out_strides2=128), "in place"),
    ("paged_evict", dict(S=1 << 40), "too large"),
    ("block_mass", dict(dtype=9), "dtype"), ("block_mass", dict(Hq=5), "divisible"), ("block_mass", dict(D=32), "head_dim"),
    ("block_mass", dict(scale=float("inf")), "scale"), ("block_mass", dict(q_strides3=2), "aligned"),
    ("block_mass", dict(q_strides2=0), "positive"), ("block_mass", dict(workspace_bytes=16), "workspace"),
    ("block_mass", dict(workspace=128), "256-byte"), ("block_mass", dict(T=1 << 30), "too large"), ("block_mass", dict(out=0), "null"),
    ("topk_distill", dict(dtype=3), "dtype"), ("topk_distill", dict(teacher_dtype=3), "dtype"), ("topk_distill", dict(K=2049), "2048"),
    ("topk_distill", dict(tau=0.0), "temperature"), ("topk_distill", dict(tau=-1.0), "temperature"),
    ("topk_distill", dict(tau=float("nan")), "temperature"), ("topk_distill", dict(loss=0), "null"),
    ("topk_distill", dict(grad=256), "null"), ("topk_distill", dict(grad=256, weight=256, stats_in=256), "alone"),
    ("topk_distill", dict(n=-1), "bad shape"), ("topk_distill", dict(n=1 << 31), "too large")])
def test_c_entries_refuse_before_any_device_work(name, change, words):
    struct, good = GOOD[name]
    lib = _lib.load()
    rc = getattr(lib, f"spruce_{name}")(_pack(struct, _fields(name), **(good | change)))
    assert rc in (_lib.ERR_INVALID, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE)
    assert words in lib.spruce_last_error().decode()
    assert getattr(lib, f"spruce_{name}")(None) == _lib.ERR_INVALID


@pytest.mark.parametrize("change", [dict(k_out=1024), dict(k_out=1024, v_out=1024), dict(k_out=1024, mass_out=1024),
                                    dict(k_out=1024, v_out=256, mass_out=1024), dict(v_cache=256, v_out=256),
                                    dict(k_out=512, v_out=256)])
def test_an_eviction_that_is_partly_in_place_is_refused(change):
    """Rows of one array would be written over before they are read, or moved twice."""
    struct, good = GOOD["paged_evict"]
    lib = _lib.load()
    assert lib.spruce_paged_evict(_pack(struct, _fields("paged_evict"), **(good | change))) == _lib.ERR_INVALID
    assert "in place" in lib.spruce_last_error().decode()


def test_empty_calls_do_nothing():
    lib = _lib.load()
    for name, change in (("paged_key_mass", dict(N=0)), ("paged_key_mass", dict(S=0)), ("paged_evict", dict(S=0)),
                         ("block_mass", dict(T=0)), ("block_mass", dict(B=0)), ("topk_distill", dict(R=0))):
        struct, good = GOOD[name]
        assert getattr(lib, f"spruce_{name}")(_pack(struct, _fields(name), **(good | change))) == _lib.OK
    assert lib.spruce_paged_attention_lse(None) == _lib.ERR_INVALID
    assert lib.spruce_block_mass_workspace_bytes(1, 28, 4, 131072, 128, 1) > 0
    assert lib.spruce_block_mass_workspace_bytes(1, 28, 3, 131072, 128, 1) == -1
    assert lib.spruce_block_mass_workspace_bytes(1, 28, 4, 131072, 96, 1) == -1


def test_a_gradient_without_columns_is_an_empty_call():
    """An empty tensor's address is null."""
    struct, good = GOOD["topk_distill"]
    for change in (dict(n=0, loss=0, stats_in=256, weight=256), dict(n=0, scores=0, loss=0, weight=256)):
        assert _lib.load().spruce_topk_distill(_pack(struct, _fields("topk_distill"), **(good | change))) == _lib.OK


# ------------------------------------------------------------------ the cache
def _tracked(monkeypatch, pages=12, page=16, layers=2):
    cut = []

    def evict(k, v, mass, table, lens, keep, **kw):
        cut.append((k.data_ptr(), table.tolist(), lens.tolist(), keep, kw))
        return None, None
    monkeypatch.setattr(native, "paged_evict", evict)
    return PagedKVCache(layers, pages, page, 2, 64, torch.float32, "cpu", track_mass=True), cut


def test_eviction_returns_pages_and_moves_positions_on(monkeypatch):
    c, cut = _tracked(monkeypatch)
    s = c.step([("a", 70), ("b", 20)])
    a = s.block_table[0].tolist()
    assert s.positions is None and s.max_position == 70 and c.free_pages == 5
    assert c.evict(["a", "b", "nobody"], 33, sinks=1, recent=4) == ["a"]
    assert [x[0] for x in cut] == [c.k[0].data_ptr(), c.k[1].data_ptr()]          # every layer
    assert cut[0][1:] == ([a], [70], 33, dict(sinks=1, recent=4, max_kv_len=70))
    assert (c.length("a"), c.position("a"), c.length("b"), c.position("b")) == (33, 70, 20, 20)
    assert c.free_pages == 7
    s = c.step([("b", 2), ("a", 3)])
    assert s.kv_lens.tolist() == [22, 36] and s.positions.tolist() == [20, 21, 70, 71, 72]
    assert (s.max_kv_len, s.max_position, s.tokens) == (36, 73, 5) and s.block_table[1, :3].tolist() == a[:3]
    assert c.step([("b", 1)]).positions is None
    c.truncate("a", 34)
    assert c.position("a") == 71
    with pytest.raises(ValueError, match="an eviction's"):
        c.truncate("a", 32)
    assert c.evict(["a", "b"], 20) == ["a", "b"] and cut[-1][2] == [34, 23]
    assert (c.position("a"), c.position("b")) == (71, 23) and c.length("a") == 20
    c.drop("a")
    assert c.position("a") == 0 and c.step([("a", 2)]).positions is None


def test_eviction_refuses(monkeypatch):
    c, cut = _tracked(monkeypatch)
    c.step([("a", 50)])
    for kw in (dict(keep=0), dict(keep=8, sinks=5, recent=4), dict(keep=8, sinks=-1), dict(keep=8, recent=-1)):
        with pytest.raises(ValueError, match="cannot keep"):
            c.evict(["a"], **kw)
    with pytest.raises(ValueError, match="appears twice"):
        c.evict(["a", "a"], 8)
    with pytest.raises(ValueError, match="without track_mass"):
        PagedKVCache(1, 4, 16, 2, 64, torch.float32, "cpu").evict(["a"], 8)
    assert c.evict(["a"], 50) == [] and not cut and c.length("a") == 50
    for kw in (dict(decay=1.5), dict(decay=-0.1), dict(observe=0)):
        with pytest.raises(ValueError):
            PagedSparseLayer(c, 0, None, **kw)


def test_a_layer_adds_weights_only_where_its_cache_keeps_them(monkeypatch):
    c, _ = _tracked(monkeypatch)
    calls = []
    for name in ("paged_append", "paged_attention", "paged_key_mass", "qk_norm_rope"):
        def call(*args, called=name, **kw):
            calls.append((called, kw))
            return args[:2] if called == "qk_norm_rope" else kw.get("q", args[0])
        monkeypatch.setattr(native, name, call)
    layer = PagedSparseLayer(c, 0, torch.zeros(100, 64), prefill=lambda q, k, v: (q, None), decay=0.5, observe=3)
    x = torch.zeros(40, 2, 64)
    layer.prefill(x, x, x, c.step([("a", 40)]))
    assert [n for n, _ in calls] == ["qk_norm_rope", "paged_append", "paged_attention", "paged_key_mass"]
    assert calls[-1][1]["decay"] == 0.0 and calls[-1][1]["max_q_len"] == 3 and calls[2][1]["lse"].shape == (3, 2)
    c.evict(["a"], 20)
    del calls[:]
    layer.extend(x[:5], x[:5], x[:5], c.step([("a", 2)]))                       # a buffer of a fixed size
    assert [n for n, _ in calls] == ["paged_append", "paged_attention", "paged_key_mass"]
    assert calls[0][1]["positions"].tolist() == [40, 41, 0, 0, 0] and calls[-1][1]["decay"] == 0.5
    step = c.step([("a", 59)])
    assert (step.max_kv_len, step.max_position) == (81, 101)
    with pytest.raises(ValueError, match="101 tokens need a rotation table"):
        layer.extend(torch.zeros(59, 2, 64), torch.zeros(59, 2, 64), torch.zeros(59, 2, 64), step)


def test_an_empty_prompt_has_no_queries_to_observe(monkeypatch):
    c, _ = _tracked(monkeypatch)
    calls = []
    for name in ("paged_append", "paged_attention", "paged_key_mass", "qk_norm_rope"):
        def call(*args, called=name, **kw):
            calls.append(called)
            return args[:2] if called == "qk_norm_rope" else args[0]
        monkeypatch.setattr(native, name, call)
    layer = PagedSparseLayer(c, 0, None, prefill=lambda q, k, v: (q, None))
    x = torch.zeros(0, 2, 64)
    assert layer.prefill(x, x, x, c.step([("a", 0)]))[0].shape == (2, 0, 64) and calls == ["qk_norm_rope", "paged_append"]


def test_drafts_weigh_when_they_are_accepted(monkeypatch):
    c, _ = _tracked(monkeypatch)
    calls = []
    for name in ("paged_append", "paged_attention", "paged_key_mass"):
        def call(*args, called=name, **kw):
            calls.append((called, args, kw))
            return kw["q"] if called == "paged_append" else args[0]
        monkeypatch.setattr(native, name, call)
    layer = PagedSparseLayer(c, 1, None, decay=0.5)
    c.step([("a", 30), ("b", 20), ("c", 5), ("d", 9)])

    def drafted():
        step = c.step([("a", 4), ("b", 3), ("c", 2), ("d", 2)])
        x = torch.randn(13, 2, 64)                                                  # a buffer of a fixed size
        out, seen = layer.draft(x, x, x, step)
        assert [n for n, _, _ in calls] == ["paged_append", "paged_attention"] and torch.equal(out, x)
        seen[1][:] = torch.arange(26.0).view(13, 2)
        del calls[:]
        return x, seen, step

    x, seen, step = drafted()
    c.truncate("a", 31)
    c.truncate("c", 4)                                                              # less than before the step
    c.drop("d")
    assert c.accepted(step) == [1, 3, 0, 0]
    layer.accept(seen, step)
    (name, (q, k, mass, table, cu, kv, lse), kw), = calls
    assert name == "paged_key_mass" and k is layer.k_cache and mass is layer.mass and table is step.block_table
    assert torch.equal(q, x[[0, 4, 5, 6]]) and torch.equal(lse, seen[1][[0, 4, 5, 6]])
    assert cu.tolist() == [0, 1, 4, 4, 4] and kv.tolist() == [31, 23, 5, 9] and cu.dtype == kv.dtype == I32
    assert kw == dict(decay=0.5, max_q_len=3, max_kv_len=step.max_kv_len)
    del calls[:]
    x, seen, step = drafted()
    layer.accept(seen, step)                                                        # all of them
    (name, args, kw), = calls
    assert args[0] is seen[0] and args[4] is step.cu_q and args[5] is step.kv_lens and kw["max_q_len"] == 4
    del calls[:]
    x, seen, step = drafted()
    for s, n in zip("abcd", (35, 26, 6, 2)):
        c.truncate(s, n)
    layer.accept(seen, step)                                                        # none
    assert not calls
    c.step([("a", 1)])
    with pytest.raises(ValueError, match="'a' has gone on"):
        layer.accept(seen, step)
    x, seen, step = drafted()
    c.evict(["b"], 20)
    with pytest.raises(ValueError, match="'b' has gone on"):
        layer.accept(seen, step)
    plain = PagedSparseLayer(PagedKVCache(1, 4, 16, 2, 64, torch.float32, "cpu"), 0, None)
    step = plain.cache.step([("a", 2)])
    out, seen = plain.draft(x[:2], x[:2], x[:2], step)
    assert seen[1] is None and plain.accept(seen, step) is None and [n for n, _, _ in calls][-1] == "paged_attention"


# ------------------------------------------------------------------ the gate
@pytest.mark.parametrize("P", [1, 3])
def test_training_scores_are_the_gates_formula(P):
    g = torch.Generator().manual_seed(1)
    gate = FlatGate(2, 16, 8)
    q, k = (torch.randn(2, 3, 5, P, 16, generator=g, dtype=torch.float16) for _ in range(2))
    s = gate_training_scores(gate, q, k)
    qp = torch.einsum("lgqpd,lde->lgqpe", q.double(), gate.Wq.double())
    kp = torch.einsum("lgkpd,lde->lgkpe", k.double(), gate.Wk.double())
    want = torch.einsum("lgqpe,lgkre->lgqkpr", qp, kp).amax((-1, -2)) / 8 ** 0.5
    assert s.requires_grad and torch.allclose(s.double(), want, atol=1e-4)
    with pytest.raises(ValueError, match="same number of prototypes"):
        gate_training_scores(gate, q, k[:, :, :, :1].expand(-1, -1, -1, P + 1, -1))
    with pytest.raises(ValueError, match="as many key blocks"):
        gate_loss(gate, q, k[:, :, :4], None, None)


def test_the_teachers_top_blocks_are_checked():
    with pytest.raises(ValueError, match="k must be positive"):
        teacher_top_blocks(torch.ones(2, 2), 0)
    ids, logits = teacher_top_blocks(torch.tensor([[0.25, 0.75]]), 5)
    assert ids.tolist() == [[1, 0]] and torch.allclose(logits.exp(), torch.tensor([[0.75, 0.25]]))
