"""What the serving operators do on the host, and rules of their kernels that only the source shows (CPU)."""
import os
import re
import subprocess
import sys

import pytest
import torch

from spruce_research_b200 import build, native
from spruce_research_b200.paged import PagedKVCache, PagedSparseLayer

CSRC = build.CSRC


def test_a_warpgroup_gives_up_registers_by_one_instruction():
    """setmaxnreg is defined only where all warps of a warpgroup execute the same one: once for each side of the split,
    under a condition on the warpgroup, before the roles of its warps part."""
    with open(os.path.join(CSRC, "paged_chunk_sm100.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert len(re.findall(r"setmaxnreg\.dec", code)) == 1 and len(re.findall(r"setmaxnreg\.inc", code)) == 1
    assert re.search(r"if \(warp >= kChunkMma\) \{\s*asm volatile\(\"setmaxnreg\.dec", code)
    assert re.search(r"\} else \{\s*asm volatile\(\"setmaxnreg\.inc", code)
    roles = {k: int(v) for k, v in re.findall(r"constexpr int kChunk(Mma|Threads) = (\d+);", code)}
    assert roles["Mma"] % 4 == 0 and roles["Threads"] == 32 * (roles["Mma"] + 4)   # whole warpgroups either side


def _cache(pages=6, page=16):
    return PagedKVCache(1, pages, page, 2, 64, torch.float32, "cpu")


def _no_kernels(monkeypatch):
    """Entry points that only note that they were called."""
    calls = []
    for name in ("paged_append", "paged_attention", "qk_norm_rope"):
        def call(*args, called=name, **kw):
            calls.append(called)
            return args[:2] if called == "qk_norm_rope" else args[0]
        monkeypatch.setattr(native, name, call)
    return calls


def test_a_layer_refuses_a_step_past_its_rotation_table(monkeypatch):
    calls = _no_kernels(monkeypatch)
    c = _cache()
    layer = PagedSparseLayer(c, 0, torch.zeros(20, 64), prefill=lambda q, k, v: (q, None))
    x = torch.zeros(21, 2, 64)
    layer.extend(x[:20], x[:20], x[:20], c.step([("a", 20)]))
    assert calls == ["paged_append", "paged_attention"]
    step = c.step([("a", 1), ("b", 3)])
    with pytest.raises(ValueError, match="21 tokens need a rotation table"):
        layer.extend(x[:4], x[:4], x[:4], step)
    step = c.step([("c", 21)])
    with pytest.raises(ValueError, match="21 tokens need a rotation table"):
        layer.prefill(x, x, x, step)
    assert calls == ["paged_append", "paged_attention"]


def test_a_layer_refuses_tensors_of_another_number_of_tokens(monkeypatch):
    """Fewer rows than the step has tokens would leave cache rows unwritten that its lengths count."""
    calls = _no_kernels(monkeypatch)
    c = _cache()
    layer = PagedSparseLayer(c, 0, torch.zeros(64, 64), prefill=lambda q, k, v: (q, None))
    x = torch.zeros(5, 2, 64)
    step = c.step([("a", 4)])
    for bad in ((x[:3], x[:4], x[:4]), (x[:4], x[:3], x[:4]), (x[:4], x[:4], x[:3])):
        with pytest.raises(ValueError, match="the step has 4 tokens"):
            layer.extend(*bad, step)
        with pytest.raises(ValueError, match="the step has 4 tokens"):
            layer.prefill(*bad, step)
    with pytest.raises(ValueError, match="the step has 4 tokens"):      # the selector would pool the rows past the prompt
        layer.prefill(x, x, x, step)
    assert not calls
    layer.prefill(x[:4], x[:4], x[:4], step)
    layer.extend(x, x, x, step)                                         # a buffer of a fixed size
    assert calls == ["qk_norm_rope", "paged_append", "paged_append", "paged_attention"]


class _Elsewhere(torch.Tensor):
    """A host tensor that says it is on GPU 1."""

    def get_device(self):
        return 1


def _elsewhere(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Elsewhere)


@pytest.fixture
def fake_gpus(monkeypatch):
    """Entry points that note their name and the current GPU; returns (the current GPU, the calls)."""
    current, made = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    class Library:
        def __getattr__(self, entry):
            return lambda args: made.append((entry, current[0])) or 0

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(native._lib, "current_device", lambda: current[0], raising=False)
    monkeypatch.setattr(native._lib, "stream_on", lambda device: 0)
    monkeypatch.setattr(native._lib, "load", Library)
    monkeypatch.setattr(native, "_paged_workspace_bytes", lambda *a: 256)
    return current, made


def _paged():
    return (_elsewhere(3, 2, 64), _elsewhere(4, 2, 16, 64), _elsewhere(1, 2, dtype=torch.int32),
            _elsewhere(2, dtype=torch.int32), _elsewhere(1, dtype=torch.int32))


def test_calls_run_on_the_gpu_of_their_tensors(fake_gpus):
    """Tensors of GPU 1 while GPU 0 is current: the stream is GPU 1's, so the launch has to be made with GPU 1 current."""
    current, made = fake_gpus
    x, cache, table, cu, kv = _paged()
    names = ["spruce_qk_norm_rope", "spruce_paged_append", "spruce_paged_attention"]
    for device in (0, 1):
        current[0] = device
        native.qk_norm_rope(x[None], x[None], _elsewhere(8, 64))
        native.paged_append(x, x, cache, cache, table, cu, kv)
        native.paged_attention(x, cache, cache, table, cu, kv, max_q_len=3, max_kv_len=3)
        assert made == [(name, 1) for name in names] and current[0] == device
        made.clear()


def test_a_workspace_with_gaps_or_repeats_is_refused(fake_gpus):
    """The kernels take its bytes as one block: an expanded element has the size of a workspace and not its memory."""
    x, cache, table, cu, kv = _paged()
    for bad in (_elsewhere(1).expand(1 << 20), _elsewhere(1 << 10, 2)[:, 0]):
        with pytest.raises(ValueError, match="workspace must be contiguous"):
            native.paged_attention(x, cache, cache, table, cu, kv, max_q_len=3, max_kv_len=3, workspace=bad)
    assert not fake_gpus[1]


def test_no_arguments_are_an_error_and_not_a_crash():
    """A null argument struct at the C entries; in a process of its own, as it could end it."""
    code = ("from spruce_research_b200 import _lib\n"
            "L = _lib.load()\n"
            "for f in (L.spruce_qk_norm_rope, L.spruce_paged_append, L.spruce_paged_attention):\n"
            "    assert f(None) == _lib.ERR_INVALID and b'null' in L.spruce_last_error()\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          cwd=build.REPO)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])


def test_a_layer_without_a_rotation_table_prefills(monkeypatch):
    """paged_append takes no table for projections that need no rotation; so does the layer, in prefill as in extend."""
    seen = []
    monkeypatch.setattr(native, "qk_norm_rope", lambda q, k, rope, **kw: seen.append((rope, kw)) or (q, k))
    monkeypatch.setattr(native, "paged_append", lambda k, v, *a, **kw: seen.append(kw.get("rope")))
    c = _cache()
    w = torch.ones(64)
    layer = PagedSparseLayer(c, 0, None, prefill=lambda q, k, v: (q, None), q_weight=w)
    x = torch.zeros(20, 2, 64)
    out, _ = layer.prefill(x, x, x, c.step([("a", 20)]))
    (rope, kw), appended = seen
    assert rope.shape == (20, 0) and rope.dtype == torch.float32 and kw["q_weight"] is w     # norms, and no angle
    assert appended is None and out.shape == (2, 20, 64)


def test_a_step_that_was_not_run_can_be_taken_back(monkeypatch):
    """A refused forward leaves the cache counting tokens that were never written, until they are truncated."""
    _no_kernels(monkeypatch)
    c = _cache(pages=6)
    layer = PagedSparseLayer(c, 0, torch.zeros(40, 64))
    x = torch.zeros(41, 2, 64)
    layer.extend(x[:20], x[:20], x[:20], c.step([("a", 20)]))
    pages = c.step([("a", 0)]).block_table[0].tolist()
    step = c.step([("a", 21), ("b", 16)])
    with pytest.raises(ValueError, match="rotation table"):
        layer.extend(x, x, x, step)
    assert c.length("a") == 41 and c.free_pages == 2
    c.truncate("a", 20)
    c.truncate("b", 0)
    c.truncate("nobody", 0)
    assert c.length("a") == 20 and c.length("b") == 0 and c.free_pages == 4
    s = c.step([("a", 12)])                     # the rest of its second page
    assert s.block_table[0].tolist() == pages and s.kv_lens.tolist() == [32] and c.free_pages == 4
    s = c.step([("c", 64)])                     # the returned pages, none of them still a's
    assert len({*pages, *s.block_table[0].tolist()}) == 6
    for seq, bad in (("a", 33), ("a", -1), ("nobody", 1)):
        with pytest.raises(ValueError, match="cannot be cut"):
            c.truncate(seq, bad)
    assert c.length("a") == 32
