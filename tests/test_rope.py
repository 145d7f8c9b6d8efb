"""Rotation tables (CPU) and the refusals of the paged entry points before any device work."""
import math

import pytest
import torch

from spruce_research_b200 import _lib, native
from spruce_research_b200.rope import rope_frequencies, rope_table


def test_table_is_the_rounded_64_bit_value():
    t = rope_table(8, 131073, 1e6, device="cpu")
    assert t.shape == (131073, 8) and t.dtype == torch.float32
    for pos in (0, 1, 4097, 131072):
        for i in range(4):
            angle = pos * 1e6 ** (-2 * i / 8)
            # one rounding of the value, and libm's 64-bit error at an angle of 1e5
            assert abs(t[pos, i].item() - math.cos(angle)) <= 2.0 ** -25 + 1e-10
            assert abs(t[pos, 4 + i].item() - math.sin(angle)) <= 2.0 ** -25 + 1e-10


def test_scalings_keep_and_divide_the_frequencies_they_name():
    plain, one = rope_frequencies(64, 1e4)
    assert one == 1.0 and plain[0] == 1.0
    lin, _ = rope_frequencies(64, 1e4, {"type": "linear", "factor": 4})
    assert torch.equal(lin, plain / 4)
    ntk, _ = rope_frequencies(64, 1e4, {"type": "ntk", "factor": 4})
    assert ntk[0] == 1.0 and abs(ntk[-1] / (plain[-1] / 4) - 1) < 1e-12      # fastest kept, slowest divided
    yarn, mult = rope_frequencies(64, 1e4, {"type": "yarn", "factor": 4, "original_positions": 4096})
    assert mult == pytest.approx(0.1 * math.log(4) + 1)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], plain[turns > 40])
    torch.testing.assert_close(yarn[turns < 0.8], plain[turns < 0.8] / 4)
    assert ((yarn <= plain) & (yarn >= plain / 4)).all()
    band, _ = rope_frequencies(64, 1e4, {"type": "banded", "factor": 8, "original_positions": 8192,
                                         "low_freq_factor": 1, "high_freq_factor": 4})
    turns = 8192 * plain / (2 * math.pi)
    assert torch.equal(band[turns >= 4], plain[turns >= 4])
    torch.testing.assert_close(band[turns <= 1], plain[turns <= 1] / 8)
    assert (band[:-1] > band[1:]).all()


@pytest.mark.parametrize("kind,args", [
    ("yarn", {"factor": 4.0, "original_max_position_embeddings": 32768}),
    ("linear", {"factor": 3.0}),
    ("default", {})])
def test_frequencies_match_the_installed_transformers(kind, args):
    """The angles a transformers model of the same rope parameters uses (float32 there)."""
    from transformers import Qwen2Config
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    cfg = Qwen2Config(hidden_size=256, num_attention_heads=2, max_position_embeddings=131072,
                      rope_parameters={"rope_type": kind, "rope_theta": 1e6, **args})
    ours = None if kind == "default" else {"type": kind, "factor": args["factor"]} | (
        {"original_positions": 32768} if kind == "yarn" else {})
    freq, mult = rope_frequencies(128, 1e6, ours)
    if kind == "default":
        want, want_mult = 1.0 / 1e6 ** (torch.arange(0, 128, 2).float() / 128), 1.0
    else:
        want, want_mult = ROPE_INIT_FUNCTIONS[kind](cfg, "cpu")
    torch.testing.assert_close(freq.float(), want, rtol=2e-6, atol=0)
    assert mult == pytest.approx(want_mult)


def test_table_refusals():
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0)):
        with pytest.raises(ValueError):
            rope_frequencies(**bad)
    with pytest.raises(ValueError, match="scaling type"):
        rope_frequencies(8, scaling={"type": "cubic", "factor": 2})
    with pytest.raises(ValueError, match="factor"):
        rope_frequencies(8, scaling={"type": "linear", "factor": 0.5})
    with pytest.raises(ValueError, match="above low_freq_factor"):
        rope_frequencies(8, scaling={"type": "banded", "factor": 2, "original_positions": 64, "low_freq_factor": 4,
                                     "high_freq_factor": 4})
    with pytest.raises(ValueError, match="positions"):
        rope_table(8, 0, device="cpu")


def test_entry_points_refuse_before_device_work():
    L = _lib.load()

    def rope(D=64, rd=64, rows=8, dtype=1, last=1, rope=16, eps=1e-6):
        strides = (64, 64, 64, last) * 4 + (0, 0)
        return L.spruce_qk_norm_rope(_lib.QK_NORM_ROPE_ARGS.pack(16, 16, 16, 16, rope, 0, 0, 0, 0, 0, *strides, dtype,
                                                                 1, 2, 1, 4, D, rows, rd, 0, eps))

    for kw, text in ((dict(D=258), "head_dim"), (dict(D=63), "head_dim"), (dict(rd=66), "rotary width"),
                     (dict(rd=3), "rotary width"), (dict(rows=0), "empty"), (dict(rope=0), "empty"),
                     (dict(dtype=3), "dtype"), (dict(last=2), "unit last stride")):
        with pytest.raises(ValueError, match=text):
            _lib.check(rope(**kw))

    def append(N=1, page=16, D=64, k=16, rd=64, rows=8, S=1, table=16):
        return L.spruce_paged_append(_lib.PAGED_APPEND_ARGS.pack(
            0, k, 16, 0, 16, 16, 16, 0, 0, 0, table, 16, 16, 0, 0, *(64,) * 14, 1, N, S, 4, 2, D, 4, page, 2, 2, rows,
            rd, 0, 1e-6))

    for kw, text in ((dict(page=24), "page_size"), (dict(D=258), "head_dim"), (dict(rows=0), "empty"),
                     (dict(k=0), "null"), (dict(table=0), "NULL"), (dict(N=-1), "bad shape"),
                     (dict(N=1 << 31), "too large")):
        with pytest.raises(ValueError, match=text):
            _lib.check(append(**kw))
    assert append(N=0) == _lib.OK and append(S=0) == _lib.OK

    def attend(D=64, Hq=4, Hkv=2, page=16, N=1, S=1, max_q=1, max_kv=16, cu=16, q=16, head=64, ws=256,
               ws_bytes=1 << 30, scale=0.1, pages=4):
        return L.spruce_paged_attention(_lib.PAGED_ATTENTION_ARGS.pack(
            q, 16, 16, 16, 16, cu, 16, ws, 0, 0, 64, 64, 64, head, 64, 64, 64, 64, 64, 64, 1, N, S, Hq, Hkv, D, pages,
            page, 2, 2, max_q, max_kv, ws_bytes, scale))

    for kw, text in ((dict(D=96), "head_dim 64 or 128"), (dict(Hq=5), "divisible"), (dict(page=24), "page_size"),
                     (dict(page=8), "page_size"), (dict(N=-1), "bad shape"), (dict(max_q=-1), "negative"),
                     (dict(max_q=1 << 30), "too long"), (dict(cu=0), "NULL"), (dict(q=0), "null"),
                     (dict(pages=0), "no pages"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
                     (dict(scale=float("inf")), "scale"), (dict(q=8), "16-byte aligned"),
                     (dict(head=60), "16-byte aligned"), (dict(ws=128), "256-byte")):
        with pytest.raises(ValueError, match=text):
            _lib.check(attend(**kw))
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.check(attend(ws_bytes=16))
    for kw in (dict(N=0), dict(S=0), dict(max_q=0)):      # nothing to do
        assert attend(**kw) == _lib.OK
    assert L.spruce_paged_attention_workspace_bytes(28, 4, 96, 1, 1) == -1
    assert L.spruce_paged_attention_workspace_bytes(28, 5, 128, 1, 1) == -1
    assert L.spruce_paged_attention_workspace_bytes(28, 4, 128, 1 << 31, 1) == -1
    assert L.spruce_paged_attention_workspace_bytes(28, 4, 128, 2048, 1) > 0


def test_cpu_tensors_are_rejected():
    x = torch.zeros(1, 2, 4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        native.qk_norm_rope(x, x, torch.zeros(4, 64))
    i = torch.zeros(1, 1, dtype=torch.int32)
    cache = torch.zeros(1, 2, 16, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        native.paged_append(x[0], x[0], cache, cache, i, i[0], i[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        native.paged_attention(x[0], cache, cache, i, i[0], i[0], max_q_len=1, max_kv_len=1)
