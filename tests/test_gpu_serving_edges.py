"""The serving operators at the edges of their contract: tokens of no sequence, bounds below the lengths, scores that are
not finite, weights near the end of fp16's range, tensors at odd addresses."""
import pytest
import torch

from spruce_research_b200 import native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 1])          # an odd base address takes the scalar kernel
@pytest.mark.parametrize("with_q", [True, False])
def test_append_leaves_out_tokens_before_the_first_sequence(shift, with_q):
    """Two sequences of a larger batch, with all its packed tokens: cu_q starts at 3, tokens 0 to 2 and 7 to 8 belong to
    none.  Their q rows are not written, nor is any cache row but the four new ones."""
    g = torch.Generator(device="cuda").manual_seed(1)
    N, Hq, Hkv, D, page = 9, 4, 2, 64, 16
    flat = torch.randn(N * (Hq + 2 * Hkv) * D + 8, generator=g, device="cuda", dtype=torch.bfloat16)
    q, k, v = flat[shift:shift + N * (Hq + 2 * Hkv) * D].view(N, Hq + 2 * Hkv, D).split([Hq, Hkv, Hkv], 1)
    cu = torch.tensor([0, 3, 5, 7, 9], device="cuda", dtype=torch.int32)[1:4]
    kv = torch.tensor([10, 18], device="cuda", dtype=torch.int32)
    table = torch.tensor([[2, 3], [0, 1]], device="cuda", dtype=torch.int32)
    kc, vc = (torch.randn(4, Hkv, page, D, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    for n, p, r in ((3, 2, 8), (4, 2, 9), (5, 1, 0), (6, 1, 1)):
        want_k[p, :, r], want_v[p, :, r] = k[n], v[n]
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    out = torch.full((N, Hq, D), 7.0, device="cuda", dtype=torch.bfloat16)
    native.paged_append(k, v, kc, vc, table, cu, kv, status=status, **(dict(q=q, q_out=out) if with_q else {}))
    assert status.item() == 0
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    if with_q:
        assert torch.equal(out[3:7], q[3:7]) and (out[:3] == 7).all() and (out[7:] == 7).all()
