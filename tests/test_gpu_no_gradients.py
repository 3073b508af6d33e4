"""The layer operators record no gradient, with operands that require one as with others, by both ways into the library."""
import pytest

import ternixengine_b200 as tb

pytestmark = pytest.mark.gpu


def test_operands_that_require_a_gradient():
    import torch
    x, w = torch.randn(5, 640, device="cuda", requires_grad=True), torch.rand(640, device="cuda", requires_grad=True)
    wp, b = torch.from_numpy(tb.synth_packed_weights(640, 192, 1)).cuda(), torch.randn(192, device="cuda", requires_grad=True)

    def calls(x, w, b, given):
        out = dict(out=torch.empty(5, 640, dtype=torch.int8, device="cuda"), row_scale=torch.empty(5, device="cuda")) if given else {}
        q, s, h = tb.rmsnorm_quantize(x, w, residual=x, residual_out=torch.empty_like(x, requires_grad=False) if given else None, **out)
        y = tb.matmul_fused(q, wp, s, 0.1, bias=b, out=torch.empty(5, 192, dtype=torch.bfloat16, device="cuda") if given else None)
        q2, s2 = tb.glu_quantize(x, x, activation="relu")
        return [q.clone(), s.clone(), h, y, q2, s2]

    for given in (False, True):
        got, want = calls(x, w, b, given), calls(x.detach(), w.detach(), b.detach(), given)
        assert not any(t.requires_grad for t in got) and all(torch.equal(p, q) for p, q in zip(got, want))
