"""A call that failed is reported once: the calls after it are not blamed for it."""
import numpy as np
import pytest

import oracle_lib
import ternixengine_b200 as tb

pytestmark = pytest.mark.gpu


def test_a_failed_call_does_not_fail_the_next_one():
    """A group cannot be made while a stream captures (it allocates); the products after that are as good as ever."""
    import torch
    a, wp = tb.synth_activations((3, 33), 1), tb.synth_packed_weights(33, 36, 2)
    ta, tw = torch.from_numpy(a).cuda(), torch.from_numpy(wp).cuda()
    out = torch.empty(1, 64, dtype=torch.int32, device="cuda")
    ga, gw = torch.zeros(1, 64, dtype=torch.int8, device="cuda"), torch.zeros(64, 16, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(Exception):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            with pytest.raises(tb.TernixError):
                tb.ProjectionGroup([(ga, gw, out)])
            raise RuntimeError("leave the capture")
    torch.cuda.synchronize()
    c = tb.matmul(ta, tw, kernel="generic")
    assert np.array_equal(c.cpu().numpy(), oracle_lib.matmul(a, wp))
    q, s = tb.quantize_rows(torch.ones(2, 64, device="cuda"))
    assert (q == 127).all()
    y = tb.matmul_fused(ta, tw, torch.ones(3, device="cuda"), 1.0, out_dtype=torch.float32)
    assert np.array_equal(y.cpu().numpy(), oracle_lib.matmul(a, wp).astype(np.float32))
