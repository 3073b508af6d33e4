"""Decode batches and layer kernels back to back on a stream, nothing between them: both let the next one begin early."""
import numpy as np
import pytest

import oracle_lib
import ternixengine_b200 as tb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["layer-batch-layer", "layer-batch-batch-layer", "product-batch"])
def test_batches_next_to_layer_kernels(order):
    """The batch reads codes that the layer kernel in front of it writes; the layer kernel behind it overwrites them.  Queued in
    one go the batches see what they see with a synchronisation after every call, and what the CPU oracle says of it."""
    import torch
    D, N = 2560, 640
    wp = [tb.synth_packed_weights(D, N, i) for i in range(2)]
    w = [torch.from_numpy(x).cuda() for x in wp]
    code, scale = torch.zeros(1, D, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")
    steps = 40
    xs = [torch.randn(1, D, device="cuda").to(torch.bfloat16) for _ in range(steps)]
    outs = [[torch.zeros(1, N, dtype=torch.int32, device="cuda") for _ in range(2)] for _ in range(steps)]
    groups = [[tb.ProjectionGroup([(code, w[i], outs[s][i])]) for i in range(2)] for s in range(steps)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = torch.zeros(1, N, dtype=torch.bfloat16, device="cuda")

    def run(sync):
        done = torch.cuda.synchronize if sync else (lambda: None)
        for s in range(steps):
            tb.rmsnorm_quantize(xs[s], out=code, row_scale=scale); done()
            if order == "product-batch":
                tb.matmul_fused(code, w[0], scale, 0.1, out=y); done()
            groups[s][0].run(status=status); done()
            if order == "layer-batch-batch-layer":
                groups[s][1].run(status=status); done()
        torch.cuda.synchronize()
        got = [[o.cpu().numpy().copy() for o in pair] for pair in outs]
        for pair in outs:
            for o in pair:
                o.zero_()
        return got

    want, got = run(True), run(False)
    for s in range(steps):
        codes = tb.rmsnorm_quantize(xs[s])[0].cpu().numpy()
        assert np.array_equal(want[s][0], oracle_lib.matmul(codes, wp[0])) and np.array_equal(want[s][0], got[s][0])
        if order == "layer-batch-batch-layer":
            assert np.array_equal(want[s][1], oracle_lib.matmul(codes, wp[1])) and np.array_equal(want[s][1], got[s][1])
    assert int(status) == 0


def test_a_batch_behind_a_kernel_longer_than_its_wait_limit():
    """The batch begins while the gate still runs, for longer than the 2 s after which a wait of the batch's would give up: the
    gate's time does not count."""
    import torch
    K, D, N = 2 ** 31 - 1025, 2560, 640
    gate = torch.ones((1, K), dtype=torch.float32, device="cuda")
    codes, scale = torch.empty((1, K), dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    wp = tb.synth_packed_weights(D, N, 1)
    out = torch.zeros(1, N, dtype=torch.int32, device="cuda")
    group = tb.ProjectionGroup([(codes[:, :D], torch.from_numpy(wp).cuda(), out)])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    start, mid, end = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    group.run(status=status)                        # whatever is set up at the first run
    torch.cuda.synchronize()
    start.record()
    tb.glu_quantize(gate, gate, activation="gelu_tanh", eps=1e-5, out=codes, row_scale=scale)
    group.run(status=status)
    end.record()
    torch.cuda.synchronize()
    print("gate and batch:", start.elapsed_time(end), "ms")
    assert int(status) == 0
    assert np.array_equal(out.cpu().numpy(), oracle_lib.matmul(np.full((1, D), 127, dtype=np.int8), wp))
