"""Problem groups one after another whose tables of TMA descriptors lie at the same address: each has to see its own
descriptors, not the ones that the TMA unit still holds from a group (or a batch) before it."""
import numpy as np
import pytest

import oracle_lib
import ternixengine_b200 as tb

pytestmark = pytest.mark.gpu

# one row: transposing GEMV; a few rows: mma.sync; some dozens: tensor-memory decode; hundreds: prefill tiles
SHAPES = {1: [(1, 256, 320), (1, 640, 192), (1, 1040, 64)], 9: [(9, 256, 320), (5, 640, 192), (16, 1040, 64)],
          40: [(40, 256, 320), (33, 640, 192), (64, 1040, 64)], 300: [(300, 256, 320), (129, 640, 512), (200, 1040, 256)]}


def problems(shapes, seed):
    import torch
    probs, expect = [], []
    for i, (m, k, n) in enumerate(shapes):
        a, w = tb.synth_activations((m, k), seed + i), tb.synth_packed_weights(k, n, seed + 50 + i)
        expect.append(oracle_lib.matmul(a, w))
        probs.append((torch.from_numpy(a).cuda(), torch.from_numpy(w).cuda(), torch.full((m, n), -7, dtype=torch.int32, device="cuda")))
    return probs, expect


@pytest.mark.parametrize("rows", list(SHAPES))
@pytest.mark.parametrize("tc3", ["1", "0"])
def test_groups_that_follow_one_another(rows, tc3, option):
    """Made, run and closed in turn, each with other sizes and operands in the same slots of the table; without a
    synchronisation of the caller's between them."""
    import torch
    if tc3 == "0" and rows < 128:
        pytest.skip("the same kernels as with tc3 = 1")
    option("tc3", tc3)
    shapes, status, seen = SHAPES[rows], torch.zeros(1, dtype=torch.int32, device="cuda"), []
    rounds = [problems(shapes[i % 3:] + shapes[:i % 3], 100 * i) for i in range(12)]
    for probs, _ in rounds:
        group = tb.ProjectionGroup(probs)
        group.run(status=status)
        seen.append([out.clone() for _, _, out in probs])
        group.close()
    for got, (_, expect) in zip(seen, rounds):
        assert all(np.array_equal(g.cpu().numpy(), e) for g, e in zip(got, expect))
    assert int(status) == 0


@pytest.mark.parametrize("rows", list(SHAPES))
def test_groups_that_live_side_by_side(rows):
    """Two tables in turn, many times."""
    shapes = SHAPES[rows]
    sets = [problems(shapes, 1), problems(shapes[::-1], 2)]
    groups = [tb.ProjectionGroup(p) for p, _ in sets]
    for turn in range(20):
        i = turn % 2
        for _, _, out in sets[i][0]:
            out.fill_(-7)
        groups[i].run()
        if turn > 17 or turn < 2:
            assert all(np.array_equal(out.cpu().numpy(), e) for (_, _, out), e in zip(*sets[i]))
