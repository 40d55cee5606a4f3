"""Every way the router's gradient of a served snapshot is summed, at sizes taken from the rules that choose among them."""
import os
import re

import numpy as np
import pytest

import ddrl_amd
import snapshot_common as sc
from test_snapshot_gpu import ask_grad, within
from test_snapshot_sizes_gpu import wide_gradient

pytestmark = pytest.mark.gpu

RULES = open(os.path.join(os.path.dirname(ddrl_amd.__file__), "csrc", "snap_internal.h")).read()
SORT_FROM = int(re.search(r"#define SNAP_SORT_FROM (\d+)", RULES).group(1))


# ---- the router's gradient, each way of summing --------------------------------------------------------------------------

def check_gradient(g, n, k, ins, outs):
    """idx anything from -1 to g, prob anything from 0 to 1 (with top_k = 1 a prob of 1 would leave no gradient)"""
    rng = np.random.RandomState(g + n + k + ins)
    s = ddrl_amd.PolicySnapshot.shaped(g, ins, outs, [], bits=32)
    x, y, dout, prob = (v.astype(np.float32) for v in (rng.uniform(-1, 1, (n, ins)), rng.standard_normal((n, k, outs)), rng.standard_normal((n, outs)), rng.uniform(0, 1, (n, k))))
    idx = rng.randint(-1, g + 1, (n, k))
    dw, db, dy = ask_grad(s, x, idx, prob, y, dout)
    ww, wb, wy, bw, bb = wide_gradient(x, idx, prob, y, dout, g)
    within(dw, ww, bw)
    within(db, wb, bb)
    within(dy, wy, 2 * sc.U * np.abs(wy) + 1e-37)
    assert np.abs(ww).max() > 100 * bw.max()                          # (the check says something)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("past", [-1, 0, 1])
def test_gradient_around_the_number_of_places_that_is_sorted(past, k):
    check_gradient(9, SORT_FROM // k + past, k, 18, 6)


@pytest.mark.parametrize("k", [1, 2, 5])
@pytest.mark.parametrize("ins", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1024])
def test_gradient_of_every_row_length(ins, k):
    check_gradient(5, SORT_FROM // 2 // k, k, ins, 3)                   # unsorted
    check_gradient(5, 3 * SORT_FROM // k, k, ins, 3)                    # sorted


@pytest.mark.parametrize("g, n, k", [(1024, 20000, 8), (600, 20000, 8), (1500, 70000, 1), (3, 400, 1), (700, 2000, 1)])
def test_gradient_of_many_blocks(g, n, k):
    """an agent's places are one or a few workgroups' work: more than 64 sorted blocks each"""
    check_gradient(g, n, k, 5, 2)
