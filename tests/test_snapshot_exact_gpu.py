"""Served snapshots where 32 bits would not do: router logits and sums over rows that need the 64 bits they are promised
(ddrl_snap_mixture*), and every way the router's gradient is summed, at sizes taken from the rules that choose among them."""
import os
import re

import numpy as np
import pytest

import ddrl_amd
import snapshot_common as sc
from test_snapshot_gpu import ask_grad, ask_mixture, within
from test_snapshot_sizes_gpu import one_net, wide_gradient

pytestmark = pytest.mark.gpu

RULES = open(os.path.join(os.path.dirname(ddrl_amd.__file__), "csrc", "snap_internal.h")).read()
SORT_FROM = int(re.search(r"#define SNAP_SORT_FROM (\d+)", RULES).group(1))
CHUNK_ROWS = int(re.search(r"#define SNAP_CHUNK_ROWS (\d+)", RULES).group(1))


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


# ---- sums over rows are 64 bits wide -------------------------------------------------------------------------------------

@pytest.mark.parametrize("g, n, spread", [(3, SORT_FROM // 2 - 2, 3), (2, SORT_FROM // 2 - 2, 2), (3, 4000, 3), (3, 40000, 3), (1100, 4000, 4), (1100, 40000, 700)])
@pytest.mark.parametrize("ins", [3, 70])
def test_sums_of_large_rows_that_cancel(g, n, spread, ins):
    """Rows of 2^20 that cancel in pairs, among rows of 2^-6.  With prob = .5, y = (s, 0), dout = 1 a row's dlogit is (s / 4, -s / 4),
    exactly; x are whole numbers.  All of it are multiples of 2^-8 below 2^42, so a sum of 64 bits is exact in any order, and
    what comes out is one rounding to 32.  A running sum of 32 bits loses the small rows next to the large."""
    rng = np.random.RandomState(n + g)
    n -= n % 4
    half = n // 4
    s = np.concatenate([rng.randint(1, 8, half) * 2.0 ** 20] * 2 + [rng.randint(-7, 8, n // 2) * 2.0 ** -6])
    s[half:2 * half] *= -1
    x = rng.randint(-7, 8, (n, ins)).astype(np.float64)
    e = rng.randint(0, spread, n)
    idx = np.stack((e, (e + 1 + rng.randint(0, spread - 1, n)) % spread), 1)
    x[half:2 * half], idx[half:2 * half] = x[:half], idx[:half]
    order = rng.permutation(n)
    s, x, idx = s[order], x[order], idx[order]
    y = np.stack((s, np.zeros(n)), 1)[..., None]
    snap = ddrl_amd.PolicySnapshot.shaped(g, ins, 1, [], bits=32)
    dw, db, _ = ask_grad(snap, x, idx, np.full((n, 2), .5), y, np.ones((n, 1)))
    ww, wb = np.zeros((g, ins)), np.zeros(g)
    for j, sign in ((0, .25), (1, -.25)):
        np.add.at(ww, idx[:, j], sign * s[:, None] * x)
        np.add.at(wb, idx[:, j], sign * s)
    assert np.array_equal(dw, ww.astype(np.float32)) and np.array_equal(db, wb.astype(np.float32))


# ---- the router's logits are 64 bits wide --------------------------------------------------------------------------------

@pytest.mark.parametrize("unit", [2.0 ** -20, 2.0 ** -28])
@pytest.mark.parametrize("bits, dims, g, n, k", [
    (4, (18, 20, 6), 40, 5, 4), (32, (18, 20, 6), 64, 3, 8), (4, (5, 20, 6), 500, 9, 2),                  # a row's workgroup is its router
    (32, (18, 20, 6), 40, CHUNK_ROWS + 900, 2), (4, (33, 20, 6), 300, CHUNK_ROWS + 4, 3),                 # one workgroup for 16 rows
    (4, (97, 20, 6), 1100, 5, 4), (32, (18, 400, 300, 6), 600, 5, 3), (4, (400, 20, 6), 300, 30, 8)])     # several, their lists merged
def test_logits_that_32_bits_cannot_tell_apart(bits, dims, g, n, k, unit):
    """A logit is a C + m r unit - a C + 1: C around 2^20 (cancels), r whole; all sums in between are whole multiples of the unit below
    2^23, so 64 bits are exact in any order.  In 32 bits the first term leaves nothing of r; with the smaller unit even the
    final values are equal.  Their differences are exact too, so prob is off by the rounding of a difference to 32
    bits (|d| U), expf (2 units in the last place, 4 U), that of the sum's terms on the average, the sum (4 U) and the
    division (2 U)."""
    rng = np.random.RandomState(g + n)
    s, _ = one_net(rng, g, dims, bits)
    ins = dims[0]
    at = (0, ins // 2, ins - 1)
    r = rng.permutation(2 ** 23)[:g] if unit > 2.0 ** -25 else np.arange(g)
    c = rng.randint(2 ** 20, 2 ** 21, g)
    rw, x = np.zeros((g, ins)), np.zeros((n, ins))
    rw[:, at[0]], rw[:, at[1]], rw[:, at[2]] = c, r, -c
    x[:, at[0]] = x[:, at[2]] = rng.randint(1, 4, n)
    x[:, at[1]] = rng.randint(1, 4, n) * unit
    assert all(np.array_equal(v.astype(np.float32), v) for v in (rw, x))
    _, idx, prob, _ = ask_mixture(s, x, rw.astype(np.float32), np.ones(g, np.float32), k)
    logits = x[:, [at[1]]] * r + 1
    want = np.argsort(-logits, 1, kind="stable")[:, :k]
    assert np.array_equal(idx, want)
    d = np.take_along_axis(logits, want, 1)
    d = d - d[:, :1]
    p = np.exp(d)
    p /= p.sum(1, keepdims=True)
    within(prob, p, p * sc.U * (np.abs(d) + (p * np.abs(d)).sum(1, keepdims=True) + 14) * 1.01 + 1e-37)
