"""Served snapshots over the sizes between which they change their way of working (ddrl_snap_*): odd k-steps and strips, routers
of every row length, few and very many places, skewed and padded batches, graphs of each, against the definition in 64-bit numpy."""
import numpy as np
import pytest
import torch

import snapshot_common as sc
import test_snapshot_gpu as base
from test_snapshot_gpu import DEV, HIDDEN, LAST, ask, ask_grad, ask_mixture, check_mixture, dev, make_flat, make_snap, within

pytestmark = pytest.mark.gpu


def one_net(rng, g, dims, bits, **kw):
    """g agents with one and the same net, loaded from one row -> snapshot, layers that look like g"""
    import ddrl_amd
    flat = make_flat(rng, 1, dims)
    s = ddrl_amd.PolicySnapshot.shaped(g, dims[0], dims[-1], dims[1:-1], HIDDEN, LAST, bits=bits)
    d = dev(flat)
    torch.cuda.synchronize()
    s.load_flat_dev(d.data_ptr(), 0)
    torch.cuda.synchronize()
    wide = lambda a: np.broadcast_to(a, (g,) + a.shape[1:])
    return s, [(wide(w), wide(b)) for w, b in sc.stored(sc.split_flat(flat, dims), bits)]


# ---- every agent's net ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("n", [1, 3, 16, 33])
@pytest.mark.parametrize("dims", [(31, 32, 33, 3), (64, 65, 96, 16), (97, 128, 129, 17), (40, 384, 260, 5), (7, 416, 353, 33), (18, 600, 500, 6), (15, 16, 48, 1)])
def test_forward_of_every_block(dims, n, bits):
    """layers whose k-steps and strips end everywhere in a block, nets that fit a workgroup's LDS and nets that do not"""
    rng = np.random.RandomState(n)
    flat = make_flat(rng, 3, dims)
    x = rng.uniform(-1, 1, (3, n, dims[0])).astype(np.float32)
    want, bound = sc.forward(sc.stored(sc.split_flat(flat, dims), bits), x, HIDDEN, LAST)
    within(ask(make_snap(flat, dims, bits), x), want, bound)


@pytest.mark.parametrize("bits", [32, 4])
def test_forward_of_very_many_rows(bits):
    """several tiles a workgroup"""
    dims, n = (5, 19, 2), 70001
    rng = np.random.RandomState(1)
    flat = make_flat(rng, 1, dims)
    x = rng.uniform(-1, 1, (1, n, 5)).astype(np.float32)
    want, bound = sc.forward(sc.stored(sc.split_flat(flat, dims), bits), x, HIDDEN, LAST)
    within(ask(make_snap(flat, dims, bits), x), want, bound)


# ---- the mixture of few places -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("g, ins, n, k", [(63, 1, 3, 2), (64, 2, 5, 3), (65, 3, 1, 4), (128, 4, 2, 5), (129, 5, 7, 1), (500, 15, 2, 6), (1000, 16, 3, 7), (1030, 17, 2, 8),
                                          (200, 31, 40, 2), (17, 33, 9, 8), (8, 1000, 3, 8), (1100, 97, 5, 4), (300, 400, 4, 2)])
def test_routers_of_every_length(g, ins, n, k, bits):
    """rows that end anywhere in a read of 4, agents that end anywhere in 64 and 16; small and large router matrices"""
    rng = np.random.RandomState(g + ins)
    s, layers = one_net(rng, g, (ins, 9, 3), bits)
    x = rng.uniform(-1, 1, (n, ins)).astype(np.float32)
    rw, rb = rng.standard_normal((g, ins)).astype(np.float32), rng.standard_normal(g).astype(np.float32)
    check_mixture(s, layers, x, rw, rb, k)
    allowed = rng.uniform(size=(n, g)) < 2.0 * k / g
    allowed[0] = False
    check_mixture(s, layers, x, rw, None, k, allowed)
    if ins <= 97:
        check_mixture(s, layers, x, np.zeros_like(rw), None, k, allowed)        # all equal: the lowest indices


@pytest.mark.parametrize("bits, dims, g, n, k", [(4, (18, 400, 300, 6), 600, 5, 8), (32, (18, 400, 300, 6), 300, 9, 2), (32, (18, 100, 100, 6), 600, 6, 8),
                                                 (4, (18, 100, 100, 6), 1500, 7, 8), (32, (18, 100, 100, 6), 40, 32, 8), (4, (30, 300, 290, 40), 20, 16, 5)])
def test_few_places_of_many_agents(bits, dims, g, n, k):
    """picks from several workgroups' lists; nets that fit together, one at a time or not at all; padded rows"""
    rng = np.random.RandomState(n)
    s, layers = one_net(rng, g, dims, bits)
    x = rng.uniform(-1, 1, (n, dims[0])).astype(np.float32)
    rw, rb = rng.standard_normal((g, dims[0])).astype(np.float32), rng.standard_normal(g).astype(np.float32)
    check_mixture(s, layers, x, rw, rb, k)
    allowed = rng.uniform(size=(n, g)) < 1.5 * k / g
    allowed[1] = False
    allowed[2] = False; allowed[2, g - 1] = True
    check_mixture(s, layers, x, rw, rb, k, allowed)
    a = ask_mixture(s, x, np.zeros_like(rw), None, k, allowed)
    assert (a[1][2] == [g - 1] + [-1] * (k - 1)).all()


def test_router_rows_that_hold_infinities_stay_apart():
    """what lies behind a router row's end, in the row after it, is never multiplied"""
    g, ins = 20, 18
    rng = np.random.RandomState(3)
    s, layers = one_net(rng, g, (ins, 9, 3), 4)
    x = rng.uniform(-1, 1, (4, ins)).astype(np.float32)
    rw = rng.standard_normal((g, ins)).astype(np.float32)
    wide = np.full((g, ins + 3), np.inf, np.float32)
    wide[:, :ins] = rw
    want = ask_mixture(s, x, rw, None, 3)
    xd, wd, out = dev(x), dev(wide), torch.zeros(4, 3, device=DEV)
    ws = torch.empty(s.mixture_workspace(4, 3), dtype=torch.uint8, device=DEV)
    s.mixture_dev(s.mixture_args(4, 3, xd.data_ptr(), wd.data_ptr(), out.data_ptr(), router_row=ins + 3, workspace=ws.data_ptr(), workspace_bytes=ws.numel()))
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want[0])
    # one router row for all agents, one state for all rows
    s.mixture_dev(s.mixture_args(4, 3, xd.data_ptr(), wd.data_ptr(), out.data_ptr(), router_row=0, x_row=0, workspace=ws.data_ptr(), workspace_bytes=ws.numel()))
    torch.cuda.synchronize()
    same = ask_mixture(s, np.tile(x[:1], (4, 1)), np.tile(rw[:1], (g, 1)), None, 3)
    assert np.array_equal(out.cpu().numpy(), same[0]) and (same[1] == np.arange(3)).all()


# ---- the mixture of many places, its gradient ----------------------------------------------------------------------------

def wide_mixture(layers, x, rw, rb, k):
    """the definition at once for all rows, every agent answering every row: -> out, bound, idx, prob, y, y's bound"""
    logits = x.astype(np.float64) @ rw.astype(np.float64).T + rb
    idx = np.argsort(-logits, 1, kind="stable")[:, :k]
    l = np.take_along_axis(logits, idx, 1)
    p = np.exp(l - l[:, :1])
    p /= p.sum(1, keepdims=True)
    y, e = sc.forward(layers, np.broadcast_to(x, (rw.shape[0],) + x.shape), HIDDEN, LAST)
    at = np.arange(x.shape[0])[:, None]
    y, e = y[idx, at], e[idx, at]
    pe = (8 + 176 + k + 1) * sc.U                                 # as in snapshot_common.mixture
    return (p[..., None] * y).sum(1), (p[..., None] * (e + (pe + (k + 1) * sc.U) * (np.abs(y) + e))).sum(1) + 1e-37, idx, p, y, e


def wide_gradient(x, idx, prob, y, dout, g):
    """snapshot_common.mixture_grad without a loop over rows"""
    x, prob, y, dout = (np.asarray(v, np.float64) for v in (x, prob, y, dout))
    n, k, a = y.shape
    ok = (idx >= 0) & (idx < g)
    p = np.where(ok, prob, 0.0)
    score, mag = (y * dout[:, None]).sum(-1), (np.abs(y) * np.abs(dout[:, None])).sum(-1)
    dl = p * (score - (p * score).sum(1, keepdims=True))
    dle = (a + k + 4) * sc.U * np.abs(p) * (mag + (np.abs(p) * mag).sum(1, keepdims=True))
    dw, db, dwe, dbe = (np.zeros((g, x.shape[1])), np.zeros(g), np.zeros((g, x.shape[1])), np.zeros(g))
    for e in range(g):
        t, j = np.nonzero(idx == e)
        dw[e], db[e], dwe[e], dbe[e] = dl[t, j] @ x[t], dl[t, j].sum(), dle[t, j] @ np.abs(x[t]), dle[t, j].sum()
    return dw, db, p[..., None] * dout[:, None], dwe + 2 * sc.U * np.abs(dw) + 1e-37, dbe + 2 * sc.U * np.abs(db) + 1e-37


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("dims, g, n, k, skew", [((18, 20, 6), 12, 4200, 2, 0), ((18, 20, 6), 12, 4200, 2, 9), ((18, 33, 17), 70, 2048, 4, 1), ((3, 9, 2), 5, 33000, 2, 1),
                                                 ((18, 400, 300, 6), 4, 4100, 2, 0), ((18, 600, 500, 6), 3, 300, 1, 3), ((9, 1024, 5), 3, 140, 2, 0), ((2, 1), 1, 9000, 1, 0), ((40, 1024, 1024, 2), 2, 150, 2, 0)])
def test_many_places(bits, dims, g, n, k, skew):
    """tiles of 16 and 32 rows, up to a router that sends (nearly) everything to few agents, more than 64 sorted blocks"""
    rng = np.random.RandomState(g)
    flat = make_flat(rng, g, dims)
    s, layers = make_snap(flat, dims, bits), sc.stored(sc.split_flat(flat, dims), bits)
    x = rng.uniform(-1, 1, (n, dims[0])).astype(np.float32)
    rw, rb = rng.standard_normal((g, dims[0])).astype(np.float32), (rng.standard_normal(g) * skew).astype(np.float32)
    out, idx, prob, y = ask_mixture(s, x, rw, rb, k)
    wo, wb, wi, wp, wy, ye = wide_mixture(layers, x, rw, rb, k)
    assert np.array_equal(idx, wi) and np.abs(prob - wp).max() <= 200 * sc.U
    within(out, wo, wb)
    within(y, wy, ye)
    again = ask_mixture(s, x, rw, rb, k)
    assert all(np.array_equal(a, b) for a, b in zip((out, idx, prob, y), again))
    dout = rng.standard_normal((n, dims[-1])).astype(np.float32)
    dw, db, dy = ask_grad(s, x, idx, prob, y, dout)
    ww, wd, wy, bw, bd = wide_gradient(x, idx, prob, y, dout, g)
    within(dw, ww, bw)
    within(db, wd, bd)
    within(dy, wy, 2 * sc.U * np.abs(wy) + 1e-37)


@pytest.mark.parametrize("g, n, k, ins, outs", [(3, 140000, 2, 2, 1), (1, 300000, 1, 1, 1), (20, 1024, 1, 300, 3), (700, 1500, 3, 18, 6), (2, 600, 2, 1024, 2), (1023, 5000, 8, 5, 2)])
def test_gradient_of_many_places(g, n, k, ins, outs):
    """several workgroups an agent, more than 256 sorted blocks, places nobody has, one agent twice in a row, rows apart"""
    import ddrl_amd
    rng = np.random.RandomState(n)
    s = ddrl_amd.PolicySnapshot.shaped(g, ins, outs, [], bits=32)
    x, y, dout = (v.astype(np.float32) for v in (rng.uniform(-1, 1, (n, ins)), rng.standard_normal((n, k, outs)), rng.standard_normal((n, outs))))
    idx, prob = rng.randint(-1, g + 1, (n, k)), rng.dirichlet(np.ones(k), n).astype(np.float32)
    idx[5] = g - 1; idx[6] = -1; idx[7] = 2 ** 31 - 1; idx[8] = -2 ** 31
    dw, db, dy = ask_grad(s, x, idx, prob, y, dout)
    ww, wd, wy, bw, bd = wide_gradient(x, idx, prob, y, dout, g)
    within(dw, ww, bw)
    within(db, wd, bd)
    within(dy, wy, 2 * sc.U * np.abs(wy) + 1e-37)
    t = [dev(v) for v in (x, idx.astype(np.int32), prob, y, dout)]
    wide, ws = torch.full((g, ins + 2), 77.0, device=DEV), torch.full((max(1, s.mixture_grad_workspace(n, k)),), 0xCD, dtype=torch.uint8, device=DEV)
    s.mixture_grad_dev(s.mixture_grad_args(n, k, *(v.data_ptr() for v in t), wide.data_ptr() + 4, d_router_row=ins + 2, workspace=ws.data_ptr(), workspace_bytes=ws.numel()))
    torch.cuda.synchronize()
    got = wide.cpu().numpy()
    assert np.array_equal(got[:, 1:-1], dw) and (got[:, [0, -1]] == 77).all()


def test_as_many_agents_as_are_sorted():
    import ddrl_amd
    g, n, k = 16383, 200, 2
    rng = np.random.RandomState(5)
    s, layers = one_net(rng, g, (2, 1), 32)
    x = rng.uniform(-1, 1, (n, 2)).astype(np.float32)
    rw = rng.standard_normal((g, 2)).astype(np.float32)
    out, idx, prob, y = ask_mixture(s, x, rw, np.zeros(g, np.float32), k)
    logits = x.astype(np.float64) @ rw.astype(np.float64).T
    wi = np.argsort(-logits, 1, kind="stable")[:, :k]
    assert np.array_equal(idx, wi)
    v, b = sc.forward([(w[:1], bb[:1]) for w, bb in layers], x[None], HIDDEN, LAST)
    within(y, np.broadcast_to(v[0][:, None], y.shape), np.broadcast_to(b[0][:, None], y.shape))
    dout = np.ones((n, 1), np.float32)
    r = 4                                                         # (the same rows four times: enough places for the sort)
    rep = lambda v: np.concatenate([v] * r)
    dw, db, _ = ask_grad(s, rep(x), rep(idx), rep(prob), rep(y), rep(dout))
    touched = np.unique(idx)
    rest = np.setdiff1d(np.arange(g), touched)
    ww, wd, _, bw, bd = sc.mixture_grad(rep(x), rep(idx), rep(prob), rep(y), rep(dout), g)
    within(dw, ww, bw)
    within(db, wd, bd)
    assert (dw[rest] == 0).all() and (db[rest] == 0).all()
    big = ddrl_amd.PolicySnapshot.shaped(g + 1, 2, 1, [], bits=32)
    with pytest.raises(ddrl_amd.DdrlError, match="16383"):
        big.mixture_workspace(n, k)
    with pytest.raises(ddrl_amd.DdrlError, match="16383"):
        big.mixture_grad_workspace(n, k)
    assert big.mixture_workspace(100, k) > 0


def test_too_many_rows_are_refused():
    import ddrl_amd
    s = ddrl_amd.PolicySnapshot.shaped(1, 1, 1, [], bits=4)
    p = dev(np.zeros(4, np.float32)).data_ptr()
    for n in (2 ** 28 + 1, 2 ** 31 - 1):
        with pytest.raises(ddrl_amd.DdrlError):
            s.forward_dev(s.forward_args(n, p, p))
        with pytest.raises(ddrl_amd.DdrlError):
            s.mixture_workspace(n, 1)
        with pytest.raises(ddrl_amd.DdrlError):
            s.mixture_grad_workspace(n, 1)


@pytest.mark.parametrize("bits, dims, g, n, k", [(4, (18, 20, 6), 10, 4096, 2), (4, (18, 20, 6), 10, 4097, 2), (32, (18, 100, 100, 6), 9, 512, 2), (32, (18, 100, 100, 6), 9, 513, 2),
                                                 (4, (18, 64, 64, 6), 64, 512, 8), (4, (18, 64, 64, 6), 64, 513, 8), (4, (130, 40, 6), 800, 600, 2), (4, (18, 33, 5), 1024, 512, 1)])
def test_rows_where_the_mixture_changes_its_way(bits, dims, g, n, k):
    rng = np.random.RandomState(g)
    s, layers = one_net(rng, g, dims, bits)
    x = rng.uniform(-1, 1, (n, dims[0])).astype(np.float32)
    rw, rb = rng.standard_normal((g, dims[0])).astype(np.float32), rng.standard_normal(g).astype(np.float32)
    allowed = rng.uniform(size=(n, g)) < 0.7
    allowed[::7] = False
    allowed[1::7] = False
    allowed[1::7, g // 2] = True
    out, idx, prob, y = ask_mixture(s, x, rw, rb, k, allowed)
    logits = np.where(allowed, x.astype(np.float64) @ rw.astype(np.float64).T + rb, -np.inf)
    wi = np.argsort(-logits, 1, kind="stable")[:, :k]
    l = np.take_along_axis(logits, wi, 1)
    have = np.isfinite(l)
    p = np.where(have, np.exp(l - np.where(have[:, :1], l[:, :1], 0)), 0)
    p = p / np.maximum(p.sum(1, keepdims=True), 1e-300)
    assert np.array_equal(idx, np.where(have, wi, -1)) and np.abs(prob - p).max() <= 200 * sc.U
    v, e = sc.forward([(w[:1], b[:1]) for w, b in layers], x[None], HIDDEN, LAST)       # all nets are one
    v, e = np.where(have[..., None], v[0][:, None], 0), np.where(have[..., None], e[0][:, None], 0)
    within(y, v, e + 1e-37)
    pe = (8 + 176 + k + 1) * sc.U                                 # as in snapshot_common.mixture
    within(out, (p[..., None] * v).sum(1), (p[..., None] * (e + (pe + (k + 1) * sc.U) * (np.abs(v) + e))).sum(1) + 1e-37)
    again = ask_mixture(s, x, rw, rb, k, allowed)
    assert all(np.array_equal(a, b) for a, b in zip((out, idx, prob, y), again))


# ---- graphs and streams of each way of working ---------------------------------------------------------------------------

@pytest.mark.parametrize("bits, dims, g, n, k", [(4, (18, 400, 300, 6), 300, 6, 8), (32, (18, 400, 300, 6), 7, 10, 2), (32, (97, 40, 6), 1100, 5, 3), (4, (18, 33, 6), 9, 4200, 2),
                                                 (32, (18, 33, 6), 9, 4200, 2), (4, (18, 40, 6), 60, 20, 5)])
def test_graphs_of_each(bits, dims, g, n, k):
    """as test_graphs: two graphs with workspaces of their own, replayed between eager calls and new inputs"""
    rng = np.random.RandomState(61)
    s = one_net(rng, g, dims, bits)[0]
    made = [base._calls(s, n, k, seed) for seed in (1, 2)]
    graphs = []
    for st, run, _ in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append(graph)
    for rep in range(4):
        for st, _, _ in made:
            st["x"].copy_(torch.from_numpy(np.random.RandomState(70 + rep).uniform(-1, 1, st["x"].shape).astype(np.float32)))
        want = []
        for st, run, results in made:
            run()
            torch.cuda.synchronize()
            want.append(results())
            for key in ("f", "out", "y", "dw"):
                st[key].zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (st, run, results), w in zip(made, want):
            assert all(np.array_equal(a, b) for a, b in zip(results(), w))


@pytest.mark.parametrize("n", [6, 300])
def test_calls_at_once(n):
    """eight mixtures of one snapshot in flight on eight streams, each with its workspace, give the bits of one after the other"""
    s = one_net(np.random.RandomState(62), 40, (18, 400, 300, 6), 4)[0]
    made = [base._calls(s, n, 3, seed) for seed in range(8)]
    want = []
    for st, run, results in made:
        run()
        torch.cuda.synchronize()
        want.append(results())
        for key in ("f", "out", "y", "dw"):
            st[key].zero_()
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for rep in range(3):
        for q, (st, run, _) in zip(streams, made):
            with torch.cuda.stream(q):
                run()
    torch.cuda.synchronize()
    for (st, run, results), w in zip(made, want):
        assert all(np.array_equal(a, b) for a, b in zip(results(), w))


# ---- what is left --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 4])
def test_an_empty_snapshot_answers_what_zero_weights_answer(bits):
    import ddrl_amd
    for dims, n in (((18, 20, 6), 1), ((18, 20, 6), 3), ((18, 400, 300, 6), 17)):
        s = ddrl_amd.PolicySnapshot.shaped(4, dims[0], dims[-1], dims[1:-1], bits=bits)
        x = np.random.RandomState(1).uniform(-1, 1, (4, n, dims[0]))
        assert (ask(s, x) == 0).all() and (s.weights() == 0).all()
        out, idx, prob, _ = ask_mixture(s, x[0], np.zeros((4, dims[0]), np.float32), None, 3)
        assert (out == 0).all() and (idx == [0, 1, 2]).all() and np.abs(prob - 1 / 3).max() <= sc.U


@pytest.mark.parametrize("n", [3, 400])
def test_logits_that_are_infinite(n):
    """an infinite logit comes first; the softmax over it is what the formula gives, not a number"""
    g, k = 30, 3
    rng = np.random.RandomState(4)
    s, layers = one_net(rng, g, (5, 9, 2), 32)
    x = rng.uniform(0.5, 1, (n, 5)).astype(np.float32)
    rw, rb = rng.standard_normal((g, 5)).astype(np.float32), rng.standard_normal(g).astype(np.float32)
    rb[[7, 22]] = np.inf
    out, idx, prob, y = ask_mixture(s, x, rw, rb, k)
    assert (idx[:, :2] == [7, 22]).all() and np.isnan(prob).all() and np.isnan(out).all() and np.isfinite(y).all()
    allowed = np.ones(g); allowed[[7, 22]] = 0
    check_mixture(s, layers, x[:40], rw, rb, k, allowed)
    rb[[7, 22]] = np.nan                                              # barred: whatever its logit is
    check_mixture(s, layers, x[:40], rw, np.where(np.isnan(rb), -np.inf, rb).astype(np.float32), k)
    a = ask_mixture(s, x, rw, rb, k, allowed)
    b = ask_mixture(s, x, rw, np.where(np.isnan(rb), 0, rb).astype(np.float32), k, allowed)
    assert all(np.array_equal(u, v) for u, v in zip(a, b))


def test_rows_that_overlap_in_memory():
    """inputs may: a sliding window over one series"""
    s, layers = one_net(np.random.RandomState(5), 3, (18, 20, 6), 4)
    series = np.random.RandomState(6).uniform(-1, 1, 50).astype(np.float32)
    xd, out = dev(series), torch.zeros(3, 33, 6, device=DEV)
    s.forward_dev(s.forward_args(33, xd.data_ptr(), out.data_ptr(), x_agent=0, x_row=1))
    torch.cuda.synchronize()
    x = np.lib.stride_tricks.sliding_window_view(series, 18)
    want, bound = sc.forward(layers, np.broadcast_to(x, (3,) + x.shape), HIDDEN, LAST)
    within(out.cpu().numpy(), want, bound)


def test_as_many_rows_as_are_served():
    """2^28 places, in the mixture and in the gradient: more threads than one launch takes.  Small whole numbers, so that every
    answer and every sum of 64 bits is exact."""
    import ddrl_amd
    n = 2 ** 28
    s = ddrl_amd.PolicySnapshot.shaped(2, 1, 1, [], 0, 0, bits=32)
    flat = dev(np.array([[3, 1], [-2, 5]], np.float32))               # weight, bias
    torch.cuda.synchronize()
    s.load_flat_dev(flat.data_ptr(), 2)
    gen = torch.Generator(DEV).manual_seed(1)
    small = lambda: torch.randint(-3, 4, (n,), generator=gen, device=DEV, dtype=torch.int8).float()
    x, rw, rb = small(), dev(np.array([[1], [-1]], np.float32)), dev(np.array([1, 0], np.float32))
    out, prob, y = (torch.full((n,), 77.0, device=DEV) for _ in range(3))
    idx = torch.full((n,), 77, dtype=torch.int32, device=DEV)
    ws = torch.empty(s.mixture_workspace(n, 1), dtype=torch.uint8, device=DEV)
    q = torch.cuda.current_stream().cuda_stream
    s.mixture_dev(s.mixture_args(n, 1, x.data_ptr(), rw.data_ptr(), out.data_ptr(), router_b=rb.data_ptr(), idx=idx.data_ptr(), prob=prob.data_ptr(), y=y.data_ptr(),
                                 workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=q))
    torch.cuda.synchronize()
    first = x + 1 >= -x
    want = torch.where(first, 3 * x + 1, -2 * x + 5)
    assert bool((idx == torch.where(first, 0, 1)).all()) and bool((prob == 1).all())
    assert bool((y == want).all()) and bool((out == want).all())
    del ws, out, want, first
    dout = small()
    prob.fill_(0.5)
    dw, db, dy = torch.zeros(2, device=DEV), torch.zeros(2, device=DEV), torch.full((n,), 77.0, device=DEV)
    ws = torch.empty(s.mixture_grad_workspace(n, 1), dtype=torch.uint8, device=DEV)
    s.mixture_grad_dev(s.mixture_grad_args(n, 1, x.data_ptr(), idx.data_ptr(), prob.data_ptr(), y.data_ptr(), dout.data_ptr(), dw.data_ptr(), db.data_ptr(), dy.data_ptr(),
                                           workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=q))
    torch.cuda.synchronize()
    assert bool((dy == 0.5 * dout).all())
    for e in range(2):
        dl = torch.where(idx == e, 0.25 * (y * dout), 0)              # .5 (s - .5 s)
        assert dw[e].item() == np.float32((dl * x).sum(dtype=torch.float64).item())
        assert db[e].item() == np.float32(dl.sum(dtype=torch.float64).item())


def test_as_many_agents_as_there_may_be():
    """2^22 - 1 agents, asked in every way"""
    import ddrl_amd
    g, k = 2 ** 22 - 1, 2
    s = ddrl_amd.PolicySnapshot.shaped(g, 1, 1, [], 0, 0, bits=4)
    gen = torch.Generator(DEV).manual_seed(2)
    flat = torch.stack((torch.tensor([.5, 1., 1.5, 2., 3., 4., 6.], device=DEV)[torch.randint(0, 7, (g,), generator=gen, device=DEV)],
                        torch.randint(-9, 10, (g,), generator=gen, device=DEV).float()), 1).contiguous()
    torch.cuda.synchronize()
    s.load_flat_dev(flat.data_ptr(), 2)
    x = torch.randint(-3, 4, (g, 1, 1), generator=gen, device=DEV, dtype=torch.int8).float()
    out = torch.full((g, 1, 1), 77.0, device=DEV)
    q = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    s.forward_dev(s.forward_args(1, x.data_ptr(), out.data_ptr(), stream=q))
    assert bool((out[:, 0, 0] == flat[:, 0] * x[:, 0, 0] + flat[:, 1]).all())
    rw = torch.zeros(g, 1, device=DEV)
    rw[[5, g - 1], 0] = torch.tensor([1., 2.], device=DEV)
    one = np.ones((1, 1), np.float32)
    got, idx, prob, y = ask_mixture(s, one, rw.cpu().numpy(), None, k)
    assert idx.tolist() == [[g - 1, 5]] and np.array_equal(y[0, :, 0], flat[[g - 1, 5]].sum(1).cpu().numpy())
    dw, db, _ = ask_grad(s, one, idx, np.array([[.5, .5]]), np.array([[[4.], [2.]]]), one)
    want = np.zeros((g, 1), np.float32)
    want[[g - 1, 5], 0] = .5, -.5                                     # .5 (4 - 3), .5 (2 - 3)
    assert np.array_equal(dw, want) and np.array_equal(db, want[:, 0])


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("n", [1, 3, 20])
def test_one_row_an_agent_packed(n, bits):
    """x_row = 0 with the agents' rows packed: agent g reads row g; out_row = 0 for a single row likewise"""
    dims, g = (18, 33, 5), 4
    rng = np.random.RandomState(n)
    flat = make_flat(rng, g, dims)
    s = make_snap(flat, dims, bits)
    x = rng.uniform(-1, 1, (g, 1, 18)).astype(np.float32)
    want, bound = sc.forward(sc.stored(sc.split_flat(flat, dims), bits), np.broadcast_to(x, (g, n, 18)), HIDDEN, LAST)
    xd, out = dev(x), torch.full((g, n, 5), 77.0, device=DEV)
    torch.cuda.synchronize()
    s.forward_dev(s.forward_args(n, xd.data_ptr(), out.data_ptr(), x_row=0, out_row=0 if n == 1 else None))
    torch.cuda.synchronize()
    within(out.cpu().numpy(), want, bound)
    xd = dev(rng.uniform(-1, 1, (1, 18)).astype(np.float32))              # one row for all agents
    torch.cuda.synchronize()
    s.forward_dev(s.forward_args(n, xd.data_ptr(), out.data_ptr(), x_agent=0, x_row=0))
    torch.cuda.synchronize()
    want, bound = sc.forward(sc.stored(sc.split_flat(flat, dims), bits), np.broadcast_to(xd.cpu().numpy(), (g, n, 18)), HIDDEN, LAST)
    within(out.cpu().numpy(), want, bound)


def test_the_host_form_refuses_before_it_reads():
    s = make_snap(make_flat(np.random.RandomState(1), 2, (3, 2)), (3, 2), 4)
    two = np.zeros(12, np.float32)
    for n in (-1, 2 ** 28 + 1, 2 ** 31 - 1):
        assert s.L.ddrl_snap_forward(s.h, n, two.ctypes.data, two.ctypes.data) == -1
        assert ("n=%d" % n).encode() in s.L.ddrl_last_error()
        assert s.L.ddrl_snap_mixture(s.h, n, 1, two.ctypes.data, two.ctypes.data, None, None, two.ctypes.data, None, None) == -1
    assert s.L.ddrl_snap_forward(s.h, 1, None, two.ctypes.data) == -1 and s.L.ddrl_snap_forward(s.h, 0, None, None) == 0


def test_strides_and_masks_over_several_launches():
    """more rows than one launch of the router takes: where a later launch starts, every array's rows are the ones a small call of
    the same rows answers; sums are exact (small whole numbers, prob = .5)"""
    import ddrl_amd
    n, k = 2 ** 26 + 5000, 2
    s = ddrl_amd.PolicySnapshot.shaped(3, 1, 1, [], 0, 0, bits=32)
    flat = dev(np.array([[3, 1], [-2, 5], [1, -4]], np.float32))
    torch.cuda.synchronize()
    s.load_flat_dev(flat.data_ptr(), 2)
    gen = torch.Generator(DEV).manual_seed(3)
    small = lambda *shape: torch.randint(-3, 4, shape, generator=gen, device=DEV, dtype=torch.int8).float()
    x, dout = small(n, 2), small(n, 3)
    allowed = (torch.rand(n, 4, generator=gen, device=DEV) < 0.6).to(torch.uint8)
    rw, rb = dev(np.array([[1], [-1], [2]], np.float32)), dev(np.array([1, 0, -1], np.float32))
    q = torch.cuda.current_stream().cuda_stream

    def ask_rows(a, b):
        m = b - a
        out, prob, y = torch.full((m, 2), 77.0, device=DEV), torch.full((m, k), 77.0, device=DEV), torch.full((m, k), 77.0, device=DEV)
        idx, ws = torch.full((m, k), 77, dtype=torch.int32, device=DEV), torch.empty(s.mixture_workspace(m, k), dtype=torch.uint8, device=DEV)
        s.mixture_dev(s.mixture_args(m, k, x[a:].data_ptr() + 4, rw.data_ptr(), out.data_ptr(), router_b=rb.data_ptr(), allowed=allowed[a:].data_ptr() + 1, idx=idx.data_ptr(),
                                     prob=prob.data_ptr(), y=y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(), x_row=2, allowed_row=4, out_row=2, stream=q))
        torch.cuda.synchronize()
        return out, idx, prob, y

    whole = ask_rows(0, n)
    assert bool((whole[0][:, 1] == 77).all())
    for a, b in ((0, 700), (2 ** 25 - 300, 2 ** 25 + 300), (2 ** 26 - 300, 2 ** 26 + 300), (n - 900, n)):
        assert all(torch.equal(u[a:b], v) for u, v in zip(whole, ask_rows(a, b)))
    _, idx, prob, y = whole
    assert bool((idx[:, 0] < 0).any()) and bool((idx[2 ** 26:, 1] >= 0).any())
    prob.fill_(0.5)
    dw, db, dy = torch.zeros(3, device=DEV), torch.zeros(3, device=DEV), torch.full((n, k), 77.0, device=DEV)
    ws = torch.empty(s.mixture_grad_workspace(n, k), dtype=torch.uint8, device=DEV)
    s.mixture_grad_dev(s.mixture_grad_args(n, k, x.data_ptr() + 4, idx.data_ptr(), prob.data_ptr(), y.data_ptr(), dout.data_ptr() + 8, dw.data_ptr(), db.data_ptr(), dy.data_ptr(),
                                           x_row=2, dout_row=3, workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=q))
    torch.cuda.synchronize()
    have = idx >= 0
    assert torch.equal(dy, torch.where(have, 0.5 * dout[:, 2:], 0.0))
    score = torch.where(have, y * dout[:, 2:], 0.0)
    dl = torch.where(have, 0.5 * (score - 0.5 * score.sum(1, keepdim=True)), 0.0)
    for e in range(3):
        mine = torch.where(idx == e, dl, 0.0).sum(1, dtype=torch.float64)
        assert dw[e].item() == np.float32((mine * x[:, 1]).sum().item()) and db[e].item() == np.float32(mine.sum().item())
