"""Served snapshots on the GPU (ddrl_snap_*), against the definition in 64-bit numpy (snapshot_common.py)."""
import numpy as np
import pytest
import torch

import snapshot_common as sc

pytestmark = pytest.mark.gpu

DEV = "cuda"
HIDDEN, LAST = 1, 2


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def make_flat(rng, g, dims, scale=1.0):
    parts = []
    for i, o in zip(dims, dims[1:]):
        parts += [rng.standard_normal((g, i * o)) * scale * 1.5 / np.sqrt(i), rng.standard_normal((g, o)) * 0.1]
    return np.concatenate(parts, 1).astype(np.float32)


def make_snap(flat, dims, bits, hidden=HIDDEN, last=LAST):
    import ddrl_amd
    s = ddrl_amd.PolicySnapshot.shaped(flat.shape[0], dims[0], dims[-1], dims[1:-1], hidden, last, bits=bits)
    d = dev(flat)
    torch.cuda.synchronize()
    s.load_flat_dev(d.data_ptr(), flat.shape[1])
    torch.cuda.synchronize()
    return s


def ask(s, x, out=None, **kw):
    """x [G, n, in] or [n, in] (shared), numpy -> [G, n, out]"""
    n = x.shape[-2]
    xd = dev(x.astype(np.float32))
    out = torch.full((s.G, n, s.out_dim), 77.0, device=DEV) if out is None else out
    a = s.forward_args(n, xd.data_ptr(), out.data_ptr(), x_agent=0 if x.ndim == 2 else None, stream=torch.cuda.current_stream().cuda_stream, **kw)
    s.forward_dev(a)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def within(got, want, bound):
    bad = ~(np.abs(got.astype(np.float64) - want) <= bound)
    assert not bad.any(), "%d of %d values off, worst %.3g of its bound" % (bad.sum(), bad.size, np.max(np.abs(got - want) / bound))


# ---- what is stored ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dims", [(1, 1), (18, 20, 6), (3, 33, 17, 5), (32, 64, 1), (45, 64, 64, 17), (129, 100, 31, 47, 2)])
@pytest.mark.parametrize("bits", [32, 4])
def test_stored_weights(dims, bits):
    rng = np.random.RandomState(1)
    flat = make_flat(rng, 5, dims)
    got = make_snap(flat, dims, bits).weights()
    want = np.concatenate([v.reshape(5, -1) for layer in sc.stored(sc.split_flat(flat, dims), bits) for v in layer], 1)
    assert np.array_equal(got, want)


def test_stored_weights_of_odd_blocks():
    """zeros, halves, a block's largest on the border of a scale, tiny blocks; one row for every agent (ld = 0)"""
    dims = (70, 9)
    flat = np.zeros((1, sc.n_params(dims)), np.float32)
    w = flat[:, :630].reshape(9, 70)
    rng = np.random.RandomState(2)
    w[1] = rng.choice([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6], 70) * rng.choice([-1, 1], 70)
    w[2] = rng.standard_normal(70) * 2.0 ** -119 / 4
    w[3] = np.float32(6) * 2.0 ** rng.randint(-20, 20, 70)
    w[4, :] = np.nextafter(np.float32(6), np.float32(7)) * np.sign(rng.standard_normal(70))
    w[5, 0] = 1
    w[6, 69] = -1
    w[7] = rng.standard_normal(70) * 2.0 ** 115
    w[8] = rng.uniform(2.0 ** -118, 2.0 ** -117, 70)
    import ddrl_amd
    s = ddrl_amd.PolicySnapshot.shaped(3, 70, 9, [], 0, 0, bits=4)
    d = dev(flat)
    torch.cuda.synchronize()
    s.load_flat_dev(d.data_ptr(), 0)
    want = np.concatenate([sc.round4(w).reshape(-1), flat[0, 630:]])
    for row in s.weights():
        assert np.array_equal(row, want)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 2.0 ** 126])
def test_a_wild_weight_answers_nan(value):
    """... for its output alone, in a net of one layer"""
    dims = (40, 19)
    flat = make_flat(np.random.RandomState(3), 2, dims)
    flat[1, 7 * 40 + 33] = value
    x = np.random.RandomState(4).uniform(-1, 1, (2, 3, 40))
    got = ask(make_snap(flat, dims, 4, 0, 0), x)
    layers = sc.stored(sc.split_flat(make_flat(np.random.RandomState(3), 2, dims), dims), 4)
    want, bound = sc.forward(layers, x.astype(np.float32), 0, 0)
    assert np.isnan(got[1, :, 7]).all()
    keep = np.ones(19, bool); keep[7] = False
    within(got[:, :, keep], want[:, :, keep], bound[:, :, keep])


@pytest.mark.parametrize("bits", [32, 4])
def test_snapshot_of_a_population(bits):
    """created from and loaded again from live nets, actor and critic; the population goes on meanwhile"""
    import ddrl_amd
    pop = ddrl_amd.PolicyPopulation(3, 18, 6, (20, 33), init_seed=5)
    s = ddrl_amd.PolicySnapshot(pop, 0, bits)
    assert (s.G, s.in_dim, s.out_dim, s.bits, s.n_params) == (3, 18, 6, bits, pop.num_params(0))
    dims = (18, 20, 33, 6)
    for seed in (1, 2):
        layers = sc.stored(sc.split_flat(pop.weights(0).astype(np.float32), dims), bits)
        assert np.array_equal(s.weights(), np.concatenate([v.reshape(3, -1) for layer in layers for v in layer], 1))
        pop.set_weights(0, make_flat(np.random.RandomState(seed), 3, dims))
        s.load(pop)
        pop.set_weights(0, pop.weights(0) * 0.5)
        s.load(pop)
    x = np.random.RandomState(6).uniform(-1, 1, (3, 18)).astype(np.float32)
    got = s.forward(x[:, None])[:, 0]
    want, bound = sc.forward(layers_now(pop, dims, bits), x[:, None], 1, 2)
    within(got, want[:, 0], bound[:, 0])
    if bits == 32:
        within(pop.infer(x), want[:, 0], bound[:, 0])


def layers_now(pop, dims, bits):
    return sc.stored(sc.split_flat(pop.weights(0).astype(np.float32), dims), bits)


def test_snapshot_of_a_learning_population():
    """every net of a DDPG population, between updates"""
    import ddrl_amd
    cfg = ddrl_amd.DdpgConfig(n_agents=2, nb_sensors=5, nb_motors=2, mini_batch_size=16, replay_memory=300, hidden_unit_a=(20,), hidden_unit_q=(30, 7))
    pop = ddrl_amd.DdpgPopulation(cfg, init_seed=1)
    rng = np.random.RandomState(0)
    pop.seed_replay([1, 2])
    for g in range(2):
        pop.replay_load(g, rng.uniform(-1, 1, (300, 14)).astype(np.float32))
    shapes = {0: (5, 20, 2), 1: (7, 30, 7, 1), 2: (5, 20, 2), 3: (7, 30, 7, 1)}
    snaps = {net: ddrl_amd.PolicySnapshot(pop, net, 32) for net in shapes}
    for _ in range(3):
        pop.update()
        for net, s in snaps.items():
            s.load(pop, net)
        for net, s in snaps.items():
            assert np.array_equal(s.weights(), pop.weights(net))
            x = rng.uniform(-1, 1, (2, 4, shapes[net][0])).astype(np.float32)
            want, bound = sc.forward(sc.split_flat(pop.weights(net), shapes[net]), x, cfg.get("hidden_layer_type"), cfg.get("actor_output_layer_type") if net in (0, 2) else 0)
            within(s.forward(x), want, bound)
            within(pop.forward_batch(net, x), want, bound)


# ---- every agent's net ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("n", [1, 2, 5, 6, 16, 17, 64, 131])
@pytest.mark.parametrize("dims", [(18, 20, 6), (3, 33, 17, 5), (45, 64, 64, 17), (129, 100, 31, 47, 2)])
def test_forward(dims, n, bits):
    rng = np.random.RandomState(n)
    flat = make_flat(rng, 5, dims)
    x = rng.uniform(-1, 1, (5, n, dims[0])).astype(np.float32)
    hidden, last = [(1, 2), (2, 0), (3, 1), (0, 3)][n % 4]
    want, bound = sc.forward(sc.stored(sc.split_flat(flat, dims), bits), x, hidden, last)
    within(ask(make_snap(flat, dims, bits, hidden, last), x), want, bound)


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("dims, n", [((1, 1), 3), ((2, 1), 1), ((18, 400, 300, 6), 1), ((18, 400, 300, 6), 40), ((1024, 1024, 1024, 1024), 1),
                                     ((1024, 1024, 1024, 1024), 21), ((7, 1024, 3, 1024, 1), 6), ((500, 16, 1000, 16), 33)])
def test_forward_of_odd_nets(dims, n, bits):
    rng = np.random.RandomState(11)
    flat = make_flat(rng, 2, dims)
    x = rng.uniform(-1, 1, (2, n, dims[0])).astype(np.float32)
    want, bound = sc.forward(sc.stored(sc.split_flat(flat, dims), bits), x, HIDDEN, LAST)
    within(ask(make_snap(flat, dims, bits), x), want, bound)


@pytest.mark.parametrize("bits", [32, 4])
def test_forward_of_many_agents(bits):
    dims, g = (18, 20, 6), 1500
    rng = np.random.RandomState(12)
    flat = make_flat(rng, g, dims)
    s = make_snap(flat, dims, bits)
    layers = sc.stored(sc.split_flat(flat, dims), bits)
    for n in (1, 30):
        x = rng.uniform(-1, 1, (g, n, 18)).astype(np.float32)
        want, bound = sc.forward(layers, x, HIDDEN, LAST)
        within(ask(s, x), want, bound)


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("n", [1, 4, 19])
def test_forward_strides_and_masks(n, bits):
    dims, g = (18, 33, 5), 6
    rng = np.random.RandomState(13)
    flat = make_flat(rng, g, dims)
    s = make_snap(flat, dims, bits)
    layers = sc.stored(sc.split_flat(flat, dims), bits)
    x = rng.uniform(-1, 1, (n, 18)).astype(np.float32)
    want, bound = sc.forward(layers, np.broadcast_to(x, (g, n, 18)), HIDDEN, LAST)
    within(ask(s, x), want, bound)                                              # the same rows for all
    one = rng.uniform(-1, 1, (g, 1, 18)).astype(np.float32)                     # one row again and again
    xd, out = dev(one), torch.zeros(g, n, 5, device=DEV)
    s.forward_dev(s.forward_args(n, xd.data_ptr(), out.data_ptr(), x_row=0, x_agent=18))
    torch.cuda.synchronize()
    w2, b2 = sc.forward(layers, np.broadcast_to(one, (g, n, 18)), HIDDEN, LAST)
    within(out.cpu().numpy(), w2, b2)
    # [n, G, ..] in and out, rows of odd length that start anywhere
    xr = rng.uniform(-1, 1, (n, g, 23)).astype(np.float32)
    xd, out = dev(xr), torch.full((n, g, 7), 77.0, device=DEV)
    mask = dev(np.array([1, 0, 2, 1, 0, 1], np.uint8))
    s.forward_dev(s.forward_args(n, xd.data_ptr() + 4 * 3, out.data_ptr() + 4, x_agent=23, x_row=23 * g, out_agent=7, out_row=7 * g, mask=mask.data_ptr()))
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    w3, b3 = sc.forward(layers, xr[:, :, 3:21].transpose(1, 0, 2), HIDDEN, LAST)
    keep = mask.cpu().numpy() != 0
    within(got[:, keep, 1:6].transpose(1, 0, 2), w3[keep], b3[keep])
    assert (got[:, ~keep] == 77).all() and (got[:, :, [0, 6]] == 77).all()


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("n", [3, 16, 40])
def test_states_that_are_not_finite_stay_in_their_rows(n, bits):
    """a NaN is a NaN in every output of its row; an infinity gives the infinities (and NaN) the formula gives, as in numpy"""
    dims = (18, 21, 6)
    rng = np.random.RandomState(14)
    flat = make_flat(rng, 2, dims)
    x = rng.uniform(-1, 1, (2, n, 18)).astype(np.float32)
    clean = x.copy()
    x[0, 1, 4] = np.nan
    x[1, 2, 17] = np.inf
    x[1, 0, 0] = 3e38
    layers = sc.stored(sc.split_flat(flat, dims), bits)
    with np.errstate(all="ignore"):
        want, bound = sc.forward(layers, x, 1, 0)
    got = ask(make_snap(flat, dims, bits, 1, 0), x)
    assert np.isnan(got[0, 1]).all()
    assert np.array_equal(np.isnan(got[1, 2]), np.isnan(want[1, 2])) and not np.isfinite(got[1, 2]).any()
    cw, cb = sc.forward(layers, clean, 1, 0)
    keep = np.ones((2, n), bool); keep[0, 1] = keep[1, 2] = keep[1, 0] = False
    within(got[keep], cw[keep], cb[keep])


def test_forward_of_no_rows_and_the_host_form():
    dims = (18, 20, 6)
    rng = np.random.RandomState(15)
    flat = make_flat(rng, 3, dims)
    s = make_snap(flat, dims, 4)
    s.forward_dev(s.forward_args(0, 0, 0))
    assert s.forward(np.zeros((3, 0, 18))).shape == (3, 0, 6)
    x = rng.uniform(-1, 1, (3, 7, 18)).astype(np.float32)
    assert np.array_equal(s.forward(x), ask(s, x))


# ---- the mixture ---------------------------------------------------------------------------------------------------------

def ask_mixture(s, x, rw, rb, k, allowed=None, stream=None, outputs=True):
    n = x.shape[0]
    keep = [dev(x.astype(np.float32)), dev(rw), None if rb is None else dev(rb), None if allowed is None else dev(allowed.astype(np.uint8))]
    out = torch.full((n, s.out_dim), 77.0, device=DEV)
    idx, prob = torch.full((n, k), 77, dtype=torch.int32, device=DEV), torch.full((n, k), 77.0, device=DEV)
    y = torch.full((n, k, s.out_dim), 77.0, device=DEV)
    ws = torch.full((max(1, s.mixture_workspace(n, k)),), 0xAB, dtype=torch.uint8, device=DEV)
    a = s.mixture_args(n, k, keep[0].data_ptr(), keep[1].data_ptr(), out.data_ptr(), router_b=0 if rb is None else keep[2].data_ptr(),
                       allowed=0 if allowed is None else keep[3].data_ptr(), allowed_row=0 if allowed is not None and allowed.ndim == 1 else None,
                       idx=idx.data_ptr() if outputs else 0, prob=prob.data_ptr() if outputs else 0, y=y.data_ptr() if outputs else 0,
                       workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    s.mixture_dev(a)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in (out, idx, prob, y)]


def check_mixture(s, layers, x, rw, rb, k, allowed=None, hidden=HIDDEN, last=LAST):
    out, idx, prob, y = ask_mixture(s, x, rw, rb, k, allowed)
    wo, wb, wi, wp, wy = sc.mixture(layers, x, rw, rb, k, allowed, hidden, last)
    assert np.array_equal(idx, wi)
    assert np.abs(prob - wp).max() <= 200 * sc.U
    within(out, wo, wb)
    assert (y[wi < 0] == 0).all() and (prob[wi < 0] == 0).all() and (out[wi[:, 0] < 0] == 0).all()
    for t, j in zip(*np.nonzero(wi >= 0)):
        e = wi[t, j]
        v, b = sc.forward([(w[e], bb[e]) for w, bb in layers], x[t:t + 1], hidden, last)
        within(y[t, j], v[0], b[0])
    out2 = ask_mixture(s, x, rw, rb, k, allowed, outputs=False)[0]
    assert np.array_equal(out, out2)
    return out, idx, prob, y


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("g, n, k", [(1, 1, 1), (2, 1, 2), (16, 1, 2), (16, 3, 1), (37, 17, 3), (100, 33, 8), (300, 9, 4), (5, 300, 2), (40, 700, 2), (9, 200, 8)])
def test_mixture(g, n, k, bits):
    dims = (18, 20, 6) if n > 100 else (18, 100, 33, 6)
    rng = np.random.RandomState(100 * g + n)
    flat = make_flat(rng, g, dims)
    x = rng.uniform(-1, 1, (n, 18)).astype(np.float32)
    rw, rb = rng.standard_normal((g, 18)).astype(np.float32), rng.standard_normal(g).astype(np.float32)
    check_mixture(make_snap(flat, dims, bits), sc.stored(sc.split_flat(flat, dims), bits), x, rw, rb if n % 2 else None, k)


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("dims, g, n, k", [((1, 1), 3, 2, 2), ((45, 64, 64, 17), 20, 40, 2), ((18, 400, 300, 6), 6, 5, 3), ((1024, 40, 1024), 3, 4, 2), ((3, 1024, 1024, 2), 2, 7, 2)])
def test_mixture_of_odd_nets(dims, g, n, k, bits):
    rng = np.random.RandomState(7)
    flat = make_flat(rng, g, dims)
    x = rng.uniform(-1, 1, (n, dims[0])).astype(np.float32)
    rw, rb = rng.standard_normal((g, dims[0])).astype(np.float32), rng.standard_normal(g).astype(np.float32)
    check_mixture(make_snap(flat, dims, bits), sc.stored(sc.split_flat(flat, dims), bits), x, rw, rb, k)


@pytest.mark.parametrize("n, g", [(4, 20), (70, 20), (400, 5)])
def test_mixture_masks(n, g):
    """rows with nothing left, with fewer than top_k, a row for all; everything to one agent"""
    dims, k = (18, 20, 6), 4
    rng = np.random.RandomState(21)
    flat = make_flat(rng, g, dims)
    s, layers = make_snap(flat, dims, 4), sc.stored(sc.split_flat(flat, dims), 4)
    x = rng.uniform(-1, 1, (n, 18)).astype(np.float32)
    rw, rb = rng.standard_normal((g, 18)).astype(np.float32), rng.standard_normal(g).astype(np.float32)
    allowed = rng.uniform(size=(n, g)) < 0.3
    allowed[0] = False
    allowed[1] = False; allowed[1, g - 1] = True
    check_mixture(s, layers, x, rw, rb, k, allowed)
    check_mixture(s, layers, x, rw, rb, k, allowed[2] * 5)
    check_mixture(s, layers, x, rw, rb, k, np.zeros(g))
    one = np.zeros(g); one[3] = 1
    check_mixture(s, layers, x, rw, rb, k, one)


def test_mixture_ties_and_wild_logits():
    """equal logits: the lower index; NaN above everything, +infinity, -infinity as barred"""
    dims, g, k = (6, 9, 3), 70, 5
    rng = np.random.RandomState(22)
    flat = make_flat(rng, g, dims)
    s, layers = make_snap(flat, dims, 32), sc.split_flat(flat, dims)
    x = rng.uniform(-1, 1, (20, 6)).astype(np.float32)
    rw = np.tile(rng.standard_normal((7, 6)).astype(np.float32), (10, 1))
    check_mixture(s, layers, x, rw, None, k)
    check_mixture(s, layers, x, np.zeros((g, 6), np.float32), np.zeros(g, np.float32), k)
    check_mixture(s, layers, x, -np.zeros((g, 6), np.float32), np.where(np.arange(g) % 2, -0.0, 0.0).astype(np.float32), k)
    rb = rng.standard_normal(g).astype(np.float32)
    rb[3:68] = -np.inf
    check_mixture(s, layers, x, rw, rb, k + 3)
    rb[:] = -np.inf
    check_mixture(s, layers, x, rw, rb, k)
    rb = rng.standard_normal(g).astype(np.float32)
    rb[[40, 11]] = np.nan
    out, idx, prob, y = ask_mixture(s, x, rw, rb, k)
    assert (idx[:, :2] == [11, 40]).all() and np.isnan(prob).all() and np.isnan(out).all()
    rest = sc.mixture(layers, x, rw, np.where(np.isnan(rb), -np.inf, rb), k, None, HIDDEN, LAST)[2]
    assert np.array_equal(idx[:, 2:], rest[:, :k - 2])
    xn = x.copy(); xn[4, 2] = np.nan                             # a state that is not a number spoils its own row
    out, idx, _, _ = ask_mixture(s, xn, rw, None, k)
    clean = ask_mixture(s, x, rw, None, k)
    assert (idx[4] == np.arange(k)).all() and np.isnan(out[4]).all()
    keep = np.arange(20) != 4
    assert np.array_equal(out[keep], clean[0][keep]) and np.array_equal(idx[keep], clean[1][keep])


def test_mixture_strides_and_the_host_form():
    dims, g, n, k = (18, 20, 6), 30, 11, 3
    rng = np.random.RandomState(23)
    flat = make_flat(rng, g, dims)
    s, layers = make_snap(flat, dims, 4), sc.stored(sc.split_flat(flat, dims), 4)
    xr, rwr = rng.uniform(-1, 1, (n, 21)).astype(np.float32), rng.standard_normal((g, 19)).astype(np.float32)
    rb, alr = rng.standard_normal(g).astype(np.float32), (rng.uniform(size=(n, 33)) < 0.5).astype(np.uint8)
    x, rw, al = xr[:, 2:20], rwr[:, 1:], alr[:, 3:]
    xd, wd, bd, ad, out = dev(xr), dev(rwr), dev(rb), dev(alr), torch.full((n, 9), 77.0, device=DEV)
    ws = torch.empty(s.mixture_workspace(n, k), dtype=torch.uint8, device=DEV)
    s.mixture_dev(s.mixture_args(n, k, xd.data_ptr() + 8, wd.data_ptr() + 4, out.data_ptr() + 4, router_b=bd.data_ptr(), allowed=ad.data_ptr() + 3,
                                 allowed_row=33, x_row=21, router_row=19, out_row=9, workspace=ws.data_ptr(), workspace_bytes=ws.numel()))
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    wo, wb, wi, wp, _ = sc.mixture(layers, x, rw, rb, k, al, HIDDEN, LAST)
    within(got[:, 1:7], wo, wb)
    assert (got[:, [0, 7, 8]] == 77).all()
    ho, hi, hp = s.mixture(x, rw, rb, k, al)
    assert np.array_equal(ho, got[:, 1:7]) and np.array_equal(hi, wi) and np.abs(hp - wp).max() <= 200 * sc.U
    s.mixture_dev(s.mixture_args(0, k, 0, 0, 0))
    assert s.mixture(np.zeros((0, 18)), rw)[0].shape == (0, 6)


# ---- its gradient --------------------------------------------------------------------------------------------------------

def ask_grad(s, x, idx, prob, y, dout, db=True, dy=True):
    n, k = idx.shape
    t = [dev(v) for v in (x.astype(np.float32), idx.astype(np.int32), prob.astype(np.float32), y.astype(np.float32), dout.astype(np.float32))]
    dw, b = torch.full((s.G, s.in_dim), 77.0, device=DEV), torch.full((s.G,), 77.0, device=DEV)
    d = torch.full((n, k, s.out_dim), 77.0, device=DEV)
    ws = torch.full((max(1, s.mixture_grad_workspace(n, k)),), 0xAB, dtype=torch.uint8, device=DEV)
    s.mixture_grad_dev(s.mixture_grad_args(n, k, *(v.data_ptr() for v in t), dw.data_ptr(), b.data_ptr() if db else 0, d.data_ptr() if dy else 0,
                                           workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return dw.cpu().numpy(), b.cpu().numpy(), d.cpu().numpy()


@pytest.mark.parametrize("g, n, k, ins, outs", [(1, 1, 1, 1, 1), (2, 3, 2, 18, 6), (16, 9, 2, 18, 6), (50, 70, 8, 45, 17), (3, 1000, 2, 18, 6), (1, 700, 1, 5, 3),
                                                (300, 130, 4, 300, 2), (4, 40, 3, 1024, 1024), (7, 600, 3, 257, 5)])
def test_mixture_gradient(g, n, k, ins, outs):
    import ddrl_amd
    rng = np.random.RandomState(g + n)
    s = ddrl_amd.PolicySnapshot.shaped(g, ins, outs, [], bits=32)
    x, y, dout = rng.uniform(-1, 1, (n, ins)), rng.standard_normal((n, k, outs)), rng.standard_normal((n, outs))
    x, y, dout = (v.astype(np.float32) for v in (x, y, dout))
    idx = np.argsort(rng.uniform(size=(n, g)), 1)[:, :k]
    prob = rng.dirichlet(np.ones(k), n).astype(np.float32)
    if n > 8:
        idx[1, -1] = -1; idx[2] = -1; idx[3, 0] = g; idx[4, 0] = 2 ** 31 - 1; idx[5, 0] = -2 ** 31        # nobody
        prob[idx < 0] = 0
    dw, db, dy = ask_grad(s, x, idx, prob, y, dout)
    ww, wb, wy, bw, bb = sc.mixture_grad(x, idx, prob, y, dout, g)
    within(dw, ww, bw)
    within(db, wb, bb)
    within(dy, wy, 2 * sc.U * np.abs(wy) + 1e-37)
    again = ask_grad(s, x, idx, prob, y, dout)
    assert all(np.array_equal(a, b) for a, b in zip((dw, db, dy), again))
    only = ask_grad(s, x, idx, prob, y, dout, db=False, dy=False)
    assert np.array_equal(only[0], dw) and (only[1] == 77).all() and (only[2] == 77).all()


def test_gradient_of_no_rows_is_zero():
    import ddrl_amd
    s = ddrl_amd.PolicySnapshot.shaped(5, 18, 6, [], bits=32)
    dw, db, _ = ask_grad(s, np.zeros((0, 18)), np.zeros((0, 2)), np.zeros((0, 2)), np.zeros((0, 2, 6)), np.zeros((0, 6)))
    assert (dw == 0).all() and (db == 0).all()


def test_gradient_against_differences():
    """L = sum(dout * out) of the mixture as it runs on the GPU's picks, differentiated in the 64-bit definition"""
    dims, g, n, k = (6, 11, 3), 12, 10, 3
    rng = np.random.RandomState(31)
    flat = make_flat(rng, g, dims)
    s, layers = make_snap(flat, dims, 4), sc.stored(sc.split_flat(flat, dims), 4)
    x = rng.uniform(-1, 1, (n, 6)).astype(np.float32)
    rw, rb = rng.standard_normal((g, 6)).astype(np.float32), rng.standard_normal(g).astype(np.float32)
    dout = rng.standard_normal((n, 3)).astype(np.float32)
    out, idx, prob, y = check_mixture(s, layers, x, rw, rb, k)
    dw, db, _ = ask_grad(s, x, idx, prob, y, dout)
    nets = [(w.astype(np.float64), b.astype(np.float64)) for w, b in layers]

    def loss(w, b):
        total = 0.0
        for t in range(n):
            l = w[idx[t]] @ x[t].astype(np.float64) + b[idx[t]]
            p = np.exp(l - l.max()); p /= p.sum()
            for j, e in enumerate(idx[t]):
                v, _ = sc.forward([(ww[e], bb[e]) for ww, bb in nets], x[t:t + 1], HIDDEN, LAST)
                total += p[j] * (dout[t] * v[0]).sum()
        return total

    w64, b64, h = rw.astype(np.float64), rb.astype(np.float64), 1e-5
    for e in range(g):
        for what, got in ((("b",), db[e]), (("w", 2), dw[e, 2]), (("w", 5), dw[e, 5])):
            hi, lo = (w64.copy(), b64.copy()), (w64.copy(), b64.copy())
            if what[0] == "b":
                hi[1][e] += h; lo[1][e] -= h
            else:
                hi[0][e, what[1]] += h; lo[0][e, what[1]] -= h
            diff = (loss(*hi) - loss(*lo)) / (2 * h)
            # central differences: h^2 / 6 of the third derivative (softmax: below 1 per row and unit of dout . y), 64-bit noise
            # 1e-15 / h; the kernel's own: some hundred U of sums of order 1 per row
            assert abs(diff - got) <= n * (h * h * 10 + 1e-9 + 400 * sc.U)


# ---- together, streams, graphs, refusals ---------------------------------------------------------------------------------

def test_a_run_of_them():
    """a population's snapshot in 4 bits answers alone and as a mixture, and the router takes a step along its gradient"""
    import ddrl_amd
    g, k, n = 24, 2, 40
    pop = ddrl_amd.PolicyPopulation(g, 18, 6, (20, 33), init_seed=5)
    dims = (18, 20, 33, 6)
    rng = np.random.RandomState(41)
    pop.set_weights(0, make_flat(rng, g, dims))
    s = ddrl_amd.PolicySnapshot(pop, 0, 4)
    layers = layers_now(pop, dims, 4)
    rw, rb = rng.standard_normal((g, 18)).astype(np.float32), np.zeros(g, np.float32)
    for step in range(3):
        x = rng.uniform(-1, 1, (n, 18)).astype(np.float32)
        goal = rng.uniform(-1, 1, (n, 6)).astype(np.float32)
        alone = ask(s, x)
        out, idx, prob, y = check_mixture(s, layers, x, rw, rb, k)
        for t, j in np.ndindex(n, k):
            within(y[t, j], alone[idx[t, j], t], 1e-5)            # (both within their bounds of the same value; these are below 5e-6)
        dout = out - goal
        dw, db, _ = ask_grad(s, x, idx, prob, y, dout)
        ww, wb, _, bw, bb = sc.mixture_grad(x, idx, prob, y, dout, g)
        within(dw, ww, bw)
        within(db, wb, bb)
        rw, rb = rw - 0.1 * dw, rb - 0.1 * db
        pop.set_weights(0, pop.weights(0) * 0.9)
        s.load(pop)
        layers = layers_now(pop, dims, 4)


def _calls(s, n, k, seed):
    """inputs, outputs and one forward, one mixture, one gradient on the current stream"""
    rng = np.random.RandomState(seed)
    st = dict(x=dev(rng.uniform(-1, 1, (n, s.in_dim)).astype(np.float32)), rw=dev(rng.standard_normal((s.G, s.in_dim)).astype(np.float32)),
              dout=dev(rng.standard_normal((n, s.out_dim)).astype(np.float32)))
    e = lambda *shape, **kw: torch.zeros(*shape, device=DEV, **kw)
    st.update(f=e(s.G, n, s.out_dim), out=e(n, s.out_dim), idx=e(n, k, dtype=torch.int32), prob=e(n, k), y=e(n, k, s.out_dim), dw=e(s.G, s.in_dim),
              db=e(s.G), dy=e(n, k, s.out_dim), ws=e(s.mixture_workspace(n, k), dtype=torch.uint8), wg=e(max(1, s.mixture_grad_workspace(n, k)), dtype=torch.uint8))

    def run():
        q = torch.cuda.current_stream().cuda_stream
        p = {key: v.data_ptr() for key, v in st.items()}
        s.forward_dev(s.forward_args(n, p["x"], p["f"], x_agent=0, stream=q))
        s.mixture_dev(s.mixture_args(n, k, p["x"], p["rw"], p["out"], idx=p["idx"], prob=p["prob"], y=p["y"], workspace=p["ws"], workspace_bytes=st["ws"].numel(), stream=q))
        s.mixture_grad_dev(s.mixture_grad_args(n, k, p["x"], p["idx"], p["prob"], p["y"], p["dout"], p["dw"], p["db"], p["dy"],
                                               workspace=p["wg"], workspace_bytes=st["wg"].numel(), stream=q))

    results = lambda: [st[key].cpu().numpy().copy() for key in ("f", "out", "idx", "prob", "y", "dw", "db", "dy")]
    return st, run, results


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("n", [3, 700])
def test_graphs(n, bits):
    """two captured graphs of one snapshot, replayed between eager calls and new inputs, against the eager bits"""
    dims = (18, 40, 6)
    s = make_snap(make_flat(np.random.RandomState(51), 30, dims), dims, bits)
    made = [_calls(s, n, 3, seed) for seed in (1, 2)]
    graphs = []
    for st, run, _ in made:
        run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        graphs.append(g)
    for rep in range(4):
        for st, _, _ in made:
            st["x"].copy_(torch.from_numpy(np.random.RandomState(60 + rep).uniform(-1, 1, st["x"].shape).astype(np.float32)))
        want = []
        for st, run, results in made:
            run()
            torch.cuda.synchronize()
            want.append(results())
            for key in ("f", "out", "y", "dw"):
                st[key].zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (st, run, results), w in zip(made, want):
            assert all(np.array_equal(a, b) for a, b in zip(results(), w))


def test_streams_and_threads():
    """calls on one snapshot from two host threads, each on a stream of its own, give the bits of calls one after the other"""
    import threading
    dims = (18, 100, 6)
    s = make_snap(make_flat(np.random.RandomState(52), 64, dims), dims, 4)
    made = [_calls(s, 400, 2, seed) for seed in (3, 4)]
    want = []
    for st, run, results in made:
        run()
        torch.cuda.synchronize()
        want.append(results())
        for key in ("f", "out", "y", "dw"):
            st[key].zero_()
    torch.cuda.synchronize()
    failed = []

    def work(run):
        try:
            q = torch.cuda.Stream()
            with torch.cuda.stream(q):
                for _ in range(20):
                    run()
            q.synchronize()
        except Exception as e:          # noqa: BLE001
            failed.append(e)

    ts = [threading.Thread(target=work, args=(run,)) for _, run, _ in made]
    [t.start() for t in ts]
    [t.join() for t in ts]
    torch.cuda.synchronize()
    assert not failed
    for (st, run, results), w in zip(made, want):
        assert all(np.array_equal(a, b) for a, b in zip(results(), w))


def test_a_load_is_not_captured():
    import ddrl_amd
    dims = (6, 8, 2)
    flat = make_flat(np.random.RandomState(53), 3, dims)
    s, d = make_snap(flat, dims, 4), dev(flat)
    x = torch.zeros(4, device=DEV)
    q = torch.cuda.Stream()
    q.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=q):
        x.add_(1)
        with pytest.raises(ddrl_amd.DdrlError) as e:
            s.load_flat_dev(d.data_ptr(), flat.shape[1], stream=torch.cuda.current_stream().cuda_stream)
    assert e.value.code == -4
    g.replay()
    torch.cuda.synchronize()
    assert (x == 1).all()


def test_refusals():
    import ddrl_amd
    dims = (6, 8, 2)
    s = make_snap(make_flat(np.random.RandomState(54), 3, dims), dims, 4)
    t = torch.zeros(4096, device=DEV)
    p = t.data_ptr()
    ws = torch.zeros(65536, dtype=torch.uint8, device=DEV)
    w = dict(workspace=ws.data_ptr(), workspace_bytes=65536)

    def refused(f, *words, code=-1):
        with pytest.raises(ddrl_amd.DdrlError) as e:
            f()
        assert e.value.code == code and all(x in str(e.value) for x in words), str(e.value)

    f = lambda **kw: s.forward_dev(s.forward_args(**{**dict(n=4, x=p, out=p + 8192), **kw}))
    refused(lambda: f(n=-1), "n=-1")
    refused(lambda: f(x=0), "x / out")
    refused(lambda: f(out=0), "x / out")
    refused(lambda: f(x=p + 2), "x / out")
    refused(lambda: f(x_row=-3), "stride of x")
    refused(lambda: f(x_agent=-2), "stride of x")
    refused(lambda: f(out_row=1), "overlap")
    refused(lambda: f(out_agent=5), "overlap")
    refused(lambda: f(out_agent=0), "overlap")
    refused(lambda: f(out_row=-7), "overlap")
    m = lambda **kw: s.mixture_dev(s.mixture_args(**{**dict(n=4, top_k=2, x=p, router_w=p + 1024, out=p + 8192), **w, **kw}))
    refused(lambda: m(n=-1), "top_k")
    refused(lambda: m(top_k=0), "top_k")
    refused(lambda: m(top_k=4), "3 agents")
    refused(lambda: m(top_k=9), "top_k")
    refused(lambda: m(n=2 ** 28), "n * top_k")
    refused(lambda: m(x=0), "NULL")
    refused(lambda: m(router_w=0), "NULL")
    refused(lambda: m(out=0), "NULL")
    refused(lambda: m(prob=p + 1), "misaligned")
    refused(lambda: m(workspace=0), "workspace")
    refused(lambda: m(workspace=ws.data_ptr() + 8), "workspace")
    refused(lambda: m(workspace_bytes=s.mixture_workspace(4, 2) - 1), "workspace")
    refused(lambda: m(out_row=1), "overlap")
    refused(lambda: m(x_row=-2), "stride")
    refused(lambda: m(router_row=-2), "stride")
    refused(lambda: m(allowed=p, allowed_row=-2), "stride")
    refused(lambda: s.mixture_workspace(3, 0), "top_k")
    r = lambda **kw: s.mixture_grad_dev(s.mixture_grad_args(**{**dict(n=4, top_k=2, x=p, idx=p, prob=p, y=p, dout=p, d_router_w=p + 8192), **w, **kw}))
    refused(lambda: r(top_k=0), "top_k")
    refused(lambda: r(idx=0), "NULL")
    refused(lambda: r(dout=0), "NULL")
    refused(lambda: r(d_router_w=0), "d_router_w")
    refused(lambda: r(d_router_row=5), "overlap")
    refused(lambda: r(dout_row=-2), "stride")
    refused(lambda: s.load_flat_dev(0, 100), "NULL")
    refused(lambda: s.load_flat_dev(p, 5), "ld=5")
    refused(lambda: ddrl_amd.PolicySnapshot.shaped(2, 3, 4, [], device=64), "device")
    # what a snapshot does not hold
    pop = ddrl_amd.PolicyPopulation(3, 6, 2, (8,), 1, 2)
    s.load(pop)
    refused(lambda: s.load(pop, 1), "net 1")
    refused(lambda: s.load(ddrl_amd.PolicyPopulation(4, 6, 2, (8,), 1, 2)), "dimensions")
    refused(lambda: s.load(ddrl_amd.PolicyPopulation(3, 6, 2, (9,), 1, 2)), "dimensions")
    refused(lambda: s.load(ddrl_amd.PolicyPopulation(3, 6, 2, (8,), 2, 2)), "dimensions")
    pop.set_gates(np.ones((3, 6)), np.ones((3, 2)))
    refused(lambda: s.load(pop), "gates", code=-4)
    cfg = ddrl_amd.DdpgConfig(n_agents=3, nb_sensors=6, nb_motors=2, mini_batch_size=16, replay_memory=300, hidden_unit_a=(8,), hidden_unit_q=(8,),
                              batch_norm_actor=7, batch_norm_critic=0)
    refused(lambda: ddrl_amd.PolicySnapshot(ddrl_amd.DdpgPopulation(cfg)), "BatchNorm")


def test_long_offsets():
    """rows more than 2^32 bytes apart, in and out"""
    dims = (6, 8, 2)
    rng = np.random.RandomState(55)
    flat = make_flat(rng, 2, dims)
    s, layers = make_snap(flat, dims, 4), sc.stored(sc.split_flat(flat, dims), 4)
    far = 1_100_000_000
    big = torch.empty(far + 100, device=DEV)
    out = torch.empty(far + 100, device=DEV)
    x = rng.uniform(-1, 1, (2, 2, 6)).astype(np.float32)
    for g in range(2):
        for t in range(2):
            big[t * far + g * 6: t * far + g * 6 + 6] = dev(x[g, t])
    s.forward_dev(s.forward_args(2, big.data_ptr(), out.data_ptr(), x_agent=6, x_row=far, out_agent=2, out_row=far))
    torch.cuda.synchronize()
    got = np.stack([[out[t * far + g * 2: t * far + g * 2 + 2].cpu().numpy() for t in range(2)] for g in range(2)])
    want, bound = sc.forward(layers, x, HIDDEN, LAST)
    within(got, want, bound)
