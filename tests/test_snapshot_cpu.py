"""Served snapshots without a GPU: the refusals that come before any device is looked for, the structures' layout, and the
definition the GPU tests compare with."""
import ctypes as C
import os

import numpy as np
import pytest

import snapshot_common as sc

HAVE_GPU = os.path.exists("/dev/kfd")


def _create(n_agents=4, in_dim=3, out_dim=2, hidden=(5,), hact=1, oact=2, bits=4, device=-1):
    import ddrl_amd
    return ddrl_amd.PolicySnapshot.shaped(n_agents, in_dim, out_dim, hidden, hact, oact, bits, device)


@pytest.mark.parametrize("bad, word", [
    (dict(n_agents=0), "n_agents"), (dict(in_dim=0), "in_dim"), (dict(in_dim=1025), "in_dim"), (dict(out_dim=0), "out_dim"),
    (dict(out_dim=2000), "out_dim"), (dict(hidden=(4, 4, 4, 4)), "n_hidden"), (dict(hidden=(0,)), "hidden[0]"),
    (dict(hidden=(5, 1025)), "hidden[1]"), (dict(hact=4), "hidden_layer_type"), (dict(oact=-1), "output_layer_type"),
    (dict(bits=8), "bits"), (dict(bits=0), "bits")])
def test_create_refuses(bad, word):
    import ddrl_amd
    with pytest.raises(ddrl_amd.DdrlError) as e:
        _create(**bad)
    assert e.value.code == -1 and word in str(e.value)


@pytest.mark.skipif(HAVE_GPU, reason="there is a GPU")
def test_no_cpu_path():
    import ddrl_amd
    with pytest.raises(ddrl_amd.DdrlError) as e:
        _create()
    assert e.value.code == -2


def test_null_handles_are_refused():
    import ddrl_amd
    from ddrl_amd import lib
    L = ddrl_amd.load()
    z = C.c_size_t()
    assert L.ddrl_snap_destroy(None) == 0
    out = C.c_void_p()
    calls = [L.ddrl_snap_shape(None, None, None, None, None, None), L.ddrl_snap_create_from(None, 0, 4, C.byref(out)), L.ddrl_snap_load(None, None, 0, None),
             L.ddrl_snap_load_flat_dev(None, None, 0, None), L.ddrl_snap_get_weights(None, None),
             L.ddrl_snap_forward_dev(None, C.byref(lib.SnapForwardArgs())), L.ddrl_snap_forward(None, 1, None, None),
             L.ddrl_snap_mixture_workspace(None, 1, 1, C.byref(z)), L.ddrl_snap_mixture_dev(None, C.byref(lib.SnapMixtureArgs())),
             L.ddrl_snap_mixture(None, 1, 1, None, None, None, None, None, None, None),
             L.ddrl_snap_mixture_grad_workspace(None, 1, 1, C.byref(z)), L.ddrl_snap_mixture_grad_dev(None, C.byref(lib.SnapMixtureGradArgs()))]
    assert calls == [-1] * len(calls)


def test_structures_have_the_c_layout():
    """64-bit platforms: int pairs, then pointers, int64_t and size_t of 8 bytes each"""
    from ddrl_amd import lib
    assert C.sizeof(lib.SnapForwardArgs) == 8 * 9
    assert C.sizeof(lib.SnapMixtureArgs) == 8 * 16
    assert C.sizeof(lib.SnapMixtureGradArgs) == 8 * 15
    assert lib.SnapMixtureArgs.x.offset == 8 and lib.SnapMixtureArgs.stream.offset == 8 * 15


def test_definition_of_four_bits():
    """the oracle against the format's own statements: the grid is kept, halves go to the even code, nothing leaves +-6 scale"""
    rng = np.random.RandomState(0)
    w = (rng.standard_normal((7, 70)) * 10 ** rng.uniform(-3, 3, (7, 1))).astype(np.float32)
    r = sc.round4(w)
    for b in range(0, 70, 32):
        v, q = w[:, b:b + 32].astype(np.float64), r[:, b:b + 32]
        a = np.abs(v).max(1)
        s = 2.0 ** np.ceil(np.log2(a / 6))
        assert np.all(a <= 6 * s) and np.all(a > 3 * s)
        m = np.abs(q) / s[:, None]
        assert np.isin(m, sc.GRID).all()
        gap = np.where(m < 2, .25, np.where(m < 4, .5, 1.0))
        assert np.all(np.abs(q - v) <= gap * s[:, None] + 1e-300)
    ties = np.array([[.25, .75, 1.25, 1.75, 2.5, 3.5, 5., 6., -.25, -.75, -5., -2.5]], np.float32)
    assert np.array_equal(sc.round4(ties)[0], [0, 1, 1, 2, 2, 4, 4, 6, 0, -1, -4, -2])


@pytest.mark.parametrize("n_agents", [2 ** 22, 2 ** 24, 2 ** 31 - 1])
def test_more_agents_than_a_launch_takes_are_refused(n_agents):
    """a workgroup an agent, 1024 threads at most, 2^32 - 1 threads in all"""
    import ddrl_amd
    with pytest.raises(ddrl_amd.DdrlError) as e:
        _create(n_agents=n_agents)
    assert e.value.code == -1 and "n_agents" in str(e.value)
