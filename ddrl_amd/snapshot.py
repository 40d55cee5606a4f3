"""Python mirror of the served snapshots (include/ddrl_pop.h, ddrl_snap_*): a copy of one net of every agent of a population,
its weights in 32 or 4 bits, that answers for every agent (`forward`) or as a mixture behind a router (`mixture`).

`forward` and `mixture` take numpy arrays.  The `_dev` calls work on device memory: `*_args` puts a call's pointers (addresses,
as torch's `data_ptr()` gives them), strides and stream (a hipStream_t, as torch's `cuda_stream`) into a structure that can be
kept and called again; the arrays behind the addresses are the caller's to keep alive.
"""
import ctypes as C

import numpy as np

from . import lib as _l
from .population import _p


def _stride(v):
    return -1 if v is None else int(v)


class PolicySnapshot:
    """One net of every agent of a population, as it was when it was loaded.

    PolicySnapshot(pop, net, bits) has the dimensions of the population's net and its parameters; PolicySnapshot.shaped(..)
    starts with zero weights.  `load` / `load_flat_dev` take new parameters."""

    def __init__(self, pop, net=0, bits=4):
        self.L = _l.load()
        h = C.c_void_p()
        _l.check(self.L.ddrl_snap_create_from(pop.h, int(net), int(bits), C.byref(h)))
        self._take(h)

    @classmethod
    def shaped(cls, n_agents, in_dim, out_dim, hidden, hidden_layer_type=1, output_layer_type=2, bits=4, device=-1):
        o = cls.__new__(cls)
        o.L = _l.load()
        hid = np.ascontiguousarray(hidden, np.int32)
        h = C.c_void_p()
        _l.check(o.L.ddrl_snap_create(int(n_agents), int(in_dim), int(out_dim), _p(hid), hid.size, int(hidden_layer_type),
                                      int(output_layer_type), int(bits), int(device), C.byref(h)))
        o._take(h)
        return o

    def _take(self, h):
        self.h = h
        v = [C.c_int() for _ in range(5)]
        _l.check(self.L.ddrl_snap_shape(h, *(C.byref(x) for x in v)))
        self.G, self.in_dim, self.out_dim, self.bits, self.n_params = (x.value for x in v)

    def close(self):
        if getattr(self, "h", None):
            self.L.ddrl_snap_destroy(self.h)
            self.h = None

    __del__ = close

    def load(self, pop, net=0, stream=0):
        _l.check(self.L.ddrl_snap_load(self.h, pop.h, int(net), stream or None))

    def load_flat_dev(self, d_flat_ptr, ld, stream=0):
        """fp32 rows [G x ld] (ld = 0: one row for every agent) already on the device"""
        _l.check(self.L.ddrl_snap_load_flat_dev(self.h, d_flat_ptr, int(ld), stream or None))

    def weights(self):
        """what the stored weights stand for, [G x n_params]; waits for everything on the GPU"""
        out = np.empty((self.G, self.n_params))
        _l.check(self.L.ddrl_snap_get_weights(self.h, _p(out)))
        return out

    # every agent's net on n rows: x [G x n x in_dim] -> [G x n x out_dim]
    def forward(self, x):
        x = np.ascontiguousarray(x, np.float32).reshape(self.G, -1, self.in_dim)
        out = np.empty((self.G, x.shape[1], self.out_dim), np.float32)
        _l.check(self.L.ddrl_snap_forward(self.h, x.shape[1], _p(x), _p(out)))
        return out

    def forward_args(self, n, x, out, x_agent=None, x_row=None, out_agent=None, out_row=None, mask=0, stream=0):
        """x_agent = 0: the same rows for all agents; a stride of None: packed"""
        return _l.SnapForwardArgs(int(n), x or None, _stride(x_agent), _stride(x_row), out or None, _stride(out_agent),
                                  _stride(out_row), mask or None, stream or None)

    def forward_dev(self, args):
        _l.check(self.L.ddrl_snap_forward_dev(self.h, C.byref(args)))

    # the mixture: x [n x in_dim], router_w [G x in_dim], router_b [G], allowed [n x G] or [G] -> out, idx, prob
    def mixture(self, x, router_w, router_b=None, top_k=2, allowed=None):
        x = np.ascontiguousarray(x, np.float32).reshape(-1, self.in_dim)
        n = x.shape[0]
        w = np.ascontiguousarray(router_w, np.float32).reshape(self.G, self.in_dim)
        b = None if router_b is None else np.ascontiguousarray(router_b, np.float32).reshape(self.G)
        al = None if allowed is None else np.ascontiguousarray(np.broadcast_to(np.asarray(allowed) != 0, (n, self.G)), np.uint8)
        out = np.empty((n, self.out_dim), np.float32)
        idx, prob = np.empty((n, top_k), np.int32), np.empty((n, top_k), np.float32)
        _l.check(self.L.ddrl_snap_mixture(self.h, n, int(top_k), _p(x), _p(w), _p(b), _p(al), _p(out), _p(idx), _p(prob)))
        return out, idx, prob

    def mixture_workspace(self, n, top_k):
        b = C.c_size_t()
        _l.check(self.L.ddrl_snap_mixture_workspace(self.h, int(n), int(top_k), C.byref(b)))
        return b.value

    def mixture_args(self, n, top_k, x, router_w, out, router_b=0, allowed=0, idx=0, prob=0, y=0, workspace=0, workspace_bytes=0,
                     x_row=None, router_row=None, allowed_row=None, out_row=None, stream=0):
        """allowed_row = 0: one row of `allowed` for all; a stride of None: packed"""
        return _l.SnapMixtureArgs(int(n), int(top_k), x or None, _stride(x_row), router_w or None, _stride(router_row), router_b or None,
                                  allowed or None, _stride(allowed_row), out or None, _stride(out_row), idx or None, prob or None,
                                  y or None, workspace or None, int(workspace_bytes), stream or None)

    def mixture_dev(self, args):
        _l.check(self.L.ddrl_snap_mixture_dev(self.h, C.byref(args)))

    def mixture_grad_workspace(self, n, top_k):
        b = C.c_size_t()
        _l.check(self.L.ddrl_snap_mixture_grad_workspace(self.h, int(n), int(top_k), C.byref(b)))
        return b.value

    def mixture_grad_args(self, n, top_k, x, idx, prob, y, dout, d_router_w, d_router_b=0, dy=0, workspace=0, workspace_bytes=0,
                          x_row=None, dout_row=None, d_router_row=None, stream=0):
        return _l.SnapMixtureGradArgs(int(n), int(top_k), x or None, _stride(x_row), idx or None, prob or None, y or None, dout or None,
                                      _stride(dout_row), d_router_w or None, _stride(d_router_row), d_router_b or None, dy or None,
                                      workspace or None, int(workspace_bytes), stream or None)

    def mixture_grad_dev(self, args):
        _l.check(self.L.ddrl_snap_mixture_grad_dev(self.h, C.byref(args)))
