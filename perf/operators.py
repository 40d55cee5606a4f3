"""Cases that measure the snapshot operators (ddrl_amd.PolicySnapshot): the nets of a population answering states from 4-bit
weights, a mixture of the nets of a population behind a router, and the router's gradient.

A case is one call on synthetic nets of random weights.  `run` computes the operator in elementary torch operations, or, where
`own` is set, makes the call that a user of the package makes.

Shapes are written "in-hidden-..-out".  The sizes are those of bench.py: the small (20), mid (100, 100) and large (400, 300)
nets of a HalfCheetah sweep (18 sensors, 6 motors; a critic reads sensors and motors, 24), the 64 x 64 nets over 45 sensors
and 17 motors of its NFAC workload, populations of up to 1024 agents.
"""
import functools
import math

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)        # the magnitudes of a 4-bit weight (E2M1); bit 3 of a code is the sign
BLOCK = 32                                             # inputs that share a scale, a power of two (E8M0)
DEVICE = "cuda"


def listed():
    return [
        # a handful of small policies asked for one action each, as on a robot: launch and latency are all there is
        dict(name="act_small", op="forward", agents=16, dims="18-20-6", acts="leaky-tanh", n=1, shared=False),
        # one action for every agent of the default sweep
        dict(name="act_mid", op="forward", agents=1024, dims="18-100-100-6", acts="leaky-tanh", n=1, shared=False),
        # the same of the large nets: reading the weights is the work
        dict(name="act_large", op="forward", agents=1024, dims="18-400-300-6", acts="leaky-tanh", n=1, shared=False),
        # a critic ensemble of odd size scoring the same 250 (state, action) rows
        dict(name="score_shared", op="forward", agents=129, dims="24-100-100-1", acts="relu-linear", n=250, shared=True),
        # a minibatch of 64 rows through every agent of a sweep of large nets: the most arithmetic
        dict(name="eval_large", op="forward", agents=1024, dims="18-400-300-6", acts="leaky-tanh", n=64, shared=False),
        # one state answered by two of sixteen policies: the latency of a mixture
        dict(name="mix_one", op="mixture", agents=16, bits=32, dims="18-100-100-6", acts="leaky-tanh", n=1, top_k=2, masked=False),
        # eight robots, a whole sweep to choose from, some of the policies withheld per robot, weights in 4 bits
        dict(name="mix_few", op="mixture", agents=1024, bits=4, dims="18-100-100-6", acts="leaky-tanh", n=8, top_k=4, masked=True),
        # an odd number of states over large nets in 32 bits
        dict(name="mix_large", op="mixture", agents=128, bits=32, dims="18-400-300-6", acts="leaky-tanh", n=33, top_k=2, masked=False),
        # a long trajectory batch over the nets of the NFAC workload
        dict(name="mix_many", op="mixture", agents=256, bits=32, dims="45-64-64-17", acts="leaky-tanh", n=4096, top_k=2, masked=False),
        # the router's gradient from a few states, as after every step online
        dict(name="grad_few", op="grad", agents=16, dims="18-6", n=9, top_k=2, masked=True),
        # and from a long trajectory batch over a whole sweep
        dict(name="grad_many", op="grad", agents=1024, dims="45-17", n=4096, top_k=4, masked=False),
    ]


def dims_of(case):
    return [int(d) for d in case["dims"].split("-")]


def weights_of(case):
    d = dims_of(case)
    return sum(a * b for a, b in zip(d, d[1:]))


def between(rng, low, high):
    """a whole number between low and high, spread over its logarithm"""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    while True:
        op = rng.choice(("forward", "mixture", "grad"))
        sensors, motors = rng.randint(3, 64), rng.randint(1, 17)
        hidden = [between(rng, 8, 400) for _ in range(rng.randint(1, 3))]
        case = dict(op=op, agents=between(rng, 1 if op == "forward" else 2, 1024))
        if op == "forward":
            case.update(dims="-".join(map(str, [sensors] + hidden + [motors])), n=between(rng, 1, 256), shared=rng.random() < 0.3,
                        acts=rng.choice(("leaky-tanh", "relu-linear", "tanh-linear")))
        else:
            case.update(n=between(rng, 1, 4096), top_k=rng.randint(1, min(8, case["agents"])), masked=rng.random() < 0.5)
            if op == "mixture":
                case.update(dims="-".join(map(str, [sensors] + hidden + [motors])), bits=rng.choice((32, 4)),
                            acts=rng.choice(("leaky-tanh", "relu-linear", "tanh-linear")))
            else:
                case.update(dims="%d-%d" % (sensors, motors))
        top = [work(c) for c in listed() if c["op"] == op]
        mine = work(case)
        if all(mine[k] <= max(t[k] for t in top) for k in ("bytes", "flops")):
            return case


def work(case):
    d, g, n = dims_of(case), case["agents"], case["n"]
    p = weights_of(case)
    outs = sum(d[1:])
    if case["op"] == "grad":
        k, s, a = case["top_k"], d[0], d[1]
        return {"bytes": 4 * (n * s + n * a + n * k * (2 + 2 * a) + g * (s + 1)), "flops": n * k * (5 * a + 2 * s + 4)}
    four = sum(o * (i / 2 + math.ceil(i / BLOCK)) for i, o in zip(d, d[1:])) + 4 * outs      # a net in 4 bits, in bytes
    if case["op"] == "forward":
        return {"bytes": g * four + 4 * n * ((1 if case["shared"] else g) * d[0] + g * d[-1]), "flops": 2 * g * n * p}
    k = case["top_k"]
    used = g * (1 - (1 - 1 / g) ** (n * k))                                                   # nets that some state chooses
    net = four if case["bits"] == 4 else 4 * (p + outs)
    return {"bytes": used * net + 4 * (g * (d[0] + 1) + n * (d[0] + d[-1]) + n * k * (2 + d[-1])) + (n * g if case["masked"] else 0),
            "flops": 2 * n * g * d[0] + 2 * n * k * p + 2 * n * k * d[-1]}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def nets(case, seed):
    """the nets of all agents: a list of (weights [agents, out, in], biases [agents, out])"""
    gen = torch.Generator(DEVICE).manual_seed(int(seed))
    d, g = dims_of(case), case["agents"]
    return [(torch.randn(g, o, i, generator=gen, device=DEVICE) * (1.5 / math.sqrt(i)), torch.randn(g, o, generator=gen, device=DEVICE) * 0.1)
            for i, o in zip(d, d[1:])]


def rows(case, seed):
    """what the nets read, and what the router chooses by"""
    gen = torch.Generator(DEVICE).manual_seed(int(seed) + 7_000_003)
    d, g, n = dims_of(case), case["agents"], case["n"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEVICE)

    if case["op"] == "forward":
        return dict(x=uniform(*((n, d[0]) if case["shared"] else (g, n, d[0]))) * 2 - 1)
    made = dict(x=uniform(n, d[0]) * 2 - 1, router_w=normal(g, d[0]) / math.sqrt(d[0]), router_b=normal(g) * 0.1, allowed=None)
    if case["masked"]:                                                 # a third withheld; now and then nothing is left
        made["allowed"] = ((uniform(n, g) > 0.33) & (uniform(n, 1) > 0.06)).to(torch.uint8)
    if case["op"] == "grad":
        made.update(y=normal(n, case["top_k"], d[1]), dout=normal(n, d[1]))
    return made


def packed(w):
    """weights in 4 bits: codes, two to a byte along the inputs, and the scales' exponents, one for 32 inputs"""
    g, o, i = w.shape
    w = torch.nn.functional.pad(w, (0, -i % BLOCK)).view(g, o, -1, BLOCK)
    mantissa, exponent = torch.frexp(w.abs().amax(-1))
    scale = torch.where(mantissa <= 0.75, exponent - 3, exponent - 2)          # the least power of two that keeps the block within 6
    scale = torch.where(mantissa == 0, torch.full_like(scale, -127), scale)
    v = torch.ldexp(w.abs(), -scale[..., None].clamp(min=-100))
    code = sum((v > t) if even else (v >= t) for t, even in                    # to the nearest, halves to the even code
               ((0.25, 1), (0.75, 0), (1.25, 1), (1.75, 0), (2.5, 1), (3.5, 0), (5.0, 1))).to(torch.uint8)
    code = (code | ((w < 0) & (code > 0)).to(torch.uint8) << 3).view(g, o, -1)
    return code[..., 0::2] | code[..., 1::2] << 4, (scale + 127).to(torch.uint8)


def prepare(case, seed):
    state = dict(case=case, **rows(case, seed))
    d, g, n = dims_of(case), case["agents"], case["n"]
    if case["op"] == "grad":
        state["idx"], state["prob"] = choose(state)
    bits = 4 if case["op"] == "forward" else case.get("bits", 32)
    if own:
        import ddrl_amd
        kinds = dict(linear=0, leaky=1, tanh=2, relu=3)
        hidden, last = (kinds[a] for a in case.get("acts", "leaky-tanh").split("-"))
        if case["op"] != "grad":
            flat = torch.cat([t.reshape(g, -1) for layer in nets(case, seed) for t in layer], 1)
            snap = ddrl_amd.PolicySnapshot.shaped(g, d[0], d[-1], d[1:-1], hidden, last, bits=bits)
            snap.load_flat_dev(flat.data_ptr(), flat.shape[1])
            torch.cuda.synchronize()
        else:
            snap = ddrl_amd.PolicySnapshot.shaped(g, d[0], d[-1], [], hidden, last, bits=bits)
        state["snap"] = snap
        stream = torch.cuda.current_stream().cuda_stream
        new = functools.partial(torch.empty, device=DEVICE)
        if case["op"] == "forward":
            state["out"] = new(g, n, d[-1])
            state["args"] = snap.forward_args(n, state["x"].data_ptr(), state["out"].data_ptr(), x_agent=0 if case["shared"] else None,
                                              stream=stream)
        elif case["op"] == "mixture":
            k = case["top_k"]
            state.update(out=new(n, d[-1]), idx=new(n, k, dtype=torch.int32), prob=new(n, k), y=new(n, k, d[-1]),
                         space=new(max(1, snap.mixture_workspace(n, k)), dtype=torch.uint8))
            state["args"] = snap.mixture_args(n, k, state["x"].data_ptr(), state["router_w"].data_ptr(), state["out"].data_ptr(),
                                              router_b=state["router_b"].data_ptr(), idx=state["idx"].data_ptr(),
                                              prob=state["prob"].data_ptr(), y=state["y"].data_ptr(),
                                              allowed=state["allowed"].data_ptr() if case["masked"] else 0,
                                              workspace=state["space"].data_ptr(), workspace_bytes=state["space"].numel(), stream=stream)
        else:
            k = case["top_k"]
            state.update(dw=new(g, d[0]), db=new(g), dy=new(n, k, d[-1]),
                         space=new(max(1, snap.mixture_grad_workspace(n, k)), dtype=torch.uint8))
            state["args"] = snap.mixture_grad_args(n, k, state["x"].data_ptr(), state["idx"].data_ptr(), state["prob"].data_ptr(),
                                                   state["y"].data_ptr(), state["dout"].data_ptr(), state["dw"].data_ptr(),
                                                   state["db"].data_ptr(), dy=state["dy"].data_ptr(),
                                                   workspace=state["space"].data_ptr(), workspace_bytes=state["space"].numel(),
                                                   stream=stream)
    elif case["op"] != "grad":
        state["layers"] = [(*packed(w), b) if bits == 4 else (w, b) for w, b in nets(case, seed)]
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        if op == "forward":
            state["snap"].forward_dev(state["args"])
            return state["out"]
        if op == "mixture":
            state["snap"].mixture_dev(state["args"])
            return dict(out=state["out"], idx=state["idx"], prob=state["prob"], y=state["y"])
        state["snap"].mixture_grad_dev(state["args"])
        return dict(dw=state["dw"], db=state["db"], dy=state["dy"])
    return dict(forward=plain_forward, mixture=plain_mixture, grad=plain_grad)[op](state)


def activation(kind, z):
    return dict(linear=lambda: z, leaky=lambda: torch.where(z > 0, z, 0.01 * z), tanh=lambda: torch.tanh(z),
                relu=lambda: torch.clamp(z, min=0))[kind]()


def matrix(layer, inputs):
    """a layer's weights as 32-bit numbers"""
    if len(layer) == 2:
        return layer[0]
    pairs, scales, _ = layer
    code = torch.stack((pairs & 15, pairs >> 4), -1).flatten(-2)
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=pairs.device)
    scale = torch.ldexp(torch.ones((), device=pairs.device), scales.int() - 127)
    return (grid[code.int()].unflatten(-1, (-1, BLOCK)) * scale[..., None]).flatten(-2)[..., :inputs]


def through(case, layers, h):
    """h [nets, inputs, rows] through the nets"""
    kinds = case["acts"].split("-")

    def step(h, at):
        z = torch.bmm(matrix(layers[at], h.shape[1]), h) + layers[at][-1][..., None]
        return activation(kinds[at == len(layers) - 1], z)

    return functools.reduce(step, range(len(layers)), h)


def plain_forward(state):
    x = state["x"]
    h = x.T.expand(state["case"]["agents"], -1, -1).contiguous() if x.dim() == 2 else x.transpose(1, 2).contiguous()
    return through(state["case"], state["layers"], h).transpose(1, 2).contiguous()


def choose(state):
    """the router: the top_k largest of the allowed logits, the lower index first among equals, and the softmax over them"""
    logits = state["x"].double() @ state["router_w"].double().T + state["router_b"].double()
    if state["allowed"] is not None:
        logits = torch.where(state["allowed"] != 0, logits, -math.inf)
    value, idx = torch.sort(logits, dim=1, descending=True, stable=True)
    value, idx = value[:, :state["case"]["top_k"]], idx[:, :state["case"]["top_k"]]
    left = value > -math.inf
    weight = torch.where(left, torch.exp(value - torch.where(left[:, :1], value[:, :1], 0.0)), 0.0)
    prob = weight / torch.where(left[:, :1], weight.sum(1, keepdim=True), 1.0)
    return torch.where(left, idx, -1).int(), prob.float()


def plain_mixture(state):
    idx, prob = choose(state)
    n, k = idx.shape
    at = idx.clamp(min=0).flatten()
    chosen = [tuple(t[at] for t in layer) for layer in state["layers"]]
    y = through(state["case"], chosen, state["x"].repeat_interleave(k, 0)[..., None]).view(n, k, -1)
    y = torch.where((idx >= 0)[..., None], y, 0.0)
    return dict(out=(prob[..., None] * y).sum(1), idx=idx, prob=prob, y=y)


def plain_grad(state):
    idx, prob, y, dout = state["idx"], state["prob"], state["y"], state["dout"]
    g, s = state["router_w"].shape
    score = (y * dout[:, None]).sum(-1)
    dlogit = prob * (score - (prob * score).sum(1, keepdim=True))
    dlogit = torch.where(idx >= 0, dlogit, 0.0)
    at = idx.clamp(min=0).flatten()
    dw = torch.zeros(g, s, dtype=torch.float64, device=idx.device)
    dw.index_add_(0, at, (dlogit[..., None] * state["x"][:, None]).flatten(0, 1).double())
    db = torch.zeros(g, dtype=torch.float64, device=idx.device)
    db.index_add_(0, at, dlogit.flatten().double())
    return dict(dw=dw.float(), db=db.float(), dy=prob[..., None] * dout[:, None])


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------------

def stands_for(w):
    """what weights rounded to 4 bits stand for, from the definition: per 32 inputs the least power of two s with max |w| <= 6 s,
    each weight to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times s, halves to the even one of the two neighbours"""
    w = w.double()
    g, o, i = w.shape
    blocks = torch.cat((w, w.new_zeros(g, o, -i % BLOCK)), 2).reshape(g, o, -1, BLOCK)
    most = blocks.abs().max(3, keepdim=True).values
    s = torch.where(most > 0, torch.exp2(torch.ceil(torch.log2(most.clamp(min=1e-300) / 6))), torch.ones_like(most))
    v = blocks / s
    grid = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return (torch.round(v / grid) * grid * s).reshape(g, o, -1)[:, :, :i]


def exact(case, seed):
    made = rows(case, seed)
    x = made["x"].double()
    if case["op"] == "grad":
        idx, prob = choose(dict(made, case=case))
        y, dout, p = made["y"].double(), made["dout"].double(), prob.double()
        n, k = idx.shape
        score = torch.einsum("nka,na->nk", y, dout)
        dlogit = p * score - p * (p * score).sum(1)[:, None]
        pick = idx.long()[..., None] == torch.arange(case["agents"], device=idx.device)          # [n, k, agents]
        spread = (pick * dlogit[..., None]).sum(1)
        return dict(dw=spread.T @ x, db=spread.sum(0), dy=p[..., None] * dout[:, None, :])
    four = case["op"] == "forward" or case["bits"] == 4
    function = dict(linear=lambda z: z, relu=lambda z: torch.relu(z), tanh=lambda z: z.tanh(), leaky=lambda z: torch.maximum(z, z / 100))
    hidden, last = (function[a] for a in case["acts"].split("-"))
    made_nets = [(stands_for(w) if four else w.double(), b.double()) for w, b in nets(case, seed)]

    def answer(h, which):
        for at, (w, b) in enumerate(made_nets):
            w, b = w[which], b[which]
            h = (h.unsqueeze(-2) @ w.transpose(-1, -2).contiguous()).squeeze(-2) + b if h.dim() == 2 else h @ w.transpose(-1, -2).contiguous() + b[:, None]
            h = last(h) if at == len(made_nets) - 1 else hidden(h)
        return h

    if case["op"] == "forward":
        parts = [slice(i, min(i + 64, case["agents"])) for i in range(0, case["agents"], 64)]
        return torch.cat([answer(x.expand(p.stop - p.start, -1, -1) if case["shared"] else x[p], p) for p in parts])
    logits = (x[:, None, :] * made["router_w"].double()[None]).sum(2) if x.shape[0] * case["agents"] < 300_000 else x @ made["router_w"].double().T
    logits = logits + made["router_b"].double()
    barred = made["allowed"] == 0 if case["masked"] else torch.zeros_like(logits, dtype=torch.bool)
    value, idx = torch.topk(logits.masked_fill(barred, -math.inf), case["top_k"], dim=1)
    none = torch.isinf(value)
    p = torch.softmax(value, 1).masked_fill(none, 0.0)
    p = torch.where(none.all(1, keepdim=True), torch.zeros_like(p), p)
    k = case["top_k"]
    ys = [answer(x, idx[:, j]).masked_fill(none[:, j, None], 0.0) for j in range(k)]
    y = torch.stack(ys, 1)
    return dict(out=(p[..., None] * y).sum(1), idx=None, prob=p, y=y)
