"""Cases of the plan operators for adapted, normalised and recurrent models, with their plain forms.

    group_norm       act(gamma (x - mean) / sqrt(var + eps) + beta) over groups of channels
    linear_adapters  act(X W^T + b + s_i (X A_i^T) U_i^T), one adapter i per row beside a shared projection
    recurrence       h_t = f h_(t-1) + (1 - f) x_t with f = sigmoid(gate), over the steps of every sequence

Where `own` is false, run() computes them with elementary torch operations; where it is true, it runs the plan that
prepare() built.  The plan owns its tensors, as in any program that uses the library: prepare() fills the input
tensors in place, which is what a gather kernel or the operation before it does.
"""
import math

import torch

own = False

DEV = "cuda"


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # every row of a recurrent state normalised by itself, four heads of 16: 15 levels of 4736 ocean cells
        dict(name="norm_rows", op="norm", samples=71040, positions=1, channels=64, groups=4, first=False, act="silu"),
        # the full-resolution level of a 256 x 256 image network
        dict(name="norm_image", op="norm", samples=1, positions=65536, channels=32, groups=8, first=False, act="silu"),
        # the upsampled volume of a 33^3 -> 66^3 super-resolution network: the largest
        dict(name="norm_volume", op="norm", samples=1, positions=287496, channels=64, groups=8, first=False, act="leaky"),
        # the bottleneck of the image network in the convolutions' own order, channels first: the smallest
        dict(name="norm_bottleneck", op="norm", samples=1, positions=1024, channels=256, groups=8, first=True, act="relu"),
        # one column asks: the weights of the projection are what is read
        dict(name="adapt_row", op="adapt", rows=1, K=768, N=768, rank=8, adapters=64, order="mixed", act="leaky"),
        # a few dozen clients at once, each with its own adapter
        dict(name="adapt_requests", op="adapt", rows=48, K=768, N=768, rank=16, adapters=64, order="mixed", act="silu"),
        # a hidden layer over all columns of a climate grid, one adapter per region, columns in any order
        dict(name="adapt_columns", op="adapt", rows=24576, K=768, N=768, rank=16, adapters=24, order="mixed", act="leaky"),
        # the first layer of a stencil network: rows of 27 floats, regions in bands
        dict(name="adapt_cells", op="adapt", rows=71040, K=27, N=64, rank=4, adapters=15, order="bands", act="relu"),
        # the head of the climate network on a part of the grid: no size is a multiple of a tile
        dict(name="adapt_head", op="adapt", rows=4099, K=556, N=368, rank=12, adapters=7, order="mixed", act=None),
        # one time step of every ocean cell with the state kept on the device
        dict(name="recur_step", op="recur", seqs=4736, steps=1, channels=64, time_major=True, ragged=False, reverse=False),
        # up the water column, every cell as deep as its sea floor
        dict(name="recur_columns", op="recur", seqs=4736, steps=15, channels=64, time_major=True, ragged=True, reverse=True),
        # two long records, one behind the other
        dict(name="recur_long", op="recur", seqs=2, steps=32768, channels=384, time_major=False, ragged=False, reverse=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "adapt", "recur"])
    if op == "norm":
        groups = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
        per = rng.choice([1, 2, 3, 4, 7, 8, 12, 16, 24, 32])
        c = groups * per
        samples = _log(rng, 1, 71040)
        most = 287496 * 64 // (samples * c)
        return dict(op="norm", samples=samples, positions=_log(rng, 1, max(1, min(287496, most))), channels=c, groups=groups,
                    first=rng.random() < 0.3, act=rng.choice([None, "relu", "leaky", "silu"]))
    if op == "adapt":
        k, n = _log(rng, 9, 768), _log(rng, 3, 768)
        return dict(op="adapt", rows=_log(rng, 1, 24576), K=k, N=n, rank=_log(rng, 1, 32) if k * n < 300000 else _log(rng, 1, 16),
                    adapters=_log(rng, 1, 64) if k * n < 300000 else _log(rng, 1, 24), order=rng.choice(["mixed", "bands"]),
                    act=rng.choice([None, "relu", "leaky", "silu"]))
    ch = _log(rng, 3, 384)
    seqs = _log(rng, 1, 4736)
    most = 2 * 32768 * 384 // (seqs * ch)
    return dict(op="recur", seqs=seqs, steps=_log(rng, 1, max(1, min(32768, most))), channels=ch, time_major=rng.random() < 0.5,
                ragged=rng.random() < 0.4, reverse=rng.random() < 0.4)


ALPHA = {"norm": 0.2, "adapt": 0.15}
EPS = 1e-5


# ---- inputs ------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    n = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    u = lambda *s: torch.rand(*s, device=DEV, generator=g)  # noqa: E731
    if case["op"] == "norm":
        b, s, c = case["samples"], case["positions"], case["channels"]
        x = n(b, c, s) if case["first"] else n(b, s, c)
        v = (lambda t: t[:, None]) if case["first"] else (lambda t: t)
        x = x * v(0.5 + u(c)) + v(2.0 * n(c))
        return dict(x=x, gamma=1.0 + 0.2 * n(c), beta=0.1 * n(c))
    if case["op"] == "adapt":
        b, k, m, r, a = case["rows"], case["K"], case["N"], case["rank"], case["adapters"]
        if case["order"] == "bands":
            index = torch.arange(b, device=DEV) * a // b
        else:
            index = (u(b) * a).long().clamp_(max=a - 1)
        index = torch.where(u(b) < 0.06, torch.full_like(index, -1), index).to(torch.int32)
        return dict(x=n(b, k), index=index, W=n(m, k) / math.sqrt(k), bias=0.1 * n(m), A=n(a, r, k) / math.sqrt(k),
                    U=0.5 * n(a, m, r) / math.sqrt(r), scale=0.5 + 1.5 * u(a))
    q, t, c = case["seqs"], case["steps"], case["channels"]
    src = n(t, q, 2 * c) if case["time_major"] else n(q, t, 2 * c)
    src[..., :c] = 1.5 * src[..., :c] + 1.0          # gates lean towards keeping the state
    d = dict(src=src, state=n(q, c))
    if case["ragged"]:
        # about one sequence in sixteen has no valid step (a land cell)
        d["lengths"] = ((u(q) * 17.0 - 1.0).clamp_(min=0.0) * t / 16.0).ceil().clamp_(max=t).to(torch.int32)
    return d


class _Memory:
    """A plan's tensor as torch sees it."""

    def __init__(self, plan, tensor, shape, kind):
        self.plan = plan
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr=kind, data=(plan.ptr(tensor), False), version=2)


class _Held:
    """Keeps a plan for as long as the state that names its tensors."""

    def __init__(self, plan):
        self.plan = plan
        self.run = plan.run

    def view(self, tensor, shape, kind="<f4"):
        t = torch.as_tensor(_Memory(self, tensor, shape, kind), device=DEV)
        assert t.data_ptr() == self.ptr(tensor)
        return t

    def ptr(self, tensor):
        return self.plan.ptr(tensor)

    def __del__(self):
        torch.cuda.synchronize()
        self.plan.close()
        from fortis_amd import lib
        lib().fortis_pool_trim()


def prepare(case, seed):
    d = _inputs(case, seed)
    if not own:
        if case["op"] == "recur":
            d["y"] = torch.zeros_like(d["src"][..., :case["channels"]]).contiguous()
        return dict(case=case, **d)
    from fortis_amd.plan import Plan
    host = lambda t: t.cpu().numpy()  # noqa: E731
    p = Plan()
    if case["op"] == "norm":
        b, s, c = case["samples"], case["positions"], case["channels"]
        t, o = p.tensor(b * s * c), p.tensor(b * s * c)
        p.group_norm(t, o, b, s, c, case["groups"], host(d["gamma"]), host(d["beta"]), eps=EPS, act=case["act"], alpha=ALPHA["norm"],
                     channels_first=case["first"])
        h = _Held(p.finalize(t, o))
        h.view(t, d["x"].shape).copy_(d["x"])
        return dict(case=case, run=h.run, out=h.view(o, d["x"].shape))
    if case["op"] == "adapt":
        b, k, m = case["rows"], case["K"], case["N"]
        t, i, o = p.tensor(b * k), p.tensor(b), p.tensor(b * m)
        p.linear_adapters(t, o, i, host(d["W"]), host(d["bias"]), host(d["A"]), host(d["U"]), b, host(d["scale"]), act=case["act"],
                          alpha=ALPHA["adapt"])
        h = _Held(p.finalize(t, o))
        h.view(t, (b, k)).copy_(d["x"])
        h.view(i, (b,), "<i4").copy_(d["index"])
        return dict(case=case, run=h.run, out=h.view(o, (b, m)))
    q, n, c = case["seqs"], case["steps"], case["channels"]
    t, o, h0, h1 = p.tensor(q * n * 2 * c), p.tensor(q * n * c), p.tensor(q * c), p.tensor(q * c)
    le = p.tensor(q) if case["ragged"] else -1
    p.recurrence(t, o, q, n, c, h_in=h0, h_out=h1, lengths=le, time_major=case["time_major"], reverse=case["reverse"])
    h = _Held(p.finalize(t, o))
    h.view(t, d["src"].shape).copy_(d["src"])
    h.view(h0, (q, c)).copy_(d["state"])
    if le >= 0:
        h.view(le, (q,), "<i4").copy_(d["lengths"])
    y = h.view(o, d["src"].shape[:2] + (c,))
    y.zero_()                                        # steps at and behind a sequence's length are not written
    return dict(case=case, run=h.run, out=dict(y=y, state=h.view(h1, (q, c))))


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _act(v, act, alpha):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "leaky":
        return torch.where(v > 0, v, alpha * v)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _norm(s):
    c = s["case"]
    b, g, per = c["samples"], c["groups"], c["channels"] // c["groups"]
    first = c["first"]
    x = s["x"].view((b, g, per, -1) if first else (b, -1, g, per))
    dims = (2, 3) if first else (1, 3)
    count = x.numel() // (b * g)
    mean = x.sum(dims, keepdim=True) / count
    dev = x - mean
    var = (dev * dev).sum(dims, keepdim=True) / count
    v = (g, per, 1) if first else (g, per)
    y = dev / torch.sqrt(var + EPS) * s["gamma"].view(v) + s["beta"].view(v)
    return _act(y, c["act"], ALPHA["norm"]).view(s["x"].shape)


def _adapt(s):
    c = s["case"]
    b, n, r, a = c["rows"], c["N"], c["rank"], c["adapters"]
    index = s["index"].long()
    row = torch.arange(b, device=DEV)
    low = (s["x"] @ s["A"].view(a * r, -1).t()).view(b, a, r)
    keep = torch.where(index >= 0, s["scale"][index.clamp(min=0)], torch.zeros_like(s["scale"][:1]))
    low = low[row, index.clamp(min=0)] * keep[:, None]
    spread = torch.zeros(b, a, r, device=DEV)
    spread[row, index.clamp(min=0)] = low
    y = s["x"] @ s["W"].t() + spread.view(b, a * r) @ s["U"].permute(0, 2, 1).reshape(a * r, n)
    return _act(y + s["bias"], c["act"], ALPHA["adapt"])


def _recur(s):
    c = s["case"]
    ch, steps = c["channels"], c["steps"]
    src = s["src"] if c["time_major"] else s["src"].transpose(0, 1)
    gate, x = src[..., :ch], src[..., ch:]
    f = 1.0 / (1.0 + torch.exp(-gate))
    v = x / (1.0 + torch.exp(gate))
    valid = None
    if "lengths" in s:
        valid = (torch.arange(steps, device=DEV)[:, None] < s["lengths"][None, :].long())[..., None]
        f, v = torch.where(valid, f, torch.ones_like(f)), torch.where(valid, v, torch.zeros_like(v))
    if c["reverse"]:
        f, v = f.flip(0), v.flip(0)
    v = torch.cat([v[:1] + f[:1] * s["state"], v[1:]])
    d = 1
    while d < steps:                                 # after a pass of distance d a place holds the last 2 d steps
        v = torch.cat([v[:d], v[d:] + f[d:] * v[:-d]])
        f = torch.cat([f[:d], f[d:] * f[:-d]])
        d *= 2
    state = v[-1].clone()
    if c["reverse"]:
        v = v.flip(0)
    y = s["y"] if c["time_major"] else s["y"].transpose(0, 1)
    y.copy_(v if valid is None else torch.where(valid, v, y))
    return dict(y=s["y"], state=state)


def run(state):
    if own:
        state["run"]()
        return state["out"]
    return {"norm": _norm, "adapt": _adapt, "recur": _recur}[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        e = case["samples"] * case["positions"] * case["channels"]
        return dict(bytes=8 * e + 8 * case["channels"], flops=8 * e)
    if case["op"] == "adapt":
        b, k, n, r = case["rows"], case["K"], case["N"], case["rank"]
        used = min(case["adapters"], b)
        return dict(bytes=4 * (b * k + b * n + n * k + n + b + used * (r * (k + n) + 1)), flops=2 * b * n * k + 2 * b * r * (k + n))
    e = case["seqs"] * case["steps"] * case["channels"]
    if case["ragged"]:
        e = e // 2                                   # lengths are spread evenly from none to all steps
    s = case["seqs"] * case["channels"]
    return dict(bytes=12 * e + 8 * s + (4 * case["seqs"] if case["ragged"] else 0), flops=10 * e)


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------------
def exact(case, seed):
    d = {k: (t if t.dtype == torch.int32 else t.double()) for k, t in _inputs(case, seed).items()}
    if case["op"] == "norm":
        x = d["x"] if case["first"] else d["x"].transpose(1, 2)              # [sample][channel][position]
        b, c, g = case["samples"], case["channels"], case["groups"]
        rows = x.reshape(b * g, -1)
        mean = rows.mean(1, keepdim=True)
        y = ((rows - mean) * (rows.var(1, unbiased=False, keepdim=True) + EPS).rsqrt()).view(b, c, -1)
        y = y * d["gamma"][:, None] + d["beta"][:, None]
        y = _act64(y, case["act"], ALPHA["norm"])
        return y if case["first"] else y.transpose(1, 2)
    if case["op"] == "adapt":
        y = d["x"] @ d["W"].t() + d["bias"]
        for i in range(case["adapters"]):
            rows = torch.nonzero(d["index"] == i).flatten()
            if rows.numel():
                y[rows] += d["scale"][i] * ((d["x"][rows] @ d["A"][i].t()) @ d["U"][i].t())
        return _act64(y, case["act"], ALPHA["adapt"])
    ch, steps = case["channels"], case["steps"]
    src = d["src"] if case["time_major"] else d["src"].transpose(0, 1)
    f = torch.sigmoid(src[..., :ch])
    add = torch.sigmoid(-src[..., :ch]) * src[..., ch:]
    h, y = d["state"], torch.zeros_like(f)
    for t in (reversed(range(steps)) if case["reverse"] else range(steps)):
        new = torch.addcmul(add[t], f[t], h)
        if case["ragged"]:
            on = (d["lengths"] > t)[:, None]
            new = torch.where(on, new, h)
            y[t] = torch.where(on, new, y[t])
        else:
            y[t] = new
        h = new
    return dict(y=y if case["time_major"] else y.transpose(0, 1), state=h)


def _act64(v, act, alpha):
    if act == "relu":
        return v.clamp(min=0)
    if act == "leaky":
        return torch.maximum(v, alpha * v)
    if act == "silu":
        return v * torch.sigmoid(v)
    return v
