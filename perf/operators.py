"""Timed cases of the operators of layered recurrent models: the gated linear recurrence and the matrix
product with bias, activation and residual in its epilogue.

Three kinds of case:

* ``scan``: ``h_t = z_t h_{t-1} + (1 - z_t) n_t`` with ``z = sigmoid``, ``n = tanh`` (or the value itself) of the two
  halves of ``gi[T, B, 2H]``; a whole sequence (``T`` > 0), with its gradients where ``train``, over ragged
  sequences where ``ragged``, or one token of a served batch (``T`` = 0: the step form).
* ``linear``: ``act(x W^T + b) + residual``, with its gradients where ``train``.
* ``block``: product, scan, product and residual one after the other, as a layer of a model has them.

Every state is float32; ``dtype`` is the type of all other tensors.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _scan(name, dtype, T, B, H, **options):
    case = dict(name=name, op="scan", dtype=dtype, T=T, B=B, H=H, train=False, ragged=False, candidate="tanh")
    case.update(options)
    return case


def _linear(name, dtype, M, K, N, **options):
    case = dict(name=name, op="linear", dtype=dtype, M=M, K=K, N=N, train=False, activation="none", residual=False)
    case.update(options)
    return case


def listed():
    return [
        # one frame of one stream, as a streaming recogniser makes it: pure latency
        _scan("scan_step_stream", "float32", 0, 1, 256),
        # one token of every sequence of a served batch
        _scan("scan_step_batch", "bfloat16", 0, 512, 1024),
        # the benchmark's training shape (64 steps, 32 sequences, 512 units)
        _scan("scan_train_short", "float32", 64, 32, 512, train=True),
        # reading one long document before answering: one sequence, so the work has to be found along time
        _scan("scan_long_prompt", "bfloat16", 32768, 1, 1024),
        # training on sequences of varying length, padded to the longest
        _scan("scan_train_ragged", "bfloat16", 1000, 24, 768, train=True, ragged=True),
        # sizes that no tile divides, unsquashed candidate
        _scan("scan_train_odd", "float32", 501, 19, 607, train=True, candidate="identity"),
        # the gates of one token of one stream
        _linear("linear_one_token", "bfloat16", 1, 1024, 2048),
        # a served batch through the wide half of a feed-forward layer
        _linear("linear_batch_tokens", "bfloat16", 48, 1024, 4096, activation="silu"),
        # float32 training on a batch of varying length (41 steps of 257 sequences), narrow input
        _linear("linear_train_ragged", "float32", 10537, 120, 608, activation="gelu", train=True),
        # long-sequence inference, the wide half of a feed-forward layer: the largest product alone
        _linear("linear_infer_wide", "bfloat16", 32768, 1024, 4096, activation="gelu"),
        # training the way back into the residual stream: the largest case
        _linear("linear_train_residual", "bfloat16", 16384, 4096, 1024, residual=True, train=True),
        # a whole recurrent block in training: gates, recurrence, output product with residual
        dict(name="block_train", op="block", dtype="float32", T=128, B=64, K=512, H=512, train=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    kind = rng.choice(["step", "scan", "scan", "scan", "linear", "linear", "linear", "block"])

    def width(low, high):
        # widths are multiples of eight in most models; one in five is not
        w = _log_int(rng, low, high)
        return w if rng.random() < 0.2 else max(8, w // 8 * 8)

    if kind == "step":
        return dict(op="scan", dtype=dtype, T=0, B=_log_int(rng, 1, 1024), H=width(32, 2048), train=False, ragged=False,
                    candidate=rng.choice(["tanh", "identity"]))
    if kind == "scan":
        T, B, H = _log_int(rng, 1, 32768), _log_int(rng, 1, 256), width(32, 2048)
        train = rng.random() < 0.6
        while T * B * H > (2 ** 24 if train else 2 ** 25):
            T, B = max(1, T * 2 // 3), max(1, B * 2 // 3)
        return dict(op="scan", dtype=dtype, T=T, B=B, H=H, train=train, ragged=rng.random() < 0.4,
                    candidate=rng.choice(["tanh", "tanh", "identity"]))
    if kind == "linear":
        M, K, N = _log_int(rng, 1, 32768), width(64, 4096), width(64, 4096)
        train = rng.random() < 0.5
        while M * K * N > (2 ** 33 if dtype == "float32" else 2 ** 36):
            M = max(1, M * 2 // 3)
        return dict(op="linear", dtype=dtype, M=M, K=K, N=N, train=train, residual=rng.random() < 0.4,
                    activation=rng.choice(["none", "relu", "silu", "gelu", "sigmoid", "tanh"]))
    T, B, H = _log_int(rng, 8, 1024), _log_int(rng, 1, 128), width(64, 1024)
    while T * B > 16384:
        T, B = max(1, T * 2 // 3), max(1, B * 2 // 3)
    return dict(op="block", dtype=dtype, T=T, B=B, K=width(64, 1024), H=H, train=rng.random() < 0.7)


# ---- inputs ---------------------------------------------------------------------------------------

def _normal(gen, dtype, *shape, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen).mul_(scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "scan":
        T, B, H = case["T"], case["B"], case["H"]
        gi = torch.randn(max(T, 1), B, 2 * H, device="cuda", generator=gen)
        # gates of a trained layer lean to keeping: memories of about ten steps in the middle, hundreds at the ends
        gi[:, :, :H].add_(torch.linspace(0.0, 5.0, H, device="cuda"))
        gi = gi.to(dtype)
        state["h"] = _normal(gen, torch.float32, B, H, scale=0.3)
        state["gi"] = gi[0] if T == 0 else gi
        state["lengths"] = torch.randint(max(1, T // 4), T + 1, (B,), device="cuda", generator=gen) if case["ragged"] else None
        if case["train"]:
            state["dout"] = _normal(gen, dtype, T, B, H, scale=1e-2)
            state["dh"] = _normal(gen, torch.float32, B, H, scale=1e-2)
        return state
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        state["x"] = _normal(gen, dtype, M, K)
        state["W"] = _normal(gen, dtype, N, K, scale=1.0 / math.sqrt(K))
        state["bias"] = _normal(gen, dtype, N, scale=0.1)
        state["residual"] = _normal(gen, dtype, M, N) if case["residual"] else None
        if case["train"]:
            state["dy"] = _normal(gen, dtype, M, N, scale=1e-2)
        return state
    T, B, K, H = case["T"], case["B"], case["K"], case["H"]
    state["x"] = _normal(gen, dtype, T, B, K)
    state["Wi"] = _normal(gen, dtype, 2 * H, K, scale=1.0 / math.sqrt(K))
    state["bi"] = torch.cat([torch.linspace(0.0, 5.0, H, device="cuda"), torch.zeros(H, device="cuda")]).to(dtype)
    state["Wo"] = _normal(gen, dtype, K, H, scale=1.0 / math.sqrt(H))
    state["bo"] = _normal(gen, dtype, K, scale=0.1)
    state["h"] = _normal(gen, torch.float32, B, H, scale=0.3)
    if case["train"]:
        state["dy"] = _normal(gen, dtype, T, B, K, scale=1e-2)
    return state


# ---- plain forms: elementary operations in 32 bits, rounded once at the end of each operator -------

def _gates(gi, candidate):
    """z, 1 - z, n and dn / dc of the two halves of gi, in gi's own precision."""
    x, c = gi.chunk(2, dim=-1)
    z, keep = 1.0 / (1.0 + torch.exp(-x)), 1.0 / (1.0 + torch.exp(x))
    n = torch.tanh(c) if candidate == "tanh" else c
    slope = 1.0 - n * n if candidate == "tanh" else torch.ones_like(n)
    return z, keep, n, slope


def _valid(lengths, T, device):
    """[T, B, 1]: whether a step lies inside its sequence."""
    return None if lengths is None else (torch.arange(T, device=device)[:, None] < lengths[None, :])[:, :, None]


def _prefix(a, b):
    """h_t = a_t h_{t-1} + b_t from h = 0, by doubling the span that each step has seen."""
    span = 1
    while span < a.shape[0]:
        b = torch.cat([b[:span], b[span:] + a[span:] * b[:-span]])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return b


def _scan_plain(gi, h0, lengths, candidate):
    T = gi.shape[0]
    z, keep, n, _ = _gates(gi.float(), candidate)
    u, valid = keep * n, _valid(lengths, T, gi.device)
    if valid is not None:
        z, u = torch.where(valid, z, 1.0), torch.where(valid, u, 0.0)
    u = torch.cat([u[:1] + z[:1] * h0, u[1:]])
    h = _prefix(z, u)
    out = h if valid is None else torch.where(valid, h, 0.0)
    return out.to(gi.dtype), h[-1], h


def _scan_plain_backward(gi, h0, lengths, candidate, h, dout, dh):
    z, keep, n, slope = _gates(gi.float(), candidate)
    valid, dout = _valid(lengths, gi.shape[0], gi.device), dout.float()
    a = z if valid is None else torch.where(valid, z, 1.0)
    b = z * dout if valid is None else torch.where(valid, z * dout, 0.0)
    b = torch.cat([b[:-1], b[-1:] + a[-1:] * dh])
    G = _prefix(a.flip(0), b.flip(0)).flip(0)
    g = dout + torch.cat([G[1:], dh[None]])
    before = torch.cat([h0[None], h[:-1]])
    dgi = torch.cat([g * (before - n) * z * keep, g * keep * slope], dim=-1)
    if valid is not None:
        dgi = torch.where(valid, dgi, 0.0)
    return dgi.to(gi.dtype), G[0]


def _activation(pre, name):
    """The activation and its slope, in pre's own precision."""
    if name == "none":
        return pre, torch.ones_like(pre)
    if name == "relu":
        return torch.where(pre > 0, pre, 0.0), (pre > 0).to(pre.dtype)
    if name == "tanh":
        y = torch.tanh(pre)
        return y, 1.0 - y * y
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(pre * math.sqrt(0.5)))
        return pre * cdf, cdf + pre * torch.exp(-0.5 * pre * pre) * (1.0 / math.sqrt(2.0 * math.pi))
    s = 1.0 / (1.0 + torch.exp(-pre))
    return (s, s * (1.0 - s)) if name == "sigmoid" else (pre * s, s * (1.0 + pre * (1.0 - s)))


def _linear_plain(x, W, bias, activation, residual):
    y, slope = _activation(x.float() @ W.float().t() + bias.float(), activation)
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype), slope


def _linear_plain_backward(x, W, slope, dy):
    d = (dy.float() * slope).reshape(-1, W.shape[0])
    flat = x.float().reshape(-1, x.shape[-1])
    dx = (d @ W.float()).reshape(x.shape)
    return dx.to(x.dtype), (d.t() @ flat).to(x.dtype), d.sum(0).to(x.dtype)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "scan":
        gi, h0, lengths = state["gi"], state["h"], state["lengths"]
        if case["T"] == 0:
            out, h_T, _ = _scan_plain(gi[None], h0, None, case["candidate"])
            return out[0], h_T
        out, h_T, h = _scan_plain(gi, h0, lengths, case["candidate"])
        if not case["train"]:
            return out, h_T
        return (out, h_T, *_scan_plain_backward(gi, h0, lengths, case["candidate"], h, state["dout"], state["dh"]))
    if case["op"] == "linear":
        x, W = state["x"], state["W"]
        y, slope = _linear_plain(x, W, state["bias"], case["activation"], state["residual"])
        if not case["train"]:
            return y
        return (y, *_linear_plain_backward(x, W, slope, state["dy"]))
    x, h0 = state["x"], state["h"]
    gi, slope_i = _linear_plain(x, state["Wi"], state["bi"], "none", None)
    out, h_T, h = _scan_plain(gi, h0, None, "tanh")
    y, slope_o = _linear_plain(out, state["Wo"], state["bo"], "none", x)
    if not case["train"]:
        return y, h_T
    dout, dWo, dbo = _linear_plain_backward(out, state["Wo"], slope_o, state["dy"])
    dgi, dh0 = _scan_plain_backward(gi, h0, None, "tanh", h, dout, torch.zeros_like(h0))
    dx, dWi, dbi = _linear_plain_backward(x, state["Wi"], slope_i, dgi)
    dx = (dx.float() + state["dy"].float()).to(x.dtype)
    return y, h_T, dx, dWi, dbi, dWo, dbo, dh0


# ---- the framework's calls -------------------------------------------------------------------------

def _leaves(*tensors):
    return [t.detach().requires_grad_(True) for t in tensors]


def _run_own(state):
    from gru_triton_b200.linear_act import linear_act
    from gru_triton_b200.scan_gated import gated_scan, gated_step

    case = state["case"]
    if case["op"] == "scan":
        gi, h0, kind = state["gi"], state["h"], case["candidate"]
        if case["T"] == 0:
            return gated_step(gi, h0, candidate=kind)
        if not case["train"]:
            return gated_scan(gi, h0, lengths=state["lengths"], candidate=kind)
        gi, h0 = _leaves(gi, h0)
        out, h_T = gated_scan(gi, h0, lengths=state["lengths"], candidate=kind)
        return (out.detach(), h_T.detach(), *torch.autograd.grad((out, h_T), (gi, h0), (state["dout"], state["dh"])))
    if case["op"] == "linear":
        x, W, bias, residual = state["x"], state["W"], state["bias"], state["residual"]
        if not case["train"]:
            return linear_act(x, W, bias, activation=case["activation"], residual=residual)
        x, W, bias = _leaves(x, W, bias)
        y = linear_act(x, W, bias, activation=case["activation"], residual=residual)
        return (y.detach(), *torch.autograd.grad(y, (x, W, bias), state["dy"]))
    names = ("x", "Wi", "bi", "Wo", "bo", "h")
    x, Wi, bi, Wo, bo, h0 = _leaves(*(state[k] for k in names)) if case["train"] else [state[k] for k in names]
    out, h_T = gated_scan(linear_act(x, Wi, bi), h0)
    y = linear_act(out, Wo, bo, residual=x)
    if not case["train"]:
        return y, h_T
    return (y.detach(), h_T.detach(), *torch.autograd.grad(y, (x, Wi, bi, Wo, bo, h0), state["dy"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    size = 4.0 if case["dtype"] == "float32" else 2.0
    if case["op"] == "scan":
        T, B, H = max(1, case["T"]), case["B"], case["H"]
        rows = T * B
        inside = rows * (0.625 if case["ragged"] else 1.0)         # mean length of a ragged batch; outputs are written whole
        moved = size * (2 * inside * H + rows * H) + 8.0 * B * H
        flops = 16.0 * inside * H
        if case["train"]:
            moved += size * (inside * H + 2 * rows * H) + 8.0 * B * H    # dout in, dgi out (gi is read once)
            flops += 20.0 * inside * H
        return {"bytes": moved, "flops": flops}
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        moved = size * (M * K + N * K + N + M * N * (2 if case["residual"] else 1))
        flops = 2.0 * M * N * K
        if case["train"]:
            moved += size * (M * N + M * K + N * K + N)
            flops *= 3
        return {"bytes": moved, "flops": flops}
    rows, K, H, B = case["T"] * case["B"], case["K"], case["H"], case["B"]
    moved = size * (2 * rows * K + 3 * H * K + 2 * H + K) + 8.0 * B * H
    flops = rows * (2.0 * 3 * H * K + 16.0 * H)
    if case["train"]:
        moved += size * (2 * rows * K + 3 * H * K + 2 * H + K) + 4.0 * B * H
        flops += rows * (4.0 * 3 * H * K + 20.0 * H)
    return {"bytes": moved, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------------

def _exact_scan(gi, h0, lengths, candidate):
    """gi, h0 in 64 bits -> every state [T + 1, B, H], one step after the other; a step behind its sequence keeps the state."""
    H = h0.shape[1]
    z = torch.sigmoid(gi[..., :H])
    n = gi[..., H:].tanh() if candidate == "tanh" else gi[..., H:]
    u = torch.sigmoid(-gi[..., :H]) * n
    if lengths is not None:
        behind = torch.arange(gi.shape[0], device=gi.device)[:, None] >= lengths
        z, u = z.masked_fill(behind[..., None], 1.0), u.masked_fill(behind[..., None], 0.0)
    states = torch.empty(gi.shape[0] + 1, *h0.shape, device=gi.device, dtype=torch.float64)
    states[0] = h0
    for t in range(gi.shape[0]):
        torch.addcmul(u[t], z[t], states[t], out=states[t + 1])
    return states


def _exact_scan_backward(gi, states, lengths, candidate, dout, dh):
    T, H = gi.shape[0], states.shape[-1]
    x, c = gi[..., :H], gi[..., H:]
    z = torch.sigmoid(x)
    n = c.tanh() if candidate == "tanh" else c
    behind = None
    if lengths is not None:
        behind = (torch.arange(T, device=gi.device)[:, None] >= lengths)[..., None]
        dout = dout.masked_fill(behind, 0.0)
    pass_on = z if behind is None else z.masked_fill(behind, 1.0)
    g, G = torch.empty_like(dout), dh
    for t in reversed(range(T)):
        torch.add(dout[t], G, out=g[t])
        G = pass_on[t] * g[t]
    dx = g * (states[:-1] - n) * z * torch.sigmoid(-x)
    dc = g * torch.sigmoid(-x)
    if candidate == "tanh":
        dc = dc / c.cosh() ** 2
    dgi = torch.cat([dx, dc], dim=-1)
    return dgi if behind is None else dgi.masked_fill(behind, 0.0), G


_EXACT_ACTIVATION = {
    "none": lambda v: v, "relu": lambda v: v.clamp(min=0), "silu": lambda v: v * torch.sigmoid(v),
    "gelu": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2.0)), "sigmoid": torch.sigmoid, "tanh": torch.tanh,
}


def _exact_linear(x, W, bias, activation, residual, dy):
    """y, and the gradients of x, W and bias where dy is given."""
    pre = torch.addmm(bias, x, W.t())
    if dy is None:
        y = _EXACT_ACTIVATION[activation](pre)
        return (y if residual is None else y + residual,)
    with torch.enable_grad():
        pre.requires_grad_(True)
        y = _EXACT_ACTIVATION[activation](pre)
        d, = torch.autograd.grad(y, pre, dy)
    y = y.detach()
    return y if residual is None else y + residual, d @ W, d.t() @ x, d.sum(0)


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in state.items()}
    if case["op"] == "scan":
        if case["T"] == 0:
            h = _exact_scan(s["gi"][None], s["h"], None, case["candidate"])[1]
            return h, h
        states = _exact_scan(s["gi"], s["h"], s["lengths"], case["candidate"])
        out = states[1:]
        if s["lengths"] is not None:
            inside = torch.arange(case["T"], device=out.device)[:, None] < s["lengths"]
            out = out * inside[..., None]
        if not case["train"]:
            return out, states[-1]
        return (out, states[-1], *_exact_scan_backward(s["gi"], states, s["lengths"], case["candidate"], s["dout"], s["dh"]))
    if case["op"] == "linear":
        got = _exact_linear(s["x"], s["W"], s["bias"], case["activation"], s["residual"], s.get("dy"))
        return got if case["train"] else got[0]
    T, B, K, H = case["T"], case["B"], case["K"], case["H"]
    flat = s["x"].reshape(T * B, K)
    gi = _exact_linear(flat, s["Wi"], s["bi"], "none", None, None)[0].reshape(T, B, 2 * H)
    states = _exact_scan(gi, s["h"], None, "tanh")
    out = states[1:].reshape(T * B, H)
    if not case["train"]:
        return _exact_linear(out, s["Wo"], s["bo"], "none", flat, None)[0].reshape(T, B, K), states[-1]
    dy = s["dy"].reshape(T * B, K)
    y, dout, dWo, dbo = _exact_linear(out, s["Wo"], s["bo"], "none", flat, dy)
    dgi, dh0 = _exact_scan_backward(gi, states, None, "tanh", dout.reshape(T, B, H), torch.zeros_like(s["h"]))
    _, dx, dWi, dbi = _exact_linear(flat, s["Wi"], s["bi"], "none", None, dgi.reshape(T * B, 2 * H))
    return y.reshape(T, B, K), states[-1], (dx + dy).reshape(T, B, K), dWi, dbi, dWo, dbo, dh0
