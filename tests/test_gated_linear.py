"""The gated linear recurrence (``scan_gated``) and the product with bias, activation and residual
(``linear_act``) against plain implementations in 64 bits; refusals; the two together as a block.

Tolerances (u = 2^-24, half a step of float32; ``half(t)`` = eps / 2 of an output type):

* scan: a state is an average of candidates and h0, so at most M = max(|n|, |h0|).  A step's gates are off by at most
  16 u of themselves, and what is not in proportion to 1 - z (the rounding of z, of the step, of a tile's product) by
  3 u M a step: |error| <= u M (16 + 3 T).  The backward recurrence is the same sum over |dout|, ``gabs``, with a factor
  |h - n| <= 2 M, and its slopes: u gabs max(1, 2 M) (32 + 6 T).
* product: S = sum |x| |W| of a result.  Operands of two fp16 planes are off by 2^-23 each, their dropped product by 2^-24;
  the tensor core truncates each of at most 32 steps of a chunk by 2 u, chunks of 64 or more terms add with u each:
  u S (80 + K / 64).  An activation adds its own 8 u of its value, and multiplies by a slope below 1.2.
* 16-bit gradients: d = dy * slope is rounded to the type, its slope to steps of 2^-15, half a step off at most:
  S_d (half(t) + u (80 + K / 64)) + S_dy 2^-16.
* every result: half(t) of itself, and half the step of the smallest numbers of its type.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from gru_triton_b200 import _lib
from gru_triton_b200.linear_act import ACTIVATIONS, linear_act
from gru_triton_b200.scan_gated import gated_scan, gated_step

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(ref, dtype):
    f = torch.finfo(dtype)
    return half(dtype) * ref.abs() + f.tiny * f.eps / 2


def close(got, ref, tol):
    assert tuple(got.shape) == tuple(ref.shape)
    off = (got.double() - ref).abs() - tol
    assert bool(torch.isfinite(got.double()).all()) and bool((off <= 0).all()), \
        f"off by {float((got.double() - ref).abs().max()):.3e}, allowed {float((tol + torch.zeros_like(ref)).min()):.3e}"


# ---- the recurrence in 64 bits -------------------------------------------------------------------

def scan64(gi, h0, lengths, candidate):
    """(out, h_T, states before each step) one step after the other."""
    gi = gi.double()
    T, B, H = gi.shape[0], gi.shape[1], gi.shape[2] // 2
    h = torch.zeros(B, H, dtype=torch.float64, device=gi.device) if h0 is None else h0.double()
    lengths = torch.full((B,), T, device=gi.device) if lengths is None else lengths.clamp(0, T)
    outs, before = [], []
    for t in range(T):
        on = (t < lengths)[:, None]
        x, c = gi[t, :, :H], gi[t, :, H:]
        n = c.tanh() if candidate == "tanh" else c
        before.append(h)
        new = torch.sigmoid(x) * h + torch.sigmoid(-x) * n
        h = torch.where(on, new, h)
        outs.append(torch.where(on, new, torch.zeros_like(new)))
    return torch.stack(outs), h, torch.stack(before)


def scan64_backward(gi, lengths, candidate, before, dout, dh):
    gi, dout, G = gi.double(), dout.double(), dh.double()
    T, B, H = gi.shape[0], gi.shape[1], gi.shape[2] // 2
    lengths = torch.full((B,), T, device=gi.device) if lengths is None else lengths.clamp(0, T)
    dgi = torch.zeros_like(gi)
    for t in reversed(range(T)):
        on = (t < lengths)[:, None]
        x, c = gi[t, :, :H], gi[t, :, H:]
        z, k = torch.sigmoid(x), torch.sigmoid(-x)
        n, slope = (c.tanh(), c.cosh() ** -2) if candidate == "tanh" else (c, torch.ones_like(c))
        g = G + dout[t]
        dgi[t] = torch.where(on, torch.cat([g * (before[t] - n) * z * k, g * k * slope], 1), torch.zeros_like(gi[t]))
        G = torch.where(on, z * g, G)
    return dgi, G


def scan_tolerance(gi, h0, T, candidate):
    c = gi.double()[..., gi.shape[2] // 2:]
    c = c[torch.isfinite(c)]
    M = float(c.abs().max()) if candidate == "identity" and c.numel() else 1.0
    M = max(M, 0.0 if h0 is None else float(h0.abs().max()))
    return M, U * M * (16 + 3 * T)


def problem(dtype, T, B, H, seed=0, lean=1.0, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(seed)
    gi = torch.randn(T, B, 2 * H, device=device, generator=gen) * 2
    gi[..., :H] += lean
    return (gi.to(dtype), torch.randn(B, H, device=device, generator=gen),
            (torch.randn(T, B, H, device=device, generator=gen)).to(dtype), torch.randn(B, H, device=device, generator=gen))


def check_scan(gi, h0, lengths, candidate, dout, dh):
    T, dtype = gi.shape[0], gi.dtype
    leaf = gi.detach().requires_grad_(True)
    leaves = [leaf] if h0 is None else [leaf, h0.detach().requires_grad_(True)]
    out, h_T = gated_scan(leaf, leaves[1] if h0 is not None else None, lengths=lengths, candidate=candidate)
    grads = torch.autograd.grad((out, h_T), leaves, (dout, dh))
    ref, ref_T, before = scan64(gi, h0, lengths, candidate)
    M, tol = scan_tolerance(gi, h0, T, candidate)
    close(out.detach(), ref, tol + rounding(ref, dtype))
    close(h_T.detach(), ref_T, tol + rounding(ref_T, torch.float32))
    inner, inner_T = gated_scan(gi, h0, lengths=lengths, candidate=candidate)          # the form without gradients
    assert torch.equal(inner, out) and torch.equal(inner_T, h_T)
    rdgi, rdh0 = scan64_backward(gi, lengths, candidate, before, dout, dh)
    _, gabs = scan64_backward(gi, lengths, candidate, before, dout.abs(), dh.abs())
    reach = float(max(gabs.max(), dh.abs().max(), dout[torch.isfinite(dout)].abs().sum(0).max() if dout.numel() else 0.0))
    tol = U * reach * max(1.0, 2 * M) * (32 + 6 * T)
    close(grads[0], rdgi, tol + rounding(rdgi, dtype))
    if h0 is not None:
        close(grads[1], rdh0, tol + rounding(rdh0, torch.float32))
    return out, h_T, grads


SCAN_SIZES = [(12, 70001, 8), (3, 70001, 5), (20, 1, 70002), (40, 3, 34), (200, 2, 1030), (600, 1, 130), (70, 260, 66),
              (9, 1, 8), (128, 1, 32), (129, 9, 2048), (1700, 1, 300), (2300, 2, 256), (1, 1, 1), (1, 3, 33), (2, 1, 8),
              (7, 2, 64), (16, 40, 72), (17, 2, 64), (63, 2, 64), (64, 5, 40), (65, 3, 96), (130, 1, 512), (300, 2, 72),
              (257, 19, 607), (1000, 1, 1024), (200, 64, 256), (2100, 1, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,B,H", SCAN_SIZES)
def test_scan_matches_64_bits(dtype, T, B, H):
    gi, h0, dout, dh = problem(dtype, T, B, H, seed=T + H)
    check_scan(gi, h0, None, "tanh", dout, dh)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,B,H", [(1, 2, 8), (40, 3, 65), (129, 4, 128), (700, 3, 200)])
def test_scan_identity_candidate_without_h0(dtype, T, B, H):
    gi, _, dout, dh = problem(dtype, T, B, H, seed=T + H)
    check_scan(gi, None, None, "identity", dout, dh)


@pytest.mark.gpu
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,H", [(5, 16), (64, 32), (150, 72), (150, 33), (513, 64)])
def test_scan_ragged_rows_ignore_their_padding(dtype, T, H, index):
    """Rows of no, one, some and all steps, lengths out of range; what lies behind a row is NaN or infinite."""
    lengths = torch.tensor([0, 1, T // 2, T - 1, T, -3, T + 9, min(T, 64), min(T, 65)], device="cuda", dtype=index)
    B = lengths.numel()
    gi, h0, dout, dh = problem(dtype, T, B, H, seed=T)
    behind = torch.arange(T, device="cuda")[:, None] >= lengths[None]
    clean_gi, clean_dout = gi.clone(), dout.clone()
    gi[behind] = float("nan")
    dout[behind] = float("inf")
    gi[-1, 0] = float("-inf")
    leaf, h = gi.requires_grad_(True), h0.requires_grad_(True)
    out, h_T = gated_scan(leaf, h, lengths=lengths)
    got = torch.autograd.grad((out, h_T), (leaf, h), (dout, dh))
    ref = check_scan(clean_gi, h0.detach(), lengths, "tanh", clean_dout, dh)
    assert torch.equal(out, ref[0]) and torch.equal(h_T, ref[1])
    assert all(torch.equal(a, b) for a, b in zip(got, ref[2]))
    assert bool((out[behind] == 0).all()) and bool((got[0][behind] == 0).all())
    for b in (0, 5):                                             # rows without steps
        assert torch.equal(h_T[b], h0[b]) and torch.equal(got[1][b], dh[b])


@pytest.mark.gpu
@pytest.mark.parametrize("T,B,H", [(1, 2, 24), (90, 2, 64), (90, 2, 33), (600, 2, 64)])
def test_scan_saturated_gates_and_nan_stay_where_they_are(T, B, H):
    gi, h0, dout, dh = problem(torch.float32, T, B, H, seed=3)
    inf = float("inf")
    gi[0, 0, :H], gi[T // 2, 0, 0], gi[T // 3, 1, H:] = inf, -inf, inf
    gi[:, 1, 1] = 60.0                                            # holds for good
    gi[:, 1, 2] = -60.0                                           # forgets at once
    gi[:, :, H + 3] *= 1e-6                                       # candidates far below one keep their precision
    check_scan(gi, h0, None, "tanh", dout, dh)
    _, h_T = gated_scan(gi, h0)
    rel = (h_T[0, 3].double() - scan64(gi, None, None, "tanh")[1][0, 3]).abs()
    assert torch.equal(h_T[1, 1], h0[1, 1]) and float(rel) < 10
    bad = gi.clone()
    bad[T // 2, 0, 5] = float("nan")
    out, _ = gated_scan(bad, h0)
    ok, _ = gated_scan(gi, h0)
    same = torch.ones(T, B, H, dtype=torch.bool, device="cuda")
    same[T // 2:, 0, 5] = False
    assert torch.equal(out[same], ok[same]) and bool(out[T // 2:, 0, 5].isnan().all())
    if T > 4:                                                    # a NaN candidate reaches no earlier step's gradient
        bad = gi.clone()
        bad[T // 2, 0, H + 5] = float("nan")
        leaf = bad.requires_grad_(True)
        dgi, = torch.autograd.grad(gated_scan(leaf, h0)[0], leaf, dout)
        assert bool(torch.isfinite(dgi[:T // 2]).all()) and bool(torch.isfinite(dgi[:, 1]).all())


@pytest.mark.gpu
def test_scan_small_candidates_keep_relative_precision():
    gi, _, _, _ = problem(torch.float32, 100, 2, 64, seed=5)
    gi[..., 64:] *= 1e-4
    out, h_T = gated_scan(gi)
    ref, ref_T, _ = scan64(gi, None, None, "tanh")
    M = float(gi[..., 64:].abs().max())
    close(out, ref, U * M * (16 + 300) + rounding(ref, torch.float32))
    close(h_T, ref_T, U * M * (16 + 300) + rounding(ref_T, torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("candidate", ["tanh", "identity"])
@pytest.mark.parametrize("T,B,H", [(1, 2, 160), (6, 3, 33), (40, 2, 96), (100, 130, 160), (200, 3, 161), (1700, 1, 300), (100, 300, 72)])
def test_scan_closed_gates_keep_relative_precision(dtype, candidate, T, B, H):
    """One step with gates from e^-1 down to e^-80 among steps that hold: what is left of h0, and of its gradient, is exact to a
    few units of itself.  e^-|x|: 2 u |x| of the exponent's two roundings, 4 u of the instruction; reciprocal and products 8 u."""
    gi = torch.zeros(T, B, 2 * H, device="cuda")
    gi[..., :H] = 60.0                                           # 1 - z = e^-60: lost beside one
    gi[T // 2, :, :H] = -torch.linspace(1, 80, H, device="cuda")
    gi = gi.to(dtype)
    _, h0, _, dh = problem(torch.float32, 1, B, H, seed=T)
    x = gi[T // 2, :, :H].double()
    z = torch.sigmoid(x)
    allowed = U * (12 + 2 * x.abs())
    leaf, h = gi.requires_grad_(True), h0.requires_grad_(True)
    out, h_T = gated_scan(leaf, h, candidate=candidate)
    dgi, dh0 = torch.autograd.grad(h_T, (leaf, h), dh)
    ref = z * h0.detach().double()
    close(h_T.detach(), ref, allowed * ref.abs())
    close(out[-1].detach(), ref, allowed * ref.abs() + rounding(ref, dtype))
    close(dh0, z * dh.double(), allowed * (z * dh.double()).abs())
    dx = dh.double() * ref * torch.sigmoid(-x)
    close(dgi[T // 2, :, :H], dx, 2 * allowed * dx.abs() + rounding(dx, dtype))
    _, new = gated_step(gi.detach()[T // 2], h0.detach(), candidate=candidate)
    close(new, ref, allowed * ref.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,H,odd", [(2500, 256, 0), (2500, 512, 0), (2100, 255, 1)])
def test_scan_where_large_clusters_cannot_be_placed(dtype, T, H, odd):
    """A device without room for clusters of 12 or 16: the same sequences in clusters of eight, either direction by itself."""
    gi, h0, dout, dh = problem(dtype, T, 1, H, seed=T)
    lib = _lib.load()
    try:
        lib.b200gru_test_limit_gated_clusters(8)
        check_scan(gi, h0, None, "tanh", dout, dh)
        leaf = gi.detach().requires_grad_(True)
        out, h_T = gated_scan(leaf, h0)
        small, = torch.autograd.grad((out, h_T), leaf, (dout, dh), retain_graph=True)
        lib.b200gru_test_limit_gated_clusters(0)
        large, = torch.autograd.grad((out, h_T), leaf, (dout, dh))
    finally:
        lib.b200gru_test_limit_gated_clusters(0)
    tol = 64 * U * float(dout.abs().max()) * 40                  # sums over memories of some ten steps, joined in another order
    close(small, large.double(), tol + 2 * rounding(large.double(), dtype))


def scan_errors(gi, h0, lengths, candidate, dout, dh):
    """(h, dgi, dh0) in 64 bits, each with what every element may be off by: the recurrence applied to the errors of its steps.

    A gate is off by u (12 + 2 |x|) of itself, a candidate by 30 u (identity: nothing) of itself, its slope by u (12 + 4 |c|).  Maps are
    folded step by step and joined at three levels, so a position meets at most 8 roundings of sums whose terms add up to ``size``
    (the recurrence of absolute values): E_t = z E_{t-1} + u ((12 + 2 |x|) (z size_{t-1} + (1 - z) |n|) + 30 (1 - z) |n| + 8 size_t), and
    likewise for the gradients from behind."""
    gi, dout, G = gi.double(), dout.double(), dh.double()
    T, B, H = gi.shape[0], gi.shape[1], gi.shape[2] // 2
    x, c = gi[..., :H], gi[..., H:]
    z, keep = torch.sigmoid(x), torch.sigmoid(-x)
    n, slope = (c.tanh(), c.cosh() ** -2) if candidate == "tanh" else (c, torch.ones_like(c))
    own = 30.0 if candidate == "tanh" else 0.0
    gate = 12 + 2 * x.abs()
    on = (torch.arange(T, device=gi.device)[:, None] < (torch.full((B,), T, device=gi.device) if lengths is None else lengths))[..., None]
    h = torch.zeros(B, H, dtype=torch.float64, device=gi.device) if h0 is None else h0.double()
    size, E = h.abs(), torch.zeros_like(h)
    hs, Es, ends = [h], [E], []
    for t in range(T):
        far = keep[t] * n[t].abs()
        new = z[t] * size + far
        E = torch.where(on[t], z[t] * E + U * (gate[t] * new + own * far + 8 * new), E)
        size = torch.where(on[t], new, size)
        h = torch.where(on[t], z[t] * h + keep[t] * n[t], h)
        hs.append(h)
        Es.append(E)
        ends.append(size)
    E, gabs = torch.zeros_like(G), G.abs()
    dgi, off = torch.zeros_like(gi), torch.zeros_like(gi)
    for t in reversed(range(T)):
        g, gsize = G + dout[t], gabs + dout[t].abs()
        E = E + U * gsize
        left, both_gates = hs[t] - n[t], z[t] * keep[t]
        dx, dc = g * left * both_gates, g * keep[t] * slope[t]
        # h itself is computed anew from the tile's first state
        wrong = Es[t + 1] + Es[t] + U * (own * n[t].abs() + left.abs())
        ex = E * left.abs() * both_gates + gsize * wrong * both_gates + U * (8 + 2 * gate[t]) * dx.abs()
        ec = E * keep[t] * slope[t] + U * (20 + gate[t] + 4 * c[t].abs()) * dc.abs()
        dgi[t] = torch.where(on[t], torch.cat([dx, dc], 1), dgi[t])
        off[t] = torch.where(on[t], torch.cat([ex, ec], 1), off[t])
        G = torch.where(on[t], z[t] * g, G)
        gabs = torch.where(on[t], z[t] * gsize, gabs)
        E = torch.where(on[t], z[t] * E + U * (gate[t] + 8) * z[t] * gsize, E)
    return (torch.stack(hs[1:]) * on, torch.stack(Es[1:]) * on), (hs[-1], Es[-1]), (dgi, off), (G, E)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("candidate", ["tanh", "identity"])
@pytest.mark.parametrize("T,B,H,ragged", [(1, 3, 33, False), (8, 3, 64, False), (70, 2, 96, True), (257, 19, 607, False), (200, 64, 256, True),
                                          (300, 300, 72, True), (600, 1, 130, False), (1000, 1, 1024, False), (1700, 1, 300, False),
                                          (2100, 1, 24, False), (2300, 2, 256, True), (2300, 1, 513, False)])
def test_scan_every_element_to_its_own_error(dtype, candidate, T, B, H, ragged):
    """Bounds that follow the recurrence, far below the values they are for: a lost carry, map or tile shows at any length."""
    gi, h0, dout, dh = problem(dtype, T, B, H, seed=T + B, lean=2.0)
    gi[..., H + 3] *= 1e-6                                       # a column of tiny candidates, of tiny states where h0 is zero
    h0[:, 3] = 0.0
    lengths = torch.linspace(T, T // 2, B, device="cuda").long() if ragged else None
    leaf, h = gi.detach().requires_grad_(True), h0.detach().requires_grad_(True)
    out, h_T = gated_scan(leaf, h, lengths=lengths, candidate=candidate)
    dgi, dh0 = torch.autograd.grad((out, h_T), (leaf, h), (dout, dh))
    for got, (ref, tol) in zip((out.detach(), h_T.detach(), dgi, dh0), scan_errors(gi, h0, lengths, candidate, dout, dh)):
        assert float(tol.norm()) <= 1e-4 * float(ref.norm())
        close(got, ref, tol + rounding(ref, got.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T", [3, 140])
def test_scan_reads_any_layout(dtype, T):
    B, H = 3, 64
    gi, h0, dout, dh = problem(dtype, T, B, H, seed=7)
    ref = check_scan(gi, h0, None, "tanh", dout, dh)

    def wide(t, front, back):
        big = torch.full((*t.shape[:-1], t.shape[-1] + front + back), float("nan"), dtype=t.dtype, device="cuda")
        big[..., front:front + t.shape[-1]] = t
        return big[..., front:front + t.shape[-1]]

    forms = {"batch first": (gi.transpose(0, 1).contiguous().transpose(0, 1), dout.transpose(0, 1).contiguous().transpose(0, 1)),
             "odd offset": (wide(gi, 1, 2), wide(dout, 3, 1)), "wide rows": (wide(gi, 8, 8), wide(dout, 0, 16)),
             "units strided": (gi.repeat_interleave(2, -1)[..., ::2], dout.transpose(1, 2).contiguous().transpose(1, 2))}
    for name, (g, d) in forms.items():
        assert torch.equal(g, gi) and torch.equal(d, dout)
        leaf, h = g.detach().requires_grad_(True), wide(h0, 1, 0).detach().requires_grad_(True)
        out, h_T = gated_scan(leaf, h)
        got = torch.autograd.grad((out, h_T), (leaf, h), (d, wide(dh, 2, 1)))
        for a, b in zip((out, h_T, *got), (ref[0], ref[1], *ref[2])):
            close(a.detach(), b.detach().double(), 2 * rounding(b.double(), dtype) + 64 * T * U * float(b.detach().abs().max()))
    # every step and row the same one: inputs of stride 0
    one = gi[:1, :1].expand(T, B, 2 * H)
    assert torch.equal(gated_scan(one)[0], gated_scan(one.contiguous())[0])
    leaf = gi.detach().requires_grad_(True)
    a, = torch.autograd.grad(gated_scan(leaf, h0)[0].sum(), leaf)                       # a gradient of stride 0
    b, = torch.autograd.grad(gated_scan(leaf, h0)[0], leaf, torch.ones_like(dout))
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_scan_gradient_of_one_output_and_broadcast_state():
    gi, h0, dout, dh = problem(torch.float32, 70, 4, 48, seed=9)
    leaf = gi.requires_grad_(True)
    out, h_T = gated_scan(leaf, h0)
    zeros = torch.zeros_like(dout), torch.zeros_like(dh)
    a = torch.autograd.grad(out, leaf, dout, retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad((out, h_T), leaf, (dout, zeros[1]), retain_graph=True)[0])
    b = torch.autograd.grad(h_T, leaf, dh, retain_graph=True)[0]
    assert torch.equal(b, torch.autograd.grad((out, h_T), leaf, (zeros[0], dh))[0])
    row = h0[0].clone().requires_grad_(True)                     # one learnt state for every row
    _, h_T = gated_scan(gi.detach(), row.expand(4, -1))
    got, = torch.autograd.grad(h_T, row, dh)
    full = h0[:1].expand(4, -1).contiguous().requires_grad_(True)
    _, h_T = gated_scan(gi.detach(), full)
    assert torch.equal(got, torch.autograd.grad(h_T, full, dh)[0].sum(0))


@pytest.mark.gpu
def test_scan_gradient_against_differences():
    gi, h0, dout, dh = problem(torch.float32, 75, 2, 40, seed=11)
    lengths = torch.tensor([75, 31], device="cuda")
    leaf, h = gi.requires_grad_(True), h0.requires_grad_(True)
    out, h_T = gated_scan(leaf, h, lengths=lengths)
    got = torch.autograd.grad((out, h_T), (leaf, h), (dout, dh))
    gen = torch.Generator(device="cuda").manual_seed(1)
    step = 1e-6
    for which in (0, 1):
        base = [gi.detach().double(), h0.detach().double()]
        way = torch.randn(base[which].shape, device="cuda", generator=gen, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            at = list(base)
            at[which] = at[which] + sign * step * way
            o, hT, _ = scan64(at[0], at[1], lengths, "tanh")
            ends.append(float((o * dout.double()).sum() + (hT * dh.double()).sum()))
        slope = (ends[0] - ends[1]) / (2 * step)
        mine = float((got[which].double() * way).sum())
        # the difference: step^2 times a third derivative, and 2^-53 of the sums over step; the gradient: as above
        scale = float((got[which].double() * way).abs().sum())
        assert abs(slope - mine) <= 1e-5 * scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("candidate", ["tanh", "identity"])
@pytest.mark.parametrize("B,H", [(1, 1), (1, 256), (5, 33), (130, 1024)])
def test_steps_walk_the_scan(dtype, candidate, B, H):
    T = 6
    gi, h0, _, _ = problem(dtype, T, B, H, seed=13)
    ref, ref_T, _ = scan64(gi, h0, None, candidate)
    _, tol = scan_tolerance(gi, h0, T, candidate)
    h, state = h0, h0.clone()
    for t in range(T):
        out, h = gated_step(gi[t], h, candidate=candidate)
        again, same = gated_step(gi[t], state, candidate=candidate, out_state=state)
        assert same is state and torch.equal(state, h) and torch.equal(out, again)
        close(out, ref[t], tol + rounding(ref[t], dtype))
    close(h, ref_T, tol + rounding(ref_T, torch.float32))
    pool = torch.full((2 * B, H + 5), 7.0, device="cuda")         # rows of a larger state table, every other one
    pool[::2, :H] = h0
    out, new = gated_step(gi[0], pool[::2, :H], candidate=candidate, out_state=pool[::2, :H])
    assert torch.equal(new, gated_step(gi[0], h0, candidate=candidate)[1])
    assert bool((pool[1::2] == 7).all()) and bool((pool[:, H:] == 7).all())


@pytest.mark.gpu
def test_step_refuses_states_that_overlap_and_gradients():
    gi, h0, _, _ = problem(torch.float32, 1, 4, 16)
    big = torch.zeros(5, 16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        gated_step(gi[0], big[:4], out_state=big[1:])
    with pytest.raises(ValueError, match="rows"):
        gated_step(gi[0], h0, out_state=h0[:1].expand(4, 16))
    with pytest.raises(ValueError, match="gradients"):
        gated_step(gi[0].requires_grad_(True), h0)
    flat = torch.zeros(4, 32, device="cuda")
    with pytest.raises(ValueError, match="gi"):
        gated_step(flat, h0, out_state=flat[:, :16])


@pytest.mark.gpu
@pytest.mark.parametrize("T,B,H", [(9, 3, 40), (64, 32, 512), (500, 2, 96), (3000, 1, 128)])
def test_scan_repeats_its_bits(T, B, H):
    gi, h0, dout, dh = problem(torch.float32, T, B, H, seed=15)
    lengths = torch.randint(0, T + 1, (B,), device="cuda")
    runs = []
    for _ in range(3):
        leaf, h = gi.detach().requires_grad_(True), h0.detach().requires_grad_(True)
        out, h_T = gated_scan(leaf, h, lengths=lengths)
        runs.append((out.detach(), h_T.detach(), *torch.autograd.grad((out, h_T), (leaf, h), (dout, dh))))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.gpu
@pytest.mark.slow
def test_scan_offsets_past_32_bits():
    """gi and out of more than 2^31 elements: the last row agrees with the same row alone."""
    T, B, H = 70016, 16, 1024
    gi = torch.empty(T, B, 2 * H, device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(0)
    row = torch.randn(T, 1, 2 * H, device="cuda", generator=gen).to(torch.bfloat16)
    gi[:, :15] = 0
    gi[:, 15:] = row
    leaf = gi.requires_grad_(True)
    out, h_T = gated_scan(leaf)
    alone, alone_T = gated_scan(row)
    assert float((out[:, 15:] - alone).abs().max()) <= 2 ** -6 and float((h_T[15] - alone_T[0]).abs().max()) <= 1e-5
    assert bool((out[:, :15] == 0).all())
    del alone
    dgi, = torch.autograd.grad(out, leaf, row[..., :H].expand(T, B, H))
    del out
    leaf1 = row.requires_grad_(True)
    ref, = torch.autograd.grad(gated_scan(leaf1)[0], leaf1, row.detach()[..., :H])
    assert float((dgi[:, 15:].float() - ref.float()).abs().max()) <= 2 ** -7 * float(ref.float().abs().max())


# ---- the product ------------------------------------------------------------------------------------

def act64(pre, name):
    return {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
            "gelu": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2.0)), "sigmoid": torch.sigmoid, "tanh": torch.tanh}[name](pre)


def linear_problem(dtype, M, K, N, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, device="cuda", generator=gen).to(dtype)
    W = (torch.randn(N, K, device="cuda", generator=gen) / math.sqrt(K)).to(dtype)
    bias = torch.randn(N, device="cuda", generator=gen).to(dtype)
    residual = torch.randn(M, N, device="cuda", generator=gen).to(dtype)
    return x, W, bias, residual, torch.randn(M, N, device="cuda", generator=gen).to(dtype)


def check_linear(x, W, bias, residual, activation, dy):
    dtype, K, N, M = x.dtype, W.shape[1], W.shape[0], x.shape[0]
    leaves = [t.detach().requires_grad_(True) for t in (x, W) + (() if bias is None else (bias,)) + (() if residual is None else (residual,))]
    it = iter(leaves[2:])
    y = linear_act(leaves[0], leaves[1], None if bias is None else next(it), activation=activation,
                   residual=None if residual is None else next(it))
    got = torch.autograd.grad(y, leaves, dy)
    inner = linear_act(x, W, bias, activation=activation, residual=residual)
    assert torch.equal(inner, y)

    x64, W64, dy64 = x.double(), W.double(), dy.double()
    pre = x64 @ W64.t() + (0 if bias is None else bias.double())
    pre.requires_grad_(True)
    a = act64(pre, activation)
    d, = torch.autograd.grad(a, pre, dy64)
    pre, a = pre.detach(), a.detach()
    ref = a if residual is None else a + residual.double()
    S = x64.abs() @ W64.abs().t() + (0 if bias is None else bias.double().abs())
    off_pre = U * S * (80 + K / 64)
    close(y.detach(), ref, 1.2 * off_pre + 8 * U * (a.abs() + pre.abs() + ref.abs()) + rounding(ref, dtype))
    # the slope's own error: |act''| <= 1 of the error of pre, a few units of itself; fixed point behind 16-bit types
    off_d = dy64.abs() * (off_pre + 16 * U)
    if activation == "relu":
        off_d = dy64.abs() * (pre.abs() <= off_pre) + 0 * d      # the sign of pre decides
    if dtype != torch.float32 and activation != "none":
        off_d = off_d + dy64.abs() * 2.0 ** -16
    # the products take d in the type: half a step of its value, or of fp16's smallest, 2^-24, where d is that small (a
    # product of one term, M or N of 1, has no larger ones beside it)
    in_product = off_d + (rounding(d, dtype) if dtype != torch.float32 and activation != "none" else 0.0)
    refs = [d @ W64, d.t() @ x64]
    sums = [d.abs() @ W64.abs(), d.abs().t() @ x64.abs()]
    carried = [in_product @ W64.abs(), in_product.t() @ x64.abs()]
    for k, terms in ((0, N), (1, M)):
        close(got[k], refs[k], carried[k] + U * sums[k] * (80 + terms / 64) + rounding(refs[k], dtype))
    if bias is not None:
        db = d.sum(0)
        close(got[2], db, off_d.sum(0) + U * d.abs().sum(0) * (80 + M / 64) + rounding(db, dtype))
    if residual is not None:
        assert torch.equal(got[-1], dy)
    return y, got


LINEAR_SIZES = [(40, 2048, 132), (1000, 132, 60), (5310, 804, 423), (300, 70000, 1), (40, 1, 70000), (70000, 1, 3),
                (70000, 3, 9), (1, 70000, 2), (5, 2048, 2048), (2, 1024, 1024), (17, 96, 130), (32, 200, 64), (1, 1, 1),
                (1, 64, 64), (2, 100, 7), (3, 129, 250), (8, 512, 1024), (9, 256, 96), (16, 65, 33), (33, 1024, 512),
                (64, 96, 260), (127, 63, 127), (128, 128, 128), (129, 72, 257), (300, 1000, 136), (1000, 120, 608),
                (2048, 512, 1024), (700, 2050, 70), (5000, 40, 24), (4100, 136, 1032)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", LINEAR_SIZES)
def test_linear_matches_64_bits(dtype, M, K, N):
    x, W, bias, residual, dy = linear_problem(dtype, M, K, N, seed=M + K + N)
    check_linear(x, W, bias, residual, "silu", dy)
    check_linear(x, W, None, None, "none", dy)


def linear_plan(M, N, K, dtype, activation="none"):
    """(CTAs to a tile, columns of a tile, K slices, blocks of 64 terms in a slice, of them in a chunk)."""
    plan = (ctypes.c_int * 5)()
    assert _lib.load().b200gru_test_linear_plan(M, N, K, 2 if dtype == torch.float32 else 1, ACTIVATIONS[activation], plan) == 0
    return tuple(plan)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("activation,residual", [("silu", True), ("gelu", False), ("none", True)])
@pytest.mark.parametrize("M,K,N", [(4104, 4104, 4104), (16400, 4096, 1024), (9000, 520, 4104)])
def test_linear_on_pairs_of_ctas(dtype, activation, residual, M, K, N):
    """256 x 256 tiles of two CTAs in the forward and in the gradients, at remainders, of many chunks, with everything an epilogue does."""
    forward, dx, dW = linear_plan(M, N, K, dtype, activation), linear_plan(M, K, N, dtype), linear_plan(N, K, M, dtype)
    assert forward[0] == dW[0] == 2 and (dx[0] == 2 or K == 520)
    if K > 4000 and dtype != torch.float32 and activation != "none":
        assert forward[2] == 1 and forward[3] > 3 * forward[4]   # totals that pass through both accumulators, more than once
    x, W, bias, r, dy = linear_problem(dtype, M, K, N, seed=N)
    check_linear(x, W, bias, r if residual else None, activation, dy)


def test_plans_of_the_large_tests():
    """Every way a product is cut has a case above: pairs with and without K slices, single CTAs of both widths, one chunk and many."""
    seen = set()
    for M, K, N in [(4104, 4104, 4104), (16400, 4096, 1024), (9000, 520, 4104), *LINEAR_SIZES]:
        for dtype in DTYPES[:2]:
            for m, n, k in ((M, N, K), (M, K, N), (N, K, M)):
                ctas, bn, splits, per, chunk = linear_plan(m, n, k, dtype)
                seen.add((dtype, ctas, bn, splits > 1, per > chunk))
    for dtype in DTYPES[:2]:
        for ctas, bn in ((2, 256), (1, 128), (1, 64)):
            assert (dtype, ctas, bn, False, True) in seen
            assert any(s[:4] == (dtype, ctas, bn, True) for s in seen) or (ctas == 2 and dtype != torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("activation", list(ACTIVATIONS))
@pytest.mark.parametrize("M,K,N", [(3, 72, 40), (40, 256, 200), (400, 264, 520)])
def test_linear_activations(dtype, activation, M, K, N):
    x, W, bias, residual, dy = linear_problem(dtype, M, K, N, seed=M)
    check_linear(x, W, bias, None, activation, dy)
    check_linear(x, W * 3, bias, residual, activation, dy)       # saturated in part


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M", [2, 40, 300])
def test_linear_reads_any_layout(dtype, M):
    K, N = 136, 264
    x, W, bias, residual, dy = linear_problem(dtype, M, K, N, seed=1)
    y, grads = check_linear(x, W, bias, residual, "gelu", dy)

    def wide(t, front, back):
        big = torch.full((*t.shape[:-1], t.shape[-1] + front + back), float("nan"), dtype=t.dtype, device="cuda")
        big[..., front:front + t.shape[-1]] = t
        return big[..., front:front + t.shape[-1]]

    def turned(t):
        return t.t().contiguous().t()

    forms = [(wide(x, 8, 16), wide(W, 16, 8), wide(residual, 8, 0), wide(dy, 0, 8)),
             (wide(x, 1, 1), wide(W, 3, 1), wide(residual, 1, 1), wide(dy, 1, 2)),
             (turned(x), turned(W), turned(residual), turned(dy))]
    for fx, fW, fr, fd in forms:
        leaves = [t.detach().requires_grad_(True) for t in (fx, fW, bias, fr)]
        out = linear_act(*leaves[:3], activation="gelu", residual=leaves[3])
        got = torch.autograd.grad(out, leaves, fd)
        assert torch.equal(out, y)
        assert all(torch.equal(a, b) for a, b in zip(got, grads))
    three = x.reshape(2, M // 2, K)                              # leading axes
    assert torch.equal(linear_act(three, W, bias, activation="gelu", residual=residual.reshape(2, M // 2, N)), y.reshape(2, M // 2, N))
    back = three.transpose(0, 1)                                 # rows in another order
    assert torch.equal(linear_act(back, W, bias), linear_act(back.contiguous(), W, bias))
    assert torch.equal(linear_act(x[0], W, bias), linear_act(x[:1], W, bias)[0])
    one = x[:1].expand(M, K)
    assert torch.equal(linear_act(one, W, bias), linear_act(one.contiguous(), W, bias))
    leaf = x.detach().requires_grad_(True)
    a, = torch.autograd.grad(linear_act(leaf, W, bias, activation="gelu").sum(), leaf)
    b, = torch.autograd.grad(linear_act(leaf, W, bias, activation="gelu"), leaf, torch.ones_like(dy))
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("activation", ["none", "gelu"])
@pytest.mark.parametrize("M, K, N", [(4, 64, 1), (40, 1, 1), (300, 128, 1), (300, 1, 72), (300, 200, 72)])
def test_linear_rows_of_stride_zero(dtype, activation, M, K, N):
    x, W, bias, residual, dy = linear_problem(dtype, M, K, N, seed=5)
    same = [x[:1].expand(M, K), W[:1].expand(N, K), bias[:1].expand(N), residual[:1, :1].expand(M, N)]
    every = dy[:1, :1].expand(M, N)
    results = []
    for form in (lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)):
        leaves = [form(t).detach().requires_grad_(True) for t in same]
        out = linear_act(*leaves[:3], activation=activation, residual=leaves[3])
        results.append((out, *torch.autograd.grad(out, leaves, form(every))))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M, K, N", [(40, 2048, 132), (1000, 132, 60), (40, 2048, 130), (300, 100, 135), (2, 60, 36)])
def test_linear_writes_inside_its_results(dtype, M, K, N):
    x, W, bias, residual, dy = linear_problem(dtype, M, K, N, seed=6)
    size, margin, lds = dtype.itemsize, 4096, (N + 7) // 8 * 8
    lib, stream = _lib.load(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def guarded(count):
        return torch.full((count + 2 * margin,), 0x5A, dtype=torch.uint8, device="cuda")

    def args(**buffers):
        a = _lib.CLinearArgs()
        a.M, a.K, a.N, a.dtype, a.activation = M, K, N, DTYPES.index(dtype), ACTIVATIONS["gelu"]
        a.x, a.ldx, a.W, a.ldw, a.lds = x.data_ptr(), K, W.data_ptr(), K, lds
        for name, t in buffers.items():
            setattr(a, name, t.data_ptr() + margin)
        return a

    def call(fn, backward, a, buffers):
        n = lib.b200gru_linear_act_workspace_bytes(ctypes.byref(a), backward)
        buffers = dict(buffers, workspace=guarded(n))
        a.workspace, a.workspace_bytes = buffers["workspace"].data_ptr() + margin, n
        assert fn(ctypes.byref(a), stream) == 0
        for name, t in buffers.items():
            assert bool((t[:margin] == 0x5A).all()) and bool((t[t.numel() - margin:] == 0x5A).all()), name

    out = dict(y=guarded(M * N * size), slope=guarded(M * lds * max(2, size)))
    a = args(**out)
    a.bias, a.residual, a.ldr, a.ldy = bias.data_ptr(), residual.data_ptr(), N, N
    call(lib.b200gru_linear_act_forward, 0, a, out)
    grads = dict(dx=guarded(M * K * size), dW=guarded(N * K * size), db=guarded(N * size))
    a = args(slope=out["slope"], **grads)
    a.dy, a.lddy = dy.data_ptr(), N
    call(lib.b200gru_linear_act_backward, 1, a, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M, K, N", [(2, 64, 130), (40, 2048, 130), (300, 128, 130), (300, 128, 132), (2100, 320, 516)])
def test_linear_slopes_of_any_row_pitch(dtype, M, K, N):
    """Slopes in rows without padding and off 16-byte boundaries, as a C caller may hold them: the same slopes and gradients."""
    x, W, bias, residual, dy = linear_problem(dtype, M, K, N, seed=7)
    lib, stream = _lib.load(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    kept = torch.float32 if dtype == torch.float32 else torch.int16

    def call(fn, backward, a):
        n = lib.b200gru_linear_act_workspace_bytes(ctypes.byref(a), backward)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), n
        assert fn(ctypes.byref(a), stream) == 0

    def run(lds, offset):
        slopes = torch.full((offset + M * lds + 8,), 77, dtype=kept, device="cuda")
        y, dx, dW, db = (torch.empty_like(t) for t in (residual, x, W, bias))
        a = _lib.CLinearArgs()
        a.M, a.K, a.N, a.dtype, a.activation = M, K, N, DTYPES.index(dtype), ACTIVATIONS["silu"]
        a.x, a.ldx, a.W, a.ldw, a.bias, a.residual, a.ldr = x.data_ptr(), K, W.data_ptr(), K, bias.data_ptr(), residual.data_ptr(), N
        a.y, a.ldy, a.slope, a.lds = y.data_ptr(), N, slopes.data_ptr() + offset * slopes.element_size(), lds
        call(lib.b200gru_linear_act_forward, 0, a)
        a.dy, a.lddy, a.dx, a.dW, a.db = dy.data_ptr(), N, dx.data_ptr(), dW.data_ptr(), db.data_ptr()
        call(lib.b200gru_linear_act_backward, 1, a)
        rows = slopes[offset:offset + M * lds].view(M, lds)
        outside = [slopes[:offset], slopes[offset + M * lds:]]
        if lds > N and offset:
            outside.append(rows[:, N:].reshape(-1))              # the padding of rows that are copied
        assert all(bool((t == 77).all()) for t in outside)
        return [rows[:, :N].contiguous(), y, dx, dW, db]

    want = run((N + 7) // 8 * 8, 0)
    for lds, offset in ((N, 0), (N, 1), (N + 3, 5)):
        for a, b in zip(run(lds, offset), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("activation", ["none", "gelu"])
@pytest.mark.parametrize("M, K, N", [(2, 131, 59), (40, 2045, 131), (300, 133, 267), (300, 130, 266), (1100, 258, 1029), (4100, 1030, 4099)])
def test_linear_of_column_blocks_of_wider_matrices(dtype, activation, M, K, N):
    """Odd widths in rows on 16-byte boundaries: what lies beside a block is neither read into a result nor written."""
    x, W, bias, residual, dy = linear_problem(dtype, M, K, N, seed=9)

    def block(t):
        big = torch.full((t.shape[0], (t.shape[1] + 7) // 8 * 8 + 16), float("nan"), dtype=dtype, device="cuda")
        big[:, 8:8 + t.shape[1]] = t
        return big[:, 8:8 + t.shape[1]]

    want = [t.detach().requires_grad_(True) for t in (x, W, bias, residual)]
    y = linear_act(*want[:3], activation=activation, residual=want[3])
    grads = torch.autograd.grad(y, want, dy)
    got = [t.detach().requires_grad_(True) for t in (block(x), block(W), bias, block(residual))]
    out = linear_act(*got[:3], activation=activation, residual=got[3])
    assert torch.equal(out, y)
    for a, b in zip(torch.autograd.grad(out, got, block(dy)), grads):
        assert torch.equal(a, b)
    # a C caller's result is such a block as well
    lib, stream = _lib.load(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    whole = torch.full((M, (N + 7) // 8 * 8 + 16), 7.0, dtype=dtype, device="cuda")
    inside = whole[:, 8:8 + N]
    a = _lib.CLinearArgs()
    a.M, a.K, a.N, a.dtype, a.activation = M, K, N, DTYPES.index(dtype), ACTIVATIONS[activation]
    a.x, a.ldx, a.W, a.ldw, a.bias = x.data_ptr(), K, W.data_ptr(), K, bias.data_ptr()
    a.residual, a.ldr, a.y, a.ldy = residual.data_ptr(), N, inside.data_ptr(), whole.shape[1]
    n = lib.b200gru_linear_act_workspace_bytes(ctypes.byref(a), 0)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    assert lib.b200gru_linear_act_forward(ctypes.byref(a), stream) == 0
    assert torch.equal(inside, y) and bool((whole[:, :8] == 7).all()) and bool((whole[:, 8 + N:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 200])
def test_linear_no_rows_some_gradients_and_special_values(M):
    x, W, bias, residual, dy = linear_problem(torch.float32, M, 64, 48)
    leaves = [t.detach().requires_grad_(True) for t in (x[:0], W, bias)]
    y = linear_act(*leaves, activation="silu")
    assert tuple(y.shape) == (0, 48)
    got = torch.autograd.grad(y, leaves, dy[:0])
    assert tuple(got[0].shape) == (0, 64) and not got[1].any() and not got[2].any()
    full = [t.detach().requires_grad_(True) for t in (x, W, bias, residual)]
    all_of = torch.autograd.grad(linear_act(*full[:3], activation="silu", residual=full[3]), full, dy)
    for k in range(4):
        some = [t.detach().requires_grad_(k == i) for i, t in enumerate((x, W, bias, residual))]
        got, = torch.autograd.grad(linear_act(*some[:3], activation="silu", residual=some[3]), some[k], dy)
        assert torch.equal(got, all_of[k])
    # a row of NaN and one of infinities stay in their rows; a zero row gives act(bias)
    bad = x.clone()
    bad[1], bad[2], bad[3] = float("nan"), float("inf"), 0.0
    for activation in ACTIVATIONS:
        out = linear_act(bad, W, bias, activation=activation)
        ok = linear_act(x, W, bias, activation=activation)
        rest = [0, 4] + list(range(5, M))
        assert torch.equal(out[rest], ok[rest]) and bool(out[1].isnan().all())
        close(out[3], act64(bias.double(), activation), 32 * U * (1 + bias.double().abs()))
    # saturated both ways
    huge = torch.full((M, 64), 1e30, device="cuda")
    one = torch.ones(2, 64, device="cuda")
    one[1] = -1
    for activation, (lo, hi) in {"relu": (0.0, None), "silu": (0.0, None), "gelu": (0.0, None), "sigmoid": (0.0, 1.0), "tanh": (-1.0, 1.0)}.items():
        leaf = huge.detach().requires_grad_(True)
        y = linear_act(leaf, one, activation=activation)
        g, = torch.autograd.grad(y, leaf, torch.ones_like(y))
        assert bool((y[:, 1] == lo).all()) and (hi is None or bool((y[:, 0] == hi).all())) and bool((y[:, 0] > 0).all())
        assert bool((g == (1.0 if hi is None else 0.0)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M", [2, 200])
def test_linear_infinity_in_a_weight_stays_in_its_column(dtype, M):
    x, W, bias, _, dy = linear_problem(dtype, M, 64, 48, seed=8)
    bad = W.clone()
    bad[5, 3] = float("inf")
    y, ok = linear_act(x, bad, bias), linear_act(x, W, bias)
    rest = [n for n in range(48) if n != 5]
    assert torch.equal(y[:, rest], ok[:, rest])
    if dtype == torch.float32 and M > 8:
        assert bool(y[:, 5].isnan().all())                       # two planes hold no infinity
    else:
        assert torch.equal(y[:, 5], torch.where(x[:, 3] > 0, math.inf, -math.inf).to(dtype))
    leaf = x.requires_grad_(True)
    dx, = torch.autograd.grad(linear_act(leaf, bad, bias), leaf, dy)
    assert not bool(torch.isfinite(dx[:, 3]).any()) and bool(torch.isfinite(dx[:, [k for k in range(64) if k != 3]]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid", "tanh"])
@pytest.mark.parametrize("M", [5, 200])
def test_linear_gradient_of_a_nan_row_is_nan_and_stays_there(dtype, activation, M):
    x, W, bias, _, dy = linear_problem(dtype, M, 64, 48)
    x[3] = float("nan")
    leaf = x.requires_grad_(True)
    dx, = torch.autograd.grad(linear_act(leaf, W, bias, activation=activation), leaf, dy)
    rest = [m for m in range(M) if m != 3]
    assert bool(dx[3].isnan().all()) and bool(torch.isfinite(dx[rest]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid", "tanh"])
@pytest.mark.parametrize("M,K", [(2, 64), (7, 64), (161, 64), (40, 2048), (20000, 64)])
def test_linear_gradient_of_saturated_units_keeps_relative_precision(dtype, activation, M, K):
    """x -> x (W the identity, zeros beside it): the gradient of x is dy act'(x), down to slopes of e^-15 (fp16) and e^-35.

    Off by: the rounding of d; the kept slope, 2^-10 (fp16) or 2^-9 (bf16) of itself, twice that at its lowest; 2 u |x| (tanh 4 u |x|) of
    an exponential's argument and 16 u of the rest; gelu 2^-11 (Phi's formula against v phi(v) in the tail); where silu's and gelu's
    slopes cross zero, 16 u absolute; fp32 gradients, a product of planes as above."""
    N = 64
    far = {"gelu": 4.5 if dtype == torch.float16 else 7.0, "tanh": 0.5 * (18 if dtype == torch.float16 else 37)}
    far = far.get(activation, 18.0 if dtype == torch.float16 else 37.0)
    x = torch.zeros(M, K, device="cuda")
    x[:, :N] = torch.linspace(-far, far, M, device="cuda")[:, None]
    x = x.to(dtype)
    W = torch.eye(N, K, device="cuda").to(dtype)
    gen = torch.Generator(device="cuda").manual_seed(M)
    dy = ((torch.rand(M, N, device="cuda", generator=gen) + 0.5) * (2.0 ** 8 if dtype == torch.float16 else 1.0)).to(dtype)
    leaf = x.requires_grad_(True)
    dx, = torch.autograd.grad(linear_act(leaf, W, activation=activation), leaf, dy)
    pre = x.detach()[:, :N].double()
    s, t = torch.sigmoid(pre), torch.sigmoid(-pre)               # written out: autograd's 1 - y loses the tails in 64 bits too
    phi = torch.exp(-0.5 * pre * pre) / math.sqrt(2 * math.pi)
    d = dy.double() * {"sigmoid": s * t, "tanh": torch.cosh(pre) ** -2, "silu": s * (1 + pre * t),
                       "gelu": 0.5 * torch.erfc(-pre / math.sqrt(2.0)) + pre * phi}[activation]
    kept = {torch.float32: U * (80 + N / 64), torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -9}[dtype]
    own = U * (16 + 4 * pre.abs()) + (2.0 ** -11 if activation == "gelu" else 0.0)
    zero = 16 * U * dy.double() * (pre.abs() < 3) * (activation in ("silu", "gelu"))
    close(dx[:, :N], d, (kept + own) * d.abs() + zero + rounding(d, dtype))
    assert not dx[:, N:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", [(4, 300, 50), (48, 512, 640), (520, 512, 640), (9000, 128, 264)])
def test_linear_repeats_its_bits(dtype, M, K, N):
    x, W, bias, residual, dy = linear_problem(dtype, M, K, N)
    runs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_(True) for t in (x, W, bias)]
        y = linear_act(*leaves, activation="tanh", residual=residual)
        runs.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.gpu
def test_linear_small_rows_beside_large_ones():
    """float32 rows and columns that differ by many powers of two keep their own precision."""
    x, W, bias, _, dy = linear_problem(torch.float32, 300, 200, 160, seed=4)
    x = x * (2.0 ** torch.randint(-30, 30, (300, 1), device="cuda"))
    W = W * (2.0 ** torch.randint(-20, 20, (160, 1), device="cuda"))
    y = linear_act(x, W)
    ref = x.double() @ W.double().t()
    S = x.double().abs() @ W.double().abs().t()
    close(y, ref, U * S * (80 + 200 / 64) + rounding(ref, torch.float32))
    leaf = x.requires_grad_(True)
    wleaf = W.requires_grad_(True)
    rows = dy * (2.0 ** torch.randint(-30, 30, (300, 1), device="cuda"))
    dx, = torch.autograd.grad(linear_act(leaf, wleaf.detach()), leaf, rows)
    ref = rows.double() @ W.double()
    # a row of d is scaled as a whole after the weight rows' own powers of two are folded in
    S = rows.double().abs() @ W.double().abs()
    top = (rows.double().abs()[:, :, None] * W.double().abs().amax(1)[None, :, None]).amax(1)
    close(dx, ref.detach(), U * S.detach() * (80 + 160 / 64) + 160 * 2.0 ** -38 * top.detach() + rounding(ref.detach(), torch.float32))


@pytest.mark.gpu
@pytest.mark.slow
def test_linear_offsets_past_32_bits():
    M, K, N = 2 ** 20 + 37, 64, 2056
    x, W, bias, _, _ = linear_problem(torch.bfloat16, 2048, K, N)
    xl = x.repeat(M // 2048 + 1, 1)[:M]
    y = linear_act(xl, W, bias, activation="relu")
    assert y.numel() > 2 ** 31
    ref = linear_act(x, W, bias, activation="relu")
    start = (M - 2048) // 2048 * 2048
    assert torch.equal(y[start:start + 2048], ref) and torch.equal(y[-37:], ref[:37])

def rounding_share(x, W, dtype, steps):
    """Of the results of a 16-bit product above 1/4 in size, the share that its sums round to another number than the exact sum does.
    A step of 16 terms that truncates loses half a unit in the last place on average, u of the running sum at most; adding a
    chunk is off by u / 2 of the total on average; the losses of different chunks add up like random signs (their sums have
    any sign).  A sum that is off by e lies on the other side of a border of its type with probability e / step."""
    parts = torch.einsum("msk,nsk->mns", x.double().unflatten(1, (-1, 16)), W.double().unflatten(1, (-1, 16)))
    total = parts.cumsum(2)
    lost = U * parts.unflatten(2, (-1, steps)).cumsum(3).abs().sum(3)
    off = (lost.square().sum(2) + (U / 2 * total[..., steps - 1::steps]).square().sum(2)).sqrt()
    ref = total[..., -1]
    step = torch.finfo(dtype).eps * torch.exp2(torch.floor(torch.log2(ref.abs().clamp(min=0.25))))
    return float((off / step)[ref.abs() >= 0.25].mean())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("activation,K,steps", [("none", 512, 8), ("none", 1024, 16), ("none", 4096, 32), ("relu", 4096, 64)])
def test_linear_16_bit_sums_are_built_in_short_chunks(dtype, activation, K, steps):
    """The share of results that are not the rounding of the exact sum (the tensor core truncates at every step: one chunk of
    all of K would leave seven times as many at K = 4096)."""
    plan = linear_plan(8192, 1024, K, dtype, activation)
    assert plan[2] == 1 and min(plan[3:]) * 4 == steps
    x, W, _, _, _ = linear_problem(dtype, 8192, K, 1024, seed=K)
    y = linear_act(x, W, activation=activation)
    ref = act64(x.double() @ W.double().t(), activation)
    here = ref.abs() >= 0.25
    n, share = int(here.sum()), rounding_share(x[:128], W, dtype, steps)
    assert int((y != ref.to(dtype))[here].sum()) <= n * share + 6 * math.sqrt(n * share)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_block_state_is_float32_of_its_gates(dtype):
    """The state behind 16-bit gates is that of these gates to float32 accuracy.  (That of other sums for the same gates is not: a gate
    on the border of two of its type's numbers may be rounded to either.)"""
    T, B, K, H = 100, 17, 512, 512
    (x, Wi, bi, _, _, h0), _ = block_problem(dtype, T, B, K, H)
    gi = linear_act(x, Wi, bi)
    _, h_T = gated_scan(gi, h0)
    ref = scan64(gi, h0, None, "tanh")[1]
    close(h_T, ref, scan_tolerance(gi, h0, T, "tanh")[1] + rounding(ref, torch.float32))
    # relative to the norm: errors of a step, about 3 u, add up over memories of ten steps
    assert float((h_T.double() - ref).norm() / ref.norm()) <= 30 * U


# ---- streams, graphs, the two together ---------------------------------------------------------------

def block(x, Wi, bi, Wo, bo, h0, lengths=None):
    out, h_T = gated_scan(linear_act(x, Wi, bi), h0, lengths=lengths)
    return linear_act(out, Wo, bo, activation="silu", residual=x), h_T


def block_problem(dtype, T, B, K, H, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=gen) * scale).to(dtype)  # noqa: E731
    return [make(T, B, K), make(2 * H, K, scale=K ** -0.5), make(2 * H), make(K, H, scale=H ** -0.5), make(K),
            torch.randn(B, H, device="cuda", generator=gen)], make(T, B, K)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,B,K,H", [(20, 3, 40, 24), (70, 4, 72, 136), (130, 8, 256, 256)])
def test_block_trains_and_serves(dtype, T, B, K, H):
    tensors, dy = block_problem(dtype, T, B, K, H)
    lengths = torch.randint(0, T + 1, (B,), device="cuda")
    lengths[0] = T
    leaves = [t.detach().requires_grad_(True) for t in tensors]
    y, h_T = block(*leaves, lengths=lengths)
    got = torch.autograd.grad(y, leaves, dy)

    def block64(x, Wi, bi, Wo, bo, h0):
        gi = x @ Wi.t() + bi
        h, outs = h0, []
        for t in range(T):
            on = (t < lengths)[:, None]
            new = torch.sigmoid(gi[t, :, :H]) * h + torch.sigmoid(-gi[t, :, :H]) * gi[t, :, H:].tanh()
            h = torch.where(on, new, h)
            outs.append(torch.where(on, new, torch.zeros_like(new)))
        pre = torch.stack(outs) @ Wo.t() + bo
        return pre * torch.sigmoid(pre) + x, h

    wide = [t.detach().double().requires_grad_(True) for t in tensors]
    ry, rh = block64(*wide)
    ref = torch.autograd.grad(ry, wide, dy.double())
    # relative to the norm: a handful of roundings of the type (gi, out, y; dout, dgi, dx), each half a step; memories of
    # about ten steps repeat that of gi
    bound = 16 * half(dtype) if dtype != torch.float32 else 512 * U
    for a, b in zip((y.detach(), h_T.detach(), *got), (ry.detach(), rh.detach(), *ref)):
        assert float((a.double() - b).norm() / b.norm()) <= bound
    # the same rows token by token
    x, Wi, bi, Wo, bo, h0 = tensors
    state = h0.clone()
    for t in range(int(lengths.min())):
        out, _ = gated_step(linear_act(x[t], Wi, bi), state, out_state=state)
        step = linear_act(out, Wo, bo, activation="silu", residual=x[t])
        assert float((step.double() - ry[t]).norm() / ry[t].norm()) <= bound


@pytest.mark.gpu
@pytest.mark.parametrize("activation", list(ACTIVATIONS))
@pytest.mark.parametrize("M", [6, 90])
def test_linear_gradient_against_differences(activation, M):
    x, W, bias, residual, dy = linear_problem(torch.float32, M, 72, 40, seed=21)
    leaves = [t.detach().requires_grad_(True) for t in (x, W, bias, residual)]
    got = torch.autograd.grad(linear_act(*leaves[:3], activation=activation, residual=leaves[3]), leaves, dy)
    gen = torch.Generator(device="cuda").manual_seed(2)
    step = 1e-6
    for which in range(4):
        base = [t.double() for t in (x, W, bias, residual)]
        way = torch.randn(base[which].shape, device="cuda", generator=gen, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            at = list(base)
            at[which] = at[which] + sign * step * way
            ends.append(float(((act64(at[0] @ at[1].t() + at[2], activation) + at[3]) * dy.double()).sum()))
        slope = (ends[0] - ends[1]) / (2 * step)
        terms = (got[which].double() * way)
        # step^2 times a third derivative and 2^-53 of the sums over step, the gradient's own error as above; a kink of relu
        # within step of a value moves the difference by that value's share
        assert abs(slope - float(terms.sum())) <= 2e-5 * float(terms.abs().sum())


@pytest.mark.gpu
def test_operators_from_two_threads():
    """Two host threads, each training a block on a stream of its own."""
    import threading
    sets = [block_problem(torch.float32, 90, 4, 64, 128, seed=s) for s in (1, 2)]
    want = []
    for tensors, dy in sets:
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        want.append(torch.autograd.grad(block(*leaves)[0], leaves, dy))
    torch.cuda.synchronize()
    got = [None, None]

    def work(k):
        tensors, dy = sets[k]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                leaves = [t.detach().requires_grad_(True) for t in tensors]
                got[k] = torch.autograd.grad(block(*leaves)[0], leaves, dy)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))


@pytest.mark.gpu
def test_operators_on_another_stream():
    tensors, dy = block_problem(torch.bfloat16, 90, 4, 64, 128)
    ref = [t.detach().requires_grad_(True) for t in tensors]
    want = torch.autograd.grad(block(*ref)[0], ref, dy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        got = torch.autograd.grad(block(*leaves)[0], leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,B,K,H", [(1, 2, 64, 64), (90, 4, 64, 128), (600, 16, 128, 256)])
def test_operators_replay_in_graphs(dtype, T, B, K, H):
    """Two captured training steps of different inputs, replayed in turn and beside each other on two streams."""
    from gru_triton_b200.graphed import GraphedStep

    def step(x, Wi, bi, Wo, bo, h0, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, Wi, bi, Wo, bo, h0)]
        y, h_T = block(*leaves)
        return (y.detach(), h_T.detach(), *torch.autograd.grad(y, leaves, dy))

    sets = [block_problem(dtype, T, B, K, H, seed=s) for s in (1, 2, 3)]
    want = [step(*t, dy) for t, dy in sets]
    graphs = [GraphedStep(step, [*t, dy]) for t, dy in sets[:2]]
    for k in (0, 1, 0):
        got = graphs[k](*sets[k][0], sets[k][1])
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))
    got = graphs[0](*sets[2][0], sets[2][1])                     # new inputs in the captured step
    assert all(torch.equal(a, b) for a, b in zip(got, want[2]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[k](*sets[k][0], sets[k][1])
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(graphs[k].static_outputs, want[k]))
    _lib.check_device_status()


# ---- refusals (no GPU) --------------------------------------------------------------------------------

def test_scan_refusals():
    gi, h0 = torch.zeros(4, 2, 16), torch.zeros(2, 8)
    for bad, match in [((gi, h0), "CUDA"), ((gi.double(), h0), "dtype"), ((gi[..., :15], h0), "2H"), ((gi[0], h0), "2H"),
                       ((gi[:0], h0), "T"), ((gi[:, :0], h0[:0]), "B"), ((gi[..., :0], h0[:, :0]), "H"),
                       ((gi, h0.half()), "float32"), ((gi, h0[:1]), "shape")]:
        with pytest.raises(ValueError, match=match):
            gated_scan(*bad)
    with pytest.raises(ValueError, match="candidate"):
        gated_scan(gi, h0, candidate="relu")
    for lengths, match in [(torch.zeros(2), "int32 or int64"), (torch.zeros(3, dtype=torch.int64), "shape"),
                           (torch.zeros(2, dtype=torch.int64), "CUDA")]:
        with pytest.raises(ValueError, match=match):
            gated_scan(gi, h0, lengths=lengths)
    for bad, match in [((gi[0], h0), "CUDA"), ((gi, h0), "2H"), ((gi[0], h0.double()), "float32"), ((gi[0, :0], h0[:0]), "B"),
                       ((gi[0], h0[:, :4]), "shape")]:
        with pytest.raises(ValueError, match=match):
            gated_step(*bad)
    with pytest.raises(ValueError, match="out_state"):
        gated_step(gi[0], h0, out_state=h0.half())
    # sizes that the 32-bit counts of the library do not hold
    with pytest.raises(ValueError, match="2\\^30"):
        gated_scan(torch.zeros(1, 1, 2).expand(2 ** 32 + 4, 1, 2))
    with pytest.raises(ValueError, match="2\\^30"):
        gated_step(torch.zeros(1, 16).expand(2 ** 29, 16), torch.zeros(1, 8).expand(2 ** 29, 8))


def test_linear_refusals():
    x, W, b, r = torch.zeros(4, 16), torch.zeros(8, 16), torch.zeros(8), torch.zeros(4, 8)
    for args, kw, match in [((x, W, b), {}, "CUDA"), ((x.double(), W.double()), {}, "dtype"), ((x, W.half()), {}, "W dtype"),
                            ((x, W[:, :8]), {}, "N, K"), ((x, W[0]), {}, "N, K"), ((x, W[:0]), {}, "N=0"), ((x, W, b[:4]), {}, "bias"),
                            ((x, W, b), {"residual": r[:1]}, "residual"), ((x, W, b), {"activation": "swish"}, "activation"),
                            ((x, W, b.half()), {}, "bias dtype"), ((x[:, :0], W[:, :0]), {}, "K=0")]:
        with pytest.raises(ValueError, match=match):
            linear_act(*args, **kw)
    with pytest.raises(ValueError, match="rows"):
        linear_act(torch.zeros(1, 16).expand(2 ** 32 + 4, 16), W)


def test_library_refuses_bad_arguments():
    """The C entries answer with a status before any device work."""
    import ctypes
    lib = _lib.load()
    a = _lib.CGatedArgs()
    assert lib.b200gru_gated_scan_forward(None, None) == 1 and lib.b200gru_gated_scan_backward(ctypes.byref(a), None) == 1
    a.T = a.B = a.H = 4
    a.gi = 256
    assert lib.b200gru_gated_scan_forward(ctypes.byref(a), None) == 1                   # no outputs
    a.dtype = 3
    assert lib.b200gru_gated_scan_forward(ctypes.byref(a), None) == 1
    a.dtype, a.lengths, a.length_bytes = 0, 256, 2
    assert lib.b200gru_gated_scan_forward(ctypes.byref(a), None) == 1
    assert lib.b200gru_gated_states_bytes(64, 200, 96) == 200 * 96 * 4 and lib.b200gru_gated_states_bytes(0, 2, 3) == 0
    assert lib.b200gru_gated_step(0, 1, 0, 4, 256, 8, 256, 4, 256, 256, 4, None) == 1
    assert lib.b200gru_gated_step(0, 1, 2, 4, 256, 8, 256, 4, 256, 256, 3, None) == 1   # rows of the new state overlap
    p = _lib.CLinearArgs()
    bad = ctypes.c_size_t(-1).value
    assert lib.b200gru_linear_act_workspace_bytes(ctypes.byref(p), 0) == bad and lib.b200gru_linear_act_forward(None, None) == 1
    p.M = p.K = p.N = p.ldx = p.ldw = 8
    p.x = p.W = 256
    assert lib.b200gru_linear_act_workspace_bytes(ctypes.byref(p), 0) != bad
    assert lib.b200gru_linear_act_forward(ctypes.byref(p), None) == 1                   # no y
    assert lib.b200gru_linear_act_backward(ctypes.byref(p), None) == 1                  # no dy
    p.dy, p.lddy, p.activation = 256, 8, 2
    assert lib.b200gru_linear_act_backward(ctypes.byref(p), None) == 1                  # no slope


# ---- calls that look past autograd (no GPU) ------------------------------------------------------------

@pytest.fixture
def opaque(monkeypatch):
    """The operators with their library calls replaced by memory that nobody wrote, on CPU tensors."""
    from gru_triton_b200 import linear_act as linear, scan_gated as scan

    def fake_scan(gi, h0, lengths, candidate, want_states):
        T, B, H = gi.shape[0], gi.shape[1], gi.shape[2] // 2
        return gi.new_zeros((T, B, H)), gi.new_zeros((B, H)), gi.new_zeros(1)

    def fake_linear(x, W, bias, residual, activation, want_slope):
        return x.new_zeros((*x.shape[:-1], W.shape[0])), None

    monkeypatch.setattr(scan, "_check_devices", lambda *a: None)
    monkeypatch.setattr(scan, "_forward", fake_scan)
    monkeypatch.setattr(linear, "_check", lambda *a: None)
    monkeypatch.setattr(linear, "_forward", fake_linear)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(opaque, grad):
    from torch.autograd import forward_ad as fwad
    gi, W = torch.randn(3, 2, 8), torch.randn(5, 8)
    for call in (lambda t: gated_scan(t), lambda t: linear_act(t, W), lambda t: linear_act(W, t[0]), lambda t: gated_step(t[0], torch.zeros(2, 4))):
        with torch.set_grad_enabled(grad), fwad.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
                call(fwad.make_dual(gi, torch.ones_like(gi)))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.jvp(lambda t: call(t), (gi,), (torch.ones_like(gi),))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.vmap(lambda t: call(t))(torch.stack([gi, gi]))


def test_traces_hold_the_operators(opaque):
    gi, W = torch.randn(3, 2, 8), torch.randn(5, 8)
    for call, t in ((lambda t: gated_scan(t), gi), (lambda t: linear_act(t, W), gi)):
        with torch.no_grad():
            graph = torch.jit.trace(call, (t,), check_trace=False).graph
        assert any(n.kind() == "prim::PythonOp" for n in graph.nodes()) and "empty" not in str(graph) and "zeros" not in str(graph)
    with pytest.raises(ValueError, match="tracing"):
        torch.jit.trace(lambda t: gated_step(t, torch.zeros(2, 4)), (gi[0],), check_trace=False)


@pytest.mark.gpu
def test_traced_calls_run_the_operators():
    gi, h0, _, _ = problem(torch.float32, 40, 3, 32, seed=2)
    W = torch.randn(24, 32, device="cuda")

    def step(gi):
        out, h_T = gated_scan(gi)
        return linear_act(out, W, activation="silu"), h_T

    with torch.no_grad():
        traced = torch.jit.trace(step, (torch.zeros_like(gi),), check_trace=False)
        for a, b in zip(traced(gi), step(gi)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("same", [True, False])
def test_step_tells_autograd_that_it_wrote_a_state(opaque, monkeypatch, same):
    from gru_triton_b200 import scan_gated as scan
    monkeypatch.setattr(scan, "call_on", lambda *a: 0)
    gi, w = torch.randn(2, 8), torch.ones(2, 4, requires_grad=True)
    state = torch.zeros(2, 4)
    loss = (w * state).sum()
    table = torch.zeros(4, 4)
    other = (w * table[:2]).sum()
    gated_step(gi, state if same else torch.zeros(2, 4), out_state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    gated_step(gi, state, out_state=table[2:])           # a view: its base counts
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        other.backward()
    version = state._version
    gated_step(gi, state)
    assert state._version == version
    with pytest.raises(ValueError, match="gradients"):
        gated_step(gi, state, out_state=torch.zeros(2, 4, requires_grad=True))
    with torch.no_grad():
        gated_step(gi, state, out_state=w)
    with torch.inference_mode():
        gated_step(gi, state.clone(), out_state=torch.zeros(2, 4))


# ---- the largest sizes (no GPU) -------------------------------------------------------------------------

def test_sizes_that_tiles_would_carry_past_32_bits_are_refused():
    row, w = torch.zeros(1, 16), torch.zeros(8, 16)
    with pytest.raises(ValueError, match="rows"):
        linear_act(row.expand(2 ** 31 - 500, 16), w)
    with pytest.raises(ValueError, match="CUDA"):                # the largest that is taken, stopped by its device
        linear_act(row.expand(2 ** 31 - 512, 16), w)
    one = torch.zeros(1, 1, 1)
    with pytest.raises(ValueError, match="units"):
        gated_scan(one.expand(1, 1, 2 ** 31))
    with pytest.raises(ValueError, match="CUDA"):
        gated_scan(one.expand(1, 1, 2 ** 31 - 128))
    with pytest.raises(ValueError, match="units"):
        gated_step(one[0].expand(1, 2 ** 31), one[0].expand(1, 2 ** 30))


def test_library_refuses_sizes_past_32_bits():
    lib = _lib.load()
    p, none = _lib.CLinearArgs(), ctypes.c_size_t(-1).value
    p.K, p.N, p.dtype, p.x, p.W, p.ldx, p.ldw = 8, 8, 1, 4096, 4096, 8, 8
    for M, taken in ((2 ** 31 - 1, False), (2 ** 31 - 16, False), (2 ** 31 - 511, False), (2 ** 31 - 512, True)):
        p.M = M
        need = lib.b200gru_linear_act_workspace_bytes(ctypes.byref(p), 0)
        assert need == (0 if taken else none)
    a = _lib.CGatedArgs()
    a.T, a.B, a.H = 1, 1, 2 ** 30 - 63
    a.gi = a.out = a.h_T = a.states = a.dgi = 4096
    a.gi_t = a.gi_b = a.out_t = a.out_b = a.dgi_t = a.dgi_b = 2 ** 31
    unsupported = lib.b200gru_gated_scan_forward(ctypes.byref(a), None)
    assert unsupported == lib.b200gru_gated_scan_backward(ctypes.byref(a), None) == 2
    assert lib.b200gru_gated_step(0, 1, 1, 2 ** 30 - 63, 4096, 2 ** 31, 4096, 2 ** 31, 4096, 4096, 2 ** 31, None) == 2
