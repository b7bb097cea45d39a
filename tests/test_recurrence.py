"""Gated linear recurrence: refusals on the CPU; on the GPU against the definition in 64 bits, forward and backward.

Tolerances follow the roundings.  With u = 2^-24 a gate's sigmoid is within 5u of its value (the exponential, one sum,
one quotient, one product), a product and a sum add u each: 8u per step relative to the sum of the absolute values of the
terms, on every path by which a term reaches a result, in whatever order the steps are joined.  That is the recursion
`E[t] = a E[t-1] + 8u G[t]` with `G` the recurrence of absolute values; the last rounding to the tensor's type adds half
a step of that type.
"""

import numpy as np
import pytest
import torch

from metta_amd.recurrence import gated_recurrence, gated_recurrence_step

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _definition(x, g, state, resets, dh=None, dlast=None):
    """numpy float64 [rows, steps, width]; returns values and error bounds (before the last rounding) by name."""
    rows, steps, width = x.shape
    with np.errstate(over="ignore"):
        a, w = 1.0 / (1.0 + np.exp(-g)), 1.0 / (1.0 + np.exp(g))
    keep = np.ones((rows, steps, 1)) if resets is None else 1.0 - resets[..., None].astype(np.float64)
    h, before, G, E, Gb, Eb = (np.zeros_like(x) for _ in range(6))
    s = np.zeros((rows, width)) if state is None else state
    sg, se = np.abs(s), np.zeros_like(s)
    for t in range(steps):
        k = keep[:, t]
        before[:, t], Gb[:, t], Eb[:, t] = s * k, sg * k, se * k
        s = a[:, t] * before[:, t] + w[:, t] * x[:, t]
        sg = a[:, t] * Gb[:, t] + w[:, t] * np.abs(x[:, t])
        se = a[:, t] * Eb[:, t] + 8 * U * sg
        h[:, t], G[:, t], E[:, t] = s, sg, se
    out = {"h": (h, E), "last": (s, se)}
    if dh is None and dlast is None:
        return out
    d = np.zeros((rows, width)) if dlast is None else dlast.copy()
    dg_, de = np.abs(d), np.zeros_like(d)
    dx, dgate, ex, eg = (np.zeros_like(x) for _ in range(4))
    for t in range(steps - 1, -1, -1):
        if dh is not None:
            d = d + dh[:, t]
            dg_ = dg_ + np.abs(dh[:, t])
            de = de + 2 * U * dg_
        slope, span = a[:, t] * w[:, t], Gb[:, t] + np.abs(x[:, t])
        dx[:, t], ex[:, t] = w[:, t] * d, w[:, t] * (de + 8 * U * dg_)
        dgate[:, t] = d * (before[:, t] - x[:, t]) * slope
        eg[:, t] = slope * (de * span + dg_ * (Eb[:, t] + 16 * U * span) + de * Eb[:, t])
        d, dg_ = keep[:, t] * a[:, t] * d, keep[:, t] * a[:, t] * dg_
        de = keep[:, t] * a[:, t] * de + 8 * U * dg_
    out.update(dx=(dx, ex), dgate=(dgate, eg), dstate=(d, de))
    return out


def _close(got, want, name):
    value, error = want
    t = got.dtype
    fi = torch.finfo(t)
    half = fi.eps / 2 * np.abs(value) + fi.smallest_normal * fi.eps / 2
    tol = error * (1 + fi.eps) + (half if t != torch.float32 else 1e-37)
    off = np.abs(got.detach().double().cpu().numpy() - value)
    assert np.all(off <= tol), f"{name}: off by {np.max(off - tol)} over the bound at {np.unravel_index(np.argmax(off - tol), off.shape)}"


def _inputs(rows, steps, width, dtype, seed=0, resets=0.05, gate_mean=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, steps, width, generator=g).to(dtype)
    gate = (torch.randn(rows, steps, width, generator=g) * 2 + gate_mean).to(dtype)
    return (x, gate, torch.randn(rows, width, generator=g), torch.rand(rows, steps, generator=g) < resets,
            torch.randn(rows, steps, width, generator=g).to(dtype), torch.randn(rows, width, generator=g))  # fmt: skip


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


# ---- refusals: on the CPU, before anything reaches a device --------------------------------------------------------


def test_refusals():
    x, s, r = torch.zeros(2, 5, 4), torch.zeros(2, 4), torch.zeros(2, 5, dtype=torch.bool)
    cases = [
        ("3D", (x[0], x[0])),
        ("even", (torch.zeros(2, 5, 3),)),
        ("same shape", (x, torch.zeros(2, 5, 3))),
        ("float32, bfloat16 or float16", (x.double(), x.double())),
        ("float32, bfloat16 or float16", (x, x.half())),
        ("state must be float32", (x, x, s.half())),
        ("rows, width", (x, x, torch.zeros(4))),
        ("rows, width", (x, x, torch.zeros(1, 4))),
        ("bool or uint8", (x, x, s, r.float())),
        ("without its last", (x, x, s, r[:, :4])),
        ("same device", (x, x, s.to("meta"))),
        ("on GPU", (x, x, s, r)),
    ]
    for text, args in cases:
        with pytest.raises(RuntimeError, match=text):
            gated_recurrence(*args)
    with pytest.raises(RuntimeError, match="2D"):
        gated_recurrence_step(x, x, s)
    with pytest.raises(RuntimeError, match="on GPU"):
        gated_recurrence_step(x[:, 0], x[:, 0], s)
    with pytest.raises(RuntimeError, match="2\\^31"):
        big = torch.zeros(1).expand(1 << 20, 1, 1 << 12)
        gated_recurrence(big, big)


def test_library_refuses_bad_arguments_before_any_launch():
    import ctypes as ct

    from metta_amd import native

    L = native.load()
    assert L.mg_gated_recurrence(None, None, None, None, None) != 0
    for change, text in (({"type": 3}, b"type"), ({"rows": -1}, b"negative"), ({"rows": 1 << 20, "width": 1 << 12}, b"2^31"), ({}, b"NULL")):
        r = native.MgRecurrence(rows=2, steps=3, width=4)
        for k, v in change.items():
            setattr(r, k, v)
        assert L.mg_gated_recurrence(ct.byref(r), None, None, None, None) != 0 and text in L.mg_last_error(), change
        assert L.mg_gated_recurrence_backward(ct.byref(r), None, 0, 0, None, None) != 0 and text in L.mg_last_error(), change
    nothing = native.MgRecurrence(rows=0, steps=3, width=4)
    assert L.mg_gated_recurrence(ct.byref(nothing), None, None, None, None) == 0


# ---- GPU ----------------------------------------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (3, 1, 5), (2, 15, 7), (2, 16, 8), (2, 17, 2), (5, 33, 33), (1, 1000, 3), (7, 65, 128), (300, 40, 100),
          (1, 4100, 64), (2, 2049, 130), (1, 129, 1000), (700, 48, 256), (300, 300, 64), (130, 600, 128), (1, 70000, 3)]  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_definition(shape, dtype):
    x, gate, state, resets, dh, dlast = _inputs(*shape, dtype, seed=sum(shape))
    want = _definition(*map(_np, (x, gate, state, resets, dh, dlast)))
    xs, gs, ss = (t.cuda().requires_grad_() for t in (x, gate, state))
    h, last = gated_recurrence(xs, gs, ss, resets.cuda())
    assert h.dtype == dtype and last.dtype == torch.float32
    grads = torch.autograd.grad([h, last], [xs, gs, ss], [dh.cuda(), dlast.cuda()])
    for name, got in zip(("h", "last", "dx", "dgate", "dstate"), (h, last, *grads)):
        _close(got, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["packed", "time_major", "sliced", "flipped_columns", "odd_offset"])
def test_layouts(layout, dtype):
    """Strided views give the values of the contiguous call, and gradients in their own layout."""
    x, gate, state, resets, dh, dlast = (t.cuda() for t in _inputs(9, 70, 24, dtype, seed=3))
    xs, gs, ss = (t.clone().requires_grad_() for t in (x, gate, state))
    h0, last0 = gated_recurrence(xs, gs, ss, resets)
    want = torch.autograd.grad([h0, last0], [xs, gs, ss], [dh, dlast])
    if layout == "packed":
        leaf = torch.cat([x, gate], -1).requires_grad_()
        h, last = gated_recurrence(leaf, None, ss, resets)
    elif layout == "time_major":
        leaf = torch.stack([x, gate]).transpose(1, 2).contiguous().requires_grad_()
        h, last = gated_recurrence(leaf[0].transpose(0, 1), leaf[1].transpose(0, 1), ss, resets.t().contiguous().t())
    elif layout == "sliced":
        leaf = torch.zeros(2, 9, 75, 31, dtype=dtype, device="cuda")
        leaf[:, :, 5:, 4:28] = torch.stack([x, gate])
        leaf.requires_grad_()
        h, last = gated_recurrence(leaf[0, :, 5:, 4:28], leaf[1, :, 5:, 4:28], ss, resets)
    elif layout == "flipped_columns":  # columns that are not adjacent
        leaf = torch.stack([x, gate], -1).requires_grad_()
        h, last = gated_recurrence(leaf[..., 0], leaf[..., 1], ss, resets)
    else:  # rows that start off every wide boundary
        flat = torch.zeros(2 * x.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = torch.stack([x, gate]).flatten()
        leaf = flat.requires_grad_()
        both = leaf[1:].view(2, *x.shape)
        h, last = gated_recurrence(both[0], both[1], ss, resets)
    got, dstate = torch.autograd.grad([h, last], [leaf, ss], [dh.transpose(0, 1).contiguous().transpose(0, 1), dlast])
    if layout == "packed":
        dx, dg = got.chunk(2, -1)
    elif layout == "time_major":
        dx, dg = got[0].transpose(0, 1), got[1].transpose(0, 1)
    elif layout == "sliced":
        dx, dg = got[0, :, 5:, 4:28], got[1, :, 5:, 4:28]
    elif layout == "flipped_columns":
        dx, dg = got.unbind(-1)
    else:
        dx, dg = got[1:].view(2, *x.shape)
    # the same arithmetic or a different split of it: either way inside the bounds of the definition
    ref = _definition(*map(_np, (x, gate, state, resets, dh, dlast)))
    for name, t in (("h", h), ("last", last), ("dx", dx), ("dgate", dg), ("dstate", dstate)):
        _close(t, ref[name], f"{layout} {name}")
    for name, t in (("h", h0), ("last", last0), ("dx", want[0]), ("dgate", want[1]), ("dstate", want[2])):
        _close(t, ref[name], f"contiguous {name}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_optional_parts(dtype):
    """No state, no resets, uint8 resets, a gradient of one output only, a state shared by all rows."""
    x, gate, state, resets, dh, dlast = _inputs(4, 50, 20, dtype, seed=8)
    xs, gs = x.cuda().requires_grad_(), gate.cuda().requires_grad_()
    h, last = gated_recurrence(xs, gs)
    ref = _definition(_np(x), _np(gate), None, None, _np(dh), None)
    _close(h, ref["h"], "h"), _close(last, ref["last"], "last")
    for name, got in zip(("dx", "dgate"), torch.autograd.grad(h, [xs, gs], dh.cuda())):
        _close(got, ref[name], name)
    h, last = gated_recurrence(xs, gs, None, resets.to(torch.uint8).cuda())
    ref = _definition(_np(x), _np(gate), None, _np(resets), None, _np(dlast))
    for name, got in zip(("dx", "dgate"), torch.autograd.grad(last, [xs, gs], dlast.cuda())):
        _close(got, ref[name], name)
    one = state[:1].cuda().requires_grad_()  # every row starts from the same learned state: its gradient is the rows' sum
    h, last = gated_recurrence(xs, gs, one.expand(4, 20), resets.cuda())
    ref = _definition(_np(x), _np(gate), _np(state[:1].expand(4, 20)), _np(resets), _np(dh), None)
    (got,) = torch.autograd.grad(h.sum() * 0 + (h.float() * dh.cuda().float()).sum(), [one])
    value, error = ref["dstate"]
    off = np.abs(_np(got)[0] - value.sum(0))
    assert np.all(off <= error.sum(0) + 8 * U * np.abs(value).sum(0))


@pytest.mark.gpu
def test_gradient_against_differences():
    x, gate, state, resets, dh, dlast = _inputs(2, 20, 6, torch.float32, seed=5)
    xs, gs, ss = (t.cuda().requires_grad_() for t in (x, gate, state))
    grads = torch.autograd.grad(gated_recurrence(xs, gs, ss, resets.cuda()), [xs, gs, ss], [dh.cuda(), dlast.cuda()])

    def loss(x, g, s):
        out = _definition(_np(x) if torch.is_tensor(x) else x, g, s, _np(resets))
        return (out["h"][0] * _np(dh)).sum() + (out["last"][0] * _np(dlast)).sum()

    base = [_np(t) for t in (x, gate, state)]
    rng, eps = np.random.default_rng(0), 1e-5
    for k in range(3):
        for _ in range(12):
            at = tuple(rng.integers(0, n) for n in base[k].shape)
            ups, downs = [b.copy() for b in base], [b.copy() for b in base]
            ups[k][at] += eps
            downs[k][at] -= eps
            slope = (loss(*ups) - loss(*downs)) / (2 * eps)
            # differences in 64 bits: their own error is of order eps^2 = 1e-10; the kernel's some hundred u
            assert abs(grads[k][at].item() - slope) <= 2e-5 * max(1.0, abs(slope)), (k, at)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_values(dtype):
    """Closed and open gates, a held tail, NaN and infinity in a state that a reset drops, every step a reset."""
    inf, n = float("inf"), 37
    x = torch.randn(2, n, 8, generator=torch.Generator().manual_seed(1)).to(dtype)
    gate = torch.zeros(2, n, 8, dtype=dtype)
    gate[0], gate[1] = inf, -inf
    state = torch.randn(2, 8)
    h, last = gated_recurrence(x.cuda(), gate.cuda(), state.cuda())
    assert torch.equal(h[0].cpu(), state[0].to(dtype).expand(n, 8))  # an open gate keeps the state exactly
    assert torch.equal(h[1].cpu(), x[1]) and torch.equal(last[0].cpu(), state[0])  # a closed one takes x exactly
    bad = torch.full((2, 8), float("nan"))
    bad[1] = inf
    resets = torch.zeros(2, n, dtype=torch.bool)
    resets[:, 0] = True
    g = torch.randn(2, n, 8, generator=torch.Generator().manual_seed(2)).to(dtype)
    leaf = bad.cuda().requires_grad_()
    h, last = gated_recurrence(x.cuda(), g.cuda(), leaf, resets.cuda())
    (ds,) = torch.autograd.grad(h.float().sum(), leaf)
    assert bool(torch.isfinite(h).all()) and bool((ds == 0).all())
    h, last = gated_recurrence(x.cuda(), g.cuda(), bad.cuda(), torch.ones(2, n, dtype=torch.bool, device="cuda"))
    w = 1.0 / (1.0 + np.exp(_np(g)))
    _close(h, (w * _np(x), 8 * U * np.abs(w * _np(x))), "all resets")
    h, _ = gated_recurrence(x.cuda(), g.cuda(), bad.cuda())
    assert bool(torch.isnan(h[0]).all())  # and without one, NaN is seen


@pytest.mark.gpu
def test_empty():
    for rows, steps, width in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        x = torch.zeros(rows, steps, width, device="cuda", requires_grad=True)
        s = torch.randn(rows, width, device="cuda", requires_grad=True)
        h, last = gated_recurrence(x, x, s)
        assert h.shape == x.shape and torch.equal(last, s)
        assert torch.equal(torch.autograd.grad(last.sum() + h.sum(), s)[0], torch.ones_like(s))
        assert torch.equal(gated_recurrence(x, x)[1], torch.zeros_like(s))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (24, 128), (5, 33), (1000, 100), (3, 2050), (4100, 256)])
def test_step(rows, width, dtype):
    x, gate, state, resets, _, _ = (t.cuda() for t in _inputs(rows, 1, width, dtype, seed=rows, resets=0.3))
    want = _definition(*map(_np, (x, gate, state, resets)))
    h, new = gated_recurrence_step(x[:, 0], gate[:, 0], state, resets[:, 0])
    _close(h, (want["h"][0][:, 0], want["h"][1][:, 0]), "h")
    _close(new, want["last"], "state")
    assert (h is new) == (dtype == torch.float32)
    packed, kept = torch.cat([x[:, 0], gate[:, 0]], -1), state.clone()
    h2, new2 = gated_recurrence_step(packed, None, kept, resets[:, 0], out_state=kept)  # in place
    assert new2 is kept and torch.equal(kept, new) and torch.equal(h2, h)
    h3, new3 = gated_recurrence_step(x[:, 0], gate[:, 0], state)
    want = _definition(_np(x), _np(gate), _np(state), None)
    _close(new3, want["last"], "no resets")


@pytest.mark.gpu
def test_steps_follow_the_scan():
    """Steps from the state that a scan left, and a segment cut in two: both go on where it stopped."""
    x, gate, state, resets, _, _ = (t.cuda() for t in _inputs(6, 90, 40, torch.bfloat16, seed=11))
    want = _definition(*map(_np, (x, gate, state, resets)))
    s = state
    for t in range(90):
        h, s = gated_recurrence_step(x[:, t], gate[:, t], s, resets[:, t])
        _close(h, (want["h"][0][:, t], want["h"][1][:, t]), f"step {t}")
    h1, mid = gated_recurrence(x[:, :37], gate[:, :37], state, resets[:, :37])
    h2, last = gated_recurrence(x[:, 37:], gate[:, 37:], mid, resets[:, 37:])
    _close(torch.cat([h1, h2], 1), want["h"], "cut in two")
    _close(last, want["last"], "last")


@pytest.mark.gpu
def test_step_refusals_on_device():
    x, s = torch.zeros(2, 4, device="cuda"), torch.zeros(2, 4, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        gated_recurrence_step(x.requires_grad_(), x, s)
    x = x.detach()
    for bad in (torch.zeros(2, 8, device="cuda")[:, ::2], torch.zeros(2, 4), torch.zeros(2, 4, device="cuda").half(), torch.zeros(4, device="cuda")):
        with pytest.raises(RuntimeError, match="out_state"):
            gated_recurrence_step(x, x, s, out_state=bad)


@pytest.mark.gpu
def test_another_stream_and_repeats():
    """On a stream of its own the results are the same to the bit, and so are those of a second run."""
    x, gate, state, resets, dh, dlast = (t.cuda() for t in _inputs(3, 3000, 50, torch.float32, seed=21))

    def once():
        leaves = [t.clone().requires_grad_() for t in (x, gate, state)]
        out = gated_recurrence(*leaves, resets)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, [dh, dlast]))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_graph_capture():
    """Two captured graphs (a rollout step in place; a segment forward) replayed in turn, against eager results."""
    x, gate, state, resets, _, _ = (t.cuda() for t in _inputs(5, 1200, 64, torch.bfloat16, seed=2))
    kept = state.clone()
    xs, gs, rs = x[:, 0].clone(), gate[:, 0].clone(), resets[:, 0].clone()
    gated_recurrence_step(xs, gs, kept.clone(), rs)
    gated_recurrence(x, gate, state, resets)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g1):
        h1, _ = gated_recurrence_step(xs, gs, kept, rs, out_state=kept)
    with torch.no_grad(), torch.cuda.graph(g2):
        h2, last2 = gated_recurrence(x, gate, state, resets)
    eager = state.clone()
    for t in range(4):
        xs.copy_(x[:, t]), gs.copy_(gate[:, t]), rs.copy_(resets[:, t])
        g1.replay()
        he, eager = gated_recurrence_step(x[:, t], gate[:, t], eager, resets[:, t])
        assert torch.equal(h1, he) and torch.equal(kept, eager), t
        x.add_(0.5)
        g2.replay()
        hs, ls = gated_recurrence(x, gate, state, resets)
        assert torch.equal(h2, hs) and torch.equal(last2, ls), t


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A view whose second row starts more than 2^32 elements after the first."""
    flat = torch.zeros((1 << 32) + 4096, dtype=torch.float16, device="cuda")
    x = torch.as_strided(flat, (2, 20, 8), (1 << 32, 8, 1))
    a, gate, state, resets, dh, dlast = _inputs(2, 20, 8, torch.float16, seed=6)
    x.copy_(a)
    h, last = gated_recurrence(x, gate.cuda(), state.cuda(), resets.cuda())
    want = _definition(*map(_np, (a, gate, state, resets)))
    _close(h, want["h"], "h"), _close(last, want["last"], "last")


@pytest.mark.gpu
def test_saved_tensors_are_watched():
    x = torch.randn(2, 40, 8, device="cuda", requires_grad=True)
    y = x * 1.0
    h, _ = gated_recurrence(y, y)
    y.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_in_a_captured_graph(dtype):
    """Forward and backward captured once, replayed on new inputs with eager work in between; other leaves do the eager part."""
    x, gate, state, resets, dh, dlast = (t.cuda() for t in _inputs(3, 700, 40, dtype, seed=12))
    leaves = [t.clone().requires_grad_() for t in (x, gate, state)]

    def once(a, b, s):
        h, last = gated_recurrence(a, b, s, resets)
        return [h, last, *torch.autograd.grad([h, last], [a, b, s], [dh, dlast])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            once(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = once(*leaves)
    for k in range(4):
        with torch.no_grad():
            for t in leaves:
                t.mul_(0.9).add_(0.1 * k)
        g.replay()
        torch.cuda.synchronize()
        want = once(*(t.detach().clone().requires_grad_() for t in leaves))
        for a, b in zip(out, want):
            assert torch.equal(a, b), k


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_saved_tensors_that_move(packed, dtype):
    """Hooks that take what was saved to the host and back give the same gradients."""
    x, gate, state, resets, dh, dlast = (t.cuda() for t in _inputs(4, 90, 24, dtype, seed=17))

    def once():
        leaf = torch.cat([x, gate], -1).requires_grad_() if packed else x.clone().requires_grad_()
        other = [] if packed else [gate.transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()]
        s = state.clone().requires_grad_()
        out = gated_recurrence(leaf * 1.0, None if packed else other[0] * 1.0, s, resets)
        return out, [leaf, s, *other]

    out, leaves = once()
    want = torch.autograd.grad(out, leaves, [dh, dlast])
    with torch.autograd.graph.save_on_cpu():
        out, leaves = once()
    junk = [torch.randn_like(x) for _ in range(8)]  # memory that was free is written over
    got = torch.autograd.grad(out, leaves, [dh, dlast])
    assert len(junk) == 8
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x = torch.randn(2, 20, 4, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(gated_recurrence(x, x)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()


@pytest.mark.gpu
def test_overlapping_states_are_refused():
    flat = torch.zeros(100, device="cuda")
    x = torch.zeros(2, 8, device="cuda")
    for at in (4, 12):
        with pytest.raises(RuntimeError, match="overlap"):
            gated_recurrence_step(x, x, flat[8:24].view(2, 8), out_state=flat[at : at + 16].view(2, 8))
    gated_recurrence_step(x, x, flat[8:24].view(2, 8), out_state=flat[24:40].view(2, 8))


@pytest.mark.gpu
def test_in_place_states_are_noticed_and_inference_mode():
    x = torch.randn(3, 8, device="cuda")
    state = torch.zeros(3, 8, device="cuda")
    w = torch.ones(3, 8, device="cuda", requires_grad=True)
    product = (w * state).sum()  # keeps the state for its gradient
    gated_recurrence_step(x, x, state, out_state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    want, _ = gated_recurrence_step(x, x, torch.zeros(3, 8, device="cuda"))
    with torch.inference_mode():
        state = torch.zeros(3, 8, device="cuda")
        h, s = gated_recurrence_step(x, x, state, out_state=state)
        y, last = gated_recurrence(x[:, None], x[:, None])
        assert s is state and torch.equal(h, want) and torch.equal(y[:, 0], want) and torch.equal(last, want)


@pytest.mark.gpu
def test_from_several_threads():
    """Calls on streams of their own, forwards and backwards, from threads at the same time."""
    from concurrent.futures import ThreadPoolExecutor

    inputs = [[t.cuda() for t in _inputs(3, 70 + 300 * k, 32, torch.bfloat16, seed=k)] for k in range(4)]

    def work(k):
        x, gate, state, resets, dh, dlast = inputs[k]
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                leaves = [t.clone().requires_grad_() for t in (x, gate, state)]
                h, last = gated_recurrence(*leaves, resets)
                out = [h.detach(), last.detach(), *torch.autograd.grad([h, last], leaves, [dh, dlast])]
            s.synchronize()
        return out

    torch.cuda.synchronize()
    want = [work(k) for k in range(4)]
    with ThreadPoolExecutor(4) as pool:
        for a, b in zip(pool.map(work, range(4)), want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 10, 8), (2, 10, 7), (2, 200, 8), (2, 200, 7), (2, 1000, 8), (1300, 40, 128)])
def test_nan_gates(shape, dtype):
    """A gate of NaN, whatever its sign, reaches every result that depends on it, up to the nearest reset and no further: walks,
    tiles, and time cut over blocks."""
    rows, steps, width = shape
    x, gate, state, resets, dh, dlast = _inputs(*shape, dtype, seed=9, resets=3.0 / steps)
    plus, minus, ints = {torch.float32: (0x7FC00000, -0x400000, torch.int32), torch.bfloat16: (0x7FC0, -0x40, torch.int16), torch.float16: (0x7E00, -0x200, torch.int16)}[dtype]
    n, bits, rng = np.zeros(shape, dtype=bool), gate.view(ints).numpy(), np.random.default_rng(1)
    for r in range(rows):
        for c in range(width):
            if (r + c) % 5 != 4:  # (the others have none)
                t = rng.integers(steps)
                bits[r, t, c], n[r, t, c] = minus if (r + c) % 2 else plus, True
    resets[1] = False
    z = resets.numpy()
    h, d, before, after = (np.zeros(shape, dtype=bool) for _ in range(4))
    s = np.zeros((rows, width), dtype=bool)
    for t in range(steps):
        before[:, t] = s & ~z[:, t, None]
        s = before[:, t] | n[:, t]
        h[:, t] = s
    back = np.zeros((rows, width), dtype=bool)
    for t in range(steps - 1, -1, -1):
        after[:, t] = back
        back = (back | n[:, t]) & ~z[:, t, None]
    want = dict(h=h, last=s, dx=after | n, dgate=after | n | before, dstate=back)
    xs, gs, ss = (t.cuda().requires_grad_() for t in (x, gate, state))
    out = gated_recurrence(xs, gs, ss, resets.cuda())
    got = [*out, *torch.autograd.grad(out, [xs, gs, ss], [dh.cuda(), dlast.cuda()])]
    for (name, nan), t in zip(want.items(), got):
        assert np.array_equal(torch.isnan(t).cpu().numpy(), nan), name
        assert bool(torch.isfinite(t[~torch.from_numpy(nan).cuda()]).all()), name


def _views(flat):
    """(what, x, gate, state, resets, out_state) that share memory otherwise than element on element."""
    v = lambda at, *shape: flat[at : at + int(np.prod(shape))].view(*shape)  # noqa: E731
    x, s = v(200, 3, 8), v(300, 3, 8)
    yield "packed projection", v(0, 3, 16), None, s, None, v(0, 3, 8)
    yield "end of a packed projection", v(0, 3, 16), None, s, None, v(40, 3, 8)
    yield "shifted x", v(0, 3, 8), x, s, None, v(4, 3, 8)
    yield "shifted gate", x, v(4, 3, 8), s, None, v(0, 3, 8)
    yield "one element of x", v(23, 3, 8), x, s, None, v(0, 3, 8)
    yield "rows further apart", v(0, 3, 16)[:, :8], x, s, None, v(0, 3, 8)
    yield "a row for all", v(0, 1, 8).expand(3, 8), x, s, None, v(0, 3, 8)
    yield "resets", x, x, s, v(0, 3, 8).view(torch.uint8).flatten()[:3], v(0, 3, 8)
    yield "16 bits", v(0, 3, 8).view(torch.bfloat16)[:, :8], v(200, 3, 8).view(torch.bfloat16)[:, :8], s, None, v(0, 3, 8)


def test_states_written_over_inputs_are_refused():
    """One thread would write what another has yet to read."""
    for what, x, gate, state, resets, out in _views(torch.zeros(400)):
        with pytest.raises(RuntimeError, match="out_state may not overlap"):
            gated_recurrence_step(x, gate, state, resets, out_state=out)
    flat = torch.zeros(400)
    a, b, s = flat[:24].view(3, 8), flat[24:48].view(3, 8), torch.zeros(3, 8)
    fine = [
        (a, b, s, b),  # element on element
        (a, b, s, a),
        (flat[100:260].view(2, 80)[:, :8], b[:2], s[:2], flat[120:136].view(2, 8)),  # between two rows
        (a[:1], b[:1], s[:1], flat[8:16].view(1, 8)),  # side by side
        (flat[:16].view(1, 16), None, s[:1], flat[:8].view(1, 8)),  # one row: candidate on candidate
    ]
    for x, gate, state, out in fine:
        with pytest.raises(RuntimeError, match="on GPU"):
            gated_recurrence_step(x, gate, state, out_state=out)


@pytest.mark.gpu
def test_states_written_element_on_element():
    x, gate, state, resets, _, _ = (t.cuda() for t in _inputs(500, 1, 64, torch.float32, seed=4, resets=0.2))
    x, gate, resets = x[:, 0].contiguous(), gate[:, 0].contiguous(), resets[:, 0].contiguous()
    want = gated_recurrence_step(x, gate, state, resets)[1]
    for k in range(2):
        both = [x.clone(), gate.clone()]
        h, s = gated_recurrence_step(*both, state, resets, out_state=both[k])
        assert s is both[k] and torch.equal(s, want)
    apart = torch.zeros(64, 500, device="cuda").t()  # columns that are not adjacent: copied before the launch
    apart.copy_(x)
    memory = torch.as_strided(apart, (500, 64), (64, 1))
    assert torch.equal(gated_recurrence_step(apart, gate, state, resets, out_state=memory)[1], want)


def test_forward_mode_is_refused():
    """A dual tensor's tangent is not dropped."""
    from torch.autograd import forward_ad

    x, s = torch.zeros(2, 5, 4), torch.zeros(2, 4)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x),), (dual(x), x), (x, dual(x)), (x, x, dual(s))):
            with pytest.raises(RuntimeError, match="gated_recurrence has no forward-mode"):
                gated_recurrence(*args)
        for args in ((dual(x[:, 0]), None, s[:, :2]), (x[:, 0], dual(x[:, 0]), s), (x[:, 0], x[:, 0], dual(s))):
            with pytest.raises(RuntimeError, match="gated_recurrence_step has no forward-mode"):
                gated_recurrence_step(*args)
        with pytest.raises(RuntimeError, match="out_state.*tangent"):
            gated_recurrence_step(x[:, 0], x[:, 0], s, out_state=dual(s.clone()))
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="on GPU"):
            gated_recurrence(dual(x))


@pytest.mark.gpu
def test_forward_mode_is_refused_on_device():
    from torch.autograd import forward_ad

    x = torch.randn(2, 20, 4, device="cuda")
    with forward_ad.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="forward-mode"):
                gated_recurrence(forward_ad.make_dual(leaf, torch.ones_like(x)))
        gated_recurrence(x)


def test_tracing_is_refused():
    """A trace would hold the results' memory and not the launches that fill it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.zeros(2, 5, 4)
    for call in (lambda t: gated_recurrence(t, t)[0], lambda t: gated_recurrence_step(t[:, 0], t[:, 0], t[:, 0])[0]):
        for leaf in (x, x.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                torch.jit.trace(call, leaf, check_trace=False)
        for mode in ("real", "fake"):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(call, tracing_mode=mode)(x)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 40])
def test_negated_views(steps):
    """Views that hold their values negated (the imaginary part of a conjugate) give what their values give, gradients too."""
    x, gate, state, _, dh, dlast = (t.cuda() for t in _inputs(3, steps, 16, torch.float32, seed=5))
    neg = lambda t: torch.complex(torch.zeros_like(t), -t).conj().imag  # noqa: E731
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    got = gated_recurrence_step(neg(x)[:, 0], neg(gate)[:, 0], neg(state))
    for a, b in zip(got, gated_recurrence_step(x[:, 0], gate[:, 0], state)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="out_state"):
        gated_recurrence_step(x[:, 0], gate[:, 0], state, out_state=torch._neg_view(state.clone()))
    leaves = [t.clone().requires_grad_() for t in (x, gate, state)]
    views = [torch._neg_view(-t) for t in leaves]
    assert all(t.is_neg() for t in views)
    out, want = gated_recurrence(*views), gated_recurrence(*leaves)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    for a, b in zip(torch.autograd.grad(out, leaves, [torch._neg_view(-dh), torch._neg_view(-dlast)]), torch.autograd.grad(want, leaves, [dh, dlast])):
        assert torch.equal(a, b)
