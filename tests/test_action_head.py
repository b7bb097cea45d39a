"""The action head (adjusted logits, sampling, re-evaluation): refusals on the CPU; on the GPU against the definition in 64
bits (numpy).

Sampled actions have to be the definition's exactly.  Tolerances of the floating results, with u = 2^-24: a distance
M - l4 is d(1 + 3u) after difference, scale and rounding, its exponential therefore within (3d + 4)u of e^-d; a sum of
them over a thread's share (at most 128 terms) and the tree over the threads adds at most 150u; log and the last rounding
a few u of the value.  So Z is within (3 mean(d) + 154)u relative, and log-probability, entropy and gradients follow by
the chain rule below.  Adjusted logits and their gradients are rounded once: half a step of their type.
"""

import numpy as np
import pytest
import torch

from metta_amd.action_head import adjust_logits, evaluate_actions, pack_allowed, sample_actions

U = 2.0**-24
INF = float("inf")
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _np(t):
    return t.detach().double().cpu().numpy()


def _adjusted(logits, allowed=None, bias=None, history=None, temperature=1.0, repetition=1.0, presence=0.0, frequency=0.0):
    """float64 [N, V] adjusted logits and slopes; `allowed` bool."""
    l = _np(logits)
    n, v = l.shape
    c = np.zeros((n, v))
    if history is not None:
        for i, row in enumerate(history.cpu().numpy()):
            for t in row[(row >= 0) & (row < v)]:
                c[i, t] += 1
    slope = np.where(c > 0, np.where(l > 0, 1 / repetition, repetition), 1.0) / temperature
    with np.errstate(invalid="ignore", over="ignore"):
        l = np.where(c > 0, np.where(l > 0, l / repetition, l * repetition), l) - frequency * c - presence * (c > 0)
        l = (l + (0.0 if bias is None else _np(bias))) / temperature
    if allowed is not None:
        a = np.broadcast_to(allowed.cpu().numpy(), l.shape)
        l, slope = np.where(a, l, -np.inf), np.where(a, slope, 0.0)
    return l, slope


def _stats(l):
    """M, e, Z, H, mean distance, mean squared distance; empty and bad rows."""
    bad = np.isnan(l).any(1) | (l == np.inf).any(1)
    l = np.where(bad[:, None], 0.0, l)
    m = l.max(1, keepdims=True)
    empty = np.isneginf(m[:, 0])
    d = np.where(empty[:, None], 0.0, np.where(empty[:, None], 0.0, m) - l)
    e = np.exp(-d)
    z = e.sum(1)
    dz = np.where(e > 0, np.where(np.isinf(d), 0.0, d), 0.0)
    return dict(m=m[:, 0], d=d, e=e, z=z, mean=(dz * e).sum(1) / z, square=(dz * dz * e).sum(1) / z, h=np.log(z) + (dz * e).sum(1) / z, bad=bad, empty=empty)


def _tol(s):
    """Bounds of log Z, of a log-probability at distance d (added by the caller) and of the entropy."""
    logz = U * (3 * s["mean"] + 154 + 2 * np.log(s["z"]))
    entropy = 2 * logz + U * (3 * s["square"] + 160 * s["mean"] + 2 * np.abs(s["h"])) + 1e-37
    return logz, entropy


def _check_rows(got_logp, got_h, l, actions):
    s = _stats(l)
    logz, tol_h = _tol(s)
    at = np.clip(actions, 0, l.shape[1] - 1)
    i = np.arange(len(at))
    inside = (actions >= 0) & (actions < l.shape[1])
    with np.errstate(invalid="ignore"):
        want = np.where(inside, l[i, at], -np.inf) - s["m"] - np.log(s["z"])
    want = np.where(s["bad"], np.nan, np.where(s["empty"], 0.0, want))
    h = np.where(s["bad"], np.nan, np.where(s["empty"], 0.0, s["h"]))
    logp, ent = _np(got_logp), _np(got_h)
    assert np.array_equal(np.isnan(logp), np.isnan(want)) and np.array_equal(np.isneginf(logp), np.isneginf(want))
    assert np.array_equal(np.isnan(ent), np.isnan(h))
    fine = np.isfinite(want)
    assert np.all(np.abs(logp - want)[fine] <= (logz + 5 * U * np.abs(want))[fine])
    fine = np.isfinite(h)
    assert np.all(np.abs(ent - h)[fine] <= tol_h[fine]), np.max((np.abs(ent - h) - tol_h)[fine])


def _picked(l, u):
    s = _stats(l)
    run = np.cumsum(s["e"], 1)
    over = run > (u[:, None] * s["z"][:, None]) if u is not None else l == l.max(1, keepdims=True)
    lastp = l.shape[1] - 1 - np.argmax(s["e"][:, ::-1] > 0, 1)
    a = np.where(over.any(1), over.argmax(1), lastp)
    return np.where(s["bad"] | s["empty"], -1, a)


def _case(n, v, dtype, seed=0, mask=True, bias="rows", length=9, scale=2.0, empty=True):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(n, v, generator=g) * scale).to(dtype)
    c = dict(temperature=0.75)
    if mask:
        c["allowed"] = torch.rand(n, v, generator=g) < 0.6
        if empty:
            c["allowed"][n // 2] = False  # a row with nothing left
    if bias:
        c["bias"] = torch.randn(*((n, v) if bias == "rows" else (v,)), generator=g)
    if length:
        c["history"] = torch.randint(-2, v + 2, (n, length), generator=g, dtype=torch.int32)  # some outside [0, V)
        c.update(repetition=1.3, presence=0.4, frequency=0.15)
    return logits, c, torch.rand(n, generator=g)


def _cuda(c):
    return {k: t.cuda() if torch.is_tensor(t) else t for k, t in c.items()}


SHAPES = [(1, 1), (3, 2), (24, 5), (1000, 5), (65, 8), (11, 9), (33, 63), (17, 64), (9, 65), (40, 157), (5, 512), (7, 513), (7, 1000), (3, 1025), (3, 2049),
          (3, 4097), (2, 8192), (2, 8193), (2, 20001), (1, 131072), (300, 33), (257, 3), (130, 6), (64, 7), (65, 4), (70, 13),
          (12, 100), (9, 180), (6, 430)]  # fmt: skip

# ---- refusals ------------------------------------------------------------------------------------------------------


def test_refusals():
    l, a = torch.zeros(3, 40), torch.ones(3, 40, dtype=torch.bool)
    h = torch.zeros(3, 4, dtype=torch.int32)
    cases = [
        ("at least one token", torch.zeros(3, 0), {}),
        ("at least one token", torch.zeros(()), {}),
        ("float32, bfloat16 or float16", l.double(), {}),
        ("temperature", l, dict(temperature=0.0)),
        ("temperature", l, dict(temperature=-1.0)),
        ("temperature", l, dict(temperature=float("nan"))),
        ("temperature", l, dict(temperature=9e-31)),
        ("temperature", l, dict(temperature=INF)),
        ("repetition", l, dict(repetition=1.1e30, history=h)),
        ("repetition", l, dict(repetition=0.0, history=h)),
        ("repetition", l, dict(repetition=INF, history=h)),
        ("finite", l, dict(presence=INF, history=h)),
        ("finite", l, dict(frequency=float("nan"), history=h)),
        ("need a history", l, dict(frequency=0.5)),
        ("allowed must be bool", l, dict(allowed=a.float())),
        ("allowed must be \\[40\\]", l, dict(allowed=a[:, :39])),
        ("allowed must be \\[40\\]", l, dict(allowed=a[:2])),
        ("allowed must be \\[2\\]", l, dict(allowed=torch.zeros(3, 3, dtype=torch.int32))),
        ("bias must be float32", l, dict(bias=torch.zeros(40).half())),
        ("bias must be \\[40\\]", l, dict(bias=torch.zeros(1, 40))),
        ("must not require", l, dict(bias=torch.zeros(40, requires_grad=True))),
        ("history must be int32", l, dict(history=h.long(), repetition=2.0)),
        ("history must be", l, dict(history=h[:2], repetition=2.0)),
        ("same device", l, dict(bias=torch.zeros(40, device="meta"))),
        ("on GPU", l, {}),
    ]
    for text, logits, c in cases:
        for call in (adjust_logits, sample_actions, lambda x, **k: evaluate_actions(x, torch.zeros(x.shape[:-1], dtype=torch.int32), **k)):
            if text == "must not require" and call is sample_actions:
                continue  # it has no gradient to lose
            with pytest.raises(RuntimeError, match=text):
                call(logits, **c)
    for bad in (a.int(), a[:, :0]):
        with pytest.raises(RuntimeError, match="bool"):
            pack_allowed(bad)


def test_library_refuses_bad_arguments_before_any_launch():
    import ctypes as ct

    from metta_amd import native

    L = native.load()
    calls = {
        "mg_adjust_logits": 2, "mg_adjust_logits_backward": 3, "mg_sample_actions": 5, "mg_evaluate_actions": 5, "mg_evaluate_actions_backward": 7,
    }  # fmt: skip
    good = dict(rows=2, width=4, temperature=1.0, repetition=1.0)
    for name, n in calls.items():
        f = getattr(L, name)
        assert f(None, *[None] * n) != 0
        for change, text in (({"type": 5}, b"type"), ({"width": 0}, b"token"), ({"rows": -1}, b"token"), ({"temperature": 0.0}, b"temperature"),
                             ({"repetition": -1.0}, b"repetition"), ({"temperature": 1e31}, b"temperature"), ({"presence": INF}, b"finite"), ({"logits": None}, b"NULL"),
                             ({"logits": 4096, "allowed": 4096, "allowed_kind": 7}, b"allowed_kind"), ({"logits": 4096}, b"NULL")):  # fmt: skip
            a = native.MgLogits(**(good | change))
            assert f(ct.byref(a), *[None] * n) != 0 and text in L.mg_last_error(), (name, change)
        assert f(ct.byref(native.MgLogits(**(good | {"rows": 0}))), *[None] * n) == 0


@pytest.mark.gpu
def test_pack_allowed_in_a_captured_graph():
    a = torch.rand(7, 157, device="cuda") < 0.5
    pack_allowed(a)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w = pack_allowed(a)
    for _ in range(4):
        a.copy_(torch.rand(7, 157, device="cuda") < 0.5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, pack_allowed(a))


def test_pack_allowed():
    for v in (1, 31, 32, 33, 157):
        a = torch.rand(4, 3, v, generator=torch.Generator().manual_seed(v)) < 0.5
        w = pack_allowed(a)
        assert w.dtype == torch.int32 and w.shape == (4, 3, (v + 31) // 32)
        at = torch.arange(v)
        assert torch.equal((w[..., at // 32] >> (at % 32)) & 1 == 1, a)


# ---- GPU ----------------------------------------------------------------------------------------------------------


def _rounded(got, want, dtype):
    fi = torch.finfo(dtype)
    g = _np(got)
    assert np.array_equal(np.isnan(g), np.isnan(want))
    over = np.abs(want) > fi.max * (1 - fi.eps / 4)  # may round to infinity or to the largest value
    assert np.array_equal(np.isinf(g)[~over], np.isinf(want)[~over])
    fine = np.isfinite(want) & ~over
    # one rounding to the type, through a rounding to 32 bits
    tol = (fi.eps / 2 + 2 * U) * np.abs(want) + fi.smallest_normal * fi.eps / 2 + 1e-37
    assert np.all(np.abs(g - want)[fine] <= tol[fine])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_adjust(shape, dtype):
    for k, kw in enumerate((dict(), dict(mask=False, bias=None), dict(bias="shared", length=300), dict(bias=None, length=0))):
        logits, c, _ = _case(*shape, dtype, seed=k, **kw)
        want, slope = _adjusted(logits, **c)
        dout = torch.randn(*shape, generator=torch.Generator().manual_seed(k)).to(dtype)
        x = logits.cuda().requires_grad_()
        dev = _cuda(c)
        out = adjust_logits(x, **dev)
        assert out.dtype == dtype and out.shape == logits.shape
        _rounded(out, want, dtype)
        (d,) = torch.autograd.grad(out, x, dout.cuda())
        _rounded(d, slope * _np(dout), dtype)
        if "allowed" in c:
            dev["allowed"] = pack_allowed(dev["allowed"])
            again = adjust_logits(x, **dev)
            assert torch.equal(again, out) and torch.equal(torch.autograd.grad(again, x, dout.cuda())[0], d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_sample(shape, dtype):
    for k, kw in enumerate((dict(), dict(mask=False, bias=None, length=0), dict(bias="shared", length=300), dict(bias=None, length=0, scale=0.0),
                            dict(mask=False, bias=None, length=0, scale=30.0))):  # fmt: skip
        logits, c, u = _case(*shape, dtype, seed=10 + k, **kw)
        l, _ = _adjusted(logits, **c)
        dev = _cuda(c)
        a, logp, h = sample_actions(logits.cuda(), u.cuda(), **dev)
        assert a.dtype == torch.int32 and not logp.requires_grad
        want = _picked(l, _np(u))
        assert np.array_equal(a.cpu().numpy(), want), (k, np.flatnonzero(a.cpu().numpy() != want))
        _check_rows(logp, h, l, want)
        if "allowed" in c:
            dev["allowed"] = pack_allowed(dev["allowed"])
            for x, y in zip(sample_actions(logits.cuda(), u.cuda(), **dev), (a, logp, h)):
                assert torch.equal(x, y)
        a, logp, h = sample_actions(logits.cuda(), **dev)  # the most likely one
        want = _picked(l, None)
        assert np.array_equal(a.cpu().numpy(), want)
        _check_rows(logp, h, l, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_evaluate(shape, dtype):
    for k, kw in enumerate((dict(), dict(mask=False, bias=None, length=0), dict(bias="shared", length=300))):
        logits, c, u = _case(*shape, dtype, seed=20 + k, **kw)
        l, slope = _adjusted(logits, **c)
        actions = _picked(l, _np(u))
        if shape[0] > 2:
            actions[0], actions[1] = shape[1], 0  # outside; perhaps masked
        g = torch.Generator().manual_seed(k)
        gp, gh = torch.randn(shape[0], generator=g), torch.randn(shape[0], generator=g)
        dev = _cuda(c)
        if k == 2:
            dev["allowed"] = pack_allowed(dev["allowed"])
        x = logits.cuda().requires_grad_()
        logp, h = evaluate_actions(x, torch.from_numpy(actions).cuda().to(torch.int32 if k else torch.int64), **dev)
        _check_rows(logp, h, l, actions)
        s = _stats(l)
        logz, tol_h = _tol(s)
        q = s["e"] / s["z"][:, None]
        i, at = np.arange(shape[0]), np.clip(actions, 0, shape[1] - 1)
        hit = np.zeros_like(q)
        hit[i, at] = (actions >= 0) & (actions < shape[1]) & np.isfinite(l[i, at])
        gpe = _np(gp) * hit.sum(1)
        lq = np.where(q > 0, -np.where(np.isinf(s["d"]), 0, s["d"]) - np.log(s["z"])[:, None], 0.0)
        for which in ("both", "logp", "entropy"):
            p_, h_ = (gpe if which != "entropy" else 0 * gpe), (_np(gh) if which != "logp" else 0 * gpe)
            want = p_[:, None] * (hit - q) - h_[:, None] * q * (lq + s["h"][:, None])
            want = np.where(s["empty"][:, None], 0.0, want * slope)
            relq = 5 * U * np.abs(lq) + logz[:, None] + 8 * U
            err = np.abs(p_)[:, None] * (q * relq + 4 * U * hit) + np.abs(h_)[:, None] * q * (
                relq * np.abs(lq + s["h"][:, None]) + 5 * U * np.abs(lq) + (logz + tol_h)[:, None] + 8 * U * (np.abs(lq) + s["h"][:, None]))  # fmt: skip
            outs, gs = {"both": ([logp, h], [gp.cuda(), gh.cuda()]), "logp": ([logp], [gp.cuda()]), "entropy": ([h], [gh.cuda()])}[which]
            (d,) = torch.autograd.grad(outs, x, gs, retain_graph=True)
            fi = torch.finfo(dtype)
            tol = err * slope + (fi.eps / 2 + 4 * U) * np.abs(want) + fi.smallest_normal * fi.eps / 2 + 1e-37
            off = np.abs(_np(d) - want)
            assert d.dtype == dtype and np.all(off <= tol), (which, k, np.max(off - tol))


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8300, 16500])
def test_many_wide_rows(v):
    """Rows beyond 8192 tokens that fill the GPU; beyond 16384 a block takes four times as many columns of each."""
    n = 1030
    logits, c, u = _case(n, v, torch.bfloat16, seed=7, length=40, scale=3.0)
    l, slope = _adjusted(logits, **c)
    dev = _cuda(c)
    a, logp, h = sample_actions(logits.cuda(), u.cuda(), **dev)
    want = _picked(l, _np(u))
    assert np.array_equal(a.cpu().numpy(), want)
    _check_rows(logp, h, l, want)
    greedy, logp, h = sample_actions(logits.cuda(), **dev)
    most = _picked(l, None)
    assert np.array_equal(greedy.cpu().numpy(), most)
    _check_rows(logp, h, l, most)
    x = logits.cuda().requires_grad_()
    logp, h = evaluate_actions(x, a, **dev)
    _check_rows(logp, h, l, want)
    (d,) = torch.autograd.grad(logp.sum() + h.sum(), x)
    s = _stats(l)
    logz, tol_h = _tol(s)
    q = s["e"] / s["z"][:, None]
    lq = np.where(q > 0, -np.where(np.isinf(s["d"]), 0, s["d"]) - np.log(s["z"])[:, None], 0.0)
    hit = np.zeros_like(q)
    hit[np.arange(n), np.clip(want, 0, v - 1)] = want >= 0
    value = np.where(s["empty"][:, None], 0.0, (hit - q - q * (lq + s["h"][:, None])) * slope)
    relq = 5 * U * np.abs(lq) + logz[:, None] + 8 * U
    err = q * relq + 4 * U * hit + q * (relq * np.abs(lq + s["h"][:, None]) + 5 * U * np.abs(lq) + (logz + tol_h)[:, None] + 8 * U * (np.abs(lq) + s["h"][:, None]))
    assert np.all(np.abs(_np(d) - value) <= err * slope + (2.0**-8 + 4 * U) * np.abs(value) + 1e-37)
    out = adjust_logits(x, **dev)
    _rounded(out, l, torch.bfloat16)


@pytest.mark.gpu
def test_gradient_against_differences():
    logits, c, _ = _case(6, 30, torch.float32, seed=4, empty=False)
    l0 = _np(logits)
    actions = _picked(_adjusted(logits, **c)[0], np.full(6, 0.4))
    x = logits.cuda().requires_grad_()
    logp, h = evaluate_actions(x, torch.from_numpy(actions).cuda(), **_cuda(c))
    (d,) = torch.autograd.grad((logp * 1.5 - h * 0.5).sum(), x)
    d = _np(d)

    def value(at, eps):
        t = torch.from_numpy(l0.copy())
        t[at] += eps
        l, _ = _adjusted(t, **c)
        s = _stats(l)
        lp = l[np.arange(6), actions] - s["m"] - np.log(s["z"])
        return (1.5 * lp - 0.5 * s["h"]).sum()

    rng = np.random.default_rng(0)
    for _ in range(60):
        at = (int(rng.integers(6)), int(rng.integers(30)))
        slope = (value(at, 1e-5) - value(at, -1e-5)) / 2e-5
        assert abs(d[at] - slope) <= 2e-5 * max(1.0, abs(slope)), at


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [5, 64, 157, 5000])
def test_masks_and_odd_values(v, dtype):
    """NaN and infinities at masked tokens count for nothing; at allowed ones they show; the type's lowest value as a
    mask; -infinity as a logit; one token left; nothing left in three ways."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(v)
    logits = torch.randn(12, v, generator=g).to(dtype)
    allowed = torch.ones(12, v, dtype=torch.bool)
    logits[0, 1], allowed[0, 1] = float("nan"), False
    logits[1, 2], allowed[1, 2] = INF, False
    logits[2, 0] = -INF
    logits[3, :4] = low  # masked the old way: as good as never
    logits[4, 1:] = low
    logits[5, :] = low  # every token: a uniform choice
    allowed[6] = False
    allowed[6, v - 1] = True  # one token left
    allowed[7] = False
    logits[8] = -INF
    logits[9], allowed[9, 3:] = -INF, False
    logits[10, v // 2] = float("nan")
    logits[11, v - 1] = INF
    u = torch.rand(12, generator=g)
    l, slope = _adjusted(logits, allowed=allowed, temperature=0.5)
    for mask in (allowed.cuda(), pack_allowed(allowed.cuda())):
        x = logits.cuda().requires_grad_()
        out = adjust_logits(x, allowed=mask, temperature=0.5)
        _rounded(out, l, dtype)
        (d,) = torch.autograd.grad(out, x, torch.ones_like(out))
        _rounded(d, slope, dtype)
        for uni in (u, None, torch.zeros(12), torch.ones(12)):
            a, logp, h = sample_actions(x, None if uni is None else uni.cuda(), allowed=mask, temperature=0.5)
            want = _picked(l, None if uni is None else _np(uni))
            assert np.array_equal(a.cpu().numpy(), want), (uni, a, want)
            _check_rows(logp, h, l, want)
        want = _picked(l, _np(u))
        logp, h = evaluate_actions(x, torch.from_numpy(want).cuda(), allowed=mask, temperature=0.5)
        _check_rows(logp, h, l, want)
        (d,) = torch.autograd.grad(logp.sum() + h.sum(), x)
        d = _np(d)
        assert np.isfinite(d[:10]).all() and np.all(d[:10][~allowed[:10].numpy()] == 0) and np.all(d[7:10] == 0)
        assert np.isnan(d[10:]).any(1).all()


@pytest.mark.gpu
def test_extreme_controls():
    """Penalties and biases that leave the range of 32 bits in between, and biases of infinity."""
    v = 70
    logits = torch.full((4, v), -3e38)
    history = torch.arange(v, dtype=torch.int32).repeat(4, 1)
    bias = torch.zeros(4, v)
    bias[1, 3], bias[2] = INF, -INF
    bias[3] = torch.linspace(-3e38, 3e38, v)
    logits[3] = -bias[3]  # cancels, up to the rounding of the penalties
    c = dict(history=history, repetition=1.5, bias=bias)
    l, _ = _adjusted(logits, **c)
    u = torch.tensor([0.31, 0.5, 0.5, 0.9])
    a, logp, h = sample_actions(logits.cuda(), u.cuda(), **_cuda(c))
    want = _picked(l, _np(u))
    assert np.array_equal(a.cpu().numpy(), want)
    _check_rows(logp, h, l, want)
    big = torch.randn(50, v, generator=torch.Generator().manual_seed(0)) + 1000.0  # large numbers, small differences
    c = dict(bias=torch.full((v,), -1000.0) + torch.randn(v, generator=torch.Generator().manual_seed(1)))
    l, _ = _adjusted(big, **c)
    u = torch.rand(50, generator=torch.Generator().manual_seed(2))
    a, _, _ = sample_actions(big.cuda(), u.cuda(), **_cuda(c))
    assert np.array_equal(a.cpu().numpy(), _picked(l, _np(u)))


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("v", [6, 100, 900, 3000, 20000])
def test_far_tokens_and_ends_of_the_temperature(v, bias):
    """Logits of 32 bits that lie further apart than their temperature allows a quotient for, under large outer gradients:
    what has no weight has no part in the gradient, and log-probabilities are right up to the last finite one."""
    logits = torch.randn(8, v, generator=torch.Generator().manual_seed(v))
    logits[:, 1] = torch.tensor([-1e38, -3.4e38, -2e38, -3e36, -1e30, -1e37, -5e37, -1e35])
    logits[4:, 2] = 1e30
    allowed = torch.ones(8, v, dtype=torch.bool)
    allowed[:, 3] = False
    kw = dict(allowed=allowed) | (dict(bias=torch.zeros(v)) if bias else {})
    actions = np.array([1, 1, 1, 1, 2, 1, 3, 0])
    for temperature in (1e-30, 1e-3, 0.02, 1.0, 1e3, 1e30):
        l, _ = _adjusted(logits, temperature=temperature, **kw)
        s = _stats(l)
        x = logits.cuda().requires_grad_()
        logp, h = evaluate_actions(x, torch.from_numpy(actions).cuda(), temperature=temperature, **_cuda(kw))
        logz, tol_h = _tol(s)
        i = np.arange(8)
        want = l[i, actions] - s["m"] - np.log(s["z"])
        big = 1.0 - 8 * U  # within roundings of the largest number a value may be infinite
        got, most = _np(logp), float(np.finfo(np.float32).max)
        fine = np.abs(want) < most * big
        assert np.all(np.isneginf(got[np.abs(want) > most * (1 + 8 * U)])) and np.all(np.abs(got - want)[fine] <= (logz + 5 * U * np.abs(want))[fine])
        assert np.all(np.abs(_np(h) - s["h"]) <= tol_h)
        for g in (1.0, 4096.0):  # a scaled loss
            (d,) = torch.autograd.grad([logp, h], x, [torch.full_like(logp, g), torch.full_like(h, g)], retain_graph=True)
            d = _np(d)
            q = s["e"] / s["z"][:, None]
            hit = np.zeros_like(q)
            hit[i, actions] = np.isfinite(l[i, actions])
            lq = np.where(q > 0, -np.where(np.isinf(s["d"]), 0, s["d"]) - np.log(s["z"])[:, None], 0.0)
            value = (hit - hit.sum(1, keepdims=True) * q - q * (lq + s["h"][:, None])) * np.where(allowed, g / temperature, 0.0)
            assert np.isfinite(d[np.abs(value) < 1e37]).all() and not np.isnan(d).any()
            # where q is nothing, nothing but the action's own gradient is left
            nothing = (s["d"] > 200) & (hit == 0)
            assert np.all(d[nothing] == 0)
            relq = 5 * U * np.abs(lq) + logz[:, None] + 8 * U
            err = q * relq + 4 * U * hit + q * (relq * np.abs(lq + s["h"][:, None]) + 5 * U * np.abs(lq) + (logz + tol_h)[:, None] + 8 * U * (np.abs(lq) + s["h"][:, None]))
            # (weights below 2^-126 may be 0: what they are multiplied by there is up to 1 + 104 + H)
            tol = (err + 2.0**-126 * 200) * g / temperature + 5 * U * np.abs(value) + 1e-37
            fine = np.abs(value) < 1e37
            assert np.all(np.abs(d - value)[fine] <= tol[fine]), (temperature, g)
        a, _, _ = sample_actions(x, torch.full((8,), 0.999, device="cuda"), temperature=temperature, **_cuda(kw))
        assert np.array_equal(a.cpu().numpy(), _picked(l, np.full(8, np.float32(0.999), dtype=np.float64)))


@pytest.mark.gpu
@pytest.mark.parametrize("controls", [False, True])
@pytest.mark.parametrize("v", [3, 8, 9, 64, 300, 700, 1500, 3000, 8000, 40000])
def test_uniforms_next_to_borders(v, controls):
    """Uniforms set right at the borders of the distribution, one step of 32 bits below, on and above them: the picked
    action is still the one of the 64-bit definition."""
    g = torch.Generator().manual_seed(v)
    logits = torch.randn(1, v, generator=g)
    c = dict(temperature=0.9)
    if controls:
        c.update(bias=torch.randn(v, generator=g), allowed=torch.rand(v, generator=g) < 0.7, history=torch.arange(0, v, 3)[None, :200].int(),
                 repetition=1.2, frequency=0.1)  # fmt: skip
        c["allowed"][1] = True
    l = _adjusted(logits, **c)[0]
    s = _stats(l)
    run = np.cumsum(s["e"][0]) / s["z"][0]
    at = np.unique(np.linspace(0, v - 2, min(v - 1, 400)).astype(int))
    border = run[at].astype(np.float32)
    u = np.concatenate([border, np.nextafter(border, np.float32(0)), np.nextafter(border, np.float32(1))])
    u = np.minimum(u, np.float32(1 - 2.0**-24))
    rows = logits.repeat(len(u), 1)
    if controls:
        c["history"] = c["history"].repeat(len(u), 1)
    a, logp, h = sample_actions(rows.cuda(), torch.from_numpy(u).cuda(), **_cuda(c))
    l = l.repeat(len(u), 0)
    want = _picked(l, u.astype(np.float64))
    assert np.array_equal(a.cpu().numpy(), want)
    _check_rows(logp, h, l, want)


@pytest.mark.gpu
def test_equal_logits_split_exactly():
    """Equal logits: borders at k / V exactly, and a uniform on a border belongs to the next token."""
    for v in (2, 4, 8, 64, 256, 8192):
        u = (torch.arange(v) / v).float()
        a, logp, h = sample_actions(torch.full((v, v), 0.7).cuda(), u.cuda())
        assert torch.equal(a.cpu(), torch.arange(v, dtype=torch.int32))
        a, _, _ = sample_actions(torch.full((3, v), 0.7, device="cuda"))
        assert torch.equal(a, torch.zeros_like(a))  # the lowest of equals


@pytest.mark.gpu
def test_shapes_and_strides():
    """Leading dimensions, none, sliced rows, columns that are not adjacent, shared controls with stride 0."""
    v = 37
    logits, c, u = _case(24, v, torch.bfloat16, seed=2)
    dev, x, uni = _cuda(c), logits.cuda(), u.cuda()
    a, logp, h = sample_actions(x, uni, **dev)
    shaped = {k: t.view(2, 3, 4, *t.shape[1:]) if torch.is_tensor(t) else t for k, t in dev.items()}
    for p, q in zip(sample_actions(x.view(2, 3, 4, v), uni.view(2, 3, 4), **shaped), (a, logp, h)):
        assert p.shape == (2, 3, 4) and torch.equal(p.flatten(), q)
    one = {k: t[3] if torch.is_tensor(t) else t for k, t in dev.items()}
    for p, q in zip(sample_actions(x[3], uni[3], **one), (a, logp, h)):
        assert p.shape == () and torch.equal(p, q[3])
    wide = torch.zeros(24, 90, dtype=torch.bfloat16, device="cuda")
    wide[:, 11 : 11 + v] = x
    assert torch.equal(sample_actions(wide[:, 11 : 11 + v], uni, **dev)[0], a)
    assert torch.equal(sample_actions(x.t().contiguous().t(), uni, **dev)[0], a)
    leaf = wide.requires_grad_()
    out = adjust_logits(leaf[:, 11 : 11 + v], **dev)
    (d,) = torch.autograd.grad(out, leaf, torch.ones_like(out[:, :1]).expand_as(out))
    plain = x.clone().requires_grad_()
    ref = adjust_logits(plain, **dev)
    assert torch.equal(out, ref) and torch.equal(d[:, 11 : 11 + v], torch.autograd.grad(ref, plain, torch.ones_like(ref))[0])
    assert torch.equal(adjust_logits(x, allowed=dev["allowed"][0], bias=dev["bias"][0]), adjust_logits(x, allowed=dev["allowed"][:1].expand(24, v), bias=dev["bias"][:1].expand(24, v)))
    empty = sample_actions(x[:0], uni[:0])
    assert all(t.shape == (0,) for t in empty)
    y = x[:0].requires_grad_()
    lp, ent = evaluate_actions(y, a[:0])
    assert torch.autograd.grad(lp.sum() + ent.sum(), y)[0].shape == (0, v) and adjust_logits(x[:0]).shape == (0, v)


@pytest.mark.gpu
def test_device_refusals():
    x = torch.zeros(3, 4, device="cuda")
    with pytest.raises(RuntimeError, match="uniforms must be float32"):
        sample_actions(x, torch.zeros(3, device="cuda").double())
    with pytest.raises(RuntimeError, match="uniforms must have"):
        sample_actions(x, torch.zeros(4, device="cuda"))
    with pytest.raises(RuntimeError, match="same device"):
        sample_actions(x, torch.zeros(3))
    with pytest.raises(RuntimeError, match="actions must be int32 or int64"):
        evaluate_actions(x, torch.zeros(3, device="cuda"))
    with pytest.raises(RuntimeError, match="actions must have"):
        evaluate_actions(x, torch.zeros(3, 1, device="cuda", dtype=torch.int32))


@pytest.mark.gpu
def test_same_actions_in_any_batch():
    """A row's action, log-probability and gradient do not depend on what else is in the batch, nor on the run."""
    for v in (5, 157, 3000):
        logits, c, u = _case(500, v, torch.float16, seed=v, length=20)
        dev, x, uni = _cuda(c), logits.cuda(), u.cuda()
        full = sample_actions(x, uni, **dev)
        for rows in (slice(0, 500), slice(7, 8), slice(100, 333)):
            part = {k: t[rows] if torch.is_tensor(t) and t.shape[0] == 500 else t for k, t in dev.items()}
            for p, q in zip(sample_actions(x[rows], uni[rows], **part), full):
                assert torch.equal(p, q[rows])


@pytest.mark.gpu
def test_graph_capture_and_streams():
    logits, c, u = _case(200, 157, torch.bfloat16, seed=9)
    dev, x, uni = _cuda(c), logits.cuda(), u.cuda()
    sample_actions(x, uni, **dev)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sample_actions(x, uni, **dev)
        adj = adjust_logits(x, **dev)
    for k in range(4):
        x.copy_(torch.randn(200, 157, generator=torch.Generator().manual_seed(k)))
        uni.copy_(torch.rand(200, generator=torch.Generator().manual_seed(k)))
        g.replay()
        for p, q in zip((*out, adj), (*sample_actions(x, uni, **dev), adjust_logits(x, **dev))):
            assert torch.equal(p, q), k
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = sample_actions(x, uni, **dev)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(other, out):
        assert torch.equal(p, q)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A view whose second row starts more than 2^32 elements after the first."""
    flat = torch.zeros((1 << 32) + 4096, dtype=torch.float16, device="cuda")
    x = torch.as_strided(flat, (2, 157), (1 << 32, 1))
    logits, c, u = _case(2, 157, torch.float16, seed=1, empty=False)
    x.copy_(logits)
    l, _ = _adjusted(logits, **c)
    a, logp, h = sample_actions(x, u.cuda(), **_cuda(c))
    assert np.array_equal(a.cpu().numpy(), _picked(l, _np(u)))
    _check_rows(logp, h, l, _picked(l, _np(u)))


@pytest.mark.gpu
@pytest.mark.parametrize("v", [5, 300, 9000])
def test_training_in_a_captured_graph(v):
    """Forward and backward captured once, replayed on new inputs with eager work in between; other leaves do the eager part."""
    logits, c, u = _case(60, v, torch.bfloat16, seed=v)
    dev, x, gp = _cuda(c), logits.cuda().requires_grad_(), u.cuda()
    actions, _, _ = sample_actions(x, gp, **dev)

    def once(t):
        logp, h = evaluate_actions(t, actions, **dev)
        adj = adjust_logits(t, **dev)
        return [logp, h, adj, *torch.autograd.grad([logp, h], [t], [gp, gp]), *torch.autograd.grad(adj, t, adj.detach().clamp(-1, 1))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            once(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = once(x)
    for k in range(4):
        with torch.no_grad():
            x.mul_(0.5).add_(0.1 * k)
        gp.uniform_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, once(x.detach().clone().requires_grad_())):
            assert torch.equal(a, b), k


@pytest.mark.gpu
@pytest.mark.parametrize("v", [7, 700, 9000])
def test_saved_tensors_that_move(v):
    """Hooks that take what was saved to the host and back give the same gradients, for sliced logits too."""
    logits, c, u = _case(20, v, torch.float16, seed=v)
    dev, gp = _cuda(c), u.cuda()
    wide = torch.zeros(20, v + 9, dtype=torch.float16, device="cuda")
    wide[:, 3 : 3 + v] = logits.cuda()
    actions, _, _ = sample_actions(wide[:, 3 : 3 + v], gp, **dev)

    def once():
        leaf = wide.clone().requires_grad_()
        view = (leaf * 1.0)[:, 3 : 3 + v]
        return leaf, [*evaluate_actions(view, actions, **dev), adjust_logits(view, **dev)]

    grads = [gp, gp, torch.ones(20, v, dtype=torch.float16, device="cuda")]
    leaf, out = once()
    (want,) = torch.autograd.grad(out, leaf, grads)
    with torch.autograd.graph.save_on_cpu():
        leaf, out = once()
    junk = [torch.randn_like(wide) for _ in range(8)]  # memory that was free is written over
    (got,) = torch.autograd.grad(out, leaf, grads)
    assert len(junk) == 8 and torch.equal(got, want)


@pytest.mark.gpu
def test_saved_tensors_are_watched_and_second_derivatives_refused():
    x = torch.randn(4, 9, device="cuda", requires_grad=True)
    y = x * 1.0
    logp, _ = evaluate_actions(y, torch.zeros(4, dtype=torch.int32, device="cuda"))
    y.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        logp.sum().backward()
    for out in (evaluate_actions(x, torch.zeros(4, dtype=torch.int64, device="cuda"))[0], adjust_logits(x)):
        (d,) = torch.autograd.grad(out.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            d.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("n,v", [(60000, 5), (20000, 64), (10000, 157), (3000, 1024), (400, 8000)])
def test_many_rows_are_the_definitions(n, v):
    """Enough rows that some targets come close to a border: the 32-bit sums do not decide those."""
    g = torch.Generator().manual_seed(n)
    logits = torch.randn(n, v, generator=g)
    for kw in ({}, dict(bias=torch.randn(v, generator=g))):
        u = torch.rand(n, generator=g)
        a, _, _ = sample_actions(logits.cuda(), u.cuda(), temperature=0.8, **_cuda(kw))
        want = _picked(_adjusted(logits, temperature=0.8, **kw)[0], _np(u))
        assert np.array_equal(a.cpu().numpy(), want)


def test_forward_mode_is_refused():
    """A dual tensor's tangent is not dropped; sampling carries no derivative of any kind."""
    from torch.autograd import forward_ad

    l, a, b = torch.zeros(3, 40), torch.zeros(3, dtype=torch.int32), torch.zeros(40)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(l, torch.ones_like(l))
        with pytest.raises(RuntimeError, match="adjust_logits has no forward-mode"):
            adjust_logits(dual)
        with pytest.raises(RuntimeError, match="evaluate_actions has no forward-mode"):
            evaluate_actions(dual, a)
        bias = forward_ad.make_dual(b, torch.ones_like(b))
        for call in (lambda: adjust_logits(l, bias=bias), lambda: evaluate_actions(l, a, bias=bias)):
            with pytest.raises(RuntimeError, match="bias is a constant"):
                call()
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="on GPU"):
            adjust_logits(dual, bias=bias)
        with pytest.raises(RuntimeError, match="on GPU"):
            sample_actions(dual)


@pytest.mark.gpu
def test_forward_mode_is_refused_on_device():
    from torch.autograd import forward_ad

    l, a = torch.randn(3, 40, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(l, torch.ones_like(l))
        for call in (lambda: adjust_logits(dual), lambda: evaluate_actions(dual, a)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        for t in sample_actions(dual):
            assert forward_ad.unpack_dual(t).tangent is None


def test_tracing_is_refused():
    """A trace would hold the results' memory and not the launches that fill it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    l, a = torch.zeros(3, 40), torch.zeros(3, dtype=torch.int32)
    for call in (lambda t: adjust_logits(t), lambda t: sample_actions(t)[1], lambda t: evaluate_actions(t, a)[0]):
        for leaf in (l, l.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                torch.jit.trace(call, leaf, check_trace=False)
        for mode in ("real", "fake"):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(call, tracing_mode=mode)(l)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [5, 64, 157, 700, 1500, 5000, 20000])
def test_gradients_of_bad_rows(v, dtype):
    """NaN or +infinity at an allowed token makes the gradient of every token that is left NaN, and of none that is not: masked,
    or at -infinity.  An infinite outer gradient passes by those, too."""
    g = torch.Generator().manual_seed(v)
    logits = torch.randn(4, v, generator=g).to(dtype)
    logits[0, 0], logits[1, v - 1], logits[:, 2] = float("nan"), INF, -INF
    allowed = torch.ones(4, v, dtype=torch.bool)
    allowed[:, 3] = False
    logits[:, 3] = float("nan")
    history = torch.tensor([[1, 2, 3, -1]], dtype=torch.int32).expand(4, 4)
    outer = torch.tensor([1.0, 1.0, INF, 1.0], device="cuda")
    for kw in (dict(), dict(bias=torch.randn(v, generator=g)), dict(history=history, repetition=1.5, presence=0.25)):
        x = logits.cuda().requires_grad_()
        out = evaluate_actions(x, torch.ones(4, dtype=torch.int32, device="cuda"), **_cuda(dict(allowed=allowed, **kw)))
        for outs in (out, out[:1], out[1:]):
            (d,) = torch.autograd.grad(outs, x, [outer] * len(outs), retain_graph=True)
            nan = torch.isnan(d).cpu()
            assert bool((d[:, 2:4] == 0).all()), "no part in the row"
            left = torch.ones(v, dtype=torch.bool)
            left[2:4] = False
            assert torch.equal(nan[0], left) and torch.equal(nan[1], left) and not bool(nan[3].any())


@pytest.mark.gpu
@pytest.mark.parametrize("v", [1, 5, 64, 157, 700, 1500, 5000, 8192, 9000, 20000])
def test_uniforms_of_nan_show(v):
    """A uniform of NaN gives action -1 and NaN, as a logit of NaN does; the rows beside it keep theirs.  Uniforms outside of
    [0, 1) are taken as 0 and as 1."""
    for kw in (dict(mask=False, bias=None, length=0), dict(empty=False)):
        logits, c, u = _case(70, v, torch.float32, seed=v, **kw)
        if "allowed" in c:
            c["allowed"][:, 0] = True  # no row is empty
        x, dev = logits.cuda(), _cuda(c)
        want = [t.clone() for t in sample_actions(x, u.cuda(), **dev)]
        bad = u.clone()
        bad[[0, 33, 69]] = torch.tensor([float("nan"), float("nan"), -float("nan")])
        got = sample_actions(x, bad.cuda(), **dev)
        for a, b in zip(got, want):
            keep = ~torch.isnan(bad).cuda()
            assert torch.equal(a[keep], b[keep])
        lost = torch.isnan(bad).cuda()
        assert bool((got[0][lost] == -1).all()) and bool(torch.isnan(got[1][lost]).all()) and bool(torch.isnan(got[2][lost]).all())
        for outside, inside in ((-1.0, 0.0), (-INF, 0.0), (INF, 1.0), (2.0, 1.0)):
            for a, b in zip(sample_actions(x, torch.full_like(u, outside).cuda(), **dev), sample_actions(x, torch.full_like(u, inside).cuda(), **dev)):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [2, 7, 100, 900, 3000, 20000])
def test_log_probabilities_of_the_furthest_tokens(v):
    """Tokens further apart than the largest number of 32 bits, which the temperature brings back into its range."""
    logits = torch.randn(4, v, generator=torch.Generator().manual_seed(v))
    logits[:, 0] = torch.tensor([3e38, 3.4e38, 2e38, 1e38])
    logits[:, 1] = torch.tensor([-3e38, -3.4e38, -2.5e38, -3.3e38])
    bias = torch.zeros(v)
    bias[0], bias[1] = 3e38, -3e38
    actions = torch.ones(4, dtype=torch.int32)
    for kw in (dict(), dict(bias=bias)):
        for temperature in (0.5, 1.0, 2.0, 4.0, 7.0, 1e10, 1e30):
            l, _ = _adjusted(logits, temperature=temperature, **kw)
            s = _stats(l)
            x = logits.cuda().requires_grad_()
            logp, h = evaluate_actions(x, actions.cuda(), temperature=temperature, **_cuda(kw))
            want, got, most = l[:, 1] - s["m"] - np.log(s["z"]), _np(logp), float(np.finfo(np.float32).max)
            # difference, scale (a rounding of its own) and product: 3u, and one for the sum
            assert np.all(np.isneginf(got[want < -most * (1 + 8 * U)])), temperature
            fine = want > -most * (1 - 8 * U)
            assert np.all(np.abs(got - want)[fine] <= (5 * U * np.abs(want))[fine]), (temperature, got, want)
            assert np.all(_np(h) == 0.0)
            (d,) = torch.autograd.grad([logp, h], x, [torch.ones_like(logp)] * 2)
            assert bool(torch.isfinite(d).all())


@pytest.mark.gpu
@pytest.mark.parametrize("v", [5, 157, 9000])
def test_negated_views(v):
    """Views that hold their values negated give what their values give, gradients too."""
    logits, c, u = _case(6, v, torch.float32, seed=v)
    dev, l, uni = _cuda(c), logits.cuda(), u.cuda()
    neg = lambda t: torch._neg_view(-t)  # noqa: E731
    other = dev | {"bias": neg(dev["bias"])}
    assert neg(l).is_neg() and torch.equal(neg(l), l)
    for a, b in zip(sample_actions(neg(l), neg(uni), **other), sample_actions(l, uni, **dev)):
        assert torch.equal(a, b)
    actions = sample_actions(l, uni, **dev)[0]

    def grads(view, kw):
        leaf = l.clone().requires_grad_()
        t = neg(leaf) if view else leaf
        w = neg if view else (lambda y: y)
        logp, h = evaluate_actions(t, actions, **kw)
        adj = adjust_logits(t, **kw)
        return [logp, h, adj, *torch.autograd.grad([logp, h], leaf, [w(uni), w(uni)]), *torch.autograd.grad(adj, leaf, w(l))]

    for a, b in zip(grads(True, other), grads(False, dev)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_evaluation_of_more_rows_than_a_grid_has_waves():
    """A wave per row joins the parts of wide rows; 2^26 of them are more threads than one dimension of a grid takes."""
    n, v = (1 << 26) + 5, 8193
    logits = torch.randn(1, v, generator=torch.Generator().manual_seed(0)).cuda()
    actions = (torch.arange(n, device="cuda", dtype=torch.int32) * 7) % v
    logp, h = evaluate_actions(logits.expand(n, v), actions)
    one, ent = evaluate_actions(logits.expand(v, v), torch.arange(v, device="cuda", dtype=torch.int32))
    assert bool((h == ent[0]).all()) and torch.equal(logp, one[actions.long()])
    some = np.arange(0, v, 100)
    _check_rows(one.cpu()[some], ent.cpu()[some], _np(logits).repeat(len(some), 0), some)


@pytest.mark.gpu
def test_exponentials_are_within_the_margin_of_sampling():
    """2^-t as the kernels compute it, for every t of 32 bits from 0 to 125.9: within the 2 units of 2^-24 that the margin of sampling
    takes for it.  Stats of (0, 0), a temperature of log2 e and an outer gradient that their factor makes 1 leave the backward
    pass of wide rows with minus the exponential itself."""
    import ctypes as ct

    from metta_amd import native

    L = native.load()
    rows, v = 16384, 8193  # column 0 is the action's
    temperature = float(np.log2(np.e))
    inv = np.float32(1.0 / temperature)
    outer = next(g for k in range(-4, 5) for g in [np.float32(1.0 / float(inv)) + np.float32(k * 2.0**-23)] if np.float32(g * inv) == np.float32(1.0))
    assert np.float32(1.0 / temperature * -1.4426950408889634) == np.float32(-1.0)
    logits = torch.zeros(rows, v, device="cuda")
    out = torch.empty_like(logits)
    actions = torch.zeros(rows, dtype=torch.int32, device="cuda")
    zero = torch.zeros(rows, device="cuda")
    stats = torch.zeros(rows, 2, dtype=torch.float64, device="cuda")
    dlogp = torch.full((rows,), float(outer), device="cuda")
    a = native.MgLogits(logits=logits.data_ptr(), rows=rows, width=v, logits_row=v, temperature=temperature, repetition=1.0)
    last = int(np.float32(125.9).view(np.int32))
    each, worst = rows * (v - 1), 0.0
    for first in range(0, last, each):
        bits = torch.arange(first, first + each, dtype=torch.int64, device="cuda").clamp_(max=last).to(torch.int32)
        t = bits.view(torch.float32).view(rows, v - 1)
        logits[:, 1:] = -t
        rc = L.mg_evaluate_actions_backward(ct.byref(a), actions.data_ptr(), zero.data_ptr(), stats.data_ptr(), dlogp.data_ptr(), None, out.data_ptr(),
                                            torch.cuda.current_stream().cuda_stream)
        assert rc == 0, L.mg_last_error()
        want = torch.exp2(-t.double())
        worst = max(worst, float(((-out[:, 1:].double() - want) / want).abs().max()))
    assert 0.0 < worst <= 2 * U, worst / U
