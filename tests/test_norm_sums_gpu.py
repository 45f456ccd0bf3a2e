"""The summed gradients of ops.gated_residual_norm (weights, biases, scales, gates of rows and columns) within a bound that a lost
term or a lost partial sum would break.

The oracle writes the backward formulas out in 64 bits and sums the terms' absolute values beside the terms.  With e = 2^-24 an
element of a sum carries at most 128 e of its absolute value: some 24 chained operations, and row sums of D terms in a tree over
lanes and waves (at most 16 serial steps in a lane, 6 + 4 levels; the stored statistics bring as many again).  "Absolute value" means: differences
are counted with both sides (|t| + |mean|, |dr| + |norm's share|).  A workgroup adds its rows one after the other in fp32 (there are 128
workgroups at least, or one per row), the rest is added in 64 bits: |error| <= (rows / 128 + 128) e sum|terms|, and e for the result.
Inputs have signs that do not cancel, so this is far below the sums themselves, which the test asserts: less than 1e-4 of the largest."""
import pytest
import torch

from tests.test_residual_norm_gpu import B16, F32

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def inputs(rows, D, xt, ht, post, pre, gate, scale):
    g = torch.Generator().manual_seed(rows + D)
    rn = lambda *s: torch.randn(*s, generator=g)
    # a value per column on top of noise: normalised rows keep its sign; no sign at all where the norm takes no mean
    lean = lambda kind: 1.5 * (rn(D).sign() if kind == "layer" else torch.ones(D)) + 0.3 * rn(rows, D)
    t = {"x": lean(pre).to(xt), "h": (0.2 * lean(post)).to(ht), "dr": (1 + 0.2 * rn(rows, D)).to(xt), "dy": (0.5 + 0.1 * rn(rows, D)).to(ht)}
    t["gate"] = {None: None, "full": rn(rows, D).to(ht), "row": rn(rows, 1), "col": rn(D)}[gate]
    t["scale"] = {None: None, "one": 0.5 + 0.1 * rn(1).abs(), "col": 0.5 + 0.1 * rn(D).abs()}[scale]
    t["post_weight"], t["pre_weight"] = 1 + 0.1 * rn(D), 1 + 0.1 * rn(D)
    t["post_bias"] = 0.1 * rn(D).abs() if post == "layer" else None
    t["pre_bias"] = 0.1 * rn(D) if pre == "layer" else None
    return t


def normed(t, kind):
    """normalised values; 1 / spread; what an error of the values is relative to"""
    m = t.mean(1, keepdim=True) if kind == "layer" else torch.zeros(len(t), 1, dtype=t.dtype)
    rstd = 1 / torch.sqrt(((t - m) ** 2).mean(1, keepdim=True) + 1e-5)
    return (t - m) * rstd, rstd, (t.abs() + m.abs()) * rstd + 1


def sums(t, post, pre, gate):
    """name -> (gradient, sum of absolute terms)"""
    d = {n: None if v is None else v.double() for n, v in t.items()}
    w1, w2 = d["post_weight"], d["pre_weight"]
    b1 = 0.0 if d["post_bias"] is None else d["post_bias"]
    act = 1.0 if gate is None else torch.sigmoid(d["gate"])
    slope = 0.0 if gate is None else act * (1 - act)
    s = 1.0 if d["scale"] is None else d["scale"]
    hh, _, hm = normed(d["h"], post)
    n, nm = hh * w1 + b1, hm * w1.abs() + abs(b1)
    r = d["x"] + s * act * n
    rh, rstd, rm = normed(r, pre)
    a = d["dy"] * w2
    mean = lambda v: v.mean(1, keepdim=True)
    du = d["dr"] + rstd * (a - (mean(a) if pre == "layer" else 0) - rh * mean(a * rh))
    dm = d["dr"].abs() + rstd * (a.abs() + mean(a.abs()) + rm * mean(a.abs() * rm))
    dn, dnm = du * s * act, dm * abs(s) * act
    out = {"pre_weight": (d["dy"] * rh, d["dy"].abs() * rm), "pre_bias": (d["dy"], d["dy"].abs()), "post_weight": (dn * hh, dnm * hm),
           "post_bias": (dn, dnm), "scale": (du * act * n, dm * act * nm)}
    out = {k: (v.sum(0), m.sum(0)) for k, (v, m) in out.items()}
    if t["scale"] is not None and t["scale"].numel() == 1:
        out["scale"] = tuple(v.sum().reshape(1) for v in out["scale"])
    if gate is not None:
        v, m = du * s * n * slope, dm * abs(s) * nm * slope
        out["gate"] = (v.sum(1, keepdim=True), m.sum(1, keepdim=True)) if gate == "row" else (v.sum(0), m.sum(0))
    return {k: v for k, v in out.items() if t[k] is not None and not (k == "gate" and gate == "full")}


@pytest.mark.parametrize("rows,D", [(3, 5), (4097, 72), (6001, 72), (4097, 300), (4097, 700), (6001, 700), (777, 1801), (2000, 2048), (777, 4999),
                                    (1000, 6200), (515, 8192), (255, 9001), (1031, 16384)])
@pytest.mark.parametrize("post,pre,gate,scale", [("rms", "rms", None, "one"), ("layer", "layer", "col", "col"), ("rms", "layer", "row", "one"),
                                                 ("rms", "rms", "full", "col"), ("rms", "rms", "col", "one")])
@pytest.mark.parametrize("types", [(F32, F32), (F32, B16), (B16, B16)], ids=["f32", "mixed", "bf16"])
def test_summed_gradients(rows, D, post, pre, gate, scale, types):
    from scpair_amd import ops
    t = inputs(rows, D, *types, post, pre, gate, scale)
    want = sums(t, post, pre, gate)
    mine = {n: v.cuda().requires_grad_() for n, v in t.items() if v is not None and n not in ("dr", "dy")}
    arg = lambda n: mine.get(n)
    r, y = ops.gated_residual_norm(mine["x"], mine["h"], gate=arg("gate"), scale=arg("scale"), post=post, post_weight=arg("post_weight"),
                                   post_bias=arg("post_bias"), pre=pre, pre_weight=arg("pre_weight"), pre_bias=arg("pre_bias"))
    names = list(want)
    got = torch.autograd.grad((r, y), [mine[n] for n in names], (t["dr"].cuda(), t["dy"].cuda()))
    for n, g in zip(names, got):
        w, m = want[n]
        bound = ((0 if n == "gate" and gate == "row" else rows / 128) + 128) * E * m + E * w.abs()
        assert g.shape == w.shape
        assert (g.cpu().double() - w).abs().sub(bound).max().item() <= 0, (n, ((g.cpu().double() - w).abs() / m).max().item() / E)
        assert bound.max().item() <= 1e-4 * w.abs().max().item(), (n, bound.max().item(), w.abs().max().item())
