"""Norms by degree with gate and residual, and gradient clipping, on the GPU against the float64
oracle.

Bounds (normwise).  fp32: a handful of roundings per element and sums of up to 2048 x 7 squares
(1e-6): 3e-6; the weights' gradients are sums over all atoms, whose rounding grows like the root
of their number against a sum that does so too: 1e-5.  bf16 features: results rounded to 8 bits,
2^-9 of the largest, which norms and gates carry on: 6e-3 (three roundings); the weights'
gradients are fp32 sums of unrounded terms for either type: 1e-5.
"""
import numpy as np
import pytest
import torch

from oracle import block as ob

from helpers import gen, normwise_err, random_rotation, wigner_d

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BOUND = {"f32": 3e-6, "bf16": 6e-3}
WEIGHT_BOUND = {"f32": 1e-5, "bf16": 1e-5}


def _np(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _inputs(n, c, dtype, seed):
    g = gen(seed)
    t = TYPES[dtype]
    return {"x": torch.randn(n, c, 16, generator=g).to(t),
            "y": (2 * torch.randn(n, c, 16, generator=g)).to(t),
            "gate": torch.randn(n, c, 4, generator=g).to(t),
            "scale": torch.randn(c, generator=g), "w_post": torch.randn(4, c, generator=g),
            "w_pre": torch.randn(4, c, generator=g),
            "gh": torch.randn(n, c, 16, generator=g).to(t),
            "gn": torch.randn(n, c, 16, generator=g).to(t)}


def _block(dev, t, gate=True, pre=True, seeds=("gh", "gn")):
    import batmobile
    names = ["x", "y", "scale", "w_post"] + (["gate"] if gate else []) + (["w_pre"] if pre else [])
    leaf = {x: t[x].to(dev).requires_grad_(True) for x in names}
    res = batmobile.gated_residual_norm(leaf["x"], leaf["y"], leaf.get("gate"), leaf["scale"],
                                        leaf["w_post"], leaf.get("w_pre"))
    h, n = res if pre else (res, None)
    outs = [o for o, s in ((h, "gh"), (n, "gn")) if o is not None and s in seeds]
    grads = torch.autograd.grad(outs, list(leaf.values()), [t[s].to(dev) for s in seeds])
    return h, n, dict(zip(names, grads))


def _check(got, want, dtype, weights=("scale", "w_post", "w_pre")):
    for name, g in got.items():
        bound = (WEIGHT_BOUND if name in weights else BOUND)[dtype]
        assert normwise_err(_np(g), want[name]) <= bound, name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(1, 1), (3, 5), (2, 16), (7, 17), (33, 32), (5, 48), (300, 64),
                                 (9, 100), (4, 128), (3, 129), (6, 300), (2, 512), (2, 700),
                                 (1, 2048)])
def test_block_norm(dev, dtype, n, c):
    t = _inputs(n, c, dtype, n + c)
    h, nn, grads = _block(dev, t)
    rh, rn, want = ob.gated_residual_norm(*[_np(t[x]) for x in ("x", "y", "gate", "scale", "w_post",
                                                                "w_pre")],
                                          gh=_np(t["gh"]), gn=_np(t["gn"]))
    assert normwise_err(_np(h), rh) <= BOUND[dtype]
    assert normwise_err(_np(nn), rn) <= BOUND[dtype]
    _check(grads, want, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gate,pre,seeds", [(False, True, ("gh", "gn")), (True, False, ("gh",)),
                                            (False, False, ("gh",)), (True, True, ("gn",)),
                                            (True, True, ("gh",))])
def test_forms(dev, dtype, gate, pre, seeds):
    """Without a gate, without the next norm, and with a gradient for one output only."""
    t = _inputs(21, 40, dtype, 5)
    h, nn, grads = _block(dev, t, gate, pre, seeds)
    rh, rn, want = ob.gated_residual_norm(
        _np(t["x"]), _np(t["y"]), _np(t["gate"]) if gate else None, _np(t["scale"]),
        _np(t["w_post"]), _np(t["w_pre"]) if pre else None,
        gh=_np(t["gh"]) if "gh" in seeds else None, gn=_np(t["gn"]) if "gn" in seeds else None)
    assert normwise_err(_np(h), rh) <= BOUND[dtype]
    if pre:
        assert normwise_err(_np(nn), rn) <= BOUND[dtype]
    if "gn" not in seeds and pre:
        assert not grads.pop("w_pre").any()
    _check(grads, want, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(1, 1), (5, 16), (130, 33), (4, 130), (2, 600)])
def test_norm_alone(dev, dtype, n, c):
    import batmobile
    t = _inputs(n, c, dtype, 9)
    x, w = t["x"].to(dev).requires_grad_(True), t["w_pre"].to(dev).requires_grad_(True)
    out = batmobile.equivariant_norm(x, w)
    gx, gw = torch.autograd.grad(out, [x, w], t["gn"].to(dev))
    _, want, g = ob.gated_residual_norm(_np(t["x"]), None, None, None, None, _np(t["w_pre"]),
                                        gn=_np(t["gn"]))
    assert normwise_err(_np(out), want) <= BOUND[dtype]
    _check({"x": gx, "w_pre": gw}, {"x": g["x"], "w_pre": g["w_pre"]}, dtype)


def test_many_rows(dev):
    """More rows than the backward's workgroups hold at once; a sample of rows, all weights."""
    t = _inputs(9001, 24, "f32", 31)
    h, nn, grads = _block(dev, t)
    rh, rn, want = ob.gated_residual_norm(*[_np(t[x]) for x in ("x", "y", "gate", "scale", "w_post",
                                                                "w_pre")],
                                          gh=_np(t["gh"]), gn=_np(t["gn"]))
    assert normwise_err(_np(nn), rn) <= BOUND["f32"]
    _check(grads, want, "f32")


def test_rows_without_rows_zeros_and_strides(dev):
    import batmobile
    w = torch.ones(4, 8, device=dev)
    x = torch.zeros(0, 8, 16, device=dev, requires_grad=True)
    out = batmobile.equivariant_norm(x, w.requires_grad_(True))
    gx, gw = torch.autograd.grad(out, [x, w], torch.zeros_like(out))
    assert out.shape == x.shape == gx.shape and not gw.any()
    # a row of zeros: 0 / sqrt(eps) = 0, finite gradients
    z = torch.zeros(2, 8, 16, device=dev, requires_grad=True)
    n = batmobile.equivariant_norm(z, w)
    (gz,) = torch.autograd.grad(n, [z], torch.ones_like(n))
    assert not n.any() and torch.allclose(gz, torch.full_like(gz, 1e3), rtol=1e-5)
    # a channel slice and an unaligned view give the results of their copies
    wide = torch.randn(5, 24, 16, device=dev)
    part = wide[:, 8:16]
    assert torch.equal(batmobile.equivariant_norm(part, w),
                       batmobile.equivariant_norm(part.contiguous(), w))
    odd = torch.randn(5 * 8 * 16 + 1, device=dev)[1:].view(5, 8, 16)
    assert torch.equal(batmobile.equivariant_norm(odd, w),
                       batmobile.equivariant_norm(odd.clone(), w))


def test_nan_and_infinities_stay_in_their_row(dev):
    import batmobile
    t = _inputs(12, 20, "f32", 41)
    clean = _block(dev, t)
    bad = dict(t, y=t["y"].clone())
    bad["y"][3, 2, 5] = float("nan")
    bad["y"][7, 0, 0] = float("inf")
    got = _block(dev, bad)
    rows = [i for i in range(12) if i not in (3, 7)]
    for a, b in ((clean[0], got[0]), (clean[1], got[1]), (clean[2]["x"], got[2]["x"]),
                 (clean[2]["y"], got[2]["y"]), (clean[2]["gate"], got[2]["gate"])):
        assert torch.equal(a[rows], b[rows])
    assert torch.isnan(got[0][3]).any()


def test_rotation(dev):
    """norm(D x) = D norm(x) for a rotation D of the components."""
    import batmobile
    t = _inputs(6, 12, "f32", 43)
    d = torch.from_numpy(wigner_d(random_rotation(2)))
    args = [t[x].to(dev) for x in ("gate", "scale", "w_post", "w_pre")]
    a = batmobile.gated_residual_norm(t["x"].to(dev), t["y"].to(dev), *args)
    b = batmobile.gated_residual_norm((t["x"].double() @ d.T).float().to(dev),
                                      (t["y"].double() @ d.T).float().to(dev), *args)
    for u, w in zip(a, b):
        assert normwise_err(_np(w), _np(u) @ d.T.numpy()) <= 1e-5


def test_gradient_against_differences(dev):
    """Step 1e-2 along each gradient, as for the attention: 1e-3."""
    import batmobile
    t = _inputs(15, 10, "f32", 45)
    _, _, grads = _block(dev, t)
    for name, g in grads.items():
        d = g / g.norm()

        def f(step):
            s = {x: v.to(dev) for x, v in t.items()}
            s[name] = s[name] + step * d
            h, n = batmobile.gated_residual_norm(s["x"], s["y"], s["gate"], s["scale"],
                                                 s["w_post"], s["w_pre"])
            return float((h.double() * s["gh"].double()).sum() +
                         (n.double() * s["gn"].double()).sum())
        want, got = (f(1e-2) - f(-1e-2)) / 2e-2, float(g.norm())
        assert abs(got - want) <= 1e-3 * got, (name, got, want)


def test_norm_refusals(dev):
    import batmobile
    x, w = torch.zeros(3, 4, 16, device=dev), torch.ones(4, 4, device=dev)
    s = torch.ones(4, device=dev)
    call = batmobile.gated_residual_norm
    with pytest.raises(RuntimeError, match="16"):
        batmobile.equivariant_norm(torch.zeros(3, 4, 9, device=dev), w)
    with pytest.raises(RuntimeError, match=r"\[4, C\]"):
        batmobile.equivariant_norm(x, torch.ones(4, 5, device=dev))
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        batmobile.equivariant_norm(x.double(), w)
    with pytest.raises(RuntimeError, match="float32"):
        batmobile.equivariant_norm(x, w.bfloat16())
    with pytest.raises(RuntimeError, match="shape of x"):
        call(x, torch.zeros(3, 5, 16, device=dev), None, s, w, w)
    with pytest.raises(RuntimeError, match="gate"):
        call(x, x, torch.zeros(3, 4, 3, device=dev), s, w, w)
    with pytest.raises(RuntimeError, match="scale"):
        call(x, x, None, torch.ones(5, device=dev), w, w)
    with pytest.raises(RuntimeError, match="type"):
        call(x, x.bfloat16(), None, s, w, w)
    with pytest.raises(RuntimeError, match="2048"):
        batmobile.equivariant_norm(torch.zeros(1, 2049, 16, device=dev),
                                   torch.ones(4, 2049, device=dev))


# ---------------------------------------------------------------------------
# clipping
# ---------------------------------------------------------------------------

def _grads(shapes, types, seed, size=1.0):
    g = gen(seed)
    return [(size * torch.randn(*s, generator=g)).to(TYPES[t]) for s, t in zip(shapes, types)]


SHAPES = [(1,), (7,), (64,), (34, 8, 8), (0,), (3, 5, 7), (8193,), (100003,), (2, 4)]


@pytest.mark.parametrize("types", [["f32"] * 9, ["bf16"] * 9, ["f32", "bf16"] * 4 + ["f32"]])
@pytest.mark.parametrize("max_norm", [0.0, 1e-3, 1.0, 1e6])
def test_clip(dev, types, max_norm):
    """Clipped values: one rounding of the factor and one of the product, 2^-23 relative to the
    largest (fp32), 2^-8 of it (bf16); the norm is summed in 64 bits: 1e-6."""
    import batmobile
    grads = _grads(SHAPES, types, 51)
    norm, out = batmobile.clip_grad_norm([g.to(dev) for g in grads], max_norm)
    rn, want = ob.clip([_np(g) for g in grads], max_norm)
    assert abs(float(norm) - rn) <= 1e-6 * rn
    for o, w, t in zip(out, want, types):
        assert o.dtype == TYPES[t]
        assert normwise_err(_np(o), w) <= (5e-7 if t == "f32" else 4e-3)


def test_clip_many_tensors_and_extreme_values(dev):
    """More tensors than a launch takes, values whose squares leave fp32's range either way."""
    import batmobile
    for size in (1e30, 1e-30):
        grads = _grads([(50 + i,) for i in range(457)], ["f32"] * 457, 53, size)
        norm, out = batmobile.clip_grad_norm([g.to(dev) for g in grads], size)
        rn, want = ob.clip([_np(g) for g in grads], float(np.float32(size)))
        assert abs(float(norm) - rn) <= 1e-6 * rn
        for o, w in zip(out, want):     # 1e-30 * 1e-24 is 0 in fp32
            assert normwise_err(_np(o), w.astype(np.float32)) <= 5e-7


def test_clip_not_finite(dev):
    """An infinite gradient gives an infinite norm and the factor 0 (0 * inf = NaN), NaN gives
    NaN everywhere, as the formula says."""
    import batmobile
    a, b = torch.ones(5, device=dev), torch.ones(300, device=dev)
    b[7] = float("inf")
    norm, (ca, cb) = batmobile.clip_grad_norm([a, b], 1.0)
    assert torch.isinf(norm) and not ca.any() and torch.isnan(cb[7]) and cb.nan_to_num().sum() == 0
    b[7] = float("nan")
    norm, (ca, cb) = batmobile.clip_grad_norm([a, b], 1.0)
    assert torch.isnan(norm) and torch.isnan(ca).all() and torch.isnan(cb).all()


def test_clip_in_place_layouts_and_streams(dev):
    """In place on parameters: transposed and gapped gradients, one without a gradient; the
    inputs made on another stream just before."""
    import batmobile
    g = gen(55)
    vals = [torch.randn(6, 10, generator=g), torch.randn(31, generator=g),
            torch.randn(9, 8, generator=g)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        p = [torch.nn.Parameter(torch.zeros(6, 10, device=dev)),
             torch.nn.Parameter(torch.zeros(31, device=dev)),
             torch.nn.Parameter(torch.zeros(9, 8, device=dev)),
             torch.nn.Parameter(torch.zeros(4, device=dev))]
        p[0].grad = vals[0].to(dev).t().contiguous().t()
        p[1].grad = torch.zeros(62, device=dev)[::2]
        p[1].grad.copy_(vals[1].to(dev))
        p[2].grad = torch.zeros(73, device=dev)[1:].view(9, 8)
        p[2].grad.copy_(vals[2].to(dev))
        norm = batmobile.clip_grad_norm_(p, 0.5)
    torch.cuda.synchronize()
    rn, want = ob.clip([_np(v) for v in vals], 0.5)
    assert abs(float(norm) - rn) <= 1e-6 * rn and p[3].grad is None
    for q, w in zip(p, want):
        assert normwise_err(_np(q.grad), w) <= 5e-7
    # below the limit nothing changes, bit for bit
    before = [q.grad.clone() for q in p[:3]]
    batmobile.clip_grad_norm_(p, 10.0)
    assert all(torch.equal(q.grad, b) for q, b in zip(p, before))


def test_clip_refusals(dev):
    import batmobile
    a = torch.ones(4, device=dev)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        batmobile.clip_grad_norm([a.double()], 1.0)
    with pytest.raises(RuntimeError, match="one tensor per"):
        batmobile.clip_grad_norm([a], 1.0, [])
    with pytest.raises(RuntimeError, match="shapes"):
        batmobile.clip_grad_norm([a], 1.0, [torch.ones(5, device=dev)])
    with pytest.raises(RuntimeError, match="type"):
        batmobile.clip_grad_norm([a], 1.0, [a.bfloat16()])


def test_second_derivative_is_refused(dev):
    import batmobile
    x = torch.randn(3, 8, 16, generator=gen(90)).to(dev).requires_grad_(True)
    n = batmobile.equivariant_norm(x, torch.ones(4, 8, device=dev))
    grad, = torch.autograd.grad(n.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


@pytest.mark.parametrize("which", ["gh", "gn"])
def test_forward_mode_of_the_backward_is_refused(dev, which):
    """A tangent on a gradient that comes in would be lost in those that go out."""
    import batmobile
    import torch.autograd.forward_ad as fw
    t = {x: v.to(dev) for x, v in _inputs(4, 8, "f32", 91).items()}
    x = t["x"].requires_grad_(True)
    h, n = batmobile.gated_residual_norm(x, *[t[k] for k in ("y", "gate", "scale", "w_post", "w_pre")])
    with fw.dual_level():
        go = {k: t[k] for k in ("gh", "gn")}
        go[which] = fw.make_dual(go[which], torch.ones_like(h))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad([h, n], x, [go["gh"], go["gn"]])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_clip_of_tensors_that_share_memory(dev, dtype):
    """A gradient listed twice in place, outs that are the gradients in another order, shifted
    views, an out behind two gradients: each result is its gradient times the factor, whatever the
    order of the writes.  Sizes of some hundred shares, tolerances as in test_clip."""
    import batmobile
    bound = 5e-7 if dtype == "f32" else 4e-3
    n = 1 << 21
    base = torch.randn(n + 64, generator=gen(92)).to(TYPES[dtype])

    def check(grads, outs):
        want = ob.clip([_np(x) for x in grads], 1.0)
        norm, res = batmobile.clip_grad_norm(grads, 1.0, outs)
        assert res is outs and abs(float(norm) - want[0]) <= 1e-6 * want[0]
        return want[1]

    for _ in range(3):
        a = base[:n].to(dev)
        want = check([a, a], [a, a])                      # twice in place
        assert normwise_err(_np(a), want[0]) <= bound
        a, b = base[:n].to(dev), base[64:].to(dev)
        want = check([a, b], [b, a])                      # exchanged
        assert normwise_err(_np(b), want[0]) <= bound
        assert normwise_err(_np(a), want[1]) <= bound
        a = base.to(dev)
        want = check([a[:n]], [a[64:]])                   # shifted
        assert normwise_err(_np(a[64:]), want[0]) <= bound
        assert torch.equal(a[:64].cpu(), base[:64])
        a, b = base.to(dev), base[5:4005].to(dev)
        want = check([a[:n], b, a[n:]], [torch.empty(n, dtype=a.dtype, device=dev), a[n - 4000:n],
                                         a[n:]])          # one gradient's end is another's out
        assert normwise_err(_np(a[n - 4000:n]), want[1]) <= bound
        assert normwise_err(_np(a[n:]), want[2]) <= bound
    # parts of one buffer, in place: no copies, the bits of separate tensors
    flat = base.to(dev)
    parts, alone = list(flat.split(1000)), [x.clone() for x in flat.split(1000)]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    batmobile.clip_grad_norm(parts, 1.0, parts)
    assert torch.cuda.max_memory_allocated() - held < 1 << 18
    _, want = batmobile.clip_grad_norm(alone, 1.0)
    assert all(torch.equal(x, y) for x, y in zip(parts, want))


def test_clip_of_a_parameter_listed_twice(dev):
    """Tied weights in two lists: counted once, scaled once, from run to run the same."""
    import batmobile
    w = torch.nn.Parameter(torch.zeros(1 << 20, device=dev))
    u = torch.nn.Parameter(torch.zeros(37, device=dev))
    gw, gu = torch.randn(1 << 20, generator=gen(93)), torch.randn(37, generator=gen(94))
    rn, want = ob.clip([_np(gw), _np(gu)], 2.0)
    for _ in range(5):
        w.grad, u.grad = gw.to(dev), gu.to(dev)
        norm = batmobile.clip_grad_norm_([w, u, w], 2.0)
        assert abs(float(norm) - rn) <= 1e-6 * rn
        assert normwise_err(_np(w.grad), want[0]) <= 5e-7
        assert normwise_err(_np(u.grad), want[1]) <= 5e-7


def test_clip_tells_autograd_what_it_writes(dev):
    """Tensors that a graph has saved and clipping writes, dense or through a copy, raise in the
    backward as with torch's own in-place operators; inference tensors have no versions."""
    import batmobile
    x = torch.ones(50, device=dev, requires_grad=True)
    for g in (torch.full((50,), 2.0, device=dev), torch.full((100,), 2.0, device=dev)[::2]):
        for write in (lambda: batmobile.clip_grad_norm([g], 1.0, [g]),
                      lambda: batmobile.clip_grad_norm([torch.ones(50, device=dev)], 1.0, [g])):
            y = (x * g).sum()
            version = g._version
            write()
            assert g._version > version
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
    p = torch.nn.Parameter(torch.ones(5, device=dev))
    loss = (p ** 3).sum()
    p.grad, = torch.autograd.grad(loss, p, create_graph=True)
    z = (p.grad ** 2).sum()
    batmobile.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.inference_mode():
        g = torch.full((4,), 2.0, device=dev)
        batmobile.clip_grad_norm([g], 1.0, [g])
        assert torch.allclose(g, torch.full_like(g, 0.5))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("max_norm", [1.0, 1e-3, 1e-6])
def test_clip_factor_below_the_normal_numbers(dev, dtype, max_norm):
    """Gradients of 1e38, whose factor lies below 2^-126 (or below fp32's smallest number) though the
    results do not: whole shares and a remainder, the bounds of test_clip."""
    import batmobile
    grads = _grads([(50,), (30011,)], [dtype] * 2, 95, 2e37)
    norm, out = batmobile.clip_grad_norm([g.to(dev) for g in grads], max_norm)
    rn, want = ob.clip([_np(g) for g in grads], float(np.float32(max_norm)))
    assert max_norm / rn < 2.0 ** -126
    for o, w in zip(out, want):
        assert normwise_err(_np(o), w) <= (5e-7 if dtype == "f32" else 4e-3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("center", [-85.0, -30.0, -12.0, 12.0, 30.0, 85.0])
def test_gates_far_from_zero(dev, dtype, center):
    """Saturated gates: h is next to nothing of y or all of it, the gate's gradient next to nothing.
    Each is compared with its own largest value (x = 0), which sigmoid or 1 - sigmoid scales."""
    t = _inputs(19, 24, dtype, 96)
    t["x"].zero_()
    t["gate"] = (t["gate"].float() + center).to(TYPES[dtype])
    pre = center > 0    # below, h is too small for a norm of it
    h, _, grads = _block(dev, t, pre=pre, seeds=("gh", "gn") if pre else ("gh",))
    rh, _, want = ob.gated_residual_norm(
        *[_np(t[x]) for x in ("x", "y", "gate", "scale", "w_post")],
        _np(t["w_pre"]) if pre else None, gh=_np(t["gh"]), gn=_np(t["gn"]) if pre else None)
    assert normwise_err(_np(h), rh) <= BOUND[dtype]
    _check(grads, want, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinite_and_nan_gates(dev, dtype):
    """-inf closes a gate, inf opens it (factors 0 and 1, no gradient), the type's largest values as
    well; a NaN stays in its row."""
    t = _inputs(30, 20, dtype, 97)
    big = torch.finfo(TYPES[dtype]).max
    for i, g in enumerate((np.inf, -np.inf, big, -big)):
        t["gate"][i::6, ::3, 1:3] = g
    h, n, grads = _block(dev, t)
    with np.errstate(over="ignore"):
        rh, rn, want = ob.gated_residual_norm(
            *[_np(t[x]) for x in ("x", "y", "gate", "scale", "w_post", "w_pre")],
            gh=_np(t["gh"]), gn=_np(t["gn"]))
    assert normwise_err(_np(h), rh) <= BOUND[dtype]
    assert normwise_err(_np(n), rn) <= BOUND[dtype]
    _check(grads, want, dtype)
    assert not grads["gate"][0, ::3, 1:3].any() and not grads["gate"][1, ::3, 1:3].any()
    t["gate"][4, 2, 1] = np.nan
    h, n, grads = _block(dev, t)
    rows = [i for i in range(30) if i != 4]
    assert torch.isnan(h[4, 2, 1:4]).all() and torch.isfinite(h[rows]).all()
    assert torch.isnan(grads["gate"][4]).any() and torch.isfinite(grads["gate"][rows]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(5003, 100), (2501, 200), (2201, 400), (1301, 700), (1101, 1500)])
def test_many_rows_of_many_channels(dev, dtype, n, c):
    """2 to 16 waves a row, each workgroup of the backward taking two rows and more in turn."""
    t = _inputs(n, c, dtype, n)
    h, nn, grads = _block(dev, t)
    rh, rn, want = ob.gated_residual_norm(*[_np(t[x]) for x in ("x", "y", "gate", "scale", "w_post",
                                                                "w_pre")],
                                          gh=_np(t["gh"]), gn=_np(t["gn"]))
    assert normwise_err(_np(h), rh) <= BOUND[dtype]
    assert normwise_err(_np(nn), rn) <= BOUND[dtype]
    _check(grads, want, dtype)


def test_clip_of_more_than_a_turn_of_the_workgroups(dev):
    """70 MB of both types, every workgroup taking shares in turn, gradients and outs at odd elements;
    the same bits as from aligned tensors."""
    import batmobile
    g = gen(98)
    sizes = [(9_000_017, "f32"), (13_000_003, "bf16"), (3, "bf16"), (2_000_001, "f32")]
    vals = [torch.randn(n, generator=g).to(TYPES[t]) for n, t in sizes]

    def odd(v):
        w = torch.empty(v.numel() + 1, dtype=v.dtype, device=dev)[1:]
        return w.copy_(v.to(dev))
    grads, outs = [odd(v) for v in vals], [odd(torch.zeros_like(v)) for v in vals]
    norm, res = batmobile.clip_grad_norm(grads, 3.0, outs)
    rn, want = ob.clip([_np(v) for v in vals], 3.0)
    assert res is outs and abs(float(norm) - rn) <= 1e-6 * rn
    for o, w, (_, t) in zip(outs, want, sizes):
        assert normwise_err(_np(o), w) <= (5e-7 if t == "f32" else 4e-3)
    norm2, aligned = batmobile.clip_grad_norm([v.to(dev) for v in vals], 3.0)
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(aligned, outs))
