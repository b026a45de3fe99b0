"""Attention over the edges of a graph on the GPU against the float64 oracle.

Bounds (normwise, max|got - want| / max|want|).  fp32: a logit is a sum of up to 256 products,
its error a few 2^-24 sqrt(256) = 1e-6 of its size (about 1), which the exponential passes on to
the probabilities; outputs and gradients stay within 1e-5.  bf16: the results are rounded to 8
bits (2^-9 = 2e-3 of the largest), the probabilities and their gradients possibly too before
they meet the rows, whose weighted sum of absolute values is at most 3 times the largest result
for these inputs: 8e-3.  The bias gradient is fp32 in either case: 1e-5.
"""
import ctypes
import os

import numpy as np
import pytest
import torch

from oracle import block as ob

from helpers import gen, normwise_err, periodic_box

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BOUND = {"f32": 1e-5, "bf16": 8e-3}


def _edges(degrees, m, seed, distinct=True):
    """src ascending within rows of the given degrees, row_ptr."""
    rng = np.random.default_rng(seed)
    src = [np.sort(rng.permutation(m)[:d] if distinct else rng.integers(0, m, d)) for d in degrees]
    row_ptr = np.concatenate([[0], np.cumsum(degrees)]).astype(np.int64)
    return np.concatenate(src + [np.zeros(0)]).astype(np.int64), row_ptr


def _inputs(n, m, e, h, kv, dk, dv, dtype, seed, bias=True):
    g = gen(seed)
    t = TYPES[dtype]
    return {"q": torch.randn(n, h, dk, generator=g).to(t),
            "k": torch.randn(m, kv, dk, generator=g).to(t),
            "v": torch.randn(m, kv, dv, generator=g).to(t),
            "bias": torch.randn(e, h, generator=g) if bias else None,
            "go": torch.randn(n, h, dv, generator=g).to(t)}


def _np(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _run(dev, plan, t, scale=None):
    """(out, grads) through autograd."""
    import batmobile
    leaf = {x: t[x].to(dev).requires_grad_(True) for x in ("q", "k", "v", "bias")
            if t[x] is not None}
    out = batmobile.neighbor_attention(leaf["q"], leaf["k"], leaf["v"], plan,
                                       bias=leaf.get("bias"), scale=scale)
    grads = torch.autograd.grad(out, list(leaf.values()), t["go"].to(dev))
    torch.cuda.synchronize()
    return out, dict(zip(leaf, grads))


def _compare(out, grads, want, wgrads, dtype, what=""):
    assert normwise_err(_np(out), want) <= BOUND[dtype], what
    for name, got in grads.items():
        bound = BOUND["f32" if name == "bias" else dtype]
        assert normwise_err(_np(got), wgrads[name]) <= bound, (what, name)


def _check(dev, src, row_ptr, m, t, dtype, order=None, src_order=None, scale=None):
    import batmobile
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev), torch.from_numpy(row_ptr).to(dev),
                                   m, order, src_order)
    out, grads = _run(dev, plan, t, scale)
    want, wg = ob.attention(_np(t["q"]), _np(t["k"]), _np(t["v"]), src, row_ptr, _np(t["bias"]),
                            scale, _np(t["go"]))
    _compare(out, grads, want, wg, dtype)
    return out, grads


# one edge to rows longer than a tile's share of the work, empty rows between
DEGREES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 0, 64, 100, 5, 5, 5, 5, 0, 0, 3, 40, 1]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,kv,dk,dv", [(1, 1, 16, 16), (4, 4, 32, 32), (4, 2, 64, 64),
                                        (8, 1, 24, 80), (2, 2, 128, 128), (3, 3, 7, 33),
                                        (2, 1, 256, 256), (2, 2, 1, 130), (1, 1, 200, 1)])
def test_sizes(dev, dtype, h, kv, dk, dv):
    m = 150
    src, row_ptr = _edges(DEGREES, m, 1)
    t = _inputs(len(DEGREES), m, len(src), h, kv, dk, dv, dtype, 2)
    out, grads = _check(dev, src, row_ptr, m, t, dtype)
    empty = torch.tensor(DEGREES) == 0
    assert not out[empty.to(dev)].any() and not grads["q"][empty.to(dev)].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,m,degree", [(1, 1, 1), (1, 5000, 5000), (3, 3000, 2500),
                                        (17, 400, 400), (40, 64, 64), (2, 10, 0)])
def test_row_lengths(dev, dtype, n, m, degree):
    """One edge, single long rows (a readout), dense rows, no edge at all; no bias."""
    src, row_ptr = _edges([degree] * n, m, 3)
    t = _inputs(n, m, len(src), 2, 2, 64, 64, dtype, 4, bias=False)
    _check(dev, src, row_ptr, m, t, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_hub_among_short_rows(dev, dtype):
    """One destination with 3001 edges among rows of 3, one source that every row reads."""
    n, m = 50, 4000
    degrees = [3] * n
    degrees[20] = 3001
    src, row_ptr = _edges(degrees, m, 5)
    src[row_ptr[:-1]] = 0
    t = _inputs(n, m, len(src), 4, 2, 48, 64, dtype, 6)
    _check(dev, src, row_ptr, m, t, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_source_hub(dev, dtype):
    """A source that 6000 destinations read: its gradients sum over a long row."""
    n, m = 6000, 20
    rng = np.random.default_rng(7)
    src = np.stack([np.zeros(n), 1 + rng.integers(0, m - 1, n)], 1).astype(np.int64).reshape(-1)
    row_ptr = np.arange(0, 2 * n + 1, 2, dtype=np.int64)
    t = _inputs(n, m, len(src), 2, 2, 32, 32, dtype, 8)
    _check(dev, src, row_ptr, m, t, dtype)


@pytest.mark.parametrize("count", [2, 40, 700])
def test_parallel_edges(dev, count):
    """The same pair several times (periodic images), each edge with a bias of its own."""
    n, m = 20, 30
    src, row_ptr = _edges([12] * n, m, 9, distinct=False)
    src = np.concatenate([np.sort(np.concatenate([src[a:b], np.full(count, 4)])) if i == 3 else
                          src[a:b] for i, (a, b) in enumerate(zip(row_ptr[:-1], row_ptr[1:]))])
    row_ptr = row_ptr + np.where(np.arange(n + 1) > 3, count, 0)
    t = _inputs(n, m, len(src), 2, 2, 32, 48, "f32", 10)
    _check(dev, src, row_ptr, m, t, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_graph_with_orders(dev, dtype):
    """A periodic box through Graph.attention_plan: the order changes no result beyond the order
    of summation, and channels as heads commute with the float64 oracle."""
    import batmobile
    n, c, h = 300, 8, 2
    pos, cell = periodic_box(n, 11)
    graph = batmobile.Graph(pos.to(dev), cell, 5.0, c)
    src, row_ptr = graph.src.cpu().numpy(), graph.row_ptr.cpu().numpy()
    t = _inputs(n, n, len(src), h, h, c // h * 16, c // h * 16, dtype, 12)
    want, wg = ob.attention(_np(t["q"]), _np(t["k"]), _np(t["v"]), src, row_ptr, _np(t["bias"]),
                            go=_np(t["go"]))
    _compare(*_run(dev, graph.attention_plan(), t), want, wg, dtype)
    _check(dev, src, row_ptr, n, t, dtype, torch.randperm(n, generator=gen(13)).to(dev),
           torch.randperm(n, generator=gen(14)).to(dev))


def test_edge_index_in_any_order(dev):
    import batmobile
    n, m, e, h = 60, 90, 900, 3
    g = gen(15)
    ei = torch.stack([torch.randint(0, m, (e,), generator=g), torch.randint(0, n, (e,), generator=g)])
    t = _inputs(n, m, e, h, 1, 40, 24, "f32", 16)
    out, grads = _run(dev, batmobile.AttentionPlan.from_edge_index(ei.to(dev), n, m), t)
    by = np.lexsort((ei[0].numpy(), ei[1].numpy()))
    row_ptr = np.searchsorted(ei[1].numpy()[by], np.arange(n + 1))
    want, wg = ob.attention(_np(t["q"]), _np(t["k"]), _np(t["v"]), ei[0].numpy()[by], row_ptr,
                            _np(t["bias"])[by], go=_np(t["go"]))
    back = np.empty_like(wg["bias"])
    back[by] = wg["bias"]
    _compare(out, grads, want, dict(wg, bias=back), "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masks(dev, dtype):
    """Bias of -inf on single edges, on whole rows, and the type's lowest value on edges and on a
    whole row (there the probabilities are equal)."""
    m = 80
    src, row_ptr = _edges([10] * 20, m, 17)
    t = _inputs(20, m, len(src), 2, 2, 32, 32, dtype, 18)
    low = torch.finfo(torch.float32).min
    b = t["bias"]
    b[0:10] = -np.inf                 # row 0: nothing left
    b[10:20, 1] = -np.inf             # row 1: nothing left for one head
    b[20:30:3] = -np.inf
    b[30:40] = low                    # row 3: all at the lowest value
    b[40:50:2] = low
    b[50:60:2] = low
    b[51:60:2] = -np.inf              # row 5: lowest values or nothing
    out, grads = _check(dev, src, row_ptr, m, t, dtype)
    assert not out[0].any() and not out[1, 1].any() and not grads["bias"][0:10].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_infinities_and_nan_stay_where_no_edge_leads(dev, dtype, value):
    """A source with NaN or infinite keys and values, and a destination with such a query and
    gradient: only rows and sources that share an unmasked edge with them may see it."""
    n, m = 40, 40
    src, row_ptr = _edges([9] * n, m, 19)
    t = _inputs(n, m, len(src), 2, 2, 64, 64, dtype, 20)
    dst = np.repeat(np.arange(n), 9)
    bad_src, bad_dst = int(src[5 * 9]), 30
    # every edge of the bad source but one row's, and of the bad destination, is masked
    hit = ((src == bad_src) & (dst != 5)) | (dst == bad_dst)
    t["bias"][torch.from_numpy(hit)] = -np.inf
    t["k"][bad_src] = value
    t["v"][bad_src, :, 3:40] = value
    t["q"][bad_dst] = value
    t["go"][bad_dst] = value
    import batmobile
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev),
                                   torch.from_numpy(row_ptr).to(dev), m)
    out, grads = _run(dev, plan, t)
    rows = torch.arange(n) != 5
    cols = torch.from_numpy(np.setdiff1d(np.arange(m), src[dst == 5]))
    clean = {x: torch.nan_to_num(t[x].clone(), nan=0.0, posinf=0.0, neginf=0.0)
             for x in ("q", "k", "v", "go")}
    want, wg = ob.attention(_np(clean["q"]), _np(clean["k"]), _np(clean["v"]), src, row_ptr,
                            _np(t["bias"]), go=_np(clean["go"]))
    assert normwise_err(_np(out)[rows], want[rows]) <= BOUND[dtype]
    assert normwise_err(_np(grads["q"])[rows], wg["q"][rows]) <= BOUND[dtype]
    assert normwise_err(_np(grads["k"])[cols], wg["k"][cols]) <= BOUND[dtype]
    assert normwise_err(_np(grads["v"])[cols], wg["v"][cols]) <= BOUND[dtype]
    assert not np.isfinite(_np(out)[5]).all()


def test_large_logits(dev):
    """Logits of some thousands: the softmax is sharp, the maximum is taken off before the
    exponential.  A logit of 1e4 carries an fp32 error of 1e-3 in the exponent, so rows are
    compared through integers, whose products are exact."""
    n, m = 20, 60
    src, row_ptr = _edges([30] * n, m, 21)
    t = _inputs(n, m, len(src), 1, 1, 16, 32, "f32", 22)
    g = gen(23)
    t["q"] = torch.randint(-30, 31, t["q"].shape, generator=g).float()
    t["k"] = torch.randint(-30, 31, t["k"].shape, generator=g).float()
    t["bias"] = torch.randint(-3, 4, t["bias"].shape, generator=g).float()
    _check(dev, src, row_ptr, m, t, "f32", scale=1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_alignment(dev, dtype):
    """q, k, v as slices of one projection, at odd element offsets, and with transposed heads."""
    import batmobile
    n, h, d = 70, 2, 32
    src, row_ptr = _edges([12] * n, n, 24)
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev), torch.from_numpy(row_ptr).to(dev))
    t = _inputs(n, n, len(src), h, h, d, d, dtype, 25)
    base, _ = _run(dev, plan, t)
    qkv = torch.cat([t[x].reshape(n, -1) for x in "qkv"], 1).to(dev)
    odd = torch.empty(n * 3 * h * d + 3, dtype=qkv.dtype, device=dev)[3:].view(n, -1)
    odd.copy_(qkv)
    for whole in (qkv, odd):
        q, k, v = (x.view(n, h, d) for x in whole.chunk(3, 1))
        out = batmobile.neighbor_attention(q, k, v, plan, bias=t["bias"].to(dev))
        assert torch.equal(out, base)
    tr = [t[x].to(dev).transpose(0, 1).contiguous().transpose(0, 1) for x in "qkv"]
    assert torch.equal(batmobile.neighbor_attention(*tr, plan, bias=t["bias"].to(dev)), base)


def test_gradient_against_differences(dev):
    """Directional derivatives of the GPU's own fp32 output: step 1e-2, truncation of the order
    of 1e-4 of the third derivative, rounding 1e-6 / 1e-2: 1e-3 of the gradient's norm."""
    import batmobile
    n, m = 30, 40
    src, row_ptr = _edges([14] * n, m, 26)
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev),
                                   torch.from_numpy(row_ptr).to(dev), m)
    t = _inputs(n, m, len(src), 4, 2, 20, 36, "f32", 27)
    _, grads = _run(dev, plan, t)
    go = t["go"].to(dev).double()
    for name in ("q", "k", "v", "bias"):
        d = grads[name] / grads[name].norm()

        def f(step):
            s = {x: t[x].to(dev) for x in ("q", "k", "v", "bias")}
            s[name] = s[name] + step * d
            return float((batmobile.neighbor_attention(s["q"], s["k"], s["v"], plan,
                                                       bias=s["bias"]).double() * go).sum())
        want = (f(1e-2) - f(-1e-2)) / 2e-2
        got = float(grads[name].norm())
        assert abs(got - want) <= 1e-3 * got, (name, got, want)


def test_results_are_deterministic_and_follow_the_stream(dev):
    """The same bits on another stream, right behind the work that makes the inputs."""
    import batmobile
    pos, cell = periodic_box(500, 28)
    plan = batmobile.Graph(pos.to(dev), cell, 5.0, 8).attention_plan()
    e = plan.src.numel()
    t = _inputs(500, 500, e, 4, 2, 64, 64, "f32", 29)
    a, ga = _run(dev, plan, t)
    big = torch.randn(4096, 4096, device=dev)
    stream = torch.cuda.Stream()
    on = {x: t[x].to(dev) for x in t}
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(5):
            big = big @ big * 1e-3
        late = {x: (v + 0 * big[0, 0].nan_to_num().to(v.dtype)) for x, v in on.items()}
        b, gb = _run(dev, plan, late)
    assert torch.equal(a, b)
    for name in ga:
        assert torch.equal(ga[name], gb[name]), name


def test_refusals(dev):
    import batmobile
    src, row_ptr = _edges([3, 3], 5, 30)
    s, r = torch.from_numpy(src).to(dev), torch.from_numpy(row_ptr).to(dev)
    plan = batmobile.AttentionPlan(s, r, 5)
    q = torch.zeros(2, 4, 8, device=dev)
    k = torch.zeros(5, 2, 8, device=dev)
    call = batmobile.neighbor_attention
    with pytest.raises(RuntimeError, match="multiple"):
        call(q, torch.zeros(5, 3, 8, device=dev), torch.zeros(5, 3, 8, device=dev), plan)
    with pytest.raises(RuntimeError, match="head size"):
        call(q, torch.zeros(5, 2, 9, device=dev), k, plan)
    with pytest.raises(RuntimeError, match="256"):
        call(q, k, torch.zeros(5, 2, 257, device=dev), plan)
    with pytest.raises(RuntimeError, match="type"):
        call(q, k.bfloat16(), k, plan)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        call(q.double(), k.double(), k.double(), plan)
    with pytest.raises(RuntimeError, match="bias"):
        call(q, k, k, plan, bias=torch.zeros(6, 3, device=dev))
    with pytest.raises(RuntimeError, match="destinations"):
        call(torch.zeros(3, 4, 8, device=dev), k, k, plan)
    with pytest.raises(RuntimeError, match="must be on"):
        call(q, k.cpu(), k, plan)
    bad = s.clone()
    bad[1] = 5
    with pytest.raises(ValueError, match="lie in"):
        batmobile.AttentionPlan(bad, r, 5)
    with pytest.raises(ValueError, match="ascend"):
        batmobile.AttentionPlan(torch.tensor([2, 1, 3, 0, 1, 2], device=dev), r, 5)
    with pytest.raises(ValueError, match="ascend"):
        batmobile.AttentionPlan(torch.tensor([2, 1, 0], device=dev),
                                torch.tensor([0, 0, 3], device=dev), 5)
    with pytest.raises(ValueError, match="row_ptr"):
        batmobile.AttentionPlan(s, torch.tensor([0, 4, 3], device=dev), 5)
    with pytest.raises(ValueError, match="int64"):
        batmobile.AttentionPlan(s.int(), r, 5)
    with pytest.raises(ValueError, match="destinations"):
        batmobile.AttentionPlan.from_edge_index(torch.stack([s, s]), 2, 5)


@pytest.mark.parametrize("e,h", [(36000, 8), (66000, 32)])
def test_bias_by_head(dev, e, h):
    """Bias and its gradient as they lie, and with so many edges and heads that they go through
    [H, E]; edges in the caller's own order as well."""
    import batmobile
    n, d = 900, 8
    g = gen(81)
    assert h == 8 or e * h >= 1 << 21
    ei = torch.stack([torch.randint(0, n, (e,), generator=g), torch.randint(0, n, (e,), generator=g)])
    t = _inputs(n, n, e, h, 4, d, d, "f32", 82)
    out, grads = _run(dev, batmobile.AttentionPlan.from_edge_index(ei.to(dev), n), t)
    by = np.lexsort((ei[0].numpy(), ei[1].numpy()))
    row_ptr = np.searchsorted(ei[1].numpy()[by], np.arange(n + 1))
    want, wg = ob.attention(_np(t["q"]), _np(t["k"]), _np(t["v"]), ei[0].numpy()[by], row_ptr,
                            _np(t["bias"])[by], go=_np(t["go"]))
    back = np.empty_like(wg["bias"])
    back[by] = wg["bias"]
    _compare(out, grads, want, dict(wg, bias=back), "f32")


@pytest.mark.parametrize("h", [1, 3, 5, 16, 17, 40])
def test_edges_by_head(bm, dev, h):
    """The transposition itself, whole and partial groups of edges and heads, with and without an
    order, there and back: exact."""
    for e in (1, 255, 256, 1000):
        x = torch.randn(e, h, generator=gen(83))
        order = torch.randperm(e, generator=gen(84))
        q = torch.zeros(4, h, 4, device=dev)
        for eid in (None, order):
            got = bm.attention_edges_by_head(x.to(dev), None if eid is None else eid.int().to(dev))
            want = x if eid is None else x[eid]
            assert torch.equal(got.cpu(), want.t())
            again = bm.attention_edges_by_head(got, None if eid is None else eid.int().to(dev), True)
            assert torch.equal(again.cpu(), x)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_key_rows_past_32_bit_offsets(dev, dtype):
    """Sources whose rows lie more than 2^32 bytes apart from the first: k and v are slices of a
    wide table, read at 64-bit offsets."""
    import batmobile
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 10 GB")
    m, h, d = 300, 2, 32
    size = 4 if dtype == "f32" else 2
    wide = (1 << 24) // size                    # 16 MB a row: 300 rows are 5 GB
    src, row_ptr = _edges([20] * 30, m, 85)
    t = _inputs(30, m, len(src), h, h, d, d, dtype, 86)
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev),
                                   torch.from_numpy(row_ptr).to(dev), m)
    want, wg = _run(dev, plan, t)
    table = torch.zeros(m, wide, dtype=TYPES[dtype], device=dev)
    k = table[:, 64:64 + h * d].view(m, h, d)
    v = table[:, 4096:4096 + h * d].view(m, h, d)
    k.copy_(t["k"].to(dev))
    v.copy_(t["v"].to(dev))
    s = {x: t[x].to(dev) for x in t}
    leaf = [s["q"].requires_grad_(True), k.detach().requires_grad_(True),
            v.detach().requires_grad_(True), s["bias"].requires_grad_(True)]
    out = batmobile.neighbor_attention(*leaf[:3], plan, bias=leaf[3])
    assert torch.equal(out, want)
    for name, got in zip(("q", "k", "v", "bias"), torch.autograd.grad(out, leaf, s["go"])):
        assert torch.equal(got, wg[name]), name


def test_plan_covers_every_edge_once(bm, dev):
    """The plan's masks, read back: every edge appears once, in its row's order, with its column;
    tiles with many edges, long rows and parallel edges are cut within the limits."""
    cases = [([5] * 40, 30, True), ([0] * 17, 5, True), ([1500, 3, 0, 40], 2000, True),
             ([200] * 33, 220, True), ([1100] * 2 + [7] * 20, 9, False), ([3] * 100, 2, False)]
    for seed, (degrees, m, distinct) in enumerate(cases):
        src, row_ptr = _edges(degrees, m, 90 + seed, distinct)
        n, e = len(degrees), len(src)
        order = torch.randperm(n, generator=gen(95))
        plan, items, parts, bad = bm.attention_plan(torch.from_numpy(row_ptr).to(dev),
                                                    torch.from_numpy(src).to(dev), order.to(dev), m,
                                                    True)
        assert bad == 0
        p = plan.cpu().numpy()
        tiles = -(-n // 16)
        max_items = tiles + e // min(max(e // 128, 64), 512)
        pad = lambda k: (k + 15) // 16 * 16
        at = 16 + pad(tiles * 16) + 3 * pad(tiles + 1)
        items_at, at = at, at + pad(max_items * 64)
        masks_at, at = at, at + pad((e // 32 + max_items) * 16)
        seen, of_tile = np.zeros(e, int), np.zeros(tiles, int)
        for i in range(items):
            rec = p[items_at + 64 * i:items_at + 64 * i + 64]
            tile, chunk, cols, part = rec[:4]
            of_tile[tile] += 1
            edge, count = rec[32:48].copy(), np.zeros(16, int)
            for c in range(-(-cols // 32)):
                for r in range(16):
                    mask = int(p[masks_at + (chunk + c) * 16 + r]) & 0xffffffff
                    for bit in range(32):
                        if mask >> bit & 1:
                            row = int(order[tile * 16 + r])
                            assert rec[16 + r] == row
                            assert row_ptr[row] <= edge[r] < row_ptr[row + 1]
                            assert 32 * c + bit < cols
                            assert p[at + (chunk + c) * 32 + bit] == src[edge[r]]
                            seen[edge[r]] += 1
                            edge[r] += 1
                            count[r] += 1
            assert (count == rec[48:64]).all()
        assert (seen == 1).all() and (of_tile >= 1).all()
        assert parts == of_tile[of_tile > 1].sum()


def test_plan_refuses_an_order_that_is_no_permutation(dev):
    import batmobile
    src, row_ptr = _edges([3] * 5, 6, 99)
    args = [torch.from_numpy(x).to(dev) for x in (src, row_ptr)]
    with pytest.raises(ValueError, match="permutation"):
        batmobile.AttentionPlan(*args, 6, torch.tensor([0, 1, 2, 3, 3], device=dev))
    with pytest.raises(ValueError, match="permutation"):
        batmobile.AttentionPlan(*args, 6, None, torch.tensor([0, 1, 2, 3, 4, 9], device=dev))


def test_memory_of_a_captured_pass(dev):
    """Forward and backward recorded into a HIP graph and replayed three times with new inputs,
    eager work between the replays: the eager bits."""
    import batmobile
    pos, cell = periodic_box(300, 101)
    plan = batmobile.Graph(pos.to(dev), cell, 5.0, 8).attention_plan()
    plan.source_side()
    e = plan.src.numel()
    s = {x: v.to(dev) for x, v in _inputs(300, 300, e, 4, 2, 64, 64, "f32", 102).items()}
    leaf = [s[x].requires_grad_(True) for x in ("q", "k", "v", "bias")]

    def step():
        out = batmobile.neighbor_attention(*leaf[:3], plan, bias=leaf[3])
        return [out] + list(torch.autograd.grad(out, leaf, s["go"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            leaf[0].copy_(torch.randn(300, 4, 64, generator=gen(103 + k)).to(dev))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_plan_refuses_an_edge_id_that_is_no_permutation(dev):
    """edge_id places the rows of the bias and of its gradient: a number past the edges would be
    an access past them."""
    import batmobile
    src, row_ptr = _edges([3] * 5, 6, 110)
    s, r = [torch.from_numpy(x).to(dev) for x in (src, row_ptr)]
    ids = torch.arange(15, device=dev)
    for at, to in ((0, 15), (0, -1), (0, 1)):
        bad = ids.clone()
        bad[at] = to
        with pytest.raises(ValueError, match="permutation"):
            batmobile.AttentionPlan(s, r, 6, edge_id=bad)
    with pytest.raises(ValueError, match="permutation"):
        batmobile.AttentionPlan(s, r, 6, edge_id=ids[:-1])
    assert batmobile.AttentionPlan(s, r, 6, edge_id=ids.flip(0)).edge_id.dtype == torch.int32
    with pytest.raises(ValueError, match="row_ptr"):
        batmobile.AttentionPlan(s, r[:1], 6)             # edges without a row


def test_second_derivative_is_refused(dev):
    import batmobile
    src, row_ptr = _edges([3] * 5, 6, 111)
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev), torch.from_numpy(row_ptr).to(dev), 6)
    q = torch.randn(5, 2, 8, generator=gen(112)).to(dev).requires_grad_(True)
    k = torch.randn(6, 2, 8, generator=gen(113)).to(dev)
    out = batmobile.neighbor_attention(q, k, k, plan)
    grad, = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


def test_plan_made_on_one_stream_and_used_on_another(dev):
    """A plan from edges in any order, made on a stream of its own; the bias and its gradient go
    by its edge_id, forward and backward, on the current stream without a wait between."""
    import batmobile
    n, m, e, h = 300, 200, 9000, 2
    g = gen(120)
    ei = torch.stack([torch.randint(0, m, (e,), generator=g), torch.randint(0, n, (e,), generator=g)])
    t = {x: None if v is None else v.to(dev) for x, v in
         _inputs(n, m, e, h, h, 16, 16, "f32", 121).items()}
    want, wg = _run(dev, batmobile.AttentionPlan.from_edge_index(ei.to(dev), n, m), t)
    for _ in range(3):
        stream = torch.cuda.Stream()
        edges = ei.to(dev)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            plan = batmobile.AttentionPlan.from_edge_index(edges, n, m)
        out, grads = _run(dev, plan, t)
        assert torch.equal(out, want)
        for name in grads:
            assert torch.equal(grads[name], wg[name]), name
        torch.cuda.synchronize()


@pytest.mark.parametrize("check", [0, 1])
@pytest.mark.parametrize("what", ["row_ptr", "order"])
def test_plan_of_arrays_that_name_edges_again_and_again(dev, what, check):
    """A row_ptr that rises and falls, and an order that holds one row only: the rows together have
    thousands of times the edges that the plan has room for.  Refused, with nothing written behind
    the plan."""
    import batmobile
    lib = ctypes.CDLL(os.path.join(os.path.dirname(batmobile.__file__), "..", "..", "lib",
                                   "libbatmobile_hip.so"))
    lib.batteries_attention_plan_bytes.restype = ctypes.c_size_t
    n, e, m = 4000, 400, 500
    src = torch.arange(e, device=dev)
    if what == "row_ptr":
        row_ptr = torch.tensor([0, e], device=dev).repeat(n // 2 + 1)[:n + 1]
        order = None
    else:
        row_ptr = torch.full((n + 1,), e, dtype=torch.long, device=dev)
        row_ptr[0] = 0
        order = torch.zeros(n, dtype=torch.long, device=dev)
    size = lib.batteries_attention_plan_bytes(ctypes.c_int64(n), ctypes.c_int64(e))
    plan = torch.full((size // 4 + 4096,), -7, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    at = lambda t: ctypes.c_void_p(None if t is None else t.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.batteries_attention_plan(at(row_ptr), at(src), at(order), ctypes.c_int64(n),
                                        ctypes.c_int64(m), ctypes.c_int64(e), check, at(plan),
                                        ctypes.c_size_t(size), stream) == 0
    head = plan[:3].tolist()
    assert head[:2] == [0, 0] and head[2] == 8 + (check and what == "row_ptr")
    assert (plan[size // 4:] == -7).all()
    with pytest.raises(ValueError, match="row_ptr|permutation"):
        batmobile.AttentionPlan(src, row_ptr, m, order, validate=bool(check))


def test_source_side_refuses_an_order_that_repeats_a_source(dev):
    import batmobile
    src, row_ptr = _edges([9] * 200, 30, 122)
    most = int(np.bincount(src).argmax())
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev), torch.from_numpy(row_ptr).to(dev),
                                   30, src_order=torch.full((30,), most, device=dev),
                                   validate=False)
    with pytest.raises(ValueError, match="src_order"):
        plan.source_side()


def test_forward_mode_of_the_backward_is_refused(dev):
    """A tangent on the gradient that comes in would be lost in the one that goes out."""
    import batmobile
    import torch.autograd.forward_ad as fw
    src, row_ptr = _edges([3] * 5, 6, 123)
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev), torch.from_numpy(row_ptr).to(dev), 6)
    q = torch.randn(5, 2, 8, generator=gen(124)).to(dev).requires_grad_(True)
    k = torch.randn(6, 2, 8, generator=gen(125)).to(dev)
    out = batmobile.neighbor_attention(q, k, k, plan)
    with fw.dual_level():
        go = fw.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, q, go)


def test_plan_made_under_inference_mode_trains(dev):
    """An evaluation pass makes the plan (and its sources' side) first, training follows on it."""
    import batmobile
    src, row_ptr = _edges([7] * 40, 30, 126)
    t = _inputs(40, 30, len(src), 2, 1, 16, 16, "f32", 127)
    s, r = torch.from_numpy(src).to(dev), torch.from_numpy(row_ptr).to(dev)
    ids = torch.randperm(len(src), generator=gen(128)).to(dev)
    want, wg = _run(dev, batmobile.AttentionPlan(s, r, 30, edge_id=ids), t)
    for early in (False, True):
        with torch.inference_mode():
            plan = batmobile.AttentionPlan(s.clone(), r.clone(), 30, edge_id=ids)
            if early:
                plan.source_side()
        out, grads = _run(dev, plan, t)
        assert torch.equal(out, want)
        for name in grads:
            assert torch.equal(grads[name], wg[name]), name


def test_rows_2_30_elements_apart(dev):
    """Strides past what the kernels take as they are: such rows are packed first, not refused."""
    import batmobile
    n, m, d = 2, 2, 16
    src, row_ptr = np.array([0, 1, 1]), np.array([0, 2, 3])
    t = _inputs(n, m, 3, 1, 1, d, d, "bf16", 129)
    plan = batmobile.AttentionPlan(torch.from_numpy(src).to(dev),
                                   torch.from_numpy(row_ptr).to(dev), m)
    want, wg = _run(dev, plan, t)
    store = torch.empty((1 << 30) + 4 * d, dtype=torch.bfloat16, device=dev)
    far = {}
    for i, x in enumerate(("q", "k", "v", "go")):
        far[x] = store[i * d:].as_strided((2, 1, d), (1 << 30, d, 1))
        far[x].copy_(t[x].to(dev))
        far[x] = far[x].detach().requires_grad_(x != "go")
    leaf = [far["q"], far["k"], far["v"], t["bias"].to(dev).requires_grad_(True)]
    out = batmobile.neighbor_attention(*leaf[:3], plan, bias=leaf[3])
    assert torch.equal(out, want)
    for name, got in zip(("q", "k", "v", "bias"), torch.autograd.grad(out, leaf, far["go"])):
        assert torch.equal(got, wg[name]), name


def _crowded(count, seed, rows=(3,)):
    """20 rows of 12 edges among 30 sources, `count` more of each of `rows` from source 4."""
    src, row_ptr = _edges([12] * 20, 30, seed, distinct=False)
    parts = [np.sort(np.concatenate([src[a:b], np.full(count if i in rows else 0, 4)]))
             for i, (a, b) in enumerate(zip(row_ptr[:-1], row_ptr[1:]))]
    return np.concatenate(parts), np.cumsum([0] + [len(x) for x in parts])


CROWDS = [(1500, (3,)), (5000, (3,)), (20000, (17,)), (90, tuple(range(20))), (400, (0, 2, 15, 16)),
          (13, tuple(range(16)))]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("count,rows", CROWDS)
def test_more_parallel_edges_than_an_item_holds(dev, dtype, count, rows, bias):
    """A column (from either side) with more edges than a part of a cut tile should have: it is cut
    within the column, so that no sum runs over thousands of equal terms in fp32."""
    src, row_ptr = _crowded(count, 130, rows)
    t = _inputs(20, 30, len(src), 4, 2, 32, 48, dtype, 131, bias)
    if bias:
        t["bias"][row_ptr[3] + 5:row_ptr[3] + 9] = -np.inf
    _check(dev, src, row_ptr, 30, t, dtype)


@pytest.mark.parametrize("count,rows", CROWDS)
def test_plan_of_crowded_columns_covers_every_edge_once(bm, dev, count, rows):
    """As test_plan_covers_every_edge_once, and no item of more than 1024 edges."""
    src, row_ptr = _crowded(count, 132, rows)
    n, e = 20, len(src)
    plan, items, parts, bad = bm.attention_plan(torch.from_numpy(row_ptr).to(dev),
                                                torch.from_numpy(src).to(dev), None, 30, True)
    p = plan.cpu().numpy()
    tiles, pad = 2, lambda k: (k + 15) // 16 * 16
    max_items = tiles + e // min(max(e // 128, 64), 512)
    items_at = 16 + pad(tiles * 16) + 3 * pad(tiles + 1)
    masks_at = items_at + pad(max_items * 64)
    ids_at = masks_at + pad((e // 32 + max_items) * 16)
    assert bad == 0 and items <= max_items
    seen, chunk_end = np.zeros(e, int), 0
    for rec in sorted(p[items_at:items_at + 64 * items].reshape(items, 64), key=lambda r: r[1]):
        chunk, cols = rec[1], rec[2]
        chunks = -(-cols // 32)
        assert chunk >= chunk_end and chunk + chunks <= e // 32 + max_items
        chunk_end = chunk + chunks
        masks = p[masks_at + chunk * 16:masks_at + (chunk + chunks) * 16].view(np.uint32)
        ids = p[ids_at + chunk * 32:ids_at + (chunk + chunks) * 32]
        bits = (masks.reshape(chunks, 16)[:, :, None] >> np.arange(32, dtype=np.uint32)) & 1
        bits = bits.transpose(1, 0, 2).reshape(16, chunks * 32)        # [row, column]
        assert not bits[:, cols:].any() and (bits.sum(1) == rec[48:64]).all()
        for r in range(16):
            edges = np.arange(rec[32 + r], rec[32 + r] + rec[48 + r])
            assert (src[edges] == ids[bits[r] == 1]).all()
            if len(edges):
                assert row_ptr[rec[16 + r]] <= edges[0] and edges[-1] < row_ptr[rec[16 + r] + 1]
            seen[edges] += 1
        assert rec[48:64].sum() <= 1024
    assert (seen == 1).all()


def test_plan_of_columns_in_no_order_is_refused(dev):
    """Long rows whose columns do not ascend, with and without the check: the cuts, which are found by
    searching, may come out anywhere in the row."""
    import batmobile
    src = torch.cat([torch.randint(0, 3, (6000,), generator=gen(133)) for _ in range(3)]).to(dev)
    row_ptr = torch.tensor([0, 6000, 12000, 18000], device=dev)
    with pytest.raises(ValueError, match="ascend"):
        batmobile.AttentionPlan(src, row_ptr, 3)
