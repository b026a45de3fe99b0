"""Bias by distance, layer norm, channel mixing, gated activation and 8-bit checkpoints without a GPU:
what is refused on the host before anything runs."""
import ctypes
import os

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ERR_ARG, ERR_WORKSPACE = -1, -2
ADDR, ODD, NONE = ctypes.c_void_p(4096), ctypes.c_void_p(4104 - 4), ctypes.c_void_p(None)


def i64(v):
    return ctypes.c_int64(v)


def size(v):
    return ctypes.c_size_t(v)


def f32(v):
    return ctypes.c_float(v)


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(REPO, "batmobile-evo_amd", "lib", "libbatmobile_hip.so"))
    for n in ("distance_bias_backward", "layer_norm_backward", "channel_mixing",
              "channel_mixing_weight_grad"):
        getattr(lib, f"batteries_{n}_workspace_bytes").restype = ctypes.c_size_t
    return lib


# the addresses are never read: every call is refused (or has nothing to do) before a launch

def _bias(lib, e=10, h=4, b=8, cutoff=5.0, lengths=ADDR, bounds=ADDR, table=ADDR, out=ADDR):
    return lib.batteries_distance_bias(lengths, bounds, table, out, NONE, i64(e), h, b, f32(cutoff),
                                       NONE)


@pytest.mark.parametrize("given", [dict(e=-1), dict(e=1 << 38), dict(h=0), dict(h=1025), dict(b=0),
                                   dict(b=4097), dict(cutoff=-1.0), dict(cutoff=float("nan")),
                                   dict(cutoff=1e-31), dict(cutoff=2e30),
                                   dict(cutoff=float("inf")), dict(lengths=NONE), dict(bounds=NONE),
                                   dict(table=NONE), dict(out=NONE)])
def test_distance_bias_refuses(lib, given):
    assert _bias(lib, **given) == ERR_ARG


def _bias_back(lib, e=10, h=4, b=8, lengths=ADDR, buckets=ADDR, g=ADDR, gt=ADDR, gl=ADDR, ws=ADDR,
               n=1 << 30):
    return lib.batteries_distance_bias_backward(lengths, buckets, g, gt, gl, i64(e), h, b, f32(5.0),
                                                ws, size(n), NONE)


@pytest.mark.parametrize("given,want", [(dict(g=NONE), ERR_ARG), (dict(buckets=NONE), ERR_ARG),
                                        (dict(lengths=NONE), ERR_ARG), (dict(ws=NONE), ERR_WORKSPACE),
                                        (dict(n=4), ERR_WORKSPACE), (dict(b=0), ERR_ARG)])
def test_distance_bias_backward_refuses(lib, given, want):
    assert _bias_back(lib, **given) == want


def _ln(lib, rows=3, d=8, eps=1e-5, dtype=0, x=ADDR, w=ADDR, y=ADDR):
    return lib.batteries_layer_norm(x, w, NONE, y, i64(rows), d, i64(d), i64(1), f32(eps), dtype, NONE)


@pytest.mark.parametrize("given", [dict(rows=-1), dict(d=0), dict(d=8193), dict(eps=-1.0),
                                   dict(eps=float("nan")), dict(dtype=2), dict(x=NONE), dict(w=NONE),
                                   dict(y=NONE), dict(x=ctypes.c_void_p(4097)),
                                   dict(y=ctypes.c_void_p(4098))])
def test_layer_norm_refuses(lib, given):
    assert _ln(lib, **given) == ERR_ARG


def _ln_back(lib, g=ADDR, gx=ADDR, gw=ADDR, ws=ADDR, n=1 << 30):
    return lib.batteries_layer_norm_backward(ADDR, ADDR, g, gx, gw, NONE, i64(3), 8, i64(8), i64(1),
                                             f32(1e-5), 0, ws, size(n), NONE)


@pytest.mark.parametrize("given,want", [(dict(g=NONE), ERR_ARG), (dict(gx=NONE), ERR_ARG),
                                        (dict(gw=NONE), ERR_ARG), (dict(ws=NONE), ERR_WORKSPACE),
                                        (dict(n=8), ERR_WORKSPACE)])
def test_layer_norm_backward_refuses(lib, given, want):
    assert _ln_back(lib, **given) == want


def _mix(lib, n=3, c=8, o=8, dtype=0, x=ADDR, w=ADDR, y=ADDR, ws=ADDR, b=1 << 30):
    return lib.batteries_channel_mixing(x, w, y, i64(n), c, o, 0, dtype, ws, size(b), NONE)


@pytest.mark.parametrize("given,want", [
    (dict(n=-1), ERR_ARG), (dict(n=1 << 31), ERR_ARG), (dict(c=0), ERR_ARG), (dict(o=2049), ERR_ARG),
    (dict(dtype=2), ERR_ARG), (dict(x=NONE), ERR_ARG), (dict(w=NONE), ERR_ARG), (dict(y=NONE), ERR_ARG),
    (dict(x=ODD), ERR_ARG), (dict(y=ODD), ERR_ARG), (dict(ws=NONE), ERR_WORKSPACE),
    (dict(b=8), ERR_WORKSPACE)])
def test_channel_mixing_refuses(lib, given, want):
    assert _mix(lib, **given) == want


@pytest.mark.parametrize("c", [8, 64, 65, 128, 256, 257, 2048])
@pytest.mark.parametrize("dtype", [0, 1])
def test_channel_mixing_refuses_a_byte_too_few(lib, c, dtype):
    need = lib.batteries_channel_mixing_workspace_bytes(c, 8, 0, dtype)
    assert need >= 16 and _mix(lib, c=c, dtype=dtype, b=need - 1) == ERR_WORKSPACE


def _mix_weight(lib, n=3, x=ADDR, codes=NONE, exps=NONE, g=ADDR, gw=ADDR, ws=ADDR, b=1 << 30):
    return lib.batteries_channel_mixing_weight_grad(x, codes, exps, g, gw, i64(n), 8, 8, 0, ws, size(b),
                                                    NONE)


@pytest.mark.parametrize("given,want", [
    (dict(x=NONE), ERR_ARG), (dict(x=NONE, codes=ADDR), ERR_ARG), (dict(x=NONE, exps=ADDR), ERR_ARG),
    (dict(g=NONE), ERR_ARG), (dict(gw=NONE), ERR_ARG), (dict(g=ODD), ERR_ARG),
    (dict(ws=NONE), ERR_WORKSPACE), (dict(b=64), ERR_WORKSPACE)])
def test_weight_gradient_refuses(lib, given, want):
    assert _mix_weight(lib, **given) == want


def test_gate_and_checkpoint_refuse(lib):
    def gate(n=3, c=8, dtype=0, x=ADDR, y=ADDR, codes=NONE, exps=NONE):
        return lib.batteries_gate_activation(x, y, codes, exps, i64(n), c, dtype, NONE)

    def back(x=ADDR, codes=NONE, exps=NONE, g=ADDR, gx=ADDR):
        return lib.batteries_gate_activation_backward(x, codes, exps, g, gx, i64(3), 8, 0, NONE)

    def encode(x=ADDR, codes=ADDR, exps=ADDR, n=3, c=8):
        return lib.batteries_checkpoint_encode(x, codes, exps, i64(n), c, 0, NONE)

    def decode(codes=ADDR, exps=ADDR, x=ADDR):
        return lib.batteries_checkpoint_decode(codes, exps, x, i64(3), 8, 0, NONE)

    for given in (dict(n=-1), dict(c=0), dict(c=2049), dict(dtype=2), dict(x=NONE), dict(y=NONE),
                  dict(codes=ADDR), dict(x=ODD), dict(codes=ODD, exps=ADDR), dict(n=1 << 31)):
        assert gate(**given) == ERR_ARG, given
    for given in (dict(x=NONE), dict(x=NONE, codes=ADDR), dict(g=NONE), dict(gx=NONE), dict(g=ODD)):
        assert back(**given) == ERR_ARG, given
    for given in (dict(x=NONE), dict(codes=NONE), dict(exps=NONE), dict(codes=ODD),
                  dict(n=1 << 28, c=64)):
        assert encode(**given) == ERR_ARG, given
    for given in (dict(x=NONE), dict(codes=NONE), dict(exps=NONE), dict(x=ODD)):
        assert decode(**given) == ERR_ARG, given


def test_nothing_to_do(lib):
    """No rows: success without an address."""
    assert _bias(lib, e=0, lengths=NONE, out=NONE) == 0
    assert _ln(lib, rows=0, x=NONE, y=NONE) == 0
    assert _mix(lib, n=0, x=NONE, w=NONE, y=NONE, ws=NONE, b=0) == 0
    assert lib.batteries_gate_activation(NONE, NONE, NONE, NONE, i64(0), 8, 0, NONE) == 0
    assert lib.batteries_checkpoint_encode(NONE, NONE, NONE, i64(0), 8, 0, NONE) == 0


def test_workspaces_stay_small(lib):
    """Partial sums: 17 MB of tables, 64 MB of weights at most, whatever the sizes."""
    for e in (1, 1000, 10 ** 6, 10 ** 9):
        for h, b in ((1, 1), (8, 256), (64, 4096), (1024, 4096)):
            n = lib.batteries_distance_bias_backward_workspace_bytes(i64(e), h, b)
            assert 4 * h * b <= n <= max(17 << 20, 4 * h * b)
        for c, o in ((1, 1), (64, 64), (128, 256), (2048, 2048)):
            n = lib.batteries_channel_mixing_weight_grad_workspace_bytes(i64(e), c, o)
            # a partial sum: 4 degrees of c x o in 4 bytes
            assert 16 * c * o <= n <= max(64 << 20, 16 * c * o)
    assert lib.batteries_layer_norm_backward_workspace_bytes(i64(10), 9000) == 0
    assert lib.batteries_channel_mixing_workspace_bytes(4000, 8, 0, 0) == 0


# ---------------------------------------------------------------------------
# forward-mode derivatives: refused before anything else, never dropped
# ---------------------------------------------------------------------------

TANGENT_CALLS = {
    "distance_bias": (lambda b, r, k, t: b.distance_bias(r, k, t, 5.0), [(6,), (3,), (4, 2)]),
    "layer_norm": (lambda b, *t: b.layer_norm(*t), [(3, 5), (5,), (5,)]),
    "channel_mixing": (lambda b, *t: b.channel_mixing(*t), [(3, 5, 16), (4, 5, 6)]),
    "gate_activation": (lambda b, x: b.gate_activation(x), [(3, 5, 16)]),
}


@pytest.mark.parametrize("name,at", [(n, i) for n, (_, s) in TANGENT_CALLS.items()
                                     for i in range(len(s))])
def test_forward_mode_derivatives_are_refused(name, at):
    import batmobile
    import torch.autograd.forward_ad as fw
    call, shapes = TANGENT_CALLS[name]
    args = [torch.ones(s) for s in shapes]
    with fw.dual_level():
        args[at] = fw.make_dual(torch.ones(shapes[at]), torch.ones(shapes[at]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(batmobile, *args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(batmobile, *args)
    with pytest.raises(RuntimeError, match="CUDA"):      # without a tangent: the next check
        call(batmobile, *[torch.ones(s) for s in shapes])


def test_modules_refuse():
    import batmobile
    with pytest.raises(ValueError, match="checkpoint"):
        batmobile.FeedForwardBlock(16, checkpoint="e5m2")
    with pytest.raises(ValueError, match="checkpoint"):
        batmobile.AttentionBlock(16, 2, checkpoint="int8")
    with pytest.raises(ValueError, match="buckets"):
        batmobile.AttentionBlock(16, 2, buckets=0)


def test_an_attention_block_without_the_options_is_as_it_was():
    """Names, order and values of the parameters."""
    import batmobile
    g = torch.Generator().manual_seed(3)
    block = batmobile.AttentionBlock(16, 4, 2, generator=g)
    assert [n for n, _ in block.named_parameters()] == ["norm", "norm_post", "scale", "w_qkv", "w_out",
                                                        "w_gate", "w1", "w2"]
    assert list(dict(block.named_buffers())) == []
    g = torch.Generator().manual_seed(3)
    for n, s in (("w_qkv", (4, 16, 32)), ("w_out", (4, 16, 16)), ("w_gate", (16, 64)), ("w1", (8, 32)),
                 ("w2", (32, 4))):
        assert torch.equal(getattr(block, n).detach(), torch.randn(*s, generator=g) / s[-2] ** 0.5)


# ---------------------------------------------------------------------------
# launches
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("c,o,dtype,n", [(128, 64, 0, (1 << 27) + 1), (65, 65, 0, (1 << 26) + 1),
                                         (300, 2048, 1, (1 << 22) + 1)])
def test_channel_mixing_refuses_more_than_a_launch_takes(lib, c, o, dtype, n):
    """One launch of the kernel for many channels: N ceil(outputs / 64) <= 2^27, more than any memory holds."""
    assert _mix(lib, n=n, c=c, o=o, dtype=dtype) == ERR_ARG
    assert n * (16 * (4 >> dtype)) * (c + o) > 288 * 2 ** 30


@pytest.mark.parametrize("c,o,dtype", [(64, 2048, 0), (256, 2048, 1)])
def test_channel_mixing_of_few_channels_has_no_such_limit(lib, c, o, dtype):
    """(a workspace too small is what is refused next)"""
    assert _mix(lib, n=(1 << 31) - 1, c=c, o=o, dtype=dtype, b=15) == ERR_WORKSPACE


def test_a_table_begins_the_same_size_for_any_number_of_buckets():
    """A lookup adds nothing up: its entries do not get smaller as buckets get finer.  The spread of 4096
    normal numbers is known to 1 / sqrt(2 * 4096) = 1.1 %; four times that of each."""
    import batmobile

    def spread(buckets, heads):
        g = torch.Generator().manual_seed(buckets)
        return float(batmobile.AttentionBlock(heads, heads, generator=g, buckets=buckets).table.detach().std())

    few, many = spread(4, 1024), spread(1024, 4)
    assert abs(few / many - 1) <= 0.09


def test_an_attention_block_kept_before_it_had_the_options_still_runs():
    """A pickled module is its attributes: one without a table and checkpoints has neither."""
    import pickle
    import batmobile
    block = batmobile.AttentionBlock(16, 4, 2)
    want = block.edge_bias(torch.linspace(0.5, 6.0, 9))
    state = {k: v for k, v in block.__dict__.items() if k not in ("table", "checkpoint")}
    old = batmobile.AttentionBlock.__new__(batmobile.AttentionBlock)
    old.__setstate__(pickle.loads(pickle.dumps(state)))
    x, w = torch.randn(3, 16, 16), block.w_out
    assert torch.equal(old.edge_bias(torch.linspace(0.5, 6.0, 9)), want)
    assert torch.equal(old.mix(x, w), block.mix(x, w))
    new = pickle.loads(pickle.dumps(batmobile.AttentionBlock(16, 4, buckets=5, checkpoint="e4m3")))
    assert new.table.shape == (5, 4) and new.checkpoint == "e4m3"
