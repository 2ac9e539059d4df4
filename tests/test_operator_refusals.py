"""What the 8-bit linear layer, the Newton-Schulz iteration and the Muon optimiser refuse, before any device work."""
import ctypes

import pytest
import torch

import dpd_amd  # noqa: F401
from dpd_amd import _lib as L
from dpd_amd.training import Muon
from dpd_amd.utils import Int8Inference, Int8Linear, int8_linear, int8_matmul, orthogonalize, quantize_rows_int8

P = (ctypes.c_float * 1024)()
PTR, NULL = ctypes.cast(P, ctypes.c_void_p), ctypes.c_void_p(0)
COEF = (ctypes.c_float * 15)(*([3.4445, -4.775, 2.0315] * 5))


def rc(name, *args):
    return getattr(L.lib(), name)(*args), L.lib().dpd_last_error().decode()


@pytest.mark.parametrize("args, code, text", [
    ((PTR, 9, 2, 8, 8, PTR, 8, PTR, NULL), 1, "type"),
    ((PTR, 0, -1, 8, 8, PTR, 8, PTR, NULL), 1, "negative"),
    ((PTR, 0, 2, 0, 8, PTR, 8, PTR, NULL), 2, "shape"),
    ((NULL, 0, 2, 8, 8, PTR, 8, PTR, NULL), 1, "null"),
    ((PTR, 0, 2, 8, 7, PTR, 8, PTR, NULL), 1, "stride"),
    ((PTR, 0, 2, 8, 8, PTR, 7, PTR, NULL), 1, "stride"),
    ((NULL, 0, 0, 8, 8, NULL, 8, NULL, NULL), 0, ""),
])
def test_quantize_rows_arguments(args, code, text):
    got, msg = rc("dpd_quantize_rows_int8", *args)
    assert got == code and (code == 0 or text in msg)


def matmul_args(**kw):
    d = dict(a=PTR, lda=16, sa=PTR, b=PTR, ldb=16, sb=PTR, bias=NULL, bt=0, M=2, N=2, K=16, out=PTR, ot=0, ldo=2, ws=NULL, wn=0, st=NULL)
    d.update(kw)
    return list(d.values())


@pytest.mark.parametrize("kw, code, text", [
    (dict(ot=3), 1, "type"), (dict(bias=PTR, bt=7), 1, "type"), (dict(M=-1), 1, "negative"), (dict(K=0), 2, "input features"),
    (dict(K=131072, lda=131072, ldb=131072), 2, "32-bit"), (dict(M=1 << 31), 2, "too many"), (dict(a=NULL), 1, "null"),
    (dict(lda=15), 1, "stride"), (dict(ldo=1), 1, "stride"), (dict(lda=1 << 23), 1, "stride"), (dict(K=15), 4, "workspace"),
    (dict(M=0, a=NULL), 0, ""), (dict(N=0, b=NULL), 0, ""),
])
def test_matmul_arguments(kw, code, text):
    got, msg = rc("dpd_int8_matmul", *matmul_args(**kw))
    assert got == code and (code == 0 or text in msg)


def test_linear_and_backward_arguments():
    ws = L.lib().dpd_int8_linear_workspace_bytes(40, 4, 16)          # few tokens need none
    ok = [PTR, 0, 40, 16, 16, PTR, PTR, NULL, 0, 4, PTR, 4, PTR, ws, NULL]
    for at, value, code, text in ((1, 5, 1, "type"), (3, 0, 2, "input features"), (0, NULL, 1, "null"), (4, 15, 1, "stride"), (11, 3, 1, "stride"),
                                  (13, ws - 1, 4, "workspace"), (5, ctypes.c_void_p(PTR.value + 8), 1, "aligned")):
        args = list(ok)
        args[at] = value
        got, msg = rc("dpd_int8_linear", *args)
        assert got == code and text in msg, (at, msg)
    n = L.lib().dpd_int8_linear_backward_workspace_bytes(2, 4, 16, 0, 1, 1, 1)
    ok = [PTR, 0, 2, 4, 16, 4, PTR, 128, PTR, PTR, 128, PTR, PTR, PTR, 0, PTR, 0, PTR, n, NULL]
    for at, value, code, text in ((1, 5, 1, "type"), (14, 5, 1, "type"), (0, NULL, 1, "null"), (6, NULL, 1, "null"), (9, NULL, 1, "null"), (5, 3, 1, "stride"),
                                  (18, n - 1, 4, "workspace"), (2, 1 << 22, 2, "too many")):
        args = list(ok)
        args[at] = value
        got, msg = rc("dpd_int8_linear_backward", *args)
        assert got == code and text in msg, (at, msg)


def test_orthogonalize_arguments():
    ok = [PTR, 0, 1, 200, 300, 5, COEF, 1e-7, 0, PTR, PTR, 1 << 40, NULL]
    wild = (ctypes.c_float * 15)(*([30.0, 0.0, 0.0] * 5))
    nan = (ctypes.c_float * 15)(*([float("nan"), 0.0, 0.0] * 5))
    for at, value, code, text in ((1, 4, 1, "type"), (2, -1, 1, "batch"), (3, -1, 1, "negative"), (4, 1 << 21, 2, "too long"), (5, 0, 2, "steps"),
                                  (5, 33, 2, "steps"), (6, wild, 2, "out of range"), (6, nan, 2, "out of range"), (7, 0.0, 2, "eps"), (7, float("nan"), 2, "eps"),
                                  (0, NULL, 1, "null"), (2, 65536, 2, "65535"), (11, 1000, 4, "workspace")):
        args = list(ok)
        args[at] = value
        got, msg = rc("dpd_orthogonalize", *args)
        assert got == code and text in msg, (at, msg)
    assert rc("dpd_orthogonalize", NULL, 0, 0, 8, 8, 5, COEF, 1e-7, 0, NULL, NULL, 0, NULL)[0] == 0      # no matrices


def test_muon_arguments():
    ptr, i64 = (ctypes.c_void_p * 2)(PTR.value, PTR.value), ctypes.c_int64 * 2
    none = (ctypes.c_void_p * 2)(PTR.value, 0)
    rows, cols = i64(200, 4), i64(200, 4)
    ok = [2, ptr, ptr, ptr, rows, cols, 0, 0.02, 0.95, 1, 0.0, 5, COEF, 1e-7, 0, PTR, 1 << 40, NULL]
    for at, value, code, text in ((0, -1, 1, "null"), (1, None, 1, "null"), (2, none, 1, "matrix 1"), (6, 3, 1, "type"), (11, 0, 2, "steps"), (13, -1.0, 2, "eps"),
                                  (16, 1000, 4, "workspace"), (4, i64(200, -4), 1, "negative")):
        args = list(ok)
        args[at] = value
        got, msg = rc("dpd_muon_step", *args)
        assert got == code and text in msg, (at, msg)


def test_workspace_sizes():
    lib = L.lib()
    assert lib.dpd_int8_row_bytes(1) == 128 and lib.dpd_int8_row_bytes(128) == 128 and lib.dpd_int8_row_bytes(129) == 256
    assert lib.dpd_orthogonalize_workspace_bytes(1, 64, 128, 1) == 256                    # runs without one
    assert lib.dpd_orthogonalize_workspace_bytes(1, 128, 129, 0) == 256 and lib.dpd_orthogonalize_workspace_bytes(1, 129, 129, 0) > 256
    assert lib.dpd_orthogonalize_workspace_bytes(1, 64, 512, 1) == 256 and lib.dpd_orthogonalize_workspace_bytes(1, 64, 640, 1) > 256
    assert lib.dpd_orthogonalize_workspace_bytes(2, 4096, 4096, 1) > lib.dpd_orthogonalize_workspace_bytes(2, 4096, 4096, 0) > 2 * 4096 * 4096 * 10
    assert lib.dpd_int8_linear_backward_workspace_bytes(10, 10, 10, 0, 0, 0, 0) == 256


def test_host_layer_refusals():
    x, w = torch.randn(3, 8), torch.randn(4, 8)
    for call in (lambda: quantize_rows_int8(x), lambda: int8_linear(x, w), lambda: Int8Linear(8, 4)(x), lambda: orthogonalize(x),
                 lambda: int8_matmul(x.to(torch.int8), x[:, 0], w.to(torch.int8), w[:, 0]),
                 lambda: Int8Inference({"weight": w.to(torch.int8), "scale": w[:, 0]})):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()


def test_muon_refusals_and_groups():
    net = torch.nn.Linear(6, 5)
    for kw in (dict(momentum=1.0), dict(lr=-1.0), dict(eps=0.0), dict(weight_decay=-0.1), dict(steps=0), dict(steps=33), dict(coefficients=(1.0, 2.0)),
               dict(coefficients=[(1.5, -0.5, 0.0)] * 4)):
        with pytest.raises(ValueError):
            Muon(net.parameters(), **kw)
    opt = Muon(net.parameters(), lr=0.1, adam=dict(lr=0.3))
    assert [g["kind"] for g in opt.param_groups] == ["matrix", "other"]
    assert [g["lr"] for g in opt.param_groups] == [0.1, 0.3]
    sched = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.5)
    opt.step()                       # no gradients: nothing to do
    sched.step()
    assert [g["lr"] for g in opt.param_groups] == [0.05, 0.15]
    net.weight.grad = torch.zeros_like(net.weight)
    with pytest.raises(RuntimeError, match="MI355X"):
        opt.step()
    for twice in ([net.weight, net.weight], [{"params": [net.weight]}, {"params": [net.weight]}]):
        with pytest.raises(ValueError, match="twice"):
            Muon(twice)
    opt = Muon([{"params": [net.weight], "lr": 0.7}, {"params": net.bias}])
    assert opt.param_groups[0]["lr"] == 0.7 and opt.param_groups[1]["kind"] == "other"


def test_muon_state_keeps_its_precision():
    """The base class casts optimiser state to the parameter's type when it is loaded; the momentum stays fp32."""
    p = torch.nn.Parameter(torch.randn(4, 6, dtype=torch.bfloat16))
    a, b = Muon([p]), Muon([p])
    m = torch.randn(4, 6)
    a.state[p]["momentum_buffer"] = m
    b.load_state_dict(a.state_dict())
    got = b.state[p]["momentum_buffer"]
    assert got.dtype == torch.float32 and torch.equal(got, m) and got.data_ptr() != m.data_ptr()


def test_train_configuration_names_the_optimizer():
    from dpd_amd.train import build_parser, create_optimizers, load_config
    config = load_config("")
    gen, disc = torch.nn.Linear(3, 2), torch.nn.Linear(3, 2)
    assert isinstance(create_optimizers(gen, disc, config)[0], torch.optim.Adam)
    config["training"]["optimizer"] = dict(config["training"]["optimizer"], type="muon", lr_matrix=0.01)
    g, d = create_optimizers(gen, disc, config)
    assert isinstance(g, Muon) and g.param_groups[0]["lr"] == 0.01 and g.param_groups[1]["lr"] == 1e-4 and isinstance(d, Muon)
    config["training"]["optimizer"]["type"] = "lion"
    with pytest.raises(ValueError, match="lion"):
        create_optimizers(gen, disc, config)
    assert build_parser().parse_args(["--optimizer", "muon"]).optimizer == "muon"


def test_serving_workspace_formula():
    """The engine computes the size of its scratch itself."""
    from dpd_amd.utils.int8 import _row_bytes
    for m, n, k in ((0, 4, 1), (1, 4, 1), (7, 9, 128), (64, 3, 129), (1000, 5, 4096)):
        assert L.lib().dpd_int8_linear_workspace_bytes(m, n, k) == m * _row_bytes(k) + (m * 4 + 255) // 256 * 256 + 256
        assert L.lib().dpd_int8_row_bytes(k) == _row_bytes(k)


def test_product_tile_option():
    for value, code in ((10, 0), (0, 0), (11, 1), (-2, 1), (-1, 0)):
        assert L.lib().dpd_set_option(b"product_tile", value) == code


def test_the_weights_of_an_engine_have_no_setter():
    eng = object.__new__(Int8Inference)
    for name in ("scale", "image", "bias"):
        with pytest.raises(AttributeError):
            setattr(eng, name, torch.zeros(3))


@pytest.mark.parametrize("kind, most", [(0, 1398080), (1, 2097088), (2, 2097088)])
def test_backward_limits_are_those_of_the_gradients_that_are_wanted(kind, most):
    """Without a workspace: code 4 says that the sizes are taken, code 2 that they are not."""
    from dpd_amd.utils.int8 import _MOST_OUTS, _MOST_TOKENS
    assert most in _MOST_OUTS.values() and _MOST_TOKENS <= most

    def call(m, n, gx=NULL, gw=NULL, gb=NULL):
        return rc("dpd_int8_linear_backward", PTR, kind, m, n, 16, n, PTR, 128, PTR, PTR, 128, PTR, gx, gw, 0, gb, 0, NULL, 0, NULL)[0]
    assert call(1 << 24, 4, gx=PTR) == 4 and call(1 << 24, 4, gb=PTR) == 4        # nothing is summed over the tokens; gb by tiles
    assert call(most, 4, gw=PTR) == 4 and call(most + 1, 4, gw=PTR) == 2
    assert call(4, most, gx=PTR) == 4 and call(4, most + 1, gx=PTR) == 2
    assert call(4, 1 << 24, gw=PTR) == 4 and call(4, 1 << 24, gb=PTR) == 4


def test_muon_options_of_a_group_hold_for_its_biases():
    a, b = torch.nn.Linear(6, 5), torch.nn.Linear(5, 4)
    opt = Muon([{"params": a.parameters(), "lr": 0.7, "weight_decay": 0.0, "steps": 3}, {"params": b.parameters(), "name": "b"}], adam=dict(lr=0.3, weight_decay=0.2))
    kinds = [(g["kind"], g["lr"], g["weight_decay"], len(g["params"])) for g in opt.param_groups]
    assert kinds == [("matrix", 0.7, 0.0, 1), ("matrix", 0.02, 0.0, 1), ("other", 0.7, 0.0, 1), ("other", 0.3, 0.2, 1)]
    assert opt.param_groups[0]["steps"] == 3 and opt.param_groups[1]["name"] == opt.param_groups[3]["name"] == "b"
    # the biases move as Adam with these options moves them, on the CPU too
    twin, before = torch.nn.Linear(6, 5), a.bias.detach().clone()
    twin.bias.data.copy_(before)
    adam = torch.optim.Adam([twin.bias], lr=0.7, weight_decay=0.0)
    a.bias.grad = twin.bias.grad = torch.linspace(-1, 1, 5)
    opt.step()
    adam.step()
    assert torch.equal(a.bias, twin.bias) and not torch.equal(a.bias, before)


@pytest.mark.parametrize("bad", [dict(momentum=2.0), dict(lr=-1.0), dict(weight_decay=-0.1), dict(eps=0.0), dict(steps=99), dict(coefficients=(1.0, 2.0))])
def test_muon_checks_the_options_of_groups(bad):
    net, more = torch.nn.Linear(6, 5), torch.nn.Linear(5, 4)
    with pytest.raises(ValueError):
        Muon([{"params": [net.weight], **bad}])
    opt = Muon(net.parameters())
    with pytest.raises(ValueError):
        opt.add_param_group({"params": list(more.parameters()), **bad})
    assert len(opt.param_groups) == 2


def test_muon_takes_groups_later():
    import copy
    net, more = torch.nn.Linear(6, 5), torch.nn.Linear(5, 4)
    first = Muon(net.parameters(), adam=dict(lr=0.3))
    for opt in (first, copy.deepcopy(first)):
        opt.add_param_group({"params": list(more.parameters()), "lr": 0.5})
        assert [(g["kind"], g["lr"]) for g in opt.param_groups] == [("matrix", 0.02), ("other", 0.3), ("matrix", 0.5), ("other", 0.5)]
        with pytest.raises(ValueError, match="twice"):
            opt.add_param_group({"params": [more.weight, more.weight]})
    with pytest.raises(ValueError, match="twice"):
        first.add_param_group({"params": [net.bias]})


def test_longest_stride_of_the_product():
    from dpd_amd.utils.int8 import _MOST_STRIDE
    assert rc("dpd_int8_matmul", *matmul_args(lda=_MOST_STRIDE, K=15))[0] == 4                # a workspace is all that is missing
    assert rc("dpd_int8_matmul", *matmul_args(lda=_MOST_STRIDE + 1, K=15))[0] == 1


def test_one_token_against_more_channels_than_one_grid_covers():
    """16 channels a workgroup of 256 threads: from 2^28 channels on the tiled product takes the token, with a workspace."""
    got, msg = rc("dpd_int8_linear", PTR, 0, 1, 16, 16, PTR, PTR, NULL, 0, (1 << 28) + 16, PTR, (1 << 28) + 16, NULL, 0, NULL)
    assert got == 4 and "workspace" in msg


def test_an_empty_optimizer_type_is_adam():
    from dpd_amd.train import create_optimizers, load_config
    config = load_config("")
    for kind in (None, "", "Adam"):
        config["training"]["optimizer"] = dict(config["training"]["optimizer"], type=kind)
        assert all(type(o) is torch.optim.Adam for o in create_optimizers(torch.nn.Linear(3, 2), torch.nn.Linear(3, 2), config))


def test_muon_takes_no_sets():
    """Their order changes from run to run, and with it what a saved state belongs to."""
    net = torch.nn.Linear(6, 5)
    for params in (set(net.parameters()), [{"params": set(net.parameters())}]):
        with pytest.raises(TypeError, match="order"):
            Muon(params)
    opt = Muon([net.weight])
    with pytest.raises(TypeError, match="order"):
        opt.add_param_group({"params": {net.bias}})
    assert Muon(net.weight).param_groups[0]["params"] == [net.weight]     # one tensor alone
