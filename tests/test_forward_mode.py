"""Forward-mode differentiation: no kernel has such a rule, so public functions take their torch path or refuse, and an op that a
tangent reaches all the same raises instead of dropping it."""

import warnings

import pytest
import torch
from torch.autograd import forward_ad

from tests.test_serving import F32, make
from tsfast_amd import dispatch, gated, mamba, ops
from tsfast_amd.gated import core, feed_hip

F64 = torch.float64


@pytest.fixture(scope="module")
def doubled():
    @ops.custom_op("tsfast_hip_test::doubled")
    def doubled(x: torch.Tensor) -> torch.Tensor:
        return x * 2

    doubled.register_fake(lambda x: torch.empty_like(x))
    doubled.register_vmap(lambda info, in_dims, x: (doubled(x), in_dims[0]))
    return doubled


WAYS = {
    "jvp": lambda f, x: torch.func.jvp(f, (x,), (x,)),
    "jacfwd": lambda f, x: torch.func.jacfwd(f)(x),
    "vmap in jvp": lambda f, x: torch.func.jvp(torch.func.vmap(f), (x,), (x,)),
    "jvp in vmap": lambda f, x: torch.func.vmap(lambda y: torch.func.jvp(f, (y,), (y,))[1])(x),
    "hessian": lambda f, x: torch.func.hessian(lambda y: (f(y) ** 2).sum())(x),
    "jvp in jvp": lambda f, x: torch.func.jvp(lambda y: torch.func.jvp(lambda w: f(y) * w, (x,), (x,))[1], (x,), (x,)),
    "compiled jvp": lambda f, x: torch.compile(lambda y: torch.func.jvp(f, (y,), (y,)), backend="eager", fullgraph=True)(x),
}


@pytest.mark.parametrize("way", WAYS)
def test_an_op_raises_where_it_would_drop_a_tangent(doubled, way):
    with pytest.raises(Exception, match="no forward-mode derivative|Observed exception"):
        WAYS[way](doubled, torch.randn(4, 3))


def test_an_op_takes_tensors_without_a_tangent(doubled):
    x = torch.randn(4, 3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        assert torch.equal(doubled(x), 2 * x)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            doubled(dual)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            doubled(x=dual)
        assert ops.has_tangent((None, (1.0, [dual]))) and not ops.has_tangent((None, x, (x, 2)))
    assert not ops.has_tangent((x,))
    assert torch.equal(torch.func.jvp(lambda y: y * doubled(x), (x,), (x,))[1], 2 * x * x)
    assert torch.equal(torch.func.vmap(doubled)(x), 2 * x)


def test_dispatch_takes_the_reference_path_for_a_tangent(monkeypatch):
    class Fused:
        supports = staticmethod(lambda *args: None)

    monkeypatch.setattr(dispatch, "_warned", set())
    pick = lambda *args: dispatch.resolve("forward.test", {"hip": Fused}, ("hip",), args)  # noqa: E731
    x = torch.randn(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        assert pick(x, None) is Fused
        with pytest.warns(RuntimeWarning, match="no forward-mode derivative"):
            assert pick(x, (None, dual)) is None
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            assert pick(dual) is None


@pytest.fixture
def stubbed(monkeypatch):
    """The fused feed-forward with its kernels replaced: CPU tensors go where GPU tensors would, through the registered op."""

    def forward(x, wg, wu, bg, bu, activation, train):
        y = torch.nn.functional.silu(x @ wg.T) * (x @ wu.T)
        return y, torch.empty(feed_hip.kept_bytes(x.shape[0], wg.shape[0], x.dtype), dtype=torch.uint8) if train else None

    monkeypatch.setattr(core, "_AUTO_ORDER", {"cpu": ("hip",)})
    monkeypatch.setattr(feed_hip, "supports", lambda *args: None)
    monkeypatch.setattr(feed_hip, "_forward", forward)
    monkeypatch.setattr(dispatch, "_warned", set())


def _near(a, b, rel):
    assert float((a - b).detach().abs().max()) <= rel * float(b.abs().max())


def _check_feed(dev, dtype, which, rel):
    r = torch.Generator(device=dev).manual_seed(0)
    tensors = [torch.randn(*s, generator=r, device=dev, dtype=dtype) for s in ((5, 4), (6, 4), (6, 4))]
    f = lambda t: gated.gated_feed_forward(*(t if i == which else s for i, s in enumerate(tensors)))  # noqa: E731
    t, tangent = tensors[which], torch.ones_like(tensors[which])
    with dispatch.use_backend("reference"):
        want, want_t = torch.func.jvp(f, (t,), (tangent,))
        want_h = torch.func.hessian(lambda s: f(s).square().sum())(t)
    assert want_t.abs().max() > 1
    got, got_t = torch.func.jvp(f, (t,), (tangent,))
    _near(got, want, rel), _near(got_t, want_t, rel)
    with forward_ad.dual_level():
        for leaf in (t, t.clone().requires_grad_()):
            _near(forward_ad.unpack_dual(f(forward_ad.make_dual(leaf, tangent))).tangent, want_t, rel)
    _near(torch.func.hessian(lambda s: f(s).square().sum())(t), want_h, rel)


@pytest.mark.filterwarnings("ignore:backend")
@pytest.mark.parametrize("which", [0, 1, 2])
def test_feed_forward_has_its_tangent(stubbed, which):
    """As the torch path has it, to float64's rounding; the forward derivative of a gradient likewise."""
    _check_feed("cpu", F64, which, 1e-12)


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:backend")
@pytest.mark.parametrize("which", [0, 1, 2])
def test_feed_forward_has_its_tangent_on_the_gpu(gpu, which):
    """The torch path twice; sums of at most 30 products in float32, 30 x 2^-24 = 2e-6 of their magnitudes, under the package's 1e-5."""
    _check_feed("cuda", F32, which, 1e-5)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_operators_in_service_refuse_tangents(dev):
    m = make(12, 8, 4, 4, 2, 3, F32, dev=dev)
    s, t, at = m["seq"], m["token"], torch.tensor([0, 12], device=dev)
    weights = dict(conv_weight=m["conv"]["weight"], conv_bias=m["conv"]["bias"], **m["proj"], A=m["A"], Dp=m["Dp"])
    calls = dict(
        conv=lambda x: mamba.mamba_conv_packed(x, at, **m["conv"]),
        conv_weight=lambda w: mamba.mamba_conv_packed(s["x"], at, w),
        ssm=lambda x: mamba.mamba_ssm_packed(x, m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at),
        step=lambda x: mamba.mamba_step(**{**t, "x": x}, **weights),
        step_state=lambda h: mamba.mamba_step(**{**t, "ssm_state": h}, **weights),
    )
    primals = dict(conv=s["x"], conv_weight=m["conv"]["weight"], ssm=s["draw"], step=t["x"], step_state=t["ssm_state"])
    before = t["ssm_state"].clone()
    for name, f in calls.items():
        x = primals[name]
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.func.jvp(f, (x,), (x,))
        with torch.no_grad(), forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
            f(forward_ad.make_dual(x, x))
    assert torch.equal(t["ssm_state"], before)
    with forward_ad.dual_level():  # a level alone asks for nothing
        assert torch.isfinite(calls["conv"](s["x"])[0]).all()
