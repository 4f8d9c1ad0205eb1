"""The gradients of layers that keep their activations in 8 bits, beside differences of the loss, one tensor at a time and along the
gradient's own signs, so that what is compared is the sum of its magnitudes.

(L(t + e d) - L(t - e d)) / 2 e of the fp32 layer, whose argument moves by e q, q = d W^T, x d^T or d: it is off by e^2 / 6 of the
third derivative (at most 1) times |q|^3, and by the fp32 results' rounding, at most 2^-20 (1 + |y|), over e.  The gradients are those
at the kept values: dz is off by 0.8 times half a step of the argument (the second derivative of gelu is at most 0.8, of silu 0.5)
beside its own rounding to the type, dw by |dz| (at most 1.13 |c|) times half a step of x more, and the results by their rounding.  Every
bound is less than half of what it bounds: gradients that are negated, doubled or zero are beyond it."""
import pytest
import torch

from test_dense_hip import HALVES, _act, _inputs, _slope, _u
from test_dense_packed_hip import _pack, _unpack

TYPES = HALVES + [torch.float32]
STEP = 2.0 ** -7
SIZES = (24, 40, 36)


def _halves(v):
    """Half a step of each value's block."""
    return torch.exp2(_pack(v)[1].double() - 134).repeat_interleave(32, -1)[:, :v.shape[1]]


def _case(dt, act, name):
    """Inputs, the direction, and by how much <gradient, direction> and the difference may be apart; in 64 bits on the CPU."""
    x, w, b, _, c = (t.double() for t in _inputs(*SIZES, dt, seed=9))
    z = x @ w.T + b
    dz, u = c * _slope(z, act), _u(dt)
    grad = {"x": dz @ w, "w": dz.T @ x, "b": dz.sum(0)}[name]
    d = grad.sign()
    q = {"x": lambda: d @ w.T, "w": lambda: x @ d.T, "b": lambda: d.expand_as(z)}[name]().abs()
    off = 0.8 * c.abs() * 1.1 * _halves(z.float()) + (2.0 ** -18 * (1 + z.abs()) + 1.13 * u) * c.abs()  # dz
    kept = {"x": lambda: off @ w.abs(), "w": lambda: off.T @ (x.abs() + _halves(x)) + (1.13 * c.abs()).T @ _halves(x), "b": lambda: off.sum(0)}[name]()
    differences = STEP ** 2 / 6 * (c.abs() * q ** 3).sum() + 2.0 ** -20 * (c.abs() * (1 + _act(z, act).abs())).sum() / STEP
    bound = (kept + (u + 2.0 ** -16) * (grad.abs() + kept)).sum() + differences
    return (x, w, b, c), d, grad, bound.item()


def _difference(layer, t, d, c, name):
    def loss(e):
        a = {k: v + e * d if k == name else v for k, v in t.items()}
        return (layer(a["x"], a["w"], a["b"]).double() * c).sum().item()

    return (loss(STEP) - loss(-STEP)) / (2 * STEP)


@pytest.mark.parametrize("name", ["x", "w", "b"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", TYPES)
def test_what_the_bound_refuses(dt, act, name):
    (x, w, b, c), d, grad, bound = _case(dt, act, name)
    diff = _difference(lambda *a: _act(a[0] @ a[1].T + a[2], act), {"x": x, "w": w, "b": b}, d, c, name)
    dz = c * _slope(_unpack(*_pack((x @ w.T + b).float()), dt), act)
    kept = {"x": lambda: dz @ w, "w": lambda: dz.T @ _unpack(*_pack(x), dt), "b": lambda: dz.sum(0)}[name]()
    assert abs((kept * d).sum() - diff) <= bound and abs((grad * d).sum() - diff) <= bound
    assert bound < 0.5 * diff
    for wrong in (-kept, 2 * kept, 0 * kept):
        assert abs((wrong * d).sum() - diff) > bound


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["x", "w", "b"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", TYPES)
def test_gradient_against_differences(dt, act, name, device):
    from maloq_amd.dense import linear_act
    (x, w, b, c), d, _, bound = _case(dt, act, name)
    x, w, b, c, d = (t.to(device) for t in (x, w, b, c, d))
    with torch.no_grad():
        diff = _difference(lambda *a: linear_act(*(t.float() for t in a), act=act), {"x": x, "w": w, "b": b}, d, c, name)
    leaves = {k: v.to(dt).requires_grad_() for k, v in (("x", x), ("w", w), ("b", b))}
    y = linear_act(leaves["x"], leaves["w"], leaves["b"], act=act, checkpoint=torch.int8)
    got, = torch.autograd.grad(y, leaves[name], c.to(dt))
    assert abs((got.double() * d).sum().item() - diff) <= bound
