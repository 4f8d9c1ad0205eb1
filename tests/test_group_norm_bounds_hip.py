"""Group norm against 64 bits with bounds from the way that each size takes, on inputs that show a place that is left out.

u = 2^-24; a sum by a chain and trees of at most L additions is off by L u of its terms' magnitudes.  A thread adds its places
one after the other, then eight columns (3), the lanes of a wave that have the same columns (log2), rows and columns that LDS holds
of the group, the lanes that do so (log2).  Of several launches: the first takes a thread's places in batches of eight, whose mean
is joined to the one before it in two roundings of the sum so far (16 + 2 a batch, with the rounding of the batch's own parts), the
second adds a group's parts by lanes, as differences from the first one's mean: those are at most the group's mean magnitude and that
of the part where it is largest.  Every place of a part, a turn, a row of column sums is one addition in dw and db.

The deviation is off by its own (L + 4) u and by what the mean is off by, beside it.  From there on as in test_group_norm_hip.py.

Inputs: few places, beside the borders of parts, threads and samples, have values of 2^12 and gradients of 2^6 where the others are
normal numbers.  Their squares are nearly all of the variance, so that any of them that is left out, or counted twice, changes every
output by several per cent, in 16 bits too: test_a_lost_place_is_seen, on the CPU.
"""
import math

import pytest
import torch

from test_dense_hip import E32, TINY, _act, _slope, _u
from test_group_norm_hip import TYPES, _inputs, _plan, _run

SIZES = [(1, 40000, 8, 2), (1, 30000, 2, 1), (2, 9000, 33, 3), (1, 4096, 512, 32), (5, 777, 330, 11), (1, 5000, 24, 24),
         (2, 600, 1030, 2), (1, 9001, 40, 1), (3, 40, 9000, 2), (2, 1000, 128, 8), (9, 256, 256, 8), (2, 100, 1000, 1), (7, 13, 48, 3)]


def _over(a, b):
    return -(-a // b)


def _log2(v):
    return max(v, 1).bit_length() - 1


class Way:
    """How a size is worked on: places of a part and of a thread, and the lengths of its sums."""

    def __init__(self, dt, n, p, channels, groups, back):
        threads, held, gpt, tiles, parts, sub, slots, span = _plan(dt, n, p, channels, groups, back)
        c, self.held, self.parts = channels // groups, threads > 0, parts
        cols = gpt * c
        if sub > 1:
            cols = _over(_over(c, _over(c, 512)), 8) * 8
            assert _over(c, cols) == sub
        self.cols = cols
        wp = 1
        while 8 * wp < cols:
            wp *= 2
        nt = threads or 256
        self.down = (span if threads else nt) // wp  # threads down a part's places
        if threads:
            self.rows, self.each = p, held
        else:
            step, cus = (4 if back else 8) * (256 // wp), torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 256
            self.rows = min(p, _over(_over(p, _over(2 * cus, n * tiles)), step) * step)
            assert _over(p, self.rows) == parts
            self.each = _over(self.rows, self.down)
        per, wave = nt // span, min(span, 64)
        lds = 1 if per > 1 else nt // 64 if wp < 64 else nt // wp
        def lanes(items):
            t = 64
            while t > 1 and t * items > nt:
                t //= 2
            return t
        t, inside = lanes(per * gpt), cols if sub > 1 else c
        across = 3 + _log2(_over(wave, wp)) + lds * _over(inside, t) + _log2(t)
        of_parts = _over(parts * sub, lanes(gpt)) + _log2(lanes(gpt))
        if threads:
            self.mean, self.sums = self.each + across + 4, self.each + across + 4
            self.columns = self.each + _over(n, slots * per) + 6 + max(nt // 64, lds) + _over(slots, 32) + 32
        else:
            self.mean, self.sums = 16 + 2 * _over(self.each, 8) + across + of_parts + 8, self.each + across + of_parts + 6
            self.columns = self.each + 6 + max(nt // 64, lds) + _over(n * parts, slots) + _over(slots, 64) + 8 + 16


def _places(p, *ways):
    """Places beside borders: of the sample, its parts, and a thread's batches."""
    some = {0, p // 3, p - 1}
    for w in ways:
        some |= {w.down - 1, w.down, w.rows - 1, w.rows, (w.parts - 1) * w.rows, (w.parts - 1) * w.rows - 1}
    return sorted(i for i in some if 0 <= i < p)


def _marked(n, p, c, dt, places, seed):
    x, w, b, g = _inputs(n, p, c, dt, seed=seed)
    x[:, places] = 2.0 ** 12
    g[:, places] = 2.0 ** 6  # (dw stays within fp16)
    return x, w.abs() + 0.25, b, g


def _sums(x, w, b, g, groups, act, eps=1e-5, lost=None):
    """Outputs and what their bounds are made of, in 64 bits; lost: (sample, place) that the forward's sums leave out, then, with
    the right statistics, the backward's."""
    n, p, c = x.shape
    x, g = (t.double().view(n, p, groups, -1) for t in (x, g))
    w, b = (t.double().view(groups, -1) for t in (w, b))
    keep = torch.ones(n, p, 1, 1, dtype=torch.float64, device=x.device)
    if lost:
        keep[lost] = 0
    over = lambda t: t.mean((1, 3), keepdim=True)

    def norm(k):
        mean = over(k * x)
        rstd = (over(k * (x - mean).square()) + eps).rsqrt()
        return rstd, (x - mean) * rstd

    y = _act(norm(keep)[1] * w + b, act)
    rstd, nx = norm(1)
    z = nx * w + b
    u = g * _slope(z, act)
    m0, m1 = over(keep * u * w), over(keep * u * w * nx)
    dx = rstd * (u * w - m0 - nx * m1)
    return {"x": x, "g": g, "w": w, "b": b, "rstd": rstd, "nx": nx, "z": z, "u": u, "m0": m0, "m1": m1, "over": over,
            "out": (y, dx, (keep * u * nx).sum((0, 1)), (keep * u).sum((0, 1)))}


def _bounds(s, act, forward, back):
    n, p, groups, c = s["x"].shape
    over, rstd, nx, z, w, u, g = (s[k] for k in ("over", "rstd", "nx", "z", "w", "u", "g"))
    size = over(s["x"].abs())
    if not forward.held:  # and the largest of a part's
        pieces = [t.abs().mean((1, 3), keepdim=True) for q in s["x"].split(forward.rows, 1) for t in q.split(min(c, forward.cols), 3)]
        size = size + torch.stack(pieces).amax(0)
    em = forward.mean * E32 * size
    en = rstd * em + nx.abs() * ((forward.mean + 8) * E32 + rstd * em)
    ez = w.abs() * en + 2 * E32 * (z.abs() + s["b"].abs())
    y = _act(z, act)
    by = 1.13 * ez + 2.0 ** -20 * (1 + z.abs()) * y.abs()
    eu = 0 * g if act == "none" else g.abs() * (0.8 * ez + 2.0 ** -20 * (1 + z.abs()))
    uw, euw = u * w, (eu + E32 * u.abs()) * w.abs()
    L = back.sums * E32
    e0 = over(euw) + L * over(uw.abs())
    e1 = over(euw * nx.abs() + uw.abs() * en) + L * over((uw * nx).abs())
    m0, m1, dx = s["m0"], s["m1"], s["out"][1]
    bx = rstd * (euw + e0 + en * m1.abs() + nx.abs() * e1 + 4 * E32 * (uw.abs() + m0.abs() + (nx * m1).abs())) + dx.abs() * ((forward.mean + 8) * E32 + rstd * em)
    every = back.columns * E32
    bw = (eu * nx.abs() + u.abs() * en).sum((0, 1)) + every * (u * nx).abs().sum((0, 1))
    bb = eu.sum((0, 1)) + every * u.abs().sum((0, 1))
    return by, bx, bw, bb


def _beyond(got, ref, bound, dt):
    """By how much of its bound the worst value is off."""
    lim = bound + _u(dt) * ref.abs() + TINY[dt]
    return ((got.double().reshape(ref.shape) - ref).abs() / lim.clamp_min(1e-300)).max().item()


def _ways(dt, n, p, c, groups):
    return Way(dt, n, p, c, groups, False), Way(dt, n, p, c, groups, True)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,p,c,groups", SIZES)
def test_a_lost_place_is_seen(n, p, c, groups, dt):
    """Each marked place, left out of the last sample's sums, takes every output beyond its bound."""
    ways = _ways(dt, n, p, c, groups)
    places = _places(p, *ways)
    x, w, b, g = _marked(n, p, c, dt, places, seed=n + c)
    s = _sums(x, w, b, g, groups, "silu")
    bounds = _bounds(s, "silu", *ways)
    assert all(_beyond(v.to(dt), v, e, dt) <= 1 for v, e in zip(s["out"], bounds))
    for place in places:
        off = _sums(x, w, b, g, groups, "silu", lost=(n - 1, place))["out"]
        for name, t, ref, bound in zip(("y", "dx", "dw", "db"), off, s["out"], bounds):
            assert _beyond(t, ref, bound, dt) > 2, (name, place, _beyond(t, ref, bound, dt))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,p,c,groups", SIZES)
def test_marked_places(n, p, c, groups, dt, device):
    ways = _ways(dt, n, p, c, groups)
    x, w, b, g = (t.to(device) for t in _marked(n, p, c, dt, _places(p, *ways), seed=n + c))
    for act in ("none", "silu", "gelu"):
        s = _sums(x, w, b, g, groups, act)
        for name, t, ref, bound in zip(("y", "dx", "dw", "db"), _run(x, w, b, g, groups, act), s["out"], _bounds(s, act, *ways)):
            assert _beyond(t, ref, bound, dt) <= 1 + 1e-6, (name, act)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,p,c,groups", SIZES + [(64, 50, 256, 256), (4, 300, 4096, 1), (300, 1, 512, 16), (5000, 1, 128, 8), (4099, 1, 7, 7), (1, 20000, 600, 1)])
def test_normal_numbers(n, p, c, groups, dt, device):
    ways = _ways(dt, n, p, c, groups)
    x, w, b, g = (t.to(device) for t in _inputs(n, p, c, dt, seed=n + c))
    for act in ("none", "silu", "gelu"):
        s = _sums(x, w, b, g, groups, act)
        for name, t, ref, bound in zip(("y", "dx", "dw", "db"), _run(x, w, b, g, groups, act), s["out"], _bounds(s, act, *ways)):
            assert _beyond(t, ref, bound, dt) <= 1 + 1e-6, (name, act)
