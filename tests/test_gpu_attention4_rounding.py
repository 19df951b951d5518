"""How far attention over a cache of 4 bits is off its formulas: as far as the roundings that its kernels are made with, and no further.

A rounding to f16 is off by at most 2^-11 of the value, and at random by r = 2^-11 sqrt(E[1 / m^2] / 3) = 2.07e-4 of it in the mean of squares, where m is a mantissa, spread evenly by its logarithm
(E = 3 / (8 ln 2)); to bf16 by 8 r.  The roundings of a row's terms meet in their sum as their squares do, as the terms themselves do, so each counts once for the output:

  streaming kernel   weights, weights times scales (beside the middle of the codes where the outputs are f16), outputs: sqrt(3) r for f16
  tensor cores       values, weights, outputs, and keys, which move a score by r times the size of a query's value: sqrt(3 + size^2) r

A mantissa's spread is not quite even: a quarter more than that is allowed.  Products rounded beside code zero, as they are without what is given back to the middle of the codes, count with the codes'
size instead of their spread, 8.3 to 3.6 for normal values in groups of 32: sqrt(2 + 5.3) r, half more than the streaming kernel's."""
import math

import pytest


torch = pytest.importorskip("torch")
from test_gpu_attention4 import forward  # noqa: E402
from test_gpu_kv4 import Cache4, backend  # noqa: E402, F401

pytestmark = pytest.mark.gpu
R16 = 2.0 ** -11 * math.sqrt(3 / (8 * math.log(2)) / 3)


def spread(c):
    """What the outputs are off by of their size, both in the mean of squares."""
    off = size = 0.0
    for i, (n, k) in enumerate(c.lens):
        keys, values = (c.held(x, c.places(i)).transpose(0, 1) for x in (True, False))
        q = c.q[c.starts[i]:c.starts[i + 1]].double().view(n, c.hk, c.hq // c.hk, c.d).permute(1, 2, 0, 3)
        s = torch.einsum("hgnd,htd->hgnt", q, keys) * c.d ** -0.5
        hidden = torch.arange(k, device="cuda") > torch.arange(k - n, k, device="cuda")[:, None]
        want = torch.einsum("hgnt,htd->hgnd", s.masked_fill(hidden, -math.inf).softmax(3), values)
        got = c.out[c.starts[i]:c.starts[i + 1]].double().view(n, c.hk, c.hq // c.hk, c.d).permute(1, 2, 0, 3)
        off, size = off + (got - want).square().sum().item(), size + want.square().sum().item()
    return math.sqrt(off / size)


SHAPES = [(64, 32), (64, 64), (96, 32), (96, 64), (128, 32), (128, 64), (192, 32), (192, 64), (256, 32), (256, 64)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("group_heads", [4, 16])
@pytest.mark.parametrize("d,group", SHAPES)
def test_spread_of_single_tokens(backend, d, group, group_heads, kind):  # noqa: F811
    c = Cache4([(1, k) for k in (2500, 3000, 4000, 2000, 2700, 3100, 2999, 2048)], 2 * group_heads, 2, d, kind, 16, group).fill().install(backend)
    forward(backend, c)
    out = 8 * R16 if kind == "bf16" else R16
    # bf16: nothing is given back, so products count with the codes' size; groups of 64 have a wider range, and codes nearer to their middle
    assert spread(c) <= 1.25 * math.hypot(out, math.sqrt(2.0 if kind == "f16" else 7.3) * R16)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1.0, 2.0])
@pytest.mark.parametrize("d,group", [(64, 32), (96, 64), (128, 32), (192, 32), (256, 64)])
def test_spread_of_chunks(backend, d, group, size, kind):  # noqa: F811
    c = Cache4([(200, 3000)], 8, 2, d, kind, 16, group).fill().install(backend)
    c.q.mul_(size)
    forward(backend, c)
    out = 8 * R16 if kind == "bf16" else R16
    assert spread(c) <= 1.25 * math.hypot(out, math.sqrt(2 + size * size) * R16)


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("heads", [4, 16])
@pytest.mark.parametrize("d,group", SHAPES)
def test_what_products_lose_is_given_back(backend, d, group, heads, page):  # noqa: F811
    """Every chunk of 16 tokens has one key of score ln(4 / 3) and fifteen of zero, so that the weights are 2^10 and 3/4 of that.  A scale's mantissa is 1 + t / 1024 with odd t, so that its
    product with 3/4 lies in the middle between two f16 numbers and loses half a step, up or down by t, 0.5 / 1540 of it.  All codes are 8 and the minimum about -7 scales, so a value is about
    one scale: the loss counts 8 times where it is not given back, 0.0024 of a value, and half where it is.

    Bound, of a value: the output's rounding, 2^-11; half of the loss, 0.5 * 0.5 / 1540; the weights, whose key is an f16 number, moved by at most 2^-12 of ln(4 / 3), in the numerator as well as
    rounded, 2^-13; sums in 32 bits, 2^-18 of the eight scales that cancel."""
    n = 1600
    c = Cache4([(1, n)], heads, 1, d, "f16", page, group)
    c.q.fill_(1.0)
    keys = torch.zeros((n, 1, d), device="cuda")
    groups = -(-d // group)
    at, none = c.places(0), torch.zeros((n, 1, groups), dtype=torch.float16, device="cuda")
    score = none.clone()
    score[::16] = math.log(4 / 3) / math.sqrt(d)
    c.put(True, at, keys, none, score)
    scale = torch.tensor([(1 + t / 1024) * 2.0 ** -(3 + i % 3) for i, t in enumerate((1, 3, 5, 7, 3, 9, 11, 1))][:groups], dtype=torch.float16, device="cuda")
    least = (-7 * scale.double()).half()
    c.put(False, at, torch.full((n, 1, d), 8.0, device="cuda"), scale.expand(n, 1, -1), least.expand(n, 1, -1))
    c.install(backend)
    forward(backend, c)
    of = torch.arange(d, device="cuda") // group
    want = (8 * scale.double() + least.double())[of]
    bound = (2.0 ** -11 + 2.0 ** -13) * want.abs() + (0.25 / 1540 + 8 * 2.0 ** -18) * scale.double()[of]
    off = ((c.out.double().view(heads, d) - want).abs() / bound).max().item()
    assert off <= 1.0, off
