"""Precision of the softmax weights in the shared-prefix decode, where nothing but them is rounded: outputs in fp32."""
import math

import pytest
import torch

from test_shared_prefix_gpu import D, Batch

pytestmark = pytest.mark.gpu

LAYOUTS = [([1, 1], 0, 70), ([1, 1], 0, 2), ([12], 2, 10), ([40], 2, 10), ([100], 2, 10), ([130], 3, 1)]


def two_levels(sizes, prefix, own, gap, vd, qd):
    """A first token `gap` (log2) above the others, which are all alike, with V = 0: the output is (1 - w_0) times the mean V of
    the others, so that an error of their one weight does not average out."""
    b = Batch(sizes, [prefix] * len(sizes), [own], 1, 1, qd=qd, vd=vd, seed=len(sizes))
    u = torch.randn(D, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda").to(qd).float()
    b.q = u.expand(b.B, 1, 1, D).to(qd).contiguous()
    b.k.zero_()
    b.r.zero_()
    b.v = (b.v.abs() + 0.5).to(vd)
    for i in range(b.B) if prefix == 0 else [0]:
        page = int(b.table[i, 0])
        k = gap * math.log(2) * math.sqrt(D) * u / u.square().sum()
        b.k[page, 0, 0] = k.to(b.k.dtype)
        b.r[page, 0, 0] = (k - b.k[page, 0, 0].float()).to(b.k.dtype)
        b.v[page, 0] = 0
    return b


def allowed(b, weight):
    """What an output may be off in fp32.  A weight may be off by `weight` of itself; a score by its fp32 sums of at most 1536
    products and by q in pieces (2^-18 of its largest element); exp2 and the sums by 2^-20."""
    out, _, lse = b.exact()
    n, d = b.lens[0], (b.q[0, 0, 0].double() @ (b.k.double() + b.r.double())[int(b.table[0, 0]), 0, 0]).abs() / math.sqrt(D)
    k1 = (b.k.double() + b.r.double())[int(b.table[0, 0]), 0, 0].abs().sum()
    score = float(1536 * 2.0 ** -24 * d * 4 + 2.0 ** -18 * b.q.abs().max().double() * k1 / math.sqrt(D))
    return out, (weight + 2 * score + 2.0 ** -20) * out.abs() + 2.0 ** -24, lse


@pytest.mark.parametrize("gap", [0.37, 1.71])
@pytest.mark.parametrize("sizes,prefix,own", LAYOUTS)
@pytest.mark.parametrize("vd,weight", [(torch.bfloat16, 2.0 ** -16), (torch.float16, 2.0 ** -12)])
def test_weights(sizes, prefix, own, gap, vd, weight):
    """bfloat16: cut to eight bits and the rest (below 2^-7) rounded to eight, 2^-16; float16: eleven bits, 2^-12."""
    b = two_levels(sizes, prefix, own, gap, vd, torch.float32)
    out, tol, _ = allowed(b, weight)
    off = (b.call().double() - out).abs()
    assert bool((off <= tol).all()), f"{float((off / out.abs().clamp(min=1e-9)).max()):.3g}, {float((off / tol).max()):.3g} of what is allowed"


@pytest.mark.parametrize("sizes,prefix,own", LAYOUTS)
def test_partials_of_bfloat16_calls(sizes, prefix, own):
    """Partials are fp32 and are merged further: they have the weights' sixteen bits, whatever the output's type."""
    b = two_levels(sizes, prefix, own, 0.37, torch.bfloat16, torch.bfloat16)
    out, tol, lse = allowed(b, 2.0 ** -16)
    part = torch.empty(b.B, 1, D + 1, device="cuda")
    got = b.call(partial_out=part)
    assert bool(((part[..., :D].double() - out).abs() <= tol).all())
    assert float((part[..., D].double() - lse).abs().max()) <= 2.0 ** -14
    assert torch.equal(got, part[..., :D].to(torch.bfloat16))


@pytest.mark.parametrize("vd", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,prefix,own", LAYOUTS)
def test_an_infinite_value_of_the_first_token(sizes, prefix, own, vd):
    """Infinity times a weight is infinity, the largest weight's too."""
    b = two_levels(sizes, prefix, own, 0.37, vd, torch.bfloat16)
    for i in range(b.B):
        b.v[int(b.table[i, 0]), 0, 0, 5] = math.inf
        b.v[int(b.table[i, 0]), 0, 0, 6] = -math.inf
    got = b.call()
    assert bool((got[..., 5] == math.inf).all()) and bool((got[..., 6] == -math.inf).all())
    got[..., 5:7] = 0
    assert bool(torch.isfinite(got).all())
