"""Rotary positions against 64 bits, over layouts, parts of the head, types, strides."""

import math

import pytest
import torch

from latentserve_b200 import rotary

pytestmark = pytest.mark.gpu


def reference(x, cos, sin, positions, interleaved, inverse=False):
    y = x.double().clone()
    r = 2 * cos.shape[1]
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None] * (-1 if inverse else 1)
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., : r // 2], y[..., r // 2: r])
    a, b = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = a, b
    else:
        y[..., : r // 2], y[..., r // 2: r] = a, b
    return y


def check(got, x, cos, sin, positions, interleaved, inverse=False):
    want = reference(x, cos, sin, positions, interleaved, inverse)
    # One rounding of half a step, and two fp32 roundings (2^-24 each) of products of |x| <= top.
    half = torch.finfo(x.dtype).eps / 2
    r = 2 * cos.shape[1]
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    top = float(x.double().abs().max()) * float(cos.abs().max().clamp(min=float(sin.abs().max())))
    err = (got.double() - want).abs()
    assert (err <= half * want.abs() + 3 * 2.0 ** -24 * 2 * top + tiny).all()
    assert torch.equal(got[..., r:], x[..., r:])


def tables(r, n, scaling=None):
    return rotary.rotary_tables(r, n, 1e4, scaling)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,r", [(128, 128), (128, 64), (64, 32), (80, 80), (80, 20), (96, 6), (2, 2), (7, 2), (256, 128)])
def test_layouts_and_types(dtype, interleaved, dim, r):
    g = torch.Generator(device="cuda").manual_seed(dim + r)
    cos, sin = tables(r, 5000)
    for tokens, hq, hk in [(1, 12, 2), (37, 3, 1), (513, 4, 4)]:
        q, k = (torch.randn(tokens, h, dim, device="cuda", generator=g).to(dtype) for h in (hq, hk))
        positions = torch.randint(0, 5000, (tokens,), device="cuda", generator=g)
        qo, ko = rotary.apply_rotary(q, k, cos, sin, positions, interleaved=interleaved)
        check(qo, q, cos, sin, positions, interleaved)
        check(ko, k, cos, sin, positions, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_many_heads_of_many_tokens(interleaved):
    """The variant with several heads a thread, a head count it does not divide."""
    g = torch.Generator(device="cuda").manual_seed(9)
    cos, sin = tables(128, 9000)
    q, k = (torch.randn(9000, h, 128, device="cuda", generator=g).half() for h in (30, 5))
    positions = torch.arange(8999, -1, -1, device="cuda")
    qo, ko = rotary.apply_rotary(q, k, cos, sin, positions, interleaved=interleaved)
    check(qo, q, cos, sin, positions, interleaved)
    check(ko, k, cos, sin, positions, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 3])
def test_views_in_place_and_neighbours(interleaved, offset):
    """Heads of a fused projection rotated in place: the values rows and everything between stay;
    with an odd offset no row is aligned."""
    g = torch.Generator(device="cuda").manual_seed(2)
    cos, sin = tables(48, 100)
    flat = torch.randn(50, 6 * 64 + 11, device="cuda", generator=g).half()
    before = flat.clone()
    heads = flat[:, offset: offset + 6 * 64].view(50, 6, 64)
    q, k = heads[:, :3], heads[:, 3:5]
    positions = torch.arange(50, 100, device="cuda")
    want = [reference(x, cos, sin, positions, interleaved) for x in (q, k)]
    qo, ko = rotary.apply_rotary(q, k, cos, sin, positions, interleaved=interleaved, q_out=q, k_out=k)
    assert qo is q and ko is k
    old = before[:, offset: offset + 6 * 64].view(50, 6, 64)
    check(q.contiguous(), old[:, :3], cos, sin, positions, interleaved)
    check(k.contiguous(), old[:, 3:5], cos, sin, positions, interleaved)
    mask = torch.ones_like(flat, dtype=torch.bool)
    mask[:, offset: offset + 5 * 64] = False
    assert torch.equal(flat[mask], before[mask])
    assert len(want) == 2


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(interleaved):
    """<w, R x> = <R^-1 w, x>: the inverse against the formula's derivative, and there and back."""
    g = torch.Generator(device="cuda").manual_seed(3)
    cos, sin = tables(32, 64)
    x, w = (torch.randn(64, 2, 48, device="cuda", generator=g) for _ in range(2))
    positions = torch.arange(64, device="cuda")
    x64 = x.double().requires_grad_()
    y = reference(x64.detach(), cos, sin, positions, interleaved)
    leaf = x.double().requires_grad_()
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    a, b = (leaf[..., 0:32:2], leaf[..., 1:32:2]) if interleaved else (leaf[..., :16], leaf[..., 16:32])
    wa, wb = (w.double()[..., 0:32:2], w.double()[..., 1:32:2]) if interleaved else (w.double()[..., :16], w.double()[..., 16:32])
    loss = ((a * c - b * s) * wa).sum() + ((b * c + a * s) * wb).sum() + (leaf[..., 32:] * w.double()[..., 32:]).sum()
    loss.backward()
    got, _ = rotary.apply_rotary(w, w[:, :0], cos, sin, positions, interleaved=interleaved, inverse=True)
    assert (got.double() - leaf.grad).abs().max() <= 8 * 2.0 ** -24 * float(w.abs().max()) * 2
    # A difference quotient of a linear function is exact but for rounding.
    i = (5, 1, 3)
    bump = x.double().clone()
    bump[i] += 1.0
    diff = ((reference(bump, cos, sin, positions, interleaved) - y) * w.double()).sum()
    assert abs(float(diff) - float(got[i])) < 1e-5
    there, _ = rotary.apply_rotary(x, x[:, :0], cos, sin, positions, interleaved=interleaved)
    back, _ = rotary.apply_rotary(there, x[:, :0], cos, sin, positions, interleaved=interleaved, inverse=True)
    # cos^2 + sin^2 of tables rounded to 2^-24, and six fp32 roundings.
    assert (back - x).abs().max() <= 12 * 2.0 ** -24 * float(x.abs().max()) * 2


def test_positions_outside_the_tables_are_nan_and_far_ones_exact():
    cos, sin = rotary.rotary_tables(64, 1_000_000, 1e6, {"type": "yarn", "factor": 8.0, "original_max_pos": 32768})
    inv, mag = rotary.rotary_frequencies(64, 1e6, {"type": "yarn", "factor": 8.0, "original_max_pos": 32768})
    x = torch.zeros(4, 1, 96, device="cuda")
    x[..., 0] = 1.0
    x[..., 64:] = 5.0
    positions = torch.tensor([999_999, 1_000_000, -1, 0], device="cuda")
    out, _ = rotary.apply_rotary(x, x, cos, sin, positions)
    assert abs(float(out[0, 0, 0]) - mag * math.cos(999_999 * float(inv[0]))) < 2.0 ** -22
    assert abs(float(out[0, 0, 32]) - mag * math.sin(999_999 * float(inv[0]))) < 2.0 ** -22
    assert out[1:3, 0, :64].isnan().all() and (out[..., 64:] == 5).all() and out[3].isfinite().all()


def test_captured_and_streams():
    g = torch.Generator(device="cuda").manual_seed(5)
    cos, sin = tables(128, 64)
    q, k = (torch.randn(16, h, 128, device="cuda", generator=g).half() for h in (12, 2))
    positions = torch.arange(16, device="cuda")
    rotary.apply_rotary(q, k, cos, sin, positions)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, _ = rotary.apply_rotary(q, k, cos, sin, positions)
    positions += 7
    graph.replay()
    torch.cuda.synchronize()
    check(qo, q, cos, sin, positions, False)


def test_refusals():
    cos, sin = tables(64, 16)
    x = torch.zeros(4, 2, 64, device="cuda")
    p = torch.arange(4, device="cuda")
    good = dict(q=x, k=x, cos=cos, sin=sin, positions=p)
    for bad in [dict(q=x.double()), dict(k=x.half()), dict(k=x[:3]), dict(q=x[..., ::2]), dict(cos=cos.half()),
                dict(sin=sin[:8]), dict(positions=p.int()), dict(positions=p[:3]), dict(positions=p.cpu()), dict(cos=cos.cpu()),
                dict(q=x[..., :32], k=x[..., :32]), dict(q_out=x[:, :1]), dict(k_out=x.half()),
                dict(q_out=x[:, :1].expand(4, 2, 64)), dict(q=x[0])]:
        a = good | bad
        with pytest.raises(ValueError):
            rotary.apply_rotary(a.pop("q"), a.pop("k"), a.pop("cos"), a.pop("sin"), a.pop("positions"), **a)
    no_q, only_k = rotary.apply_rotary(x[:, :0], x + 1, cos, sin, p)
    assert no_q.shape == (4, 0, 64)
    check(only_k, x + 1, cos, sin, p, False)
    row = torch.ones(1, 1, 64, device="cuda")
    wide, _ = rotary.apply_rotary(row.expand(4, 2, 64), x, cos, sin, p)              # broadcast inputs
    check(wide, torch.ones(4, 2, 64, device="cuda"), cos, sin, p, False)
    none, _ = rotary.apply_rotary(x[:0], x[:0], cos, sin, p[:0])
    assert none.shape == (0, 2, 64)
