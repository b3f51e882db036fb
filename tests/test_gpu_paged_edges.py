"""Paged-cache operators on the MI355X where a rule or a type reaches its edge: probabilities far below a row's largest,
tables wider than their sequences, gradients, caches without pages, keys cut where tiles outnumber places, pages that
refill a wave's window.  Plain forms and bounds: tests/paged_ref.py."""
import math

import pytest
import torch

from tests import paged_ref as R
from tests.test_gpu_paged import check, gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def ops():
    from ospo_amd import ops as _ops
    return _ops


def fill_seq(s, b, total, page, k, v):
    """Positions 0 .. total - 1 of sequence b from k, v [total, hk, d]."""
    j = torch.arange(total, device=DEV)
    p = s["table"][b].long()[j // page]
    s["kc"][p, :, j % page], s["vc"][p, :, j % page] = k, v


@pytest.mark.parametrize("new,total,gap", [(1, 600, 18.5), (1, 3000, 18.5), (1, 600, 14.484375), (5, 600, 14.484375),
                                           (130, 600, 14.484375), (130, 3000, 14.484375)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_small_probabilities_keep_their_sum(new, total, gap, d, dtype):
    """A first key that takes nearly all of a row and whose value is zero: the output is what is left for all others,
    each with e^-gap of its probability (2^-26.7 and 2^-20.9: in fp16 zero, and a subnormal with 5 % of rounding).

    Bound: the others' scores are equal and exact, so their probability is off by the exponent's fp32 rounding (2^-24 of
    at most 64, times ln 2), exp2's last bit and its own rounding h; sums of kv terms by 2 kv u; no term in the row's
    largest probability."""
    hq, hk, page = 4, 2, 16
    s = R.build([new], [total], hq=hq, hk=hk, d=d, page=page, dtype=dtype, seed=21, device=DEV)
    g = gen(22)
    k = torch.randn(total, hk, d, generator=g, device=DEV)
    v = 64 + 8 * torch.randn(total, hk, d, generator=g, device=DEV)
    k[:, :, 0], k[0, :, 0], v[0] = 0.0, 1.0, 0.0
    fill_seq(s, 0, total, page, k.to(dtype), v.to(dtype))
    gap = float(torch.tensor(gap).to(dtype))
    s["q"].zero_()
    s["q"][:, :, 0] = gap
    out = ops().paged_attn(s["q"], s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], 1.0)
    h, u = R.HALF[dtype], 2.0 ** -24
    vd = v.to(dtype).double()
    for r in range(new):
        kv = total - new + r + 1
        rest = math.exp(-gap) * vd[1:kv].sum(0) / (1 + (kv - 1) * math.exp(-gap))  # [hk, d]
        ref = rest.repeat_interleave(hq // hk, 0)
        ok, worst = R.within(out[r], ref, (h + 2 * kv * u + 2.0 ** -17) * ref.abs(), dtype)
        assert ok, (r, worst)


# ---------------------------------------------------------------- gradients
def turn(x, cos, sin, il):
    """The formula in elementary 64-bit operations that autograd follows."""
    half = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if il else (x[..., :half], x[..., half:2 * half])
    a, b = a * c - b * s, b * c + a * s
    y = torch.stack([a, b], -1).flatten(-2) if il else torch.cat([a, b], -1)
    return torch.cat([y, x[..., 2 * half:]], -1)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("hk", [0, 2])
def test_rotary_records_gradients(dtype, il, back, hk):
    """Against the formula's gradient: each value is two products and a sum in fp32, rounded once (rotate's bound)."""
    n, hq, d, rot = 33, 5, 64, 48
    g = gen(31)
    q = torch.randn(n, hq, d, generator=g, device=DEV).to(dtype).requires_grad_()
    k = torch.randn(n, hk, d, generator=g, device=DEV).to(dtype).requires_grad_() if hk else None
    pos = torch.randint(0, 512, (n,), generator=g, device=DEV).int()
    tab = ops().rotary_tables(512, rot, 10000.0, DEV)
    got = ops().rotary(q, k, pos, tab, interleaved=il, backward=back)
    with torch.no_grad():
        plain = ops().rotary(q, k, pos, tab, interleaved=il, backward=back)
    cos, sin = (t[pos.long()] for t in tab)
    for x, y, p in ((q, got[0], plain[0]), (k, got[1], plain[1])):
        if x is None:
            assert y is None
            continue
        assert torch.equal(y, p) and y.requires_grad
        dy = torch.randn(x.shape, generator=g, device=DEV).to(dtype)
        x64 = x.detach().double().requires_grad_()
        turn(x64, cos, -sin if back else sin, il).backward(dy.double())
        (dx,) = torch.autograd.grad(y, x, dy, retain_graph=True)
        _, tol = R.rotate(dy, torch.atan2(sin.double(), cos.double()), 1.0, il)
        ok, worst = R.within(dx, x64.grad, tol, dtype)
        assert ok, worst


def test_rotary_gradients_of_one_output_expanded_and_twice():
    n, d = 9, 32
    g = gen(32)
    q, k = (torch.randn(n, h, d, generator=g, device=DEV, requires_grad=True) for h in (4, 2))
    pos = torch.arange(n, device=DEV).int()
    tab = ops().rotary_tables(16, d, 10000.0, DEV)
    qo, ko = ops().rotary(q, k, pos, tab)
    one = torch.ones(n, 2, d, device=DEV)
    want = ops().rotary(one, None, pos, tab, backward=True)[0]
    ko.sum().backward()  # the gradient of a sum comes expanded; q has no part in it
    assert q.grad is None and torch.equal(k.grad, want)
    # one of two that wants a gradient; two in one backward pass
    q2 = q.detach()
    qo, ko = ops().rotary(q2, k, pos, tab)
    (dk,) = torch.autograd.grad(ko.sum() + (qo * qo).sum(), k)
    assert torch.equal(dk, want)
    # the gradient's gradient: f = sum (R q)^2 w, df/dq = 2 R^T (w R q), its derivative along u is 2 R^T (w R u)
    w, u = (torch.randn(n, 4, d, generator=g, device=DEV) for _ in range(2))
    y, _ = ops().rotary(q, None, pos, tab)
    (dq,) = torch.autograd.grad((y * y * w).sum(), q, create_graph=True)
    (h,) = torch.autograd.grad((dq * u).sum(), q)
    with torch.no_grad():
        ru = ops().rotary(u, None, pos, tab)[0]
        ref = 2 * ops().rotary(w * ru, None, pos, tab, backward=True)[0]
    # each of the two rotations and two products rounds its values once: 8 half steps of |w| |u| sums of two
    assert float((h - ref).abs().max()) <= 8 * 2.0 ** -24 * 2 * 2 * float((w.abs().max() * u.abs().max()) * 2)


def test_rotary_gradient_matches_differences_through_autograd():
    """Along a direction u: the map is linear, so a difference over a step of 1 is exact up to rounding."""
    n, h, d, rot = 17, 3, 64, 40
    g = gen(33)
    x, u, dy = (torch.randn(n, h, d, generator=g, device=DEV) for _ in range(3))
    pos = torch.arange(n, device=DEV).int()
    tab = ops().rotary_tables(64, rot, 10000.0, DEV, {"type": "ntk", "factor": 4.0})
    x.requires_grad_()
    y, _ = ops().rotary(x, None, pos, tab, interleaved=True)
    y.backward(dy)
    with torch.no_grad():
        z, _ = ops().rotary(x + u, None, pos, tab, interleaved=True)
        lhs = (dy.double() * (z.double() - y.double())).sum()
        rhs = (x.grad.double() * ((x + u) - x).double()).sum()
        lim = 8 * 2.0 ** -24 * float((dy.abs().double() * (y.abs() + z.abs() + 1)).sum())
    assert abs(float(lhs - rhs)) <= lim


def test_rotary_gradient_captured():
    """Forward and backward of a step in one graph, replayed with other values beside eager work."""
    n, d = 40, 64
    pos = torch.arange(n, device=DEV).int()
    tab = ops().rotary_tables(64, d, 10000.0, DEV)
    x = torch.zeros(n, 4, d, device=DEV, requires_grad=True)
    dy = torch.zeros(n, 4, d, device=DEV)

    def step():
        y, _ = ops().rotary(x, None, pos, tab)
        return torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx = step()
    for i in range(3):
        dy.copy_(torch.randn(n, 4, d, generator=gen(40 + i), device=DEV))
        pos.copy_((torch.arange(n, device=DEV) + i) % 64)
        graph.replay()
        want = ops().rotary(dy, None, pos, tab, backward=True)[0]
        torch.cuda.synchronize()
        assert torch.equal(dx, want), i


# ------------------------------------------------------- caches without pages
@pytest.mark.parametrize("pages,columns", [(0, 3), (4, 0), (0, 0)])
def test_cache_without_pages(pages, columns):
    """No row is stored, every query is turned, and a row of the attention sees nothing."""
    n, hq, hk, d = 5, 4, 2, 64
    g = gen(51)
    q, k, v = (torch.randn(n, h, d, generator=g, device=DEV).to(BF) for h in (hq, hk, hk))
    kc = torch.randn(pages, hk, 16, d, generator=g, device=DEV).to(BF)
    vc = kc.clone()
    table = torch.zeros(2, columns, dtype=torch.int32, device=DEV)
    q_start = torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV)
    kv_len = torch.tensor([9, 3], dtype=torch.int32, device=DEV)
    tab = ops().rotary_tables(16, d, 10000.0, DEV)
    q_out = ops().paged_append(k, v, kc, vc, table, q_start, kv_len, q=q, rope=tab)
    pos = torch.tensor([7, 8, 0, 1, 2], dtype=torch.int32, device=DEV)
    assert torch.equal(q_out, ops().rotary(q, None, pos, tab)[0])
    assert torch.equal(kc, vc)  # (as they were)
    lse = torch.zeros(n, hq, device=DEV)
    out = ops().paged_attn(q_out, kc, vc, table, q_start, kv_len, 0.1, lse=lse)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


# ---------------------------------------------------------- cutting the keys
@pytest.mark.parametrize("new,total,hq,hk", [
    ([1] * 32, [24 + 19 * i for i in range(32)], 32, 32),  # a sampling step: more tiles than places, nothing to cut
    ([200, 90, 150], [200, 300, 150], 8, 8),               # many rows, too short to cut
    ([1, 1], [5000, 300], 8, 2),                           # long enough
    ([200, 90, 1], [200, 6000, 150], 8, 4)])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
def test_a_wider_table_cuts_no_more(new, total, hq, hk, d, dtype):
    """A table with room for longer sequences (a captured step's) gives the same bits: its keys are cut by the lengths
    on the device, where some sequence is long enough."""
    s = R.build(new, total, hq=hq, hk=hk, d=d, page=16, dtype=dtype, seed=61, device=DEV)
    want, wl = check(s, d ** -0.5)
    wide = torch.zeros(len(new), 2048, dtype=torch.int32, device=DEV)
    wide[:, : s["table"].shape[1]] = s["table"]
    got, gl = check(dict(s, table=wide), d ** -0.5)
    assert torch.equal(got, want) and torch.equal(gl, wl)
