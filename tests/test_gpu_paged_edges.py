"""Paged-cache operators on the MI355X where a rule or a type reaches its edge: probabilities far below a row's largest,
tables wider than their sequences, gradients, caches without pages, keys cut where tiles outnumber places, pages that
refill a wave's window.  Plain forms and bounds: tests/paged_ref.py."""
import math

import pytest
import torch

from tests import paged_ref as R
from tests.paged_cases import WAYS, WINDOWS
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


def spot_check(c, d, dtype, seed):
    """A batch against the plain form, heads and sequences thinned where the batch is large (each head and each sequence is
    an item of its own): the first and last sequences and every fifth, the first, middle and last key/value heads."""
    new, kv, hq, hk, page = c["new"], c["kv"], c["hq"], c["hk"], c["page"]
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = [-(-t // page) for t in kv]
    order = torch.randperm(sum(pages) + 2, generator=g, device=DEV)
    kc = torch.randn(order.numel(), hk, page, d, generator=g, device=DEV, dtype=dtype)
    vc = torch.randn(order.numel(), hk, page, d, generator=g, device=DEV, dtype=dtype)
    table = torch.zeros(len(new), c["columns"], dtype=torch.int32, device=DEV)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at: at + p].int()
        if kv[b] % page:  # slots behind the end
            kc[order[at + p - 1], :, kv[b] % page:] = math.nan
            vc[order[at + p - 1], :, kv[b] % page:] = math.nan
        at += p
    q = torch.randn(sum(new), hq, d, generator=g, device=DEV, dtype=dtype)
    q_start = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    kv_len = torch.tensor(kv, dtype=torch.int32, device=DEV)
    lse = torch.full((sum(new), hq), 3.0, device=DEV)
    out = ops().paged_attn(q, kc, vc, table, q_start, kv_len, d ** -0.5, lse=lse)
    again = ops().paged_attn(q, kc, vc, table, q_start, kv_len, d ** -0.5)
    assert torch.equal(out, again)
    seqs = sorted({0, len(new) - 1, *range(0, len(new), 5)})
    for h in sorted({0, hk // 2, hk - 1}):
        heads = slice(h * (hq // hk), (h + 1) * (hq // hk))
        for b in seqs:
            rows = slice(int(q_start[b]), int(q_start[b + 1]))
            one = torch.tensor([0, new[b]], dtype=torch.int32)
            ref, rl, tol, ltol, _ = R.attend(q[rows, heads], kc[:, h: h + 1], vc[:, h: h + 1], table[b: b + 1], one,
                                             kv_len[b: b + 1], d ** -0.5)
            ok, worst = R.within(out[rows, heads], ref, tol, dtype)
            assert ok, (b, h, worst)
            assert bool(((lse[rows, heads].double() - rl).abs() <= ltol).all()), (b, h)
    assert bool(out.isfinite().all()) and bool(lse.isfinite().all())


@pytest.mark.parametrize("name,d", [(n, d) for n in sorted(WAYS) for d in WAYS[n]["d"]])
def test_every_way_of_the_rule(name, d):
    spot_check(WAYS[name], d, HF if d == 64 else BF, 71)


@pytest.mark.parametrize("name", sorted(WINDOWS))
def test_windows_of_page_numbers(name):
    spot_check(WINDOWS[name], WINDOWS[name]["d"], BF, 72)


# ------------------------------------------------------------ many rows, more
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("new,total,at", [(130, 700, 3), (130, 700, 400), (130, 700, 640), (2, 700, 300)])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF), (256, BF)])
def test_values_that_are_not_finite_while_maxima_rise(value, new, total, at, d, dtype):
    """Keys lengthen along the sequence, so that maxima rise by many powers of two from tile to tile, and one visible value
    is not finite.  Its probability in 32 bits is zero for most later rows, where a product of zero and infinity may be
    NaN: its column of its head is infinite or NaN, all else is as without it."""
    s = R.build([new], [total], hq=4, hk=2, d=d, page=16, dtype=dtype, seed=81, device=DEV)
    j = torch.arange(total, device=DEV)
    p = s["table"][0].long()[j // 16]
    f = (1 + j.float() / 8).clamp(max=90.0)[:, None, None]
    s["kc"][p, :, j % 16] = (s["kc"][p, :, j % 16].float() * f).to(dtype)
    check(s, d ** -0.5)
    args = (s["q"], s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], d ** -0.5)
    lse = torch.zeros(new, 4, device=DEV)
    clean = ops().paged_attn(*args)
    s["vc"][p[at], 1, at % 16, d - 3] = value
    got = ops().paged_attn(*args, lse=lse)
    first = max(0, at - (total - new))  # rows from here on see it
    assert bool((~got[first:, 2:, d - 3].isfinite()).all())
    got[first:, 2:, d - 3] = clean[first:, 2:, d - 3]
    assert torch.allclose(got.float(), clean.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
    assert bool(lse.isfinite().all())


@pytest.mark.parametrize("new,total", [([70, 3], [200, 130]), ([1, 2], [200, 30])])
def test_slots_far_apart(new, total):
    """Slots 2^26 elements apart (16 of them are 2 GiB), where the many-row kernel's 32-bit byte offsets end."""
    hk, d, page, stride = 2, 128, 16, 1 << 26
    s = R.build(new, total, hq=4, hk=hk, d=d, page=page, dtype=BF, seed=91, device=DEV)
    want, wl = check(s, d ** -0.5)
    far = {}
    for name in ("kc", "vc"):
        c = s[name]
        flat = torch.empty(stride * (page - 1) + c.shape[0] * hk * d, dtype=BF, device=DEV)
        far[name] = flat.as_strided(c.shape, (hk * d, d, stride, 1))
        far[name].copy_(c)
    got, gl = check(dict(s, **far), d ** -0.5)
    assert torch.equal(got, want) and torch.equal(gl, wl)
    g = gen(92)
    k, v = (torch.randn(sum(new), hk, d, generator=g, device=DEV).to(BF) for _ in range(2))
    ops().paged_append(k, v, s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"])
    ops().paged_append(k, v, far["kc"], far["vc"], s["table"], s["q_start"], s["kv_len"])
    assert torch.equal(far["kc"], s["kc"]) and torch.equal(far["vc"], s["vc"])
