"""Paged-cache operators on the MI355X against their plain forms in 64 bits: rotary positions (both directions), the
append, and the attention of new tokens.  Bounds: tests/paged_ref.py."""
import math

import pytest
import torch

from tests import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _lib():
    from ospo_amd import _lib
    _lib.lib()


def ops():
    from ospo_amd import ops as _ops
    return _ops


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def angles(positions, rot, theta=10000.0):
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    return positions.double()[:, None] * f


# ------------------------------------------------------------------ rotary
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("n,hq,hk,d,rot,il", [
    (1, 1, 0, 128, 128, False), (1, 32, 32, 128, 128, False), (37, 28, 4, 128, 64, True), (5, 3, 1, 80, 80, False),
    (129, 7, 7, 64, 24, False), (129, 7, 7, 64, 24, True), (65, 2, 1, 128, 50, False), (65, 2, 1, 128, 50, True),
    (33, 5, 2, 256, 256, False), (33, 5, 2, 256, 256, True), (9, 4, 4, 36, 2, True), (9, 4, 4, 35, 10, False),
    (601, 32, 8, 128, 128, True)])
@pytest.mark.parametrize("backward", [False, True])
def test_rotary(dtype, n, hq, hk, d, rot, il, backward):
    g = gen(n * 7 + d + rot)
    q = torch.randn(n, hq, d, generator=g, device=DEV).to(dtype)
    k = torch.randn(n, hk, d, generator=g, device=DEV).to(dtype) if hk else None
    pos = torch.randint(0, 4096, (n,), generator=g, device=DEV).int()
    tab = ops().rotary_tables(4096, rot, 10000.0, DEV)
    got = ops().rotary(q, k, pos, tab, interleaved=il, backward=backward)
    for x, y in zip((q, k), got):
        if x is None:
            assert y is None
            continue
        ref, tol = R.rotate(x, angles(pos, rot), 1.0, il, backward)
        ok, worst = R.within(y, ref, tol, dtype)
        assert ok, worst
        assert torch.equal(y[..., rot:], x[..., rot:])


def test_rotary_far_positions():
    """At position 10^6 the angles still come from 64 bits."""
    pos = torch.tensor([999_999, 524_288, 1], dtype=torch.int32, device=DEV)
    q = torch.randn(3, 2, 64, generator=gen(1), device=DEV)
    y, _ = ops().rotary(q, None, pos, ops().rotary_tables(1_000_000, 64, 10000.0, DEV))
    ref, tol = R.rotate(q, angles(pos, 64), 1.0, False)
    ok, worst = R.within(y, ref, tol, FP)
    assert ok, worst


@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rotary_strides_in_place_and_streams(il, dtype):
    """Views of a packed projection, a head-major layout, an odd offset, in place, on another stream."""
    n, hq, hk, d, rot = 45, 6, 2, 64, 48
    g = gen(5)
    pos = torch.randint(0, 100, (n,), generator=g, device=DEV).int()
    tab = ops().rotary_tables(100, rot, 10000.0, DEV)
    packed = torch.randn(n, (hq + 2 * hk) * d, generator=g, device=DEV).to(dtype)
    q, k = packed[:, : hq * d].view(n, hq, d), packed[:, hq * d: (hq + hk) * d].view(n, hk, d)
    want = ops().rotary(q.contiguous(), k.contiguous(), pos, tab, interleaved=il)
    major = torch.empty(hq, n, d, device=DEV, dtype=dtype).transpose(0, 1)
    odd = torch.empty(n * hk * d + 1, device=DEV, dtype=dtype)[1:].view(n, hk, d)
    got = ops().rotary(q, k, pos, tab, interleaved=il, out=(major, odd))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rest = packed[:, (hq + hk) * d:].clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops().rotary(q, k, pos, tab, interleaved=il, out=(q, k))
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(rest, packed[:, (hq + hk) * d:])


def test_rotary_clamps_positions_and_empty():
    tab = ops().rotary_tables(10, 64, 10000.0, DEV)
    q = torch.randn(4, 2, 64, generator=gen(2), device=DEV)
    a, _ = ops().rotary(q, None, torch.tensor([-5, 2 ** 31 - 1, 9, 0], dtype=torch.int32, device=DEV), tab)
    b, _ = ops().rotary(q, None, torch.tensor([0, 9, 9, 0], dtype=torch.int32, device=DEV), tab)
    assert torch.equal(a, b)
    e, _ = ops().rotary(q[:0], None, torch.zeros(0, dtype=torch.int32, device=DEV), tab)
    assert e.shape == (0, 2, 64)


def test_rotary_gradient_matches_differences():
    """<dy, R(x + t u) - R(x)> / t = <R^T dy, u>: R is linear, so t = 1 is exact; fp32, with a table magnitude."""
    n, h, d, rot = 17, 3, 64, 40
    g = gen(9)
    x, u, dy = (torch.randn(n, h, d, generator=g, device=DEV) for _ in range(3))
    pos = torch.arange(n, device=DEV).int()
    for il in (False, True):
        tab = ops().rotary_tables(64, rot, 10000.0, DEV, {"type": "yarn", "factor": 4.0, "original": 16})
        r = lambda t, **kw: ops().rotary(t, None, pos, tab, interleaved=il, **kw)[0].double()  # noqa: E731
        lhs = (dy.double() * (r(x + u) - r(x))).sum()
        rhs = (r(dy, backward=True) * (x + u - x).double()).sum()
        # both sides round each of n h d outputs once or twice: 2^-24 of their magnitudes
        lim = 8 * 2.0 ** -24 * float((dy.abs().double() * (r(x).abs() + r(x + u).abs() + 1)).sum())
        assert abs(float(lhs - rhs)) <= lim


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("new,total,page,hq,hk,d,rot,il,layout", [
    ([1], [1], 16, 4, 4, 128, 128, False, "pages"),
    ([1, 1, 1], [600, 24, 17], 16, 32, 32, 128, 128, False, "pages"),
    ([5, 0, 1, 130, 3], [5, 40, 1, 500, 64], 24, 14, 2, 64, 32, True, "pages"),
    ([33, 2], [33, 9], 1, 3, 1, 128, 0, False, "slots"),
    ([200], [1000], 100, 8, 8, 256, 24, False, "slots"),
    ([7, 8], [7, 8], 7, 0, 3, 36, 10, True, "pages"),
    ([1] * 70, list(range(1, 71)), 8, 2, 1, 64, 64, False, "pages")])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_paged_append(new, total, page, hq, hk, d, rot, il, layout, dtype):
    s = R.build(new, total, hq=max(hq, 1), hk=hk, d=d, page=page, dtype=dtype, seed=3, device=DEV, layout=layout, lead=2,
                tail=3)
    n = s["q"].shape[0]
    g = gen(4)
    packed = torch.randn(n, (hq + 2 * hk), d, generator=g, device=DEV).to(dtype)
    q, k, v = packed[:, :hq], packed[:, hq: hq + hk], packed[:, hq + hk:]
    tab = ops().rotary_tables(max(total), rot, 10000.0, DEV) if rot else None
    want_k, want_v = s["kc"].double(), s["vc"].double()
    tol_k = torch.zeros_like(want_k)
    q_out = torch.full((n, hq, d), 7.0, device=DEV).to(dtype) if hq else None
    seq = torch.full((n,), -1)
    for b in range(len(new)):
        seq[int(s["q_start"][b]): int(s["q_start"][b + 1])] = b
    pos = torch.zeros(n, dtype=torch.int64)
    for r in range(n):
        if seq[r] >= 0:
            pos[r] = total[seq[r]] - int(s["q_start"][seq[r] + 1]) + r
    pos = pos.to(DEV)
    zero = torch.zeros(n, rot // 2, dtype=torch.float64, device=DEV)
    ang = angles(pos.int(), rot) if rot else zero
    rk, tk = R.rotate(k, ang, 1.0, il)
    for r in range(n):
        if seq[r] >= 0:
            p = int(s["table"][seq[r], int(pos[r]) // page])
            want_k[p, :, int(pos[r]) % page], want_v[p, :, int(pos[r]) % page] = rk[r], v[r].double()
            tol_k[p, :, int(pos[r]) % page] = tk[r]
    got = ops().paged_append(k, v, s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], q=q if hq else None,
                             q_out=q_out, rope=tab, interleaved=il)
    ok, worst = R.within(s["kc"], want_k, tol_k, dtype)
    assert ok, worst
    assert torch.equal(s["vc"].double(), want_v)
    if hq:
        own = (seq >= 0).to(DEV)
        rq, tq = R.rotate(q, ang, 1.0, il)
        ok, worst = R.within(got[own], rq[own], tq[own], dtype)
        assert ok, worst
        assert bool((got[~own] == 7.0).all())
    else:
        assert got is None


def test_paged_append_missing_pages_and_positions():
    """Rows whose page or position does not exist are not stored; all others are."""
    s = R.build([4, 2, 3], [20, 2, 6], hq=2, hk=2, d=64, page=8, dtype=BF, seed=1, device=DEV)
    s["table"][0, 2] = -1            # positions 16 .. 19 of sequence 0: its four new rows
    s["table"][1, 0] = s["kc"].shape[0]
    s["kv_len"][2] = 2               # three rows, two positions: the first row has position -1
    n = s["q"].shape[0]
    k, v = (torch.randn(n, 2, 64, generator=gen(i), device=DEV).to(BF) for i in (1, 2))
    kc, vc = s["kc"].clone(), s["vc"].clone()
    ops().paged_append(k, v, s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"])
    p = int(s["table"][2, 0])
    kc[p, :, :2], vc[p, :, :2] = k[7:9].transpose(0, 1), v[7:9].transpose(0, 1)
    assert torch.equal(kc, s["kc"]) and torch.equal(vc, s["vc"])


# --------------------------------------------------------------- attention
def check(s, scale, causal=True, q=None, fill=3.0, **kw):
    q = s["q"] if q is None else q
    n, hq, d = q.shape
    out = torch.full((n, hq, d), fill, device=DEV).to(q.dtype)
    lse = torch.full((n, hq), fill, device=DEV)
    got = ops().paged_attn(q, s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], scale, start=s["start"],
                           causal=causal, out=kw.get("out", out), lse=lse)
    ref, rl, tol, ltol, owned = R.attend(q, s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], scale, s["start"],
                                         causal)
    ok, worst = R.within(got[owned], ref[owned], tol[owned], q.dtype)
    assert ok, worst
    empty = rl == -math.inf
    assert torch.equal(lse[owned] == -math.inf, empty[owned])
    live = owned[:, None] & ~empty
    assert bool(((lse.double() - rl).abs()[live] <= ltol[live]).all())
    assert bool((got[empty & owned[:, None]] == 0).all())
    if "out" not in kw:
        assert bool((got[~owned] == fill).all()) and bool((lse[~owned] == fill).all())
    return got, lse


SHAPES = [  # new, total, page, hq, hk
    ([1], [1], 16, 4, 4),
    ([1], [600], 16, 32, 32),
    ([1], [33], 1, 1, 1),
    ([1, 1, 1, 1], [640, 24, 1, 333], 24, 8, 2),
    ([1] * 9, [5, 64, 65, 127, 128, 129, 4096, 1, 2], 64, 28, 4),
    ([2, 0, 1, 5], [2, 77, 4000, 130], 7, 6, 2),
    ([31], [31], 100, 4, 1),
    ([64], [64], 16, 2, 2),
    ([65, 129], [65, 700], 128, 3, 3),
    ([257, 1, 30], [257, 3000, 1030], 24, 16, 4),
    ([600], [600], 8, 2, 1),
    ([3], [1500], 16, 33, 1),
    ([128], [129], 256, 64, 1),
]


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, HF), (256, BF), (128, HF), (64, BF)])
@pytest.mark.parametrize("new,total,page,hq,hk", SHAPES)
def test_paged_attn(new, total, page, hq, hk, d, dtype):
    s = R.build(new, total, hq=hq, hk=hk, d=d, page=page, dtype=dtype, seed=len(new) + d, device=DEV, lead=1, tail=2,
                fill=math.nan)
    check(s, d ** -0.5)


@pytest.mark.parametrize("new,total,start", [
    ([1, 1, 1], [50, 50, 50], [0, 49, 50]),            # the last row sees nothing
    ([70, 3, 40], [300, 3, 40], [250, 1, 39]),         # rows before the start see nothing
    ([5, 5], [5, 2], [0, 0]),                          # more rows than positions: the first rows see nothing
    ([1, 1], [0, 900], [0, 880]),
    ([200], [1024], [1000])])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_paged_attn_rows_without_keys(new, total, start, causal, d):
    s = R.build(new, total, hq=6, hk=2, d=d, page=16, dtype=BF, seed=2, device=DEV, start=start, tail=1, fill=math.inf)
    for b, a in enumerate(start):  # keys in front of the start are not there either
        for p in range(min(a, total[b])):
            s["kc"][int(s["table"][b, p // 16]), :, p % 16] = math.nan
            s["vc"][int(s["table"][b, p // 16]), :, p % 16] = math.nan
    check(s, d ** -0.5, causal)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("new,total,hk,d", [(40, 100, 1, 128), (150, 150, 2, 64), (3, 70, 2, 256)])
def test_paged_attn_later_values_do_not_reach_earlier_rows(value, new, total, hk, d):
    """A value of infinity or NaN at one position: rows in front of it are as without it, rows from it on get it."""
    s = R.build([new], [total], hq=2 * hk, hk=hk, d=d, page=16, dtype=BF, seed=8, device=DEV)
    args = (s["q"], s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], d ** -0.5)
    clean = ops().paged_attn(*args)
    at = total - new // 2 - 1
    s["vc"][int(s["table"][0, at // 16]), 0, at % 16, 5] = value
    got = ops().paged_attn(*args)
    row = at - (total - new)
    # rows in front: the same up to the order of one tile's sum (an fp32 rounding, then the stored one)
    assert torch.allclose(got[:row].float(), clean[:row].float(), rtol=2.0 ** -7, atol=2.0 ** -9)
    hit = got[row:, : 2, 5].float()  # the value's head, its group's two query heads
    assert bool((hit.isnan() if math.isnan(value) else hit == value).all())
    keep = torch.ones_like(got[row:], dtype=torch.bool)
    keep[:, :2, 5] = False
    assert bool(got[row:][keep].isfinite().all())


@pytest.mark.parametrize("new,total,page,hq,hk", [
    ([8, 8], [300, 40], 16, 8, 2),
    ([20, 1, 1, 1], [900, 64, 5, 33], 24, 8, 2),
    ([9, 3], [5000, 3], 64, 28, 4),
    ([33, 31], [1500, 31], 16, 4, 4),  # on both sides of the rule
    ([32], [2000], 8, 2, 2),
    ([33], [2000], 8, 2, 2)])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF), (256, BF)])
def test_paged_attn_a_few_tiles_of_rows(new, total, page, hq, hk, d, dtype):
    s = R.build(new, total, hq=hq, hk=hk, d=d, page=page, dtype=dtype, seed=15, device=DEV, tail=1, fill=math.nan)
    check(s, d ** -0.5)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("new,at", [(70, 10), (70, 300), (2, 300)])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF), (256, BF)])
def test_paged_attn_values_that_are_not_finite(value, new, at, d, dtype):
    """At a key that every row sees, in the first tile and in the middle: its column of its head, and nothing else."""
    s = R.build([new], [500], hq=8, hk=2, d=d, page=16, dtype=dtype, seed=13, device=DEV)
    args = (s["q"], s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], d ** -0.5)
    clean = ops().paged_attn(*args)
    s["vc"][int(s["table"][0, at // 16]), 1, at % 16, d - 3] = value
    got = ops().paged_attn(*args)
    hit = got[:, 4:, d - 3].float()
    assert bool((hit.isnan() if math.isnan(value) else hit == value).all())
    got[:, 4:, d - 3] = clean[:, 4:, d - 3]
    assert torch.allclose(got.float(), clean.float(), rtol=2.0 ** -7, atol=2.0 ** -9)


@pytest.mark.parametrize("new,total", [([130], [700]), ([1, 1, 1], [700, 64, 129]), ([70, 1], [65, 3000])])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF), (256, BF), (128, HF)])
@pytest.mark.parametrize("down", [False, True])
def test_paged_attn_scores_that_grow(new, total, d, dtype, down):
    """Keys that lengthen (or shorten) along the sequence: maxima rise by many powers of two from tile to tile, and
    what was summed before has to follow."""
    s = R.build(new, total, hq=8, hk=2, d=d, page=16, dtype=dtype, seed=12, device=DEV)
    for b, t in enumerate(total):
        for i in range(-(-t // 16)):
            pos = torch.arange(16, device=DEV) + 16 * i
            f = 1 + ((t - pos).clamp(min=0) if down else pos).float() / 8
            page = int(s["table"][b, i])
            s["kc"][page] = (s["kc"][page].float() * f.clamp(max=90.0)[None, :, None]).to(dtype)
    check(s, d ** -0.5)


def test_paged_attn_many_sequences():
    """More sequences than a wave has lanes, of all lengths, some cut into chunks: single tokens, and chunks beside
    them; rows of none between."""
    total = [1 + (37 * i * i) % 700 for i in range(150)]
    total[3], total[70], total[149] = 9000, 5000, 3000
    for new in ([1] * 150, [0 if i % 7 == 0 else min(total[i], 1 + 40 * (i % 3 == 0)) for i in range(150)]):
        s = R.build(new, total, hq=4, hk=1, d=64, page=16, dtype=BF, seed=14, device=DEV, lead=2, tail=3)
        check(s, 0.125)


def test_paged_attn_nothing_to_do():
    s = R.build([1], [40], hq=4, hk=2, d=64, page=16, dtype=BF, seed=1, device=DEV)
    none = ops().paged_attn(s["q"][:0], s["kc"], s["vc"], s["table"], torch.zeros(2, dtype=torch.int32, device=DEV),
                            s["kv_len"], 0.1)
    assert none.shape == (0, 4, 64)
    out = torch.full((1, 4, 64), 3.0, device=DEV).to(BF)
    ops().paged_attn(s["q"], s["kc"], s["vc"], s["table"][:0], s["q_start"][:1], s["kv_len"][:0], 0.1, out=out)
    assert bool((out == 3).all())


@pytest.mark.parametrize("new,total", [([1, 1], [700, 90]), ([130], [900])])
@pytest.mark.parametrize("d", [64, 128])
def test_paged_attn_strides_streams_and_offsets(new, total, d):
    """Queries as views of a packed projection, at an odd offset, head-major outputs, a slot-major cache, another
    stream: the same bits as the plain layout."""
    hq, hk = 6, 3
    s = R.build(new, total, hq=hq, hk=hk, d=d, page=16, dtype=BF, seed=4, device=DEV)
    want, wl = check(s, d ** -0.5)
    n = sum(new)
    packed = torch.zeros(n, (hq + 2) * d, device=DEV, dtype=BF)
    packed[:, d: (hq + 1) * d] = s["q"].reshape(n, -1)
    odd = torch.zeros(n * hq * d + 3, device=DEV, dtype=BF)[3:].view(n, hq, d)
    odd.copy_(s["q"])
    major = torch.empty(hq, n, d, device=DEV, dtype=BF).transpose(0, 1)
    off = torch.empty(n * hq * d + 1, device=DEV, dtype=BF)[1:].view(n, hq, d)
    lse = torch.empty(hq, n, device=DEV).t()
    st = torch.cuda.Stream()
    args = (s["table"], s["q_start"], s["kv_len"], d ** -0.5)
    slots = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (s["kc"], s["vc"])]
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a = ops().paged_attn(packed[:, d: (hq + 1) * d].view(n, hq, d), s["kc"], s["vc"], *args, out=major, lse=lse)
        b = ops().paged_attn(odd, *slots, *args, out=off)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(a, want) and torch.equal(b, want) and torch.equal(lse, wl)


def test_paged_attn_long_context_split():
    """One token over 70,000 keys of grouped heads, and a chunk over 20,000: keys cut into many chunks and joined;
    the same bits each time."""
    for new, total, hq, hk in (([1, 1], [70_001, 300], 8, 1), ([48], [20_000], 8, 2)):
        s = R.build(new, total, hq=hq, hk=hk, d=128, page=64, dtype=BF, seed=6, device=DEV)
        a, la = check(s, 128 ** -0.5)
        b, lb = check(s, 128 ** -0.5)
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_paged_cache_offsets_past_32_bits():
    """Pages whose elements lie behind 2^31 (and bytes behind 2^32)."""
    hk, page, d = 2, 64, 128
    pages = 2 ** 31 // (hk * page * d) + 40
    kc = torch.empty(pages, hk, page, d, dtype=BF, device=DEV)
    vc = torch.empty_like(kc)
    total, new = 500, 3
    ids = torch.arange(pages - 1, pages - 9, -1)
    table = ids.int()[None].to(DEV)
    small = R.build([new], [total], hq=4, hk=hk, d=d, page=page, dtype=BF, seed=5, device=DEV, spare=0)
    for i in range(8):
        p = int(small["table"][0, i])
        kc[ids[i]], vc[ids[i]] = small["kc"][p], small["vc"][p]
    big = dict(small, kc=kc, vc=vc, table=table)
    k, v = (torch.randn(new, hk, d, generator=gen(i), device=DEV).to(BF) for i in (1, 2))
    tab = ops().rotary_tables(total, d, 10000.0, DEV)
    for s in (small, big):
        ops().paged_append(k, v, s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], rope=tab)
    a = ops().paged_attn(small["q"], small["kc"], small["vc"], small["table"], small["q_start"], small["kv_len"], 0.1)
    b = ops().paged_attn(big["q"], kc, vc, table, big["q_start"], big["kv_len"], 0.1)
    assert torch.equal(a, b)


def test_paged_attn_missing_pages_leave_other_sequences_alone():
    s = R.build([1, 4, 1], [100, 60, 300], hq=4, hk=2, d=64, page=16, dtype=BF, seed=7, device=DEV)
    args = lambda t, kl: (s["q"], s["kc"], s["vc"], t, s["q_start"], kl, 0.125)  # noqa: E731
    want = ops().paged_attn(*args(s["table"], s["kv_len"]))
    t = s["table"].clone()
    t[1, :2] = torch.tensor([-7, 2 ** 30], dtype=torch.int32)
    kl = s["kv_len"].clone()
    got = ops().paged_attn(*args(t, kl))
    assert torch.equal(got[0], want[0]) and torch.equal(got[5], want[5])
    kl[1] = 2 ** 31 - 1  # clamped to the block table's width
    got = ops().paged_attn(*args(s["table"], kl))
    assert torch.equal(got[0], want[0]) and torch.equal(got[5], want[5])
    assert bool(got.isfinite().all())


# ---------------------------------------------------------------- together
def _layer(s, packed, hq, hk, d, tab, il):
    n = packed.shape[0]
    x = packed.view(n, hq + 2 * hk, d)
    q = ops().paged_append(x[:, hq: hq + hk], x[:, hq + hk:], s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"],
                           q=x[:, :hq], rope=tab, interleaved=il)
    return ops().paged_attn(q, s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], d ** -0.5)


@pytest.mark.parametrize("il", [False, True])
def test_chunks_then_tokens_equal_one_prompt(il):
    """A prompt taken in chunks and then token by token gives the rows that one call over all of it gives, and both the
    plain causal attention of the turned queries and keys."""
    T, hq, hk, d, page = 150, 6, 2, 64, 24
    packed = torch.randn(T, (hq + 2 * hk) * d, generator=gen(11), device=DEV).to(BF)
    tab = ops().rotary_tables(256, d, 10000.0, DEV)

    def fresh():
        return R.build([T], [T], hq=hq, hk=hk, d=d, page=page, dtype=BF, seed=1, device=DEV, fill=math.nan)

    one = fresh()
    whole = _layer(one, packed, hq, hk, d, tab, il)
    s, rows, at = fresh(), [], 0
    for m in (70, 1, 1, 50, 1, 27):
        s["q_start"] = torch.tensor([0, m], dtype=torch.int32, device=DEV)
        s["kv_len"] = torch.tensor([at + m], dtype=torch.int32, device=DEV)
        rows.append(_layer(s, packed[at: at + m], hq, hk, d, tab, il))
        at += m
    got = torch.cat(rows)
    pos = torch.arange(T, device=DEV).int()
    x = packed.view(T, hq + 2 * hk, d)
    q, k = ops().rotary(x[:, :hq], x[:, hq: hq + hk], pos, tab, interleaved=il)
    assert torch.equal(R.gather(one["kc"], one["table"][0], T, page).transpose(0, 1), k)
    ref, _, tol, _, _ = R.attend(q, one["kc"], one["vc"], one["table"], torch.tensor([0, T]), torch.tensor([T]),
                                 d ** -0.5)
    for y in (whole, got):
        ok, worst = R.within(y, ref, tol, BF)
        assert ok, worst


def test_padded_rows_match_the_dense_cache():
    """Left-padded rows (the sampler's) over the paged cache against ospo_attn_cache on the dense one, which rounds its
    scores twice to bf16 (each 2^-9 of a score of at most |s| = 6: e^(2^-8 6) - 1 < 2.4 %)."""
    rows, H, T = 4, 4, 100
    start = [0, 3, 17, 60]
    s = R.build([1] * rows, [T] * rows, hq=H, hk=H, d=128, page=16, dtype=BF, seed=12, device=DEV, start=start, q_scale=1.0)
    got, _ = check(s, 128 ** -0.5)
    dense = [torch.stack([R.gather(c, s["table"][r], T, 16) for r in range(rows)]).contiguous()
             for c in (s["kc"], s["vc"])]
    out = torch.empty(rows, H * 128, device=DEV, dtype=BF)
    pos = torch.tensor([T - 1], dtype=torch.int32, device=DEV)
    ops().attn_cache(s["q"].reshape(rows, -1), *dense, rows, 1, H, T, s["start"], pos, 128 ** -0.5, out)
    assert float((out.view(rows, H, 128).float() - got.float()).norm() / got.float().norm()) < 0.024


def test_captured_step_follows_the_lengths():
    """One decode step captured once; at each replay it follows the lengths, pages and inputs on the device.  Two
    graphs with workspaces of their own, replayed in turn beside eager work."""
    hq, hk, d, page, rows = 8, 2, 64, 16, 3
    total = [40, 700, 5]
    s = R.build([1] * rows, [t + 8 for t in total], hq=hq, hk=hk, d=d, page=page, dtype=BF, seed=13, device=DEV)
    tab = ops().rotary_tables(1024, d, 10000.0, DEV)
    packed = torch.zeros(rows, (hq + 2 * hk) * d, device=DEV, dtype=BF)
    s["kv_len"].copy_(torch.tensor(total, dtype=torch.int32))
    _layer(s, packed, hq, hk, d, tab, False)  # warm-up: it stores a key, so the twin is taken after it
    twin = {k: v.clone() if torch.is_tensor(v) else v for k, v in s.items()}
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _layer(s, packed, hq, hk, d, tab, False)
        graphs.append((g, out))
    for step in range(6):
        x = torch.randn(rows, (hq + 2 * hk) * d, generator=gen(100 + step), device=DEV).to(BF)
        s["kv_len"] += 1
        twin["kv_len"] += 1
        packed.copy_(x)
        g, out = graphs[step % 2]
        g.replay()
        eager = _layer(twin, x, hq, hk, d, tab, False)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), step
        assert torch.equal(s["kc"], twin["kc"]) and torch.equal(s["vc"], twin["vc"])


def test_two_calls_at_once():
    """The same cache read by two streams at once: every call has a workspace of its own."""
    s = R.build([1], [30_000], hq=8, hk=1, d=128, page=64, dtype=BF, seed=14, device=DEV)
    args = (s["q"], s["kc"], s["vc"], s["table"], s["q_start"], s["kv_len"], 0.09)
    want = ops().paged_attn(*args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops().paged_attn(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
