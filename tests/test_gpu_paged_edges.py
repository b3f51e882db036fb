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
