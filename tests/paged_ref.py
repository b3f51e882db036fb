"""Plain 64-bit forms of the paged-cache operators and the error bounds their kernels are held to."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}  # half a step of the subnormals


def rotate(x, angle, mag, interleaved, backward=False):
    """x [n, heads, d], angle [n, rot / 2] (64 bits) -> (y, bound of |kernel - y|)."""
    half = angle.shape[1]
    x = x.double()
    c, s = (angle.cos() * mag)[:, None], (angle.sin() * mag)[:, None]
    if backward:
        s = -s
    a, b = ((x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved
            else (x[..., :half], x[..., half:2 * half]))
    y, tol = x.clone(), torch.zeros_like(x)
    ya, yb = a * c - b * s, b * c + a * s
    # fp32: each table value, each product and the sum rounded once: at most 4 half steps of |a| m + |b| m
    e = (a.abs() + b.abs()) * mag * 4 * 2.0 ** -24
    for dst, va, vb in ((y, ya, yb), (tol, e, e)):
        if interleaved:
            dst[..., 0:2 * half:2], dst[..., 1:2 * half:2] = va, vb
        else:
            dst[..., :half], dst[..., half:2 * half] = va, vb
    return y, tol


def within(got, ref, tol, dtype):
    """|got - ref| <= tol + half a step of the stored type (of a value up to |ref| + tol)."""
    err = (got.double() - ref).abs()
    lim = tol + HALF[dtype] * (ref.abs() + tol) + TINY[dtype]
    bad = ~(err <= lim)
    return not bool(bad.any()), float((err / lim.clamp_min(1e-300)).max()) if err.numel() else 0.0


def gather(cache, table, n, page):
    """Rows 0 .. n - 1 of a sequence from a cache [pages, heads, page, d] -> [heads, n, d]."""
    j = torch.arange(n, device=cache.device)
    return cache[table.long()[j // page], :, j % page].transpose(0, 1)


def attend(q, kc, vc, table, q_start, kv_len, scale, start=None, causal=True):
    """Per sequence and head in 64 bits -> out, lse, bound of out, bound of lse, rows that belong to a sequence.

    Bounds (u = 2^-24, h = half a step of the cache's type): a score's fp32 sum of d products is off by at most
    d u sum|q k|, its scaling and exponent by a few u of its size, so a probability by e = 2 (d + 8) u S (S = scale
    times the row's largest sum |q||k|); rounding a probability to the cache's type adds h (or 2^-25 of the row's
    maximum where fp16 is subnormal); fp32 sums over n keys add n u of the sum of magnitudes.  An output is a mean of
    v with weights p / sum p: off by at most (h + 2 e + 2 n u) A, A = the mean of |v|, and n 2^-25 max|v| in fp16."""
    n, hq, d = q.shape
    page, hk = kc.shape[2], kc.shape[1]
    u, h = 2.0 ** -24, HALF[kc.dtype]
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    tol, lse = torch.zeros_like(out), torch.full((n, hq), -math.inf, dtype=torch.float64, device=q.device)
    ltol = torch.zeros_like(lse)
    owned = torch.zeros(n, dtype=torch.bool, device=q.device)
    for b in range(table.shape[0]):
        q0, q1, kv = int(q_start[b]), int(q_start[b + 1]), int(kv_len[b])
        m = q1 - q0
        owned[q0:q1] = True
        if m <= 0 or kv <= 0:
            continue
        k, v = gather(kc, table[b], kv, page).double(), gather(vc, table[b], kv, page).double()
        pos = torch.arange(kv - m, kv, device=q.device) if causal else torch.full((m,), kv - 1, device=q.device)
        key = torch.arange(kv, device=q.device)
        seen = (key[None] <= pos[:, None]) & (key[None] >= (int(start[b]) if start is not None else 0))
        for j in range(hq):
            kh, vh = k[j // (hq // hk)], v[j // (hq // hk)]
            x = q[q0:q1, j].double()
            w = torch.where(seen, x @ kh.t() * scale, -math.inf)
            size = torch.where(seen, x.abs() @ kh.abs().t() * scale, 0.0).amax(1)
            top = w.amax(1, keepdim=True)
            p = torch.where(seen, (w - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
            total = p.sum(1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            some = seen.any(1)
            # a value that no row of a column sees must not enter, whatever it is
            use = seen.any(0)[:, None]
            o = p @ torch.where(use, vh, 0.0)
            mean = p @ torch.where(use, vh.abs(), 0.0)
            e = 2 * (d + 8) * u * size[:, None]
            out[q0:q1, j] = o
            tol[q0:q1, j] = (h + 2 * e + 2 * kv * u) * mean
            if kc.dtype == torch.float16:
                tol[q0:q1, j] += kv * 2.0 ** -25 * torch.where(use, vh.abs(), 0.0).amax()
            lse[q0:q1, j] = torch.where(some, (top + torch.where(total == 0, 1.0, total).log()).squeeze(1), -math.inf)
            ltol[q0:q1, j] = torch.where(some, (e.squeeze(1) + 2 * kv * u + 4 * u * lse[q0:q1, j].abs() + 4 * u), 0.0)
    return out, lse, tol, ltol, owned


def build(new, total, *, hq, hk, d, page, dtype, seed, device, start=None, spare=2, layout="pages", lead=0, tail=0,
          fill=0.0, q_scale=1.5):
    """A ragged batch and its paged cache: pages in a random order, slots behind a sequence's length and spare pages
    hold ``fill``; ``lead`` / ``tail`` rows of no sequence around the batch."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    pages = [-(-max(t, 0) // page) for t in total]
    order = torch.randperm(sum(pages) + spare, generator=g)
    most = max(pages + [1])
    table = torch.zeros(len(new), most, dtype=torch.int32)
    shape = (order.numel(), hk, page, d)
    kc, vc = torch.full(shape, fill), torch.full(shape, fill)
    at = 0
    for b, (t, p) in enumerate(zip(total, pages)):
        ids = order[at: at + p]
        at += p
        table[b, :p] = ids.int()
        for c in (kc, vc):
            x = torch.full((p * page, hk, d), fill)
            x[:max(t, 0)] = r(max(t, 0), hk, d)
            c[ids] = x.view(p, page, hk, d).transpose(1, 2)
    n = lead + sum(new) + tail
    s = dict(q=(r(n, hq, d) * q_scale).to(dtype).to(device), table=table.to(device),
             q_start=torch.tensor([lead + sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=device),
             kv_len=torch.tensor(list(total), dtype=torch.int32, device=device),
             start=None if start is None else torch.tensor(list(start), dtype=torch.int32, device=device))
    for name, c in (("kc", kc), ("vc", vc)):
        c = c.to(dtype).to(device)
        if layout == "slots":  # [pages, slots, heads, d] in memory
            c = c.transpose(1, 2).contiguous().transpose(1, 2)
        s[name] = c
    return s
