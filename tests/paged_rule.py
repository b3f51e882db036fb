"""The attention's launch rule restated (ospo_amd/csrc/paged_attn.hip: make_plan, even_chunk, pick_chunk, find_item): what a
call's shapes bound, and how its lengths are cut within that."""
import numpy as np

f32 = np.float32


def plan(rows, S, hq, hk, d, most, cus=256):
    """What the host makes of the shapes."""
    g = hq // hk
    few = rows * g <= 32 * S
    bm, ku = (16, 128) if few else (128 if d > 128 else 256, 64)
    pairs = min(rows * g // bm + S, rows * -(-g // bm)) * hk
    slots = cus * ({64: 4, 128: 3, 256: 2}[d] if few else 1)
    least = -(-rows * g // bm) * hk
    host = 640 + 384 * pairs // slots if few else 256 + 2048 * pairs // slots
    bar = min(host, 256 + 1536 * pairs // slots) if few else 96 + 1900 * pairs // slots
    split = most > host and least < 4 * slots and least * S < 1 << 30
    items = pairs if not split else slots if pairs <= slots else pairs + 4 * slots
    return dict(few=few, bm=bm, ku=ku, g=g, pairs=pairs, slots=slots, bar=bar, split=split, items=items,
                cap=min(slots * bm * (4 if few and pairs > slots else 1), rows * g * hk * -(-most // ku)))


def even_chunk(p, hk, tiles, units, longest):
    """Key blocks of a chunk, and the way that it was found."""
    total = f32(sum(f32(t) * f32(u) for t, u in zip(tiles, units)))
    base, most = sum(tiles), max([1] + [u for t, u in zip(tiles, units) if t])
    if longest <= p["bar"]:
        return 0x7fffffff, "whole"
    base, total = max(1, base * hk), f32(total * f32(hk))
    even = f32(total / f32(p["slots"]))
    if base > p["slots"]:
        return int(max(f32(4), min(f32(most), np.ceil(even if base >= 4 * p["slots"] else f32(0.25) * even)))), "rounds"
    lo, times = max(f32(1), np.ceil(even)), p["slots"] // base
    hi = f32((most + times - 1) // times)
    if p["slots"] > base:
        hi = min(hi, np.ceil(f32(1.00001) * total / f32(p["slots"] - base)) + f32(1))
    hi = max(lo, hi) + (f32(4) if most > 1 << 22 else f32(0))
    for i in range(4):
        c = int(lo + (hi - lo) * f32(0.25) * f32(i))
        if hk * sum(t * ((u - 1) // c + 1) for t, u in zip(tiles, units)) <= p["slots"]:
            return c, "step"
        if hi - lo < 1:
            break
    return int(hi), "last"


def cut(rows, new, kv, start, hq, hk, d, most):
    """How a batch is cut: items, (tile, head) pairs, rows of partial results, chunks of each sequence, and the way."""
    p = plan(rows, len(new), hq, hk, d, most)
    g, bm, ku = p["g"], p["bm"], p["ku"]
    tiles = [-(-n * g // bm) for n in new]
    units = [-(-k // ku) - a // ku if k > a else 1 for k, a in zip(kv, start)]
    way, need, c = "off", 0, 0x7fffffff
    if p["split"]:
        c, way = even_chunk(p, hk, tiles, units, max([0] + [k - a for k, a, t in zip(kv, start, tiles) if t]))
        while True:
            need = hk * sum(n * g * nch for n, nch in zip(new, [(u - 1) // c + 1 for u in units]) if nch > 1)
            if need <= p["cap"]:
                break
            c, way = int(np.ceil(f32(c) * max(f32(need) / f32(p["cap"]), f32(1.125)))), "room"
    nch = [(u - 1) // c + 1 for u in units]
    return dict(p, chunk=c, way=way, need=need, nch=nch, units=units, tiles=tiles, pairs_made=hk * sum(tiles),
                items_made=hk * sum(t * n for t, n in zip(tiles, nch)))
