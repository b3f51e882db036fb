"""The attention's launch rule over random batches: what the lengths on the device make of a call never passes what the
host sized for its shapes, and the cases of the GPU tests take the ways that they are there for."""
import math
import random

import pytest

from ospo_amd import _lib
from tests import paged_rule as P
from tests.paged_cases import WAYS, WINDOWS


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def test_a_batch_never_passes_its_bounds():
    rng, ways = random.Random(5), {}
    for _ in range(12000):
        S, hk = rng.choice([1, 2, 3, 8, 32, 64, 100, 200]), rng.choice([1, 2, 3, 4, 8, 16, 32])
        hq, d = hk * rng.choice([1, 2, 4, 7, 8]), rng.choice([64, 128, 256])
        mix, most_new, reach = rng.random(), rng.choice([4, 40, 600, 4000]), rng.choice([300, 1000, 8000, 70000, 500000])
        new = [int(rng.random() > 0.1) if rng.random() < mix else _log(rng, 1, most_new) for _ in range(S)]
        kv = [_log(rng, 1, reach) if rng.random() < 0.7 else rng.choice([0, 1, reach]) for _ in range(S)]
        start = [rng.randint(0, k) if rng.random() < 0.2 else 0 for k in kv]
        rows = sum(new) + rng.choice([0, 0, 5])
        if rows == 0:
            continue
        r = P.cut(rows, new, kv, start, hq, hk, d, max(kv + [1]) * rng.choice([1, 1, 4, 20]))
        assert r["pairs_made"] <= r["pairs"] and r["items_made"] <= r["items"], r
        assert r["need"] <= r["cap"], r
        for u, n in zip(r["units"], r["nch"]):  # chunks of ceil(u / n) blocks: each of the n begins inside the keys
            size = -(-u // n)
            assert size <= r["chunk"] and n * size >= u
        key = (r["few"], r["way"])
        ways[key] = ways.get(key, 0) + 1
    for few in (True, False):
        for way in ("off", "whole", "rounds", "step", "last", "room"):
            assert ways.get((few, way), 0) > (0 if way == "room" else 5), (few, way, ways)


def test_the_host_sizes_what_the_rule_says():
    for rows, S, hq, hk, d, page, columns in ((32, 32, 32, 32, 128, 16, 2048), (575, 64, 32, 8, 128, 64, 128),
                                              (2048, 64, 32, 8, 256, 64, 4096), (1, 1, 8, 1, 64, 16, 4000)):
        p = P.plan(rows, S, hq, hk, d, page * columns)
        want = 32 + 32 * p["pairs"] + p["cap"] * (4 * d + 8) if p["split"] else 0
        assert _lib.query("ospo_paged_attn_ws_bytes", rows, S, hq, hk, d, page, columns) == want


@pytest.mark.parametrize("name", sorted(WAYS))
def test_cases_take_their_ways(name):
    c = WAYS[name]
    for d in c["d"]:
        r = P.cut(sum(c["new"]), c["new"], c["kv"], [0] * len(c["kv"]), c["hq"], c["hk"], d, c["page"] * c["columns"])
        assert (r["few"], r["way"]) == (c["few"], c["way"]), r
        assert (r["few"], r["way"] in ("off", "whole")) == (c["few"], max(r["nch"]) == 1)


@pytest.mark.parametrize("name", sorted(WINDOWS))
def test_windows_are_refilled(name):
    """A wave holds 64 page numbers, and the next 64 on their way."""
    c = WINDOWS[name]
    r = P.cut(sum(c["new"]), c["new"], c["kv"], [0] * len(c["kv"]), c["hq"], c["hk"], c["d"], c["page"] * c["columns"])
    assert r["few"] == c["few"] and r["nch"][0] == c["nch"]
    keys = min(-(-r["units"][0] // r["nch"][0]) * r["ku"], c["kv"][0])
    assert (-(-keys // c["page"]) - 1) // 64 == c["refills"]
