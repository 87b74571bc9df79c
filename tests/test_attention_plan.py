"""How attention's tiles are dealt out (csrc/attention_plan.hpp), on the CPU:
the slots of every sequence's tiles are its own and within the grid, the parts
of a split have room in the workspace."""

from __future__ import annotations

import os
import random
import shutil
import subprocess

import pytest

from conftest import PKG_DIR

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include "attention_plan.hpp"
using namespace mhc;
int main() {
  long packed, Tq, Tk, B, H, Hk, d, fp32;
  static const int32_t some[1] = {0};
  while (scanf("%ld %ld %ld %ld %ld %ld %ld %ld", &packed, &Tq, &Tk, &B, &H, &Hk, &d, &fp32) == 8) {
    AttDims n = {packed ? some : nullptr, packed ? some : nullptr, nullptr, Tq, Tk, (int)B, B ? (int)(Tq / B) : 0,
                 B ? (int)(Tk / B) : 0, (int)H, (int)Hk, (int)d, 1};
    const AttSplit s = att_split(n, 256);
    const AttBwdPlan p = att_bwd_plan(n, fp32, att_big_head(n, fp32), 256);
    printf("%lld %lld %lld %d %d %lld %zu %d %zu %zu %d %lld %d\n", (long long)att_slots(packed, Tq, (int)B, n.Sq, 128),
           (long long)att_slots(packed, Tq, (int)B, n.Sq, 256), (long long)att_slots(packed, Tk, (int)B, n.Sk, 128),
           s.use, s.splits, (long long)s.slots, s.bytes(n), p.splits, p.delta_bytes, p.part_bytes, p.keys, (long long)p.slots, att_blocks(n, att_big_head(n, fp32), 256));
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("plan")
    src = d / "plan.cpp"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-I", os.path.join(PKG_DIR, "csrc"), str(src), "-o", str(d / "plan")], check=True)

    def run(rows):
        text = "\n".join(" ".join(str(int(v)) for v in r) for r in rows)
        out = subprocess.run([str(d / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        names = ("slots128", "slots256", "slots_k", "use", "splits", "split_slots", "bytes", "parts", "delta", "part_bytes", "keys", "key_slots", "blocks")
        return [dict(zip(names, map(int, line.split()))) for line in out.splitlines()]

    return run


def _starts(rng, B, T):
    cuts = sorted(rng.randint(0, T) for _ in range(B - 1)) if rng.random() < 0.5 else sorted(
        rng.choice([0, T, rng.randint(0, T)]) for _ in range(B - 1))
    end = rng.choice([T, rng.randint(cuts[-1] if cuts else 0, T)])
    return [0, *[min(c, end) for c in cuts], end]


def _find(cu, T, R, slot, scale=1):
    """slot_sequence's search: 64 candidates a step."""
    cu = [min(max(c, 0), T) for c in cu]
    cu[0] = 0
    lo, n = 0, len(cu)
    while n > 1:
        step = (n + 63) // 64
        hit = max(1, sum(1 for lane in range(64) if lane * step < n and cu[lo + lane * step] * scale // R + lo + lane * step <= slot))
        skip = (hit - 1) * step
        lo += skip
        n = min(step, n - skip)
    return lo


def test_every_tile_has_a_slot_of_its_own(plan):
    """.. found again by the kernels' search, for tiles of 128 and 256 queries and
    for tiles of 32 rows of G a query; rows behind the last sequence too."""
    rng = random.Random(1)
    for _ in range(120):
        B, T = rng.choice([1, 2, 7, 63, 64, 65, 130, 700]), rng.choice([1, 5, 127, 128, 129, 1000, 5000])
        G = rng.choice([1, 3, 4, 7, 40])
        cu = _starts(rng, B, T)
        got = plan([(1, T, T, B, G, 1, 64, 0)])[0]
        tall = plan([(1, T, 100000, B, 128, 128, 128, 0)])[0]
        assert tall["keys"] == 256 and got["keys"] == 128 and got["key_slots"] == got["slots_k"]
        for R, scale, slots in ((128, 1, got["slots128"]), (256, 1, got["slots256"]), (32, G, got["split_slots"])):
            seen = set()
            ends = cu[1:] + [T]
            for b, (lo, hi) in enumerate(zip(cu, ends)):
                for tile in range(-(-(hi - lo) * scale // R)):
                    slot = lo * scale // R + b + tile
                    assert slot < slots and slot not in seen
                    seen.add(slot)
                    assert _find(cu, T, R, slot, scale) == b


def test_wrong_starts_stay_inside():
    """Starts that fall, or leave the buffer, lead to some sequence, never past the last."""
    rng = random.Random(2)
    for _ in range(300):
        B, T = rng.choice([1, 2, 64, 65, 200]), rng.choice([1, 100, 1000])
        cu = [rng.choice([rng.randint(-5, T + 5), -(1 << 31), (1 << 31) - 1]) for _ in range(B + 1)]
        for slot in (0, 1, T // 128 + B):
            assert 0 <= _find(cu, T, 128, slot) <= B


def test_parts_fit_their_workspace(plan):
    rng = random.Random(3)
    rows = []
    for _ in range(2000):
        B, Hk, G = rng.choice([1, 2, 16, 64, 300]), rng.choice([1, 2, 8, 16]), rng.choice([1, 4, 7])
        packed = rng.random() < 0.5
        Sq, Sk = rng.choice([1, 2, 64, 1000, 16384]), rng.choice([1, 300, 5000, 1 << 20])
        rows.append((packed, B * Sq, B * Sk, B, G * Hk, Hk, rng.choice([64, 128, 256]), rng.random() < 0.3))
    for r, p in zip(rows, plan(rows)):
        _, Tq, Tk, B, H, Hk, d, _ = r
        assert 1 <= p["parts"] <= 16 and p["splits"] >= 1
        assert p["bytes"] == (p["splits"] * Tq * H * (d + 2) * 4 if p["use"] and p["splits"] > 1 else 0)
        assert p["delta"] >= H * Tq * 4 and p["delta"] % 256 == 0
        assert p["part_bytes"] == (p["parts"] * 2 * Tk * Hk * d * 4 if p["parts"] > 1 else 0)
        # a part of the keys has a tile for each wave, one of the queries 64 rows or more
        assert p["splits"] <= max(1, -(-Tk // B) // 128) and p["parts"] <= max(1, -(-Tq // B) * (H // Hk) // 64)


def test_nothing_to_split(plan):
    for r in ((1, 0, 0, 3, 4, 2, 64, 0), (0, 0, 0, 0, 4, 2, 64, 0), (1, 10, 10, 0, 4, 2, 64, 0)):
        p = plan([r])[0]
        assert p["use"] == 0 and p["splits"] == p["parts"] == 1 and p["bytes"] == p["part_bytes"] == 0


def test_gpu_tests_reach_every_kernel(plan):
    """The calls of the GPU tests choose the kernels that they are there for (256 compute units)."""
    from test_gpu_attention_blocks import OF_128, OF_256, PAIRS, _lengths
    for heads, kind, d, longest, fp32 in ((PAIRS, 2, 64, 700, 0), (PAIRS, 2, 128, 700, 1), (OF_128, 0, 128, 700, 0),
                                          (OF_128, 0, 256, 700, 0), (OF_128, 0, 64, 700, 1), (OF_256, 1, 128, 1200, 0)):
        for seed in (5, 9, 64, 72, 96, 128, 192, 256):
            T = sum(_lengths(seed, 70, longest))
            p = plan([(1, T, T, 70, *heads, d, fp32)])[0]
            assert p["use"] == 0 and p["blocks"] == kind, (heads, seed, p)
            assert p["keys"] == (256 if kind == 1 else 128)
    # parts of the keys, and none; parts of the queries, and none
    one = plan([(0, 1, 5000, 1, 8, 1, 64, 0), (0, 3, 6300, 3, 4, 4, 128, 1), (1, 5, 5, 1, 4, 2, 64, 0), (1, 1030, 1030, 1, 2, 1, 64, 0)])
    assert [p["use"] for p in one] == [1, 1, 1, 1]
    assert one[0]["splits"] > 1 and one[1]["splits"] > 1 and one[2]["splits"] == one[2]["parts"] == 1 and one[3]["parts"] > 1
