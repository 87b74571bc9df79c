"""The calls of the GPU tests of norms and of fp16's range choose the kernels that
they are there for (256 compute units)."""

from __future__ import annotations

import pytest

from test_attention_plan import plan  # noqa: F401 (a fixture)

KIND = {"pairs": 2, "pairs_128": 2, "of_128": 0, "of_256": 1, "wide": None}


def _chosen(p, name):
    if name == "split":
        return p["use"] == 1
    return p["use"] == 0 and KIND[name] in (None, p["blocks"]) and (name != "of_256" or p["keys"] == 256)


def test_norms(plan):  # noqa: F811
    from test_gpu_attention_norms import CALLS, KERNELS
    rows = []
    for name, d, dtype, _ in CALLS:
        lengths, H, Hk, _ = KERNELS[name]
        rows.append((name, (1, sum(lengths), sum(lengths), len(lengths), H, Hk, d, dtype == "f32")))
    for (name, r), p in zip(rows, plan([r for _, r in rows])):
        assert _chosen(p, name), (name, r, p)


def test_f16_range(plan):  # noqa: F811
    from test_gpu_attention_f16_range import KERNELS
    for (name, (T, H, Hk, d)), p in zip(KERNELS.items(), plan([(0, T, T, 1, H, Hk, d, 0) for T, H, Hk, d in KERNELS.values()])):
        assert _chosen(p, name), (name, p)


@pytest.mark.parametrize("rows,kinds", [([(0, n, 1024, 1, H, Hk, 128, 0) for n, H, Hk in (
    (1, 4, 1), (40, 2, 1), (1100, 4, 4), (3500, 16, 16), (3500, 32, 8), (4200, 128, 8))], ("split", "split", "split", "pairs", "of_128", "of_256")),
    ([(1, 40, 16000, 3, 4, 2, 64, 0), (1, 1000, 1000, 3, 32, 2, 64, 0), (1, 1000, 1000, 3, 64, 2, 64, 0)], ("split", "pairs", "pairs"))])
def test_weights_and_guards(plan, rows, kinds):  # noqa: F811
    got = ["split" if p["use"] else {v: k for k, v in KIND.items() if k != "pairs_128"}[p["blocks"]] for p in plan(rows)]
    assert tuple(got) == kinds
