"""Every kernel that a plan may choose for a product of the gated feed-forward
block runs in some shape of tests/test_gpu_gated_ffn_plans.py: the plans of
many random shapes are collected on the CPU (256 CUs), and each (product, size
of an element, tile, direct to LDS or not, whole or in runs, tail or not) among
them has to be among those of that list.  A change of the plans' costs that
leaves a kernel without a test fails here, and names it."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import PKG_DIR
from test_gpu_gated_ffn_plans import SHAPES

REACH = r"""
#include <math.h>
#include <stdio.h>
#include <map>
#include <random>
#include <set>
#include <string>
#include "gated_ffn_plan.hpp"
using namespace mhc;

template <typename F>
static void roles(const FfnDims& d, size_t es, F&& visit) {
  static const char* const kTiles[] = {"16x128", "64x128", "64x64", "128x128", "128x256", "256x256"};
  for (int back = 0; back < 2; ++back) {
    static const char* const kProducts[2][4] = {{"hidden", "out"}, {"grad_hidden", "grad_x", "grad_w_down", "grad_w_gate_up"}};
    const FfnLines l(d, es, back, 256);
    const FfnShapes f(d, l, back);
    for (int i = 0; i < f.n; ++i) {
      const GemmPlans p = plan_gemm(f.s[i], es, 256);
      if (p.main_rows == 0) {
        visit(std::string(kProducts[back][i]) + " few rows, " + std::to_string(8 * es) + " bits");
        continue;
      }
      for (int tail = 0; tail <= (p.main_rows < f.s[i].M); ++tail) {
        const GemmPlan& q = tail ? p.tail : p.main;
        visit(std::string(kProducts[back][i]) + " " + kTiles[q.kind] + ", " + std::to_string(8 * es) + " bits" +
              (q.dma ? "" : ", registers") + (q.run_tiles ? ", runs" : "") + (tail ? ", tail" : ""));
      }
    }
  }
}

int main() {
  std::set<std::string> tested;
  FfnDims d;
  int es;
  while (scanf("%ld %d %d %d %d", (long*)&d.T, &d.D, &d.F, &d.O, &es) == 5)
    roles(d, es, [&](const std::string& r) { tested.insert(r); });
  std::mt19937_64 rng(5);
  auto uni = [&](double a, double b) { return a + (b - a) * (double)(rng() >> 11) / 9007199254740992.0; };
  auto logu = [&](double a, double b) { return (int64_t)exp2(uni(log2(a), log2(b))); };
  std::map<std::string, FfnDims> missing;
  std::set<std::string> seen;
  for (int i = 0; i < 600000; ++i) {
    const bool round = rng() % 4 != 0;
    auto width = [&] { const int64_t w = logu(64, 9000); return (int)(round ? (w + 63) / 64 * 64 : w); };
    d = {logu(1, 9000), width(), width(), width()};
    if (rng() % 5 == 0) d.T = 256 * logu(1, 30) + logu(1, 64);
    es = rng() % 3 ? 2 : 4;
    if ((double)d.T * d.F * (d.D + d.O) > 2e11) continue;  // a second's test
    roles(d, es, [&](const std::string& r) {
      seen.insert(r);
      if (!tested.count(r)) missing[r] = d;
    });
  }
  for (auto& [r, e] : missing)
    printf("not tested: %s (by T=%ld D=%d F=%d O=%d)\n", r.c_str(), (long)e.T, e.D, e.F, e.O);
  printf("%zu roles\n", seen.size());
  return !missing.empty() || seen.size() < 200;
}
"""


def test_every_role_is_tested(tmp_path):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    src, exe = tmp_path / "reach.cpp", tmp_path / "reach"
    src.write_text(REACH)
    subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(PKG_DIR, "csrc"), str(src), "-o",
                    str(exe)], check=True)
    shapes = "\n".join(f"{T} {D} {F} {O} {4 if dtype == 'f32' else 2}" for T, D, F, O, dtype in SHAPES)
    p = subprocess.run([str(exe)], input=shapes, capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stdout
