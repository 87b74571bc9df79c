"""How the gated feed-forward block's products are dealt out (csrc/gemm_plan.hpp,
csrc/gated_ffn_plan.hpp), on the CPU: every step of every tile is some block's,
once; every partial sum has a slot of its own inside the workspace; the join
reads exactly the slots of its tile, in order of k; padded copies and partial
sums do not overlap.  The walks repeat the kernels' indexing."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import PKG_DIR

WALK = r"""
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <random>
#include <vector>
#include "gated_ffn_plan.hpp"
using namespace mhc;

static long bad = 0, runs = 0, tails = 0, kinds[kKinds] = {}, few = 0;

static void fail(const char* what, const GemmShape& s, size_t es, int cus) {
  if (bad++ < 20)
    printf("%s: la=%d lb=%d epi=%d M=%lld N=%lld K=%lld es=%zu cus=%d\n", what, s.la, s.lb, s.epi, (long long)s.M,
           (long long)s.N, (long long)s.K, es, cus);
}

static void walk(const GemmShape& s, int64_t M, const GemmPlan& p, size_t es, int cus, size_t part) {
  GemmShape rows = s;
  rows.M = M;
  const KernelCost& c = kCosts[p.kind];
  const int64_t tiles = tiles_of(rows, c.bm, c.bn);
  const int64_t steps = (s.K * (int64_t)es + 127) / 128 * s.segments;
  ++kinds[p.kind];
  if (p.whole_tiles + p.run_tiles != tiles) fail("tiles", s, es, cus);
  if (s.la == kCol && c.bm < 64) fail("a kCol tile of fewer than 64 rows", s, es, cus);
  if (p.kind >= kWide128 && !p.dma) fail("a large tile through registers", s, es, cus);
  if (p.run_tiles == 0) return;
  ++runs;
  if ((size_t)2 * p.run_blocks * c.bm * c.bn * 4 > part) fail("partial sums past the workspace", s, es, cus);
  std::vector<std::vector<RunPiece>> of(p.run_tiles);
  for (int64_t b = 0; b < p.run_blocks; ++b) {
    int64_t have = 0;
    for (int i = 0;; ++i) {
      RunPiece r;
      if (!run_piece(b, i, p.run_tiles, (int)steps, p.run_blocks, &r)) break;
      if (i > 1) fail("a third piece", s, es, cus);
      if (r.tile < 0 || r.tile >= p.run_tiles || r.s0 < 0 || r.s1 > steps) { fail("a piece out of range", s, es, cus); break; }
      if (r.slot >= 2 * (int64_t)p.run_blocks) fail("a slot out of range", s, es, cus);
      have += r.s1 - r.s0;
      of[r.tile].push_back(r);
    }
    if (have < 1 || have != run_start(b + 1, p.run_tiles, (int)steps, p.run_blocks) - run_start(b, p.run_tiles, (int)steps, p.run_blocks))
      fail("a run's steps", s, es, cus);
  }
  for (int64_t t = 0; t < p.run_tiles; ++t) {
    int64_t at = 0;  // blocks were walked in order, so the pieces are in order of k
    for (const RunPiece& r : of[t]) {
      if (r.s0 != at) fail("a gap in a tile's steps", s, es, cus);
      at = r.s1;
    }
    if (at != steps) fail("a tile's last steps", s, es, cus);
    const RunBlocks rb = run_blocks_of(t, p.run_tiles, (int)steps, p.run_blocks);
    if (of[t].size() == 1) {
      if (rb.first != rb.last || of[t][0].slot != -1) fail("a whole tile that is joined", s, es, cus);
      continue;
    }
    if (rb.last - rb.first != (int64_t)of[t].size()) { fail("the join's blocks", s, es, cus); continue; }
    for (int64_t b = rb.first; b < rb.last; ++b)
      if (of[t][b - rb.first].slot != 2 * b + (b == rb.first && rb.begun_before)) fail("the join's slots", s, es, cus);
  }
}

static void product(const GemmShape& s, size_t es, int cus, size_t part) {
  const GemmPlans p = plan_gemm(s, es, cus);
  if (p.main_rows == 0) {
    ++few;
    if (s.M > kFewRows || s.la != kRow || s.lb != kRow) fail("no plan", s, es, cus);
    return;
  }
  walk(s, p.main_rows, p.main, es, cus, part);
  if (p.main_rows < s.M) ++tails, walk(s, s.M - p.main_rows, p.tail, es, cus, part);
}

static long copies = 0;

static void pass(const FfnDims& d, size_t es, int cus, bool back) {
  const FfnLines l(d, es, back, cus);
  const FfnWorkspace w(d, es, back, cus);
  const FfnShapes f(d, l, back);
  for (int i = 0; i < f.n; ++i) product(f.s[i], es, cus, w.part);
  copies += l.copy_D || l.copy_F || l.copy_O;
  // copies: whole 16-byte lines that hold the rows, in regions that hold them
  for (auto [copied, n, ld] : {std::tuple<bool, int64_t, int64_t>{l.copy_D, d.D, l.D}, {l.copy_F, d.F, l.F}, {l.copy_O, d.O, l.O}})
    if (copied ? ld < n || ld * es % 16 != 0 : ld != n) fail("a copy's lines", f.s[0], es, cus);
  if (l.copy_D && (w.x < (size_t)d.T * l.D * es || w.w < (size_t)d.F * l.D * es)) fail("copies of x, w", f.s[0], es, cus);
  if (l.copy_F && w.w_down < (size_t)d.O * l.F * es) fail("copy of w_down", f.s[0], es, cus);
  if (l.copy_O && w.grad_out < (size_t)d.T * l.O * es) fail("copy of grad_out", f.s[0], es, cus);
  if (w.hidden < (size_t)d.T * hidden_ld(d.F) * es) fail("hidden", f.s[0], es, cus);
  for (size_t n : {w.hidden, w.x, w.w, w.w_down, w.grad_out})
    if (n % 256 != 0) fail("a region's alignment", f.s[0], es, cus);
  if (w.bytes(back) != (back ? 2 : 1) * w.hidden + w.x + 2 * w.w + w.w_down + w.grad_out + w.part) fail("the sum", f.s[0], es, cus);
}

static void block(const FfnDims& d, size_t es, int cus) {
  for (int back = 0; back < 2; ++back) pass(d, es, cus, back);
}

int main() {
  std::mt19937_64 rng(1);
  auto uni = [&](double a, double b) { return a + (b - a) * (double)(rng() >> 11) / 9007199254740992.0; };
  auto logu = [&](double a, double b) { return (int64_t)exp2(uni(log2(a), log2(b))); };
  for (int i = 0; i < 6000; ++i) {
    const bool round = rng() % 2;
    auto width = [&] { const int64_t w = logu(1, 8000); return (int)(round && w >= 64 ? w / 64 * 64 : w); };
    FfnDims d = {logu(1, 20000), width(), (int)(1 + width() * uni(1, 3)), 0};
    if (round) d.F = (d.F + 63) / 64 * 64;
    d.O = rng() % 4 ? d.D : width();
    if (rng() % 5 == 0) d.T = 256 * logu(1, 40) + logu(1, 64);
    block(d, rng() % 3 ? 2 : 4, rng() % 8 ? 256 : (int)logu(1, 304));
  }
  for (int k = 0; k < kKinds; ++k) printf("%s%ld", k ? " " : "", kinds[k]);
  printf(" of each kernel, %ld few rows, %ld in runs, %ld tails, %ld copies, %ld faults\n", few, runs, tails, copies, bad);
  for (long n : kinds)
    if (n < 50) return 1;
  return bad || runs < 500 || tails < 50 || few < 100 || copies < 500;
}
"""


def test_every_step_once_and_every_sum_in_its_place(tmp_path):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text("#include <tuple>\n" + WALK)
    subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(PKG_DIR, "csrc"), str(src), "-o",
                    str(exe)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stdout
