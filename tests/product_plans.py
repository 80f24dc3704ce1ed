"""Shapes of products by the plan they are meant for, and the plans that the library's rule
gives them (csrc/product_plan.h, compiled for the host)."""

from __future__ import annotations

import shutil
import subprocess
from typing import NamedTuple

from conftest import PKG

SMS = 148  # of a B200

_MAIN = r"""
#include <cinttypes>
#include <cstdio>
#include "product_plan.h"
int main() {
    int64_t t, k, n;
    int half, sms;
    while (std::scanf("%" SCNd64 " %" SCNd64 " %" SCNd64 " %d %d", &t, &k, &n, &half, &sms) == 5) {
        const tlb::ProductPlan p = tlb::plan_product(t, n, k, half != 0, sms);
        std::printf("%d %d %d %d %d %d %d %zu\n", p.tile_tokens, p.split, p.pair, p.chunks,
                    p.pieces, p.stages, p.ctas, p.smem);
    }
}
"""


class Plan(NamedTuple):
    tile_tokens: int
    split: int
    pair: int
    chunks: int
    pieces: int
    stages: int
    ctas: int
    smem: int

    def kind(self) -> str:
        if self.pair:
            return "pair"
        return f"cluster of {self.split}" if self.split > 1 else f"{self.chunks} a stage"


class Planner:
    def __init__(self, folder):
        (folder / "main.cpp").write_text(_MAIN)
        self.program = folder / "plans"
        subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O1", f"-I{PKG / 'csrc'}",
                        str(folder / "main.cpp"), "-o", str(self.program)], check=True)

    def __call__(self, shapes, sms=SMS) -> list[Plan]:
        """shapes: (tokens, width, features, results in 16 bits)."""
        lines = "".join(f"{t} {k} {n} {int(half)} {sms}\n" for t, k, n, half in shapes)
        out = subprocess.run([str(self.program)], input=lines, capture_output=True, text=True,
                             check=True).stdout
        return [Plan(*map(int, line.split())) for line in out.splitlines()]


# By kind of plan. "1 a stage" and "2 a stage": single CTAs with stages of one or two chunks of
# 128 values. Each kind has tiles of more stages than the ring holds, several tiles a CTA (or
# cluster, or pair), and a last group of 16 values.
SHAPES = {
    "1 a stage": [(1024, 2048, 2560), (640, 1168, 4096), (256, 1168, 16384), (1500, 272, 16384),
                  (128, 4112, 20000)],
    "2 a stage": [(64, 2048, 16384), (64, 1168, 20000), (300, 8192, 9728), (16, 272, 2560)],
    "cluster of 2": [(300, 8192, 2048), (9, 4112, 20000)],
    "cluster of 4": [(64, 8192, 2048), (33, 8192, 20000), (200, 4112, 640)],
    "pair": [(2048, 4096, 4096), (2500, 1168, 9728), (700, 4112, 20000)],
}
CASES = [shape for shapes in SHAPES.values() for shape in shapes]
