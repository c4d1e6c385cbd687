"""The barriers of attend_tiles (csrc/sc_attention_tile.cu) as a model whose every interleaving is
walked through on the CPU: no warp reads sums that a product still has to reach, no score lands on
weights that a product still reads, nothing waits for ever.

Agents are the warp that issues the products, the tensor cores (products end in the order they were
issued in) and softmax warps, each of which may lag behind the others and may or may not raise its
maximum at any tile.  Waits name a phase by its parity, as the hardware's do.  Which phase a softmax warp
waits for before it hands its last weights over comes from csrc/sc_tile_waits.h itself.
"""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest

from conftest import REPO

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")

WARPS = 2  # of the four; what two can do to one another, more can


@pytest.fixture(scope="module")
def phase_before_weights(tmp_path_factory):
    out = tmp_path_factory.mktemp("waits")
    src, so = out / "waits.cpp", out / "waits.so"
    src.write_text('#include "sc_tile_waits.h"\n'
                   'extern "C" int phase(int q, int i, int n) { return sc::phase_before_weights(q, i, n); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{REPO}/intelligent-bell_b200/csrc", str(src),
                    "-o", str(so)], check=True)
    return ctypes.CDLL(str(so)).phase


def passes(over: int, phase: int) -> bool:
    """Whether a wait for ``phase`` returns when that many phases of the barrier are over."""
    return over & 1 != phase & 1


def issued_products(n_q: int, n: int):
    """The issuing warp's steps: ('score' or 'sum', row tile, token tile, waits), a wait being a barrier and
    a phase.  One row tile: two score buffers in turn; two: one each."""
    steps = []
    if n_q == 1:
        steps.append(("score", 0, 0, []))
        for i in range(n):
            if i + 1 < n:
                steps.append(("score", 0, i + 1, [("o", 0, i - 1)] if i > 0 else []))
            steps.append(("sum", 0, i, [("p", i & 1, i >> 1)]))
        return steps
    steps += [("score", q, 0, []) for q in range(2)]
    for i in range(n):
        for q in range(2):
            steps.append(("sum", q, i, [("p", q, i)]))
            if i + 1 < n:
                steps.append(("score", q, i + 1, [("o", q, i)]))
    return steps


def faults(n_q: int, n: int, before) -> set[str]:
    """What can go wrong in some interleaving of n token tiles."""
    steps = issued_products(n_q, n)
    found: set[str] = set()
    buf = lambda q, i: i & 1 if n_q == 1 else q
    turn = lambda i: i >> 1 if n_q == 1 else i  # of a score buffer
    warps = [(q, w) for q in range(n_q) for w in range(WARPS)]
    # state: steps issued, steps ended, and per softmax warp (tile, stage)
    # stages: 0 waits for scores, 1 may raise, 2 hands over, 3 waits for the sums, 4 done
    start = (0, 0, tuple((0, 0) for _ in warps))
    seen, todo = {start}, [start]
    while todo:
        issued, ended, at = todo.pop()
        done = [s for s in steps[:ended]]
        sums = [sum(1 for s in done if s[0] == "sum" and s[1] == q) for q in range(n_q)]  # o phases over
        scores = [sum(1 for s in done if s[0] == "score" and buf(s[1], s[2]) == b) for b in range(2)]
        handed = [0, 0]  # p phases over: the slowest warp's
        for b in range(2):
            tiles = [[i for i in range(n) if buf(q, i) == b] for q in range(n_q)]
            per = [sum(1 for i in tiles[q] if i < t or (i == t and s >= 3))
                   for (q, _), (t, s) in zip(warps, at) if tiles[q]]
            handed[b] = min(per) if per else 0
        after = []
        if ended < issued:
            after.append((issued, ended + 1, at))
        if issued < len(steps):
            kind, q, i, waits = steps[issued]
            if all(passes(sums[k] if w == "o" else handed[k], ph) for w, k, ph in waits):
                if kind == "score" and i - (2 if n_q == 1 else 1) >= sums[q]:
                    found.add("scores land on weights that a product still reads")
                if kind == "sum" and handed[buf(q, i)] <= turn(i):
                    found.add("a product reads weights that are not there")
                after.append((issued + 1, ended, at))
        for k, ((q, _), (i, stage)) in enumerate(zip(warps, at)):
            def to(*x):
                after.append((issued, ended, at[:k] + (x,) + at[k + 1:]))

            if stage == 0 and passes(scores[buf(q, i)], turn(i)):
                if scores[buf(q, i)] <= turn(i):
                    found.add("weights of scores that are not there")
                to(i, 1)
            elif stage == 1:
                to(i, 2)  # keeps its maximum
                if i > 0 and passes(sums[q], i - 1):
                    if sums[q] < i:
                        found.add("sums scaled while a product reaches them")
                    to(i, 2)
            elif stage == 2:
                phase = before(n_q, i, n)
                if phase < 0 or passes(sums[q], phase):
                    if phase >= 0 and sums[q] <= phase:
                        found.add("a wait answered by an earlier phase")
                    to(*((i, 3) if i == n - 1 else (i + 1, 0)))
            elif stage == 3 and passes(sums[q], n - 1):
                if sums[q] < n:
                    found.add("sums read before the last products")
                to(i, 4)
        if not after and not (ended == len(steps) and all(s == 4 for _, s in at)):
            found.add("waits for ever")
        for x in after:
            if x not in seen:
                seen.add(x)
                todo.append(x)
    return found


@pytest.mark.parametrize("n_q", [1, 2])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
def test_every_interleaving_is_sound(phase_before_weights, n_q, n):
    assert faults(n_q, n, phase_before_weights) == set()


@pytest.mark.parametrize("n", [2, 3, 4])
def test_the_model_sees_what_the_wait_is_for(n):
    """Without it a warp that is a tile ahead takes the phase two before for the last one."""
    assert faults(1, n, lambda q, i, m: -1) == {"sums read before the last products"}
    assert faults(2, n, lambda q, i, m: -1) == set()
