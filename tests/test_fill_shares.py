"""Shares of the zeros that are written beside a sort cover every byte once, whatever the size."""

import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if not cxx:
        pytest.skip("no host compiler")
    exe = str(tmp_path_factory.mktemp("fill") / "fill_shares")
    subprocess.run([cxx, "-O1", "-std=c++17", "-o", exe, os.path.join(HERE, "fill_shares.cpp")], check=True)

    def run(cases):
        out = subprocess.run([exe], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in out.stdout.splitlines()]
    return run


def test_every_byte_once(replay):
    rng = random.Random(1)
    tables = [(8193, 1, 2), (1001, 1113, 2), (50257, 1201, 2), (32001, 769, 2), (513, 7681, 2), (128257, 2817, 2), (262145, 8194, 2), (262145, 4097, 4),
              (300001, 4129, 4), (2 ** 31 - 65536, 40, 4)]
    tables += [(rng.randint(1, 10 ** rng.randint(1, 6)), rng.randint(1, 10 ** rng.randint(1, 4)), rng.choice([2, 4])) for _ in range(20000)]
    cases = [(vocab * cols * size, shares, threads) for vocab, cols, size in tables for shares in (2, 4, 6, 8) for threads in (256, 512, 1024)]
    cases += [(4096 * shares * k + more, shares, 512) for shares in (2, 4, 6, 8) for k in (0, 1, 7) for more in range(2 * shares)]
    bad = [(c, r) for c, r in zip(cases, replay(cases), strict=True) if r != (0, 0, 0)]
    assert not bad, bad[:10]
