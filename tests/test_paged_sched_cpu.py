"""CPU: the work line of the paged-attention kernels (paged_sched.cuh), run on
the host: every unit's keys come exactly once, in order, whatever the lengths
and however many steps they are."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    exe = tmp_path_factory.mktemp("sched") / "paged_sched_host"
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "zlift_b200", "csrc"),
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
                    os.path.join(ROOT, "tests", "paged_sched_host.cpp"), "-o", str(exe)], check=True)

    def run(tokens, keys, least, pieces, causal, heads, page, table_pages, seqs):
        text = [tokens, keys, least, pieces, int(causal), heads, page, table_pages, len(seqs)]
        text += [x for pair in seqs for x in pair]
        out = subprocess.run([str(exe)], input=" ".join(map(str, text)), capture_output=True, text=True,
                             check=True, timeout=300).stdout.split()
        return [int(x) for x in out]                         # step, units, keys, bad
    return run


def expected(tokens, causal, heads, seqs):
    units = keys = 0
    for n, length in seqs:
        for i in range(0, n, tokens):
            units += 1
            keys += max(0, min(length, length - n + min(n, i + tokens))) if causal else length
    return [units * heads, keys * heads]


CALLS = {
    "one token": (1, 16, 3, 64, True, 2, 16, 64, [(1, 515)]),
    "no keys": (4, 32, 3, 64, True, 8, 16, 4, [(1, 0), (3, 0)]),
    "rows that see nothing": (32, 128, 2, 20, True, 3, 16, 4, [(90, 40), (5, 1)]),
    "empty sequences": (2, 16, 3, 64, True, 4, 8, 40, [(0, 9), (3, 300), (0, 0), (0, 5), (1, 17), (0, 3)]),
    "more sequences than lanes": (1, 64, 3, 300, True, 2, 16, 64, [(i % 3, 7 * i % 900) for i in range(133)]),
    "one unit for all pieces": (3, 16, 3, 592, True, 1, 64, 2048, [(3, 131072)]),
    "chunks": (64, 128, 2, 148, True, 8, 16, 256, [(2048, 4096), (1033, 1100), (2047, 3000), (1500, 1500)]),
    "not causal": (64, 128, 2, 148, False, 8, 16, 256, [(2048, 4096), (1, 1100), (70, 30)]),
}


@pytest.mark.parametrize("name", CALLS)
def test_every_key_once(walk, name):
    c = CALLS[name]
    step, units, keys, bad = walk(*c)
    assert bad == 0 and step == c[1] and [units, keys] == expected(c[0], c[4], c[5], c[8])


def test_more_steps_than_32_bits(walk):
    """A long chunk in tiles of a token each: 131072 x 4096 steps on average, for
    each of 8 heads, is 2^32."""
    seqs = [(131072, 131072)]
    step, units, keys, bad = walk(1, 16, 3, 48, True, 8, 16, 8192, seqs)
    assert bad == 0 and step > 16 and [units, keys] == expected(1, True, 8, seqs)


def test_a_wide_table_alone_costs_nothing(walk):
    """A table for long contexts and a batch of single tokens: fine steps."""
    seqs = [(1, 100 + i) for i in range(96)]
    step, units, keys, bad = walk(1, 16, 3, 64, True, 8, 16, 8192, seqs)
    assert bad == 0 and step == 16 and [units, keys] == expected(1, True, 8, seqs)


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(walk, seed):
    r = random.Random(seed)
    seqs = [(r.choice([0, 1, 1, r.randint(1, 400)]), r.randint(0, 3000)) for _ in range(r.randint(1, 70))]
    seqs.append((1, 5))
    tokens, keys = r.choice([(1, 16), (4, 32), (6, 64), (32, 128)])
    call = (tokens, keys, r.randint(1, 3), r.choice([1, 7, 60, 148]), r.random() < 0.7, r.randint(1, 8), 16,
            200, seqs)
    step, units, found, bad = walk(*call)
    assert bad == 0 and step == keys and [units, found] == expected(tokens, call[4], call[5], seqs)
