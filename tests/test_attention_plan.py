"""The plan of an attention call (csrc/attention_kv4.hip, on the CPU): launches that HIP takes, of every request once, over
sizes up to those that the entry point accepts."""
from __future__ import annotations

import ctypes
import itertools
import random

import pytest

CUS = 256
F32, BF16, F16 = 0, 1, 2


class Launch(ctypes.Structure):
    _fields_ = [("prompt", ctypes.c_bool), ("tiles", ctypes.c_int), ("parts", ctypes.c_int), ("per", ctypes.c_int),
                ("waves", ctypes.c_int), ("least", ctypes.c_int), ("most", ctypes.c_int)]


class Plan(ctypes.Structure):
    _fields_ = [("launch", Launch * 2), ("launches", ctypes.c_int), ("splits", ctypes.c_int)]


@pytest.fixture(scope="module")
def plan(pkg):
    # pfng::plan_attention(int, long, long, int, int, int, long, long, bool, int)
    f = pkg.lib()._ZN4pfng14plan_attentionEilliiillbi
    f.restype = Plan
    f.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int64,
                  ctypes.c_int64, ctypes.c_bool, ctypes.c_int]
    return lambda kind, tokens, requests, heads, kv_heads, dim, max_added, max_length, causal=True: f(
        kind, tokens, requests, heads, kv_heads, dim, max_added, max_length, causal, CUS)


def check(plan, kind, tokens, requests, heads, kv_heads, dim, max_added, max_length, causal=True):
    case = (kind, tokens, requests, heads, kv_heads, dim, max_added, max_length, causal)
    p = plan(*case)
    assert p.launches in (1, 2), case
    launches = list(p.launch)[:p.launches]
    for a in launches:
        assert a.tiles >= 1 and 1 <= a.parts <= 256 and a.per >= 1 and a.waves in (4, 8), case
        threads = 64 * (a.waves if not a.prompt else 4 if dim == 256 else 8)
        # HIP takes fewer than 2^32 threads a launch
        assert requests * kv_heads * a.tiles * a.parts * threads < 1 << 32, (case, a.tiles, a.parts, threads)
    # every number of new tokens belongs to one launch
    for added in {0, 1, 3, 4, 5, 6, 100, max_added, tokens, (1 << 30)}:
        assert sum(a.least <= added <= a.most for a in launches) == 1, case
    assert p.splits == max(a.parts for a in launches), case
    if p.splits > 1:  # joined by 16 threads a row, or by 256 a row where there are few
        rows = tokens * heads
        assert rows * 16 + 256 < 1 << 32, case
        if p.splits > 4 and rows <= 512 * p.splits:
            assert rows * 256 < 1 << 32, case
    return p


@pytest.mark.parametrize("tokens,requests,max_added,max_length", [
    (32768 + 1023, 1024, 32768, 32768),    # a long prompt beside running requests
    (131072 + 255, 256, 131072, 131072),
    (8192 + 4095, 4096, 8192, 8192),
    (512, 512, 131072, 8192),              # max_added far above what is there
    (1, 1, 1 << 30, 1 << 30),
    (4096, 4096, 1 << 30, 1 << 30),
])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_steps(plan, tokens, requests, max_added, max_length, kind, dim):
    for heads, kv_heads in ((64, 8), (64, 64), (32, 1), (128, 8)):
        check(plan, kind, tokens, requests, heads, kv_heads, dim, max_added, max_length)


def test_drawn_steps(plan):
    """Requests, tokens and hints over their whole ranges."""
    rng = random.Random(0)
    whole = lambda top: int(2 ** rng.uniform(0, top))
    for _ in range(20000):
        kv_heads = rng.choice([1, 2, 3, 8, 40, 128])
        heads = kv_heads * rng.choice([1, 2, 4, 7, 16])
        requests = min(whole(24), ((1 << 24) - 1) // kv_heads)
        tokens = rng.choice([requests, requests - 1 + whole(20), whole(24)])
        tokens = min(tokens, (1 << 32) // heads)
        check(plan, rng.choice([F32, BF16, F16]), tokens, requests, heads, kv_heads, rng.choice([64, 128, 256]),
              rng.choice([1, whole(10), whole(30), max(1, tokens)]), rng.choice([0, whole(15), whole(30)]), rng.random() < 0.8)


def test_ordinary_steps_are_two_launches_where_prompts_and_running_requests_meet(plan):
    p = check(plan, BF16, 2048 + 31, 32, 32, 8, 128, 2048, 8192)
    assert p.launches == 2 and p.launch[0].prompt and not p.launch[1].prompt
    assert (p.launch[0].least, p.launch[1].most) == (5, 4) and p.launch[0].tiles == 2048 * 4 // 256
    for requests, added in itertools.product((1, 8), (1, 64, 4096)):
        assert check(plan, BF16, requests * added, requests, 32, 8, 128, added, 8192).launches == 1
