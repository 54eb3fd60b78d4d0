"""Launches of attention_kv4 that the sizes of an ordinary test do not reach, on the GPU against 64 bits: each test asserts
that the plan takes the path that it is for."""
from __future__ import annotations

import numpy as np
import pytest

import kv_reference as R
from test_attention_plan import BF16, F16, F32, plan  # noqa: F401 (a fixture)
from test_gpu_attention_kv4 import BOTH, KINDS, Setup, check
from test_gpu_attention_kv4_unseen import put

pytestmark = pytest.mark.gpu

TYPES = {"f32": F32, "bf16": BF16, "f16": F16}


def planned(plan, s, kind, added, group, max_added, max_length, causal=True):
    p = plan(TYPES[kind], sum(added), len(added), s.kv_heads * group, s.kv_heads, s.dim, max_added, max_length, causal)
    return list(p.launch)[:p.launches]


def parts_of(launch, s, r, added, window, tile_rows, group):
    """The parts that the first row tile of request r has of its keys, as the kernels count them."""
    keys = 64 * 128 // s.dim if launch.prompt else 32
    first = s.lengths[r] - added
    low = max(0, first - window + 1) // keys * keys if window else 0
    steps = -(-(min(first + -(-tile_rows // group), s.lengths[r]) - low) // keys)
    per = launch.per if steps <= launch.per * launch.parts else -(-steps // launch.parts)
    return -(-steps // per)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,heads", [(64, 1), (128, 1), (256, 1), (128, 2)])
@pytest.mark.parametrize("window", [0, 1500])
def test_prompts_in_parts(hip, plan, torch_gpu, kind, dim, heads, window):
    """The tile kernel with a row's keys in several parts; with a window parts that start behind the first key."""
    s = Setup(torch_gpu, [3000], heads, dim, 16, seed=dim + window)
    launch, = planned(plan, s, kind, [100], 4, 2048, 3000)
    assert launch.prompt and parts_of(launch, s, 0, 100, window, 256 if dim < 256 else 128, 4) > 1
    check(hip, s, 4, [100], kind, window=window, max_added=2048, max_length=3000)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_nan_in_one_part_of_a_prompt(hip, plan, torch_gpu, kind, dim):
    """A value of one part's keys: its block of the rows that see it, through the join."""
    torch = torch_gpu
    s = Setup(torch, [3000], 1, dim, 16, seed=2)
    launch, = planned(plan, s, kind, [100], 4, 2048, 3000)
    assert launch.prompt and parts_of(launch, s, 0, 100, 0, 256, 4) > 1
    q = torch.randn(100, 4, dim, device="cuda").to(getattr(torch, KINDS[kind]))
    starts = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    cache, table, lengths = s.device()
    print(f"nan in a part: dim={dim} {kind}", flush=True)
    for window in (0, 60):
        run = lambda: hip.attention_kv4(q, cache, table, lengths, starts, max_added=2048, max_length=3000, window=window)
        clean = run()
        for token in (1000, 2890, 2950):
            slots = torch.from_numpy(s.slots(0, np.array([token])).astype(np.int32)).cuda()
            saved = cache.clone()
            k, v = hip.kv4_read(cache, slots, dim)
            v[0, 0, 40] = float("nan")
            hip.kv4_store(k, v, slots, cache)
            got = run()
            cache.copy_(saved)
            position = torch.arange(2900, 3000, device="cuda")
            sees = (position >= token) & ((position - token < window) | (window == 0))
            assert got[sees][:, :, 32:64].isnan().all()
            keep = torch.ones_like(got, dtype=torch.bool)
            keep[sees, :, 32:64] = False
            # the tile is marked: its exponents move their base earlier
            assert torch.allclose(got[keep].float(), clean[keep].float(), rtol=2.0 ** -6, atol=1e-3)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 400])
def test_a_tiled_prompt_beside_running_requests(hip, plan, torch_gpu, kind, dim, window):
    added = [1, 90, 4, 5, 0, 2]
    s = Setup(torch_gpu, [1500, 800, 40, 300, 70, 1100], 1, dim, 16, seed=dim)
    launches = planned(plan, s, kind, added, 8, 1500, 3000)
    assert [a.prompt for a in launches] == [True, False] and launches[1].parts > 1
    check(hip, s, 8, added, kind, window=window, max_added=1500, max_length=3000)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_more_row_tiles_than_planned(hip, plan, torch_gpu, dim):
    """max_added below what a request adds: a workgroup of the tile kernel takes several row tiles."""
    s = Setup(torch_gpu, [900], 1, dim, 16, seed=dim)
    launch, = planned(plan, s, "bf16", [700], 4, 520, 4000)
    assert launch.prompt and launch.tiles * (256 if dim < 256 else 128) < 700 * 4
    check(hip, s, 4, [700], "bf16", max_added=520, max_length=4000)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [700, 1501])
def test_windows_in_parts(hip, plan, torch_gpu, kind, dim, window):
    """Single tokens whose window starts inside a later page, in several parts of their keys."""
    s = Setup(torch_gpu, [3000, 2011, 100], 2, dim, 16, seed=window)
    launch, = planned(plan, s, kind, [1, 1, 1], 2, 1, 3000)
    assert not launch.prompt and parts_of(launch, s, 0, 1, window, 16, 2) > 1
    check(hip, s, 2, [1, 1, 1], kind, window=window, max_length=3000)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_many_steps_of_a_wave(hip, plan, torch_gpu, kind):
    """More than 64 steps a wave: its pages are looked up 64 steps at a time."""
    s = Setup(torch_gpu, [17500], 1, 64, 16, seed=1)
    launch, = planned(plan, s, kind, [1], 4, 1, 32)
    assert launch.parts == 1 and 17500 // 32 // launch.waves > 64
    check(hip, s, 4, [1], kind, max_length=32)


@pytest.mark.parametrize("page", [256, 1024])
@pytest.mark.parametrize("kind,dim", [("f32", 128), ("bf16", 64), ("bf16", 256)])
def test_large_pages(hip, torch_gpu, page, kind, dim):
    s = Setup(torch_gpu, [1500, 300], 2, dim, page, seed=page)
    check(hip, s, 2, [1, 1], kind)
    check(hip, s, 2, [40, 70], kind)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window", [5, 33, 100])
def test_windows_of_wide_heads(hip, torch_gpu, kind, window):
    s = Setup(torch_gpu, [150, 61], 1, 256, 16, seed=window)
    check(hip, s, 2, [70, 20], kind, window=window)
    check(hip, s, 2, [1, 1], kind, window=window, with_starts=True)


@pytest.mark.parametrize("most", BOTH)
@pytest.mark.parametrize("starts,rows", [([0, 4, 1000], {0: (0, 4), 1: (4, 10)}), ([-5, 4, 10], {0: (0, 4), 1: (4, 10)}),
                                         ([6, 2, 10], {1: (2, 10)}), ([3, 3, 7], {1: (3, 7)})])
def test_starts_outside_the_tokens(hip, torch_gpu, most, starts, rows):
    """Starts are cut to the tokens there are: what they leave a request is right, and nothing around the result is written."""
    torch = torch_gpu
    s = Setup(torch, [40, 40], 1, 64, 16, seed=14)
    cache, table, lengths = s.device()
    q = torch.randn(10, 2, 64, device="cuda")
    buffer = torch.full((30, 3, 64), 7.0, device="cuda")
    print(f"starts {starts} max_added={most}", flush=True)
    hip.attention_kv4(q, cache, table, lengths, torch.tensor(starts, dtype=torch.int32, device="cuda"), max_added=most,
                      out=buffer[10:20, :2])
    got = buffer.cpu()
    assert (got[:10] == 7).all() and (got[20:] == 7).all() and (got[:, 2] == 7).all()
    for r, (a, b) in rows.items():
        want, bound = R.attention(q[a:b].double().cpu().numpy(), s.k[r], s.v[r], s.ks[r], s.vs[r], 40 - (b - a), 40, True, 0,
                                  64 ** -0.5, "f32")
        assert (np.abs(got[10 + a:10 + b, :2].double().numpy() - want) <= bound).all()


def test_values_that_grow_over_eight_orders(hip, torch_gpu):
    """From 1e-4 to 1e4 along the context, in every type's kernels of few and of many rows."""
    s = Setup(torch_gpu, [800], 1, 128, 16, seed=8)
    rng = np.random.default_rng(2)
    for i in range(800):
        put(s, 1, i, rng.standard_normal((1, 128)) * 10.0 ** (i / 100 - 4))
    for kind in KINDS:
        for added in ([1], [60]):
            check(hip, s, 2, added, kind, with_starts=True)


def test_a_hint_far_above_the_tokens(hip, plan, torch_gpu):
    """512 single tokens with a max_added of 131072: one row tile of many has work, and the launch has to be one."""
    torch = torch_gpu
    s = Setup(torch, [40] * 512, 8, 64, 16, seed=3, extra=1)
    assert max(a.tiles for a in planned(plan, s, "bf16", [1] * 512, 8, 131072, 8192)) > 100
    cache, table, lengths = s.device()
    q = torch.randn(512, 64, 64, device="cuda").bfloat16()
    print("hint of 131072", flush=True)
    want = hip.attention_kv4(q, cache, table, lengths)
    got = hip.attention_kv4(q, cache, table, lengths, max_added=131072, max_length=8192)
    assert torch.allclose(got.float(), want.float(), rtol=2.0 ** -7, atol=1e-2)
