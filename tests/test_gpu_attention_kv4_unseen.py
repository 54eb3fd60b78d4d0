"""What a row does not see does not reach it: finite keys and values of any size beside much smaller ones, on the GPU
against 64 bits (kv_reference.py; its bounds go by what a row sees)."""
from __future__ import annotations

import numpy as np
import pytest

import kv_reference as R
from test_gpu_attention_kv4 import BOTH, KINDS, Setup

pytestmark = pytest.mark.gpu


def put(s, half, position, x):
    """Overwrites one token's keys or values (kv_heads, dim) of request 0, in the cache and in what the checks know."""
    codes, scales = R.quantize(x.astype(np.float32))
    s.cache.store(half, int(s.slots(0, np.array([position]))[0]), codes, scales)
    (s.k, s.v)[half][0][position] = R.values(codes, scales)
    (s.ks, s.vs)[half][0][position] = scales


def attend(hip, s, q, added, kind, most, window=0):
    torch = s.torch
    cache, table, lengths = s.device()
    starts = torch.tensor([0, added], dtype=torch.int32, device="cuda")
    print(f"unseen: lengths={s.lengths} dim={s.dim} {kind} max_added={most} window={window}", flush=True)
    return hip.attention_kv4(q, cache, table, lengths, starts, max_added=most, window=window)


def queries(torch, s, added, group, kind, size):
    q = size * np.random.default_rng(3).standard_normal((added, s.kv_heads * group, s.dim))
    return torch.from_numpy(q.astype(np.float32)).cuda().to(getattr(torch, KINDS[kind]))


def within(s, q, got, kind, window=0):
    want, bound = s.want(q.double().cpu().numpy(), [q.shape[0]], True, window, s.dim ** -0.5, kind)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), f"worst error is {(err / np.maximum(bound, 1e-300)).max()} of the bound"


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,group", [(64, 2), (128, 1), (128, 4), (256, 1)])
@pytest.mark.parametrize("most", BOTH)
@pytest.mark.parametrize("size", [1e2, 1e5])
def test_a_large_value_reaches_those_who_see_it(hip, torch_gpu, kind, dim, group, most, size):
    """Values around 1e-3 (scales around 2^-12) and one token's of `size`: rows before it are as exact as without it,
    wherever it lies in a step of 32 keys, in a tile of rows and in a group of tokens that are decoded together."""
    s = Setup(torch_gpu, [50], 1, dim, 16, seed=dim, v_size=1e-3)
    q = queries(torch_gpu, s, 50, group, kind, 0.3)
    clean = attend(hip, s, q, 50, kind, most)
    within(s, q, clean, kind)
    for token in (3, 15, 31, 32, 49):
        saved = s.v[0][token].copy(), s.vs[0][token].copy(), s.cache.bytes.copy()
        put(s, 1, token, size * np.linspace(0.5, 1, dim)[None] * (1 - 2 * (np.arange(dim) % 2)))
        got = attend(hip, s, q, 50, kind, most)
        within(s, q, got, kind)
        if most == 1:  # the same sums in the same order
            assert torch_gpu.equal(got[:token], clean[:token])
        s.v[0][token], s.vs[0][token], s.cache.bytes = saved


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("most", BOTH)
def test_a_large_key_reaches_those_who_see_it(hip, torch_gpu, kind, dim, most):
    """Keys around 1e-4, whose scales are below the normal numbers of fp16, and one token's of 1e5."""
    s = Setup(torch_gpu, [50], 1, dim, 16, seed=dim, k_size=1e-4)
    q = queries(torch_gpu, s, 50, 1, kind, 3e4)
    for token in (15, 31, 32):
        saved = s.k[0][token].copy(), s.ks[0][token].copy(), s.cache.bytes.copy()
        put(s, 0, token, 1e5 * np.linspace(0.5, 1, dim)[None] * (1 - 2 * (np.arange(dim) % 2)))
        within(s, q, attend(hip, s, q, 50, kind, most), kind)
        s.k[0][token], s.ks[0][token], s.cache.bytes = saved


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("most", BOTH)
@pytest.mark.parametrize("window", [9, 40])
def test_a_large_value_before_the_window(hip, torch_gpu, kind, most, window):
    """Rows whose window has left the large token behind, beside rows that still see it."""
    s = Setup(torch_gpu, [90], 1, 128, 16, seed=5, v_size=1e-3)
    q = queries(torch_gpu, s, 60, 2, kind, 0.3)
    for token in (20, 44, 60):
        saved = s.v[0][token].copy(), s.vs[0][token].copy(), s.cache.bytes.copy()
        put(s, 1, token, 1e5 * np.linspace(0.5, 1, 128)[None])
        within(s, q, attend(hip, s, q, 60, kind, most, window), kind, window)
        s.v[0][token], s.vs[0][token], s.cache.bytes = saved
