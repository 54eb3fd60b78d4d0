"""Scores of any size that fp32 holds: the exponents' base is a whole number in fp32, and past 2^24 it cannot stand
everywhere."""
from __future__ import annotations

import numpy as np
import pytest

import kv_reference as R
from test_gpu_attention_kv4 import BOTH, KINDS, Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("most", BOTH)
@pytest.mark.parametrize("alike", [False, True])
def test_scores_past_the_units_of_fp32(hip, torch_gpu, kind, dim, most, alike):
    """Queries from 1e6 to 1e12 times as large as usual. alike: keys of whole numbers of which a few differ by little, so
    that scores lie within some units of each other."""
    torch = torch_gpu
    s = Setup(torch, [80], 1, dim, 16, seed=dim)
    if alike:
        from test_gpu_attention_kv4_unseen import put
        rng = np.random.default_rng(1)
        one = 8.0 * (1 - 2 * rng.integers(0, 2, dim))
        one[1::32] = 1
        for i in range(80):
            x = one.copy()
            x[1::32] = rng.integers(-1, 2, dim // 32)
            put(s, 0, i, x[None])
    cache, table, lengths = s.device()
    starts = torch.tensor([0, 80], dtype=torch.int32, device="cuda")
    for size in 10.0 ** np.arange(6, 12.5, 0.5):
        q = size * np.random.default_rng(3).standard_normal((80, 1, dim))
        if alike:
            q = size * np.sign(s.k[0][40, 0]) * np.ones((80, 1, 1))
            q[:, :, 1::32] = 1e-6 * size
        q = torch.from_numpy(q.astype(np.float32)).cuda().to(getattr(torch, KINDS[kind]))
        print(f"scores: dim={dim} {kind} max_added={most} alike={alike} size={size}", flush=True)
        got = hip.attention_kv4(q, cache, table, lengths, starts, max_added=most).double().cpu().numpy()
        assert np.isfinite(got).all()
        x = q.double().cpu().numpy()
        for i in range(80):
            seen = s.v[0][:i + 1, 0]
            # a mean of what the row sees, whatever the weights
            room = 2.0 ** -7 * np.abs(seen).max(0)
            assert (got[i, 0] <= seen.max(0) + room).all() and (got[i, 0] >= seen.min(0) - room).all()
            scores = dim ** -0.5 * (s.k[0][:i + 1, 0] @ x[i, 0])
            order = np.argsort(scores)
            reach = dim ** -0.5 * (np.abs(x[i, 0]) @ (8 * np.repeat(np.abs(s.ks[0][:i + 1, 0]), 32, -1)).T).max()
            # one score above the others by more than keys and queries of 11 bits leave open
            if i == 0 or scores[order[-1]] - scores[order[-2]] > reach * 2.0 ** -9 + 30:
                only = seen[order[-1]]
                # the result's rounding, and for bf16 those of a probability and of a value to fp16
                assert (np.abs(got[i, 0] - only) <= R.rounding(only, kind) + 2.0 ** -11 * np.abs(only) + 1e-6).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("most", BOTH)
def test_queries_up_to_the_end_of_fp32(hip, torch_gpu, kind, dim, most):
    """Queries of 1e34 to 3e38 with keys of 1e-6: scores that fp32 holds, and the largest of which takes all."""
    torch = torch_gpu
    s = Setup(torch, [40], 1, dim, 16, seed=dim, k_size=1e-6)
    cache, table, lengths = s.device()
    starts = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    for size in (1e34, 1e36, 1e37, 1e38, 3e38):
        q = size * np.random.default_rng(3).uniform(-1, 1, (40, 1, dim))
        q = torch.from_numpy(q.astype(np.float32)).cuda().to(getattr(torch, KINDS[kind]))
        print(f"scores: dim={dim} {kind} max_added={most} size={size}", flush=True)
        got = hip.attention_kv4(q, cache, table, lengths, starts, max_added=most).double().cpu().numpy()
        assert np.isfinite(got).all()
        x = q.double().cpu().numpy()
        for i in range(40):
            scores = dim ** -0.5 * (s.k[0][:i + 1, 0] @ x[i, 0])
            order = np.argsort(scores)
            reach = dim ** -0.5 * (np.abs(x[i, 0]) @ (8 * np.repeat(np.abs(s.ks[0][:i + 1, 0]), 32, -1)).T).max()
            if i == 0 or scores[order[-1]] - scores[order[-2]] > reach * 2.0 ** -9:
                only = s.v[0][order[-1], 0]
                assert (np.abs(got[i, 0] - only) <= R.rounding(only, kind) + 2.0 ** -11 * np.abs(only) + 1e-6).all()
