"""Sizes whose launch HIP would not take (2^32 threads and more) are refused as arguments, before the device is touched
(CPU only)."""
from __future__ import annotations

import pytest

from test_kv_api import attend, norm, read, store

# a row is a token's head; 8 elements a thread, whole workgroups of 256
REFUSED = [
    (norm, {"tokens": 1 << 28, "heads": 1, "dim": 128}),
    (norm, {"tokens": 1 << 27, "heads": 1, "dim": 256, "rot": 256}),
    (norm, {"tokens": 1 << 29, "heads": 1, "dim": 64, "rot": 64}),
    (norm, {"tokens": (1 << 28) - 15, "heads": 1, "dim": 128}),  # one more workgroup than there may be
    (store, {"tokens": 1 << 27, "heads": 1, "dim": 256, "pages": 1 << 20}),
    (store, {"tokens": 1 << 28, "heads": 1, "pages": 1 << 20}),
    (store, {"tokens": 1 << 25, "heads": 8, "pages": 1 << 20, "stride": 1024}),
    (read, {"tokens": 1 << 27, "heads": 1, "dim": 256}),
    (read, {"tokens": 1 << 29, "heads": 1, "dim": 64}),
    (attend, {"requests": 1 << 23, "tokens": 1 << 23, "kv_heads": 2}),
    (attend, {"requests": 1 << 24, "tokens": 4, "kv_heads": 1}),
]


@pytest.mark.parametrize("call,change", REFUSED, ids=[f"{c.__name__}-{k}" for c, k in REFUSED])
def test_refused(pkg, call, change):
    assert call(pkg.lib(), **change) == pkg.ERR_INVALID_ARGUMENT
    assert pkg.last_error()


def test_workspace_query_refuses_the_same(pkg):
    f = pkg.lib().pfng_hip_attention_kv4_workspace_size
    assert f(1, 1 << 23, 1 << 23, 4, 2, 128, 1, 1, 64) == -1 and pkg.last_error()
    assert f(1, 4, 1 << 24, 4, 1, 128, 1, 1, 64) == -1


@pytest.mark.parametrize("call,change", [
    (norm, {"tokens": (1 << 28) - 16, "heads": 1, "dim": 128}), (store, {"tokens": (1 << 28) - 16, "heads": 1, "pages": 1 << 20}),
    (read, {"tokens": (1 << 28) - 16, "heads": 1}), (attend, {"requests": (1 << 23) - 1, "tokens": (1 << 23) - 1, "kv_heads": 2}),
])
def test_up_to_there_arguments_are_taken(pkg, call, change):
    """Without a device the call gets as far as the launch."""
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("would launch on pointers that are none")
    assert call(pkg.lib(), **change) == pkg.ERR_HIP
