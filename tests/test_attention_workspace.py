"""The workspace of linear attention against the sizes that the header states."""
import ctypes

import pytest

from salt_b200 import _lib

F32, F16, BF16 = 0, 1, 2
PARTS = {F32: 3, F16: 2, BF16: 1}


def up(n):
    return -(-n // 256) * 256


def planes(kind, batch, n, heads, dim):
    return up(2 * PARTS[kind] * batch * n * heads * (-(-dim // 8) * 8))


def asked(batch, n, heads, kv, dk, dv, kind, backward=False):
    Args = _lib.LinearAttentionBackwardArgs if backward else _lib.LinearAttentionArgs
    a = Args(batch=batch, len=n, heads=heads, kv_heads=kv, dim_k=dk, dim_v=dv, type=kind, scale=1.0)
    for name, width in (("q", heads * dk), ("k", kv * dk), ("v", kv * dv), ("out", heads * dv),
                        ("dout", heads * dv), ("dq", heads * dk), ("dk", kv * dk),
                        ("dv", kv * dv)):
        if not hasattr(a, name):
            continue
        setattr(a, name, 2)  # bfloat16 off every boundary; nothing is read
        setattr(a, name + "_stride", width)
        setattr(a, name + "_batch_stride", width * n)
    a.log_decay = 16
    size = ctypes.c_size_t(0)
    lib = _lib.lib()
    query = (lib.salt_linear_attention_backward_workspace_size if backward
             else lib.salt_linear_attention_workspace_size)
    _lib.check(query(bytes(a), ctypes.byref(size)))
    return size.value


CASES = ((64, 100, 8, 8, 64, 64), (64, 37, 8, 2, 1, 1), (32, 300, 16, 4, 75, 50), (64, 1, 4, 1, 128, 9))


@pytest.mark.parametrize("kind", PARTS)
@pytest.mark.parametrize("batch, n, heads, kv, dk, dv", CASES)
def test_planes_and_shared_heads(kind, batch, n, heads, kv, dk, dv):
    """Enough heads to keep rows whole."""
    rows = (planes(kind, batch, n, heads, dk) + planes(kind, batch, n, kv, dk)
            + planes(kind, batch, n, kv, dv))
    assert asked(batch, n, heads, kv, dk, dv, kind) == rows
    rows += planes(kind, batch, n, heads, dv)
    if kv < heads:
        rows += up(4 * batch * n * heads * max(dk, dv))
    assert asked(batch, n, heads, kv, dk, dv, kind, backward=True) == rows


@pytest.mark.parametrize("kind", PARTS)
@pytest.mark.parametrize("backward", (False, True))
def test_states_of_segments(kind, backward):
    """Few heads: at most 64 states a head beside the planes."""
    batch, n, heads, dk, dv = 1, 20000, 2, 64, 48
    rest = asked(batch, n, heads, heads, dk, dv, kind, backward) - sum(
        planes(kind, batch, n, heads, d) for d in ((dk, dk, dv, dv) if backward else (dk, dk, dv)))
    state = 4 * heads * dk * dv
    assert 2 * state <= rest <= up(64 * state) and rest % state < 256
