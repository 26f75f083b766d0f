"""not-gpu: the buffers that the head losses ask for, against what their documentation promises."""
import ctypes

import pytest

from neuron_interpolation_model_fusion_amd import _lib

MIB = 1 << 20


def _bytes(n, d, v, dtype, k, ldw):
    p = ctypes.c_void_p(4096)
    h = _lib.HeadDesc(hidden=p, ldh=d, weight=p, ldw=ldw, rows=n, features=d, classes=v, dtype=dtype, reduction=_lib.NIF_REDUCE_MEAN,
                      labels=p if k == 0 else None, top_indices=p if k else None, top_values=p if k else None, top=k, temperature=1.0)
    at = ctypes.byref(h)
    return [f(at) for f in (_lib.lib.nif_head_state_bytes, _lib.lib.nif_head_forward_workspace_bytes, _lib.lib.nif_head_backward_workspace_bytes)]


@pytest.mark.parametrize('dtype, e', [(_lib.NIF_F32, 4), (_lib.NIF_BF16, 2), (_lib.NIF_F16, 2)])
@pytest.mark.parametrize('n', [1, 40, 513, 8192, 100000, 1 << 20, 1 << 24, 1 << 27])
@pytest.mark.parametrize('d, v', [(8, 5), (64, 32000), (77, 9001), (4096, 131072), (2050, 100001)])
def test_memory_is_within_the_stated_bounds(dtype, e, n, d, v):
    rows, wide = -(-n // 256) * 256, -(-d // 64) * 64  # of the packed hidden rows
    for k in (0, 32):
        for ldw in (d, d + 1):
            state, forward, backward = _bytes(n, d, v, dtype, k, ldw)
            assert state <= rows * wide * e + 64 * MIB + rows * (max(k, 1) * 12 + 24) + 4096
            piece = max(256 * MIB, 1024 * max(rows, wide) * e) + 256 * rows * e  # of dz, or of a weight that is packed
            splits = 1024 * MIB  # partial sums of split products: of few tiles only
            assert forward <= rows * (v // 32 + 16) * 8 + piece + splits
            assert backward <= 2 * piece + rows * (d + 4) * 4 + splits + rows * 8


def test_the_statistics_of_many_rows():
    """Of large products 8 bytes for 128 classes of a row (f32: 64)."""
    n, d, v = 1 << 20, 64, 32000
    assert _bytes(n, d, v, _lib.NIF_BF16, 0, d)[1] <= n * (v / 128 + 8) * 8 + 8 * MIB
    assert _bytes(n, d, v, _lib.NIF_F32, 0, d)[1] <= n * (v / 64 + 8) * 8 + 8 * MIB
