"""The paged cache's C ABI and Python checks that need no GPU."""
from __future__ import annotations

import ctypes as C
import os

import numpy as np
import pytest


@pytest.fixture(scope="module")
def built(tg):
    if not os.path.exists(tg.LIB_PATH):
        tg.build()
    return tg


def test_null_handles_are_refused(built):
    L = built.lib()
    h, d = C.c_void_p(), built.tg_paged_desc()
    bad = built.TG_ERR_INVALID_ARG
    assert L.tg_paged_create(None, C.byref(d), C.byref(h)) == bad
    assert L.tg_paged_destroy(None) == built.TG_OK
    assert L.tg_paged_layer_ptrs(None, 0, C.byref(h), None, None) == bad
    assert L.tg_paged_append(None, None, 0, 1, 1, None, None, None, 1, None, None, None, None) == bad
    assert L.tg_paged_attention(None, None, 0, 1, None, None, None, 1, None) == bad
    assert L.tg_paged_attention_shared(None, None, 0, 1, None, None, None, 1, 0, None) == bad
    assert L.tg_paged_select(None, None, 0, 1, None, None, None, 1, 0, 0, 1, None) == bad
    assert L.tg_paged_attention_sparse(None, None, 0, 1, None, None, None, 1, 1, None, None) == bad


def test_argument_checks_of_the_binding(built):
    f = np.zeros((3, 128), np.float32)
    assert built._rows(f, 128, "k") == 3
    with pytest.raises(ValueError):
        built._rows(f, 100, "k")
    with pytest.raises(ValueError):
        built._rows(f.astype(np.float64), 128, "k")
    i = np.zeros(4, np.int32)
    assert built._ints(i, 4, "pos") == i.ctypes.data and built._ints(None, 4, "pos") is None
    for bad in (i.astype(np.int64), i.astype(np.uint32), i[:3]):
        with pytest.raises(ValueError):
            built._ints(bad, 4, "pos")
    with pytest.raises(ValueError):
        built._table_shape(i)
    assert built._table_shape(np.zeros((2, 5), np.int32)) == (2, 5)


class DeviceTensor:
    """What the binding looks at of a device tensor."""

    def __init__(self, n, dtype):
        import torch
        self._n, self.dtype, self.device = n, dtype, torch.device("cuda", 0)

    def numel(self):
        return self._n

    def element_size(self):
        return self.dtype.itemsize

    def data_ptr(self):
        return 0


@pytest.mark.parametrize("name,good", [("DTYPE_BF16", "bfloat16"), ("DTYPE_F32", "float32")])
def test_pools_of_another_type_are_refused(built, name, good):
    """Types of the same size among them: their bits would be read as the
    cache's type.  The right type goes on to the library, which has no context
    here."""
    import torch

    class Backend:
        device, handle = 0, None

    right = getattr(torch, good)
    for wrong in (torch.float16, torch.int16, torch.int32, torch.float64, torch.bfloat16,
                  torch.float32, torch.uint8):
        for at in ("k", "v", "bounds"):
            types = {"k": right, "v": right, "bounds": right, at: wrong}
            pools = {x: DeviceTensor(4 * 2 * (16 if x != "bounds" else 2) * 64, t)
                     for x, t in types.items()}
            with pytest.raises(built.TGError if wrong == right else ValueError) as e:
                built.PagedKVCache(Backend(), 1, 4, 16, dtype=getattr(built, name), **pools)
            if wrong != right:
                assert str(e.value).startswith(f"{at} is ")
