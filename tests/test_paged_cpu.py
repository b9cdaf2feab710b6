"""CPU tests of the paged cache's host side: argument checks that need no device,
and the C entry points' refusals that come before any CUDA call."""
import ctypes as C

import numpy as np
import pytest


def test_public_names():
    import kvforge_b200 as K
    for name in ("PagedKVCache", "PagedBatch", "Eviction"):
        assert name in K.__all__ and hasattr(K, name)


def test_constructor_refuses_before_it_allocates():
    import torch
    import kvforge_b200 as K
    with pytest.raises(TypeError):
        K.PagedKVCache(4, 1, 64, dtype=torch.int8)
    for bad in (dict(page_size=48), dict(page_size=256), dict(head_dim=0), dict(head_dim=300), dict(num_heads=0),
                dict(num_pages=0), dict(num_layers=0)):
        with pytest.raises(K.KvForgeError):
            K.PagedKVCache(**{**dict(num_pages=4, num_heads=1, head_dim=64), **bad})


def test_host_arrays():
    from kvforge_b200.paged import _ints
    a, n = _ints([[1, 2, 3], [], [4]])
    assert n == 3 and list(a) == [1, 2, 3, 0, 0, 0, 4, 0, 0]
    a, n = _ints([])
    assert n == 1 and list(a) == [0]
    a, n = _ints([[]])
    assert n == 1 and list(a) == [0]


def test_null_context_is_refused():
    from kvforge_b200 import _lib as L
    lib = L.lib()
    pool = L.PagedPool(L.IN_F16, 16, 1, 4, 1, 64, 256, 256, 256)
    plan = C.c_void_p()
    one = np.ones(1, np.int32)
    assert lib.kvf_paged_plan_create(None, C.byref(pool), 1, one.ctypes.data, one.ctypes.data, one.ctypes.data, 1, 1, 0,
                                     0, C.byref(plan), None) == L.ERR_INVALID_CONFIG
    assert lib.kvf_paged_append(None, None, C.byref(pool), 0, None, 1, 1, None, 1, 1, None) == L.ERR_INVALID_CONFIG
    assert lib.kvf_paged_attention(None, None, C.byref(pool), 0, None, 1, 1, 1.0, -1.0, None, None,
                                   None) == L.ERR_INVALID_CONFIG
    assert lib.kvf_paged_gather(None, C.byref(pool), 0, None, 1, None, None, None) == L.ERR_INVALID_CONFIG
    assert lib.kvf_paged_evict(None, C.byref(pool), 1, None, None, 1, 1, 0, 0, None, 1, None,
                               None) == L.ERR_INVALID_CONFIG
    assert lib.kvf_paged_plan_free(None) == L.OK
