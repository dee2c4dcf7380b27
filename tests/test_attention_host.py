"""CPU: host side of the decode-attention and page entry points (no context, no GPU)."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests.attend_util import tree_words


def test_tree_mask_follows_the_parents():
    import kvmem_b200 as K
    rng = np.random.default_rng(0)
    for n in (1, 2, 31, 32, 33, 100):
        parents = [-1 if i == 0 else int(rng.integers(-1, i)) for i in range(n)]
        see = np.zeros((n, n), bool)
        for i in range(n):
            j = i
            while j >= 0:
                see[i, j] = True
                j = parents[j]
        assert torch.equal(K.tree_mask(parents), tree_words(see))
    assert K.tree_mask([]).shape == (0, 1)


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 2, 0], [-2]])
def test_tree_mask_refuses(parents):
    import kvmem_b200 as K
    with pytest.raises(K.KvmError) as e:
        K.tree_mask(parents)
    assert e.value.code == K._abi.ERR_INVALID_ARGUMENT
    words = (C.c_uint32 * 4)()
    assert K._abi.load().kvm_tree_mask((C.c_int32 * 33)(*([-1] * 33)), 33, 1, words) == K._abi.ERR_INVALID_ARGUMENT


def test_null_handles_are_refused_before_any_cuda_call():
    import kvmem_b200 as K
    A, lib = K._abi, K._abi.load()
    r, kc, lay = A.Rows(), A.KCache(), A.StageLayout()
    assert lib.kvm_window_attention(None, C.byref(A.WindowDesc()), C.byref(r), C.byref(kc), C.byref(kc), C.byref(r), None, None) == A.ERR_INVALID_ARGUMENT
    assert lib.kvm_tree_attention(None, None, C.byref(A.TreeDesc()), lay, C.byref(r), C.byref(kc), C.byref(kc), C.byref(r), None, None) == A.ERR_INVALID_ARGUMENT
    assert lib.kvm_pool_fork(None, None, lay, None, None, 1, 1, 0, None) == A.ERR_INVALID_ARGUMENT
    assert lib.kvm_pool_copy(None, None, lay, None, 1, 0, None) == A.ERR_INVALID_ARGUMENT
    assert lib.kvm_pool_free(None, None, None, 1, None, None, 1, None) == A.ERR_INVALID_ARGUMENT
    assert lib.kvm_pool_compact(None, None, lay, None, 1, None, 0, None) == A.ERR_INVALID_ARGUMENT
    assert lib.kvm_pool_tables(None, None, None) == A.ERR_INVALID_ARGUMENT


def test_cache_layout_of_strided_planes():
    import kvmem_b200 as K
    k = torch.zeros(3, 5, 4, 8, dtype=torch.float16)
    L = K.cache_layout(k[:, 1:], k[1:])
    assert L.planes == 2 and L.dev_base[0] == k.data_ptr() + 64 and L.dev_row_stride[0] == 320
    assert L.dev_slot_stride[1] == 64 and L.bytes[1] == 64
    with pytest.raises(K.KvmError):
        K.cache_layout(k.transpose(2, 3))
