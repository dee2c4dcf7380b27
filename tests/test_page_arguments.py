"""CPU: numbers that do not fit the library's 32-bit arguments are refused before any call, not taken modulo 2^32."""
import ctypes as C
import types

import pytest
import torch


class Calls:
    """Stands for the library: remembers what was called."""

    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        return lambda *a: (self.seen.append((name, a)), 0)[1]


@pytest.fixture
def pool(monkeypatch):
    import kvmem_b200 as K
    from kvmem_b200 import recall
    monkeypatch.setattr(recall, "_stream_on", lambda device, stream: 0)
    p = K.ResidencyPool.__new__(K.ResidencyPool)
    p.ctx = types.SimpleNamespace(lib=Calls(), h=C.c_void_p(1), device=-1)  # (-1: CPU tensors' get_device())
    p.h, p.rows, p.pages, p.slots = None, 4, 10, 4
    return p


@pytest.fixture
def layout():
    import kvmem_b200 as K
    return K.cache_layout(torch.zeros(4, 4, 16, dtype=torch.uint8))


BAD = [-1, 1 << 32, (1 << 32) + 2, -(1 << 32)]


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("call", [
    lambda p, L, x: p.fork(L, [0], [1], page_end=x),
    lambda p, L, x: p.fork(L, [0], [1], ctas=x),
    lambda p, L, x: p.fork(L, [x], [1]),
    lambda p, L, x: p.fork(L, [0], [x]),
    lambda p, L, x: p.copy_pages(L, [(0, 0, 1, 1)], ctas=x),
    lambda p, L, x: p.copy_pages(L, [(0, 0, 1, 1), (x, 0, 2, 1)]),
    lambda p, L, x: p.copy_pages(L, [(0, x, 1, 1)]),
    lambda p, L, x: p.copy_pages(L, [(0, 0, x, 1)]),
    lambda p, L, x: p.copy_pages(L, [(0, 0, 1, x)]),
    lambda p, L, x: p.free([x], torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)),
    lambda p, L, x: p.compact(L, [x]),
    lambda p, L, x: p.compact(L, [0], ctas=x),
])
def test_out_of_range(pool, layout, call, bad):
    import kvmem_b200 as K
    with pytest.raises(K.KvmError) as e:
        call(pool, layout, bad)
    assert e.value.code == K._abi.ERR_INVALID_ARGUMENT
    assert not pool.ctx.lib.seen


def test_numbers_in_range_go_through(pool, layout):
    pool.fork(layout, [0], [1], page_end=0xFFFFFFFF, ctas=3)
    pool.copy_pages(layout, [(0, 1, 2, 3)], ctas=7)
    pool.copy_pages(layout, torch.tensor([[0, 1, 2, 3]], dtype=torch.int32))
    pool.free([3], torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    pool.compact(layout, ctas=9)
    names = [n for n, _ in pool.ctx.lib.seen]
    assert names == ["kvm_pool_fork", "kvm_pool_copy", "kvm_pool_copy", "kvm_pool_free", "kvm_pool_compact"]
    fork = pool.ctx.lib.seen[0][1]
    assert list(fork[3]) == [0] and list(fork[4]) == [1] and fork[5:8] == (1, 0xFFFFFFFF, 3)
    assert list(pool.ctx.lib.seen[-1][1][3]) == [0, 1, 2, 3]
