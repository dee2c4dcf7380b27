"""CPU: a bound workspace lives as long as the context may write to it."""
import gc
import weakref

import pytest
import torch


class Calls:
    def __init__(self, bind=0):
        self.bind = bind

    def kvm_ctx_create(self, device, handle):
        return 0

    def kvm_ctx_bind_workspace(self, *a):
        return self.bind

    def kvm_ctx_destroy(self, h):
        return 0


@pytest.fixture
def make(monkeypatch):
    from kvmem_b200 import recall

    def new(lib):
        monkeypatch.setattr(recall.A, "load", lambda: lib)
        c = recall.RecallContext(0)
        c.h = object()
        return c

    return new


def alive(ref):
    gc.collect()
    return ref() is not None


def test_a_bound_workspace_is_held(make):
    c = make(Calls())
    t = torch.empty(1024, dtype=torch.uint8)
    first = weakref.ref(t)
    c.bind_workspace(t)
    del t
    assert alive(first)
    t = torch.empty(512, dtype=torch.uint8)
    second = weakref.ref(t)
    c.bind_workspace(t)
    del t
    assert not alive(first) and alive(second)
    c.close()
    assert not alive(second)


def test_a_refused_workspace_is_not(make):
    import kvmem_b200 as K
    c = make(Calls(bind=K._abi.ERR_INVALID_ARGUMENT))
    t = torch.empty(1024, dtype=torch.uint8)
    ref = weakref.ref(t)
    with pytest.raises(K.KvmError):
        c.bind_workspace(t)
    del t
    assert not alive(ref)
