"""GPU: a bf16 tail beside quantised pages keeps bf16's whole range below fp16's largest value.

Bounds for a row that sees the tail alone, with u = 2^-8 for the rounding of the output and A = sum_t p_t |v_t|: K and V are
exact in every form. The tcgen05 kernel takes P as the sum of two bf16 numbers, what is left is 2^-8 2^-8 of it; the mma.sync kernel
takes one, 2^-8. Queries: bf16 numbers after a division of their row by a power of two, exact down to 2^-30 of the row's
largest, and off by at most 2^-38 of it below. Logits as in tests/attend_util.py, delta undoubled: (D / 16 + 8) 2^-22 S and
D 2^-38 scale max|q| max|k| (twice, for the query's and the key's rows). The second product is summed in 32 bits over T keys by
steps of 16: (T / 16 + 8) 2^-22 A."""
import math

import numpy as np
import pytest
import torch

from tests import util as U
from tests.attend_util import attend64
from tests.test_gpu_tree import Problem

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def near(out, lse, q, k, v, see, scale, p_err):
    """out [N][Hq][D], lse [N][Hq] against 64 bits, bounds as above. q [N][Hq][D], k, v [T][Hkv][D]."""
    o, l64, size, delta = attend64(q, k, v, see, scale)
    dim = q.shape[-1]
    delta = delta + 2 * dim * 2.0 ** -38 * scale * q.double().abs().amax() * k.double().abs().amax()
    p_err = p_err + (k.shape[0] / 16 + 8) * 2.0 ** -22
    tol = 1.1 * (2.0 ** -8 * o.abs() + p_err * size + 2 * delta[..., None] * size) + 1e-44
    g = out.double().cpu()
    assert torch.isfinite(g).all()
    worst = float(((g - o).abs() / tol).max())
    assert worst <= 1.0, f"error {worst:.3g} of its bound"
    if lse is not None:
        assert ((lse.double().cpu() - l64).abs() <= 1.1 * delta + 2.0 ** -20 + l64.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("splits", ["1", "3"])
@pytest.mark.parametrize("case", [
    # nodes, hq, hkv, dim, page, recent
    (1, 24, 4, 256, 256, 300),
    (16, 24, 4, 256, 128, 131),
    (9, 16, 2, 128, 32, 700),   # more key tiles than the kernel keeps scales of
    (33, 12, 3, 64, 16, 1200),
])
@pytest.mark.parametrize("k_exp,v_exp", [(0, -30), (-40, 0), (-60, -70), (10, -20)])
def test_small_values_of_the_tail(ctx, monkeypatch, kernel, splits, case, k_exp, v_exp):
    """Keys and values far below fp16's range; queries as much above it where the keys are below."""
    monkeypatch.setenv("KVM_ATTEND", kernel)
    monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    nodes, hq, hkv, dim, page, recent = case
    p = Problem(ctx, 51, 1, nodes, hq, hkv, dim, page, 4, 3, [3 * page], [recent], torch.bfloat16,
                kinds=(U.Q8_0, U.Q4_0), garbage=True)
    p.q = torch.ldexp(p.q.float(), torch.tensor(-k_exp)).to(torch.bfloat16)
    used = recent + nodes
    for i, e in enumerate((k_exp, v_exp)):
        p.tail[i] = torch.ldexp(p.tail[i].float(), torch.tensor(e)).to(torch.bfloat16)
        p.tail_d[i][:, :used] = p.tail[i][:, :used].to(DEV)
    out, lse = p.call(lists=[[]])
    ctx.check_status()
    see = torch.cat([torch.ones(nodes, recent, dtype=torch.bool), torch.from_numpy(p.see[0])], 1)
    near(out[0], lse[0], p.q[0], p.tail[0][0, :used], p.tail[1][0, :used], see, 1 / math.sqrt(dim),
         2.0 ** -16 if kernel == "tc" else 2.0 ** -8)


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("dim,page", [(256, 64), (128, 64), (64, 64)])
def test_small_values_of_the_tail_behind_pages(ctx, monkeypatch, kernel, dim, page):
    """The tail's tokens outweigh the pages' by e^60, so its small values are all that is left."""
    monkeypatch.setenv("KVM_ATTEND", kernel)
    monkeypatch.setenv("KVM_ATTEND_SPLITS", "1")
    nodes, recent = 5, 200
    p = Problem(ctx, 52, 1, nodes, 8, 2, dim, page, 6, 4, [6 * page - 9], [recent], torch.bfloat16,
                kinds=(U.Q8_0, U.Q8_0))
    used = recent + nodes
    scale = 1 / math.sqrt(dim)
    p.q = torch.zeros_like(p.q)
    p.q[..., 0] = 1.0
    # first key coordinates: pages as encoded (|scale * k| below a few units), tail 100 / scale and up
    p.tail[0] = (torch.randn(p.tail[0].shape, generator=torch.Generator().manual_seed(5)) * 0.5).to(torch.bfloat16)
    p.tail[0][..., 0] += 100 / scale
    p.tail[1] = torch.ldexp(p.tail[1].float(), torch.tensor(-40)).to(torch.bfloat16)
    for i in range(2):
        p.tail_d[i][:] = p.tail[i].to(DEV)
    kmax = float(p.vals[0].abs().max()) * scale
    assert kmax < 20
    out, lse = p.call()
    ctx.check_status()
    see = torch.cat([torch.ones(nodes, recent, dtype=torch.bool), torch.from_numpy(p.see[0])], 1)
    near(out[0], lse[0], p.q[0], p.tail[0][0, :used], p.tail[1][0, :used], see, scale, 2.0 ** -16 if kernel == "tc" else 2.0 ** -8)


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinite_values_of_a_node_stay_with_those_that_see_it(ctx, monkeypatch, kernel, dim):
    """An infinite V value and a tiny one beside it: infinite where it is seen, exact elsewhere."""
    monkeypatch.setenv("KVM_ATTEND", kernel)
    nodes, recent, j = 12, 70, 5
    p = Problem(ctx, 53, 1, nodes, 6, 2, dim, 32, 5, 3, [96], [recent], torch.bfloat16, kinds=(U.Q4_0, U.Q4_0))
    p.tail[1] = torch.ldexp(p.tail[1].float(), torch.tensor(-35)).to(torch.bfloat16)
    p.tail_d[1][:] = p.tail[1].to(DEV)
    p.tail_d[1][0, recent + j, :, 3::8] = float("inf")
    out, lse = p.call(lists=[[]])
    ctx.check_status()
    sees = p.see[0][:, j]
    assert sees.any() and not sees.all()
    vis = torch.cat([torch.ones(nodes, recent, dtype=torch.bool), torch.from_numpy(p.see[0])], 1)
    got = out[0].cpu()
    for i in np.flatnonzero(sees):
        assert (got[i, :, 3::8] == float("inf")).all()
    # the other dims of rows that see it, and all dims of rows that do not
    used = recent + nodes
    k, v = p.tail[0][0, :used], p.tail[1][0, :used].clone()
    clean = got.clone()
    v[recent + j, :, 3::8] = 0
    ref = attend64(p.q[0], k, v, vis, 1 / math.sqrt(dim))[0]
    clean[torch.from_numpy(np.flatnonzero(sees))[:, None], :, torch.arange(3, dim, 8)[None]] = \
        ref[torch.from_numpy(np.flatnonzero(sees))[:, None], :, torch.arange(3, dim, 8)[None]].to(torch.bfloat16)
    near(clean, lse[0], p.q[0], k, v, vis, 1 / math.sqrt(dim), 2.0 ** -16 if kernel == "tc" else 2.0 ** -8)
