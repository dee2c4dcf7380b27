"""64-bit attention and error bounds for the decode-attention tests.

Bounds, for an output o = sum_t p_t v_t / l of type t with unit roundoff u = eps / 2 (a rounding is off by at most half
a step): the kernels round P (or P times a block's scale) to t and the result to t, so |err| <= u (A + |o|) with
A = sum_t p_t |v_t| / l, to first order. Logits come from exact products summed in 32 bits: the sum of D products by
steps of 16 is off by at most (D / 16 + 8) 2^-22 S with S = scale * sum_d |q_d k_d| (8 more steps for the scale, the
max and exp2), which shifts each p_t by that, relative: 2 delta A, delta the largest over the row's keys. fp16 P below
its subnormal step lose at most 2^-25 each against a row maximum of 1: T 2^-25 max|v|; with block scales the same
after the lift by 64. A factor 1.1 covers the second order.

Pages decoded to fp16 (the tcgen05 kernel): each K and V value code * scale is rounded to fp16 once, 2^-11 relative, which
shifts a logit by at most 2^-11 S and o by at most 2^-11 A more; values below fp16's smallest normal number by 2^-25 each,
which D 2^-25 scale max|q| and 2^-25 cover."""
import numpy as np
import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend64(q, k, v, see, scale, decoded=False):
    """q [N][Hq][D], k, v [T][Hkv][D], see bool [N][T] -> out, lse, A, delta (float64, per row and head)."""
    q, k, v = q.double(), k.double(), v.double()
    n, hq, dim = q.shape
    g = hq // k.shape[1] if k.shape[1] else 1
    out = torch.zeros(n, hq, dim, dtype=torch.float64)
    size = torch.zeros(n, hq, dim, dtype=torch.float64)
    lse = torch.full((n, hq), -float("inf"), dtype=torch.float64)
    delta = torch.zeros(n, hq, dtype=torch.float64)
    for i in range(n):
        t = see[i].nonzero()[:, 0]
        if not len(t):
            continue
        for h in range(hq):
            kk, vv = k[t, h // g], v[t, h // g]
            s = kk @ q[i, h] * scale
            delta[i, h] = ((dim / 16 + 8) * 2.0 ** -22 + (2.0 ** -11 if decoded else 0)) * float((kk.abs() @ q[i, h].abs()).max()) * scale
            if decoded:
                delta[i, h] += dim * 2.0 ** -25 * scale * float(q[i, h].abs().max())
            lse[i, h] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[i, h])
            out[i, h], size[i, h] = p @ vv, p @ vv.abs()
            if decoded:  # u (A + |o|) + 2^-11 A + 2^-25 with u the output type's, so at most twice u A where u = 2^-11
                size[i, h] = 2 * size[i, h] + 2.0 ** -13
    return out, lse, size, delta


def check(got, got_lse, exp, dtype, keys, vmax):
    """got [N][Hq][D] of dtype and got_lse [N][Hq] (or None) against attend64's result."""
    out, lse, size, delta = exp
    u = UNIT[dtype]
    g = got.double().cpu()
    tol = 1.1 * (u * (size + out.abs()) + 2 * delta[..., None] * size) + (keys * 2.0 ** -25 * vmax if dtype == torch.float16 else 0) + 1e-30
    err = (g - out).abs()
    assert torch.isfinite(g).all(), "non-finite outputs"
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.3g} of its bound"
    if got_lse is not None:
        L = got_lse.double().cpu()
        assert (torch.isinf(L) == torch.isinf(lse)).all() and (L[torch.isinf(L)] < 0).all()
        f = ~torch.isinf(lse)
        # 32-bit sums of partial sums: 2^-20 relative covers 16 roundings per partial sum and their joining.
        assert ((L[f] - lse[f]).abs() <= delta[f] * 1.1 + 2.0 ** -20 + lse[f].abs() * 2.0 ** -22).all()


def tree_words(see):
    """bool [..][N][N] -> int32 [..][N][words]"""
    n = see.shape[-1]
    words = max(1, -(-n // 32))
    bits = np.zeros(see.shape[:-1] + (words * 32,), np.uint8)
    bits[..., :n] = see
    return torch.from_numpy(np.packbits(bits, axis=-1, bitorder="little").view(np.int32).copy())
