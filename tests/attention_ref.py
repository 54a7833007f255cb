"""Attention in 64 bits from its definition, and how far a kernel that keeps 32-bit sums may be from it."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # half a unit in the last place, relative


def rows64(q, k, v, scale, seen):
    """q [rows, dim], k, v [keys, dim] of one head; row i sees the keys below seen[i] that are not None in k.
    Returns out, lse and two bounds' ingredients: sum of weights times |v|, largest scale * sum |q||k|."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    out, lse = torch.zeros(len(q), v.shape[1], dtype=torch.float64), torch.full((len(q),), -math.inf, dtype=torch.float64)
    mass, size = torch.zeros_like(out), torch.zeros(len(q), dtype=torch.float64)
    for i, n in enumerate(seen):
        if n <= 0:
            continue
        s = (k[:n] @ q[i]) * scale
        lse[i] = torch.logsumexp(s, 0)
        w = torch.softmax(s, 0)
        out[i], mass[i] = w @ v[:n], w @ v[:n].abs()
        size[i] = (k[:n].abs() @ q[i].abs()).max() * scale
    return out, lse, mass, size


def allowed_error(kind, dim, keys, out, lse, mass, size, largest_v):
    """Of out and of lse.

    A score is a sum of `dim` products in 32 bits: at most (dim + 8) units of `size` off, the scale's and
    log2(e)'s products among them; the exponential's argument is rounded again (4 units of size + 1), the sums
    over the keys add at most keys + 32 units.  Weights off by a factor of 1 + d move the quotient by 2 d
    of `mass`.  In 16 bits the weights are rounded once more, and so is the result; weights below fp16's
    normal range (kept 2^10 above one, for the largest) lose up to 2^-35 of the largest each."""
    unit32 = 2.0 ** -24
    d = unit32 * ((dim + 8) * size + 4 * (size + 1) + keys + 32)
    rel = UNIT[kind]
    err = rel * out.abs() + 2 * d[:, None] * mass
    if kind != "f32":
        err = err + rel * mass * 1.01
    if kind == "f16":
        err = err + keys * 2.0 ** -34 * largest_v + 2.0 ** -25
    return err + 1e-30, d + 2.0 ** -23 * lse.abs().nan_to_num(posinf=0.0, neginf=0.0) + 1e-30


def check(kind, dim, keys, got_out, got_lse, want, largest_v):
    """One head's rows against rows64's answer."""
    out, lse, mass, size = want
    err, err_lse = allowed_error(kind, dim, keys, out, lse, mass, size, largest_v)
    got_out, got_lse = got_out.double().cpu(), got_lse.double().cpu()
    off = (got_out - out).abs()
    assert (off <= err).all(), "out: %g over its bound" % (off - err).max()
    empty = torch.isinf(lse)
    assert (got_out[empty] == 0).all() and torch.isneginf(got_lse[empty]).all()
    off = (got_lse - lse).abs()[~empty]
    assert (off <= err_lse[~empty]).all(), "lse"
