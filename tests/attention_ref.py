"""Attention with a window, its gradients and rotary positions from their
definitions in 64 bits, each with how far a kernel may be off: tolerances
count the roundings that a kernel makes on the way.

u: half a step of the tensors' type relative to a value; w: that of the
weights P and dS where a kernel rounds them for the tensor cores (bf16), and
of fp32 otherwise. A score's fp32 error is (dh + 4) 2^-24 of sum |q||k|, which
is the relative error of its exponential; sums of n terms add n 2^-24, and
the hardware's exponential and logarithm 2^-20. A weight below fp32's smallest
normal number, 2^-126, may count as 0 (of scores some 90 below the row's
largest), and so may a result: TINY of what it multiplies, and of 1."""
import math

import torch


TINY = 2.0 ** -125


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def mask(n, m, window, sinks, device):
    """Which of m keys each of the last n of them sees."""
    i = torch.arange(m - n, m, device=device)[:, None]
    j = torch.arange(m, device=device)[None]
    return (j <= i) & ((i - j < window) | (j < sinks) if window else torch.ones_like(j <= i))


def attend(q, k, v, seen, scale, dtype, dout=None, summed=False):
    """One head: q [n, dh], k, v [m, dh] in 64 bits. out, lse and with dout dq, dk, dv, each beside its tolerance.
    summed: D = sum_j p_j dP_j, not from the rounded out: it was that first, then the sum of P (dP - D) was added."""
    u, w = half_step(dtype), half_step(dtype)
    m, dh = k.shape
    e = 2.0 ** -24
    z = torch.where(seen, q @ k.t() * scale, -math.inf)
    size = torch.where(seen, q.abs() @ k.abs().t() * scale, 0).amax(1, keepdim=True)
    p = torch.softmax(z, 1).nan_to_num(0)
    off = 2 * ((dh + 4) * size + m) * e + 2.0 ** -20  # of a weight, relative
    out = p @ v
    out_tol = u * out.abs() + ((w + 2 * off) * p + TINY) @ v.abs() + TINY
    lse = torch.logsumexp(z, 1)
    lse_tol = off[:, 0] + 2.0 ** -22 * lse.abs()
    got = dict(out=(out, out_tol), lse=(lse, lse_tol))
    if dout is None:
        return got
    dp, D = dout @ v.t(), (dout * out).sum(1, keepdim=True)
    ds = p * (dp - D)
    many = dh * e
    size_p, size_D = dout.abs() @ v.abs().t(), (dout.abs() * out.abs()).sum(1, keepdim=True)
    off_D = (dout.abs() * out_tol).sum(1, keepdim=True) + many * size_D
    if summed:  # what was wrong before is left as far as the weights' sum is off 1
        mean = (p * size_p).sum(1, keepdim=True)
        off_D = off * (off_D + mean + size_D) + (many + m * e) * (2 * mean + size_D)
    off_s = (w + m * e) * ds.abs() + p * (off * (size_p + size_D) + many * size_p + off_D) + TINY * (size_p + size_D)
    got["dv"] = (p.t() @ dout, u * (p.t() @ dout).abs() + ((w + 2 * off) * p + TINY).t() @ dout.abs() + TINY)
    got["dq"] = (scale * ds @ k, u * (scale * ds @ k).abs() + scale * off_s @ k.abs() + TINY)
    got["dk"] = (scale * ds.t() @ q, u * (scale * ds.t() @ q).abs() + scale * off_s.t() @ q.abs() + TINY)
    return got


def packed(q, k, v, offsets, window, sinks, scale, dtype, dout=None, summed=False):
    """All sequences and heads: {name: (value, tolerance)}, rows of no sequence 0."""
    T, Hq, dh = q.shape
    Hkv = k.shape[1]
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)  # noqa: E731
    shapes = dict(out=(T, Hq, dh), lse=(T, Hq))
    if dout is not None:
        shapes |= dict(dq=(T, Hq, dh), dk=(T, Hkv, dh), dv=(T, Hkv, dh))
    full = {n: (z(*s), z(*s)) for n, s in shapes.items()}
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        if hi == lo:
            continue
        seen = mask(hi - lo, hi - lo, window, sinks, q.device)
        for h in range(Hq):
            hk = h // (Hq // Hkv)
            got = attend(q[lo:hi, h].double(), k[lo:hi, hk].double(), v[lo:hi, hk].double(), seen, scale, dtype,
                         None if dout is None else dout[lo:hi, h].double(), summed)
            for n, pair in got.items():
                at = hk if n in ("dk", "dv") else h
                for f, x in zip(full[n], pair):
                    f[lo:hi, at] += x
    full["lse"] = tuple(x.t() for x in full["lse"])
    return full


def turn(x, pos, freq, axis, interleaved, scale, back=False):
    """Rotary positions: x [T, H, dh], pos [axes, T], axis [pairs]."""
    a = (pos[axis].double() * freq.double()[:, None]).t()[:, None]
    if back:
        a = -a
    n = freq.numel()
    y = x.double().clone()
    first = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    second = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    x0, x1 = x[..., first].double(), x[..., second].double()
    y[..., first] = scale * (x0 * a.cos() - x1 * a.sin())
    y[..., second] = scale * (x1 * a.cos() + x0 * a.sin())
    return y


def turn_tolerance(x, n, interleaved, scale, dtype, y):
    """Half a step of y's type, and of each product of a pair four roundings in fp32 and a sine's 2^-21."""
    pairs = x[..., :2 * n].double().abs()
    size = torch.zeros_like(x, dtype=torch.float64)
    if interleaved:
        both = pairs[..., 0::2] + pairs[..., 1::2]
        size[..., :2 * n] = both.repeat_interleave(2, -1)
    else:
        both = pairs[..., :n] + pairs[..., n:]
        size[..., :2 * n] = torch.cat([both, both], -1)
    return half_step(dtype) * y.abs() + abs(scale) * size * 2.0 ** -20


def close(got, want, tol, what=""):
    """Every value within its tolerance; infinities and NaN where they are wanted."""
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    fine = same | ((got - want).abs() <= tol)
    bad = ~fine
    if bad.any():
        i = tuple(x[0].item() for x in bad.nonzero(as_tuple=True))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i].item()} for "
                             f"{want[i].item()} within {tol[i].item()}")
