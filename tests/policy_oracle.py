"""The policy operators from their definitions in 64 bits (numpy, step by step), each with a bound on what float arithmetic may be off.

Bounds count roundings, u = 2^-24 each (half a step of float32; 2^-53 for double).  A recurrence's value is a sum of terms x_j a_{j+1} ..
a_t.  However the time axis is cut, a term meets one rounding a step (in a product of gates or in a fused multiply-add) and
one for every run of 16 steps folded, so with M_t = |a_t| M_{t-1} + |x_t| its error is at most 2 u D_t, D_t = |a_t| D_{t-1} + M_t.
An output of a narrower type adds half a step of it: finfo.eps / 2 of the value (and half its smallest step near zero)."""
import numpy as np
import torch

U32, U64 = 2.0 ** -24, 2.0 ** -53


def np64(t):
    return t.detach().cpu().double().numpy()


def rounded(value, off, dtype):
    """bound after one rounding to dtype of something that is `off` off value"""
    f = torch.finfo(dtype)
    return off + (np.abs(value) + off) * (f.eps / 2) + f.smallest_normal * f.eps / 2


def scan(x, gate, state, done, reverse, u=U32):
    """x [T, E, C], gate [T, E, H] or a float -> dict of float64 arrays: y, last, their bounds, and what the gradients need"""
    x = np64(x)
    T, E, C = x.shape
    a = np.full((T, E, C), float(gate)) if not isinstance(gate, torch.Tensor) else np.repeat(np64(gate), C // gate.shape[2], axis=2) if C else np.zeros((T, E, C))
    d = np.zeros((T, E), bool) if done is None else done.cpu().numpy() != 0
    s = np.zeros((E, C)) if state is None else np64(state)
    order = list(range(T))[::-1] if reverse else list(range(T))
    y, k, M, D, kD = np.zeros_like(x), np.zeros_like(x), np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)
    cut = np.zeros((T, E), bool)
    h, m, dd = s, np.abs(s), np.zeros((E, C))
    for n, t in enumerate(order):
        c = d[t] if reverse else (d[t - 1] if n else np.zeros(E, bool))
        cut[t] = c
        h, m, dd = (np.where(c[:, None], 0.0, v) for v in (h, m, dd))
        k[t], kD[t] = h, dd
        forget = a[t] == 0
        with np.errstate(invalid="ignore"):
            h = np.where(forget, x[t], a[t] * h + x[t])
            m = np.where(forget, np.abs(x[t]), np.abs(a[t]) * m + np.abs(x[t]))
            dd = np.where(forget, m, np.abs(a[t]) * dd + m)
        y[t], M[t], D[t] = h, m, dd
    if not reverse and T:
        h, dd = np.where(d[-1][:, None], 0.0, h), np.where(d[-1][:, None], 0.0, dd)
    return dict(y=y, ybound=2 * u * D, last=h, lastbound=2 * u * dd, a=a, k=k, kbound=2 * u * kD, cut=cut, done=d, order=order)


def scan_grad(f, dy, dlast, heads, reverse, u=U32):
    """gradients of scan()'s y and last: dx, dgate, dstate and their bounds"""
    T, E, C = f["y"].shape
    dy = np.zeros((T, E, C)) if dy is None else np64(dy)
    r = np.zeros((E, C)) if dlast is None else np64(dlast)
    if not reverse and T:
        r = np.where(f["done"][-1][:, None], 0.0, r)
    m, dd = np.abs(r), np.zeros((E, C))
    dx, gD = np.zeros_like(dy), np.zeros_like(dy)
    for t in f["order"][::-1]:
        g = dy[t] + r
        m = np.abs(dy[t]) + m
        dd = dd + m  # one rounding of the sum
        dx[t], gD[t] = g, dd
        c = f["cut"][t][:, None]
        r, m, dd = (np.where(c, 0.0, np.abs(f["a"][t]) * v if v is not g else f["a"][t] * v) for v in (g, m, dd))
        dd = dd + m  # and one of the product
    gb = 2 * u * gD
    per = dx * f["k"]
    perb = np.abs(f["k"]) * gb + np.abs(dx) * f["kbound"] + gb * f["kbound"]
    split = (T, E, heads, C // heads if heads else 0)
    # a head's sum: products one rounding, at most 6 butterflies + 1 pair + partial sums of every 64 lanes
    n = 8 + 1 + (C // max(heads, 1)) // 64
    return dict(dx=dx, dxbound=gb, dgate=per.reshape(split).sum(-1), dgatebound=(perb + n * u * (np.abs(per) + perb)).reshape(split).sum(-1), dstate=r, dstatebound=2 * u * dd)


def advantages(reward, value, last_value, done, gamma, lam, first):
    """(advantage, return) in plane order"""
    r, v = np64(reward), np64(value)
    P, E, n = r.shape
    after = np.zeros((E, n)) if last_value is None else np64(last_value)
    d = np.zeros((P, E, n), bool) if done is None else np.broadcast_to((done.cpu().numpy() != 0).reshape(P, E, -1), (P, E, n))
    adv, ret, nxt = np.zeros_like(r), np.zeros_like(r), np.zeros((E, n))
    for s in range(P - 1, -1, -1):
        p = (first + s) % P
        adv[p] = r[p] - v[p] + np.where(d[p], 0.0, gamma * after) + np.where(d[p], 0.0, gamma * lam * nxt)
        ret[p] = adv[p] + v[p]
        nxt, after = adv[p], v[p]
    return adv, ret


def logits(l, tokens=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None, dz=None):
    """l [R, V], tokens [R, L], bias [B, V], allowed bool [R, V] (already spread over the rows): z, its bound, and with dz the gradients"""
    l, (R, V) = np64(l), l.shape
    seen, count = np.zeros((R, V), bool), np.zeros((R, V))
    row = lambda v: np64(v).reshape(R, 1) if isinstance(v, torch.Tensor) else np.full((R, 1), np.float32(v), np.float64)  # noqa: E731
    rep, pres, freq = row(repetition), row(presence), row(frequency)
    if tokens is not None:
        tok = tokens.cpu().numpy().astype(np.int64)
        for r in range(R):
            n = tok.shape[1] if lengths is None else min(max(int(lengths[r]), 0), tok.shape[1])
            k = 0 if prompt_lengths is None else max(int(prompt_lengths[r]), 0)
            for i in range(n):
                if 0 <= tok[r, i] < V:
                    seen[r, tok[r, i]] = True
                    count[r, tok[r, i]] += i >= k
    with np.errstate(invalid="ignore", over="ignore"):
        factor = np.where(seen, np.where(l > 0, 1 / rep, np.broadcast_to(rep, (R, V))), 1.0)
        scaled = np.where(seen, np.where(l > 0, l / rep, l * rep), l)
        taken = np.where(count > 0, pres + freq * count, 0.0)
        b = np.zeros((1, V)) if bias is None else np64(bias)
        b = np.tile(b, (R // b.shape[0], 1)) if R else np.zeros((0, V))
        z = scaled - taken + b
        # at most five float operations, each rounding a value no larger than the sum of the sizes
        off = 5 * U32 * (np.abs(scaled) + np.where(count > 0, np.abs(pres) + np.abs(freq) * count, 0.0) + np.abs(b))
    ok = np.ones((R, V), bool) if allowed is None else allowed
    z, off = np.where(ok, z, -np.inf), np.where(ok, off, 0.0)
    out = dict(z=z, bound=np.where(np.isfinite(z), off, 0.0))
    if dz is not None:
        d = np.where(ok, np64(dz), 0.0)
        out["dlogits"], out["dlogitsbound"] = d * factor, 2 * U32 * np.abs(d * factor)
        if bias is not None:
            B = bias.shape[0]
            out["dbias"] = d.reshape(-1, B, V).sum(0)
            out["dbiasbound"] = (R // B) * U32 * np.abs(d).reshape(-1, B, V).sum(0)  # one rounding a term, in any order
    return out


def close(got, want, bound, what=""):
    """|got - want| <= bound; infinities and NaN where they belong"""
    got = np64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what
    bad = ~(np.abs(got - np.where(fine, want, 0)) <= bound) & fine
    if bad.any():
        i = tuple(int(k) for k in np.argwhere(bad)[0])
        raise AssertionError("%s: %d of %d past their bound; first at %s: %r, %r wanted, bound %.3g" % (what, bad.sum(), bad.size, i, got[i], want[i], bound[i]))
