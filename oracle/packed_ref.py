"""TEST INFRASTRUCTURE -- 64-bit oracles of attention over packed sequences, the
rotation by several axes and 8-bit integer rows, from their definitions, on the
CPU; never used by the product."""
from __future__ import annotations

import math

import torch


def _sequences(offsets):
    ends = [int(x) for x in offsets]
    return [slice(a, b) for a, b in zip(ends, ends[1:]) if b > a]


def packed_attention_ref(q, k, v, offsets, causal=True):
    """(O, LSE, weight, scores): float64; ``weight`` is sum_j P_j |v_j| of every output, ``scores`` the
    largest sum_d |q_d k_jd| / sqrt(D) of every row.  Rows of no sequence: 0 and -inf."""
    q, k, v = q.double(), k.double(), v.double()
    h, t, d = q.shape
    g = h // k.shape[0]
    o, weight = torch.zeros_like(q), torch.zeros_like(q)
    lse, scores = torch.full((h, t), -math.inf, dtype=torch.float64), torch.zeros(h, t, dtype=torch.float64)
    for at in _sequences(offsets):
        n = at.stop - at.start
        for i in range(h):
            a, b, c = q[i, at], k[i // g, at], v[i // g, at]
            x = a @ b.T / math.sqrt(d)
            if causal:
                x = x.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf)
            lse[i, at] = torch.logsumexp(x, -1)
            p = torch.exp(x - lse[i, at, None])
            o[i, at], weight[i, at] = p @ c, p @ c.abs()
            scores[i, at] = (a.abs() @ b.abs().T).amax(-1) / math.sqrt(d)
    return o, lse, weight, scores


def packed_attention_bwd_ref(q, k, v, o, lse, do, offsets, causal=True):
    """((dq, dk, dv), bounds, noise): float64, from the forward's outputs as they
    are given.  ``bounds`` are the gradients' sums over magnitudes, ``noise`` the
    same sums with dS_pj replaced by P_pj (sum |dO v_j| + sum |dO O|), what the error of
    dO . v_j - D_p is relative to."""
    q, k, v, o, lse, do = (x.double() for x in (q, k, v, o, lse, do))
    h, t, d = q.shape
    g, r = h // k.shape[0], 1 / math.sqrt(d)
    outs = [[torch.zeros_like(x) for x in (q, k, v)] for _ in range(3)]
    for at in _sequences(offsets):
        n = at.stop - at.start
        for i in range(h):
            j = i // g
            a, b, c, e = q[i, at], k[j, at], v[j, at], do[i, at]
            p = torch.exp(a @ b.T * r - lse[i, at, None])
            if causal:
                p = p.tril()
            ds = p * (e @ c.T - (e * o[i, at]).sum(-1, keepdim=True))
            size = p * (e.abs() @ c.abs().T + (e * o[i, at]).abs().sum(-1, keepdim=True))
            for which, (x, y, w) in enumerate(((ds, p, 0), (ds.abs(), p, 1), (size, p, 1))):
                one = (lambda z: z.abs()) if w else (lambda z: z)
                outs[which][0][i, at] = x @ one(b) * r
                outs[which][1][j, at] += x.T @ one(a) * r
                outs[which][2][j, at] += y.T @ one(e)
    return outs


def axes_angles_ref(positions, freq, sections):
    """[B, S, R] angles: positions [axes, B, S], one frequency a pair."""
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    return torch.stack([positions[a].double() * f for a, f in zip(axis, freq.double())], -1)


def rope_axes_ref(x, angle, interleaved=False, back=False):
    """(out, bound): [B, H, S, D] with angle [B, S, R]; ``bound`` is |a| + |b| of the pair behind each output."""
    x = x.double()
    r = angle.shape[-1]
    c, s = angle.cos()[:, None], angle.sin()[:, None] * (-1 if back else 1)
    a, b = (x[..., 0:2 * r:2], x[..., 1:2 * r:2]) if interleaved else (x[..., :r], x[..., r:2 * r])
    out, bound = x.clone(), x.abs()
    parts = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r), slice(r, 2 * r))
    out[..., parts[0]], out[..., parts[1]] = a * c - b * s, b * c + a * s
    bound[..., parts[0]] = bound[..., parts[1]] = a.abs() + b.abs()
    return out, bound


RECIPROCAL = float(torch.tensor(1.0) / torch.tensor(127.0))   # rounded to fp32


def quantize_ref(x):
    """(codes, scale): one value at a time, ties to even."""
    codes, scales = torch.zeros(x.shape, dtype=torch.int8), torch.zeros(x.shape[0])
    for m, row in enumerate(x.double()):
        if not bool(row.isfinite().all()):
            scales[m] = math.nan
            continue
        scales[m] = max(float((row.abs().max() * RECIPROCAL).float()), 2.0 ** -126)
        s = float(scales[m])
        for k, value in enumerate(row.tolist()):
            # s and the value are dyadic: the quotient's distance from whole numbers is exact in integers
            num, den = (abs(value)).as_integer_ratio()
            sn, sd = s.as_integer_ratio()
            num, den = num * sd, den * sn
            whole, rest = divmod(num, den)
            whole += 2 * rest > den or (2 * rest == den and whole % 2 == 1)
            codes[m, k] = -whole if value < 0 else whole
    return codes, scales


def gemm_int8_ref(a, b, a_scale, b_scale):
    """float64 [M, N]; the sums are whole numbers below 2^53."""
    return (a.double() @ b.double().T) * a_scale.double()[:, None] * b_scale.double()
