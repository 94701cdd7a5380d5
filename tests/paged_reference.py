"""Plain float64 forms of the paged key-value cache operators, one sequence and head after another (CPU or GPU tensors,
no code of the library), and the tolerances of the tests."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}   # half a step, relative


def rotate(x, rope_row, interleaved):
    """x [heads, d] float64, rope_row [rotary] float64 (cosines, sines)."""
    r = rope_row.numel()
    x = x.clone()
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        c, s = rope_row[i], rope_row[r // 2 + i]
        xa, xb = x[:, a].clone(), x[:, b].clone()
        x[:, a], x[:, b] = xa * c - xb * s, xb * c + xa * s
    return x


def sequence(pool, table_row, n, page, head, scale=None):
    """float64 [n, d]: the first n tokens of a sequence for one head."""
    rows = [pool[int(table_row[p // page]), p % page, head] for p in range(n)]
    if not rows:
        return torch.zeros(0, pool.shape[3], dtype=torch.float64, device=pool.device)
    x = torch.stack([r.double() for r in rows])
    return x if scale is None else x * scale[head].double()


def attend(q, k, v, scale):
    """(out, lse, mass) of one query: q [d], k and v [n, d] float64.  mass = largest scale * sum_d |q_d k_d|."""
    if k.shape[0] == 0:
        return torch.zeros_like(q), -math.inf, 0.0
    logits = (k @ q) * scale
    out = torch.softmax(logits, 0) @ v
    return out, float(torch.logsumexp(logits, 0)), float((abs(scale) * (k.abs() @ q.abs())).max())


def attention_tolerance(out, n, d, mass, v_max, dtype, single_p):
    """Largest error the kernel may make against float64, per element of `out`.

    The result is rounded once: half a step of `dtype`.  Before that, in fp32:
      * a logit is a sum of d exact products; each partial sum is off by at most 2^-23 of the sum of the magnitudes
        (tensor cores truncate, hence a whole step): delta = (d + 4) 2^-23 mass, 4 for the scaling and the exponent;
      * a weight exp(s) / sum then is off by a factor of at most 1 + 2 delta + 2^-21 (2^-22 for each exponential);
      * a weight enters the product with V as two 16-bit terms (relative error 2^-16) or, where the result is bf16 and
        the pages hold 8 bits, as one fp16 term (2^-11);
      * n products are added, again 2^-23 each (n + 64: the joins of parts), and the weights add up to 1, so every
        relative error of a weight or a sum is an error of at most that times the largest |v|."""
    delta = (d + 4) * 2.0 ** -23 * mass
    rel = 2 * delta + 2.0 ** -21 + (2.0 ** -11 if single_p else 2.0 ** -16) + (n + 64) * 2.0 ** -23
    return HALF[dtype] * out.abs() + rel * v_max + (2.0 ** -25 if dtype == torch.float16 else 0.0)   # fp16: subnormal step


def lse_tolerance(lse, n, d, mass):
    """delta as above for the largest logit's error, the relative error of the sum, and the rounding of the result."""
    return (d + 4) * 2.0 ** -23 * mass + (n + 64) * 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -22 * abs(lse)


def scores(q, low, high):
    """float64 score of one page for one key head: q [g, d], low and high [d]."""
    if not bool((low.isfinite() & high.isfinite()).all()):
        return math.inf
    s = torch.maximum(q * low, q * high).sum(1)
    return float(torch.where(s.isfinite(), s, torch.full_like(s, math.inf)).max())


def select(score, top, sink, recent):
    """Pages chosen from a list of scores."""
    n = len(score)
    if n <= top:
        return list(range(n))
    middle = sorted(range(sink, n - recent), key=lambda i: (-score[i], i))[: top - sink - recent]
    return sorted(list(range(sink)) + middle + list(range(n - recent, n)))
