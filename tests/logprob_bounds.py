"""How far the log-probability kernels may be from the definition in 64 bits,
from the additions that a term really goes through.

u = 2^-24.  A thread adds e^(x - r) about a reference r that is at most 6 below
the largest value so far; r moves (a factor e^(r - r') on the sums) when it is
left behind by more than 6, and once more at each join.  With d = x - M:

 - a term: x - r rounds (u), its product with log2 e is 2u more, the exponential
   4u (2 ulp): (3 |x - r| + 4) u.  A move by D is (3 |D| + 4) u, and u for the
   product.  Along a term's way |x - r| and the moves add up to |d| + 12 at the
   most (12 where x was 6 above r), a thread's own moves are one for each 6 of
   that, and there are at most 3 joins: (3 (|d| + 12) + 4 + 5 (|d| + 12) / 6 + 15) u,
   at most (4 |d| + 65) u.
 - the sum: u for each of the L additions on the way, all of positive numbers.

So log s is off by z = u (4 A1 + 65 + L) with A1 = sum p |d|, and by logf's one
ulp, 2 u |log s| with log s <= log Z + 6; x - r and the result round besides.
t = sum e^(x - r) (x - r) takes the same way with at most |d| + 12 in place of 1,
and 8 u more for that factor: t / s is off by
u sum p (4 |d| + 73 + L) (|d| + 12), and by z + 2u of itself, at most A1 + 6."""
import math

import torch

from score_util import logprobs64

U = 2.0 ** -24


def walk_chain(V, bytes_each):
    """Additions of token_logprobs: a thread's 64 bytes a trip in two halves, the
    trips of a block that has the row to itself, joins of 32 lanes, warps, blocks."""
    threads = 128 if V * bytes_each <= 128 * 1024 else 256
    values = 64 // bytes_each
    trips = -(-(V + 16) // (values * threads))
    return values // 2 + 1 + trips + 15


def head_chain(T, V, sms=148):
    """Additions of the head scoring that stores no logits: 32 columns at a time in
    two halves, the tiles of a part, two joins."""
    tt, vt, slots = -(-T // 256), -(-V // 256), sms // 2
    best = None
    for g in range(min(tt, slots), 0, -1):
        C = min(vt, slots // g, 160)
        cost = -(-tt // g) * (-(-vt // C) + 0.5)
        if best is None or cost < best[0]:
            best = cost, C
    return 17 + 4 * -(-vt // best[1]) + 10


def bounded64(logits, tokens, k, chain):
    """logprobs64's values with these bounds; check_logprobs adds the rounding of
    the result, 4 u (|value| + 1)."""
    ref = logprobs64(logits, tokens, k)
    x = logits.detach().cpu().double()
    for t in range(x.shape[0]):
        M = x[t].max()
        if ref["tol_z"][t] == 0.0:  # an empty row, or one that is not all numbers
            continue
        d = torch.where(torch.isinf(x[t]), 0.0, x[t] - M).abs()
        e = torch.exp(x[t] - M)
        Z = e.sum()
        p = e / Z
        a1, logz = (p * d).sum().item(), math.log(Z)
        z = U * (4 * a1 + 65 + chain)
        last = U * (2 * (logz + 6) + 6)  # log s, and x - r with r up to 6 below M
        ref["tol_z"][t] = z + last
        ref["tol_h"][t] = z + last + U * (p * (4 * d + 73 + chain) * (d + 12)).sum().item() + (z + 2 * U) * (a1 + 6)
    return ref
