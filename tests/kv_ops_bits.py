"""Bars for attention over the Q8_0 KV cache that see how many bits the
operands have, where kv_ops_util's bar, in units of max |V|, does not.

Random caches (`row_errors`, `row_bar`).  An output is sum p_t V_t with V_t of
mean zero, and an operand's rounding gives each weight a relative error
delta_t of its own: the error sum delta_t p_t V_t is to the output as delta is
to one, in norms over a head's dims.  With S the largest
sqrt(sum (q_d K_td)^2) / sqrt(hd), delta's root mean square is at most the sum of
  S 2^-22                  a query in two f16 terms
  S sqrt(hd + 8) 2^-24     the products' f32 sums, roundings independent
  2^-21                    exp2, the weight's and the value's two terms
  sqrt(L / 16 + 64) 2^-24  the f32 sums over L rows
and a head's norms, of 32 dims at least, leave that by a factor below 6.  One
f16 term in place of two is 2^-12 / sqrt(3) = 1.4e-4 of any of them.

One row far above the others, with value zero (`sink`).  All scores are 0 but
for row 0, whose score is `gap`: q and K are integers and powers of two, and
the values positive, so an output is sum p_t V_t of equal signs and its
relative error is at most the largest of the weights'.  A weight 2^-x of the
largest is right to 2^-38 of that, so to 2^(x - 38) of itself, its product with
a scale in the upper half of its range to four times that (kv_ops.hpp); the
row's own weight, in the sum that divides, has the score's rounding: three of
the factor log2(e) / sqrt(hd) and one more, times gap.  The sums of the
products and of the weights run in pieces of at most L / 16 + 64 f32
additions; equal terms on a large sum round the same way each time, so their
errors add up: 0.377 of a weight on one of 2^13, 190 times, where a step is
2^-10, is off by up to 190 2^-11 = 2^-16.4 of the sum.
  gap 2^-22 + 5 exp(gap) 2^-38 + 2^-21 + 2 (L / 16 + 64) 2^-24
"""
import numpy as np

from kv_ops_util import HostCache


def row_errors(out, ref, hd):
    """Error norm / output norm of every row and head."""
    o, r = (np.asarray(x, np.float64).reshape(-1, hd) for x in (out, ref))
    return np.linalg.norm(o - r, axis=1) / np.linalg.norm(r, axis=1)


def row_bar(host, q, rows):
    hd = host.hd
    k2 = host.values("k") ** 2
    group = q.shape[1] // hd // host.n_kv
    q2 = q.astype(np.float64).reshape(q.shape[0], host.n_kv, group, hd) ** 2
    S = max(np.sqrt((q2[:, kv].reshape(-1, hd) @ k2[:, kv].T).max() / hd) for kv in range(host.n_kv))
    return 6 * (S * (2.0 ** -22 + np.sqrt(hd + 8) * 2.0 ** -24) + 2.0 ** -21 + np.sqrt(rows / 16 + 64) * 2.0 ** -24)


def sink(rows, n_kv, hd, gap, n_tok, n_head, seed):
    """(cache, queries, the gap as it is): row 0 has score `gap` for every
    query, all others 0."""
    host = HostCache(rows, n_kv, hd, seed)
    r = np.random.default_rng(seed)
    host.k_qs[:] = r.integers(-127, 128, host.k_qs.shape)
    host.k_qs[:, ::hd] = 0
    host.k_qs[0, ::hd] = 64
    host.k_d[:] = 2.0 ** -6
    host.v_qs[:] = r.integers(64, 128, host.v_qs.shape)
    host.v_qs[0] = 0
    host.v_d[:] = 2.0 ** -7
    q = np.zeros((n_tok, n_head, hd), np.float32)
    q[:, :, 0] = np.round(gap * np.sqrt(hd))
    return host, q.reshape(n_tok, -1), float(q[0, 0, 0]) / np.sqrt(hd)


def sink_bar(gap, rows):
    return gap * 2.0 ** -22 + 5 * np.exp(gap) * 2.0 ** -38 + 2.0 ** -21 + 2 * (rows / 16 + 64) * 2.0 ** -24
