"""Plain 64-bit forms of the group operators, and what their results may be off by.

The reference attends token t of sequence i over the prefix rows and its own
rows up to its own position, per query head, in float64.  Next to the output it
returns, per output element, how far a kernel may be off it:

  P   the weights enter the second product rounded to bf16: one rounding (off by
      at most 2^-8 of the weight) with bf16 activations, two (hi + lo parts, off
      by at most 2^-16) with fp32 ones.  That moves the output by at most
      e_P * A, A = sum(w |v|) / sum(w).
  q   exact with bf16 activations; hi + lo parts, off by at most 2^-16 |q|, with
      fp32 ones: a score moves by at most 2^-16 B, B = max_j sum_d |q_d k_jd| *
      scale, a normalised weight by at most twice that relatively.
  sum fp32 sums of the scores (head_dim terms) and of the outputs (steps of 16
      positions, each part of P by itself), off by at most 2^-23 per step (the
      tensor core truncates), and 2^-22 of a weight for the exponential.
  out rounded once to the output type.
"""
import numpy as np

import oracle as O


def reference(q, parts, scale, bf16):
    """q [t][hd] of one query head; parts: list of (k, v) float64 [n][hd] whose
    rows all t queries see, the last one causally: query j sees its first
    n - t + j + 1 rows.  Returns (out, tol), float64 [t][hd]."""
    t, hd = q.shape
    k = np.concatenate([p[0] for p in parts])
    v = np.concatenate([p[1] for p in parts])
    n = len(k)
    seen = np.arange(n)[None, :] <= (n - t + np.arange(t))[:, None]
    s = np.where(seen, q @ k.T * scale, -np.inf)
    w = np.where(seen, np.exp(s - s.max(1, keepdims=True)), 0.0)
    l = w.sum(1, keepdims=True)
    out = (w @ v) / l
    A = (w @ np.abs(v)) / l
    B = np.where(seen, np.abs(q) @ np.abs(k).T * scale, 0.0).max(1, keepdims=True)
    e_p, e_q, terms = (2.0 ** -8, 0.0, 1) if bf16 else (2.0 ** -16, 2.0 ** -16, 2)
    steps = terms * (n / 16 + 8)
    e = e_p + 2 * (e_q + terms * hd * 2.0 ** -23) * B + 2 * steps * 2.0 ** -23 + 2.0 ** -21
    tol = A * e + np.abs(out) * (2.0 ** -8 if bf16 else 2.0 ** -23)
    return out, tol


def group_reference(q, prefix, owns, n_new, nkv, scale, bf16):
    """q [total][nh][hd] float64, prefix (k, v) [P][nkv][hd] or None, owns: per
    sequence (k, v) [len][nkv][hd] with its new rows.  (out, tol) as q."""
    out, tol = np.empty_like(q), np.empty_like(q)
    nh, at = q.shape[1], 0
    for (k, v), t in zip(owns, n_new):
        for h in range(nh if t else 0):
            c = h * nkv // nh
            parts = [(prefix[0][:, c], prefix[1][:, c])] if prefix is not None else []
            parts.append((k[:, c], v[:, c]))
            out[at:at + t, h], tol[at:at + t, h] = reference(q[at:at + t, h], parts, scale, bf16)
        at += t
    return out, tol


def bf16(x):
    """x rounded to bf16: (bits uint16, values float64)."""
    b = O.f32_to_bf16(np.ascontiguousarray(x, np.float32))
    return b, O.bf16_to_f32(b).astype(np.float64)
