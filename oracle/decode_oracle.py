"""Test infrastructure only: numpy f64 oracle of the decoding operators
(include/trba_decode.h and LinearInt4 of include/trba_ops.h), written from
their definitions.  Nothing in the product imports this file."""
from __future__ import annotations

import numpy as np

NEG = -np.inf


def log_probs(row: np.ndarray) -> np.ndarray:
    """f64 log softmax of one row; NaN counts as -inf, +inf tokens share."""
    row = np.where(np.isnan(row), NEG, np.asarray(row, np.float64))
    m = row.max()
    if m == NEG:
        return row
    if m == np.inf:
        return np.where(row == np.inf, -np.log((row == np.inf).sum()), NEG)
    z = row - m
    return z - np.log(np.exp(z).sum())


def totals(logits, scores, finished, eos) -> np.ndarray:
    """f64 scores [lines, beams, vocab] of every continuation."""
    scores = np.asarray(scores, np.float32)
    L, K = scores.shape
    logits = np.asarray(logits, np.float64).reshape(L, K, -1)
    out = np.full(logits.shape, NEG)
    for b in range(L):
        for k in range(K):
            s = float(scores[b, k])
            if not s > NEG:
                continue
            if finished is not None and finished[b, k]:
                out[b, k, eos] = s
            else:
                out[b, k] = s + log_probs(logits[b, k])
    with np.errstate(over="ignore"):  # what f32 cannot hold is no continuation
        out[~(out.astype(np.float32) > NEG)] = NEG
    return out


def beam_select(logits, scores, finished=None, eos=-1):
    """(scores f64, tokens, parents, finished), [lines, beams] each."""
    tot = totals(logits, scores, finished, eos)
    L, K, V = tot.shape
    res = [np.empty((L, K)), np.empty((L, K), np.int32), np.empty((L, K), np.int32), np.empty((L, K), bool)]
    for b in range(L):
        flat = tot[b].ravel()
        order = np.argsort(-flat, kind="stable")[:K]
        for k in range(K):
            at = order[k] if k < len(order) else 0
            if k >= len(order) or flat[at] == NEG:
                vals = (NEG, max(eos, 0), k, eos >= 0)
            else:
                p, t = divmod(int(at), V)
                vals = (flat[at], t, p, eos >= 0 and (t == eos or (finished is not None and bool(finished[b, p]))))
            for r, v in zip(res, vals):
                r[b, k] = v
    return res


def beam_sequences(tokens, parents, eos=-1, pad=0):
    T, L, K = tokens.shape
    seq, lengths = np.full((L, K, T), pad, np.int32), np.empty((L, K), np.int32)
    for b in range(L):
        for k in range(K):
            path, slot = [], k
            for t in range(T - 1, -1, -1):
                if not 0 <= slot < K:
                    path = None
                    break
                path.append(int(tokens[t, b, slot]))
                slot = int(parents[t, b, slot])
            if path is None:
                lengths[b, k] = -1
                continue
            path.reverse()
            n = path.index(eos) if eos in path else T
            seq[b, k, :n] = path[:n]
            lengths[b, k] = n
    return seq, lengths


def int4_quantize(w: np.ndarray, group: int):
    """codes [out, ceil(in / 2)] uint8 (even input in the low half) and scales
    [out, groups] of f32 weights: scale = max |w| / 7, halves away from zero."""
    w = np.asarray(w, np.float32)
    n, k = w.shape
    groups = -(-k // group)
    q = np.full((n, k + (k & 1)), 8, np.uint8)
    scales = np.ones((n, groups), np.float32)
    for g in range(groups):
        part = w[:, g * group:(g + 1) * group]
        mx = np.abs(part).max(1)
        s = np.where(mx > 0, (mx / np.float32(7)).astype(np.float32), np.float32(1))
        scales[:, g] = s
        v = np.clip((part / s[:, None]).astype(np.float32), -7, 7).astype(np.float64)
        q[:, g * group:g * group + part.shape[1]] = (np.sign(v) * np.floor(np.abs(v) + 0.5)).astype(np.int8) + 8
    return (q[:, ::2] | (q[:, 1::2] << 4)).astype(np.uint8), scales


def int4_weights(codes, scales, ins: int, group: int) -> np.ndarray:
    """f64 [out, in] of the codes and scales."""
    q = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)[:, :ins].astype(np.float64) - 8
    return q * np.repeat(np.asarray(scales, np.float64), group, 1)[:, :ins]
