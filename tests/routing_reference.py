"""Routing's definition in 64 bits (numpy, one token at a time), and how far fp32 weights and gradients may be from it."""

from __future__ import annotations

import numpy as np

HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}
TINY = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25, "float32": 2.0 ** -150}


def scores_of(logits: np.ndarray, scoring: str) -> np.ndarray:
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            return 1 / (1 + np.exp(-logits))
        e = np.exp(logits - logits.max())
        return e / e.sum()


def _order(values: np.ndarray, open_: np.ndarray) -> list[int]:
    """The open ones, largest first, NaN after all numbers, equal ones by index."""
    at = [i for i in range(len(values)) if open_[i]]
    return sorted(at, key=lambda i: (np.isnan(values[i]), -values[i] if not np.isnan(values[i]) else 0.0, i))


def choose(logits, top_k, *, scoring="softmax", bias=None, groups=1, top_groups=None, group_score="max", **_) -> list[int]:
    """One token's experts, the best first; -1 where there are no more."""
    experts = len(logits)
    with np.errstate(all="ignore"):
        score = scores_of(logits, scoring)
        open_ = logits != -np.inf
        choice = logits
        if bias is not None:
            open_ = open_ & (bias != -np.inf)
            choice = score + bias
        if groups > 1:
            per = experts // groups
            value, some = np.zeros(groups), np.zeros(groups, bool)
            for g in range(groups):
                inside = slice(g * per, (g + 1) * per)
                part = choice if bias is not None or group_score == "max" else score
                best = _order(part[inside], open_[inside])
                some[g] = len(best) > 0
                value[g] = sum(part[inside][i] for i in best[:2 if group_score == "top2" else 1])
            kept = _order(value, some)
            kept += [g for g in range(groups) if not some[g]]
            keep = np.zeros(groups, bool)
            keep[kept[:top_groups or groups]] = True
            open_ = open_ & np.repeat(keep, per)
    chosen = _order(choice, open_)[:top_k]
    return chosen + [-1] * (top_k - len(chosen))


def weights_of(logits, chosen, *, scoring="softmax", renormalize=True, scale=1.0, **_) -> np.ndarray:
    with np.errstate(all="ignore"):
        score = scores_of(logits, scoring)
        has = np.array(chosen) >= 0
        w = np.where(has, score[np.array(chosen)], 0.0)
        if renormalize:
            if scoring == "softmax" and np.isfinite(logits.max()) and not np.isnan(logits).any():
                # relative to the largest chosen one, where all the token's scores may be too small for any number
                top = logits[np.array(chosen)][has].max() if has.any() else 0.0
                w = np.where(has, np.exp(logits[np.array(chosen)] - top), 0.0)
                w = w / w.sum() if has.any() else w
            else:
                w = w / max(w.sum(), 2.0 ** -100) if not np.isnan(w.sum()) else np.where(has, np.nan, 0.0)
        return np.where(has, w * scale, 0.0)


def order_of(experts: np.ndarray, count: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """(ends, rows, source) of choices (tokens, top_k)."""
    flat = experts.reshape(-1)
    source = np.full(flat.size, -1)
    rows = np.full(flat.size, -1)
    ends, at = [], 0
    for e in range(count):
        for i in np.nonzero(flat == e)[0]:
            source[at], rows[i] = i, at
            at += 1
        ends.append(at)
    return np.array(ends), rows.reshape(experts.shape), source


def route(logits: np.ndarray, top_k: int, *, mask=None, **rules):
    """(weights, experts, ends, rows, source)."""
    tokens, count = logits.shape
    experts = np.full((tokens, top_k), -1)
    weights = np.zeros((tokens, top_k))
    for t in range(tokens):
        if mask is None or mask[t]:
            experts[t] = choose(logits[t], top_k, **rules)
            weights[t] = weights_of(logits[t], experts[t], **rules)
    return (weights, experts, *order_of(experts, count))


def unit(logits: np.ndarray) -> float:
    """A weight's relative error in fp32. exp is within 2 steps of 2^-23 and its argument, a difference, within half a step
    of at most D, the row's range; so is each term of a sum of at most 32 numbers in a lane and 5 more over the warp; a score
    and a renormalised one are quotients of two such (twice that), with a rounding each, and the scale's."""
    finite = logits[np.isfinite(logits)]
    spread = float(finite.max() - finite.min()) if finite.size else 0.0
    return 2.0 ** -24 * (2 * (4 + spread + 37) + 4)


def gradient(logits, experts, g, *, scoring="softmax", renormalize=True, scale=1.0, **_):
    """(the logits' gradient, what its errors are relative to): every difference counts with the size of its terms."""
    tokens, count = logits.shape
    out, size = np.zeros((tokens, count)), np.zeros((tokens, count))
    for t in range(tokens):
        has = experts[t] >= 0
        at = experts[t][has]
        if not has.any():
            continue
        gs = g[t][has] * scale
        score = scores_of(logits[t], scoring)
        if scoring == "sigmoid":
            inner, inner_size = gs, np.abs(gs)
            if renormalize:
                total = score[at].sum()
                if total < 2.0 ** -100:
                    inner, inner_size = gs / 2.0 ** -100, np.abs(gs) / 2.0 ** -100
                else:
                    inner = (gs - (gs * score[at]).sum() / total) / total
                    inner_size = (np.abs(gs) + (np.abs(gs) * score[at]).sum() / total) / total
            slope = score[at] / (1 + np.exp(logits[t][at]))
            out[t][at], size[t][at] = inner * slope, inner_size * slope
        elif renormalize:
            share = weights_of(logits[t], list(experts[t]), scoring=scoring)[has]
            out[t][at] = share * (gs - (gs * share).sum())
            size[t][at] = share * (np.abs(gs) + (np.abs(gs) * share).sum())
        else:
            mean, mean_size = (gs * score[at]).sum(), (np.abs(gs) * score[at]).sum()
            out[t], size[t] = -score * mean, score * mean_size
            out[t][at] += score[at] * gs
            size[t][at] += score[at] * np.abs(gs)
    return out, size
