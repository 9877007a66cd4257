"""Top-p sampling and draft verification in 64 bits, row by row, and chunk attention in 64 bits: the
definitions that the kernels of the speculative step are checked against."""
from __future__ import annotations

import math

import numpy as np
import torch


def row_probs(logits: torch.Tensor, temperature: float, top_p: float) -> np.ndarray:
    """Kept, renormalised probabilities of one row: tokens ranked by value (lower index first among equals),
    kept while the mass ranked before them is at most top_p. temperature <= 0 or NaN: one at the argmax. NaN
    and -inf are no tokens; a row without tokens is all 0."""
    x = logits.double().cpu().numpy().copy()
    x[np.isnan(x)] = -np.inf
    p = np.zeros_like(x)
    top = x.max()
    if top == -np.inf:
        return p
    if not temperature > 0:
        p[int(np.argmax(x))] = 1.0
        return p
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / np.float64(temperature)))
    w[np.isnan(w) | (x == -np.inf)] = 0.0
    if top_p < 1:
        order = np.argsort(-x, kind="stable")
        ws = w[order]
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        p[order] = np.where(before <= max(top_p, 0.0) * w.sum(), ws, 0.0)
    else:
        p = w
    return p / p.sum()


def drawable(p: np.ndarray) -> np.ndarray:
    """Weights below 2^-45 of the largest cannot be drawn (weights are multiples of 2^-44)."""
    return np.where(p < 2.0**-45 * p.max(), 0.0, p)


def draw(p: np.ndarray, u: float) -> int:
    """First index whose running sum exceeds u times the whole; 0 when there is no mass."""
    c = np.cumsum(p)
    if c[-1] == 0:
        return 0
    return int(np.searchsorted(c, np.float64(u) * c[-1], side="right"))


def sample(logits, temperature, top_p, uniform):
    p = [row_probs(l, float(t), float(k)) for l, t, k in zip(logits, temperature, top_p)]
    return np.array([draw(drawable(r), float(u)) for r, u in zip(p, uniform)], dtype=np.int32), np.stack(p) if p else None


def verify(logits, tokens, indptr, uniform, temperature, top_p, draft_probs=None):
    """(accepted, next token) of every request."""
    accepted, following = [], []
    vocab = logits.shape[1]
    tok, u = [int(t) for t in tokens], [float(x) for x in uniform]
    for i, (a, b) in enumerate(zip(indptr[:-1], indptr[1:])):
        a, b = int(a), int(b)
        if a == b:
            accepted.append(0)
            following.append(-1)
            continue
        r = a
        while True:
            p = drawable(row_probs(logits[r], float(temperature[i]), float(top_p[i])))
            if r == b - 1:
                break
            x = tok[r + 1]
            q = np.zeros(vocab)
            if draft_probs is not None:
                q = draft_probs[r].double().cpu().numpy()
            elif 0 <= x < vocab:
                q[x] = 1.0
            inside = 0 <= x < vocab
            if not (inside and u[r] * q[x] < p[x]):
                rest = np.maximum(p - q, 0.0)
                p = rest if rest.sum() > 0 else p
                break
            r += 1
        accepted.append(r - a)
        following.append(draw(p, u[b - 1]))
    return np.array(accepted, dtype=np.int32), np.array(following, dtype=np.int32)


def chunk_attention(q, pages, qo, kv_indices, kv_indptr, lens, scale=None):
    """(out, lse, A, B) in float64 on q's device: the result, its log-sum-exp, and what error bounds need: A =
    sum_t p |v| per element and B = max_t sum_d |q_d k_d| scale per row. `lens`: kv length of every request; row j
    of n sees positions <= len - n + j."""
    _, _, ps, hkv, d = pages.shape
    nnz, hq, _ = q.shape
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    dev = q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    size = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.full((nnz, hq), -math.inf, dtype=torch.float64, device=dev)
    reach = torch.zeros((nnz, hq), dtype=torch.float64, device=dev)
    for i, n_kv in enumerate(int(x) for x in lens):
        a, b = int(qo[i]), int(qo[i + 1])
        if a == b or n_kv <= 0:
            continue
        kv = pages[kv_indices[int(kv_indptr[i]): int(kv_indptr[i + 1])].long()]
        k = kv[:, 0].reshape(-1, hkv, d)[:n_kv].double().repeat_interleave(g, 1).transpose(0, 1)
        v = kv[:, 1].reshape(-1, hkv, d)[:n_kv].double().repeat_interleave(g, 1).transpose(0, 1)
        for j in range(a, b):
            seen = n_kv - (b - a) + (j - a) + 1
            if seen <= 0:
                continue
            x = (k[:, :seen] @ q[j].double()[:, :, None]).squeeze(-1) * scale
            p = torch.softmax(x, dim=-1)
            lse[j] = torch.logsumexp(x, dim=-1)
            out[j] = (p[:, None] @ v[:, :seen]).squeeze(1)
            size[j] = (p[:, None] @ v[:, :seen].abs()).squeeze(1)
            reach[j] = ((k[:, :seen].abs() @ q[j].double().abs()[:, :, None]).squeeze(-1) * abs(scale)).amax(-1)
    return out, lse, size, reach
