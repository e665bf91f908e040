"""Plain 64-bit forms of the operators of requests: attention over pages, adapters, controls on logits."""
import math

import torch


def paged_attention(q, k_cache, v_cache, table, lens, scale=None):
    """(result, sum of weight x |value|) of every row; rows without tokens give zeros."""
    rows, hq, d = q.shape
    page, hk = k_cache.shape[1], k_cache.shape[2]
    out, mass = torch.zeros(rows, hq, d, dtype=torch.float64, device=q.device), torch.zeros(rows, hq, d, dtype=torch.float64, device=q.device)
    scale = d ** -0.5 if scale is None else scale
    for r, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        used = table[r, :-(-n // page)].long()
        k, v = k_cache[used].reshape(-1, hk, d)[:n].double(), v_cache[used].reshape(-1, hk, d)[:n].double()
        w = torch.softmax(scale * torch.einsum("hgd,thd->hgt", q[r].double().view(hk, -1, d), k), dim=-1)
        out[r] = torch.einsum("hgt,thd->hgd", w, v).reshape(hq, d)
        mass[r] = torch.einsum("hgt,thd->hgd", w, v.abs()).reshape(hq, d)
    return out, mass


def adapters(y, x, pairs, scales, index):
    """(y + scale B A x, |scale| |B| |A| |x|); ``pairs[slot]``: (A, B) per part, or None."""
    y, x = y.double(), x.double()
    out, mass = y.clone(), torch.zeros_like(y)
    for r, s in enumerate(index):
        if s < 0 or pairs[s] is None:
            continue
        at = 0
        for part, n in pairs[s]:
            if part is not None:
                a, b = (t.double() for t in part)
                out[r, at:at + n] += scales[s] * (b @ (a @ x[r]))
                mass[r, at:at + n] = abs(scales[s]) * (b.abs() @ (a.abs() @ x[r].abs()))
            at += n
    return out, mass


def controls(logits, history=None, prompt=0, repetition=1.0, frequency=0.0, presence=0.0, biases=(), mask=None, dtype=torch.float64):
    """One row of logits after its controls, step by step in ``dtype``. ``history``: tokens; ``biases``: (token, value) pairs;
    ``mask``: list of 32-bit words."""
    v = logits.to(dtype).clone()
    num = lambda x: torch.tensor(x, dtype=torch.float32).to(dtype)
    history = [] if history is None else history
    for t in sorted(set(h for h in history if 0 <= h < len(v))):
        n = sum(1 for h in history[prompt:] if h == t)
        v[t] = v[t] / num(repetition) if v[t] > 0 else v[t] * num(repetition)
        v[t] = v[t] - num(frequency) * num(float(n))
        if n:
            v[t] = v[t] - num(presence)
    total = {}
    for t, b in biases:
        if 0 <= t < len(v):
            total[t] = total[t] + num(b) if t in total else num(b)
    for t, b in total.items():
        v[t] = v[t] + b
    if mask is not None:
        for t in range(len(v)):
            if not (int(mask[t // 32]) >> (t % 32)) & 1:
                v[t] = -math.inf
    return v
