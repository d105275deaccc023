"""64-bit definitions of the operators of a decode step with drafted tokens (CPU or GPU tensors)."""
from __future__ import annotations

import math

import torch


def visible(positions: torch.Tensor, num_keys: int, window: int, sinks: int) -> torch.Tensor:
    """[rows, keys]: whether the row at each position sees each key."""
    t, j = positions.view(-1, 1), torch.arange(num_keys, device=positions.device).view(1, -1)
    seen = j <= t
    if window:
        seen = seen & ((j > t - window) | (j < sinks))
    return seen


def sequence_keys(cache: torch.Tensor, table: torch.Tensor, num_keys: int) -> torch.Tensor:
    """Rows [num_keys, kv_heads, D] (fp64) of a paged cache [pages, block, kv_heads, D]; rows of pages that the
    table does not have (below 0) are zeros."""
    block = cache.shape[1]
    j = torch.arange(num_keys, device=cache.device)
    page = table.to(torch.int64)[j // block]
    rows = cache[page.clamp(min=0), j % block].double()
    return torch.where((page >= 0).view(-1, 1, 1), rows, torch.zeros_like(rows))


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, window: int, sinks: int,
              scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """softmax(scale q K) V of rows q [rows, heads, D] at the positions over k / v [keys, kv_heads, D], all fp64:
    (output, root of the mean square of V under the softmax).  Keys that a row does not see may hold anything;
    rows that see none give zeros."""
    rows, heads, d = q.shape
    group = heads // k.shape[1]
    seen = visible(positions, k.shape[0], window, sinks)
    out, rms = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        score = (q[:, h] @ kh.T * scale).masked_fill(~seen, -math.inf)
        p = torch.nan_to_num(torch.softmax(score, -1)) if k.shape[0] else score
        if not bool(torch.isfinite(vh).all()):
            vh = torch.where(seen.any(0).view(-1, 1), vh, torch.zeros_like(vh))
        out[:, h], rms[:, h] = p @ vh, (p @ vh.square()).sqrt()
    return out, rms


def step(context_lens, new_lens, tables, free_pages, num_free, block, total_rows, window, sinks):
    """The metadata of a step on lists of ints, sequence by sequence; returns (positions, slots, cu_q, cu_k, lengths,
    tables, free_pages, num_free)."""
    tables, free = [list(t) for t in tables], list(free_pages)
    context = [max(n, 0) for n in context_lens]
    fresh = [0 if n < 0 else max(m, 0) for n, m in zip(context_lens, new_lens)]
    rows = [max(m, 0) for m in new_lens]     # idle places (below 0) have rows too
    for table, n, m in zip(tables, context, fresh):
        for t in range(n, n + m):
            page = t // block
            if page < len(table) and table[page] < 0 and num_free > 0:
                num_free -= 1
                table[page] = free[num_free]
    if window:
        for table, n in zip(tables, context):
            for page in range(len(table)):
                keys = range(page * block, (page + 1) * block)
                if keys[0] >= sinks and keys[-1] <= n - window and table[page] >= 0:
                    free[num_free] = table[page]
                    num_free += 1
                    table[page] = -1
    positions, slots, cu_q, cu_k = [], [], [0], [0]
    for table, n, m, k in zip(tables, context, fresh, rows):
        for t in range(n, n + m):
            page = table[t // block] if t // block < len(table) else -1
            positions.append(t)
            slots.append(page * block + t % block if page >= 0 else -1)
        positions += [0] * (k - m)
        slots += [-1] * (k - m)
        cu_q.append(cu_q[-1] + k)
        cu_k.append(cu_k[-1] + n + m)
    pad = max(0, total_rows - len(positions))
    return (positions[:total_rows] + [0] * pad, slots[:total_rows] + [-1] * pad, cu_q, cu_k,
            [n + m for n, m in zip(context, fresh)], tables, free, num_free)


def _count(x: float) -> int:
    """What a probability counts as."""
    return 0 if math.isnan(x) else int(min(max(x, 0.0), 1.0) * 2 ** 42)


def verify(drafts, target, draft, u, u_last):
    """One sequence's verification in whole numbers: drafts a list, target [K + 1, V] and draft [K, V] (or None) tensors
    of the caller's type, u a list, u_last a number; returns the emitted tokens."""
    kept, weights = [], None
    vocab = target.shape[1]
    for i, d in enumerate(drafts):
        if not 0 <= d < vocab:
            break
        q = 1.0 if draft is None else float(draft[i, d])
        if u[i] * q < float(target[i, d]):   # (a product of two fp32 numbers is exact in 64 bits)
            kept.append(d)
            continue
        if draft is None:
            weights = target[i].float().clone()
            weights[d] = 0.0
        else:
            weights = target[i].float() - draft[i].float()
        break
    n = len(kept)
    for w in ([] if weights is None else [weights]) + [target[n].float()]:
        counts = [_count(x) for x in w.tolist()]
        total = sum(counts)
        if total > 0:
            break
    else:
        return kept + [-1]
    r = 0.0 if math.isnan(u_last) else min(max(u_last, 0.0), 1.0 - 2.0 ** -24)
    goal = int(r * 2 ** 24) * total // 2 ** 24
    upto = 0
    for v, c in enumerate(counts):
        upto += c
        if upto > goal:
            return kept + [v]
