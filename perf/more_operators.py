"""The operators of a decode step with drafted tokens over a windowed cache that are measured, with their plain forms.

Four operators, each as a user of the package calls it:
  decode   attention of the last 1 .. n tokens of each sequence over the paged bf16 cache, with a sliding
           window and a few first tokens (sinks) that stay visible; n > 1 are drafted tokens to be verified;
  prefill  the same mask for prompts and for the next piece of a long prompt;
  step     block tables and slot maps built on the GPU from the sequences' lengths: pages taken from a free
           list where a table has none, pages behind the window given back, positions and slots of every
           new row;
  verify   drafted tokens accepted or refused against the target's probabilities from given random
           numbers, and the token after them sampled.

The mask: row r of a sequence's n has position t = len - n + r and sees key j iff j <= t and (window == 0 or
j > t - window or j < sinks).

The sampled token is exact: a probability x counts as floor(clamp(x, 0, 1) * 2^42) (x = fp32(p - q) at a refused
draft), and the token is the first whose cumulative count passes floor(floor(u * 2^24) * total / 2^24).
"""
import math

import torch

own = False

D = 128            # head size
COUNT = 2.0 ** 42  # what a probability of 1 counts as
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ACCEPT = 0.75      # about the share of drafted tokens that the inputs below get accepted


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One request alone, one token a step, a short window: the smallest call, latency.
        {"name": "decode_one", "op": "decode", "seqs": 1, "rows": 1, "min_len": 6001, "max_len": 6001, "heads": 16,
         "kv_heads": 2, "block": 256, "window": 1024, "sinks": 4, "released": True},
        # A decode step of 64 requests of ragged lengths, a quarter of them shorter than the window: bandwidth.
        {"name": "decode_batch_64", "op": "decode", "seqs": 64, "rows": 1, "min_len": 2700, "max_len": 10700,
         "heads": 28, "kv_heads": 4, "block": 256, "window": 4096, "sinks": 4, "released": True},
        # The same step with four drafted tokens behind each last one.
        {"name": "decode_drafts_64", "op": "decode", "seqs": 64, "rows": 5, "min_len": 2700, "max_len": 10700,
         "heads": 28, "kv_heads": 4, "block": 256, "window": 4096, "sinks": 4, "released": False},
        # Drafted tokens of two long requests that see every key: few rows over a very long axis.
        {"name": "decode_drafts_two_long", "op": "decode", "seqs": 2, "rows": 4, "min_len": 100003, "max_len": 131071,
         "heads": 16, "kv_heads": 2, "block": 256, "window": 0, "sinks": 0, "released": False},
        # A whole prompt with a 4K image (20 + 10549 + 48 tokens) under a window, 7B shapes: matrix products.
        {"name": "prefill_prompt_4k_image", "op": "prefill", "seqs": 1, "rows": 10617, "before": 0, "heads": 28,
         "kv_heads": 4, "block": 256, "window": 4096, "sinks": 4},
        # The next pieces of two long prompts, whose earlier pages are mostly behind the window.
        {"name": "prefill_pieces_of_two", "op": "prefill", "seqs": 2, "rows": 513, "before": 20011, "heads": 16,
         "kv_heads": 2, "block": 256, "window": 1024, "sinks": 4},
        # The metadata of a decode step of a few requests: the smallest call, latency.
        {"name": "step_decode_8", "op": "step", "seqs": 8, "min_new": 1, "max_new": 1, "min_len": 700,
         "max_len": 10700, "block": 256, "width": 44, "window": 0, "sinks": 0},
        # Of 256 requests with four drafted tokens each, whose pages behind the window are given back.
        {"name": "step_drafts_256", "op": "step", "seqs": 256, "min_new": 5, "max_new": 5, "min_len": 2700,
         "max_len": 10700, "block": 256, "width": 44, "window": 4096, "sinks": 4},
        # Of 64 prompts of up to a 4K image: every page is taken from the list.
        {"name": "step_prompts_64", "op": "step", "seqs": 64, "min_new": 48, "max_new": 10617, "min_len": 0,
         "max_len": 0, "block": 256, "width": 44, "window": 0, "sinks": 0},
        # One request with four drafted tokens: latency.
        {"name": "verify_one", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 151936, "dtype": "fp32",
         "draft_probs": True, "ragged": False},
        # 64 requests with up to four.
        {"name": "verify_batch_64", "op": "verify", "seqs": 64, "drafts": 4, "vocab": 152064, "dtype": "fp32",
         "draft_probs": True, "ragged": True},
        # 256 requests whose drafts were looked up in their own text, so that they have no probabilities.
        {"name": "verify_lookup_256", "op": "verify", "seqs": 256, "drafts": 3, "vocab": 151936, "dtype": "bf16",
         "draft_probs": False, "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads = rng.choice([(28, 4), (16, 2), (16, 2), (28, 4), (32, 8), (8, 8), (12, 1), (32, 2)])
    block = rng.choice([256, 256, 128])
    op = rng.choice(["decode", "decode", "prefill", "step", "verify", "verify"])
    window = rng.choice([0, _log(rng, 1, 8192), _log(rng, 128, 8192)])
    sinks = rng.choice([0, 4, rng.randint(1, 300)]) if window else 0
    if op == "decode":
        seqs = _log(rng, 1, 100)
        rows = rng.choice([1, 1, 2, 3, 5, 8])
        longest = _log(rng, rows, max(rows, min(131072, 1000000 // (seqs * kv_heads))))
        return {"op": "decode", "seqs": seqs, "rows": rows, "min_len": max(rows, longest - _log(rng, 1, longest + 1)),
                "max_len": longest, "heads": heads, "kv_heads": kv_heads, "block": block, "window": window,
                "sinks": sinks, "released": rng.random() < 0.5}
    if op == "prefill":
        return {"op": "prefill", "seqs": rng.randint(1, 3), "rows": _log(rng, 1, 5000),
                "before": rng.choice([0, _log(rng, 1, 5000)]), "heads": heads, "kv_heads": kv_heads, "block": block,
                "window": window, "sinks": sinks}
    if op == "step":
        seqs, most = _log(rng, 1, 400), rng.choice([1, rng.randint(2, 9), _log(rng, 10, 6000)])
        longest = rng.choice([0, _log(rng, 1, 30000)])
        return {"op": "step", "seqs": seqs, "min_new": rng.choice([most, 0]), "max_new": most,
                "min_len": longest // 3, "max_len": longest, "block": block, "width": (longest + most) // block + 2,
                "window": window, "sinks": sinks}
    seqs, drafts = _log(rng, 1, 100), rng.randint(0, 8)
    vocab = _log(rng, 1000, min(160000, 50000000 // (seqs * (drafts + 1))))
    return {"op": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab,
            "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "draft_probs": rng.random() < 0.6,
            "ragged": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _permutation(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def _lengths(case, seed):
    """(new rows, lengths with them) of each sequence."""
    import random
    r = random.Random(seed)
    if case["op"] == "decode":
        return [case["rows"]] * case["seqs"], [r.randint(case["min_len"], case["max_len"]) for _ in range(case["seqs"])]
    if case["op"] == "prefill":
        new = [max(1, case["rows"] - 37 * i) for i in range(case["seqs"])]
        return new, [n + case["before"] for n in new]
    same = random.Random(case["seqs"])                                   # (the rows of all seeds are as many)
    new = [same.randint(case["min_new"], case["max_new"]) for _ in range(case["seqs"])]
    r.shuffle(new)
    return new, [n + r.randint(case["min_len"], case["max_len"]) for n in new]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "verify":
        return _prepare_verify(s, case, g, seed)
    new, lens = _lengths(case, seed)
    block = case["block"]
    if case["op"] == "step":
        before = [n - k for n, k in zip(lens, new)]
        held = [(b + block - 1) // block for b in before]
        pool = case["seqs"] * case["width"] + 3
        order = _permutation(g, pool).to(torch.int32)
        tables, at = [], 0
        for n, b in zip(held, before):
            # pages far behind the window went back in earlier steps, the last one or two did not yet
            first = (case["sinks"] + block - 1) // block
            gone = max(first, (b - case["window"] + 1) // block - 2) if case["window"] else 0
            tables.append([-1 if first <= p < gone else at + p for p in range(n)] + [-1] * (case["width"] - n))
            at += n
        tables = torch.tensor(tables, device="cuda")
        s["block_tables"] = torch.where(tables >= 0, order[tables.clamp(min=0)], -1).to(torch.int32)
        taken = torch.zeros(pool, dtype=torch.bool, device="cuda")
        taken[s["block_tables"][s["block_tables"] >= 0].long()] = True
        free = _permutation(g, pool)
        free = free[~taken[free]].to(torch.int32)
        s["free_pages"] = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
        s["free_pages"][:free.numel()] = free
        s["num_free"] = torch.tensor([free.numel()], dtype=torch.int32, device="cuda")
        s["lens"] = torch.tensor(before, dtype=torch.int32, device="cuda")
        s["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        s["rows"] = sum(new) + 3                                         # a captured step has room to spare
        return s
    heads, kv_heads = case["heads"], case["kv_heads"]
    widths = [max(1, (n + block - 1) // block) for n in lens]
    pages = sum(widths) + 2
    order = _permutation(g, pages)
    tables, at = [], 0
    for n, k, w in zip(lens, new, widths):
        first = (case["sinks"] + block - 1) // block
        gone = (n - k - case["window"] + 1) // block if case["window"] and case.get("released", True) else 0
        tables.append([-1 if first <= p < gone else at + p for p in range(w)] + [-1] * (max(widths) - w))
        at += w
    tables = torch.tensor(tables, device="cuda")
    s["tables"] = torch.where(tables >= 0, order[tables.clamp(min=0)], -1).to(torch.int32)
    size = torch.exp(0.5 * _normal(g, D))
    s["k_cache"], s["v_cache"] = (torch.empty(pages, block, kv_heads, D, dtype=torch.bfloat16, device="cuda")
                                  for _ in range(2))
    step = max(1, (1 << 22) // (block * kv_heads))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        s["k_cache"][p:p + n] = _normal(g, n, block, kv_heads, D) * size
        s["v_cache"][p:p + n] = _normal(g, n, block, kv_heads, D)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["softmax_scale"] = 1.0 / math.sqrt(D)
    s["max_len"] = max(widths) * block
    if case["op"] == "decode":
        s["q"] = (1.5 * _normal(g, len(lens), case["rows"], heads, D)).to(torch.bfloat16)
        return s
    cu_q, cu_k = [0], [0]
    for a, b in zip(new, lens):
        cu_q.append(cu_q[-1] + a)
        cu_k.append(cu_k[-1] + b)
    s["q"] = (1.5 * _normal(g, cu_q[-1], heads, D)).to(torch.bfloat16)
    s["cu_q"], s["cu_k"] = cu_q, cu_k
    if own:  # the plan of the step, which every layer of it shares
        from vlcache_b200 import ops
        s["plan"] = ops.build_prefill_plan(cu_q, cu_k, heads, kv_heads, device="cuda", window=case["window"],
                                           sinks=case["sinks"])
    return s


def _prepare_verify(s, case, g, seed):
    seqs, drafts, vocab, dtype = case["seqs"], case["drafts"], case["vocab"], TYPES[case["dtype"]]
    s["p"] = torch.empty(seqs, drafts + 1, vocab, dtype=dtype, device="cuda")
    s["q"] = torch.empty(seqs, drafts, vocab, dtype=dtype, device="cuda") if case["draft_probs"] else None
    s["drafts"] = torch.empty(seqs, drafts, dtype=torch.int64, device="cuda")
    step = max(1, (1 << 24) // (vocab * (drafts + 1)))
    for i in range(0, seqs, step):
        n = min(step, seqs - i)
        logits = 5.0 * _normal(g, n, drafts + 1, vocab)
        p = torch.softmax(logits, -1)
        s["p"][i:i + n] = p
        near = torch.softmax(logits[:, :drafts] + 0.6 * _normal(g, n, drafts, vocab), -1)
        if case["draft_probs"]:
            s["q"][i:i + n] = near
        if drafts:
            pick = near if case["draft_probs"] else p[:, :drafts]
            noise = torch.empty_like(pick).exponential_(generator=g)
            token = (pick / noise).argmax(-1)
            best = p[:, :drafts].argmax(-1)
            lucky = torch.rand(n, drafts, generator=g, device="cuda") < 0.6
            s["drafts"][i:i + n] = token if case["draft_probs"] else torch.where(lucky, best, token)
    if case["ragged"]:  # requests with fewer drafts: padded with -1
        import random
        r = random.Random(seed)
        count = torch.tensor([r.randint(0, drafts) for _ in range(seqs)], device="cuda")
        s["drafts"].masked_fill_(torch.arange(drafts, device="cuda") >= count.view(-1, 1), -1)
    s["u"] = torch.rand(seqs, drafts, generator=g, device="cuda")
    s["u_last"] = torch.rand(seqs, generator=g, device="cuda")
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if s["op"] == "decode":
        return _run_decode(s)
    if s["op"] == "prefill":
        return _run_prefill(s)
    if s["op"] == "step":
        return _run_step(s)
    return _run_verify(s)


def _softmax_v(score, v):
    """Rows of softmax(score) v; rows that see nothing are zeros."""
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, torch.ones_like(total), total)


def _run_decode(s):
    c = s["case"]
    if own:
        from vlcache_b200 import ops
        return ops.decode_attention_window(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["max_len"],
                                           s["softmax_scale"], c["window"], c["sinks"])
    seqs, n, heads, kv_heads = c["seqs"], c["rows"], c["heads"], c["kv_heads"]
    group = heads // kv_heads
    q = s["q"].float().view(seqs, n, kv_heads, group, D).permute(0, 2, 1, 3, 4).flatten(2, 3)
    pages = s["tables"].long().clamp(min=0)
    key = torch.arange(pages.shape[1] * c["block"], device=q.device)
    at = (s["lens"].view(-1, 1) - n + torch.arange(n, device=q.device)).repeat_interleave(group, 1)[:, None, :, None]
    seen = key <= at
    if c["window"]:
        seen &= (key > at - c["window"]) | (key < c["sinks"])
    o = torch.empty(seqs, kv_heads, n * group, D, device=q.device)
    for h in range(kv_heads):
        k = s["k_cache"][pages, :, h].flatten(1, 2).float()              # [seqs, keys, D]
        score = (q[:, h] @ k.transpose(-1, -2)) * s["softmax_scale"]
        score = torch.where(seen[:, 0], score, -math.inf)
        o[:, h] = _softmax_v(score, s["v_cache"][pages, :, h].flatten(1, 2).float())
    return o.view(seqs, kv_heads, n, group, D).permute(0, 2, 1, 3, 4).reshape(seqs, n, heads, D).to(torch.bfloat16)


def _run_prefill(s):
    c = s["case"]
    if own:
        from vlcache_b200 import ops
        return ops.prefill_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["plan"], s["softmax_scale"])
    heads, kv_heads = c["heads"], c["kv_heads"]
    group = heads // kv_heads
    out = torch.empty_like(s["q"])
    for i in range(len(s["cu_q"]) - 1):
        a, b = s["cu_q"][i], s["cu_q"][i + 1]
        n, m = b - a, s["cu_k"][i + 1] - s["cu_k"][i]
        pages = s["tables"][i, :(m + c["block"] - 1) // c["block"]].long().clamp(min=0)
        key = torch.arange(m, device=out.device)
        at = torch.arange(m - n, m, device=out.device).view(-1, 1)
        seen = key <= at
        if c["window"]:
            seen &= (key > at - c["window"]) | (key < c["sinks"])
        for h in range(kv_heads):
            k = s["k_cache"][pages, :, h].flatten(0, 1)[:m].float()
            v = s["v_cache"][pages, :, h].flatten(0, 1)[:m].float()
            q = s["q"][a:b, h * group:(h + 1) * group].float().transpose(0, 1)
            score = torch.where(seen, (q @ k.T) * s["softmax_scale"], -math.inf)
            out[a:b, h * group:(h + 1) * group] = _softmax_v(score, v).transpose(0, 1).to(torch.bfloat16)
            del score
    return out


def _run_step(s):
    c = s["case"]
    if own:
        from vlcache_b200 import ops
        positions, slots, cu_q, cu_k, lens = ops.step_metadata(
            s["lens"], s["new"], s["block_tables"], s["free_pages"], s["num_free"], c["block"], s["rows"], c["window"],
            c["sinks"])
        return positions, slots, cu_q, cu_k, lens, s["block_tables"], s["free_pages"], s["num_free"]
    block, tables, free = c["block"], s["block_tables"], s["free_pages"]
    before, new = s["lens"].long(), s["new"].long()
    page = torch.arange(tables.shape[1], device=tables.device)
    first, last = (before // block).view(-1, 1), ((before + new - 1) // block).view(-1, 1)
    need = (page >= first) & (page <= last) & (new.view(-1, 1) > 0) & (tables < 0)
    nth = (need.flatten().cumsum(0) - 1).view_as(need)
    count = s["num_free"].long()
    got = need & (nth < count)
    pages = torch.where(got, free[(count - 1 - nth).clamp(0, free.numel() - 1)], tables)
    count = count - got.sum()
    if c["window"]:
        behind = ((before - c["window"] + 1) // block).view(-1, 1)       # (floor: none where it is negative)
        gone = (page >= (c["sinks"] + block - 1) // block) & (page < behind) & (pages >= 0)
        nth = (gone.flatten().cumsum(0) - 1).view_as(gone)
        where = torch.where(gone, count + nth, free.numel()).flatten()   # the others: one past the end
        free.copy_(torch.cat((free, free.new_zeros(1))).scatter(0, where, pages.flatten())[:-1])
        pages = torch.where(gone, -1, pages)
        count = count + gone.sum()
    tables.copy_(pages)
    s["num_free"].copy_(count)
    zero = torch.zeros(1, dtype=torch.int64, device=tables.device)
    cu_q, cu_k = torch.cat((zero, new.cumsum(0))), torch.cat((zero, (before + new).cumsum(0)))
    row = torch.arange(s["rows"], device=tables.device)
    seq = torch.searchsorted(cu_q[1:], row, right=True).clamp(max=c["seqs"] - 1)
    live = row < cu_q[-1]
    positions = torch.where(live, before[seq] + row - cu_q[seq], 0)
    at = pages[seq, (positions // block).clamp(max=tables.shape[1] - 1)].long()
    slots = torch.where(live & (at >= 0), at * block + positions % block, -1)
    return (positions, slots.to(torch.int32), cu_q.to(torch.int32), cu_k.to(torch.int32),
            (before + new).to(torch.int32), tables, free, s["num_free"])


def _run_verify(s):
    if own:
        from vlcache_b200 import ops
        return ops.verify_drafts(s["drafts"], s["p"], s["q"], s["u"], s["u_last"])
    drafts, p = s["drafts"], s["p"]
    seqs, most = drafts.shape
    token = drafts.clamp(min=0).unsqueeze(-1)
    there = p[:, :most].gather(-1, token).squeeze(-1).double()
    chance = s["u"].double()
    if s["q"] is not None:                                               # (the product of two fp32 is exact in 64 bits)
        chance = chance * s["q"].gather(-1, token).squeeze(-1).double()
    taken = ((drafts >= 0) & (chance < there)).long().cumprod(-1).sum(-1)
    row = torch.arange(seqs, device=p.device)
    weight = p[row, taken].float()
    if most:
        stop = taken.clamp(max=most - 1)
        refused = ((taken < most) & (drafts[row, stop] >= 0)).view(-1, 1)
        if s["q"] is not None:
            weight = torch.where(refused, weight - s["q"][row, stop].float(), weight)
        else:
            other = torch.arange(p.shape[-1], device=p.device) != drafts[row, stop].view(-1, 1)
            weight = torch.where(refused & ~other, torch.zeros_like(weight), weight)
    upto = (weight.clamp(0, 1) * COUNT).long().cumsum(-1)
    total = upto[:, -1:]
    u = (s["u_last"].view(-1, 1) * 2.0 ** 24).long()
    goal = u * (total >> 24) + ((u * (total & 0xffffff)) >> 24)
    last = torch.searchsorted(upto, goal, right=True)
    place = torch.arange(most + 1, device=p.device)
    tokens = torch.where(place < taken.view(-1, 1), torch.cat((drafts, last), 1), -1)
    tokens = torch.where(place == taken.view(-1, 1), last, tokens)
    return tokens, (taken + 1).to(torch.int32)


# ------------------------------------------------------------------ what a pass cannot do without
def _seen(n, m, window, sinks):
    """(query, key) pairs that the mask leaves of n rows at the end of m keys, and keys that any row sees."""
    if not window:
        return n * m - n * (n - 1) / 2, m
    pairs = sum(min(t + 1, window) + min(sinks, max(0, t + 1 - window)) for t in range(m - n, m))
    low = max(0, m - n - window + 1)
    return pairs, m - low + min(sinks, low)


def work(case):
    if case["op"] == "verify":
        size = 4 if case["dtype"] == "fp32" else 2
        # one row of p, and where a draft is refused (ACCEPT: the share that is not) one of q
        rows = 1 + (1 - ACCEPT ** case["drafts"] if case["draft_probs"] else 0)
        return {"bytes": case["seqs"] * (rows * case["vocab"] * size + case["drafts"] * (2 * size + 20) + 8),
                "flops": case["seqs"] * case["vocab"] * 3}
    if case["op"] == "step":
        rows, block = case["seqs"] * (case["min_new"] + case["max_new"]) / 2, case["block"]
        entries = rows / block + case["seqs"] * (3 if case["window"] else 1)
        return {"bytes": rows * 12 + case["seqs"] * 20 + entries * 8, "flops": 0}
    heads, kv_heads = case["heads"], case["kv_heads"]
    if case["op"] == "decode":
        m = (case["min_len"] + case["max_len"]) // 2
        pairs, keys = _seen(min(case["rows"], m), m, case["window"], case["sinks"])
        rows = case["rows"]
        return {"bytes": case["seqs"] * (keys * 2 * kv_heads * D * 2 + rows * heads * D * 4),
                "flops": case["seqs"] * 4 * pairs * heads * D}
    new, lens = _lengths(case, 0)
    total = {"bytes": 0, "flops": 0}
    for n, m in zip(new, lens):
        pairs, keys = _seen(n, m, case["window"], case["sinks"])
        total["bytes"] += keys * 2 * kv_heads * D * 2 + n * heads * D * 4
        total["flops"] += 4 * pairs * heads * D
    return total


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"decode": _exact_attention, "prefill": _exact_attention, "step": _exact_step,
            "verify": _exact_verify}[case["op"]](case, seed, s)


def _exact_attention(case, seed, s):
    new, lens = _lengths(case, seed)
    heads, kv_heads, block = case["heads"], case["kv_heads"], case["block"]
    q = s["q"].flatten(0, -3).double()
    out, at = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0
    for i, (n, m) in enumerate(zip(new, lens)):
        t = torch.arange(m - n, m, device="cuda").view(-1, 1)
        j = torch.arange(m, device="cuda").view(1, -1)
        hidden = j > t
        if case["window"]:
            hidden = hidden | ((t - j >= case["window"]) & (j >= case["sinks"]))
        rows = torch.arange(m, device="cuda")
        slot = s["tables"][i].long()[rows // block].clamp(min=0) * block + rows % block
        for h in range(heads):
            k = s["k_cache"].flatten(0, 1)[slot, h * kv_heads // heads].double()
            v = s["v_cache"].flatten(0, 1)[slot, h * kv_heads // heads].double()
            score = (q[at:at + n, h] @ k.T * s["softmax_scale"]).masked_fill_(hidden, -math.inf)
            out[at:at + n, h] = torch.softmax(score, -1) @ v
        at += n
    return out.view(s["q"].shape)


def _exact_step(case, seed, s):
    """The step as a loop over sequences and pages."""
    block, window = case["block"], case["window"]
    tables, free = s["block_tables"].tolist(), s["free_pages"].tolist()
    count, new, before = int(s["num_free"]), s["new"].tolist(), s["lens"].tolist()
    for table, n, b in zip(tables, new, before):
        for p in range(b // block, (b + n - 1) // block + 1 if n > 0 else 0):
            if table[p] < 0 and count > 0:
                count -= 1
                table[p] = free[count]
    if window:
        for table, b in zip(tables, before):
            for p in range(-(-case["sinks"] // block), len(table)):
                if (p + 1) * block <= b - window + 1 and table[p] >= 0:
                    free[count], table[p] = table[p], -1
                    count += 1
    positions, slots, cu_q, cu_k = [], [], [0], [0]
    for table, n, b in zip(tables, new, before):
        positions += range(b, b + n)
        slots += [table[t // block] * block + t % block if table[t // block] >= 0 else -1 for t in range(b, b + n)]
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + b + n)
    spare = s["rows"] - len(positions)
    i32 = dict(dtype=torch.int32, device="cuda")
    return (torch.tensor(positions + [0] * spare, dtype=torch.int64, device="cuda"),
            torch.tensor(slots + [-1] * spare, **i32), torch.tensor(cu_q, **i32), torch.tensor(cu_k, **i32),
            torch.tensor([b + n for b, n in zip(before, new)], **i32), torch.tensor(tables, **i32),
            torch.tensor(free, **i32), torch.tensor([count], **i32))


def _exact_verify(case, seed, s):
    """Request by request; whole counts below 2^53 are exact in 64-bit floating point too."""
    drafts, most = s["drafts"].tolist(), case["drafts"]
    u, u_last = s["u"].tolist(), s["u_last"].tolist()
    tokens, counts = [], []
    for b in range(case["seqs"]):
        kept, last = [], None
        for i, d in enumerate(drafts[b]):
            if d < 0:
                break
            q = 1.0 if s["q"] is None else float(s["q"][b, i, d])
            if u[b][i] * q < float(s["p"][b, i, d]):
                kept.append(d)
                continue
            last = s["p"][b, i].float().clone()
            if s["q"] is None:
                last[d] = 0.0
            else:
                last -= s["q"][b, i].float()
            break
        if last is None:
            last = s["p"][b, len(kept)].float()
        upto = torch.cumsum(torch.floor(last.double().clamp(0.0, 1.0) * COUNT), 0)
        total = int(upto[-1])
        goal = int(math.floor(u_last[b] * 2 ** 24)) * total // 2 ** 24
        kept.append(int((upto <= goal).sum()))
        counts.append(len(kept))
        tokens.append(kept + [-1] * (most + 1 - len(kept)))
    return (torch.tensor(tokens, dtype=torch.int64, device="cuda"),
            torch.tensor(counts, dtype=torch.int32, device="cuda"))
