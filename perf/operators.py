"""The operators around the paged cache that are measured, with their plain forms.

Five operators, each as a user of the package calls it:
  rope     rotary positions with several axes (time, height, width) of new rows, fused with the
           scatter into the bf16 paged cache;
  store4   the same fused with the quantising scatter into the 4-bit cache, then the dense
           read-back of that cache (the values it stands for);
  attend4  attention over the 4-bit cache, for single tokens (decode) and for prompts (prefill);
  shift4   the move of reused image rows inside the 4-bit cache with the re-rotation of K by the
           position delta, all layers at once, then the read-back;
  pages    copying pages of every layer and rewriting the block tables (fork, compaction).

The 4-bit cache: groups of 16 consecutive dims of a head hold e2m1 codes (two per byte, the even
dim in the low nibble) and one e4m3 scale s; the value is g * s * code with g a power of two per
cache.  s = e4m3(min(max|x / g| / 6, 448)), code = e2m1(x / g / s), both rounded to nearest even;
codes are 0 where s is 0.  A page of one layer's K or V is [kv_heads][block * 64 code bytes, then
block * 8 scale bytes].
"""
import math

import torch

own = False

D = 128            # head size
HALF = D // 2
GROUP = 16         # dims that share a scale
ROW = 72           # bytes of one head's row: 64 of codes, 8 of scales
MAX_POS = 32768
THETA = 1e6
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of a few running requests: latency.
        {"name": "rope_decode_8", "op": "rope", "tokens": 8, "heads": 28, "kv_heads": 4, "sections": "16,24,24",
         "block": 256},
        # All rows of a prompt with a 4K image (20 + 10549 + 48 tokens), 7B shapes: bandwidth.
        {"name": "rope_prompt_4k_image", "op": "rope", "tokens": 10617, "heads": 28, "kv_heads": 4,
         "sections": "16,24,24", "block": 256},
        # One decode step of 64 requests into the 4-bit cache.
        {"name": "store4_decode_64", "op": "store4", "tokens": 64, "heads": 28, "kv_heads": 4, "sections": "16,24,24",
         "block": 256, "k_exp": 0, "v_exp": -3},
        # A whole prompt with a 4K image into the 4-bit cache, 3B shapes.
        {"name": "store4_prompt_4k_image", "op": "store4", "tokens": 10617, "heads": 16, "kv_heads": 2,
         "sections": "16,24,24", "block": 256, "k_exp": 1, "v_exp": -3},
        # One short request alone: the smallest call, latency.
        {"name": "decode4_one_short", "op": "attend4", "mode": "decode", "seqs": 1, "min_len": 700, "max_len": 700,
         "heads": 16, "kv_heads": 2, "block": 256, "k_exp": 0, "v_exp": -3},
        # The 256 concurrent sequences of the decode benchmark, ragged lengths: bandwidth.
        {"name": "decode4_batch_256", "op": "attend4", "mode": "decode", "seqs": 256, "min_len": 2700,
         "max_len": 10700, "heads": 28, "kv_heads": 4, "block": 256, "k_exp": 0, "v_exp": -3},
        # Few rows over a very long axis: the work has to be split and joined.
        {"name": "decode4_two_long", "op": "attend4", "mode": "decode", "seqs": 2, "min_len": 100003,
         "max_len": 131071, "heads": 28, "kv_heads": 4, "block": 256, "k_exp": 1, "v_exp": -2},
        # The warm request of the prefill benchmark: 10 % of a 4K image's rows and the text over all keys.
        {"name": "prefill4_warm_4k_image", "op": "attend4", "mode": "prefill", "seqs": 1, "prefix": 20, "image": 10549,
         "suffix": 48, "recompute": 1055, "heads": 16, "kv_heads": 2, "block": 256, "k_exp": 0, "v_exp": -3},
        # A 1024-token image moved by a few positions in one layer: the smallest move.
        {"name": "shift4_small_image", "op": "shift4", "rows": 922, "layers": 1, "kv_heads": 2, "block": 256,
         "dt": 16, "dh": 16, "dw": 16},
        # A 1080p image's reused rows in all 36 layers.
        {"name": "shift4_1080p_image", "op": "shift4", "rows": 2556, "layers": 36, "kv_heads": 2, "block": 256,
         "dt": 389, "dh": 389, "dw": 389},
        # Three requests fork: the half-filled last page of each is copied before it is written.
        {"name": "pages_fork_3", "op": "pages", "pages": 16, "moves": 3, "layers": 36, "kv_heads": 2, "block": 256,
         "seqs": 4},
        # Compaction of a fragmented pool: pages move to its front and the block tables follow.
        {"name": "pages_compact_48", "op": "pages", "pages": 128, "moves": 48, "layers": 28, "kv_heads": 4,
         "block": 256, "seqs": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads = rng.choice([(28, 4), (16, 2), (16, 2), (28, 4), (32, 8), (8, 8), (12, 1)])
    block = rng.choice([256, 256, 128])
    base = {"heads": heads, "kv_heads": kv_heads, "block": block}
    exps = {"k_exp": rng.randint(-2, 3), "v_exp": rng.randint(-5, 1)}
    sections = rng.choice(["16,24,24", "16,24,24", "24,20,20", "22,21,21", "64", "11,53"])
    op = rng.choice(["rope", "store4", "decode", "decode", "prefill", "shift4", "pages"])
    if op == "rope":
        return {"op": "rope", "tokens": _log(rng, 1, 9000), "sections": sections, **base}
    if op == "store4":
        return {"op": "store4", "tokens": _log(rng, 1, 9000), "sections": sections, **base, **exps}
    if op == "decode":
        seqs = _log(rng, 1, 200)
        longest = _log(rng, 1, min(131072, 3000000 // (seqs * kv_heads)))
        return {"op": "attend4", "mode": "decode", "seqs": seqs, "min_len": max(0, longest - _log(rng, 1, longest + 1)),
                "max_len": longest, **base, **exps}
    if op == "prefill":
        image = _log(rng, 1, 6000)
        return {"op": "attend4", "mode": "prefill", "seqs": rng.randint(1, 3), "prefix": _log(rng, 1, 300),
                "image": image, "suffix": _log(rng, 1, 200), "recompute": rng.randint(0, max(1, image // 8)),
                **base, **exps}
    if op == "shift4":
        return {"op": "shift4", "rows": _log(rng, 1, 2500), "layers": rng.choice([1, 4, 28]), "kv_heads": min(kv_heads, 2),
                "block": block, "dt": rng.choice([0, 1]) * rng.randint(-900, 900), "dh": rng.randint(-900, 900),
                "dw": rng.randint(-900, 900)}
    pages = rng.randint(8, 120)
    return {"op": "pages", "pages": pages, "moves": rng.randint(1, pages // 3), "layers": rng.choice([1, 28, 36]),
            "kv_heads": rng.choice([1, 2]), "block": block, "seqs": rng.randint(1, 6)}


# ------------------------------------------------------------------ the 4-bit form, in elementary operations
def _views(cache):
    """Codes [.., block, 64] and scales [.., block, 8] of pages [.., block * 72]."""
    block = cache.shape[-1] // ROW
    return cache[..., :block * 64].unflatten(-1, (block, 64)), cache[..., block * 64:].unflatten(-1, (block, 8))


def _quantise(x):
    """fp32 rows [.., 128] (already divided by g): packed codes [.., 64] and scale bytes [.., 8]."""
    x = x.unflatten(-1, (D // GROUP, GROUP))
    s8 = (x.abs().amax(-1) / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = s8.float().unsqueeze(-1)
    a = torch.where(s == 0, torch.zeros_like(x), x / s)
    m = a.abs()
    # ties go to the even code: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75).to(torch.uint8) + (m > 1.25).to(torch.uint8)
            + (m >= 1.75).to(torch.uint8) + (m > 2.5).to(torch.uint8) + (m >= 3.5).to(torch.uint8)
            + (m > 5.0).to(torch.uint8))
    code = (code + (a < 0).to(torch.uint8) * 8).flatten(-2)
    return code[..., 0::2] + code[..., 1::2] * 16, s8.view(torch.uint8)


def _dequantise(codes, scales, table):
    """fp32 values [.., 128] (without g) of codes [.., 64] and scale bytes [.., 8]; table: [256, 2]."""
    v = table[codes.int()].flatten(-2).unflatten(-1, (D // GROUP, GROUP))
    return (v * scales.view(torch.float8_e4m3fn).float().unsqueeze(-1)).flatten(-2)


def _code_table(device):
    one = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=device)
    byte = torch.arange(256, device=device)
    return torch.stack((one[byte % 16], one[byte // 16]), -1)


def _rotate(x, cos, sin):
    """Rotate-half pairs (j, j + 64) of fp32 rows; each product and sum is rounded on its own."""
    a, b = x[..., :HALF], x[..., HALF:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _rope_plain(x, s):
    pair = torch.arange(HALF, device=x.device)
    pos = s["positions"][s["axis"]].T                                   # [N, 64]: each pair's own axis
    cos, sin = s["table"][pos, pair], s["table"][pos, pair + HALF]
    return _rotate(x.float(), cos.unsqueeze(1), sin.unsqueeze(1)).to(torch.bfloat16)


# ------------------------------------------------------------------ inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _cache4(g, pages, kv_heads, block, exp):
    """Pages filled with quantised rows, made in pieces."""
    cache = torch.empty(pages, kv_heads, block * ROW, dtype=torch.uint8, device="cuda")
    codes, scales = _views(cache)
    size = torch.exp(0.5 * _normal(g, D))
    step = max(1, (1 << 20) // (kv_heads * block))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        codes[p:p + n], scales[p:p + n] = _quantise(_normal(g, n, kv_heads, block, D) * size * 2.0 ** -exp)
    return cache


def _rope_table():
    freq = 1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D))
    angle = torch.outer(torch.arange(MAX_POS, dtype=torch.float32, device="cuda"), freq)
    return torch.cat((angle.cos(), angle.sin()), -1)


def _permutation(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "op": case["op"], "code_table": _code_table("cuda")}
    block, kv_heads = case["block"], case["kv_heads"]
    if case["op"] in ("rope", "store4"):
        n, heads = case["tokens"], case["heads"]
        sections = [int(x) for x in case["sections"].split(",")]
        s["sections"] = tuple(sections)
        s["axis"] = torch.repeat_interleave(torch.arange(len(sections), device="cuda"),
                                            torch.tensor(sections, device="cuda"), output_size=HALF)
        s["positions"] = torch.randint(0, MAX_POS, (len(sections), n), generator=g, device="cuda")
        s["table"] = _rope_table()
        qkv = (_normal(g, n, heads + 2 * kv_heads, D) * torch.exp(0.5 * _normal(g, D))).to(torch.bfloat16).flatten(1)
        s["q"] = qkv[:, :heads * D].view(n, heads, D)                    # views of the projection's rows
        s["k"] = qkv[:, heads * D:(heads + kv_heads) * D].view(n, kv_heads, D)
        s["v"] = qkv[:, (heads + kv_heads) * D:].view(n, kv_heads, D)
        pages = (n + block - 1) // block + 1
        s["slots"] = _permutation(g, pages * block)[:n].to(torch.int32)
        if case["op"] == "rope":
            s["k_cache"] = _normal(g, pages, block, kv_heads, D).to(torch.bfloat16)
            s["v_cache"] = _normal(g, pages, block, kv_heads, D).to(torch.bfloat16)
        else:
            s["k_scale"], s["v_scale"] = 2.0 ** case["k_exp"], 2.0 ** case["v_exp"]
            s["k_cache"] = _cache4(g, pages, kv_heads, block, case["k_exp"])
            s["v_cache"] = _cache4(g, pages, kv_heads, block, case["v_exp"])
            s["tables"] = _permutation(g, pages).to(torch.int32).view(1, pages)
            s["total"] = pages * block
            s["cu_k"] = torch.tensor([0, s["total"]], dtype=torch.int32, device="cuda")
    elif case["op"] == "attend4":
        s["k_scale"], s["v_scale"] = 2.0 ** case["k_exp"], 2.0 ** case["v_exp"]
        s["softmax_scale"] = 1.0 / math.sqrt(D)
        heads = case["heads"]
        q_lens, k_lens, shared = _lengths(case, seed)
        tables, at = [], 0
        for i, n in enumerate(k_lens):
            width = max(1, (n + block - 1) // block)
            tables.append(list(range(at, at + width)))
            if not shared or i % 2:                                      # the first part of a warm request reads the
                at += width                                              # front of the second part's pages
        pages = at + 2
        order = _permutation(g, pages)
        w = max(len(t) for t in tables)
        padded = torch.tensor([t + [-1] * (w - len(t)) for t in tables], device="cuda")
        s["tables"] = torch.where(padded >= 0, order[padded.clamp(min=0)], padded).to(torch.int32)
        s["lens"] = torch.tensor(k_lens, dtype=torch.int32, device="cuda")
        s["k_cache"] = _cache4(g, pages, kv_heads, block, case["k_exp"])
        s["v_cache"] = _cache4(g, pages, kv_heads, block, case["v_exp"])
        s["max_len"] = w * block
        if case["mode"] == "decode":
            s["q"] = (2.0 * _normal(g, len(k_lens), heads, D)).to(torch.bfloat16)
        else:
            cu_q, cu_k = [0], [0]
            for a, b in zip(q_lens, k_lens):
                cu_q.append(cu_q[-1] + a)
                cu_k.append(cu_k[-1] + b)
            s["q"] = (2.0 * _normal(g, cu_q[-1], heads, D)).to(torch.bfloat16)
            s["max_q"] = max(q_lens)
            s["cu_q"] = torch.tensor(cu_q, dtype=torch.int32, device="cuda")
            s["cu_k"] = torch.tensor(cu_k, dtype=torch.int32, device="cuda")
            if own:  # the plan of the step, which every layer of it shares
                from vlcache_b200 import ops
                s["plan"] = ops.build_prefill_plan(cu_q, cu_k, heads, kv_heads, device="cuda")
    elif case["op"] == "shift4":
        rows, layers = case["rows"], case["layers"]
        half = (rows + block - 1) // block + 1
        cache = _cache4(g, 2 * layers * 2 * half, kv_heads, block, 0)
        s["cache"] = cache.view(2, layers, 2 * half, kv_heads, block * ROW)
        order = _permutation(g, 2 * half)
        row = torch.arange(rows, device="cuda")
        old = row + 37 % block                                           # the image starts inside a page
        s["src"] = (order[old // block] * block + old % block).to(torch.int32)
        s["dst"] = (order[half + row // block] * block + row % block).to(torch.int32)
        s["tables"] = order[half:half + (rows + block - 1) // block].to(torch.int32).view(1, -1)
        s["total"] = rows
        s["cu_k"] = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        s["delta"] = (case["dt"], case["dh"], case["dw"])
        s["cos"], s["sin"], s["moves"] = _delta_tables(s["delta"])
    else:
        pages, layers = case["pages"], case["layers"]
        s["cache"] = torch.empty(2, layers, pages, block, kv_heads, D, dtype=torch.bfloat16, device="cuda")
        s["cache"].normal_(generator=g)
        order = _permutation(g, pages)
        m = case["moves"]
        s["src"], s["dst"] = order[:m].to(torch.int32), order[m:2 * m].to(torch.int32)
        s["map"] = torch.arange(pages, dtype=torch.int32, device="cuda")
        s["map"][s["src"].long()] = s["dst"]
        live = torch.cat((order[:m], order[2 * m:]))                     # the pages in use before the moves
        s["tables"] = live[torch.randint(0, live.numel(), (case["seqs"], 11), generator=g, device="cuda")].to(torch.int32)
        s["tables"][:, 9:] = -1
    return s


def _lengths(case, seed):
    """(query lengths, key lengths, whether sequences come in pairs that share pages)."""
    import random
    r = random.Random(seed)
    if case["mode"] == "decode":
        k = [r.randint(case["min_len"], case["max_len"]) for _ in range(case["seqs"])]
        return [1] * len(k), k, False
    q, k = [], []
    for _ in range(case["seqs"]):
        a, n = case["prefix"] + case["recompute"], case["prefix"] + case["image"] + case["suffix"]
        q += [a, case["suffix"]]
        k += [a, n]
    return q, k, True


def _delta_tables(delta):
    """cos, sin [64] of each pair's rotation (sections 16, 24, 24) and whether its group of 16 pairs moves."""
    a = torch.tensor([float(delta[0])] * 16 + [float(delta[1])] * 24 + [float(delta[2])] * 24, dtype=torch.float64)
    p = (torch.tensor(THETA, dtype=torch.float64) ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).float()
    a = a * (1.0 / p).double()
    moves = (a != 0).view(4, GROUP).any(-1)
    return a.cos().float().cuda(), a.sin().float().cuda(), moves.repeat(2).cuda()


# ------------------------------------------------------------------ one pass
def run(s):
    if s["op"] == "rope":
        return _run_rope(s)
    if s["op"] == "store4":
        return _run_store4(s)
    if s["op"] == "attend4":
        return _run_attend4(s)
    if s["op"] == "shift4":
        return _run_shift4(s)
    return _run_pages(s)


def _run_rope(s):
    if own:
        from vlcache_b200 import ops
        q = ops.mrope_store_kvcache(s["positions"], s["q"], s["k"], s["v"], s["table"], s["k_cache"], s["v_cache"],
                                    s["slots"], s["sections"])
        return q, s["k_cache"], s["v_cache"]
    slots = s["slots"].long()
    s["k_cache"].flatten(0, 1)[slots] = _rope_plain(s["k"], s)
    s["v_cache"].flatten(0, 1)[slots] = s["v"]
    return _rope_plain(s["q"], s), s["k_cache"], s["v_cache"]


def _read_back(cache, s, scale):
    """Rows [.., total, kv_heads, 128] of the one sequence of `tables`, as bf16 values."""
    pages = cache[..., s["tables"][0].long(), :, :]
    v = (_dequantise(*_views(pages), s["code_table"]) * scale).to(torch.bfloat16)
    return v.transpose(-3, -2).flatten(-4, -3)[..., :s["total"], :, :]


def _run_store4(s):
    if own:
        from vlcache_b200 import ops
        q = ops.rope_store_kvcache_fp4(s["positions"], s["q"], s["k"], s["v"], s["table"], s["k_cache"], s["v_cache"],
                                       s["slots"], s["sections"], s["k_scale"], s["v_scale"])
        k, v = ops.gather_kvcache_fp4(s["k_cache"], s["v_cache"], s["tables"], s["cu_k"], s["total"], s["k_scale"],
                                      s["v_scale"])
        return q, k, v
    slots, block = s["slots"].long(), s["case"]["block"]
    page, row = slots // block, slots % block
    codes, scales = _views(s["k_cache"])
    codes[page, :, row], scales[page, :, row] = _quantise(_rope_plain(s["k"], s).float() / s["k_scale"])
    codes, scales = _views(s["v_cache"])
    codes[page, :, row], scales[page, :, row] = _quantise(s["v"].float() / s["v_scale"])
    return _rope_plain(s["q"], s), _read_back(s["k_cache"], s, s["k_scale"]), _read_back(s["v_cache"], s, s["v_scale"])


def _run_attend4(s):
    decode = s["case"]["mode"] == "decode"
    if own:
        from vlcache_b200 import ops
        if decode:
            return ops.decode_attention_fp4(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["max_len"],
                                            s["softmax_scale"], s["k_scale"], s["v_scale"])
        return ops.prefill_attention_fp4(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["cu_k"], s["plan"],
                                         s["softmax_scale"], s["k_scale"], s["v_scale"])
    q, heads, kv_heads, block = s["q"].float(), s["case"]["heads"], s["case"]["kv_heads"], s["case"]["block"]
    tables, lens = s["tables"].long().clamp(min=0), s["lens"].long()
    seqs, width = tables.shape
    key = torch.arange(width * block, device=q.device).view(1, width, 1, 1, block)
    k = _dequantise(*_views(s["k_cache"][tables]), s["code_table"])      # [seqs, width, kv_heads, block, 128]
    if decode:
        rows = q.view(seqs, 1, kv_heads, heads // kv_heads, D)
        last = (lens - 1).view(seqs, 1, 1, 1, 1)                         # the last key that the row sees
    else:
        token = torch.arange(q.shape[0], device=q.device)
        seq = torch.searchsorted(s["cu_q"][1:].long(), token, right=True)
        i = token - s["cu_q"].long()[seq]
        rows = torch.zeros(seqs, s["max_q"], heads, D, device=q.device)
        rows[seq, i] = q
        rows = rows.view(seqs, s["max_q"], kv_heads, heads // kv_heads, D).transpose(1, 2).flatten(2, 3).unsqueeze(1)
        q_lens = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
        at = torch.arange(s["max_q"], device=q.device).repeat_interleave(heads // kv_heads)
        last = ((lens - q_lens).view(seqs, 1) + at).view(seqs, 1, 1, -1, 1)
    score = (rows @ k.transpose(-1, -2)) * (s["softmax_scale"] * s["k_scale"])
    del k
    score = torch.where(key <= torch.minimum(last, lens.view(seqs, 1, 1, 1, 1) - 1), score, -math.inf)
    top = score.amax((1, 4), keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum((1, 4))
    v = _dequantise(*_views(s["v_cache"][tables]), s["code_table"]) * s["v_scale"]
    o = (p @ v).sum(1) / torch.where(total == 0, torch.ones_like(total), total).unsqueeze(-1)
    if decode:
        return o.view(seqs, heads, D).to(torch.bfloat16)
    o = o.view(seqs, kv_heads, s["max_q"], heads // kv_heads, D).transpose(1, 2).flatten(2, 3)
    return o[seq, i].to(torch.bfloat16)


def _run_shift4(s):
    cache = s["cache"]
    if own:
        from vlcache_b200 import ops
        ops.mrope_shift_fp4(cache, s["src"], s["dst"], s["delta"], rope_theta=THETA)
        return ops.gather_kvcache_fp4(cache[0], cache[1], s["tables"], s["cu_k"], s["total"])
    block = s["case"]["block"]
    src, dst = s["src"].long(), s["dst"].long()
    codes, scales = _views(cache)                                        # [2, layers, pages, kv_heads, block, ..]
    c, f = codes[:, :, src // block, :, src % block], scales[:, :, src // block, :, src % block]
    c, f = c.clone(), f.clone()                                          # [rows, 2, layers, kv_heads, ..]
    x = _rotate(_dequantise(c[:, 0], f[:, 0], s["code_table"]), s["cos"], s["sin"]).to(torch.bfloat16).float()
    new_c, new_f = _quantise(x)
    # a group whose pairs all stay keeps its bits
    c[:, 0] = torch.where(s["moves"].repeat_interleave(GROUP // 2), new_c, c[:, 0])
    f[:, 0] = torch.where(s["moves"], new_f, f[:, 0])
    codes[:, :, dst // block, :, dst % block], scales[:, :, dst // block, :, dst % block] = c, f
    return _read_back(cache[0], s, 1.0), _read_back(cache[1], s, 1.0)


def _run_pages(s):
    if own:
        from vlcache_b200 import ops
        ops.copy_kv_pages(s["cache"], s["src"], s["dst"])
        ops.remap_block_tables(s["tables"], s["map"])
        return s["cache"], s["tables"]
    s["cache"][:, :, s["dst"].long()] = s["cache"][:, :, s["src"].long()]
    s["tables"].copy_(torch.where(s["tables"] >= 0, s["map"][s["tables"].clamp(min=0).long()], s["tables"]))
    return s["cache"], s["tables"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    block, kv_heads = case["block"], case["kv_heads"]
    if case["op"] in ("rope", "store4"):
        n, heads = case["tokens"], case["heads"]
        axes = len(case["sections"].split(","))
        table = min(n, MAX_POS) * D * 4
        read = n * ((heads + 2 * kv_heads) * D * 2 + 8 * axes + 4) + table
        flops = n * (heads + kv_heads) * HALF * 6
        if case["op"] == "rope":
            return {"bytes": read + n * (heads + 2 * kv_heads) * D * 2, "flops": flops}
        total = ((n + block - 1) // block + 1) * block
        write = n * (heads * D * 2 + 2 * kv_heads * ROW)
        return {"bytes": read + write + total * 2 * kv_heads * (ROW + D * 2), "flops": flops + 4 * n * 2 * kv_heads * D}
    if case["op"] == "attend4":
        heads = case["heads"]
        if case["mode"] == "decode":
            keys = case["seqs"] * (case["min_len"] + case["max_len"]) / 2
            return {"bytes": keys * 2 * kv_heads * ROW + case["seqs"] * heads * D * 4, "flops": 4 * keys * heads * D}
        a, n = case["prefix"] + case["recompute"], case["prefix"] + case["image"] + case["suffix"]
        u = case["suffix"]
        seen = a * (a + 1) / 2 + u * n - u * (u - 1) / 2
        return {"bytes": case["seqs"] * ((a + u) * heads * D * 4 + n * 2 * kv_heads * ROW),
                "flops": case["seqs"] * 4 * seen * heads * D}
    if case["op"] == "shift4":
        rows = case["rows"] * case["layers"] * kv_heads
        return {"bytes": rows * 2 * (2 * ROW + ROW + D * 2) + case["rows"] * 8, "flops": rows * HALF * 6}
    return {"bytes": case["moves"] * 2 * case["layers"] * block * kv_heads * D * 2 * 2 + case["seqs"] * 11 * 8, "flops": 0}


# ------------------------------------------------------------------ the definitions, in 64 bits
def _exact_values(cache):
    """64-bit values [.., block, 128] of pages, one nibble and one scale field at a time."""
    codes, scales = _views(cache)
    nibble = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int64)
    e, m = (nibble >> 1) & 3, (nibble & 1).double()
    mag = torch.where(e == 0, 0.5 * m, torch.exp2((e - 1).double()) * (1 + 0.5 * m))
    mag = torch.where(nibble >= 8, -mag, mag)
    b = scales.to(torch.int64)
    e, m = (b >> 3) & 15, (b & 7).double()
    s = torch.where(e == 0, m / 8 * 2.0 ** -6, torch.exp2((e - 7).double()) * (1 + m / 8))
    return mag * s.repeat_interleave(GROUP, -1)


def _exact_quantised(x):
    """The values that rows x (64 bits, divided by g) are held as."""
    x = x.unflatten(-1, (D // GROUP, GROUP))
    t = (x.abs().amax(-1, keepdim=True) / 6).clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)  # spacing of e4m3 around t
    s = torch.round(t / step) * step                                     # round() takes ties to even
    y = torch.where(s > 0, x.abs() / torch.where(s > 0, s, 1.0), 0.0)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))         # spacing of e2m1 around y
    y = torch.clamp(torch.round(y / step) * step, max=6.0)
    return (torch.sign(x) * y * s).flatten(-2)


def _exact_rope(x, s):
    x, out = x.double(), torch.empty(x.shape, dtype=torch.float64, device=x.device)
    start = 0
    for axis, n in enumerate(s["sections"]):
        row = s["table"].double()[s["positions"][axis]].unsqueeze(1)
        lo, hi = slice(start, start + n), slice(HALF + start, HALF + start + n)
        out[..., lo] = x[..., lo] * row[..., lo] - x[..., hi] * row[..., hi]
        out[..., hi] = x[..., hi] * row[..., lo] + x[..., lo] * row[..., hi]
        start += n
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    block, kv_heads = case["block"], case["kv_heads"]
    if case["op"] == "rope":
        k, v = s["k_cache"].double().flatten(0, 1), s["v_cache"].double().flatten(0, 1)
        k[s["slots"].long()], v[s["slots"].long()] = _exact_rope(s["k"], s), s["v"].double()
        shape = s["k_cache"].shape
        return _exact_rope(s["q"], s), k.view(shape), v.view(shape)
    if case["op"] == "store4":
        outs = []
        for cache, x, g in ((s["k_cache"], _exact_rope(s["k"], s).to(torch.bfloat16).double(), s["k_scale"]),
                            (s["v_cache"], s["v"].double(), s["v_scale"])):
            rows = _exact_values(cache).transpose(1, 2).flatten(0, 1)    # [slots, kv_heads, 128]
            rows[s["slots"].long()] = _exact_quantised(x / g)            # a key is held in bf16 before it is quantised
            outs.append((rows.unflatten(0, (-1, block))[s["tables"][0].long()].flatten(0, 1)) * g)
        return _exact_rope(s["q"], s), outs[0], outs[1]
    if case["op"] == "attend4":
        heads = case["heads"]
        q_lens, k_lens, _ = _lengths(case, seed)
        if sum(a * b for a, b in zip(q_lens, k_lens)) * heads > 4e9:
            return None
        outs, at = [], 0
        for i, (a, n) in enumerate(zip(q_lens, k_lens)):
            pages = s["tables"][i][:max(1, (n + block - 1) // block)].long()
            k = (_exact_values(s["k_cache"][pages]) * s["k_scale"]).transpose(0, 1).flatten(1, 2)[:, :n]
            v = (_exact_values(s["v_cache"][pages]) * s["v_scale"]).transpose(0, 1).flatten(1, 2)[:, :n]
            q = s["q"][at:at + a].double().view(a, kv_heads, -1, D).permute(1, 2, 0, 3)
            score = q @ k.unsqueeze(1).transpose(-1, -2) * s["softmax_scale"]
            seen = torch.arange(n, device="cuda") <= torch.arange(n - a, n, device="cuda").view(-1, 1)
            p = torch.softmax(score.masked_fill(~seen, -math.inf), -1) if n else score
            outs.append((torch.nan_to_num(p) @ v.unsqueeze(1)).permute(2, 0, 1, 3).reshape(a, heads, D))
            at += a
        return torch.cat(outs)
    if case["op"] == "shift4":
        src, dst = s["src"].long(), s["dst"].long()
        outs = []
        for which in (0, 1):
            rows = _exact_values(s["cache"][which]).transpose(2, 3).flatten(1, 2)  # [layers, slots, kv_heads, 128]
            x = rows[:, src]
            if which == 0:
                a, b = x[..., :HALF], x[..., HALF:]
                cos, sin = s["cos"].double(), s["sin"].double()
                y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(torch.bfloat16).double()
                x = torch.where(s["moves"].repeat_interleave(GROUP), _exact_quantised(y), x)
            rows[:, dst] = x
            pages = rows.unflatten(1, (-1, block))[:, s["tables"][0].long()]
            outs.append(pages.flatten(1, 2)[:, :s["total"]])
        return outs[0], outs[1]
    return None
