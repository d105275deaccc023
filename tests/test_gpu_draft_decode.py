"""A decode step with drafted tokens over a windowed cache, on the device: windowed attention (decode and prefill)
against 64 bits, the step's metadata and the verification of drafts against whole numbers."""
import math

import numpy as np
import pytest
import torch

from oracle import draft_decode as oracle

pytestmark = pytest.mark.gpu

D = 128
STEP = 2.0 ** -8   # half a step of bf16, relative


def _ops():
    from vlcache_b200 import ops
    return ops


def _caches(g, pages, block, kv_heads, joined=True):
    both = torch.randn(2, pages, block, kv_heads, D, generator=g, device="cuda").to(torch.bfloat16)
    return (both[0], both[1]) if joined else (both[1].clone(), both[0].clone())


def _tables(g, lens, block, spare=1):
    """Block tables of sequences of these lengths over pages in a random order; (tables, pages)."""
    widths = [(n + block - 1) // block for n in lens]
    pages = sum(widths) + 2
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    out, at = [], 0
    for w in widths:
        out.append(order[at:at + w] + [-1] * (max(widths) + spare - w))
        at += w
    return torch.tensor(out, dtype=torch.int32, device="cuda"), pages


def _release(tables, lens, new, block, window, sinks):
    """Entries of pages that no row sees become -1."""
    for i, (n, m) in enumerate(zip(lens, new)):
        for page in range(tables.shape[1]):
            first, last = page * block, page * block + block - 1
            if window and first >= sinks and last <= n - m - window:
                tables[i, page] = -1


def _spoil(cache, tables, lens, new, window, sinks, value):
    """`value` in every row that no query row sees (free pages, behind the windows, past the ends)."""
    block = cache.shape[1]
    keep = torch.zeros(cache.shape[:2], dtype=torch.bool, device=cache.device)
    for i, (n, m) in enumerate(zip(lens, new)):
        if n == 0:
            continue
        seen = oracle.visible(torch.arange(n - m, n, device=cache.device), n, window, sinks).any(0)
        j = torch.nonzero(seen).flatten()
        keep[tables[i].long()[j // block], j % block] = True
    cache[~keep] = value


def _decode(tables, lens, new, q, k_cache, v_cache, window, sinks, scale, **kw):
    block = k_cache.shape[1]
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return _ops().decode_attention_window(q, k_cache, v_cache, tables, lens_t, kw.pop("bound", max(lens + [1])), scale,
                                          window, sinks, **kw)


def _check_decode(got, tables, lens, n, q, k_cache, v_cache, window, sinks, scale):
    for i, m in enumerate(lens):
        k, v = (oracle.sequence_keys(c, tables[i], m) for c in (k_cache, v_cache))
        pos = torch.arange(m - n, m, device="cuda")
        want, rms = oracle.attention(q[i].double().view(n, -1, D), k, v, pos, window, sinks, scale)
        # P is off by STEP of itself in numerator and denominator alike: STEP * sum p |v - o| <= STEP * rms;
        # the output's rounding is STEP of it; fp32 scores and sums of up to 2^8 natural logs are off by less
        # than 2^-12 of the terms.
        tol = (STEP + 2.0 ** -12) * (rms + want.abs()) + 1e-30
        off = (got[i].double().view(n, -1, D) - want).abs()
        assert bool((off <= tol).all()), (i, m, float((off / tol).max()))


CASES = [
    # heads, kv_heads, tokens, block, window, sinks, lengths
    (16, 2, 1, 256, 1024, 4, [6001]),
    (16, 2, 1, 256, 0, 0, [1, 2, 15, 16, 17, 255, 256, 257, 0, 1000]),
    (28, 4, 1, 64, 100, 4, [1, 50, 100, 101, 104, 105, 164, 300, 999]),
    (28, 4, 5, 256, 512, 4, [5, 4, 1, 0, 511, 512, 513, 516, 517, 2000]),
    (28, 4, 2, 128, 1, 0, [2, 129, 1000]),
    (16, 2, 3, 32, 33, 20, [3, 40, 53, 54, 200, 1000]),
    (8, 8, 8, 256, 300, 300, [8, 299, 300, 301, 600, 601, 1500]),
    (12, 1, 1, 256, 64, 1, [700, 64, 65]),
    (12, 1, 5, 256, 700, 100, [3000, 701, 60]),
    (32, 2, 8, 256, 1000, 4, [5000, 8]),
    (16, 1, 8, 32, 77, 5, [400, 9, 1]),
    (4, 4, 1, 96, 50, 3, [500, 47, 48, 49]),
    (2, 2, 31, 256, 20, 2, [500, 31, 12]),
    (7, 1, 7, 64, 200, 33, [1000, 7, 300]),       # 49 rows: two tiles for four warps
    (28, 4, 3, 256, 128, 0, [900, 3, 130]),       # 21: three tiles
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("joined", [True, False])
def test_decode_window(case, joined):
    heads, kv_heads, n, block, window, sinks, lens = case
    g = torch.Generator(device="cuda").manual_seed(heads * 1000 + n * 100 + window)
    tables, pages = _tables(g, lens, block)
    k_cache, v_cache = _caches(g, pages, block, kv_heads, joined)
    q = (1.5 * torch.randn(len(lens), n, heads, D, generator=g, device="cuda")).to(torch.bfloat16)
    new = [min(n, m) for m in lens]
    _spoil(k_cache, tables, lens, new, window, sinks, math.nan)
    _spoil(v_cache, tables, lens, new, window, sinks, math.inf)
    _release(tables, lens, new, block, window, sinks)
    scale = 1 / math.sqrt(D)
    got = _decode(tables, lens, new, q, k_cache, v_cache, window, sinks, scale)
    assert _ops().device_error() == 0
    _check_decode(got, tables, lens, n, q, k_cache, v_cache, window, sinks, scale)
    again = _decode(tables, lens, new, q, k_cache, v_cache, window, sinks, scale)
    assert torch.equal(got, again)


def test_decode_window_batch():
    """Many pairs: shares that end inside pairs, and whole ones."""
    g = torch.Generator(device="cuda").manual_seed(5)
    lens = [int(x) for x in np.random.default_rng(3).integers(0, 3000, 90)]
    tables, pages = _tables(g, lens, 256)
    k_cache, v_cache = _caches(g, pages, 256, 4)
    for n in (1, 3):
        q = torch.randn(len(lens), n, 28, D, generator=g, device="cuda").to(torch.bfloat16)
        for window, sinks in ((0, 0), (700, 4)):
            got = _decode(tables, lens, None, q, k_cache, v_cache, window, sinks, 0.1)
            _check_decode(got, tables, lens, n, q, k_cache, v_cache, window, sinks, 0.1)
    assert _ops().device_error() == 0


def test_decode_window_without_a_window_is_decode():
    g = torch.Generator(device="cuda").manual_seed(8)
    lens = [1, 300, 2222, 7000]
    tables, pages = _tables(g, lens, 256)
    k_cache, v_cache = _caches(g, pages, 256, 2)
    q = torch.randn(4, 16, D, generator=g, device="cuda").to(torch.bfloat16)
    a = _decode(tables, lens, None, q, k_cache, v_cache, 0, 0, 0.09)
    b = _ops().decode_attention(q, k_cache, v_cache, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), 7000,
                                0.09)
    assert a.shape == b.shape == (4, 16, D)
    _check_decode(a.unsqueeze(1), tables, lens, 1, q.unsqueeze(1), k_cache, v_cache, 0, 0, 0.09)
    assert float((a.float() - b.float()).abs().max()) < 2e-2


PREFILL = [
    # heads, kv_heads, block, window, sinks, [(query rows, keys)]
    (16, 2, 256, 128, 4, [(700, 700)]),
    (16, 2, 256, 1, 0, [(300, 300), (17, 400)]),
    (28, 4, 128, 300, 130, [(1, 1), (600, 900), (0, 0), (33, 1500)]),
    (28, 4, 256, 1000, 4, [(2500, 2500)]),
    (8, 8, 256, 129, 128, [(260, 520), (128, 128)]),
    (12, 1, 256, 77, 1000, [(900, 2000)]),
    (16, 2, 256, 5000, 4, [(500, 700)]),       # a window that hides nothing
    (16, 2, 128, 512, 4, [(48, 9000)]),        # few rows: split and merged
]


@pytest.mark.parametrize("case", PREFILL, ids=lambda c: "-".join(map(str, c[:5])))
@pytest.mark.parametrize("way", ["paged", "inflight", "contiguous"])
def test_prefill_window(case, way):
    ops = _ops()
    heads, kv_heads, block, window, sinks, seqs = case
    g = torch.Generator(device="cuda").manual_seed(heads + window)
    new, lens = [a for a, _ in seqs], [b for _, b in seqs]
    tables, pages = _tables(g, lens, block)
    k_cache, v_cache = _caches(g, pages, block, kv_heads)
    q = (1.5 * torch.randn(sum(new), heads, D, generator=g, device="cuda")).to(torch.bfloat16)
    cu_q, cu_k = np.cumsum([0] + new), np.cumsum([0] + lens)
    _spoil(k_cache, tables, lens, new, window, sinks, math.nan)
    _spoil(v_cache, tables, lens, new, window, sinks, math.inf)
    full = tables.clone()
    _release(tables, lens, new, block, window, sinks)
    plan = ops.build_prefill_plan(cu_q, cu_k, heads, kv_heads, device="cuda", window=window, sinks=sinks)
    scale = 1 / math.sqrt(D)
    rows = [(cache.flatten(0, 1)[full[i].long()[torch.arange(m, device="cuda") // block] * block
                                 + torch.arange(m, device="cuda") % block])
            for cache in (k_cache, v_cache) for i, m in enumerate(lens)]
    k_rows, v_rows = torch.cat(rows[:len(lens)]), torch.cat(rows[len(lens):])
    if way == "contiguous":
        got = ops.prefill_attention(q, k_rows, v_rows, None, plan, scale)
    elif way == "paged":
        got = ops.prefill_attention(q, k_cache, v_cache, tables, plan, scale)
    else:  # the new rows' keys and values as the projection left them
        own = torch.cat([torch.arange(cu_k[i + 1] - n, cu_k[i + 1], device="cuda") for i, n in enumerate(new)])
        got = ops.prefill_attention(q, k_cache, v_cache, tables, plan, scale, k_new=k_rows[own], v_new=v_rows[own])
    assert ops.device_error() == 0
    for i, (n, m) in enumerate(seqs):
        want, rms = oracle.attention(q[cu_q[i]:cu_q[i + 1]].double(), k_rows[cu_k[i]:cu_k[i + 1]].double(),
                                     v_rows[cu_k[i]:cu_k[i + 1]].double(), torch.arange(m - n, m, device="cuda"), window,
                                     sinks, scale)
        # P is off by STEP of itself (sum p |v| <= rms), a split tile's parts by STEP of themselves
        # (again <= rms), the output by STEP of itself.
        tol = (STEP + 2.0 ** -12) * (2 * rms + want.abs()) + 1e-30
        off = (got[cu_q[i]:cu_q[i + 1]].double() - want).abs()
        assert n == 0 or bool((off <= tol).all()), (i, float((off / tol).max()))


def _step_case(r, b, most_new, longest, block, window, sinks, pool=None):
    lens = [int(x) for x in r.integers(0, longest + 1, b)]
    new = [int(x) for x in r.integers(0, most_new + 1, b)]
    if b > 2:
        lens[1] = -1
        new[2] = 0
    width = (longest + most_new) // block + 2
    need = sum((n + block - 1) // block for n in lens if n > 0)
    pool = need + b * (most_new // block + 2) if pool is None else need + pool
    pages = r.permutation(pool + 3).tolist()
    tables = []
    for n in lens:
        held = (max(n, 0) + block - 1) // block
        t = [pages.pop() for _ in range(held)]
        gone = max(0, (n - window + 1) // block - 2) if window else 0
        first = -(-sinks // block)
        for p in range(first, min(gone, held)):   # given back earlier
            pages.append(t[p])
            t[p] = -1
        if held and r.random() < 0.3:              # a page left by refused drafts
            t += [pages.pop()] if pages else []
        tables.append(t + [-1] * (width - len(t)))
    free = pages + [-7] * (sum(map(len, tables)) + 5)
    return lens, new, tables, free, len(pages)


@pytest.mark.parametrize("b,most_new,longest,block,window,sinks", [
    (1, 1, 0, 256, 0, 0), (1, 5, 700, 256, 0, 0), (8, 1, 4000, 256, 1024, 4), (33, 5, 900, 16, 100, 20),
    (70, 9, 3000, 128, 512, 300), (300, 3, 2000, 64, 1, 0), (5, 4000, 100, 256, 0, 0), (17, 700, 2000, 32, 600, 4),
    (129, 40, 0, 7, 3, 0), (1000, 5, 300, 256, 64, 4),
])
def test_step_metadata(b, most_new, longest, block, window, sinks):
    ops = _ops()
    r = np.random.default_rng(b + most_new)
    lens, new, tables, free, count = _step_case(r, b, most_new, longest, block, window, sinks)
    total = sum(max(n, 0) for n, m in zip(new, lens) if m >= 0) + 5
    want = oracle.step(lens, new, tables, free, count, block, total, window, sinks)
    i32 = dict(dtype=torch.int32, device="cuda")
    # a row stride of its own, with guards behind the tables' rows
    wide = torch.full((b, len(tables[0]) + 3), -9, **i32)
    wide[:, :len(tables[0])] = torch.tensor(tables, **i32)
    tables_t, free_t = wide[:, :len(tables[0])], torch.tensor(free, **i32)
    count_t, lens_t, new_t = torch.tensor([count], **i32), torch.tensor(lens, **i32), torch.tensor(new, **i32)
    got = ops.step_metadata(lens_t, new_t, tables_t, free_t, count_t, block, total, window, sinks)
    assert ops.device_error() == 0
    for a, w in zip(got + (tables_t, free_t, count_t), want[:7] + ([want[7]],)):
        assert a.tolist() == w
    assert bool((wide[:, len(tables[0]):] == -9).all()) and lens_t.tolist() == lens
    # the same step again finds its pages in the tables
    twice = ops.step_metadata(lens_t, new_t, tables_t, free_t, count_t, block, total, window, sinks)
    assert all(torch.equal(x, y) for x, y in zip(got, twice)) and int(count_t) == want[7]


def _probabilities(g, b, rows, vocab, dtype, spread=3.0):
    return torch.softmax(spread * torch.randn(b, rows, vocab, generator=g, device="cuda"), -1).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("b,k,vocab", [(1, 4, 1000), (3, 0, 257), (40, 3, 4099), (7, 31, 33), (20, 2, 1), (5, 8, 32003),
                                       (9, 1, 20000)])
@pytest.mark.parametrize("sampled", [True, False])
def test_verify_drafts(dtype, b, k, vocab, sampled):
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(b * 100 + k)
    p = _probabilities(g, b, k + 1, vocab, dtype)
    q = _probabilities(g, b, k, vocab, dtype)
    if k:
        q = (0.8 * p[:, :k].float() + 0.2 * q.float()).to(dtype)
        drafts = torch.multinomial(q.flatten(0, 1).float(), 1, generator=g).view(b, k)
    else:
        drafts = torch.empty(b, 0, dtype=torch.int64, device="cuda")
    for i in range(0, b, 3):
        drafts[i, i % (k + 1):] = -1
    u, u_last = torch.rand(b, k, generator=g, device="cuda"), torch.rand(b, generator=g, device="cuda")
    tokens, emitted = ops.verify_drafts(drafts, p, q if sampled else None, u, u_last)
    assert ops.device_error() == 0
    for i in range(b):
        want = oracle.verify(drafts[i].tolist(), p[i].cpu(), q[i].cpu() if sampled else None, u[i].tolist(),
                             float(u_last[i]))
        assert int(emitted[i]) == len(want) and tokens[i].tolist() == want + [-1] * (k + 1 - len(want))
