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


def _check_decode(got, tables, lens, n, q, k_cache, v_cache, window, sinks, scale, scores=0.0):
    for i, m in enumerate(lens):
        k, v = (oracle.sequence_keys(c, tables[i], m) for c in (k_cache, v_cache))
        pos = torch.arange(m - n, m, device="cuda")
        want, rms = oracle.attention(q[i].double().view(n, -1, D), k, v, pos, window, sinks, scale)
        # P is off by STEP of itself in numerator and denominator alike: STEP * sum p |v - o| <= STEP * rms;
        # the output's rounding is STEP of it; fp32 scores and sums of up to 2^8 natural logs are off by less
        # than 2^-12 of the terms.  `scores`: what scores are off by beyond that, and so the logarithms of P.
        tol = (STEP + 2.0 ** -12) * (rms + want.abs()) + 2 * math.expm1(scores) * rms + 1e-30
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
    total = sum(new) + 5
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


# ------------------------------------------------------------------ decode: what a call may bring
def _small(seed=1, lens=(200, 70, 333), n=2, heads=16, kv_heads=2, block=64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = list(lens)
    tables, pages = _tables(g, lens, block)
    k_cache, v_cache = _caches(g, pages, block, kv_heads)
    q = torch.randn(len(lens), n, heads, D, generator=g, device="cuda").to(torch.bfloat16)
    return g, lens, tables, k_cache, v_cache, q


@pytest.mark.parametrize("lens", [(200, 70, 333), (9000,) * 40])   # clusters, and the line of chunks
def test_decode_window_strides_out_and_workspace(lens):
    g, lens, tables, k_cache, v_cache, q = _small(lens=lens)
    b, n, heads, _ = q.shape
    want = _decode(tables, lens, None, q, k_cache, v_cache, 50, 3, 0.1)
    rows = torch.full((b * n, 20 * D), math.nan, dtype=torch.bfloat16, device="cuda")   # a projection's rows
    view = rows[:, :heads * D].view(b, n, heads, D)
    view.copy_(q)
    into = torch.full((b * n + 1, heads + 1, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = into[:b * n, :heads].view(b, n, heads, D)
    need = _ops().decode_window_workspace_bytes(b, n, heads, 2, max(lens), 50, 3)
    wide = torch.full((b, tables.shape[1] + 5), -3, dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = tables
    got = _decode(wide[:, :tables.shape[1]], lens, None, view, k_cache, v_cache, 50, 3, 0.1, out=out,
                  workspace=torch.empty(need + 16, dtype=torch.uint8, device="cuda"))
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
    assert bool((into[b * n:] == 7).all()) and bool((into[:, heads:] == 7).all())   # rows behind stay as they were
    three = _decode(tables, lens, None, q[:, 1].contiguous(), k_cache, v_cache, 50, 3, 0.1)
    assert three.shape == (b, heads, D)
    _check_decode(three.unsqueeze(1), tables, lens, 1, q[:, 1:].contiguous(), k_cache, v_cache, 50, 3, 0.1)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = _decode(tables, lens, None, q, k_cache, v_cache, 50, 3, 0.1)
    other.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [0.3, -0.3, 0.0])
def test_decode_window_scales_and_broken_queries(scale):
    g, lens, tables, k_cache, v_cache, q = _small()
    q[0, 1, 3, 5], q[1, 0, 0, 0], q[2, 1, 15, 127] = math.inf, math.nan, -math.inf
    got = _decode(tables, lens, None, q, k_cache, v_cache, 40, 0, scale)
    broken = ~torch.isfinite(q).all(-1)
    assert int(broken.sum()) == 3 and bool(torch.isnan(got[broken]).all()) and bool(torch.isfinite(got[~broken]).all())
    clean = torch.where(broken.unsqueeze(-1), torch.zeros_like(q), q)
    got = torch.where(broken.unsqueeze(-1), _decode(tables, lens, None, clean, k_cache, v_cache, 40, 0, scale), got)
    _check_decode(got, tables, lens, 2, clean, k_cache, v_cache, 40, 0, scale)


def test_decode_window_large_scores():
    """Scores that rise by some 2 a key to well over a thousand: the maximum keeps moving."""
    g, lens, tables, k_cache, v_cache, q = _small(lens=(700,))
    for j in range(700):
        k_cache[tables[0, j // 64], j % 64] = q[0, 0, 0] * (j / 64)
    got = _decode(tables, lens, None, q, k_cache, v_cache, 0, 0, 1.0)
    # A score is a sum of 128 products in fp32, each sum off by 2^-24 of sum |q k| at most, then scaled in two
    # roundings: 130 steps of it.
    most = float(q[0].double().abs().sum(-1).max() * k_cache.double().abs().max())
    most = min(most, float((q[0].double().abs() @ (q[0, 0, 0].double().abs() * 11)).max()) * 1.01)
    _check_decode(got, tables, lens, 2, q, k_cache, v_cache, 0, 0, 1.0, scores=130 * 2.0 ** -24 * most)


@pytest.mark.parametrize("lens", [(200, 70, 333), (9000,) * 40])
def test_decode_window_bad_pages_and_lengths(lens):
    ops = _ops()
    g, lens, tables, k_cache, v_cache, q = _small(lens=lens)
    pages = k_cache.shape[0]
    for bad in (-1, pages, 1 << 30, -(1 << 31)):
        broken = tables.clone()
        broken[1, 0] = bad
        got = _decode(broken, lens, None, q, k_cache, v_cache, 0, 0, 0.1)
        assert ops.device_error() == 102
        keys = k_cache.clone(), v_cache.clone()   # its keys count as zeros
        for c in keys:
            c[tables[1, 0].long()] = 0
        _check_decode(got, tables, lens, 2, q, *keys, 0, 0, 0.1)
    # a table too narrow for the length: the same
    narrow = tables[:, :1].contiguous()
    got = _decode(narrow, lens, None, q, k_cache, v_cache, 0, 0, 0.1)
    assert ops.device_error() == 102 and bool(torch.isfinite(got).all())
    # a length past the host's bound is cut to it
    got = _decode(tables, lens, None, q, k_cache, v_cache, 30, 2, 0.1, bound=100)
    assert ops.device_error() == 104
    cut = [min(n, 100) for n in lens]
    _check_decode(got, tables, cut, 2, q, k_cache, v_cache, 30, 2, 0.1)
    lens_t = torch.tensor([-5] + lens[1:], dtype=torch.int32, device="cuda")
    got = ops.decode_attention_window(q, k_cache, v_cache, tables, lens_t, max(lens), 0.1)
    assert ops.device_error() == 0 and bool((got[0] == 0).all())


def test_decode_window_no_sequences():
    _, _, tables, k_cache, v_cache, q = _small()
    got = _decode(tables[:0], [], None, q[:0], k_cache, v_cache, 8, 0, 0.1)
    assert got.shape == (0, 2, 16, D)


@pytest.mark.parametrize("lens", [(200, 70, 333), (6000,) * 40])
def test_decode_window_captured(lens):
    """Two graphs of their own workspaces, replayed in turn and at once, follow lengths and tables that change."""
    g, lens, tables, k_cache, v_cache, q = _small(lens=lens)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs, graphs, outs = [q, q.flip(0).contiguous()], [], []
    for x in qs:
        _ops().decode_attention_window(x, k_cache, v_cache, tables, lens_t, max(lens), 0.1, 60, 4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_ops().decode_attention_window(x, k_cache, v_cache, tables, lens_t, max(lens), 0.1, 60, 4))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for cut in (0, 3, 64):
        lens_t.copy_(torch.tensor([max(0, n - cut) for n in lens], dtype=torch.int32))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for x, out in zip(qs, outs):
            _check_decode(out, tables, [max(0, n - cut) for n in lens][:3], 2, x, k_cache, v_cache, 60, 4, 0.1)
    assert _ops().device_error() == 0


def test_decode_window_pages_beyond_4_gb():
    """Pages whose byte offset passes 32 bits, the caches in either order."""
    g = torch.Generator(device="cuda").manual_seed(3)
    pages, block, kv_heads = 9000, 256, 4
    both = torch.empty(2, pages, block, kv_heads, D, dtype=torch.bfloat16, device="cuda")
    both[:, -4:].normal_(generator=g)
    tables = torch.tensor([[pages - 1, pages - 3], [pages - 2, pages - 4]], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 1, 28, D, generator=g, device="cuda").to(torch.bfloat16)
    for k_cache, v_cache in ((both[0], both[1]), (both[1], both[0])):
        got = _decode(tables, [400, 512], None, q, k_cache, v_cache, 300, 4, 0.1)
        _check_decode(got, tables, [400, 512], 1, q, k_cache, v_cache, 300, 4, 0.1)


# ------------------------------------------------------------------ step: what goes wrong
def test_step_metadata_without_room():
    ops = _ops()
    i32 = dict(dtype=torch.int32, device="cuda")

    def step(lens, new, tables, free, count, total, **kw):
        a = [torch.tensor(x, **i32) for x in (lens, new, tables, free, [count])]
        return ops.step_metadata(*a, 4, total, **kw), a
    # two pages for three that are missing: the last sequence's slots are -1
    got, a = step([3, 0], [2, 5], [[5, -1], [-1, -1]], [9, 8, 7], 2, 7)
    assert ops.device_error() == 105 and got[1].tolist() == [23, 32, 36, 37, 38, 39, -1] and int(a[4]) == 0
    assert a[2].tolist() == [[5, 8], [9, -1]] and got[0].tolist() == [3, 4, 0, 1, 2, 3, 4]
    # past the table
    got, a = step([7], [3], [[5, 6]], [9], 1, 3)
    assert ops.device_error() == 102 and got[1].tolist() == [27, -1, -1] and int(a[4]) == 1
    # fewer rows than the step has
    got, a = step([0, 0], [2, 2], [[-1], [-1]], [9, 8], 2, 3)
    assert ops.device_error() == 104 and got[1].tolist() == [32, 33, 36] and got[2].tolist() == [0, 2, 4]
    # a free list that is full takes nothing more
    got, a = step([9], [0], [[1, 2, 3]], [4, 5], 2, 0, window=1)
    assert ops.device_error() == 105 and a[3].tolist() == [4, 5] and a[2].tolist() == [[-1, -1, 3]] and int(a[4]) == 2
    # slots past 32 bits
    got, a = step([0], [1], [[1 << 30]], [9], 0, 1)
    assert ops.device_error() == 101 and got[1].tolist() == [-1]
    # idle places have rows; negative new lengths are none
    got, a = step([-1, 2, -7, 4], [2, -3, 1, 1], [[-1], [1], [-1], [-1]], [9], 1, 5)
    assert ops.device_error() == 102 and got[0].tolist() == [0, 0, 0, 4, 0] and got[1].tolist() == [-1] * 5
    assert got[2].tolist() == [0, 2, 2, 3, 4] and got[4].tolist() == [0, 2, 0, 5]
    # no sequences
    got = ops.step_metadata(*(torch.empty(n, **i32) for n in ((0,), (0,), (0, 4), (2,))), torch.zeros(1, **i32), 4, 3)
    assert ops.device_error() == 0 and got[0].tolist() == [0] * 3 and got[1].tolist() == [-1] * 3 and got[2].tolist() == [0]


def test_step_metadata_many_rows_of_idle_places():
    """The second launch (many rows) with idle places, empty ones and rows to spare."""
    ops = _ops()
    r = np.random.default_rng(5)
    lens = [int(x) for x in r.integers(0, 300, 40)]
    new = [int(x) for x in r.integers(0, 900, 40)]
    for i in (0, 7, 39):
        lens[i] = -1
    new[3] = new[38] = 0
    tables = [[-1] * 40 for _ in lens]
    free = r.permutation(1700).tolist()
    for t, n in zip(tables, lens):
        for p in range((max(n, 0) + 31) // 32):
            t[p] = free.pop()
    count = len(free)
    free += [0] * 300
    total = sum(new) + 4097
    want = oracle.step(lens, new, tables, free, count, 32, total, 100, 4)
    i32 = dict(dtype=torch.int32, device="cuda")
    a = [torch.tensor(x, **i32) for x in (lens, new, tables, free, [count])]
    got = ops.step_metadata(*a, 32, total, 100, 4)
    assert ops.device_error() == 0
    for x, w in zip(got + (a[2], a[3], a[4]), want[:7] + ([want[7]],)):
        assert x.tolist() == w


# ------------------------------------------------------------------ verification: what goes wrong
def _verify_one(drafts, p, q, u, u_last, dtype=torch.float32):
    p = torch.tensor([p], dtype=dtype, device="cuda")
    q = None if q is None else torch.tensor([q], dtype=dtype, device="cuda")
    k = len(drafts)
    got = _ops().verify_drafts(torch.tensor([drafts], dtype=torch.int64, device="cuda").view(1, k), p, q,
                               torch.tensor([u], dtype=torch.float32, device="cuda").view(1, k),
                               torch.tensor([u_last], dtype=torch.float32, device="cuda"))
    want = oracle.verify(drafts, p[0].cpu(), None if q is None else q[0].cpu(), torch.tensor(u).tolist(),
                         float(torch.tensor(u_last)))
    assert int(got[1]) == len(want) and got[0][0].tolist() == want + [-1] * (k + 1 - len(want))
    return want


def test_verify_drafts_borders():
    half = [0.5, 0.5, 0.0]
    assert _verify_one([], [half], None, [], 0.5) == [1]                   # half of the counts belong to token 0
    assert _verify_one([], [half], None, [], 0.5 - 2.0 ** -24) == [0]
    assert _verify_one([], [[0.0, 0.25, 0.0, 0.75]], None, [], 0.0) == [1]  # the first with any weight
    assert _verify_one([0], [half, half], [half], [1.0 - 2.0 ** -24], 0.0) == [0, 0]   # equal: accepted below 1
    assert _verify_one([2], [half, half], [half], [0.0], 0.9) == [1]      # 0 < 0 does not hold, and p - q is 0: p
    assert _verify_one([0], [[0.25, 0.5, 0.25], half], None, [0.25], 0.0) == [1]      # 0.25 < 0.25 does not hold
    assert _verify_one([0], [[0.25, 0.5, 0.25], half], None, [0.2499], 0.0) == [0, 0]
    assert _verify_one([1], [[1.0, 0.0], half[:2]], [[0.0, 1.0]], [0.0], 0.99) == [0]
    assert _verify_one([0, 1], [half, half, half], [half, half], [0.1, 0.1], 0.7) == [0, 1, 1]
    assert _verify_one([0, -1, 1], [half] * 4, None, [0.1, 0.1, 0.1], 0.7) == [0, 1]   # -1 ends the drafts


def test_verify_drafts_rows_that_are_no_probabilities():
    nan, inf = math.nan, math.inf
    assert _verify_one([], [[nan, -1.0, 0.5, inf]], None, [], 0.2) == [2]   # NaN and below 0 count 0, above 1 as 1
    assert _verify_one([], [[nan, -1.0, 0.5, inf]], None, [], 0.9) == [3]
    assert _verify_one([], [[0.0, 0.0]], None, [], 0.5) == [-1]
    assert _verify_one([], [[nan, nan]], None, [], 0.5) == [-1]
    assert _verify_one([1], [[0.0, nan], [0.5, 0.5]], [[0.5, 0.5]], [0.5], 0.5) == [-1]
    assert _verify_one([0], [[nan, 1.0], [0.5, 0.5]], [[0.5, 0.5]], [0.5], 0.5) == [1]   # NaN accepts nothing
    for u in (1.0, 2.0, inf):
        assert _verify_one([], [[0.5, 0.5]], None, [], u) == [1]
    for u in (-0.5, nan, -inf):
        assert _verify_one([], [[0.5, 0.5]], None, [], u) == [0]
    assert _verify_one([], [[1e-30, 2.0 ** -42, 2.0 ** -43]], None, [], 0.9) == [1]   # what counts below one is nothing
    assert _ops().device_error() == 0


def test_verify_drafts_past_the_vocabulary():
    ops = _ops()
    p = torch.full((2, 3, 5), 0.2, device="cuda")
    drafts = torch.tensor([[1, 5], [1 << 40, 0]], device="cuda")
    tokens, emitted = ops.verify_drafts(drafts, p, None, torch.zeros(2, 2, device="cuda"), torch.zeros(2, device="cuda"))
    assert ops.device_error() == 106 and emitted.tolist() == [2, 1] and tokens.tolist() == [[1, 0, -1], [0, -1, -1]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 15, 16, 17, 1023, 8191, 8193, 1 << 18])
def test_verify_drafts_alignments(dtype, vocab):
    """Rows that begin at every place of a 16-byte word, p's and q's alike and apart; every token can come."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(vocab)
    b, k = 9, 1
    for apart in (0, 1):
        room = vocab + 16
        big_p = torch.full((b, k + 1, room), math.nan, dtype=dtype, device="cuda")
        big_q = torch.full((b, k, room), math.nan, dtype=dtype, device="cuda")
        drafts = torch.randint(0, vocab, (b, k), generator=g, device="cuda")
        u, u_last = torch.rand(b, k, generator=g, device="cuda"), torch.rand(b, generator=g, device="cuda")
        u_last[0], u_last[1] = 0.0, 1 - 2.0 ** -24   # the first and the last token that have weight
        flat = torch.full((2, vocab), 1 / vocab, device="cuda")
        for shift in range(8):
            p, q = big_p[..., shift:shift + vocab], big_q[..., (shift + apart) % 8:(shift + apart) % 8 + vocab]
            p.copy_(_probabilities(g, b, k + 1, vocab, dtype))
            p[:2] = flat.to(dtype)
            q.copy_(_probabilities(g, b, k, vocab, dtype))
            for draft in (q, None):
                tokens, emitted = ops.verify_drafts(drafts, p, draft, u, u_last)
                some = range(b) if vocab < 10000 else range(0, 3)
                for i in some:
                    want = oracle.verify(drafts[i].tolist(), p[i].cpu(), None if draft is None else draft[i].cpu(),
                                         u[i].tolist(), float(u_last[i]))
                    assert tokens[i, :len(want)].tolist() == want and int(emitted[i]) == len(want)
            if vocab > 10000 and shift == 2:
                break
    assert ops.device_error() == 0


def test_verify_drafts_many_sequences_and_lengths():
    """More sequences than clusters fit at once, lengths moved on in place, the call captured."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(2)
    b, k, vocab = 700, 2, 900
    p, q = _probabilities(g, b, k + 1, vocab, torch.float32), _probabilities(g, b, k, vocab, torch.float32)
    drafts = torch.randint(0, vocab, (b, k), generator=g, device="cuda")
    u, u_last = torch.rand(b, k, generator=g, device="cuda") ** 4, torch.rand(b, generator=g, device="cuda")
    lens = torch.arange(-2, b - 2, dtype=torch.int32, device="cuda")
    before = lens.clone()
    tokens, emitted = ops.verify_drafts(drafts, p, q, u, u_last, lens)
    assert torch.equal(lens, torch.where(before < 0, before, before + emitted))
    for i in range(0, b, 7):
        want = oracle.verify(drafts[i].tolist(), p[i].cpu(), q[i].cpu(), u[i].tolist(), float(u_last[i]))
        assert tokens[i].tolist() == want + [-1] * (k + 1 - len(want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.verify_drafts(drafts, p, q, u, u_last)
    p.copy_(p.flip(0)), q.copy_(q.flip(0)), drafts.copy_(drafts.flip(0)), u.copy_(u.flip(0)), u_last.copy_(u_last.flip(0))
    graph.replay()
    assert torch.equal(out[0], tokens.flip(0)) and torch.equal(out[1], emitted.flip(0))
    empty = ops.verify_drafts(drafts[:0], p[:0], q[:0], u[:0], u_last[:0])
    assert empty[0].shape == (0, k + 1) and empty[1].shape == (0,)


# ------------------------------------------------------------------ a run of them together
class _Model:
    """Two attention layers over embeddings of the tokens, one with a sliding window; logits from their outputs."""

    def __init__(self, seed, vocab=97, heads=8, kv_heads=2, window=40, sinks=3, all_windowed=True):
        from vlcache_b200.layers.attention import Attention
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.vocab = heads, kv_heads, vocab
        self.embed = torch.randn(vocab, (heads + 2 * kv_heads) * D, generator=g, device="cuda").to(torch.bfloat16)
        self.head = torch.randn(heads * D, vocab, generator=g, device="cuda") * 0.08
        self.layers = [Attention(heads, D, 0.1, kv_heads, window, sinks),
                       Attention(heads, D, 0.1, kv_heads, window if all_windowed else None, sinks)]

    def rows(self, tokens, positions):
        x = self.embed[tokens.clamp(min=0)] * (1 + 0.1 * torch.sin(positions)).unsqueeze(-1).to(torch.bfloat16)
        x = x.view(-1, self.heads + 2 * self.kv_heads, D)
        return x[:, :self.heads], x[:, self.heads:-self.kv_heads], x[:, -self.kv_heads:]

    def caches(self, pages, block):
        for i, layer in enumerate(self.layers):
            layer.k_cache, layer.v_cache = (torch.zeros(pages, block, self.kv_heads, D, dtype=torch.bfloat16, device="cuda")
                                            for _ in range(2))

    def __call__(self, tokens, positions):
        q, k, v = self.rows(tokens, positions)
        o = sum(layer(q, k.contiguous(), v.contiguous()).reshape(-1, self.heads * D).float() for layer in self.layers)
        return torch.softmax(o @ self.head, -1)

    def plain(self, tokens):
        """Probabilities behind each token of one sequence, from 64-bit attention over all of it."""
        pos = torch.arange(len(tokens), device="cuda")
        q, k, v = (x.double() for x in self.rows(torch.tensor(tokens, device="cuda"), pos))
        o = sum(oracle.attention(q, k, v, pos, l.sliding_window, l.num_sinks, 0.1)[0] for l in self.layers)
        return torch.softmax(o.flatten(1) @ self.head.double(), -1)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("all_windowed", [True, False])
def test_draft_decode_together(captured, all_windowed):
    """Prompts through the windowed prefill, then steps of drafts: what is emitted is what each sequence alone, by
    64-bit attention over all of its tokens, gives its probabilities to; pages go back and are used again."""
    from vlcache_b200.engine.draft_decode import DraftDecode
    from vlcache_b200.engine.page_pool import PagePool
    from vlcache_b200.utils.context import reset_context, set_context
    ops = _ops()
    block, places, drafts_n = 32, 4, 3
    model = _Model(7, all_windowed=all_windowed)
    pool = PagePool(200, block)
    model.caches(200, block)
    window = 40 if all_windowed else 0
    d = DraftDecode(pool, places, 16, drafts_n, window, 3 if window else 0)
    assert d.lend(40)
    r = np.random.default_rng(4)
    histories = {0: [int(x) for x in r.integers(0, 97, 50)], 1: [int(x) for x in r.integers(0, 97, 7)],
                 3: [int(x) for x in r.integers(0, 97, 133)]}

    def prompt(place, tokens):
        table = pool.allocate(pool.pages_for(len(tokens)))
        n = len(tokens)
        slots = torch.tensor([table[t // block] * block + t % block for t in range(n)], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        # this layer stack has no residual path, so one call fills every layer's cache
        set_context(True, cu, cu, n, n, slots, None, None, cu_seqlens_q_host=[0, n], cu_seqlens_k_host=[0, n])
        probs = model(torch.tensor(tokens, device="cuda"), torch.arange(n, device="cuda"))
        want = model.plain(tokens)
        assert float((probs.double() - want).abs().max()) < 0.05
        d.admit(place, table, n)
        return int(probs[-1].argmax())

    last = {p: prompt(p, h) for p, h in histories.items()}
    tokens_in = torch.zeros(places, drafts_n + 1, dtype=torch.int64, device="cuda")
    u, u_last = torch.zeros(places, drafts_n, device="cuda"), torch.zeros(places, device="cuda")

    def step():
        positions = d.begin()
        probs = model(tokens_in.flatten(), positions).view(places, drafts_n + 1, -1)
        return (probs,) + d.finish(tokens_in[:, 1:].contiguous(), probs, None, u, u_last)

    graph = None
    for turn in range(14):
        guess = torch.full((places, drafts_n + 1), -1, dtype=torch.int64)
        for p in histories:   # drafts: the right ones up to somewhere, then others
            row, good = [last[p]], int(r.integers(0, drafts_n + 1))
            for i in range(drafts_n):
                best = int(model.plain(histories[p] + row)[-1].argmax())
                row.append(best if i < good else int(r.integers(0, 97)))
            guess[p] = torch.tensor(row)
        tokens_in.copy_(guess)
        u.copy_(torch.tensor(r.random((places, drafts_n)) * 0.2, dtype=torch.float32))
        u_last.copy_(torch.tensor(r.random(places), dtype=torch.float32))
        lens = {p: len(h) for p, h in histories.items()}
        if captured and graph is None:
            saved = [t.clone() for t in (d.context_lens, d.block_tables, d.free_pages, d.num_free)]
            step()   # what a first call sets up
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                probs, tokens, emitted = step()
            for t, s in zip((d.context_lens, d.block_tables, d.free_pages, d.num_free), saved):
                t.copy_(s)
        if graph is not None:
            graph.replay()
        else:
            probs, tokens, emitted = step()
        assert ops.device_error() == 0
        for p in histories:
            want = model.plain(histories[p] + guess[p].tolist())[lens[p]:]
            # An output is off by STEP * (2 rms + |o|) < 0.02 a layer, of either sign; a logit sums 512 of each of the
            # two layers' (8 heads of 128, summed by pairs) times 0.08: 0.02 * 0.08 * sqrt(2048) = 0.07 would be
            # the deviation if all were that far off, and a probability moves by a quarter of it at most.
            assert float((probs[p].double() - want).abs().max()) < 0.05, (turn, p)
            out = oracle.verify(guess[p, 1:].tolist(), probs[p].cpu(), None, u[p].tolist(), float(u_last[p]))
            assert tokens[p].tolist() == out + [-1] * (drafts_n + 1 - len(out)) and int(emitted[p]) == len(out)
            histories[p] += guess[p, :len(out)].tolist()
            last[p] = out[-1]
            assert int(d.context_lens[p]) == len(histories[p])
        if window:   # pages wholly behind the window went back, the first stays (its sinks)
            for p, h in histories.items():
                live = [i for i, x in enumerate(d.block_tables[p].tolist()) if x >= 0]
                gone = (lens[p] - window + 1) // block
                assert 0 in live and all(i == 0 or i >= gone for i in live)
        pages = [x for row in d.block_tables.tolist() for x in row if x >= 0] + d.free_pages[:int(d.num_free)].tolist()
        assert len(pages) == len(set(pages))   # no page is twice in use
        if turn == 8:   # one leaves, another comes
            d.retire(0)
            del histories[0]
            histories[2] = [int(x) for x in r.integers(0, 97, 64)]
            last[2] = prompt(2, histories[2])
    for p in histories:
        d.retire(p)
    d.settle()
    assert pool.num_free == 200 and pool.refs == [0] * 200
    reset_context()


# ------------------------------------------------------------------ further calls that the documentation allows
@pytest.mark.parametrize("lens", [(200, 70, 333), (9000,) * 40])
def test_decode_window_in_place(lens):
    """The output over the query."""
    g, lens, tables, k_cache, v_cache, q = _small(lens=lens)
    want = _decode(tables, lens, None, q, k_cache, v_cache, 70, 4, 0.1)
    got = _decode(tables, lens, None, q, k_cache, v_cache, 70, 4, 0.1, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, want)


def test_decode_window_many_short_sequences():
    g = torch.Generator(device="cuda").manual_seed(11)
    lens = [int(x) for x in np.random.default_rng(1).integers(0, 40, 2500)]
    tables, pages = _tables(g, lens, 32)
    k_cache, v_cache = _caches(g, pages, 32, 1)
    q = torch.randn(len(lens), 2, 8, D, generator=g, device="cuda").to(torch.bfloat16)
    got = _decode(tables, lens, None, q, k_cache, v_cache, 9, 2, 0.1)
    assert _ops().device_error() == 0
    pick = list(range(0, 2500, 37))
    _check_decode(got[pick], tables[pick], [lens[i] for i in pick], 2, q[pick], k_cache, v_cache, 9, 2, 0.1)
    assert bool((got[[i for i, n in enumerate(lens) if n == 0]] == 0).all())


@pytest.mark.parametrize("lens", [(500, 77), (20000, 9999)])
def test_decode_window_one_cache_for_both(lens):
    """Keys that are the values (one tensor): copied apart, since their distance is 0."""
    g, lens, tables, k_cache, _, q = _small(lens=lens)
    got = _decode(tables, lens, None, q, k_cache, k_cache, 0, 0, 0.1)
    _check_decode(got, tables, lens, 2, q, k_cache, k_cache, 0, 0, 0.1)


@pytest.mark.parametrize("head_dim", [80, 96, 128])
def test_prefill_window_head_dims(head_dim):
    """Contiguous keys and values of narrower heads, whole and split tiles."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(head_dim)
    new, lens = [300, 9], [300, 5000]
    cu_q, cu_k = np.cumsum([0] + new), np.cumsum([0] + lens)
    q, k, v = (torch.randn(n, h, head_dim, generator=g, device="cuda").to(torch.bfloat16)
               for n, h in ((309, 16), (5300, 2), (5300, 2)))
    plan = ops.build_prefill_plan(cu_q, cu_k, 16, 2, head_dim, device="cuda", window=1500, sinks=4)
    assert plan.num_parts > 0
    got = ops.prefill_attention(q, k, v, None, plan, 0.1)
    assert ops.device_error() == 0
    for i, (n, m) in enumerate(zip(new, lens)):
        want, rms = oracle.attention(q[cu_q[i]:cu_q[i + 1]].double(), k[cu_k[i]:cu_k[i + 1]].double(),
                                     v[cu_k[i]:cu_k[i + 1]].double(), torch.arange(m - n, m, device="cuda"), 1500, 4, 0.1)
        tol = (STEP + 2.0 ** -12) * (2 * rms + want.abs()) + 1e-30   # (as test_prefill_window)
        assert bool(((got[cu_q[i]:cu_q[i + 1]].double() - want).abs() <= tol).all())


def test_prefill_window_over_a_4_bit_cache_and_refusals():
    """A windowed plan over keys read back from 4 bits is the one over those keys in bf16; scales that are not
    positive are refused."""
    ops = _ops()
    from vlcache_b200._lib import VLCError
    from vlcache_b200.layers.attention import Attention
    from vlcache_b200.utils.context import reset_context, set_context
    g = torch.Generator(device="cuda").manual_seed(4)
    n, block = 700, 128
    k, v = (torch.randn(n, 2, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(300, 16, D, generator=g, device="cuda").to(torch.bfloat16)
    k4, v4 = (torch.zeros(6, 2, block * 72, dtype=torch.uint8, device="cuda") for _ in range(2))
    ops.store_kvcache_fp4(k, v, k4, v4, torch.arange(n, dtype=torch.int32, device="cuda"))
    tables = torch.arange(6, dtype=torch.int32, device="cuda").view(1, 6)
    cu_k = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    plan = ops.build_prefill_plan([0, 300], [0, n], 16, 2, device="cuda", window=200, sinks=4)
    a = ops.prefill_attention_fp4(q, k4, v4, tables, cu_k, plan, 0.1)
    kb, vb = ops.gather_kvcache_fp4(k4, v4, tables, cu_k, n)
    assert torch.equal(a, ops.prefill_attention(q, kb, vb, None, plan, 0.1)) and ops.device_error() == 0
    for scale in (0.0, -0.1, math.nan):
        with pytest.raises(VLCError):
            ops.prefill_attention(q, kb, vb, None, plan, scale)
    layer = Attention(16, D, 0.1, 2, 200)
    layer.k_cache, layer.v_cache = k4, v4
    set_context(False, slot_mapping=torch.full((1,), -1, dtype=torch.int32, device="cuda"), context_lens=cu_k[1:],
                block_tables=tables)
    with pytest.raises(ValueError, match="4-bit"):
        layer(q[:1], k[:1], v[:1])
    layer = Attention(16, D, 0.1, 2)
    layer.k_cache, layer.v_cache = (torch.zeros(6, block, 2, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    set_context(False, slot_mapping=torch.full((3,), -1, dtype=torch.int32, device="cuda"),
                context_lens=cu_k.clone(), block_tables=tables.expand(2, 6).contiguous())
    with pytest.raises(ValueError, match="3 rows for 2 sequences"):
        layer(q[:3], k[:3], v[:3])
    reset_context()


def test_prefill_window_plans_are_pairs(cuda_lib):
    ops = _ops()
    try:
        ops.set_prefill_kernel(ops.PREFILL_QUADS)
        plan = ops.build_prefill_plan([0, 700], [0, 900], 16, 2, device="cuda", window=100)
        assert int(plan.host[21]) == 0 and int(plan.host[22]) == 100
    finally:
        ops.set_prefill_kernel(ops.PREFILL_DEFAULT)


@pytest.mark.parametrize("b", [8193, 65535])
def test_step_metadata_many_sequences(b):
    """The most sequences: a page of two tokens each."""
    ops = _ops()
    i32 = dict(dtype=torch.int32, device="cuda")
    lens = torch.arange(b, **i32) % 3 - 1              # idle, empty, one token
    tables = torch.full((b, 2), -1, **i32)
    one = (lens == 1).nonzero().flatten()
    tables[one, 0] = one.int()
    free = torch.arange(b, 3 * b, **i32)
    count, new = torch.tensor([2 * b], **i32), torch.full((b,), 2, **i32)
    positions, slots, cu_q, cu_k, after = ops.step_metadata(lens, new, tables, free, count, 2, 2 * b)
    assert ops.device_error() == 0
    missing = (lens >= 0).long()                        # empty: its first page; one token: its second
    nth = missing.cumsum(0) - 1
    page = torch.where(missing > 0, 3 * b - 1 - nth, -1)
    want = torch.full((b, 2), -1, dtype=torch.int64, device="cuda")
    want[:, 0] = torch.where(lens == 0, page, torch.where(lens == 1, torch.arange(b, device="cuda"), -1))
    want[:, 1] = torch.where(lens == 1, page, -1)
    assert torch.equal(tables.long(), want) and int(count) == 2 * b - int(missing.sum())
    start = lens.clamp(min=0).long()
    pos = torch.stack((start, start + 1), 1)
    live = (lens >= 0).view(-1, 1)
    assert torch.equal(positions.view(b, 2), torch.where(live, pos, 0))
    slot = want.gather(1, (pos // 2).clamp(max=1)) * 2 + pos % 2
    assert torch.equal(slots.view(b, 2).long(), torch.where(live, slot, -1))
    assert torch.equal(cu_q.long(), 2 * torch.arange(b + 1, device="cuda"))
    assert torch.equal(after.long(), torch.where(lens >= 0, start + 2, 0)) and int(cu_k[-1]) == int(after.sum())


def test_verify_drafts_shared_rows():
    """One distribution for all sequences (strides of 0), and random numbers likewise."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(6)
    p = _probabilities(g, 1, 3, 5000, torch.float32).expand(50, 3, 5000)
    u = torch.rand(1, 2, generator=g, device="cuda").expand(50, 2)
    drafts = torch.randint(0, 5000, (1, 2), generator=g, device="cuda").expand(50, 2)
    tokens, emitted = ops.verify_drafts(drafts, p, None, u, torch.full((50,), 0.3, device="cuda"))
    assert bool((tokens == tokens[0]).all()) and bool((emitted == emitted[0]).all())
    want = oracle.verify(drafts[0].tolist(), p[0].cpu(), None, u[0].tolist(), float(torch.tensor(0.3)))
    assert tokens[0].tolist() == want + [-1] * (3 - len(want))


# ------------------------------------------------------------------ decode of more than 24 rows a KV head
MANY_ROWS = [
    # heads, kv_heads, tokens, block, window, sinks: 28, 35, 48, 56, 72, 91, 112 and 128 rows
    (14, 2, 4, 256, 700, 4),
    (14, 2, 5, 32, 129, 20),
    (32, 2, 3, 96, 0, 0),
    (7, 1, 8, 160, 128, 0),
    (24, 2, 6, 128, 300, 130),
    (14, 2, 13, 64, 1, 0),
    (7, 1, 16, 256, 1000, 1),
    (16, 1, 8, 32, 255, 300),
]


@pytest.mark.parametrize("case", MANY_ROWS, ids=lambda c: "-".join(map(str, c)))
def test_decode_window_many_rows(case):
    """Lengths around the chunks' borders, pairs that blocks share, rows that see nothing, and NaN and infinities
    in every key and value that no row sees."""
    heads, kv_heads, n, block, window, sinks = case
    g = torch.Generator(device="cuda").manual_seed(heads + n + block)
    lens = [0, 1, n, 127, 128, 129, 255, 256, 257, 383, 4000] + [int(x) for x in np.random.default_rng(n).integers(1, 2500, 50)]
    tables, pages = _tables(g, lens, block)
    k_cache, v_cache = _caches(g, pages, block, kv_heads, joined=n % 2 == 0)
    q = (1.5 * torch.randn(len(lens), n, heads, D, generator=g, device="cuda")).to(torch.bfloat16)
    new = [min(n, m) for m in lens]
    _spoil(k_cache, tables, lens, new, window, sinks, math.nan)
    _spoil(v_cache, tables, lens, new, window, sinks, math.inf)
    _release(tables, lens, new, block, window, sinks)
    got = _decode(tables, lens, new, q, k_cache, v_cache, window, sinks, 0.09)
    assert _ops().device_error() == 0
    _check_decode(got, tables, lens, n, q, k_cache, v_cache, window, sinks, 0.09)
    assert torch.equal(got, _decode(tables, lens, new, q, k_cache, v_cache, window, sinks, 0.09, out=q))   # in place


@pytest.mark.parametrize("scale", [0.3, -0.3, 0.0])
def test_decode_window_many_rows_scales_and_broken_queries(scale):
    g, lens, tables, k_cache, v_cache, q = _small(lens=(200, 70, 3330), n=5)
    q[0, 1, 3, 5], q[1, 0, 0, 0], q[2, 4, 15, 127] = math.inf, math.nan, -math.inf
    got = _decode(tables, lens, None, q, k_cache, v_cache, 40, 0, scale)
    broken = ~torch.isfinite(q).all(-1)
    assert int(broken.sum()) == 3 and bool(torch.isnan(got[broken]).all()) and bool(torch.isfinite(got[~broken]).all())
    clean = torch.where(broken.unsqueeze(-1), torch.zeros_like(q), q)
    again = _decode(tables, lens, None, clean, k_cache, v_cache, 40, 0, scale)
    _check_decode(again, tables, lens, 5, clean, k_cache, v_cache, 40, 0, scale)
    assert torch.equal(got[~broken], again[~broken])


def test_decode_window_many_rows_large_scores():
    """Scores that rise along the keys: the maxima move again and again."""
    g, lens, tables, k_cache, v_cache, q = _small(lens=(3000, 2000), n=4)
    rising = torch.linspace(0.1, 3, 3000, device="cuda")
    for i, m in enumerate(lens):
        at, row = tables[i].long()[torch.arange(m, device="cuda") // 64], torch.arange(m, device="cuda") % 64
        k_cache[at, row] = (k_cache[at, row].float() * rising[:m, None, None]).to(torch.bfloat16)
    got = _decode(tables, lens, None, q, k_cache, v_cache, 0, 0, 0.5)
    # a score is off by 130 steps of fp32 of sum |q k| at most (128 products, two roundings of the scale)
    most = 0.5 * float(q.double().abs().sum(-1).max() * k_cache.double().abs().max())
    most = min(most, 0.5 * float((q.double() ** 2).sum(-1).max().sqrt() * (k_cache.double() ** 2).sum(-1).max().sqrt()))
    _check_decode(got, tables, lens, 4, q, k_cache, v_cache, 0, 0, 0.5, scores=130 * 2.0 ** -24 * most)


def test_decode_window_many_rows_bad_pages_and_lengths():
    ops = _ops()
    g, lens, tables, k_cache, v_cache, q = _small(lens=(200, 70, 5000), n=4, block=32)
    for bad in (-1, k_cache.shape[0], 1 << 30, -(1 << 31)):
        broken = tables.clone()
        broken[2, 7], broken[1, 1] = bad, bad
        got = _decode(broken, lens, None, q, k_cache, v_cache, 0, 0, 0.1)
        assert ops.device_error() == 102
        keys = k_cache.clone(), v_cache.clone()   # their keys count as zeros, the others of their chunks stay
        for c in keys:
            c[tables[2, 7].long()] = 0
            c[tables[1, 1].long()] = 0
        _check_decode(got, tables, lens, 4, q, *keys, 0, 0, 0.1)
    got = _decode(tables[:, :1].contiguous(), lens, None, q, k_cache, v_cache, 0, 0, 0.1)
    assert ops.device_error() == 102 and bool(torch.isfinite(got).all())
    got = _decode(tables, lens, None, q, k_cache, v_cache, 30, 2, 0.1, bound=100)
    assert ops.device_error() == 104
    _check_decode(got, tables, [min(m, 100) for m in lens], 4, q, k_cache, v_cache, 30, 2, 0.1)


def test_decode_window_many_rows_strides_and_captured():
    """A projection's rows, a caller's output and workspace; two graphs at once that follow changed lengths."""
    ops = _ops()
    g, lens, tables, k_cache, v_cache, q = _small(lens=(900, 70, 5000), n=4)
    rows = torch.full((12, 20 * D), math.nan, dtype=torch.bfloat16, device="cuda")
    view = rows[:, :16 * D].view(3, 4, 16, D)
    view.copy_(q)
    into = torch.full((13, 17, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = into[:12, :16].view(3, 4, 16, D)
    need = ops.decode_window_workspace_bytes(3, 4, 16, 2, 5000, 600, 3)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ops.decode_attention_window(view, k_cache, v_cache, tables, lens_t, 5000, 0.1, 600, 3, out,
                                torch.empty(need, dtype=torch.uint8, device="cuda"))
    _check_decode(out, tables, lens, 4, q, k_cache, v_cache, 600, 3, 0.1)
    assert bool((into[12:] == 7).all()) and bool((into[:, 16:] == 7).all())
    qs, graphs, outs = [q, q.flip(0).contiguous()], [], []
    for x in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.decode_attention_window(x, k_cache, v_cache, tables, lens_t, 5000, 0.1, 600, 3))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for cut in (0, 3, 64):
        now = [max(0, m - cut * 2) for m in lens]
        lens_t.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for x, o in zip(qs, outs):
            _check_decode(o, tables, now, 4, x, k_cache, v_cache, 600, 3, 0.1)
    assert ops.device_error() == 0


def test_decode_window_many_rows_pages_beyond_4_gb():
    g = torch.Generator(device="cuda").manual_seed(3)
    pages, block, kv_heads = 9000, 256, 4
    both = torch.empty(2, pages, block, kv_heads, D, dtype=torch.bfloat16, device="cuda")
    both[:, -4:].normal_(generator=g)
    tables = torch.tensor([[pages - 1, pages - 3], [pages - 2, pages - 4]], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 5, 28, D, generator=g, device="cuda").to(torch.bfloat16)
    got = _decode(tables, [400, 512], None, q, both[0], both[1], 300, 4, 0.1)
    _check_decode(got, tables, [400, 512], 5, q, both[0], both[1], 300, 4, 0.1)


@pytest.mark.parametrize("head_dim", [80, 128])
@pytest.mark.parametrize("window", [0, 6000, 20000])
def test_prefill_window_split_tiles_that_see_all_keys(head_dim, window):
    """No window, and windows that hide nothing: the parts of split tiles are fp32, P's rounding and the output's
    are the only ones."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(head_dim)
    new, lens = [48, 9], [6000, 500]
    cu_q, cu_k = np.cumsum([0] + new), np.cumsum([0] + lens)
    q, k, v = (torch.randn(n, h, head_dim, generator=g, device="cuda").to(torch.bfloat16)
               for n, h in ((57, 16), (6500, 2), (6500, 2)))
    plan = ops.build_prefill_plan(cu_q, cu_k, 16, 2, head_dim, device="cuda", window=window)
    assert plan.num_parts > 0
    got = ops.prefill_attention(q, k, v, None, plan, 0.1)
    assert ops.device_error() == 0
    for i, (n, m) in enumerate(zip(new, lens)):
        want, rms = oracle.attention(q[cu_q[i]:cu_q[i + 1]].double(), k[cu_k[i]:cu_k[i + 1]].double(),
                                     v[cu_k[i]:cu_k[i + 1]].double(), torch.arange(m - n, m, device="cuda"), 0, 0, 0.1)
        tol = (STEP + 2.0 ** -12) * (rms + want.abs()) + 1e-30
        assert bool(((got[cu_q[i]:cu_q[i + 1]].double() - want).abs() <= tol).all())
