"""A decode step with drafted tokens on the device, further: what its inputs may hold and which calls may follow one
another."""
import math

import pytest
import torch

from oracle import draft_decode as oracle

pytestmark = pytest.mark.gpu

D = 128


def _ops():
    from vlcache_b200 import ops
    return ops


# ------------------------------------------------------------------ verification
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("vocab", [5, 64, 1000, 40003])
@pytest.mark.parametrize("sampled", [True, False])
def test_verify_drafts_counts_negative_zeros_as_none(dtype, vocab, sampled):
    """Probabilities of -0.0 (and -0.0 - 0.0 at a refused draft) count 0, in whole vectors and at a row's ends."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(vocab)
    b, k = 12, 2
    p = torch.softmax(2 * torch.randn(b, k + 1, vocab, generator=g, device="cuda"), -1).to(dtype)
    q = torch.softmax(2 * torch.randn(b, k, vocab, generator=g, device="cuda"), -1).to(dtype)
    zero = torch.rand(p.shape, generator=g, device="cuda") < 0.5
    zero[..., 0] = zero[..., -1] = True
    zero[..., vocab // 2] = False
    p = torch.where(zero, torch.full_like(p, -0.0), p)
    q = torch.where(zero[:, :k] & (torch.rand(q.shape, generator=g, device="cuda") < 0.7), torch.zeros_like(q), q)
    assert bool(torch.signbit(p[..., 0]).all())
    drafts = torch.randint(0, vocab, (b, k), generator=g, device="cuda")
    u, u_last = torch.rand(b, k, generator=g, device="cuda"), torch.rand(b, generator=g, device="cuda")
    tokens, emitted = ops.verify_drafts(drafts, p, q if sampled else None, u, u_last)
    assert ops.device_error() == 0
    for i in range(b):
        want = oracle.verify(drafts[i].tolist(), p[i].cpu(), q[i].cpu() if sampled else None, u[i].tolist(),
                             float(u_last[i]))
        assert tokens[i].tolist() == want + [-1] * (k + 1 - len(want)) and int(emitted[i]) == len(want)


# ------------------------------------------------------------------ steps that find no page
def _stored(table, length, rows, block):
    """Leading rows of a step at positions length .. that the table has pages for."""
    for r in range(rows):
        if (length + r) // block >= len(table) or table[(length + r) // block] < 0:
            return r
    return rows


@pytest.mark.parametrize("blocks", [1, 8])   # of the cluster that takes a sequence
def test_verify_drafts_of_rows_without_pages(blocks):
    """A draft in a row without a page is none, a sequence without a page for its first row emits nothing; idle places
    and sequences whose rows have pages are verified as without tables."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(3)
    b, k, vocab, block, width = (600 if blocks == 1 else 12), 3, 517, 4, 5
    p = torch.softmax(2 * torch.randn(b, k + 1, vocab, generator=g, device="cuda"), -1)
    q = torch.softmax(2 * torch.randn(b, k, vocab, generator=g, device="cuda"), -1)
    drafts = torch.randint(0, vocab, (b, k), generator=g, device="cuda")
    u, u_last = torch.rand(b, k, generator=g, device="cuda") ** 4, torch.rand(b, generator=g, device="cuda")
    lens = (torch.arange(b, device="cuda") * 7 % 23 - 1).int()   # -1: idle; up to 21, past the table of 20 tokens
    tables = torch.where(torch.rand(b, width, generator=g, device="cuda") < 0.3, -1, 9).int()
    wide = torch.full((b, width + 2), 7, dtype=torch.int32, device="cuda")   # pages behind a row's end are not its own
    wide[:, :width] = tables
    before = lens.clone()
    tokens, emitted = ops.verify_drafts(drafts, p, q, u, u_last, lens, wide[:, :width], block)
    seen = set()
    for i in range(b):
        n = int(before[i])
        rows = k + 1 if n < 0 else _stored(tables[i].tolist(), n, k + 1, block)
        seen.add(rows)
        ds = [d if r + 1 < rows else -1 for r, d in enumerate(drafts[i].tolist())]
        want = [] if rows == 0 else oracle.verify(ds, p[i].cpu(), q[i].cpu(), u[i].tolist(), float(u_last[i]))
        assert tokens[i].tolist() == want + [-1] * (k + 1 - len(want)) and int(emitted[i]) == len(want), i
        assert int(lens[i]) == (n if n < 0 else n + len(want))
    assert seen >= {0, 4} and ops.device_error() == 0
    # slots past 32 bits are none
    far = torch.full((1, 1), 1 << 29, dtype=torch.int32, device="cuda")
    got = ops.verify_drafts(drafts[:1], p[:1], q[:1], u[:1], u_last[:1], torch.zeros(1, dtype=torch.int32, device="cuda"),
                            far, block)
    assert int(got[1]) == 0
    # no table at all
    none = ops.verify_drafts(drafts[:2], p[:2], q[:2], u[:2], u_last[:2], before[1:3].clone(), tables[:2, :0], block)
    assert none[1].tolist() == [0, 0] and none[0].tolist() == [[-1] * (k + 1)] * 2


@pytest.mark.parametrize("all_windowed", [True, False])
def test_draft_decode_without_pages(all_windowed):
    """Steps while the lent pages run out, and at a table's end: rows without a page are not verified, no length
    counts a token that is not in the cache, and sequences go on when pages are lent, from the same token."""
    from test_gpu_draft_decode import _Model

    from vlcache_b200.engine.draft_decode import DraftDecode
    from vlcache_b200.engine.page_pool import PagePool
    from vlcache_b200.utils.context import reset_context, set_context
    import numpy as np
    ops = _ops()
    block, places, k, most = 32, 3, 3, 4
    model = _Model(11, all_windowed=all_windowed)
    pool = PagePool(60, block)
    model.caches(60, block)
    for layer in model.layers:   # what a recycled page holds
        layer.k_cache.fill_(3.0)
        layer.v_cache.fill_(30.0)
    window = 40 if all_windowed else 0
    d = DraftDecode(pool, places, most, k, window, 3 if window else 0)
    r = np.random.default_rng(9)
    histories = {0: [int(x) for x in r.integers(0, 97, 61)], 1: [int(x) for x in r.integers(0, 97, 95)],
                 2: [int(x) for x in r.integers(0, 97, 30)]}
    last = {}
    for place, tokens in histories.items():
        table, n = pool.allocate(pool.pages_for(len(tokens))), len(tokens)
        slots = torch.tensor([table[t // block] * block + t % block for t in range(n)], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        set_context(True, cu, cu, n, n, slots, None, None, cu_seqlens_q_host=[0, n], cu_seqlens_k_host=[0, n])
        last[place] = int(model(torch.tensor(tokens, device="cuda"), torch.arange(n, device="cuda"))[-1].argmax())
        d.admit(place, table, n)
    seen, errors = set(), set()
    for turn in range(250):
        if all(len(h) == most * block for h in histories.values()) and 0 in seen:
            break
        if turn in (6, 9, 30):
            assert d.lend(1)
        if turn == 40:
            assert d.lend(20)
        guess = torch.full((places, k + 1), -1, dtype=torch.int64)
        for p in histories:
            row = [last[p]]
            for _ in range(k):   # the right drafts, mostly
                best = int(model.plain(histories[p] + row)[-1].argmax())
                row.append(best if r.random() < 0.7 else int(r.integers(0, 97)))
            guess[p] = torch.tensor(row)
        tokens_in = guess.cuda()
        u = torch.tensor(r.random((places, k)) * 0.2, dtype=torch.float32, device="cuda")
        u_last = torch.tensor(r.random(places), dtype=torch.float32, device="cuda")
        positions = d.begin()
        tables = d.block_tables.tolist()
        probs = model(tokens_in.flatten(), positions).view(places, k + 1, -1)
        tokens, emitted = d.finish(tokens_in[:, 1:].contiguous(), probs, None, u, u_last)
        errors.add(ops.device_error())
        for p, h in histories.items():
            rows = _stored(tables[p], len(h), k + 1, block)
            seen.add(rows)
            want = model.plain(h + guess[p].tolist())[len(h):]
            # (an output's error as in the test of steps with pages: below 0.05)
            assert float((probs[p].double() - want)[:rows].abs().max() if rows else 0.0) < 0.05, (turn, p, rows)
            ds = [x if i + 1 < rows else -1 for i, x in enumerate(guess[p, 1:].tolist())]
            out = [] if rows == 0 else oracle.verify(ds, probs[p].cpu(), None, u[p].tolist(), float(u_last[p]))
            assert tokens[p].tolist() == out + [-1] * (k + 1 - len(out)) and int(emitted[p]) == len(out), (turn, p)
            if out:
                h += guess[p, :len(out)].tolist()
                last[p] = out[-1]
            assert int(d.context_lens[p]) == len(h) <= most * block
    assert 0 in seen and k + 1 in seen and len(seen) > 2 and errors - {0} <= {102, 105} and len(errors) > 1
    assert all(len(h) == most * block for h in histories.values())   # and every table ended full
    for p in histories:
        d.retire(p)
    d.settle()
    assert pool.num_free == 60 and pool.refs == [0] * 60
    reset_context()


def test_one_token_steps_to_the_table_end():
    """Steps without drafts over layers without a window (the one-token decode), up to and past a full table."""
    from test_gpu_draft_decode import _Model

    from vlcache_b200.engine.draft_decode import DraftDecode
    from vlcache_b200.engine.page_pool import PagePool
    from vlcache_b200.layers.attention import Attention
    from vlcache_b200.utils.context import reset_context, set_context
    import numpy as np
    ops = _ops()
    block, places = 256, 2
    model = _Model(5)
    model.layers = [Attention(model.heads, D, 0.1, model.kv_heads) for _ in range(2)]
    pool = PagePool(6, block)
    model.caches(6, block)
    d = DraftDecode(pool, places, 2, 0)
    r = np.random.default_rng(2)
    histories = {0: [int(x) for x in r.integers(0, 97, 505)], 1: [int(x) for x in r.integers(0, 97, 254)]}
    last = {}
    for place, tokens in histories.items():
        table, n = pool.allocate(pool.pages_for(len(tokens))), len(tokens)
        slots = torch.tensor([table[t // block] * block + t % block for t in range(n)], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        set_context(True, cu, cu, n, n, slots, None, None, cu_seqlens_q_host=[0, n], cu_seqlens_k_host=[0, n])
        last[place] = int(model(torch.tensor(tokens, device="cuda"), torch.arange(n, device="cuda"))[-1].argmax())
        d.admit(place, table, n)
    none = torch.zeros(places, 0, device="cuda")
    for turn in range(12):
        if turn == 5:
            assert d.lend(1)   # place 1 stands at 256 tokens until now
        positions = d.begin()
        probs = model(torch.tensor([last[0], last[1]], device="cuda"), positions).view(places, 1, -1)
        tokens, emitted = d.finish(none.long(), probs, None, none, torch.full((places,), 0.5, device="cuda"))
        assert ops.device_error() in (0, 102, 104, 105)
        for p, h in histories.items():
            stored = len(h) < 512 and (p == 0 or len(h) < 256 or turn >= 5)
            assert int(emitted[p]) == int(stored), (turn, p)
            if stored:
                want = model.plain(h + [last[p]])[-1]
                assert float((probs[p, 0].double() - want).abs().max()) < 0.05   # (as in the test of steps with pages)
                h.append(last[p])
                last[p] = int(tokens[p, 0])
            assert int(d.context_lens[p]) == len(h)
    assert len(histories[0]) == 512 and len(histories[1]) == 256 + 7
    reset_context()


def test_draft_decode_over_a_compacted_pool():
    """Tables and free list through the page map: lent pages and sequences' are the pool's still, each once."""
    from vlcache_b200.engine.draft_decode import DraftDecode
    from vlcache_b200.engine.page_pool import PagePool
    from vlcache_b200.utils.context import reset_context
    ops = _ops()
    pool = PagePool(30, 32)
    d = DraftDecode(pool, 3, 6, 2)
    filler = pool.allocate(9)
    assert d.lend(4)
    tables = {0: pool.allocate(3), 2: pool.allocate(2)}
    d.admit(0, tables[0], 95)   # the next step takes a page
    d.admit(2, tables[2], 33)
    pool.free(filler)
    src, dst, page_map = pool.compact()
    assert src and max(dst) < 9
    on_device = torch.from_numpy(page_map).cuda()
    for t in (d.block_tables, d.free_pages.view(1, -1)):
        ops.remap_block_tables(t, on_device)
    assert ops.device_error() == 0
    d.begin()
    assert ops.device_error() == 0 and int(d.num_free) == 3
    held = [p for row in d.block_tables.tolist() for p in row if p >= 0] + d.free_pages[:3].tolist()
    assert sorted(held) == list(range(9)) and all(pool.refs[p] == 1 for p in held)
    assert d.block_tables[0, :3].tolist() == [int(page_map[p]) for p in tables[0]]
    for p in (0, 2):
        d.retire(p)
    d.settle()
    assert pool.num_free == 30 and pool.refs == [0] * 30
    reset_context()


# ------------------------------------------------------------------ one call behind another
@pytest.mark.parametrize("rows,window", [(700, 0), (700, 100), (20000, 0), (20000, 1000)])   # one launch of metadata, and two
def test_prefill_reads_tables_of_the_step_before(rows, window):
    """Block tables that vlc_step_metadata has just written, by the prefill launched directly behind it, which starts
    before that kernel has ended."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(rows)
    seqs, block = 4, 256
    each = rows // seqs
    held = (each + block - 1) // block
    pages = 2 * seqs * held
    k_cache, v_cache = (torch.randn(pages, block, 2, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(seqs * each, 16, D, generator=g, device="cuda").to(torch.bfloat16)
    cu = [i * each for i in range(seqs + 1)]
    plan = ops.build_prefill_plan(cu, cu, 16, 2, device="cuda", window=window or None)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, new = torch.zeros(seqs, **i32), torch.full((seqs,), each, **i32)
    tables = torch.full((seqs, held), -1, **i32)
    out = torch.empty_like(q)
    workspace = torch.empty(max(1, plan.workspace_bytes), dtype=torch.uint8, device="cuda")
    for turn in range(6):
        free = torch.randperm(pages, generator=g, device="cuda").int()
        count = torch.tensor([pages], **i32)
        tables.fill_(-1)   # a stale entry would be an error, or another turn's page
        torch.cuda.synchronize()
        ops.step_metadata(lens, new, tables, free, count, block, seqs * each)
        ops.prefill_attention(q, k_cache, v_cache, tables, plan, 0.1, out=out, workspace=workspace)
        got = out.clone()
        torch.cuda.synchronize()
        assert ops.device_error() == 0 and int((tables < 0).sum()) == 0
        assert torch.equal(got, ops.prefill_attention(q, k_cache, v_cache, tables, plan, 0.1)), turn


# ------------------------------------------------------------------ windowed prefill over a 4-bit cache
@pytest.mark.parametrize("window,sinks", [(100, 0), (200, 4), (64, 130), (1, 0), (333, 64)])
def test_prefill_window_over_a_4_bit_cache_without_hidden_pages(window, sinks):
    """Pages that no row sees are not read: entries of -1 change nothing and record nothing; pages that rows see are."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(window)
    block, seqs = 64, [(50, 1500), (0, 400), (130, 130), (1, 700), (300, 2000)]
    new, lens = [a for a, _ in seqs], [b for _, b in seqs]
    cu_q, cu_k = ([sum(x[:i]) for i in range(len(x) + 1)] for x in (new, lens))
    widths = [(n + block - 1) // block for n in lens]
    pages = sum(widths)
    k4, v4 = (torch.randint(0, 256, (pages, 2, block * 72), generator=g, device="cuda", dtype=torch.int32)
              .to(torch.uint8) for _ in range(2))
    k, v = (torch.randn(pages * block, 2, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    ops.store_kvcache_fp4(k, v, k4, v4, torch.arange(pages * block, dtype=torch.int32, device="cuda"))
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    tables = torch.full((len(seqs), max(widths)), -1, dtype=torch.int32, device="cuda")
    for i, w in enumerate(widths):
        tables[i, :w] = torch.tensor([order.pop() for _ in range(w)], dtype=torch.int32)
    q = torch.randn(sum(new), 16, D, generator=g, device="cuda").to(torch.bfloat16)
    cu = torch.tensor(cu_k, dtype=torch.int32, device="cuda")
    plan = ops.build_prefill_plan(cu_q, cu_k, 16, 2, device="cuda", window=window, sinks=sinks)
    want = ops.prefill_attention_fp4(q, k4, v4, tables, cu, plan, 0.1)
    kb, vb = ops.gather_kvcache_fp4(k4, v4, tables, cu, cu_k[-1])
    assert torch.equal(want, ops.prefill_attention(q, kb, vb, None, plan, 0.1)) and ops.device_error() == 0
    gone = 0
    for i, (n, m) in enumerate(seqs):
        for page in range(widths[i]):
            if n == 0 or (page * block >= sinks and (page + 1) * block <= m - n - window + 1):
                tables[i, page] = -1
                gone += 1
    assert gone > 20
    # (what the workspace holds where nothing is read is not seen)
    workspace = torch.full((ops.prefill_fp4_workspace_bytes(plan, 2),), 255, dtype=torch.uint8, device="cuda")
    got = ops.prefill_attention_fp4(q, k4, v4, tables, cu, plan, 0.1, workspace=workspace)
    assert torch.equal(got, want) and ops.device_error() == 0
    tables[4, widths[4] - 1] = -1   # one that its rows see
    ops.prefill_attention_fp4(q, k4, v4, tables, cu, plan, 0.1, workspace=workspace)
    assert ops.device_error() == 102


# ------------------------------------------------------------------ windowed prefill, to the bound of 32-bit parts
STEP = 2.0 ** -8   # half a step of bf16, relative


def _prefill_cases():
    from test_gpu_draft_decode import PREFILL
    return [(*c, D) for c in PREFILL] + [(16, 2, 256, 40, 3, [(300, 300), (9, 5000)], d) for d in (80, 96, 112)] + \
        [(16, 2, 256, 3000, 4, [(48, 9000)], D), (28, 4, 256, 6000, 300, [(20, 12000), (7, 30)], D)]


@pytest.mark.parametrize("case", _prefill_cases(), ids=lambda c: "-".join(map(str, (c[0], c[1], c[3], c[4], c[6]))))
def test_prefill_window_keeps_parts_in_32_bits(case):
    """P's rounding (STEP of itself, sum p |v| <= rms) and the output's (STEP of it) are the only ones, also where a
    window hides keys and tiles are split: 2^-12 for what fp32 scores, sums and parts are off by."""
    ops = _ops()
    heads, kv_heads, _, window, sinks, seqs, head_dim = case
    g = torch.Generator(device="cuda").manual_seed(heads + window + head_dim)
    cu_q, cu_k = ([sum(x[:i]) for i in range(len(x) + 1)] for x in ([a for a, _ in seqs], [b for _, b in seqs]))
    q = (1.5 * torch.randn(cu_q[-1], heads, head_dim, generator=g, device="cuda")).to(torch.bfloat16)
    k, v = (torch.randn(cu_k[-1], kv_heads, head_dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    plan = ops.build_prefill_plan(cu_q, cu_k, heads, kv_heads, head_dim, device="cuda", window=window, sinks=sinks)
    assert plan.num_parts > 0 or window < 3000
    got = ops.prefill_attention(q, k, v, None, plan, 0.09)
    assert ops.device_error() == 0
    for i, (n, m) in enumerate(seqs):
        want, rms = oracle.attention(q[cu_q[i]:cu_q[i + 1]].double(), k[cu_k[i]:cu_k[i + 1]].double(),
                                     v[cu_k[i]:cu_k[i + 1]].double(), torch.arange(m - n, m, device="cuda"), window, sinks,
                                     0.09)
        off = (got[cu_q[i]:cu_q[i + 1]].double() - want).abs()
        assert bool((off <= (STEP + 2.0 ** -12) * (rms + want.abs()) + 1e-30).all()), i


# ------------------------------------------------------------------ positions of several axes
def test_draft_decode_positions_of_several_axes():
    """A step's rows behind images: each place's offset on the device makes [axes, rows] of the positions."""
    from vlcache_b200.engine.draft_decode import DraftDecode
    from vlcache_b200.engine.page_pool import PagePool
    from vlcache_b200.layers.rotary_embedding import get_mrope
    from vlcache_b200.utils.context import reset_context
    ops = _ops()
    pool = PagePool(12, 32)
    d = DraftDecode(pool, 3, 4, 2)
    assert d.lend(4)
    d.admit(0, pool.allocate(2), 50)
    d.admit(2, pool.allocate(1), 9)
    offsets = torch.tensor([-30, 0, 7], device="cuda")   # (idle places: 0)
    positions = d.begin()
    axes = (positions.view(3, -1) + offsets.view(-1, 1)).view(1, -1).expand(3, -1)
    assert axes.tolist() == [[20, 21, 22, 0, 0, 0, 16, 17, 18]] * 3
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.randn(9, h, D, generator=g, device="cuda").to(torch.bfloat16) for h in (4, 2))
    rot = get_mrope(D, D, 64, 1e6).cuda()
    for a, b in zip(rot(axes, q, k), rot(axes.contiguous(), q, k)):
        assert torch.equal(a, b)
    assert ops.device_error() == 0
    reset_context()
