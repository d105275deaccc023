"""Host side of a decode step with drafted tokens over a windowed cache: windowed prefill plans, the 64-bit
definitions, the bookkeeping of pages and the refusals, none of which needs a GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import draft_decode as oracle


# ------------------------------------------------------------------ the definitions
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (3, 0), (3, 2), (100, 4), (5, 100)])
def test_oracle_mask_row_by_row(window, sinks):
    seen = oracle.visible(torch.arange(0, 12), 12, window, sinks)
    for t in range(12):
        keys = {j for j in range(t + 1) if not window or j > t - window or j < sinks}
        assert set(torch.nonzero(seen[t]).flatten().tolist()) == keys


def test_oracle_attention_is_softmax():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 128, generator=g, dtype=torch.float64) for n, h in ((3, 4), (9, 2), (9, 2)))
    out, _ = oracle.attention(q, k, v, torch.tensor([5, 6, -1]), 0, 0, 0.1)
    want = torch.softmax(q[0, 3] @ k[:6, 1].T * 0.1, -1) @ v[:6, 1]
    assert torch.allclose(out[0, 3], want) and torch.equal(out[2], torch.zeros(4, 128, dtype=torch.float64))


def test_oracle_verify_samples_the_distributions():
    """Over many draws the first emitted token follows the target's probabilities, whatever the draft's are."""
    r = np.random.default_rng(0)
    p = torch.tensor([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]], dtype=torch.float32)
    q = torch.tensor([[0.2, 0.2, 0.6]], dtype=torch.float32)
    n, count = 6000, [0, 0, 0]
    for _ in range(n):
        d = int(r.choice(3, p=[0.2, 0.2, 0.6]))
        count[oracle.verify([d], p, q, [float(np.float32(r.random()))], float(np.float32(r.random())))[0]] += 1
    # a count of n draws at probability x is off by 5 deviations once in two million
    for c, x in zip(count, (0.5, 0.3, 0.2)):
        assert abs(c - n * x) < 5 * math.sqrt(n * x * (1 - x))


# ------------------------------------------------------------------ windowed plans
def _plan_blocks(plan):
    """(query token, KV head, key block) that each unit's tiles run over, and the plan's fields."""
    h = plan.host
    units = h[int(h[13]):int(h[13]) + int(h[3]) * 17].reshape(-1, 17)
    window, sinks = int(h[22]), int(h[23])
    out = {}
    for u in units.tolist():
        low = u[13]
        begin = max(0, low - window + 1) // 128 if window else 0
        first = min(begin, -(-sinks // 128))
        tiles = [(u[7], u[8], u[9], u[2], u[3])] + ([(u[11], u[12], u[13], u[2], u[15])] if u[12] > 0 else [])
        for q0, n, pos, b0, b1 in tiles:
            assert not window or pos >= low
            for b in range(b0, b1):
                block = b if b < first else b + begin - first
                for t in range(n):
                    key = (q0 + t, u[1], block)
                    assert key not in out
                    out[key] = pos + t
    return out, window, sinks


@pytest.mark.parametrize("heads,kv_heads", [(16, 2), (28, 4), (8, 8), (12, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (127, 4), (128, 128), (129, 129), (700, 4), (64, 1000)])
def test_window_plan_covers_what_rows_see(cuda_lib, heads, kv_heads, window, sinks):
    """Every visible key of every row is in exactly one of its units' blocks, blocks are never run twice, and
    those that no row of a pair of tiles sees are skipped."""
    from vlcache_b200 import ops
    new, lens = [300, 1, 0, 77], [300, 900, 40, 2100]
    cu_q, cu_k = np.cumsum([0] + new), np.cumsum([0] + lens)
    plan = ops.build_prefill_plan(cu_q, cu_k, heads, kv_heads, num_sms=16, window=window, sinks=sinks)
    blocks, w, s = _plan_blocks(plan)
    assert (w, s) == (window, sinks)
    tile = 128 // (heads // kv_heads)
    for i, (n, m) in enumerate(zip(new, lens)):
        for r in range(n):
            t = m - n + r
            seen = {j // 128 for j in range(t + 1) if j > t - window or j < sinks}
            for g in range(kv_heads):
                run = {b for b in range(-(-m // 128)) if (cu_q[i] + r, g, b) in blocks}
                assert seen <= run
                # of a pair of tiles (2 tile rows) nothing before its first row's window is run, but sinks
                low = max(0, t - 2 * tile + 2 - window)
                assert all(b * 128 < sinks or (b + 1) * 128 > low for b in run)
    assert all(blocks[k] == lens[np.searchsorted(cu_q, k[0], side="right") - 1]
               - new[np.searchsorted(cu_q, k[0], side="right") - 1]
               + k[0] - cu_q[np.searchsorted(cu_q, k[0], side="right") - 1] for k in blocks)


def test_window_that_hides_nothing_is_the_plan_without(cuda_lib):
    from vlcache_b200 import ops
    a = ops.build_prefill_plan([0, 700], [0, 900], 16, 2, num_sms=16, window=900, sinks=3)
    b = ops.build_prefill_plan([0, 700], [0, 900], 16, 2, num_sms=16)
    assert np.array_equal(a.host, b.host) and a.workspace_bytes == b.workspace_bytes
    c = ops.build_prefill_plan([0, 20], [0, 9000], 16, 2, num_sms=148, window=4000)
    assert c.num_parts > 0 and c.workspace_bytes == c.num_parts * 128 * (128 * 4 + 8)   # parts in fp32


def test_window_of_0_is_the_plan_without_but_for_split_tiles(cuda_lib):
    from vlcache_b200 import ops
    a = ops.build_prefill_plan([0, 700], [0, 900], 16, 2, num_sms=16, window=0)
    b = ops.build_prefill_plan([0, 700], [0, 900], 16, 2, num_sms=16)
    assert a.num_parts == 0 and np.array_equal(a.host, b.host)
    for window in (0, 9000):
        a = ops.build_prefill_plan([0, 20], [0, 9000], 16, 2, num_sms=148, window=window)
        b = ops.build_prefill_plan([0, 20], [0, 9000], 16, 2, num_sms=148)
        assert a.num_parts == b.num_parts > 0 and a.num_units == b.num_units
        assert a.workspace_bytes == a.num_parts * 128 * (128 * 4 + 8)
        assert b.workspace_bytes == b.num_parts * 128 * (128 * 2 + 8)   # bf16, as plans without a window were
    a = ops.build_prefill_plan([0, 20], [0, 9000], 16, 2, num_sms=148, window=0, causal=False)
    b = ops.build_prefill_plan([0, 20], [0, 9000], 16, 2, num_sms=148, causal=False)
    assert np.array_equal(a.host, b.host)


def test_window_plan_refusals(cuda_lib):
    from vlcache_b200 import ops
    from vlcache_b200._lib import VLCError
    for kw in (dict(window=-1), dict(window=5, sinks=-1), dict(window=(1 << 30) + 1), dict(window=5, causal=False)):
        with pytest.raises(VLCError):
            ops.build_prefill_plan([0, 64], [0, 64], 16, 2, num_sms=8, **kw)


# ------------------------------------------------------------------ refusals before a launch
def test_c_abi_refuses_before_a_launch(cuda_lib):
    one = ctypes.c_void_p(64)   # never dereferenced: validation fails first

    def decode(q=one, stride=2048, seqs=1, tokens=1, heads=16, pages=4, block=256, kv=2, d=128, ts=4, tw=4, bound=1000,
               window=0, sinks=0, scale=1.0, out=one, ws=None, nbytes=0):
        return cuda_lib.vlc_decode_attn_window(q, stride, seqs, tokens, heads, one, one, pages, block, kv, d, one, ts,
                                               tw, one, bound, window, sinks, scale, out, stride, ws, nbytes, None)
    assert decode(seqs=-1) == 2 and decode(tokens=0) == 2 and decode(heads=15) == 2 and decode(pages=0) == 2
    assert decode(window=-1) == 2 and decode(sinks=-1) == 2 and decode(bound=-1) == 2 and decode(bound=(1 << 30) + 1) == 2
    assert decode(seqs=65536) == 2 and decode(tw=-1) == 2
    assert decode(d=64) == 5 and decode(block=48) == 5 and decode(block=0) == 5 and decode(tokens=17) == 5
    assert decode(scale=math.inf) == 5 and decode(scale=math.nan) == 5
    assert decode(q=None) == 1 and decode(out=None) == 1
    assert decode(stride=2044) == 3 and decode(stride=1024) == 3 and decode(ts=3) == 3
    assert decode(q=ctypes.c_void_p(72)) == 4
    assert decode(seqs=200, bound=100000) == 6 and decode(seqs=200, bound=100000, ws=one, nbytes=64) == 6
    assert decode(seqs=0) == 0

    def step(lens=one, new=one, seqs=3, tables=one, ts=4, width=4, block=256, window=0, sinks=0, pages=one, capacity=9,
             free=one, rows=5, cu=one):
        return cuda_lib.vlc_step_metadata(lens, new, seqs, tables, ts, width, block, window, sinks, pages, capacity, free,
                                          one, one, rows, cu, one, one, None)
    assert step(seqs=-1) == 2 and step(block=0) == 2 and step(window=-1) == 2 and step(rows=-1) == 2
    assert step(capacity=-1) == 2 and step(seqs=65535, width=1 << 20, ts=1 << 20) == 2
    assert step(lens=None) == 1 and step(tables=None) == 1 and step(pages=None) == 1 and step(free=None) == 1
    assert step(cu=None) == 1 and step(ts=3) == 3

    def verify(drafts=one, seqs=1, n=2, p=one, q=one, vocab=100, dtype=0, u=one, last=one):
        return cuda_lib.vlc_verify_drafts(drafts, n, seqs, n, p, 300, 100, q, 200, 100, vocab, dtype, u, n, last, one, one,
                                          None, None)
    assert verify(seqs=-1) == 2 and verify(n=-1) == 2 and verify(vocab=0) == 2
    assert verify(n=32) == 5 and verify(vocab=(1 << 18) + 1) == 5 and verify(dtype=3) == 5
    assert verify(drafts=None) == 1 and verify(p=None) == 1 and verify(u=None) == 1 and verify(last=None) == 1
    assert verify(seqs=0) == 0


def test_workspace_sizes(cuda_lib):
    from vlcache_b200 import ops
    assert ops.decode_window_workspace_bytes(1, 1, 16, 2, 1000) == 0                  # one launch, no parts
    small, large = (ops.decode_window_workspace_bytes(64, n, 28, 4, 9000, 4096, 4) for n in (1, 5))
    assert 0 < small < large
    for bad in ((64, 0, 28, 4, 9000), (64, 1, 27, 4, 9000), (64, 1, 28, 4, -1), (64, 19, 28, 4, 9000), (0, 1, 28, 4, 9)):
        assert ops.decode_window_workspace_bytes(*bad) == 0


def _decode_args(**kw):
    bf16 = dict(dtype=torch.bfloat16)
    a = dict(q=torch.zeros(3, 2, 16, 128, **bf16), k_cache=torch.zeros(4, 64, 2, 128, **bf16),
             v_cache=torch.zeros(4, 64, 2, 128, **bf16), block_tables=torch.zeros(3, 2, dtype=torch.int32),
             context_lens=torch.ones(3, dtype=torch.int32), max_context_len=100, softmax_scale=0.1)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,what", [
    (dict(q=torch.zeros(3, 2, 16, 128)), "q: bf16"),
    (dict(q=torch.zeros(16, 128, dtype=torch.bfloat16)), "q: bf16"),
    (dict(q=torch.zeros(3, 2, 128, 16, dtype=torch.bfloat16).transpose(2, 3)), "contiguous"),
    (dict(q=torch.zeros(2, 3, 16, 128, dtype=torch.bfloat16).transpose(0, 1)), "one token stride"),
    (dict(k_cache=torch.zeros(4, 64, 2, 128)), "k_cache"),
    (dict(v_cache=torch.zeros(4, 32, 2, 128, dtype=torch.bfloat16)), "k_cache"),
    (dict(k_cache=torch.zeros(4, 2, 64, 128, dtype=torch.bfloat16).transpose(1, 2)), "k_cache"),
    (dict(block_tables=torch.zeros(2, 2, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(3, 2)), "block_tables"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int32).T), "rows must be contiguous"),
    (dict(context_lens=torch.ones(2, dtype=torch.int32)), "context_lens"),
    (dict(context_lens=torch.ones(3)), "context_lens"),
    (dict(max_context_len=-1), "max_context_len"), (dict(max_context_len=(1 << 30) + 1), "max_context_len"),
    (dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(window=1 << 40), "window"),
    (dict(out=torch.zeros(3, 16, 128, dtype=torch.bfloat16)), "out"),
    (dict(out=torch.zeros(3, 2, 16, 128)), "out"),
    (dict(workspace=torch.zeros(64, 2, dtype=torch.uint8).T), "workspace"),
    ({}, "CUDA tensors only"),
])
def test_decode_refusals(cuda_lib, change, what):
    from vlcache_b200 import ops
    with pytest.raises(ValueError, match=what):
        ops.decode_attention_window(**_decode_args(**change))


def test_decode_refuses_other_types(cuda_lib):
    from vlcache_b200 import ops
    with pytest.raises(TypeError, match="q must be a tensor"):
        ops.decode_attention_window(**_decode_args(q=[1.0]))
    with pytest.raises(TypeError):
        ops.decode_attention_window(**_decode_args(softmax_scale="0.1"))
    with pytest.raises((TypeError, ValueError)):
        ops.decode_attention_window(**_decode_args(max_context_len="many"))


def _step_args(**kw):
    i32 = dict(dtype=torch.int32)
    a = dict(context_lens=torch.ones(3, **i32), new_lens=torch.ones(3, **i32), block_tables=torch.zeros(3, 4, **i32),
             free_pages=torch.zeros(9, **i32), num_free=torch.zeros(1, **i32), block_size=256, total_rows=3)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,what", [
    (dict(context_lens=torch.ones(3)), "context_lens"), (dict(new_lens=torch.ones(2, dtype=torch.int32)), "new_lens"),
    (dict(new_lens=torch.ones(6, dtype=torch.int32)[::2]), "new_lens"),
    (dict(block_tables=torch.zeros(2, 4, dtype=torch.int32)), "block_tables"),
    (dict(free_pages=torch.zeros(9)), "free_pages"), (dict(free_pages=torch.zeros(18, dtype=torch.int32)[::2]), "free_pages"),
    (dict(num_free=torch.zeros(2, dtype=torch.int32)), "num_free"), (dict(block_size=0), "block_size"),
    (dict(total_rows=-1), "total_rows"), (dict(window=-1), "window"), (dict(sinks=1 << 31), "sinks"),
    ({}, "CUDA tensors only"),
])
def test_step_refusals(cuda_lib, change, what):
    from vlcache_b200 import ops
    with pytest.raises(ValueError, match=what):
        ops.step_metadata(**_step_args(**change))


def _verify_args(**kw):
    a = dict(drafts=torch.zeros(3, 2, dtype=torch.int64), target_probs=torch.zeros(3, 3, 50),
             draft_probs=torch.zeros(3, 2, 50), u=torch.zeros(3, 2), u_last=torch.zeros(3))
    a.update(kw)
    return a


@pytest.mark.parametrize("change,what", [
    (dict(drafts=torch.zeros(3, 2, dtype=torch.int32)), "drafts"), (dict(drafts=torch.zeros(6, dtype=torch.int64)), "drafts"),
    (dict(drafts=torch.zeros(2, 3, dtype=torch.int64).T), "drafts"),
    (dict(drafts=torch.zeros(3, 32, dtype=torch.int64)), "31 drafts"),
    (dict(target_probs=torch.zeros(3, 2, 50)), "target_probs"),
    (dict(target_probs=torch.zeros(3, 3, 50, dtype=torch.float64)), "target_probs"),
    (dict(target_probs=torch.zeros(3, 3, 0), draft_probs=None), "vocabulary"),
    (dict(target_probs=torch.zeros(3, 3, 100)[..., ::2]), "target_probs"),
    (dict(target_probs=torch.zeros(1, 1, 1).expand(3, 3, (1 << 18) + 1), draft_probs=None), "vocabulary"),
    (dict(draft_probs=torch.zeros(3, 3, 50)), "draft_probs"), (dict(draft_probs=torch.zeros(3, 2, 51)), "draft_probs"),
    (dict(draft_probs=torch.zeros(3, 2, 50, dtype=torch.bfloat16)), "draft_probs"),
    (dict(u=torch.zeros(3, 3)), "u: fp32"), (dict(u=torch.zeros(3, 2, dtype=torch.float64)), "u: fp32"),
    (dict(u_last=torch.zeros(2)), "u_last"), (dict(u_last=torch.zeros(6)[::2]), "u_last"),
    (dict(context_lens=torch.zeros(2, dtype=torch.int32)), "context_lens"),
    ({}, "CUDA tensors only"),
])
def test_verify_refusals(cuda_lib, change, what):
    from vlcache_b200 import ops
    with pytest.raises(ValueError, match=what):
        ops.verify_drafts(**_verify_args(**change))


# ------------------------------------------------------------------ the engine's bookkeeping
def _decoder(pages=20, **kw):
    from vlcache_b200.engine.draft_decode import DraftDecode
    from vlcache_b200.engine.page_pool import PagePool
    pool = PagePool(pages, 32)
    return pool, DraftDecode(pool, **{**dict(places=3, max_pages=6, num_drafts=2, device="cpu"), **kw})


def test_draft_decode_pages_come_and_go():
    pool, d = _decoder()
    assert d.lend(5) and pool.num_free == 15 and int(d.num_free) == 5 and d.free_pages[:5].tolist() == [0, 1, 2, 3, 4]
    assert d.lend(0) and not d.lend(16) and int(d.num_free) == 5 and pool.num_free == 15
    table = pool.allocate(2)
    d.admit(1, table, 40)
    assert d.context_lens.tolist() == [-1, 40, -1] and d.block_tables[1].tolist() == table + [-1] * 4
    assert d.retire(1) == 40 and pool.num_free == 15 and d.context_lens.tolist() == [-1] * 3
    d.settle()
    assert pool.num_free == 20 and int(d.num_free) == 0 and pool.refs == [0] * 20


def test_draft_decode_refusals():
    from vlcache_b200.engine.draft_decode import DraftDecode
    from vlcache_b200.engine.page_pool import PagePool
    pool, d = _decoder()
    for bad in (dict(places=0), dict(max_pages=0), dict(num_drafts=-1)):
        with pytest.raises(ValueError):
            _decoder(**bad)
    with pytest.raises(ValueError, match="multiple of 32"):
        DraftDecode(PagePool(4, 48), 1, 2, 1, device="cpu")
    table = pool.allocate(2)
    for place, t, n, what in ((3, table, 1, "outside"), (0, table, 65, "does not hold"), (0, table, -1, "does not hold"),
                              (0, table + pool.allocate(5), 1, "at most"), (0, table + [table[0]], 1, "twice"),
                              (0, [19], 1, "not this table's alone"), (0, [-1], 1, "not this table's alone")):
        with pytest.raises(ValueError, match=what):
            d.admit(place, t, n)
    fork, _ = pool.fork(table, 64)
    with pytest.raises(ValueError, match="not this table's alone"):   # shared pages would be given back twice
        d.admit(0, table, 64)
    pool.free(fork)
    d.admit(0, table, 64)
    with pytest.raises(ValueError, match="taken"):
        d.admit(0, pool.allocate(1), 1)
    with pytest.raises(ValueError, match="idle"):
        d.retire(1)
    with pytest.raises(ValueError, match="drafts"):
        d.finish(torch.zeros(3, 3, dtype=torch.int64), None, None, None, None)


def test_attention_layer_arguments():
    from vlcache_b200.layers.attention import Attention
    for kw in (dict(sliding_window=0), dict(sliding_window=-5), dict(sliding_window=5, num_sinks=-1)):
        with pytest.raises(ValueError):
            Attention(16, 128, 0.1, 2, **kw)
    plain, windowed = Attention(16, 128, 0.1, 2, None, 4), Attention(16, 128, 0.1, 2, 100, 4)
    assert (plain.sliding_window, plain.num_sinks) == (0, 0) and (windowed.sliding_window, windowed.num_sinks) == (100, 4)
