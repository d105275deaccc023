"""Host side of a decode step with drafted tokens, further: refusals and bookkeeping, none of which needs a GPU."""
import ctypes

import pytest
import torch


# ------------------------------------------------------------------ verification with block tables
def _verify_args(**kw):
    a = dict(drafts=torch.zeros(3, 2, dtype=torch.int64), target_probs=torch.zeros(3, 3, 50), draft_probs=None,
             u=torch.zeros(3, 2), u_last=torch.zeros(3), context_lens=torch.zeros(3, dtype=torch.int32),
             block_tables=torch.zeros(3, 4, dtype=torch.int32), block_size=32)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,what", [
    (dict(context_lens=None), "with context_lens"), (dict(block_tables=torch.zeros(2, 4, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(3, 4)), "block_tables"),
    (dict(block_tables=torch.zeros(4, 3, dtype=torch.int32).T), "rows must be contiguous"),
    (dict(block_size=0), "block_size"), (dict(block_size=1 << 31), "block_size"), ({}, "CUDA tensors only"),
    (dict(block_tables=None), "block_size: with block_tables"),   # rows that it was to leave out would count
])
def test_verify_refuses_tables(cuda_lib, change, what):
    from vlcache_b200 import ops
    with pytest.raises(ValueError, match=what):
        ops.verify_drafts(**_verify_args(**change))


def test_verify_takes_a_block_size_with_tables(cuda_lib):
    from vlcache_b200 import ops
    with pytest.raises(TypeError):
        ops.verify_drafts(**_verify_args(block_size=None))


def test_c_abi_verify_refuses_tables(cuda_lib):
    one = ctypes.c_void_p(64)   # never dereferenced: validation fails first

    def verify(seqs=2, lens=one, tables=one, stride=4, width=4, block=32, vocab=100):
        return cuda_lib.vlc_verify_stored_drafts(one, 2, seqs, 2, one, 300, 100, one, 200, 100, vocab, 0, one, 2, one, one,
                                                 one, lens, tables, stride, width, block, None)
    assert verify(block=0) == 2 and verify(width=-1) == 2 and verify(vocab=0) == 2
    assert verify(lens=None) == 1 and verify(tables=None) == 1 and verify(stride=3) == 3
    assert verify(seqs=0) == 0 and verify(seqs=0, lens=None, tables=None) == 0


# ------------------------------------------------------------------ waits that give up
def _source(name):
    from pathlib import Path

    import vlcache_b200
    return (Path(vlcache_b200.__file__).parent / "csrc" / name).read_text()


def test_wide_decode_warps_give_up_together():
    """A wait that gives up ends a role for all lanes of a warp or for none: lanes that left alone would be waited for by
    the others at their next vote, for ever.  Only the products' role, which is one lane, leaves by itself; the softmax
    warps, whose barriers need all of them, never leave."""
    import re
    src = _source("decode_window_wide.cu")
    kernel = src[src.index("window_decode_wide_kernel(const"):src.index("static int launch(")]
    roles = re.split(r"  // -{20,} (?=K and V copies|products|Q:|softmax)", kernel)
    assert len(roles) == 5
    copies, products, queries, softmax = roles[1:]
    leaves = r"!wait\(|= wait\(|return wait\("   # something depends on a lane's own result
    assert re.search(r"empty_now = .*\|\| wait\(.*\n.*\n *if \(!__all_sync\(0xffffffffu, empty_now\)\) return false;", copies)
    assert not re.search(leaves, copies)
    assert "!warp_wait(" in queries and not re.search(leaves, queries)
    assert "if (lane == 0 && count > 0)" in products and "!wait(" in products
    assert not re.search(leaves, softmax) and "break;" not in softmax and "return;" not in softmax
    common = _source("common.cuh")
    helper = common[common.index("bool warp_wait_or_abort("):]
    assert "__all_sync(0xffffffffu, wait_or_abort(" in helper[:helper.index("}")]


def test_prefill_softmax_warps_never_leave_a_wait():
    """The prefill's softmax warps meet at warp and named barriers: none of them leaves its role where a wait gave up.
    The copies' roles give theirs in flight more time."""
    import re
    src = _source("prefill_attn.cu")
    kernels = re.split(r"__global__ void", src)[1:3]
    for kernel in kernels:
        roles = re.split(r"  // -{20,} (?=Q producer|K/V producer|MMA issuer|softmax)", kernel)
        assert len(roles) == 5
        softmax = roles[4]
        assert softmax.count("wait_or_abort(") == 3
        assert not re.search(r"!\s*wait_or_abort\(|return wait_or_abort\(|\bok\b|\bbreak;", softmax)
        assert "drain_ring(bars.q_full" in roles[1]
        assert "drain_ring(bars.k_full" in roles[2] and "drain_ring(bars.v_full" in roles[2]


def test_projection_epilogues_never_leave_a_wait():
    """The projections' epilogue warps meet at named barriers and take tickets that the next launch relies on."""
    import re
    src = _source("gemm.cu")
    epilogues = re.findall(r"  // -{20,} epilogue \(warps 2-5.*?\n  __syncthreads\(\);", src, flags=re.S)
    assert len(epilogues) == 2
    for role in epilogues:
        assert role.count("wait_or_abort(") == 1 and not re.search(r"!\s*wait_or_abort\(|\bbreak;", role)
    assert src.count("drain_ring(full, it, ") == 2


# ------------------------------------------------------------------ windowed plans
def test_windowed_plan_holds_first_keys(cuda_lib):
    from vlcache_b200 import ops
    cu_q, cu_k = [0, 5, 5, 300, 301], [0, 1000, 1400, 1695, 1700]
    plan = ops.build_prefill_plan(cu_q, cu_k, 16, 2, num_sms=8, window=100, sinks=4)
    assert plan.host[plan.lows_at:].tolist() == [1000 - 5 - 99, -1, 0, 0] and plan.lows_at == int(plan.host[15])
    assert ops.build_prefill_plan(cu_q, cu_k, 16, 2, num_sms=8).lows_at is None
    hides_nothing = ops.build_prefill_plan([0, 20], [0, 9000], 16, 2, num_sms=148, window=0)   # split: parts in 32 bits
    assert hides_nothing.host[hides_nothing.lows_at:].tolist() == [0]


@pytest.mark.parametrize("window,parts,wide", [
    (None, None, False), (0, None, True), (None, torch.float32, True), (0, torch.float32, True),
    (None, torch.bfloat16, False), (0, torch.bfloat16, False), (4000, None, True), (4000, torch.float32, True),
    (9000, torch.float32, True),
])
def test_plan_parts_have_a_named_type(cuda_lib, window, parts, wide):
    """What split tiles are kept in goes by a name; no window and a window of 0 are the same mask under either."""
    from vlcache_b200 import ops
    plan = ops.build_prefill_plan([0, 20], [0, 9000], 16, 2, num_sms=148, window=window, parts=parts)
    assert plan.num_parts > 0 and plan.workspace_bytes == plan.num_parts * 128 * (128 * (4 if wide else 2) + 8)
    if not window:   # the same mask, and so the same plan
        other = ops.build_prefill_plan([0, 20], [0, 9000], 16, 2, num_sms=148, window=0 if wide else None)
        assert plan.host.tolist() == other.host.tolist()
    whole = ops.build_prefill_plan([0, 700], [0, 900], 16, 2, num_sms=16, window=window, parts=parts)
    assert whole.num_parts == 0 and whole.workspace_bytes == 0


def test_plan_parts_refusals(cuda_lib):
    from vlcache_b200 import ops
    for kw in (dict(parts=torch.float16), dict(parts="fp32"), dict(parts=torch.bfloat16, window=100),
               dict(parts=torch.float32, causal=False)):
        with pytest.raises(ValueError, match="parts"):
            ops.build_prefill_plan([0, 64], [0, 64], 16, 2, num_sms=8, **kw)


def test_c_abi_gather_of_seen_keys_refuses(cuda_lib):
    one = ctypes.c_void_p(64)   # never dereferenced: validation fails first

    def gather(seqs=1, lows=one, sinks=0, block=64):
        return cuda_lib.vlc_gather_seen_kvcache_fp4(one, one, 0, 1, 4, block, 2, 128, one, 4, 4, one, seqs, 100, 1.0, 1.0,
                                                    one, one, 256, 0, lows, sinks, None)
    assert gather(sinks=-1) == 2 and gather(lows=None) == 1 and gather(block=48) == 5 and gather(seqs=0, lows=None) == 0


# ------------------------------------------------------------------ the engine's bookkeeping
def _decoder(pages=20, **kw):
    from vlcache_b200.engine.draft_decode import DraftDecode
    from vlcache_b200.engine.page_pool import PagePool
    pool = PagePool(pages, 32)
    return pool, DraftDecode(pool, **{**dict(places=3, max_pages=6, num_drafts=2, device="cpu"), **kw})


@pytest.mark.parametrize("window,sinks,tokens", [(40, 3, 170), (40, 0, 170), (1, 0, 161), (33, 64, 192), (100, 5, 190)])
def test_admit_takes_a_table_whose_hidden_pages_are_gone(window, sinks, tokens):
    """Entries of -1 where no later row sees a key, and nowhere else: the pages that a step would give back."""
    pool, d = _decoder(window=window, sinks=sinks)
    full = pool.allocate(6)
    seen = {j // 32 for j in range(tokens + 1) if j > tokens - window or j < sinks}
    hidden = [i for i in range(6) if i not in seen]
    assert hidden or window == 100
    table = [-1 if i in hidden else p for i, p in enumerate(full)]
    pool.free([full[i] for i in hidden])
    for i in sorted(seen & set(range(6))):
        with pytest.raises(ValueError, match="not this table's alone"):
            d.admit(0, [-1 if x == i else p for x, p in enumerate(table)], tokens)
    assert int(d.context_lens[0]) == -1
    for bad in (-2, 20):
        for i in hidden:
            with pytest.raises(ValueError, match="not this table's alone"):
                d.admit(0, [bad if x == i else p for x, p in enumerate(table)], tokens)
    d.admit(0, table, tokens)
    assert d.block_tables[0].tolist() == table and int(d.context_lens[0]) == tokens
    assert d.retire(0) == tokens and pool.num_free == 20 and pool.refs == [0] * 20


def test_admit_without_a_window_needs_every_page():
    pool, d = _decoder()
    table = pool.allocate(3)
    with pytest.raises(ValueError, match="not this table's alone"):
        d.admit(0, [-1] + table[1:], 96)


def test_admit_refuses_pages_that_the_decoder_has():
    """A page of another place's table, or one that was lent, would be written by two sequences and given back twice."""
    pool, d = _decoder()
    table = pool.allocate(2)
    d.admit(0, table, 64)
    for other in (table, pool.allocate(1) + table[1:]):
        with pytest.raises(ValueError, match="another place's table"):
            d.admit(1, other, 40)
    assert d.lend(2)
    lent = d.free_pages[:2].tolist()
    with pytest.raises(ValueError, match="was lent"):
        d.admit(1, lent, 40)
    d.settle()   # now they are the pool's, and nobody's
    assert d.retire(0) == 64
    d.admit(1, table[:0], 0)
    assert int(d.context_lens[1]) == 0
    again = pool.allocate(4)   # pages that the decoder had are a table's again
    d.admit(2, again, 100)
    assert d.block_tables[2].tolist() == again + [-1, -1]


# ------------------------------------------------------------------ rows of a decode step
@pytest.mark.parametrize("rows,lens,tokens,refused", [
    (4, 2, None, True), (3, 2, None, True), (4, 2, 2, False), (2, 2, 2, False), (6, 2, 2, True), (3, 2, 2, True),
    (2, 2, None, False), (1, 2, None, False), (2, 2, 0, True),
])
def test_attention_takes_the_tokens_that_the_context_says(rows, lens, tokens, refused, monkeypatch):
    """Twice as many rows as lengths are no two tokens each unless the context says so: a slip in the lengths is
    refused before anything runs."""
    from vlcache_b200 import ops
    from vlcache_b200.layers.attention import Attention
    from vlcache_b200.utils.context import reset_context, set_context
    calls = []
    monkeypatch.setattr(ops, "decode_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(ops, "decode_window_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(ops, "decode_attention", lambda q, *a, **k: calls.append(q.shape) or q)
    monkeypatch.setattr(ops, "decode_attention_window", lambda q, *a, **k: calls.append((q.shape, a[2].shape, a[3].shape)) or q)
    layer = Attention(4, 128, 0.1, 2)
    layer.k_cache, layer.v_cache = (torch.zeros(2, 32, 2, 128, dtype=torch.bfloat16) for _ in range(2))
    kw = {} if tokens is None else dict(num_tokens=tokens)
    try:
        set_context(False, context_lens=torch.ones(lens, dtype=torch.int32),
                    block_tables=torch.zeros(lens, 1, dtype=torch.int32), **kw)
        q = torch.zeros(rows, 4, 128, dtype=torch.bfloat16)
        if refused:
            with pytest.raises(ValueError, match=f"decode: {rows} rows for {lens} sequences"):
                layer(q, None, None)
            assert not calls
        else:
            layer(q, None, None)
            n = tokens or 1
            assert calls == ([((rows // n, n, 4, 128), (rows // n, 1), (rows // n,))] if n > 1 else [(rows, 4, 128)])
    finally:
        reset_context()


def test_draft_decode_says_its_tokens(monkeypatch):
    from vlcache_b200 import ops
    from vlcache_b200.utils.context import get_context, reset_context
    _, d = _decoder()
    monkeypatch.setattr(ops, "step_metadata", lambda *a: (torch.zeros(9),) * 4 + (d.context_lens,))
    try:
        d.begin()
        assert get_context().num_tokens == 3 and not get_context().is_prefill
    finally:
        reset_context()


# ------------------------------------------------------------------ the build
@pytest.mark.parametrize("torch_there", [True, False])
def test_library_is_built_without_torch(torch_there, monkeypatch, tmp_path):
    """The library needs no torch: without it the build leaves the binding out (and says so in its stamp)."""
    from pathlib import Path

    from vlcache_b200 import build
    for name in ("LIB_PATH", "BINDING_PATH", "STAMP_PATH", "BUILD_DIR"):
        monkeypatch.setattr(build, name, tmp_path / name)
    with_torch = build.source_hash()
    if not torch_there:
        real_spec, real_version = build.importlib.util.find_spec, build.importlib.metadata.version

        def version(name):
            if name == "torch":
                raise build.importlib.metadata.PackageNotFoundError(name)
            return real_version(name)
        monkeypatch.setattr(build.importlib.util, "find_spec", lambda n, *a: None if n == "torch" else real_spec(n, *a))
        monkeypatch.setattr(build.importlib.metadata, "version", version)
    tools = []

    def run(cmd, **kw):
        tools.append(Path(cmd[0]).name)
        out = Path(cmd[cmd.index("-o") + 1])
        out.parent.mkdir(parents=True, exist_ok=True)
        out.write_text("built")
        return build.subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(build.subprocess, "run", run)
    assert build.build() == build.LIB_PATH and build.LIB_PATH.exists() and build.is_fresh()
    assert build.BINDING_PATH.exists() == torch_there and tools.count("g++") == (2 if torch_there else 0)
    assert tools.count("nvcc") == len(build.CUDA_SOURCES) + len(build.CPP_SOURCES) + 1
    assert (build.source_hash() == with_torch) == torch_there
    tools.clear()
    build.build()
    assert not tools   # fresh


@pytest.mark.parametrize("num_drafts", [0, 1, 5])
def test_draft_decode_bounds_lengths_by_its_tables(num_drafts, monkeypatch):
    """A step that begins in a table is not cut, one that begins at its end is: a single token's length never passes
    the table, which the one-token decode reads unchecked."""
    from vlcache_b200 import ops
    from vlcache_b200.utils.context import get_context, reset_context
    _, d = _decoder(num_drafts=num_drafts)
    monkeypatch.setattr(ops, "step_metadata", lambda *a: (torch.zeros(9),) * 4 + (d.context_lens,))
    try:
        d.begin()
        bound, room = get_context().max_context_len, 6 * 32
        assert (room - 1) + (num_drafts + 1) <= bound < room + (num_drafts + 1)
    finally:
        reset_context()


def test_draft_decode_refuses_more_drafts_than_a_verification_takes():
    for bad in (dict(num_drafts=32), dict(places=65536)):
        with pytest.raises(ValueError, match="places"):
            _decoder(**bad)
    _decoder(num_drafts=31)
