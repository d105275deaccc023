"""Host side of the 4-bit cache, the page pool and the several-axes rotary: the oracle's
rounding, the pool's bookkeeping, and the refusals, none of which needs a GPU."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import fp4


# ------------------------------------------------------------------ the oracle's rounding
def test_oracle_scale_grid_rounds_as_float8():
    """The oracle's e4m3 list and its rounding agree with torch's cast (finite, up to 448)."""
    x = torch.cat([torch.logspace(-12, 2.65, 4001), torch.tensor([0.0, 448.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    x = x.clamp(max=448.0)
    ours = fp4.nearest(x.double().numpy(), fp4.E4M3)
    assert np.array_equal(ours.astype(np.uint8), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_oracle_code_ties_go_to_even():
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    assert fp4.nearest(ties, fp4.E2M1).tolist() == [0, 2, 2, 4, 4, 6, 6]
    assert fp4.nearest(np.array([6.0, 7.9, 1e9]), fp4.E2M1).tolist() == [7, 7, 7]


def test_oracle_values_fit_bf16():
    """Every product of a code and a scale is exact in bf16 (and so in fp32 and f16)."""
    v = torch.from_numpy(fp4.E2M1[:, None] * fp4.E4M3[None, :])
    assert torch.equal(v.to(torch.bfloat16).double(), v) and torch.equal(v.to(torch.float16).double(), v)


def test_quantising_without_division_is_exact():
    """The kernels' arithmetic, in numpy's fp32, over every bf16 magnitude and every scale: a
    product with the reciprocal put on the grid of 2^-11 rounds to e2m1 as the exact quotient
    does, and a product with 1/6 rounds to e4m3 as the quotient by 6 does.  The reciprocal is
    taken one step high and low too, as an approximate one may be."""
    f = np.float32
    x = np.arange(0x7f80, dtype=np.uint32)
    x = (x << 16).view(f)                                            # all finite magnitudes
    top = np.minimum(x.astype(np.float64) / 6, 448)
    with np.errstate(over="ignore"):
        assert np.array_equal(fp4.nearest(np.minimum(x * (f(1) / f(6)), f(448)).astype(np.float64), fp4.E4M3),
                              fp4.nearest(top, fp4.E4M3))
        grid = f(1.5 * 4096)
        for s in fp4.E4M3[1:]:
            y = x[x <= 20 * s]                                       # the codes stop at 6
            want = fp4.nearest(y.astype(np.float64) / s, fp4.E2M1)
            inv = f(1) / f(s)
            for i in (inv, np.nextafter(inv, f(0)), np.nextafter(inv, f(4096))):
                for sign in (f(1), f(-1)):
                    q = (y.astype(np.float64) * sign * i + grid).astype(f) - grid   # one rounding, as fma has
                    assert np.array_equal(fp4.nearest(np.abs(q.astype(np.float64)), fp4.E2M1), want)


def test_oracle_pages_round_trip():
    r = np.random.default_rng(0)
    pages = r.integers(0, 256, size=(3, 2, 64 * fp4.ROW), dtype=np.uint8)
    assert np.array_equal(fp4.join_pages(*fp4.split_pages(pages)), pages)


# ------------------------------------------------------------------ page pool
def test_page_pool_allocate_fork_free():
    from vlcache_b200.engine.page_pool import PagePool
    pool = PagePool(8, 4)
    a = pool.allocate(3)
    assert a == [0, 1, 2] and pool.num_free == 5
    table, copies = pool.fork(a, 9)           # two full pages and one token
    assert table[:2] == a[:2] and copies == [(2, table[2])] and table[2] not in a
    full, none = pool.fork(a, 8)              # exactly two pages: nothing to copy
    assert full == a[:2] and none == []
    empty, none = pool.fork(a, 0)
    assert empty == [] and none == []
    pool.free(a)
    assert pool.num_free == 5                 # page 2 came back, 0 and 1 are still shared
    pool.free(full)
    pool.free(table)
    assert pool.num_free == 8 and pool.refs == [0] * 8


def test_page_pool_without_room_changes_nothing():
    from vlcache_b200.engine.page_pool import PagePool
    pool = PagePool(2, 4)
    a = pool.allocate(2)
    before = list(pool.refs)
    assert pool.allocate(1) is None and pool.fork(a, 7) is None and pool.refs == before
    for bad in (lambda: pool.fork(a, 9), lambda: pool.fork([5], 1), lambda: pool.free([0, 0]), lambda: pool.free([-1]),
                lambda: pool.allocate(-1), lambda: PagePool(0)):
        with pytest.raises(ValueError):
            bad()
    assert pool.refs == before


@pytest.mark.parametrize("seed", range(5))
def test_page_pool_compact(seed):
    """After compaction the used pages are the first ones, every table still names the page
    that holds its contents, and no page is both written and read by the copies."""
    from vlcache_b200.engine.page_pool import PagePool, remap
    r = np.random.default_rng(seed)
    pool = PagePool(40, 4)
    tables = [pool.allocate(int(n)) for n in r.integers(1, 6, 8)]
    shared, copies = pool.fork(tables[0], 4 * len(tables[0]))
    assert copies == []
    tables.append(shared)
    for i in sorted(r.choice(8, 4, replace=False).tolist(), reverse=True):
        pool.free(tables.pop(i))
    content = np.arange(40) + 1000
    want = [[content[p] for p in t] for t in tables]
    src, dst, page_map = pool.compact()
    assert not set(src) & set(dst)
    content[dst] = content[src]
    tables = [remap(t, page_map) for t in tables]
    assert [[content[p] for p in t] for t in tables] == want
    live = {p for t in tables for p in t}
    assert live == set(range(len(live))) and pool.num_free == 40 - len(live)
    assert pool.compact()[:2] == ([], [])
    for t in tables:
        pool.free(t)
    assert pool.num_free == 40


def test_copy_pages_refuses_bad_lists():
    from vlcache_b200.engine.kv_cache import copy_pages
    cache = torch.zeros(2, 1, 4, 8)
    copy_pages(cache, [], [])
    for src, dst in (([0], [0, 1]), ([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(ValueError):
            copy_pages(cache, src, dst)


# ------------------------------------------------------------------ sizing
def test_cache_budget_of_the_4bit_cache():
    from vlcache_b200.engine.kv_cache import allocate_kv_cache, cache_budget
    args = dict(mem_info=(150 << 30, 180 << 30), peak_bytes=0, current_bytes=0)
    b16 = cache_budget(28, 4, 128, 3584, **args)
    b4 = cache_budget(28, 4, 128, 3584, kv_format="fp4", **args)
    assert b4.kv_block_bytes * 256 == b16.kv_block_bytes * 72
    assert b4.num_encoder_blocks == b16.num_encoder_blocks and b4.num_kvcache_blocks > 3.5 * b16.num_kvcache_blocks
    t = allocate_kv_cache(None, 2, 3, 4, block_size=64, device="cpu", kv_format="fp4")
    assert t.dtype == torch.uint8 and tuple(t.shape) == (2, 2, 3, 4, 64 * 72)
    for bad in (dict(kv_format="int4"), dict(kv_format="fp4", head_dim=64), dict(kv_format="fp4", block_size=100)):
        with pytest.raises(ValueError):
            allocate_kv_cache(None, 1, 1, 1, device="cpu", **bad)


def test_mrope_section_is_checked():
    from vlcache_b200.layers.rotary_embedding import MRotaryEmbedding
    assert MRotaryEmbedding(128, 128, 16, 1e4, (22, 21, 21)).mrope_section == (22, 21, 21)
    for bad in ((16, 24, 23), (80, -16), ()):
        with pytest.raises(ValueError):
            MRotaryEmbedding(128, 128, 16, 1e4, bad)


# ------------------------------------------------------------------ refusals of the C ABI
P = ctypes.c_void_p(4096)   # never read: the checks come first
SEC3 = (ctypes.c_int32 * 3)(16, 24, 24)
NULL, SHAPE, STRIDE, ALIGN, UNSUPPORTED, WORKSPACE = 1, 2, 3, 4, 5, 6


def _call(lib, name, defaults, **changes):
    args = dict(defaults)
    for k, v in changes.items():
        assert k in args, k
        args[k] = v
    return getattr(lib, name)(*args.values())


ROPE = dict(positions=P, axis_stride=4, num_axes=3, sections=SEC3, q=P, q_stride=512, q_out=P, q_out_stride=512, key=P,
            key_stride=256, value=P, value_stride=256, table=P, max_position=64, k_cache=P, v_cache=P, slots=P,
            num_slots=256, k_out=None, k_out_stride=0, tokens=4, heads=4, kv_heads=2, head_dim=128, stream=None)
ROPE4 = {k: v for k, v in ROPE.items() if k not in ("num_slots", "k_out", "k_out_stride", "tokens", "heads", "kv_heads",
                                                    "head_dim", "stream")}
ROPE4.update(num_pages=4, block=64, k_scale=1.0, v_scale=0.5, tokens=4, heads=4, kv_heads=2, head_dim=128, stream=None)
STORE4 = dict(key=P, key_stride=256, value=P, value_stride=256, k_cache=P, v_cache=P, slots=P, num_pages=4, block=64,
              k_scale=1.0, v_scale=1.0, tokens=4, kv_heads=2, head_dim=128, stream=None)
GATHER = dict(k=P, v=P, layer_stride=0, layers=1, num_pages=4, block=64, kv_heads=2, head_dim=128, tables=P,
              table_stride=2, width=2, cu=P, seqs=2, total=100, k_scale=1.0, v_scale=1.0, k_out=P, v_out=P, row=256,
              out_layer=0, stream=None)
SHIFT4 = dict(k=P, v=P, layer_stride=0, layers=1, num_pages=4, block=64, kv_heads=2, head_dim=128, src=P, dst=P, rows=4,
              delta=SEC3, section=SEC3, theta=1e6, stream=None)
DECODE4 = dict(q=P, q_stride=512, seqs=2, heads=4, k=P, v=P, num_pages=4, block=64, kv_heads=2, head_dim=128, tables=P,
               table_stride=2, width=2, lens=P, max_len=128, scale=0.1, k_scale=1.0, v_scale=1.0, out=P, out_stride=512,
               ws=None, ws_bytes=0, stream=None)
COPY = dict(base=P, plane_stride=4096, planes=2, page_bytes=1024, pages=4, src=P, dst=P, pairs=2, stream=None)
REMAP = dict(tables=P, row_stride=4, rows=2, width=4, map=P, pages=8, stream=None)
odd = ctypes.c_void_p(4100)

REFUSALS = [
    ("vlc_mrope_store_kvcache", ROPE, dict(head_dim=64), UNSUPPORTED),
    ("vlc_mrope_store_kvcache", ROPE, dict(num_axes=5), UNSUPPORTED),
    ("vlc_mrope_store_kvcache", ROPE, dict(num_axes=0), UNSUPPORTED),
    ("vlc_mrope_store_kvcache", ROPE, dict(num_axes=2), SHAPE),            # 16 + 24 pairs
    ("vlc_mrope_store_kvcache", ROPE, dict(sections=(ctypes.c_int32 * 3)(96, -16, -16)), SHAPE),
    ("vlc_mrope_store_kvcache", ROPE, dict(axis_stride=3), STRIDE),
    ("vlc_mrope_store_kvcache", ROPE, dict(q_stride=504), STRIDE),
    ("vlc_mrope_store_kvcache", ROPE, dict(value_stride=100), STRIDE),
    ("vlc_mrope_store_kvcache", ROPE, dict(key=odd), ALIGN),
    ("vlc_mrope_store_kvcache", ROPE, dict(positions=None), NULL),
    ("vlc_mrope_store_kvcache", ROPE, dict(slots=None), NULL),             # no cache and no k_out
    ("vlc_mrope_store_kvcache", ROPE, dict(tokens=-1), SHAPE),
    ("vlc_mrope_store_kvcache", ROPE, dict(tokens=0), 0),
    ("vlc_rope_store_kvcache_fp4", ROPE4, dict(block=96), UNSUPPORTED),
    ("vlc_rope_store_kvcache_fp4", ROPE4, dict(k_scale=3.0), UNSUPPORTED),  # not a power of two
    ("vlc_rope_store_kvcache_fp4", ROPE4, dict(v_scale=0.0), UNSUPPORTED),
    ("vlc_rope_store_kvcache_fp4", ROPE4, dict(v_scale=float("nan")), UNSUPPORTED),
    ("vlc_rope_store_kvcache_fp4", ROPE4, dict(v_scale=-1.0), UNSUPPORTED),
    ("vlc_rope_store_kvcache_fp4", ROPE4, dict(num_pages=0), SHAPE),
    ("vlc_rope_store_kvcache_fp4", ROPE4, dict(v_cache=None), NULL),
    ("vlc_store_kvcache_fp4", STORE4, dict(head_dim=80), UNSUPPORTED),
    ("vlc_store_kvcache_fp4", STORE4, dict(key_stride=252), STRIDE),
    ("vlc_store_kvcache_fp4", STORE4, dict(key=None), NULL),
    ("vlc_store_kvcache_fp4", STORE4, dict(k_cache=odd), ALIGN),
    ("vlc_store_kvcache_fp4", STORE4, dict(tokens=0), 0),
    ("vlc_gather_kvcache_fp4", GATHER, dict(block=0), UNSUPPORTED),
    ("vlc_gather_kvcache_fp4", GATHER, dict(total=-1), SHAPE),
    ("vlc_gather_kvcache_fp4", GATHER, dict(layers=2), STRIDE),
    ("vlc_gather_kvcache_fp4", GATHER, dict(row=128), STRIDE),
    ("vlc_gather_kvcache_fp4", GATHER, dict(table_stride=1), STRIDE),
    ("vlc_gather_kvcache_fp4", GATHER, dict(v_out=odd), ALIGN),
    ("vlc_gather_kvcache_fp4", GATHER, dict(cu=None), NULL),
    ("vlc_gather_kvcache_fp4", GATHER, dict(seqs=0), 0),
    ("vlc_mrope_shift_fp4", SHIFT4, dict(section=(ctypes.c_int32 * 3)(16, 24, 20)), SHAPE),
    ("vlc_mrope_shift_fp4", SHIFT4, dict(layers=3), STRIDE),
    ("vlc_mrope_shift_fp4", SHIFT4, dict(head_dim=64), UNSUPPORTED),
    ("vlc_mrope_shift_fp4", SHIFT4, dict(src=None), NULL),
    ("vlc_mrope_shift_fp4", SHIFT4, dict(rows=0), 0),
    ("vlc_decode_attn_fp4", DECODE4, dict(heads=5), SHAPE),
    ("vlc_decode_attn_fp4", DECODE4, dict(heads=34, q_stride=34 * 128, out_stride=34 * 128), UNSUPPORTED),  # 17 a head
    ("vlc_decode_attn_fp4", DECODE4, dict(block=32), UNSUPPORTED),
    ("vlc_decode_attn_fp4", DECODE4, dict(block=1 << 21), UNSUPPORTED),
    ("vlc_gather_kvcache_fp4", GATHER, dict(block=1 << 21), UNSUPPORTED),
    ("vlc_store_kvcache_fp4", STORE4, dict(block=1 << 21), UNSUPPORTED),
    ("vlc_decode_attn_fp4", DECODE4, dict(out_stride=256), STRIDE),
    ("vlc_decode_attn_fp4", DECODE4, dict(q=odd), ALIGN),
    ("vlc_decode_attn_fp4", DECODE4, dict(lens=None), NULL),
    ("vlc_decode_attn_fp4", DECODE4, dict(max_len=100000), WORKSPACE),
    ("vlc_decode_attn_fp4", DECODE4, dict(k_scale=1.5), UNSUPPORTED),
    ("vlc_decode_attn_fp4", DECODE4, dict(seqs=0), 0),
    ("vlc_copy_pages", COPY, dict(page_bytes=1000), STRIDE),
    ("vlc_copy_pages", COPY, dict(plane_stride=2048), STRIDE),
    ("vlc_copy_pages", COPY, dict(base=odd), ALIGN),
    ("vlc_copy_pages", COPY, dict(src=None), NULL),
    ("vlc_copy_pages", COPY, dict(pairs=0), 0),
    ("vlc_remap_block_tables", REMAP, dict(row_stride=2), STRIDE),
    ("vlc_remap_block_tables", REMAP, dict(map=None), NULL),
    ("vlc_remap_block_tables", REMAP, dict(rows=0), 0),
]


@pytest.mark.parametrize("name,defaults,changes,status", REFUSALS,
                         ids=[f"{r[0][4:]}-{'-'.join(r[2])}-{i}" for i, r in enumerate(REFUSALS)])
def test_c_abi_refusals(cuda_lib, name, defaults, changes, status):
    assert _call(cuda_lib, name, defaults, **changes) == status


def test_ops_refuse_cpu_tensors(cuda_lib):
    from vlcache_b200 import ops
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    cache = torch.zeros(2, 2, 64 * 72, dtype=torch.uint8)
    ints = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.store_kvcache_fp4(x, x, cache, cache, ints),
                 lambda: ops.mrotary_embedding(torch.zeros(3, 2, dtype=torch.int64), x, x, torch.zeros(4, 128)),
                 lambda: ops.decode_attention_fp4(x, cache, cache, ints.view(2, 1), ints, 64, 0.1),
                 lambda: ops.gather_kvcache_fp4(cache, cache, ints.view(2, 1), ints, 4),
                 lambda: ops.mrope_shift_layer_fp4(cache, cache, ints, ints, (1, 1, 1)),
                 lambda: ops.copy_kv_pages(torch.zeros(2, 1, 2, 16), ints, ints),
                 lambda: ops.remap_block_tables(ints.view(1, 2), ints)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ bounds and arguments at their ends
@pytest.mark.parametrize("seqs,heads,kv_heads", [(64, 28, 4), (200, 16, 2), (100, 32, 2), (1, 16, 2)])
def test_decode_workspace_of_a_zero_bound(cuda_lib, seqs, heads, kv_heads):
    """A bound of 0 (every sequence is empty) is a bound of 1 for the size as for the call, and a
    byte less is refused."""
    need = cuda_lib.vlc_decode_fp4_workspace_size(seqs, heads, kv_heads, 0)
    assert need == cuda_lib.vlc_decode_fp4_workspace_size(seqs, heads, kv_heads, 1)
    assert (need > 0) == (seqs > 1)          # one sequence: clusters take whole pairs, without a workspace
    if need:
        stride = heads * 128
        assert _call(cuda_lib, "vlc_decode_attn_fp4", DECODE4, seqs=seqs, heads=heads, kv_heads=kv_heads, max_len=0,
                     q_stride=stride, out_stride=stride, ws=P, ws_bytes=need - 1) == WORKSPACE


def test_get_mrope_takes_a_list():
    """mrope_section as model configs hold it; the instance is the tuple's."""
    from vlcache_b200.layers.rotary_embedding import get_mrope
    rot = get_mrope(128, 128, 16, 1e4, [16, 24, 24])
    assert rot.mrope_section == (16, 24, 24)
    assert get_mrope(128, 128, 16, 1e4, (16, 24, 24)) is rot and get_mrope(128, 128, 16, 1e4) is rot
    assert get_mrope(128, 128, 16, 1e4, [22, 21, 21]).mrope_section == (22, 21, 21)
    with pytest.raises(ValueError):
        get_mrope(128, 128, 16, 1e4, [16, 24, 23])


@pytest.mark.parametrize("shape,swap", [((1, 2, 5, 4, 16), (0, 1)), ((2, 3, 1, 4, 16), None), ((2, 1, 5, 4, 16), None),
                                        ((2, 5, 1, 4, 16), (1, 2)), ((3, 2, 5, 8), None)])
def test_page_copies_stay_inside_the_cache(monkeypatch, shape, swap):
    """The planes and pages that the launch is given tile the cache's own memory, also where a dim
    of size 1 has a stride that says nothing (one layer of a cache allocated layer first; one page)."""
    from vlcache_b200 import ops
    cache = torch.zeros(shape, dtype=torch.bfloat16)
    if swap:
        cache = cache.transpose(*swap)
    assert cache.is_contiguous()
    calls = []
    monkeypatch.setattr(ops, "_device", lambda *t: 0)
    monkeypatch.setattr(ops, "_launch", lambda dev, name, *args: calls.append(args))
    pages = torch.zeros(1, dtype=torch.int32)
    ops.copy_kv_pages(cache, pages, pages)
    base, plane_stride, planes, page_bytes, num_pages = calls[0][:5]
    assert base == cache.data_ptr() and planes == cache.shape[0] * cache.shape[1] and num_pages == cache.shape[2]
    assert page_bytes * num_pages == plane_stride and plane_stride * planes == cache.nbytes


def test_remap_of_a_padded_host_table():
    """Padding stays padding, as ops.remap_block_tables leaves it; other entries outside the pool are refused."""
    from vlcache_b200.engine.page_pool import PagePool, remap
    pool = PagePool(6, 4)
    first, second = pool.allocate(2), pool.allocate(2)
    pool.free(first)
    page_map = pool.compact()[2]
    assert remap(second + [-1, -1], page_map) == [0, 1, -1, -1]
    for bad in ([6], [-2]):
        with pytest.raises(ValueError):
            remap(bad, page_map)


def test_decode_refuses_a_strided_workspace(cuda_lib, monkeypatch):
    """The parts are written to consecutive bytes: a strided view's lie between another tensor's."""
    from vlcache_b200 import ops
    calls = []
    monkeypatch.setattr(ops, "_device", lambda *t: 0)
    monkeypatch.setattr(ops, "_launch", lambda dev, name, *args: calls.append(args))
    q, cache = torch.zeros(3, 4, 128, dtype=torch.bfloat16), torch.zeros(2, 2, 64 * 72, dtype=torch.uint8)
    ints = torch.zeros(3, dtype=torch.int32)
    need = ops.decode_fp4_workspace_bytes(3, 4, 2, 5000)
    call = lambda ws: ops.decode_attention_fp4(q, cache, cache, ints.view(3, 1), ints, 5000, 0.1, workspace=ws)  # noqa: E731
    whole = torch.zeros(need, 2, dtype=torch.uint8)
    with pytest.raises(ValueError):
        call(whole[:, 0])
    assert not calls
    call(whole.view(-1)[:need])
    assert calls[0][-2:] == (whole.data_ptr(), need)


@pytest.mark.parametrize("steps", [2, 3])
def test_quantising_bears_the_approximate_reciprocal(steps):
    """The codes with 1 / s off by two and three fp32 steps: the approximate division that makes it
    is off by two units in the last place at most."""
    f = np.float32
    x = (np.arange(0x7f80, dtype=np.uint32) << 16).view(f)
    grid = f(1.5 * 4096)
    for s in fp4.E4M3[1:]:
        y = x[x <= 20 * s]
        want = fp4.nearest(y.astype(np.float64) / s, fp4.E2M1)
        for end in (f(0), f(4096)):
            inv = f(1) / f(s)
            for _ in range(steps):
                inv = np.nextafter(inv, end)
            q = (y.astype(np.float64) * inv + grid).astype(f) - grid
            assert np.array_equal(fp4.nearest(np.abs(q.astype(np.float64)), fp4.E2M1), want)
