"""GPU tests of the several-axes rotary, the 4-bit cache (store, read-back, attention, move of
reused rows) and the page copies, against the 64-bit oracle (oracle/fp4.py).

Where the result is defined by roundings (codes, scales, copies) it has to be equal, bytes or
values.  Attention is held to a bound that follows from its arithmetic, per element:
  decode   2^-8 |o| for the bf16 output, and (2^-11 + 2^-14 B + 2^-15) sum_j p_j |v_j|: P rounds
           to f16 (2^-11); a score's fp32 error is below 2^-15 B (128 products and as many
           additions of at most one 2^-23 each, with B = scale * max_j sum_d |q_d K_jd|), which
           changes p and its sum by 2^-14 B at most together; sums of P V and of the parts, some
           hundred additions of 2^-23: 2^-15.
  prefill  the same with P in bf16 (2^-8) and the parts of a split tile in bf16 (2^-8).
"""
import math

import numpy as np
import pytest
import torch

from oracle import fp4, mrope as omr, rope as orope

pytestmark = pytest.mark.gpu
D = 128
SCALE = 1 / math.sqrt(D)


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from vlcache_b200 import ops
    ops.device_error(reset=True)
    return ops


@pytest.fixture(autouse=True)
def no_device_error(ops):
    yield
    assert ops.device_error(reset=True) == 0


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bits(t):
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def _pages(seed, pages, hk, block, size=1.0):
    """Random 4-bit pages: quantised normal rows (uint8 CPU tensor)."""
    r = np.random.default_rng(seed)
    c, s = fp4.quantise(r.normal(size=(pages, hk, block, D)) * size)
    return torch.from_numpy(fp4.join_pages(c, s))


# ------------------------------------------------------------------ several axes
SECTIONS = [(16, 24, 24), (24, 20, 20), (22, 21, 21), (64,), (11, 53), (0, 64, 0), (8, 8, 24, 24)]


def _axes_reference(x, positions, sections, table):
    """oracle/rope.py at each axis, columns taken by section: bf16 bits [N, heads, 128]."""
    axis = np.repeat(np.arange(len(sections)), sections)
    per_axis = [orope.rope_rows(_bits(x), positions[a].numpy(), table[:, 0].numpy()) for a in range(len(sections))]
    out = np.empty_like(per_axis[0])
    for j in range(64):
        out[..., j], out[..., 64 + j] = per_axis[axis[j]][..., j], per_axis[axis[j]][..., 64 + j]
    return out


@pytest.mark.parametrize("sections", SECTIONS)
@pytest.mark.parametrize("N,H,Hk", [(1, 28, 4), (7, 16, 2), (130, 12, 1), (33, 8, 8)])
def test_mrope_store_matches_oracle(ops, sections, N, H, Hk):
    from vlcache_b200.layers.rotary_embedding import rope_cos_sin_cache
    g = _gen(N + len(sections))
    table = rope_cos_sin_cache(D, 4096, 1e6)
    pos = torch.randint(0, 4096, (len(sections), N), generator=g)
    qkv = torch.randn(N, H + 2 * Hk, D, generator=g).to(torch.bfloat16)
    q, k, v = qkv.split((H, Hk, Hk), 1)
    slots = torch.randperm(512, generator=g)[:N].to(torch.int32)
    slots[::5] = -1
    kc = torch.randn(2, 256, Hk, D, generator=g).to(torch.bfloat16)
    vc = torch.randn(2, 256, Hk, D, generator=g).to(torch.bfloat16)
    q_ref, k_ref = _axes_reference(q, pos, sections, table), _axes_reference(k, pos, sections, table)
    kc_ref, vc_ref = _bits(kc).reshape(512, Hk, D).copy(), _bits(vc).reshape(512, Hk, D).copy()
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            kc_ref[s], vc_ref[s] = k_ref[i], _bits(v)[i]
    dq, dk, dv = qkv.cuda().split((H, Hk, Hk), 1)
    dkc, dvc, t = kc.cuda(), vc.cuda(), table.cuda()
    q_rot, k_rot = ops.mrotary_embedding(pos.cuda(), dq, dk, t, sections)
    out = ops.mrope_store_kvcache(pos.cuda(), dq, dk, dv, t, dkc, dvc, slots.cuda(), sections, out=dq)
    assert out.data_ptr() == dq.data_ptr()      # in place
    for got, ref in ((q_rot, q_ref), (k_rot, k_ref), (out, q_ref)):
        assert np.array_equal(_bits(got), ref)
    assert np.array_equal(_bits(dkc).reshape(512, Hk, D), kc_ref)
    assert np.array_equal(_bits(dvc).reshape(512, Hk, D), vc_ref)


@pytest.mark.parametrize("N,H,Hk,sections", [(4011, 28, 4, (16, 24, 24)), (12001, 6, 1, (22, 21, 21)),
                                             (6001, 16, 2, (64,))])
def test_mrope_many_tokens_are_few_tokens_rows(ops, N, H, Hk, sections):
    """A prompt's rows come out as they do in calls of a few tokens each, into either cache and
    without one: skipped slots, bad slots and bad positions among them."""
    from vlcache_b200.layers.rotary_embedding import rope_cos_sin_cache
    g = _gen(N)
    table = rope_cos_sin_cache(D, 1024, 1e6).cuda()
    pos = torch.randint(0, 1024, (len(sections), N), generator=g)
    pos[-1, 77] = 1024
    pos, qkv = pos.cuda(), torch.randn(N, H + 2 * Hk, D, generator=g).to(torch.bfloat16).cuda()
    q, k, v = qkv.split((H, Hk, Hk), 1)
    pages = (N + 255) // 256 + 1
    slots = torch.randperm(pages * 256, generator=g)[:N].to(torch.int32)
    slots[::11], slots[5] = -1, pages * 256
    slots = slots.cuda()
    zeros = lambda fmt: [torch.zeros(*((pages, 256, Hk, D) if fmt == "bf16" else (pages, Hk, 256 * 72)),  # noqa: E731
                                     dtype=torch.bfloat16 if fmt == "bf16" else torch.uint8, device="cuda")
                         for _ in "kv"]
    rows = [slice(i, i + 100) for i in range(0, N, 100)]
    for fmt, store in (("bf16", ops.mrope_store_kvcache), ("fp4", ops.rope_store_kvcache_fp4)):
        many, few = zeros(fmt), zeros(fmt)
        out, parts = torch.zeros(N, H, D, dtype=torch.bfloat16, device="cuda"), torch.zeros_like(q)
        store(pos, q, k, v, table, *many, slots, sections, out=out)
        assert ops.device_error(reset=True) in (101, 103)
        for r in rows:
            store(pos[:, r], q[r], k[r], v[r], table, *few, slots[r], sections, out=parts[r])
        assert ops.device_error(reset=True) in (101, 103)
        assert torch.equal(out, parts) and bool(out[-1].any()) and not bool(out[77].any())
        assert all(torch.equal(a, b) and bool(a.any()) for a, b in zip(many, few))
    good = pos.clamp(max=1023)
    a, b = ops.mrotary_embedding(good, q, k, table, sections)
    for r in rows:
        x, y = ops.mrotary_embedding(good[:, r], q[r], k[r], table, sections)
        assert torch.equal(a[r], x) and torch.equal(b[r], y)


def test_mrope_on_equal_axes_is_rope(ops):
    """Text rows: equal positions on every axis (one row, broadcast) give the one-axis bits."""
    from vlcache_b200.layers.rotary_embedding import rope_cos_sin_cache
    g = _gen(5)
    table = rope_cos_sin_cache(D, 2048, 1e6).cuda()
    q = torch.randn(100, 16, D, generator=g).to(torch.bfloat16).cuda()
    k = torch.randn(100, 2, D, generator=g).to(torch.bfloat16).cuda()
    pos = torch.randint(0, 2048, (100,), generator=g).cuda()
    want = ops.rotary_embedding(pos, q, k, table)
    for p in (pos.expand(3, 100), pos.repeat(3, 1), pos.repeat(5, 1)[::2]):
        got = ops.mrotary_embedding(p, q, k, table)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_mrope_against_transformers_formula(ops):
    """Image rows at (t, h, w) grid positions: the fp32 formula of the multimodal rotary on the
    same inputs.  The table's angles are fp32 products in both; its cos/sin may differ by an
    fp32 step from the formula's and the kernel's sum of two products carries three roundings:
    2^-22 (|x1| + |x2|), then half a bf16 step."""
    from vlcache_b200.layers.rotary_embedding import get_mrope
    g = _gen(6)
    pos = torch.from_numpy(omr.vision_positions(37, 12, 9))
    x = torch.randn(108, 4, D, generator=g).to(torch.bfloat16)
    rot = get_mrope(D, D, 4096, 1e6).cuda()
    got, _ = rot(pos.cuda(), x.cuda(), x.cuda())
    ref = omr.apply_mrope(x.float(), pos.numpy())
    bound = ref.abs() * 2.0 ** -8 + 2.0 ** -22 * (x.float().abs() + omr.rotate_half(x.float()).abs()) * 1.01
    assert bool(((got.float().cpu() - ref).abs() <= bound).all())


def test_mrope_bad_rows_are_flagged_and_skipped(ops):
    from vlcache_b200.layers.rotary_embedding import rope_cos_sin_cache
    table = rope_cos_sin_cache(D, 64, 1e6).cuda()
    g = _gen(7)
    q, k, v = (torch.randn(3, h, D, generator=g).to(torch.bfloat16).cuda() for h in (4, 2, 2))
    pos = torch.tensor([[0, 1, 2], [0, 64, 2], [0, 1, 2]]).cuda()      # token 1: its second axis is past the table
    for fmt in ("bf16", "fp4"):
        kc = (torch.zeros(1, 64, 2, D, dtype=torch.bfloat16) if fmt == "bf16" else
              torch.zeros(1, 2, 64 * 72, dtype=torch.uint8)).cuda()
        vc, out = kc.clone(), torch.zeros_like(q)
        slots = torch.tensor([0, 1, 64], dtype=torch.int32).cuda()     # slot 64 of 64
        store = ops.mrope_store_kvcache if fmt == "bf16" else ops.rope_store_kvcache_fp4
        store(pos, q, k, v, table, kc, vc, slots, (16, 24, 24), out=out)
        assert ops.device_error(reset=True) in (101, 103)
        assert int(out[1].abs().sum() == 0) and bool(out[0].any()) and bool(out[2].any())
        if fmt == "bf16":
            assert bool(kc[0, 0].any()) and not bool(kc[0, 1:].any())
            assert bool(vc[0, 1].any()) and not bool(vc[0, 2:].any())
        else:
            c, s = fp4.split_pages(kc.cpu().numpy())
            assert c[0, :, 0].any() and not c[0, :, 1:].any() and not s[0, :, 1:].any()
            c, s = fp4.split_pages(vc.cpu().numpy())
            assert c[0, :, 1].any() and not c[0, :, 2:].any()


# ------------------------------------------------------------------ storing in 4 bits
def _special_rows(n, hk, g):
    """Normal rows with groups at the edges of the formats."""
    x = torch.randn(n, hk, D, generator=g)
    x[0] = 0                                           # all-zero groups
    if n > 4:
        x[1] *= 2.0 ** -11                             # scales that are subnormal or 0
        x[2] *= 3000.0                                 # scales that saturate
        x[3] = torch.tensor([0.25, -0.75, 1.25, 1.75, 2.5, -3.5, 5.0, 6.0]).repeat(16) * 1.125   # code ties
        x[4] = 2.0 ** -30
    if n > 8:
        x[5, :, 16:32] = 3 * 2.0 ** -10 * 6            # a scale tie
        x[6, 0, 17] = float("nan")
        x[7, 0, 40] = float("inf")
        x[7, 0, 41] = -float("inf")
        x[8, 0, 5] = -float("nan")
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("N,Hk,block,kg,vg", [(1, 1, 64, 1.0, 1.0), (9, 2, 256, 2.0, 0.125), (200, 4, 128, 1.0, 2.0 ** -5),
                                              (65, 8, 64, 2.0 ** -20, 2.0 ** 10)])
def test_store_fp4_bytes(ops, N, Hk, block, kg, vg):
    g = _gen(N)
    pages = (N + block - 1) // block + 2
    kc, vc = _pages(1, pages, Hk, block), _pages(2, pages, Hk, block)
    k, v = (_special_rows(N, Hk, g).float() * s for s in (kg, vg))
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    slots = torch.randperm(pages * block, generator=g)[:N].to(torch.int32)
    slots[3::7] = -1
    dkc, dvc = kc.cuda(), vc.cuda()
    ops.store_kvcache_fp4(k.cuda(), v.cuda(), dkc, dvc, slots.cuda(), kg, vg)
    for got, cache, x, s in ((dkc, kc, k, kg), (dvc, vc, v, vg)):
        want = fp4.split_pages(fp4.store(cache.numpy(), x.double().numpy(), slots.numpy(), s))
        have = fp4.split_pages(got.cpu().numpy())
        nan = np.repeat(want[1] == 127, 16, -1)        # of a NaN group only the scale counts
        assert np.array_equal(want[1], have[1])
        zero = (want[0] & 7 == 0) & (have[0] & 7 == 0)  # -0 and 0 are one value
        assert bool(((want[0] == have[0]) | zero | nan).all())


@pytest.mark.parametrize("H,Hk,N", [(28, 4, 37), (16, 2, 3), (12, 1, 66), (8, 8, 1)])
def test_rope_store_fp4_is_rope_then_store(ops, H, Hk, N):
    """Fused and unfused give the same bytes, on one axis and on three; q/k/v are views of one
    projection row and q is rotated in place."""
    from vlcache_b200.layers.rotary_embedding import rope_cos_sin_cache
    g = _gen(N)
    table = rope_cos_sin_cache(D, 1024, 1e6).cuda()
    qkv = torch.randn(N, H + 2 * Hk, D, generator=g).to(torch.bfloat16).cuda()
    slots = torch.randperm(256, generator=g)[:N].to(torch.int32).cuda()
    for section, axes in ((None, 0), ((64,), 1), ((16, 24, 24), 3), ((21, 22, 21), 3)):
        pos = torch.randint(0, 1024, (axes, N) if axes else (N,), generator=g).cuda()
        q, k, v = qkv.clone().split((H, Hk, Hk), 1)
        caches = [torch.zeros(2, Hk, 128 * 72, dtype=torch.uint8, device="cuda") for _ in range(4)]
        q_rot, k_rot = (ops.rotary_embedding(pos, q.contiguous(), k.contiguous(), table) if section is None else
                        ops.mrotary_embedding(pos, q, k, table, section))
        ops.store_kvcache_fp4(k_rot, v, caches[0], caches[1], slots, 0.5, 0.25)
        out = ops.rope_store_kvcache_fp4(pos, q, k, v, table, caches[2], caches[3], slots, section, 0.5, 0.25, out=q)
        assert torch.equal(out, q_rot)
        assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
        assert bool(caches[2].any())


# ------------------------------------------------------------------ reading back
@pytest.mark.parametrize("lens,block,hk", [([5], 64, 1), ([0, 1, 63, 64, 65, 0, 200], 64, 2), ([700, 3], 256, 4),
                                           ([128] * 9, 128, 2)])
def test_gather_fp4_is_exact(ops, lens, block, hk):
    pages = sum((n + block - 1) // block for n in lens) + 3
    kc, vc = _pages(3, pages, hk, block), _pages(4, pages, hk, block)
    order = torch.randperm(pages, generator=_gen(1)).tolist()
    width = max(1, max((n + block - 1) // block for n in lens))
    tables, at = [], 0
    for n in lens:
        w = (n + block - 1) // block
        tables.append(order[at:at + w] + [-1] * (width - w))
        at += w
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    total = int(cu[-1])
    k_out = torch.full((total + 5, hk, D), 7.0, dtype=torch.bfloat16, device="cuda")
    v_out = torch.full((total + 5, hk, D), 7.0, dtype=torch.bfloat16, device="cuda")
    bt = torch.tensor(tables, dtype=torch.int32).cuda()
    ops.gather_kvcache_fp4(kc.cuda(), vc.cuda(), bt, torch.from_numpy(cu).cuda(), total + 5, 4.0, 0.25, k_out, v_out)
    for out, cache, g in ((k_out, kc, 4.0), (v_out, vc, 0.25)):
        want = np.concatenate([fp4.sequence(cache.numpy(), t, n, g) for t, n in zip(tables, lens)])
        assert np.array_equal(out[:total].double().cpu().numpy(), want)
        assert bool((out[total:] == 7).all())          # rows behind the last sequence stay
    # several layers at once: each layer's rows are that layer's own
    kv = torch.stack([torch.stack([kc, vc]), torch.stack([vc, kc])]).cuda()
    a, b = ops.gather_kvcache_fp4(kv[0], kv[1], bt, torch.from_numpy(cu).cuda(), total, 1.0, 1.0)
    assert a.shape == (2, total, hk, D) and torch.equal(a[0], b[1]) and torch.equal(a[1], b[0])


def test_gather_fp4_flags_bad_pages_and_lengths(ops):
    kc = _pages(5, 2, 1, 64).cuda()
    bt = torch.tensor([[0, 9], [-1, 1]], dtype=torch.int32).cuda()
    cu = torch.tensor([0, 100, 200], dtype=torch.int32).cuda()
    k, _ = ops.gather_kvcache_fp4(kc, kc, bt, cu, 200)
    assert ops.device_error(reset=True) == 102
    assert bool(k[:64].any()) and not bool(k[64:164].any()) and bool(k[164:].any())
    out = torch.full((150, 1, D), 3.0, dtype=torch.bfloat16, device="cuda")
    guard = torch.full((200, 1, D), 3.0, dtype=torch.bfloat16, device="cuda")[:150]
    bt = torch.tensor([[0, 1], [0, 1]], dtype=torch.int32).cuda()
    ops.gather_kvcache_fp4(kc, kc, bt, cu, 150, k_out=out, v_out=guard)   # cu_seqlens_k says 200
    assert ops.device_error(reset=True) == 104
    assert bool((guard._base[150:] == 3).all())


# ------------------------------------------------------------------ attention
def _paged(seed, lens, hk, block, poison=True, size=1.0):
    """Caches and tables; rows behind a sequence's end hold NaN scales, as memory never written may."""
    pages = sum(max(1, (n + block - 1) // block) for n in lens) + 2
    kc, vc = _pages(seed, pages, hk, block, size), _pages(seed + 1, pages, hk, block, size)
    order = torch.randperm(pages, generator=_gen(seed)).tolist()
    width = max(max(1, (n + block - 1) // block) for n in lens)
    tables, at = [], 0
    for n in lens:
        w = (n + block - 1) // block
        tables.append(order[at:at + w] + [-1] * (width - w))
        at += w
        if poison and n % block:
            for c in (kc, vc):
                page = c[order[at - 1]]
                page[:, block * 64 + (n % block) * 8:] = 255
                page[:, (n % block) * 64:block * 64] = 255
    return kc, vc, torch.tensor(tables, dtype=torch.int32)


def _check_attention(out, q, kc, vc, tables, q_lens, k_lens, scale, kg, vg, p_error, margins=None, what=""):
    at, worst = 0, 0.0
    q64 = q.double().cpu().numpy()
    for i, (a, n) in enumerate(zip(q_lens, k_lens)):
        k = fp4.sequence(kc.numpy(), tables[i].tolist(), n, kg)
        v = fp4.sequence(vc.numpy(), tables[i].tolist(), n, vg)
        rows = q64[at:at + a]
        ref, size = fp4.attend(rows, k, v, scale)
        G = q.shape[1] // kc.shape[1]
        got = out[at:at + a].double().cpu().numpy()
        assert np.isfinite(got).all()
        if n:
            B = scale * np.einsum("ahd,nhd->ahn", np.abs(rows), np.abs(np.repeat(k, G, 1))).max(-1)[..., None]
        else:
            B = 0.0
        bound = 2.0 ** -8 * np.abs(ref) + (p_error + 2.0 ** -14 * B + 2.0 ** -15) * size
        err = np.abs(got - ref)
        worst = max(worst, float((err / np.maximum(bound, 1e-30)).max(initial=0)))
        at += a
    assert worst <= 1.0, worst


DECODE = [  # H, Hk, block, lens
    (16, 2, 256, [1]),
    (16, 2, 64, [0, 1, 15, 16, 17, 63, 64, 65, 0]),
    (28, 4, 256, [700, 2, 511, 512, 513]),
    (12, 1, 128, [300, 0, 129]),             # 12 query heads a KV head: two column tiles
    (16, 1, 64, [130, 77]),                  # 16
    (9, 1, 64, [200]),
    (8, 8, 64, [100, 33]),                   # one query head a KV head
    (28, 4, 256, [5000, 40, 2049]),          # several splits
    (4, 4, 128, [20011]),
    (28, 4, 64, [255, 256, 257, 0, 768, 1023, 1024]),   # whole pairs of 4, 8 and 16 chunks
    (32, 2, 128, [1024, 256, 3]),
]


@pytest.mark.parametrize("H,Hk,block,lens", DECODE)
def test_decode_fp4(ops, H, Hk, block, lens):
    kc, vc, bt = _paged(11, lens, Hk, block)
    q = (2 * torch.randn(len(lens), H, D, generator=_gen(3))).to(torch.bfloat16)
    ctx = torch.tensor(lens, dtype=torch.int32)
    for bound in (max(max(lens), 1), 30000):   # whole pairs to a block, where they are short; the line of chunks
        out = torch.full((len(lens), H, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        got = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), ctx.cuda(), bound, SCALE, 2.0, 0.25,
                                       out=out)
        assert got.data_ptr() == out.data_ptr()
        _check_attention(out, q, kc, vc, bt, [1] * len(lens), lens, SCALE, 2.0, 0.25, 2.0 ** -11)


@pytest.mark.parametrize("H,Hk", [(28, 4), (40, 4)])   # 7 and 10 query heads a KV head
def test_decode_fp4_of_many_ragged_sequences(ops, H, Hk):
    """More pairs than SMs, some of them in dozens of parts, some in one, some empty."""
    lens = [int(x) for x in torch.randint(0, 300, (60,), generator=_gen(21))]
    lens[7], lens[8], lens[59] = 2000, 0, 1500
    kc, vc, bt = _paged(23, lens, Hk, 64)
    q = torch.randn(len(lens), H, D, generator=_gen(5)).to(torch.bfloat16)
    out = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(),
                                   torch.tensor(lens, dtype=torch.int32).cuda(), 2000, SCALE)
    _check_attention(out, q, kc, vc, bt, [1] * len(lens), lens, SCALE, 1.0, 1.0, 2.0 ** -11)


@pytest.mark.parametrize("size,qsize", [(300.0, 1e4), (2.0 ** -6, 2.0 ** -20), (1.0, 1e30)])
def test_decode_fp4_extreme_magnitudes(ops, size, qsize):
    """Keys at the ends of the scales' range, queries far outside f16's: the power of two that q
    is scaled by keeps both exact, and scores are as large or small as they should be."""
    lens, H, Hk = [300, 70], 8, 2
    kc, vc, bt = _paged(13, lens, Hk, 64, size=size)
    q = (qsize * torch.randn(2, H, D, generator=_gen(4))).to(torch.bfloat16)
    scale = min(1.0, 1.0 / (qsize * size))
    for bound in (512, 5000):
        out = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(),
                                       torch.tensor(lens, dtype=torch.int32).cuda(), bound, scale)
        _check_attention(out, q, kc, vc, bt, [1, 1], lens, scale, 1.0, 1.0, 2.0 ** -11)


@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_decode_fp4_zero_and_negative_scale(ops, scale):
    """A scale of 0 weighs every key alike; a negative one favours the least similar."""
    lens, H, Hk = [700, 65, 1], 8, 2
    kc, vc, bt = _paged(39, lens, Hk, 64)
    q = torch.randn(3, H, D, generator=_gen(10)).to(torch.bfloat16)
    out = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(),
                                   torch.tensor(lens, dtype=torch.int32).cuda(), np.int64(700), np.float32(scale))
    for i, n in enumerate(lens):
        k, v = (fp4.sequence(c.numpy(), bt[i].tolist(), n) for c in (kc, vc))
        ref, size = fp4.attend(q[i:i + 1].double().numpy(), k, v, float(np.float32(scale)))
        B = abs(scale) * float(np.abs(q[i].double().numpy()).max() * np.abs(k).sum(-1).max())
        bound = 2.0 ** -8 * np.abs(ref) + (2.0 ** -11 + 2.0 ** -14 * B + 2.0 ** -15) * size
        assert bool((np.abs(out[i:i + 1].double().cpu().numpy() - ref) <= bound).all())


def test_image_rows_move_layer_by_layer_in_4_bits(ops):
    """copy_image_kv_per_layer on its own stream gives copy_image_kv's bytes."""
    from vlcache_b200.engine import kv_cache as kvc
    kv = torch.stack([torch.stack([_pages(61 + 2 * x + y, 6, 2, 64) for x in range(3)]) for y in (0, 1)]).cuda()
    src, dst = kvc.image_reuse_slots(10, 140, 13, [3, 4, 5], 7, [0, 1, 2], 64)
    a, b = kv.clone(), kv.clone()
    kvc.copy_image_kv(a, src, dst, (3, 3, 3))
    events = kvc.copy_image_kv_per_layer(b, torch.from_numpy(src).cuda(), torch.from_numpy(dst).cuda(), (3, 3, 3),
                                         torch.cuda.Stream())
    for e in events:
        torch.cuda.current_stream().wait_event(e)
    assert len(events) == 3 and torch.equal(a, b) and not torch.equal(a, kv)


def test_decode_fp4_order_and_sharing_of_the_caches(ops):
    """K before V, V before K, and one cache for both give what each place holds."""
    lens, H, Hk = [400, 129], 16, 2
    kc, vc, bt = _paged(37, lens, Hk, 64, poison=False)
    q = torch.randn(2, H, D, generator=_gen(9)).to(torch.bfloat16)
    ctx = torch.tensor(lens, dtype=torch.int32).cuda()
    call = lambda k, v: ops.decode_attention_fp4(q.cuda(), k, v, bt.cuda(), ctx, 400, SCALE)  # noqa: E731
    a, b = torch.stack([kc, vc]).cuda(), torch.stack([vc, kc]).cuda()
    first, second = call(a[0], a[1]), call(b[1], b[0])
    assert torch.equal(first, second)
    _check_attention(first, q, kc, vc, bt, [1, 1], lens, SCALE, 1.0, 1.0, 2.0 ** -11)
    _check_attention(call(a[0], a[0]), q, kc, kc, bt, [1, 1], lens, SCALE, 1.0, 1.0, 2.0 ** -11)


def test_decode_fp4_flat_and_peaked(ops):
    """One key far above a flat rest: the rest's weights, 2^-26 of the peak each and below f16's
    smallest number, still add up (65536 of them are 2^-10 of the whole)."""
    n, block = 65537, 256
    x = np.zeros((n, 1, D))
    x[0, 0, 0] = 6.0
    pages = (n + block - 1) // block
    empty = np.zeros((pages, 1, block * 72), np.uint8)
    kc = torch.from_numpy(fp4.store(empty, x[:1], [0]))
    c, s = fp4.split_pages(empty)
    c[...], s[...] = 7, 0x38                                   # V: 6 everywhere
    c[0, :, 0], s[0, :, 0] = 0, 0                              # but 0 at the peak
    vc = torch.from_numpy(fp4.join_pages(c, s))
    q = torch.zeros(1, 1, D, dtype=torch.bfloat16)
    q[0, 0, 0] = 1.0
    scale = 26 * math.log(2) / 6
    bt = torch.arange(pages, dtype=torch.int32).view(1, -1)
    out = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(),
                                   torch.tensor([n], dtype=torch.int32).cuda(), n, scale)
    want = 6 * 65536 * 2.0 ** -26 / (1 + 65536 * 2.0 ** -26)
    # B = scale * |q k| = 18.1 in natural units; only the sizes count here
    assert bool(((out.double() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -14 * 18.1 + 2.0 ** -15)).all())


@pytest.mark.parametrize("bound", [256, 4096])
def test_decode_fp4_flags_bad_pages_and_lengths(ops, bound):
    kc, vc, bt = _paged(17, [256, 256], 1, 64, poison=False)
    q = torch.randn(2, 8, D, generator=_gen(5)).to(torch.bfloat16)
    lens = torch.tensor([256, 256], dtype=torch.int32).cuda()
    good = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), lens, bound, SCALE)
    bad = bt.clone()
    bad[1, 0], bad[1, 2] = -1, 10 ** 6
    out = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bad.cuda(), lens, bound, SCALE)
    assert ops.device_error(reset=True) == 102
    assert torch.equal(out[0], good[0])
    # the keys of the bad entries are left out
    left = torch.cat([bt[1, 1:2], bt[1, 3:4]]).view(1, 2)
    _check_attention(out[1:], q[1:], kc, vc, left, [1], [128], SCALE, 1.0, 1.0, 2.0 ** -11)
    lens[0] = 100000                                  # above what the grid was sized for
    out = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), lens, bound, SCALE)
    assert ops.device_error(reset=True) in (102, 104)
    assert bound > 256 or torch.equal(out[1], good[1])   # (a line of other shares adds in another order)


def test_decode_fp4_nan_key_reaches_its_own_sequence_only(ops):
    kc, vc, bt = _paged(19, [90, 90], 1, 64, poison=False)
    page = int(bt[1, 0])
    kc[page, 0, 64 * 64 + 5 * 8 + 2] = 0x7f                    # a NaN scale of key 5
    q = torch.randn(2, 4, D, generator=_gen(6)).to(torch.bfloat16)
    for bound in (128, 2048):
        out = ops.decode_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(),
                                       torch.tensor([90, 90], dtype=torch.int32).cuda(), bound, SCALE)
        assert bool(torch.isfinite(out[0]).all()) and bool(torch.isnan(out[1]).all())


def test_decode_fp4_strided_graph_streams(ops):
    """q and out rows inside wider buffers; the call captured in a graph and replayed with other
    lengths and tables; two graphs with workspaces of their own on two streams."""
    H, Hk, lens = 28, 4, [3000, 700, 1]
    kc, vc, bt = _paged(23, lens, Hk, 256)
    dk, dv = kc.cuda(), vc.cuda()
    wide = torch.randn(3, H * D + 64, generator=_gen(7)).to(torch.bfloat16).cuda()
    q = wide[:, :H * D].view(3, H, D)
    out_wide = torch.zeros(3, H * D + 8, dtype=torch.bfloat16, device="cuda")
    out = out_wide[:, :H * D].view(3, H, D)
    ctx, table = torch.tensor(lens, dtype=torch.int32).cuda(), bt.cuda()
    call = lambda o, w: ops.decode_attention_fp4(q, dk, dv, table, ctx, 3328, SCALE, out=o, workspace=w)  # noqa: E731
    ws = [torch.empty(ops.decode_fp4_workspace_bytes(3, H, Hk, 3328), dtype=torch.uint8, device="cuda") for _ in "ab"]
    assert ws[0].numel() > 0
    eager = call(None, None)
    assert torch.equal(call(out, ws[0]), eager) and not bool(out_wide[:, H * D:].any())
    graphs, outs, streams = [], [torch.zeros_like(eager) for _ in "ab"], [torch.cuda.Stream() for _ in "ab"]
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            call(outs[i], ws[i])
        graphs.append(graph)
    for new in (lens, [2999, 0, 256]):
        ctx.copy_(torch.tensor(new, dtype=torch.int32))
        want = call(None, None)
        torch.cuda.synchronize()
        for _ in range(5):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        # bit for bit: the third sequence reads on into rows of NaN at its second length
        assert np.array_equal(_bits(outs[0]), _bits(want)) and np.array_equal(_bits(outs[1]), _bits(want))
    del graphs


PREFILL = [  # H, Hk, block, (q_len, k_len)
    (16, 2, 256, [(1, 1)]),
    (28, 4, 256, [(1, 300), (17, 17), (64, 500), (5, 257)]),
    (16, 2, 128, [(130, 130), (48, 900), (1, 1024)]),
    (8, 8, 64, [(33, 65), (2, 2)]),
    (12, 1, 64, [(40, 200)]),
]


@pytest.mark.parametrize("H,Hk,block,lens", PREFILL)
def test_prefill_fp4(ops, H, Hk, block, lens):
    q_lens, k_lens = [a for a, _ in lens], [b for _, b in lens]
    kc, vc, bt = _paged(29, k_lens, Hk, block)
    cu_q, cu_k = np.concatenate([[0], np.cumsum(q_lens)]), np.concatenate([[0], np.cumsum(k_lens)])
    q = (2 * torch.randn(int(cu_q[-1]), H, D, generator=_gen(8))).to(torch.bfloat16)
    plan = ops.build_prefill_plan(cu_q, cu_k, H, Hk, device="cuda")
    cu = torch.tensor(cu_k, dtype=torch.int32).cuda()
    out = ops.prefill_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), cu, plan, SCALE, 0.5, 2.0)
    _check_attention(out, q, kc, vc, bt, q_lens, k_lens, SCALE, 0.5, 2.0, 2.0 ** -7)
    # exactly the bf16 attention over the read-back rows
    k, v = ops.gather_kvcache_fp4(kc.cuda(), vc.cuda(), bt.cuda(), cu, int(cu_k[-1]), 0.5, 2.0)
    assert torch.equal(out, ops.prefill_attention(q.cuda(), k, v, None, plan, SCALE))
    ws = torch.empty(ops.prefill_fp4_workspace_bytes(plan, Hk), dtype=torch.uint8, device="cuda")
    again = ops.prefill_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), cu, plan, SCALE, 0.5, 2.0, workspace=ws)
    assert torch.equal(out, again)


def test_long_cache_offsets_pass_32_bits(ops):
    """Pages beyond 4 GB of each cache: store, read back, attend, move and copy there."""
    hk, block = 4, 256
    pages = 60000                                       # 60000 * 73728 B = 4.4 GB
    kv = torch.zeros(2, 1, pages, hk, block * 72, dtype=torch.uint8, device="cuda")
    kc, vc = kv[0, 0], kv[1, 0]
    g = _gen(9)
    rows = torch.randn(300, hk, D, generator=g).to(torch.bfloat16).cuda()
    table = [pages - 1, pages - 3]
    slots = torch.tensor([table[i // block] * block + i % block for i in range(300)], dtype=torch.int32).cuda()
    ops.store_kvcache_fp4(rows, rows, kc, vc, slots)
    bt = torch.tensor([table], dtype=torch.int32).cuda()
    cu = torch.tensor([0, 300], dtype=torch.int32).cuda()
    k, v = ops.gather_kvcache_fp4(kc, vc, bt, cu, 300)
    c, s = fp4.quantise(rows.double().cpu().numpy())
    want = fp4.values(c, s)
    assert np.array_equal(k.double().cpu().numpy(), want) and torch.equal(k, v)
    q = torch.randn(1, 8, D, generator=g).to(torch.bfloat16)
    out = ops.decode_attention_fp4(q.cuda(), kc, vc, bt, cu[1:], 512, SCALE)
    ref, size = fp4.attend(q.double().numpy(), want, want, SCALE)
    assert bool((np.abs(out.double().cpu().numpy() - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -9 * size).all())
    near = torch.arange(300, dtype=torch.int32).cuda()
    ops.mrope_shift_fp4(kv, slots, near, (0, 0, 0))
    k2, v2 = ops.gather_kvcache_fp4(kc, vc, torch.tensor([[0, 1]], dtype=torch.int32).cuda(), cu, 300)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    ops.copy_kv_pages(kv, torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor([pages - 7, 5], dtype=torch.int32).cuda())
    assert torch.equal(kv[:, :, pages - 7], kv[:, :, pages - 1]) and torch.equal(kv[:, :, 5], kv[:, :, pages - 3])


# ------------------------------------------------------------------ moving reused rows
@pytest.mark.parametrize("rows,hk,layers,block,delta", [(1, 1, 1, 64, (5, 5, 5)), (70, 2, 3, 64, (-900, 0, 0)),
                                                        (33, 4, 2, 128, (0, 31, 7)), (200, 2, 1, 256, (0, 0, 0)),
                                                        (130, 1, 2, 64, (12345, -12345, 1))])
def test_shift_fp4_bytes(ops, rows, hk, layers, block, delta):
    half = (rows + block - 1) // block + 1
    kv = torch.stack([torch.stack([_pages(31 + 2 * x + y, 2 * half, hk, block) for x in range(layers)]) for y in (0, 1)])
    g = _gen(rows)
    src = torch.randperm(half * block, generator=g)[:rows]
    dst = torch.randperm(half * block, generator=g)[:rows] + half * block
    dev = kv.cuda()
    ops.mrope_shift_fp4(dev, src.to(torch.int32).cuda(), dst.to(torch.int32).cuda(), delta)
    cos, sin = omr.shift_table(delta)
    turned = np.repeat([any(delta[0 if j < 16 else 1 if j < 40 else 2] for j in range(16 * m, 16 * m + 16))
                        for m in range(4)] * 2, 16)
    for layer in range(layers):
        for which in (0, 1):
            codes, scale = (a.copy() for a in fp4.split_pages(kv[which, layer].numpy()))
            c = codes[src // block, :, src % block]
            s = scale[src // block, :, src % block]
            if which == 0:
                x = fp4.values(c, s).astype(np.float32)
                x1, x2 = x[..., :64], x[..., 64:]
                y = np.concatenate([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)    # fp32, op by op
                y = omr.bf16_bits_to_f32(omr.f32_to_bf16_bits(y)).astype(np.float64)
                nc, ns = fp4.quantise(y)
                c = np.where(turned, nc, c)
                s = np.where(turned[::16], ns, s)
            codes[dst // block, :, dst % block], scale[dst // block, :, dst % block] = c, s
            have = fp4.split_pages(dev[which, layer].cpu().numpy())
            assert np.array_equal(have[1], scale)
            same = (have[0] == codes) | ((have[0] & 7 == 0) & (codes & 7 == 0))
            assert bool(same.all())


def test_shift_fp4_in_place_and_per_layer(ops):
    """In place turns K where it lies and leaves V; a layer alone gives the bytes of all layers."""
    kv = torch.stack([torch.stack([_pages(41 + 2 * x + y, 3, 2, 64) for x in range(2)]) for y in (0, 1)]).cuda()
    slots = torch.arange(10, 90, dtype=torch.int32).cuda()
    away = slots + 92
    moved, placed = kv.clone(), kv.clone()
    ops.mrope_shift_fp4(moved, slots, away, (3, 5, 7))
    ops.mrope_shift_fp4(placed, slots, None, (3, 5, 7))
    assert torch.equal(placed[1], kv[1])
    cu = torch.tensor([0, 192], dtype=torch.int32).cuda()
    bt = torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda()
    a, _ = ops.gather_kvcache_fp4(moved[0], moved[1], bt, cu, 192)
    b, _ = ops.gather_kvcache_fp4(placed[0], placed[1], bt, cu, 192)
    assert torch.equal(a[:, 102:182], b[:, 10:90])
    for layer in range(2):
        one = kv.clone()
        ops.mrope_shift_layer_fp4(one[0, layer], one[1, layer], slots, away, (3, 5, 7))
        assert torch.equal(one[:, layer], moved[:, layer]) and torch.equal(one[:, 1 - layer], kv[:, 1 - layer])
    ops.mrope_shift_fp4(kv, torch.tensor([0, -1, 192], dtype=torch.int32).cuda(), None, (1, 1, 1))
    assert ops.device_error(reset=True) == 101


# ------------------------------------------------------------------ pages
@pytest.mark.parametrize("shape,dtype", [((2, 3, 9, 64, 2, 128), torch.bfloat16), ((2, 2, 9, 4, 128 * 72), torch.uint8),
                                         ((2, 1, 9, 16), torch.uint8), ((2, 1, 12, 5, 7, 16), torch.float16)])
def test_copy_kv_pages(ops, shape, dtype):
    cache = torch.randint(0, 256, (math.prod(shape) * dtype.itemsize,), dtype=torch.uint8, generator=_gen(2))
    cache = cache.cuda().view(dtype).view(shape)
    raw = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    src = torch.tensor([0, 3, 0, -1, 8], dtype=torch.int32).cuda()     # one page twice, a padding pair, onto itself
    dst = torch.tensor([1, 5, 2, -1, 8], dtype=torch.int32).cuda()
    want = cache.clone()
    want[:, :, [1, 5, 2]] = want[:, :, [0, 3, 0]]
    ops.copy_kv_pages(cache, src, dst)
    assert torch.equal(raw(cache), raw(want))
    ops.copy_kv_pages(cache, src[:0], dst[:0])
    before = raw(cache).clone()
    ops.copy_kv_pages(cache, torch.tensor([0, shape[2], -2], dtype=torch.int32).cuda(),
                      torch.tensor([shape[2], 1, 1], dtype=torch.int32).cuda())
    assert ops.device_error(reset=True) == 102
    assert torch.equal(raw(cache), before)


def test_remap_block_tables(ops):
    g = _gen(3)
    wide = torch.randint(-1, 50, (7, 40), generator=g, dtype=torch.int32)
    page_map = torch.randperm(50, generator=g).to(torch.int32)
    want = torch.where(wide >= 0, page_map[wide.clamp(min=0).long()], wide)
    dev = wide.cuda()
    part = dev[:, 3:36]
    ops.remap_block_tables(part, page_map.cuda())
    assert torch.equal(dev[:, 3:36].cpu(), want[:, 3:36])
    assert torch.equal(dev[:, :3].cpu(), wide[:, :3]) and torch.equal(dev[:, 36:].cpu(), wide[:, 36:])
    bad = torch.tensor([[50, -2, 1]], dtype=torch.int32).cuda()
    ops.remap_block_tables(bad, page_map.cuda())
    assert ops.device_error(reset=True) == 102
    assert bad.tolist() == [[50, -2, int(page_map[1])]]


# ------------------------------------------------------------------ refusals of the ops
def test_ops_refusals(ops):
    x = torch.zeros(2, 2, D, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(2, 4, D, dtype=torch.bfloat16, device="cuda")
    c = torch.zeros(2, 2, 64 * 72, dtype=torch.uint8, device="cuda")
    s = torch.zeros(2, dtype=torch.int32, device="cuda")
    t = torch.zeros(8, D, device="cuda")
    pos = torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    bt = s.view(2, 1)
    bad = [
        lambda: ops.store_kvcache_fp4(x.float(), x, c, c, s),
        lambda: ops.store_kvcache_fp4(x, x[:1], c, c, s),
        lambda: ops.store_kvcache_fp4(x, x, c, c[:1], s),
        lambda: ops.store_kvcache_fp4(x, x, c[:, :1], c[:, :1], s),
        lambda: ops.store_kvcache_fp4(x, x, c, c, s[:1]),
        lambda: ops.store_kvcache_fp4(x, x, c, c, s.long()),
        lambda: ops.store_kvcache_fp4(x, x, c[..., :100], c[..., :100], s),
        lambda: ops.store_kvcache_fp4(x.transpose(1, 2), x, c, c, s),
        lambda: ops.store_kvcache_fp4(x, x, c, c, s.cpu()),
        lambda: ops.rope_store_kvcache_fp4(pos, q, x, x, t, c, c, s),                       # three axes, no section
        lambda: ops.rope_store_kvcache_fp4(pos[:2], q, x, x, t, c, c, s, (16, 24, 24)),
        lambda: ops.rope_store_kvcache_fp4(pos.int(), q, x, x, t, c, c, s, (16, 24, 24)),
        lambda: ops.rope_store_kvcache_fp4(pos, q, x, x, t.half(), c, c, s, (16, 24, 24)),
        lambda: ops.rope_store_kvcache_fp4(pos, q, x, x, t, c, c, s, (16, 24, 24), out=x),
        lambda: ops.mrope_store_kvcache(pos, q, x, x, t, c, c, s),                          # not a bf16 cache
        lambda: ops.decode_attention_fp4(q, c, c, bt[:1], s, 64, 0.1),
        lambda: ops.decode_attention_fp4(q, c, c, bt.long(), s, 64, 0.1),
        lambda: ops.decode_attention_fp4(q, c, c, bt, s[:1], 64, 0.1),
        lambda: ops.decode_attention_fp4(q.view(1, 2, 4, D), c, c, bt, s, 64, 0.1),
        lambda: ops.gather_kvcache_fp4(c, c, bt, s, 4),                                     # one sequence, two tables
        lambda: ops.gather_kvcache_fp4(c, c, bt[:1], s, 4, k_out=x),
        lambda: ops.mrope_shift_fp4(c, s, s, (1, 1, 1)),
        lambda: ops.mrope_shift_layer_fp4(c, c, s, s[:1], (1, 1, 1)),
        lambda: ops.copy_kv_pages(c.view(2, 1, 2, -1)[:, :, :1], s, s),
        lambda: ops.copy_kv_pages(c.view(2, 1, 2, -1), s, s[:1]),
        lambda: ops.remap_block_tables(bt.long(), s),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print(i)
    for call in (lambda: ops.store_kvcache_fp4(x, x, c, c, s, k_scale=3.0),
                 lambda: ops.decode_attention_fp4(q[:, :3].contiguous(), c, c, bt, s, 64, 0.1),
                 lambda: ops.mrotary_embedding(pos, q, x, t, (16, 24, 25))):
        with pytest.raises(RuntimeError):
            call()
    # no tokens, no rows: nothing to do
    ops.store_kvcache_fp4(x[:0], x[:0], c, c, s[:0])
    assert ops.decode_attention_fp4(q[:0], c, c, bt[:0], s[:0], 64, 0.1).shape == (0, 4, D)
    assert not bool(c.any())


def test_bounds_outside_32_bits_are_refused(ops):
    q = torch.zeros(1, 2, D, dtype=torch.bfloat16, device="cuda")
    c = torch.zeros(1, 2, 64 * 72, dtype=torch.uint8, device="cuda")
    s = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bound in (-1, 2 ** 30 + 1, 2 ** 32 + 64):
        with pytest.raises(ValueError):
            ops.decode_attention_fp4(q, c, c, s.view(1, 1), s, bound, 0.1)


def test_page_copies_of_host_lists_are_not_captured(ops):
    from vlcache_b200.engine import kv_cache as kvc
    kv = torch.arange(2 * 4 * 64 * 72, device="cuda").to(torch.uint8).view(2, 1, 4, 1, 64 * 72)
    src, dst = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (1, 3))
    before = kv.clone()
    ops.copy_kv_pages(kv, dst, dst)   # (loads the kernel)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            kvc.copy_pages(kv, [1], [3])
        ops.copy_kv_pages(kv, src, dst)
    graph.replay()
    before[:, :, 3] = before[:, :, 1]
    assert torch.equal(kv, before)


# ------------------------------------------------------------------ together, as an engine runs them
@pytest.mark.parametrize("axes", [1, 3])
def test_attention_layers_over_a_4bit_cache(ops, axes):
    """A cold prompt, a warm request whose image rows are reused from it, a fork of that request
    and a decode step of both, through Attention, the metadata builder, the image move and the
    page pool.  The 4-bit cache is followed byte by byte with the ops by themselves, and the
    outputs are those of the bf16 layer over the read-back values where it computes the same."""
    from vlcache_b200.engine import kv_cache as kvc
    from vlcache_b200.engine.page_pool import PagePool
    from vlcache_b200.layers.attention import Attention
    from vlcache_b200.layers.rotary_embedding import get_mrope, get_rope, image_position_delta
    from vlcache_b200.utils import context as ctx
    H, Hk, L = 16, 2, 1
    g = _gen(51)
    attn = Attention(H, D, SCALE, Hk)
    holder = torch.nn.ModuleList([attn])
    kv = kvc.allocate_kv_cache(holder, L, 16, Hk, kv_format="fp4")
    kv.zero_()
    attn.k_scale, attn.v_scale = 1.0, 0.25
    rot = (get_mrope(D, D, 4096, 1e6) if axes == 3 else get_rope(D, D, 4096, 1e6)).cuda()
    widen = (lambda p: p.repeat(3, 1)) if axes == 3 else (lambda p: p)  # noqa: E731
    pool = PagePool(16)

    def rows(n):
        x = torch.randn(n, H + 2 * Hk, D, generator=g).to(torch.bfloat16).cuda()
        return x.split((H, Hk, Hk), 1)

    def gathered(table, n):
        return ops.gather_kvcache_fp4(attn.k_cache, attn.v_cache, torch.tensor([table], dtype=torch.int32).cuda(),
                                      torch.tensor([0, n], dtype=torch.int32).cuda(), n, attn.k_scale, attn.v_scale)

    builder = kvc.WarmPrefillBuilder(H, Hk)
    # cold: the step's own K and V in bf16; the cache gets their quantised rows
    old = pool.allocate(pool.pages_for(420))
    batch = builder.upload(builder.build([kvc.WarmRequest(420, old)]))
    q, k, v = rows(420)
    o = attn(q, k, v, positions=widen(batch.device_tensors["positions"]), rotary_emb=rot)
    q_rot, k_rot = rot(widen(batch.device_tensors["positions"]), q, k)
    assert torch.equal(o, ops.prefill_attention(q_rot, k_rot, v, None, batch.plan, SCALE))
    gk, gv = gathered(old, 420)
    c, s = fp4.quantise(k_rot.double().cpu().numpy())
    assert np.array_equal(gk.double().cpu().numpy(), fp4.values(c, s))
    c, s = fp4.quantise(v.double().cpu().numpy(), 0.25)
    assert np.array_equal(gv.double().cpu().numpy(), fp4.values(c, s, 0.25))
    # warm: the image (rows 20..400 of the old request) at 53.. of a new one, 40 of its rows again
    n, start, end, R = 460, 53, 433, 40
    new = pool.allocate(pool.pages_for(n))
    src, dst = kvc.image_reuse_slots(start, end, R, new, 20, old)
    kvc.copy_image_kv(kv, src, dst, image_position_delta(20, start))
    batch = builder.upload(builder.build([kvc.WarmRequest(n, new, start, end, R, True)]))
    q, k, v = rows(int(batch.cu_seqlens_q[-1]))
    pos = widen(batch.device_tensors["positions"])
    o = attn(q, k, v, positions=pos, rotary_emb=rot)
    gk, gv = gathered(new, n)
    a = start + R
    both = [torch.cat([x[:a], x]) for x in (gk, gv)]
    assert torch.equal(o, ops.prefill_attention(rot(pos, q, k)[0], *both, None, batch.plan, SCALE))
    assert torch.equal(gv[start + R:end], gathered(old, 420)[1][20 + R:400])       # moved V rows as they were
    # fork, then one decode step of both requests
    forked, copies = pool.fork(new, n)
    assert len(copies) == 1
    kvc.copy_pages(kv, *zip(*copies))
    assert all(torch.equal(x, y) for x, y in zip(gathered(forked, n), (gk, gv)))
    positions = kvc.prepare_decode([n + 1, n + 1], [new, forked])
    q, k, v = rows(2)
    o = attn(q, k, v, positions=widen(positions), rotary_emb=rot)
    assert o.shape == (2, 1, H, D)
    q_rot = rot(widen(positions), q, k)[0]
    for i, table in enumerate((new, forked)):
        gk2, gv2 = gathered(table, n + 1)
        assert torch.equal(gk2[:n], gk) and torch.equal(gv2[:n], gv)
        ref, size = fp4.attend(q_rot[i:i + 1].double().cpu().numpy(), gk2.double().cpu().numpy(),
                               gv2.double().cpu().numpy(), SCALE)
        B = SCALE * float((q_rot[i].double().abs().max() * gk2.double().abs().sum(-1).max()))
        bound = 2.0 ** -8 * np.abs(ref) + (2.0 ** -11 + 2.0 ** -14 * B + 2.0 ** -15) * size
        assert bool((np.abs(o[i].double().cpu().numpy() - ref) <= bound).all())
    # the old request ends; compaction moves pages, the tables follow, the values stay
    pool.free(old)
    moved_src, moved_dst, page_map = pool.compact()
    assert len(moved_src) > 0
    kvc.copy_pages(kv, moved_src, moved_dst)
    table = torch.tensor([new], dtype=torch.int32).cuda()
    ops.remap_block_tables(table, torch.from_numpy(page_map).cuda())
    assert all(torch.equal(x[:n], y) for x, y in zip(gathered(table[0].tolist(), n + 1), (gk, gv)))
    ctx.reset_context()


def test_projection_into_a_4bit_cache(ops):
    """QKVParallelLinear.forward_rope_store with a 4-bit cache and with several axes: what the
    projection, the rotation and the scatter give one by one."""
    from vlcache_b200.engine.kv_cache import allocate_kv_cache
    from vlcache_b200.layers.attention import Attention
    from vlcache_b200.layers.linear import QKVParallelLinear
    from vlcache_b200.layers.rotary_embedding import get_mrope
    from vlcache_b200.utils import context as ctx
    H, Hk, hidden, n = 4, 2, 256, 9
    g = _gen(61)
    lin = QKVParallelLinear(hidden, D, H, Hk, bias=True)
    lin.weight.data = torch.randn(lin.weight.shape, generator=g).to(torch.bfloat16).mul_(0.05).cuda()
    lin.bias.data = torch.randn(lin.bias.shape, generator=g).to(torch.bfloat16).cuda()
    x = torch.randn(n, hidden, generator=g).to(torch.bfloat16).cuda()
    pos = torch.randint(0, 100, (3, n), generator=g).cuda()
    rot = get_mrope(D, D, 128, 1e6).cuda()
    slots = torch.randperm(256, generator=g)[:n].to(torch.int32).cuda()
    ctx.set_context(False, slot_mapping=slots)
    for fmt in ("fp4", "bf16"):
        attn = Attention(H, D, SCALE, Hk)
        kv = allocate_kv_cache(torch.nn.ModuleList([attn]), 1, 1, Hk, kv_format=fmt)
        kv.zero_()
        out = lin.forward_rope_store(x, pos, rot, attn)
        q, k, v = lin(x).view(n, H + 2 * Hk, D).split((H, Hk, Hk), 1)
        q_rot, k_rot = rot(pos, q, k)
        other = torch.zeros_like(kv)
        if fmt == "fp4":
            ops.store_kvcache_fp4(k_rot, v, other[0, 0], other[1, 0], slots)
        else:
            ops.store_kvcache(k_rot, v.contiguous(), other[0, 0], other[1, 0], slots)
        assert torch.equal(out, q_rot) and torch.equal(kv, other)
    ctx.reset_context()


# ------------------------------------------------------------------ calls at the ends of their ranges
@pytest.mark.parametrize("seqs,H,Hk", [(1, 16, 2), (64, 28, 4), (100, 32, 2)])
def test_decode_fp4_zero_bound(ops, seqs, H, Hk):
    """All sequences empty and a bound of 0, with fewer and with more pairs than SMs: zeros."""
    c = torch.full((1, Hk, 64 * 72), 255, dtype=torch.uint8, device="cuda")
    q = torch.randn(seqs, H, D, generator=_gen(1)).to(torch.bfloat16).cuda()
    lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    bt = torch.full((seqs, 1), -1, dtype=torch.int32, device="cuda")
    out = torch.full((seqs, H, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(ops.decode_fp4_workspace_bytes(seqs, H, Hk, 0), dtype=torch.uint8, device="cuda")
    for w in (None, ws):
        ops.decode_attention_fp4(q, c, c, bt, lens, 0, SCALE, out=out, workspace=w)
        assert not bool(out.any())           # (a NaN counts as true)
        out.fill_(float("nan"))


def test_copy_kv_pages_of_a_large_pool(ops):
    """More pairs than a grid has rows (65535): a compaction of a pool of small pages, bad pairs and
    padding behind that border among them."""
    n = 140010
    cache = torch.randint(0, 256, (2, 2, n, 32), dtype=torch.uint8, generator=_gen(4)).cuda()
    src = torch.arange(n - 70000, n, dtype=torch.int32, device="cuda")
    dst = torch.randperm(n - 70000, generator=_gen(5))[:70000].to(torch.int32).cuda()
    good = torch.ones(70000, dtype=torch.bool, device="cuda")
    good[69990:69993] = False
    want = cache.clone()
    want[:, :, dst[good].long()] = cache[:, :, src[good].long()]
    src[69990], dst[69991] = n, -3
    src[69992] = dst[69992] = -1
    ops.copy_kv_pages(cache, src, dst)
    assert ops.device_error(reset=True) == 102
    assert torch.equal(cache, want)


@pytest.mark.parametrize("H,Hk", [(8, 2), (20, 2)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_decode_fp4_non_finite_query(ops, H, Hk, bad):
    """A head whose query holds an infinity has scores of +-infinity or NaN only, and a softmax of
    those is NaN, all of them -infinity included (the keys have one sign where q is infinite).  The
    other heads keep their bits, and a sequence without keys its zeros."""
    lens, block = [700, 0, 65], 64
    r = np.random.default_rng(7)
    x = -np.abs(r.normal(size=(14, Hk, block, D))) - 0.5
    kc = torch.from_numpy(fp4.join_pages(*fp4.quantise(x)))
    vc = _pages(8, 14, Hk, block)
    bt = torch.arange(14, dtype=torch.int32)
    bt = torch.stack([bt[:11], torch.full((11,), -1, dtype=torch.int32), torch.cat([bt[11:13], bt[:1].expand(9)])]).cuda()
    ctx = torch.tensor(lens, dtype=torch.int32).cuda()
    q = torch.randn(3, H, D, generator=_gen(9)).to(torch.bfloat16).cuda()
    for bound in (704, 5000):
        call = lambda x: ops.decode_attention_fp4(x, kc.cuda(), vc.cuda(), bt, ctx, bound, SCALE)  # noqa: E731
        good, other = call(q), q.clone()
        other[:, 1, 0], other[:, H - 1, 3] = bad, bad
        out = call(other)
        assert not bool(out[1].any())
        hit = torch.zeros(H, dtype=torch.bool)
        hit[1] = hit[H - 1] = True
        for i in (0, 2):
            assert bool(torch.isnan(out[i, hit]).all())
            assert bool(torch.isfinite(good[i]).all()) and torch.equal(out[i, ~hit], good[i, ~hit])


# ------------------------------------------------------------------ every scale and magnitude on the device
def _sweep_rows(groups):
    """bf16 rows [n, 1, 128] of groups of 16 (float32 values that bf16 holds), the last row filled up."""
    flat = np.concatenate(groups).astype(np.float32)
    flat = np.concatenate([flat, np.zeros(-len(flat) % D, np.float32)])
    return torch.from_numpy(flat).view(-1, 1, D).to(torch.bfloat16)


def _sweep_codes():
    """For each scale s: groups whose largest element is 6 s (which makes the scale s) and whose others
    sweep the bf16 magnitudes from 2^-4 s (below, the code is 0) to 6 s, in both signs."""
    mags = (np.arange(0x7f80, dtype=np.uint32) << 16).view(np.float32)
    out = []
    for s in fp4.E4M3[1:]:
        y = mags[(mags >= s / 16) & (mags <= 6 * s)]
        y = np.concatenate([y, -y, np.zeros(-2 * len(y) % 15, np.float32)]).reshape(-1, 15)
        out.append(np.concatenate([np.full((len(y), 1), 6 * s), y], 1).ravel())
    return _sweep_rows(out)


def _sweep_scales():
    """A group for each bf16 magnitude, as its largest element among smaller ones."""
    mags = (np.arange(0x7f80, dtype=np.uint32) << 16).view(np.float32)
    part = (np.arange(16) % 8 / 8.0 * np.where(np.arange(16) < 8, 1, -1)).astype(np.float32)
    part[0] = 1.0
    x = torch.from_numpy(mags[:, None] * part[None]).to(torch.bfloat16).float().numpy()
    return _sweep_rows([x.ravel()])


@pytest.mark.parametrize("sweep", [_sweep_codes, _sweep_scales])
@pytest.mark.parametrize("g", [1.0, 2.0 ** -5])
def test_store_fp4_over_every_scale_and_magnitude(ops, sweep, g):
    x = sweep()
    n, block = x.shape[0], 64
    rows = (x.float() * g).to(torch.bfloat16)
    pages = (n + block - 1) // block
    kc, vc = (torch.zeros(pages, 1, block * 72, dtype=torch.uint8, device="cuda") for _ in "kv")
    slots = torch.randperm(pages * block, generator=_gen(n))[:n].to(torch.int32)
    ops.store_kvcache_fp4(rows.cuda(), -rows.cuda(), kc, vc, slots.cuda(), g, g)
    at = slots.long()
    for cache, sign in ((kc, 1.0), (vc, -1.0)):
        codes, scale = (a[at // block, :, at % block] for a in fp4.split_pages(cache.cpu().numpy()))
        want_codes, want_scale = fp4.quantise(sign * rows.double().numpy(), g)
        assert np.array_equal(scale, want_scale)
        zero = (codes & 7 == 0) & (want_codes & 7 == 0)
        assert bool(((codes == want_codes) | zero).all())


# ------------------------------------------------------------------ axes that differ, through the layers
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
def test_attention_layers_at_image_positions(ops, fmt):
    """A cold prompt with an image, a warm request that reuses the image further on, and a decode
    step, with (time, height, width) positions that differ between the axes: the cache holds the
    oracle's rotated rows, and the outputs are those of the attention over what the cache holds.
    The moved rows are what new rows at their new positions would be: two bf16 roundings of the pair
    (x1, x2) of radius r before the last turn's own, each 2^-8 of a component, give 2^-8 sqrt(2) r +
    2 * 2^-8 |z|, and the fp32 angles 2^-16 r."""
    from vlcache_b200.engine import kv_cache as kvc
    from vlcache_b200.layers.attention import Attention
    from vlcache_b200.layers.rotary_embedding import get_mrope, image_position_delta
    from vlcache_b200.utils import context as ctx
    H, Hk, gh, gw = 16, 2, 13, 17
    image = gh * gw
    g = _gen(71)
    attn = Attention(H, D, SCALE, Hk)
    kv = kvc.allocate_kv_cache(torch.nn.ModuleList([attn]), 1, 8, Hk, kv_format=fmt)
    kv.zero_()
    rot = get_mrope(D, D, 512, 1e6, [16, 24, 24])
    table = rot.cos_sin_cache.cpu()
    rot = rot.cuda()

    def positions(start, tail):     # text, the image from `start` on, text from the image's largest position on
        return torch.from_numpy(np.concatenate([omr.text_positions(0, start), omr.vision_positions(start, gh, gw),
                                                omr.text_positions(start + max(gh, gw), tail)], 1))

    def rows(n):
        return torch.randn(n, H + 2 * Hk, D, generator=g).to(torch.bfloat16).cuda().split((H, Hk, Hk), 1)

    def bf16(bits):
        return torch.from_numpy(bits.view(np.int16).copy()).view(torch.bfloat16).cuda()

    def held(x):                    # a row as the cache holds it
        if fmt == "bf16":
            return x
        return torch.from_numpy(fp4.values(*fp4.quantise(x.double().cpu().numpy()))).to(torch.bfloat16).cuda()

    def cached(pages, n):
        if fmt == "fp4":
            return ops.gather_kvcache_fp4(attn.k_cache, attn.v_cache, torch.tensor([pages], dtype=torch.int32).cuda(),
                                          torch.tensor([0, n], dtype=torch.int32).cuda(), n)
        return [c[pages].flatten(0, 1)[:n] for c in (attn.k_cache, attn.v_cache)]

    builder = kvc.WarmPrefillBuilder(H, Hk)
    # cold: 20 rows of text, the image, 30 rows of text
    n = 20 + image + 30
    old = [6, 1]
    batch = builder.upload(builder.build([kvc.WarmRequest(n, old)]))
    pos, (q, k, v) = positions(20, 30), rows(n)
    assert len(set(map(tuple, pos.T.tolist()))) > image and bool((pos[0] != pos[1]).any())
    o = attn(q, k, v, positions=pos.cuda(), rotary_emb=rot)
    q_rot, k_rot = (bf16(_axes_reference(x.cpu(), pos, (16, 24, 24), table)) for x in (q, k))
    assert torch.equal(o, ops.prefill_attention(q_rot, k_rot, v.contiguous(), None, batch.plan, SCALE))
    for got, want in zip(cached(old, n), (k_rot, v)):
        assert torch.equal(got, held(want))
    raw_k, old_k = k, k_rot
    # warm: the image from row 53 on, 40 of its rows again
    start, again = 53, 40
    n, new = start + image + 25, [0, 4]
    src, dst = kvc.image_reuse_slots(start, start + image, again, new, 20, old)
    kvc.copy_image_kv(kv, src, dst, image_position_delta(20, start))
    batch = builder.upload(builder.build([kvc.WarmRequest(n, new, start, start + image, again, True)]))
    pos = positions(start, 25)
    fresh = torch.cat([torch.arange(start + again), torch.arange(start + image, n)])
    q, k, v = rows(len(fresh))
    o = attn(q, k, v, positions=pos[:, fresh].contiguous().cuda(), rotary_emb=rot)
    q_rot, k_rot = (bf16(_axes_reference(x.cpu(), pos[:, fresh], (16, 24, 24), table)) for x in (q, k))
    ck, cv = cached(new, n)
    for got, want in ((ck, k_rot), (cv, v)):
        assert torch.equal(got[fresh.cuda()], held(want))
    both = [torch.cat([x[:start + again], x]) for x in (ck, cv)]
    assert torch.equal(o, ops.prefill_attention(q_rot, *both, None, batch.plan, SCALE))
    if fmt == "bf16":
        mine = slice(start + again, start + image)
        x = raw_k[20 + again:20 + image].float()
        z = bf16(_axes_reference(x.to(torch.bfloat16).cpu(), pos[:, mine], (16, 24, 24), table)).float()
        r = (x ** 2 + omr.rotate_half(x) ** 2).sqrt()
        bound = 2.0 ** -8 * (math.sqrt(2) * r * 1.01 + 2 * z.abs() * 1.01) + 2.0 ** -16 * r
        assert bool(((ck[mine].float() - z).abs() <= bound).all())
        assert not torch.equal(ck[mine], old_k[20 + again:20 + image])
    # decode: one token further, its axes apart
    kvc.prepare_decode([n + 1], [new])
    pos = torch.tensor([[90], [71], [85]])
    q, k, v = rows(1)
    o = attn(q, k, v, positions=pos.cuda(), rotary_emb=rot)
    q_rot, k_rot = (bf16(_axes_reference(x.cpu(), pos, (16, 24, 24), table)) for x in (q, k))
    ck2, cv2 = cached(new, n + 1)
    assert torch.equal(ck2[:n], ck) and torch.equal(cv2[:n], cv)
    assert torch.equal(ck2[n:], held(k_rot)) and torch.equal(cv2[n:], held(v))
    bt, lens = torch.tensor([new], dtype=torch.int32).cuda(), torch.tensor([n + 1], dtype=torch.int32).cuda()
    decode = ops.decode_attention_fp4 if fmt == "fp4" else ops.decode_attention
    assert torch.equal(o[:, 0], decode(q_rot, attn.k_cache, attn.v_cache, bt, lens, ctx.get_context().max_context_len
                                       or 512, SCALE))
    ctx.reset_context()


# ------------------------------------------------------------------ forms that the tests above leave out
@pytest.mark.parametrize("block", [192, 320])
def test_blocks_that_are_no_power_of_two(ops, block):
    """Store, read back, attend (both decode kernels and the prefill), move and copy in pages of a
    multiple of 64 rows that is no power of two."""
    H, Hk, lens = 12, 3, [700, 1, 383]
    kc, vc, bt = _paged(81, lens, Hk, block)
    cu_k = np.concatenate([[0], np.cumsum(lens)])
    cu = torch.tensor(cu_k, dtype=torch.int32).cuda()
    q = torch.randn(3, H, D, generator=_gen(1)).to(torch.bfloat16)
    ctx = torch.tensor(lens, dtype=torch.int32).cuda()
    dk, dv, dbt = kc.cuda(), vc.cuda(), bt.cuda()
    for bound in (700, 5000):
        out = ops.decode_attention_fp4(q.cuda(), dk, dv, dbt, ctx, bound, SCALE)
        _check_attention(out, q, kc, vc, bt, [1] * 3, lens, SCALE, 1.0, 1.0, 2.0 ** -11)
    q_lens = [40, 1, 300]
    plan = ops.build_prefill_plan(np.concatenate([[0], np.cumsum(q_lens)]), cu_k, H, Hk, device="cuda")
    q = torch.randn(sum(q_lens), H, D, generator=_gen(2)).to(torch.bfloat16)
    out = ops.prefill_attention_fp4(q.cuda(), dk, dv, dbt, cu, plan, SCALE)
    _check_attention(out, q, kc, vc, bt, q_lens, lens, SCALE, 1.0, 1.0, 2.0 ** -7)
    # rows stored over the first sequence's, on both sides of its page borders, then read back
    rows = torch.randn(300, Hk, D, generator=_gen(3)).to(torch.bfloat16)
    at = torch.arange(150, 450)
    slots = (bt[0].long()[at // block] * block + at % block).to(torch.int32)
    kv = torch.stack([dk, dv]).unsqueeze(1)
    ops.store_kvcache_fp4(rows.cuda(), rows.cuda(), kv[0, 0], kv[1, 0], slots.cuda())
    k, v = ops.gather_kvcache_fp4(kv[0, 0], kv[1, 0], dbt, cu, int(cu_k[-1]))
    want = fp4.values(*fp4.quantise(rows.double().numpy()))
    assert np.array_equal(k[150:450].double().cpu().numpy(), want) and torch.equal(k[150:450], v[150:450])
    assert np.array_equal(k[:150].double().cpu().numpy(), fp4.sequence(kc.numpy(), bt[0].tolist(), 150))
    # moved without a turn to pages of their own, and those pages copied
    free = [p for p in range(kc.shape[0]) if p not in bt.tolist()[0][:3]][:2]
    if 2 * block >= 300:
        to = (torch.tensor(free)[torch.arange(300) // block] * block + torch.arange(300) % block).to(torch.int32)
        ops.mrope_shift_fp4(kv, slots.cuda(), to.cuda(), (0, 0, 0))
        moved, _ = ops.gather_kvcache_fp4(kv[0, 0], kv[1, 0], torch.tensor([free], dtype=torch.int32).cuda(),
                                          torch.tensor([0, 300], dtype=torch.int32).cuda(), 300)
        assert torch.equal(moved, k[150:450])
    page = kv[:, :, free[0]].clone()
    ops.copy_kv_pages(kv, torch.tensor(free[:1], dtype=torch.int32).cuda(), torch.tensor(free[1:], dtype=torch.int32).cuda())
    assert torch.equal(kv[:, :, free[1]], page)


def test_gather_fp4_into_outputs_of_16_byte_alignment(ops):
    kc, vc, bt = _paged(83, [200, 70], 2, 64)
    cu = torch.tensor([0, 200, 270], dtype=torch.int32).cuda()
    want = ops.gather_kvcache_fp4(kc.cuda(), vc.cuda(), bt.cuda(), cu, 270, 2.0, 0.5)
    for a, b in ((8, 0), (0, 8), (8, 8)):
        outs = [torch.full((270 * 2 * D + 24,), 7.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
        k, v = outs[0][a:a + 270 * 2 * D].view(270, 2, D), outs[1][b:b + 270 * 2 * D].view(270, 2, D)
        assert (k.data_ptr() | v.data_ptr()) % 32 == 16
        ops.gather_kvcache_fp4(kc.cuda(), vc.cuda(), bt.cuda(), cu, 270, 2.0, 0.5, k, v)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
        assert bool((outs[0][a + 270 * 2 * D:] == 7).all()) and bool((outs[1][b + 270 * 2 * D:] == 7).all())


@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
def test_rotary_of_many_tokens_in_place(ops, fmt):
    """A prompt's q rotated where it lies, in the projection's rows, is the q of a separate output."""
    from vlcache_b200.layers.rotary_embedding import rope_cos_sin_cache
    N, H, Hk = 6011, 28, 4
    g = _gen(91)
    table = rope_cos_sin_cache(D, 1024, 1e6).cuda()
    pos = torch.randint(0, 1024, (3, N), generator=g).cuda()
    qkv = torch.randn(N, H + 2 * Hk, D, generator=g).to(torch.bfloat16).cuda()
    slots = torch.randperm(24 * 256, generator=g)[:N].to(torch.int32).cuda()
    shape, dtype = ((24, 256, Hk, D), torch.bfloat16) if fmt == "bf16" else ((24, Hk, 256 * 72), torch.uint8)
    caches = [torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(4)]
    store = ops.mrope_store_kvcache if fmt == "bf16" else ops.rope_store_kvcache_fp4
    q, k, v = qkv.split((H, Hk, Hk), 1)
    apart = store(pos, q, k, v, table, *caches[:2], slots, (16, 24, 24))
    mine = qkv.clone()
    q, k, v = mine.split((H, Hk, Hk), 1)
    out = store(pos, q, k, v, table, *caches[2:], slots, (16, 24, 24), out=q)
    assert out.data_ptr() == mine.data_ptr() and torch.equal(out, apart) and not torch.equal(out, qkv[:, :H])
    assert torch.equal(mine[:, H:], qkv[:, H:])
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("hk", [1, 3])
def test_shift_fp4_of_k_alone(ops, hk):
    kv = torch.stack([_pages(93 + x, 4, hk, 64) for x in (0, 1)]).cuda()
    src = torch.arange(5, 100, dtype=torch.int32).cuda()
    both, alone = kv.clone(), kv.clone()
    ops.mrope_shift_layer_fp4(both[0], both[1], src, src + 128, (3, 4, 5))
    ops.mrope_shift_layer_fp4(alone[0], None, src, src + 128, (3, 4, 5))
    assert torch.equal(alone[0], both[0]) and torch.equal(alone[1], kv[1]) and not torch.equal(both[1], kv[1])


def test_prefill_fp4_without_mask_and_with_idle_sequences(ops):
    """Every row sees all keys of its sequence; sequences without query rows, and without keys, between others."""
    H, Hk, q_lens, k_lens = 16, 2, [3, 0, 0, 70, 0], [200, 65, 0, 70, 1]
    kc, vc, bt = _paged(95, k_lens, Hk, 64)
    cu_q, cu_k = np.concatenate([[0], np.cumsum(q_lens)]), np.concatenate([[0], np.cumsum(k_lens)])
    cu = torch.tensor(cu_k, dtype=torch.int32).cuda()
    q = torch.randn(73, H, D, generator=_gen(6)).to(torch.bfloat16)
    for causal in (True, False):
        plan = ops.build_prefill_plan(cu_q, cu_k, H, Hk, device="cuda", causal=causal)
        out = ops.prefill_attention_fp4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), cu, plan, SCALE)
        if causal:
            _check_attention(out, q, kc, vc, bt, q_lens, k_lens, SCALE, 1.0, 1.0, 2.0 ** -7)
        else:      # each row by itself is the last of its sequence
            rows = [(i, r) for i, n in enumerate(q_lens) for r in range(n)]
            for at, (i, _) in enumerate(rows):
                _check_attention(out[at:at + 1], q[at:at + 1], kc, vc, bt[i:i + 1], [1], [k_lens[i]], SCALE, 1.0, 1.0,
                                 2.0 ** -7)


def test_prefill_fp4_of_no_rows(ops):
    kc, vc, bt = _paged(97, [65], 2, 64)
    plan = ops.build_prefill_plan([0, 0], [0, 65], 16, 2, device="cuda")
    out = ops.prefill_attention_fp4(torch.empty(0, 16, D, dtype=torch.bfloat16, device="cuda"), kc.cuda(), vc.cuda(),
                                    bt.cuda(), torch.tensor([0, 65], dtype=torch.int32).cuda(), plan, SCALE)
    assert out.shape == (0, 16, D)


def test_a_step_captured_and_replayed(ops):
    """Rotary and scatter, prefill, decode, move and read-back captured together on a stream of their
    own, and replayed with other rows, positions and slots, against the same calls made eagerly."""
    from vlcache_b200.layers.rotary_embedding import rope_cos_sin_cache
    H, Hk, block, n = 16, 2, 64, 300
    g = _gen(99)
    table = rope_cos_sin_cache(D, 512, 1e6).cuda()
    pos = torch.randint(0, 512, (3, n), generator=g).cuda()
    qkv = torch.randn(n, H + 2 * Hk, D, generator=g).to(torch.bfloat16).cuda()
    kv = torch.stack([torch.stack([_pages(101 + x, 12, Hk, block)]) for x in (0, 1)]).cuda()
    order = torch.randperm(12, generator=g).to(torch.int32)
    bt, to = order[:5].view(1, 5).cuda(), order[5:10].view(1, 5).cuda()
    row = torch.arange(n, device="cuda")
    slots = (bt[0].long()[row // block] * block + row % block).to(torch.int32)
    away = (to[0].long()[row // block] * block + row % block).to(torch.int32)
    cu, lens = torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    plan = ops.build_prefill_plan([0, n], [0, n], H, Hk, device="cuda")
    ws = torch.empty(ops.prefill_fp4_workspace_bytes(plan, Hk), dtype=torch.uint8, device="cuda")
    ws2 = torch.empty(ops.decode_fp4_workspace_bytes(1, H, Hk, 5000), dtype=torch.uint8, device="cuda")

    def step(cache):
        q, k, v = qkv.split((H, Hk, Hk), 1)
        q = ops.rope_store_kvcache_fp4(pos, q, k, v, table, cache[0, 0], cache[1, 0], slots, (16, 24, 24))
        a = ops.prefill_attention_fp4(q, cache[0, 0], cache[1, 0], bt, cu, plan, SCALE, workspace=ws)
        ops.mrope_shift_fp4(cache, slots, away, (7, 3, 5))
        b = ops.decode_attention_fp4(q[-1:], cache[0, 0], cache[1, 0], to, lens, 5000, SCALE, workspace=ws2)
        c = ops.decode_attention_fp4(q[-1:], cache[0, 0], cache[1, 0], to, lens, 512, SCALE)
        return (a, b, c) + ops.gather_kvcache_fp4(cache[0, 0], cache[1, 0], to, cu, n)

    step(kv.clone())
    mine = kv.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        outs = step(mine)
    for seed in (1, 2):
        qkv.copy_(torch.randn(qkv.shape, generator=_gen(seed)))
        pos.copy_(torch.randint(0, 512, (3, n), generator=_gen(seed)))
        want_cache = mine.clone()
        want = step(want_cache)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(mine, want_cache) and all(torch.equal(x, y) for x, y in zip(outs, want))
    del graph
