"""GPU tests of the 4-bit decode where the keys of all pairs form one line that the grid's warps
share (bounds above 1024 keys, or more pairs than SMs), with several chunks a warp: the cursor over
pages, heads, sequences and empty ones, the ring's stages used again, sums rescaled when a later
chunk raises the maximum, several pairs in a warp and parts on both sides of it.

Against 64-bit sums of the values that the cache holds, to the bound of
tests/test_gpu_cache_formats.py: 2^-8 |o| + (2^-11 + 2^-14 B + 2^-15) sum_j p_j |v_j| with
B = |scale| max_j sum_d |q_d K_jd|.
"""
import math

import numpy as np
import pytest
import torch

from oracle import fp4

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


def _values(cache, table, n, g=1.0):
    """Float64 values [n, Hk, 128] of a sequence's first n keys."""
    block = cache.shape[-1] // 72
    pages = cache[table[:(n + block - 1) // block].long()]
    packed, scale = pages[..., :block * 64].unflatten(-1, (block, 64)), pages[..., block * 64:].unflatten(-1, (block, 8))
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    mag = torch.tensor(np.concatenate([fp4.E2M1, -fp4.E2M1]), device=cache.device)
    e4m3 = torch.tensor(np.concatenate([fp4.E4M3, [np.nan]]), device=cache.device)
    v = mag[codes.int()] * e4m3[(scale & 127).int()].repeat_interleave(16, -1) * g
    return v.transpose(1, 2).flatten(0, 1)[:n]


def _check(out, q, kc, vc, bt, lens, scale=SCALE, kg=1.0, vg=1.0, left_out=()):
    """left_out: (sequence, first key, key after the last) of keys that do not count."""
    H, Hk = q.shape[1], kc.shape[1]
    worst = 0.0
    for i, n in enumerate(lens):
        if n == 0:
            assert not bool(out[i].any())
            continue
        keep = torch.ones(n, dtype=torch.bool, device=kc.device)
        for s, a, b in left_out:
            if s == i:
                keep[a:b] = False
        table = bt[i].clamp(0, kc.shape[0] - 1)
        k, v = _values(kc, table, n, kg)[keep], _values(vc, table, n, vg)[keep]
        rows = q[i].double().view(Hk, H // Hk, D)
        for h in range(Hk):
            s = rows[h] @ k[:, h].T
            p = torch.softmax(s * scale, -1)
            ref, size = p @ v[:, h], p @ v[:, h].abs()
            B = abs(scale) * (rows[h].abs() @ k[:, h].abs().T).amax(-1, keepdim=True)
            bound = 2.0 ** -8 * ref.abs() + (2.0 ** -11 + 2.0 ** -14 * B + 2.0 ** -15) * size
            got = out[i].view(Hk, H // Hk, D)[h].double()
            assert bool(torch.isfinite(got).all())
            worst = max(worst, float(((got - ref).abs() / bound.clamp(min=1e-30)).max()))
    assert worst <= 1.0, worst


def _line(seed, lens, hk, block):
    """Caches of random codes and tables in random page order.  Every other sequence's K scales rise
    by 2^4 along it, so that later chunks raise the maximum past the slack; what lies behind a
    sequence's end is 255 in codes and scales (NaN)."""
    r = np.random.default_rng(seed)
    need = [(n + block - 1) // block for n in lens]
    pages = sum(need) + 2
    caches = []
    for _ in "kv":
        codes = r.integers(0, 256, (pages, hk, block * 64), dtype=np.uint8)
        scales = r.integers(0x30, 0x40, (pages, hk, block * 8), dtype=np.uint8)
        caches.append((codes, scales))
    order = r.permutation(pages)
    tables, at = np.full((len(lens), max(max(need), 1)), -1, np.int32), 0
    for i, n in enumerate(lens):
        mine = order[at:at + need[i]]
        at += need[i]
        tables[i, :len(mine)] = mine
        if i % 2:
            rise = (0x20 + np.arange(len(mine) * block) * 32 // max(n, 1)).clip(0, 0x40).astype(np.uint8)
            caches[0][1][mine] = np.repeat(rise.reshape(len(mine), 1, block), 8, -1)
        if n % block:
            for codes, scales in caches:
                codes[mine[-1], :, (n % block) * 64:] = 255
                scales[mine[-1], :, (n % block) * 8:] = 255
    kc, vc = (torch.from_numpy(np.concatenate(c, -1)).cuda() for c in caches)
    return kc, vc, torch.from_numpy(tables).cuda()


def _warps(ops, seqs, H, Hk, bound):
    """Warps of the grid, from the workspace: [warps][2][group] rows of 130 floats, and a place a pair."""
    return (ops.decode_fp4_workspace_bytes(seqs, H, Hk, bound) - seqs * Hk * 8) // (2 * (H // Hk) * 130 * 4)


def _q(seed, seqs, H):
    return torch.randn(seqs, H, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


RAGGED = [(28, 4, 64), (28, 4, 256), (40, 4, 64), (16, 8, 128)]   # 7, 7, 10 (two column tiles) and 2 heads a KV head


@pytest.mark.parametrize("H,Hk,block", RAGGED)
def test_many_chunks_a_warp(ops, H, Hk, block):
    """Several chunks and pairs a warp, empty sequences first, last and in runs between others."""
    r = np.random.default_rng(H + block)
    lens = r.integers(0, 3300, 80).tolist()
    lens[0] = lens[17] = lens[18] = lens[19] = lens[79] = 0
    lens[5], lens[40], lens[41] = 1, 6000, 64
    kc, vc, bt = _line(3, lens, Hk, block)
    assert sum((n + 63) // 64 for n in lens) * Hk > 4 * _warps(ops, 80, H, Hk, 6000)
    q, ctx = _q(4, 80, H), torch.tensor(lens, dtype=torch.int32).cuda()
    out = torch.full((80, H, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.decode_attention_fp4(q, kc, vc, bt, ctx, 6000, SCALE, 0.5, 2.0, out=out)
    _check(out, q, kc, vc, bt, lens, SCALE, 0.5, 2.0)
    assert torch.equal(out, ops.decode_attention_fp4(q, kc, vc, bt, ctx, 6000, SCALE, 0.5, 2.0))


@pytest.mark.parametrize("H,Hk,block", RAGGED)
def test_bad_pages_inside_a_run(ops, H, Hk, block):
    """Table entries outside the cache, at the start, in the middle and at the end of sequences whose
    chunks lie inside a warp's run: recorded, their keys left out, all else as it is."""
    r = np.random.default_rng(H + block)
    lens = r.integers(1100, 2400, 80).tolist()
    kc, vc, bt = _line(5, lens, Hk, block)
    assert sum((n + 63) // 64 for n in lens) * Hk > 4 * _warps(ops, 80, H, Hk, 2400)
    left_out = []
    for seq, page, entry in ((3, 0, -1), (20, 2, 10 ** 6), (21, 1, -7), (50, (lens[50] - 1) // block, kc.shape[0])):
        bt[seq, page] = entry
        left_out.append((seq, page * block, (page + 1) * block))
    q, ctx = _q(6, 80, H), torch.tensor(lens, dtype=torch.int32).cuda()
    out = ops.decode_attention_fp4(q, kc, vc, bt, ctx, 2400, SCALE)
    assert ops.device_error(reset=True) == 102
    _check(out, q, kc, vc, bt, lens, left_out=left_out)


@pytest.mark.parametrize("H,Hk,n", [(4, 4, 140001), (16, 1, 310001)])
def test_one_long_sequence(ops, H, Hk, n):
    lens = [n]
    kc, vc, bt = _line(7, [0, n], Hk, 256)     # the second of two: its scales rise
    bt = bt[1:].contiguous()
    assert (n + 63) // 64 * Hk > 4 * _warps(ops, 1, H, Hk, n)
    q = _q(8, 1, H)
    out = ops.decode_attention_fp4(q, kc, vc, bt, torch.tensor(lens, dtype=torch.int32).cuda(), n, SCALE)
    _check(out, q, kc, vc, bt, lens)


@pytest.mark.parametrize("H,Hk", [(8, 2), (20, 2)])
@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_zero_and_negative_scale(ops, H, Hk, scale):
    """A scale of 0 weighs every key alike; a negative one favours the least similar; whole chunks and a cut one."""
    lens = [700, 65, 1, 128]
    kc, vc, bt = _line(9, lens, Hk, 64)
    q = _q(10, 4, H)
    assert _warps(ops, 4, H, Hk, 5000) > 1
    out = ops.decode_attention_fp4(q, kc, vc, bt, torch.tensor(lens, dtype=torch.int32).cuda(), 5000, scale)
    _check(out, q, kc, vc, bt, lens, scale)


def test_order_and_sharing_of_the_caches(ops):
    """K before V, V before K, and one cache for both give what each place holds."""
    lens, H, Hk = [400, 129, 3000], 16, 2
    kc, vc, bt = _line(11, lens, Hk, 64)
    q, ctx = _q(12, 3, H), torch.tensor(lens, dtype=torch.int32).cuda()
    call = lambda k, v: ops.decode_attention_fp4(q, k, v, bt, ctx, 5000, SCALE)  # noqa: E731
    a, b = torch.stack([kc, vc]), torch.stack([vc, kc])
    first, second = call(a[0], a[1]), call(b[1], b[0])
    assert torch.equal(first, second)
    _check(first, q, kc, vc, bt, lens)
    _check(call(a[0], a[0]), q, kc, kc, bt, lens)


def test_pages_beyond_4_gb(ops):
    """Pages past 32-bit offsets of either cache, whose distance is past them too."""
    lens, H, Hk, block = [700, 2600], 8, 4, 256
    small = _line(13, lens, Hk, block)
    pages = 60000                                       # 60000 * 73728 B = 4.4 GB
    kv = torch.full((2, pages, Hk, block * 72), 255, dtype=torch.uint8, device="cuda")
    places = torch.randperm(small[0].shape[0], generator=torch.Generator().manual_seed(1)).cuda() + pages - small[0].shape[0]
    kv[0, places], kv[1, places] = small[0], small[1]
    bt = torch.where(small[2] >= 0, places[small[2].clamp(min=0).long()].to(torch.int32), small[2])
    q, ctx = _q(14, 2, H), torch.tensor(lens, dtype=torch.int32).cuda()
    out = ops.decode_attention_fp4(q, kv[0], kv[1], bt, ctx, 5000, SCALE)
    _check(out, q, small[0], small[1], small[2], lens)
    assert torch.equal(out, ops.decode_attention_fp4(q, *small, ctx, 5000, SCALE))
