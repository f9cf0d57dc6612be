"""The 8-bit key/value cache on the GPU: append, attention, block weights and eviction against their definitions
in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from cache8_util import BLOCK, CODE_MAX, attention, decode, evicted, held, within

pytestmark = pytest.mark.gpu

FORMATS = ["e4m3", "int8"]


def _cache(seqs, heads, d, capacity, fmt, shuffle=True, seed=0):
    """An empty cache whose tensors hold the worst of leftovers (NaN codes and scales), its places shuffled."""
    from semblo_amd.kv_cache8 import QuantizedKVCache
    cache = QuantizedKVCache(num_seqs=seqs, num_kv_heads=heads, head_dim=d, capacity=capacity, fmt=fmt, device="cuda")
    cache.codes_k.fill_(0x7F if fmt == "e4m3" else 0x80)
    cache.codes_v.fill_(0xFF if fmt == "e4m3" else 0x80)
    cache.scales.fill_(float("nan"))
    cache.tail.fill_(float("nan"))
    if shuffle:
        gen = torch.Generator().manual_seed(seed)
        order = torch.rand(cache.tables.table.shape, generator=gen).argsort(-1)
        cache.tables.table.copy_(order)
    return cache


def _rows(t, heads, d, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(t, heads, d, generator=gen) * scale).bfloat16().cuda()


def _offsets(rows, first=0):
    out = [first]
    for n in rows:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def _state(cache):
    """What a cache's sequences hold, block by block in order (free places left out)."""
    out = []
    for s in range(cache.num_seqs):
        for h in range(cache.num_kv_heads):
            n = int(cache.lengths[s, h])
            place = cache.tables.table[s, h, :-(-n // BLOCK)].long()
            out += [cache.codes_k[s, h][place], cache.codes_v[s, h][place], cache.scales[:, s, h][:, place],
                    cache.tables.weights[s, h, :-(-n // BLOCK)]]
            if n:
                out.append(cache.tail[:, s, h, :(n - 1) % BLOCK + 1])
                assert int(cache.tables.open_block[s, h]) == (n - 1) // BLOCK
    return out


def _half_step(x, scale, fmt):
    """How far a code's value may be from x: half a step, which is 2^-4 of an e4m3 number, or 2^-10 among the
    subnormals, and 1/2 of an integer.  The quotient x / scale is rounded once before, by 2^-24 of itself, so
    a quotient within that of a tie goes to the other side: |code - x / scale| <= 1/2 + 2^-24 |x / scale|, and times
    the scale half a step + 2^-24 |x| (e4m3 likewise)."""
    half = torch.maximum(x.abs() * 2.0 ** -4, 2.0 ** -10 * torch.as_tensor(scale, dtype=torch.float64)) \
        if fmt == "e4m3" else 0.5 * scale
    return half + x.abs() * 2.0 ** -24


def _same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.shape == y.shape and torch.equal(x.view(torch.uint8) if x.dtype != torch.uint8 else x,
                                                  y.view(torch.uint8) if y.dtype != torch.uint8 else y)


# -- append -------------------------------------------------------------------------------


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 128, 200])
def test_append_quantises_each_block_by_its_largest_value(fmt, d, n):
    cache = _cache(2, 3, d, 256, fmt)
    k, v = _rows(2 * n, 3, d, 1, 3.0), _rows(2 * n, 3, d, 2, 0.01)
    cache.append(k, v)
    assert (cache.lengths == n).all() and not cache.overflowed()
    for s in range(2):
        for h in range(3):
            place = cache.tables.table[s, h].long().cpu()
            got = held(cache, s, h)
            for t, x in enumerate((k, v)):
                x = x[s * n:(s + 1) * n, h].double().cpu()
                blocks = torch.nn.functional.pad(x, (0, 0, 0, -n % BLOCK)).view(-1, BLOCK, d)
                most = blocks.abs().amax((1, 2))
                scale = cache.scales[t, s, h].cpu()[place][:len(blocks)].double()
                # the scale is one fp32 division of the largest value
                assert bool(((scale - most / CODE_MAX[fmt]).abs() <= 2.0 ** -24 * scale).all())
                step = scale.repeat_interleave(BLOCK)[:n, None]
                assert bool(((got[t] - x).abs() <= _half_step(x, step, fmt)).all())
            # rows behind the last are codes of 0
            if n % BLOCK:
                last = place[n // BLOCK]
                assert not cache.codes_k[s, h, last, n % BLOCK:].any() and not cache.codes_v[s, h, last, :, n % BLOCK:].any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [128, 256])
def test_append_holds_the_same_however_the_rows_are_split(fmt, d):
    rows = [150, 0, 64, 259]
    k, v = _rows(sum(rows), 2, d, 3), _rows(sum(rows), 2, d, 4)
    whole = _cache(4, 2, d, 320, fmt)
    whole.append(k, v, offsets=_offsets(rows))
    assert whole.lengths[:, 0].tolist() == rows
    first = _offsets(rows).tolist()
    for cuts, hint in (([1, 1, 1, 1], 1), ([37, 9, 64, 65], 7), ([149, 5, 63, 130], None), ([149, 5, 63, 200], 1)):
        parts = _cache(4, 2, d, 320, fmt)
        at = [0] * 4
        while at != rows:
            n = [min(c, r - a) for c, r, a in zip(cuts, rows, at)]
            take = torch.cat([torch.arange(f + a, f + a + m) for f, a, m in zip(first, at, n)]).cuda()
            parts.append(k[take], v[take], offsets=_offsets(n), max_rows=hint)
            at = [a + m for a, m in zip(at, n)]
        _same(_state(parts), _state(whole))


def test_append_takes_rows_of_any_layout():
    d, n = 128, 70
    plain = _cache(2, 2, d, 128, "e4m3")
    k, v = _rows(2 * n, 2, d, 5), _rows(2 * n, 2, d, 6)
    plain.append(k, v)
    fused = torch.zeros(2 * n, 5, d, dtype=torch.bfloat16, device="cuda")
    fused[:, 1:3], fused[:, 3:5] = k, v
    odd = torch.zeros(2 * n, 2, d + 1, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(v)
    for kk, vv in ((fused[:, 1:3], fused[:, 3:5]), (k.permute(1, 0, 2).contiguous().permute(1, 0, 2), odd)):
        cache = _cache(2, 2, d, 128, "e4m3")
        cache.append(kk, vv)
        _same(_state(cache), _state(plain))


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_writes_over_rejected_rows(fmt):
    d = 128
    k, v = _rows(300, 2, d, 7), _rows(300, 2, d, 8)
    want = _cache(1, 2, d, 320, fmt)
    want.append(k[:200], v[:200])
    cache = _cache(1, 2, d, 320, fmt)
    start = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")     # noqa: E731
    cache.append(k[:195], v[:195])
    cache.weights.fill_(3.0)
    cache.append(k[200:204], v[200:204])                   # a guess, rejected
    cache.append(k[195:200], v[195:200], start=start(195))
    assert cache.weights[0, 0].tolist() == [3.0] * 5          # no block was begun
    cache.weights.zero_()
    _same(_state(cache), _state(want))
    cache.append(k[200:270], v[200:270])                   # past the block's end, and back to a block's start
    cache.append(k[192:200], v[192:200], start=start(192))
    _same(_state(cache), _state(want))
    # cut off without new rows, then on from there
    cache.append(k[:0], v[:0], start=start(128))
    assert cache.lengths[0].tolist() == [128, 128]
    cache.append(k[128:200], v[128:200])
    _same(_state(cache), _state(want))
    # into a block whose rows are there in codes alone: those rows come back from them, and
    # the new block holds them to two roundings
    before = held(cache, 0, 1)[0][64:100]
    cache.append(k[100:101], v[100:101], start=start(100))
    assert cache.lengths[0].tolist() == [101, 101] and cache.tables.open_block[0].tolist() == [1, 1]
    after, scale = held(cache, 0, 1)[0], float(cache.scales[0, 0, 1, cache.tables.table[0, 1, 1].long()])
    x = before.abs() * (1 + 2.0 ** -8)
    assert bool(((after[64:100] - before).abs() <= before.abs() * 2.0 ** -8 + _half_step(x, scale, fmt)).all())
    # a start past the end is the end
    cache.append(k[101:103], v[101:103], start=start(5000))
    assert cache.lengths[0].tolist() == [103, 103]


def test_append_drops_rows_without_room_and_says_so():
    cache = _cache(2, 1, 128, 128, "e4m3")
    k, v = _rows(300, 1, 128, 9), _rows(300, 1, 128, 10)
    cache.append(k[:260], v[:260], offsets=_offsets([200, 60]))
    assert cache.lengths[:, 0].tolist() == [128, 60] and cache.overflowed()
    want = _cache(2, 1, 128, 128, "e4m3")
    want.append(torch.cat([k[:128], k[200:260]]), torch.cat([v[:128], v[200:260]]), offsets=_offsets([128, 60]))
    _same(_state(cache), _state(want))
    cache.append(k[:2], v[:2])                             # one is full, the other goes on
    assert cache.lengths[:, 0].tolist() == [128, 61]
    cache.reset()
    assert not cache.overflowed() and not cache.lengths.any()
    with pytest.raises(ValueError):
        cache.append(k[:258], v[:258])


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_of_zeros_tiny_huge_and_not_finite_values(fmt):
    d = 128
    cache = _cache(1, 1, d, 384, fmt)
    k = torch.zeros(320, 1, d, dtype=torch.bfloat16, device="cuda")
    k[64:128] = 3.3e38
    k[128:192, :, ::2] = 1e-39                     # subnormal
    k[192:256] = 1.0
    k[200, 0, 5] = float("inf")
    k[256:] = _rows(64, 1, d, 1)
    v = k.clone()
    v[200, 0, 5] = float("nan")
    cache.append(k, v)
    for x in held(cache, 0, 0):
        assert not x[:64].any()
        assert bool(((x[64:128] / 3.3e38 - 1).abs() < 2.0 ** -4).all())
        assert float(x[128:192].abs().max()) <= 2e-39
        assert x[192:256].isnan().all()                    # the block that holds it
        assert torch.isfinite(x[256:]).all()
    # rows that do not see that block are finite, those that do are not
    q = _rows(100, 1, d, 2)
    cache.append(k[:0], v[:0], start=torch.tensor([192], dtype=torch.int32, device="cuda"))
    cache.append(_rows(20, 1, d, 3), _rows(20, 1, d, 4))
    assert torch.isfinite(cache.attend(q[:20])).all()
    cache.append(k[200:201], v[200:201])
    out = cache.attend(q[:2])
    assert out[1].isnan().all()


# -- attention ------------------------------------------------------------------------------


@pytest.mark.parametrize("fmt,d", [("e4m3", 128), ("e4m3", 256), ("int8", 128), ("int8", 256)])
@pytest.mark.parametrize("hkv,g", [(1, 1), (2, 2), (1, 4), (2, 8), (1, 16), (1, 3)])
@pytest.mark.parametrize("n", [1, 2, 5, 8, 17, 40, 130])
def test_attend_matches_the_definition(fmt, d, hkv, g, n):
    lengths = [300, 0, 1, 64, 65, 127]
    cache = _cache(len(lengths), hkv, d, 448, fmt)
    total = sum(lengths)
    cache.append(_rows(total, hkv, d, 11, 1.5), _rows(total, hkv, d, 12), offsets=_offsets(lengths))
    q = _rows(n * len(lengths), hkv * g, d, 13, 1.5)
    cache.weights.fill_(0.5)
    out, lse = cache.attend(q, return_lse=True, accumulate=True)
    want, want_lse, added, tol, ltol = attention(cache, q, [n] * len(lengths))
    within(out, want, tol, "out")
    within(lse, want_lse, ltol, "lse")
    # a row without keys gives exactly 0
    assert not out.view(len(lengths), n, -1)[1].any() and lse.view(len(lengths), n, -1)[1].isneginf().all()
    # a weight sums n g probabilities, each off as in the bound of out, in fp32
    bound = 0.5 * 2.0 ** -23 + added * (2 * float((ltol[torch.isfinite(want_lse)]).max()) + 2.0 ** -17)
    within(cache.weights, added + 0.5, bound + 2.0 ** -23, "weights")
    assert torch.equal(cache.attend(q), out)               # the same bits, weighed or not


@pytest.mark.parametrize("fmt", FORMATS)
def test_attend_ragged_rows(fmt):
    lengths, rows = [200, 33, 0, 500, 64, 7], [1, 40, 3, 0, 130, 9]
    d, hkv, hq = 128, 2, 8
    cache = _cache(6, hkv, d, 512, fmt)
    cache.append(_rows(sum(lengths), hkv, d, 14), _rows(sum(lengths), hkv, d, 15), offsets=_offsets(lengths))
    q = _rows(sum(rows) + 20, hq, d, 16)
    first = 4                                              # rows before and behind the sequences' own
    want, want_lse, _, tol, ltol = attention(cache, q, rows, first)
    for hint in (None, 1, 8, 64, 130):
        out = torch.full_like(q, 7.0)
        _, lse = cache.attend(q, offsets=_offsets(rows, first), max_rows=hint, out=out, return_lse=True)
        mine = slice(first, first + sum(rows))
        within(out[mine], want[mine], tol[mine], f"out, hint {hint}")
        within(lse[mine], want_lse[mine], ltol[mine], f"lse, hint {hint}")
        assert (out[:first] == 7).all() and (out[first + sum(rows):] == 7).all()


def test_attend_takes_offsets_of_many_sequences_and_none_with_rows():
    cache = _cache(200, 1, 128, 64, "e4m3")
    lengths = [(7 * i) % 65 for i in range(200)]
    cache.append(_rows(sum(lengths), 1, 128, 1), _rows(sum(lengths), 1, 128, 2), offsets=_offsets(lengths))
    rows = [i % 3 for i in range(200)]
    q = _rows(sum(rows), 2, 128, 3)
    want, want_lse, _, tol, _ = attention(cache, q, rows)
    for hint in (None, 2):
        within(cache.attend(q, offsets=_offsets(rows), max_rows=hint), want, tol, "out")
    out = torch.full_like(q, 3.0)
    cache.attend(q, offsets=_offsets([0] * 200), out=out)
    assert (out == 3).all()
    assert cache.attend(q[:0]).shape == (0, 2, 128)


@pytest.mark.parametrize("fmt", FORMATS)
def test_attend_over_blocks_of_very_unequal_size(fmt):
    """Keys that draw all attention behind ones that drew it before, values whose scales lie far apart."""
    d = 128
    cache = _cache(1, 1, d, 1024, fmt)
    k, v = _rows(1000, 1, d, 17), _rows(1000, 1, d, 18)
    k *= torch.linspace(0.2, 12, 1000, device="cuda")[:, None, None].bfloat16()
    v *= (10.0 ** torch.linspace(-3, 3, 16, device="cuda")).repeat_interleave(64)[:1000, None, None].bfloat16()
    for flip in (False, True):
        cache.reset()
        cache.append(k.flip(0) if flip else k, v.flip(0) if flip else v)
        for n in (1, 70):
            q = _rows(n, 4, d, 19, 3.0)
            out, lse = cache.attend(q, return_lse=True)
            want, want_lse, _, tol, ltol = attention(cache, q, [n])
            within(out, want, tol, "out")
            within(lse, want_lse, ltol, "lse")


def test_attend_long_enough_for_every_share_of_the_keys():
    d, length = 128, 20011
    cache = _cache(1, 2, d, 20480, "e4m3")
    cache.append(_rows(length, 2, d, 20), _rows(length, 2, d, 21))
    for n in (1, 3, 20, 70):
        q = _rows(n, 8, d, 22, 2.0)
        out, lse = cache.attend(q, return_lse=True, accumulate=True)
        want, want_lse, added, tol, ltol = attention(cache, q, [n])
        within(out, want, tol, "out")
        within(lse, want_lse, ltol, "lse")
        within(cache.weights, added, added * (2 * float(ltol.max()) + 2.0 ** -17) + 2.0 ** -23, "weights")
        cache.weights.zero_()


def test_attend_scale_strides_and_given_out():
    d = 256
    cache = _cache(2, 2, d, 128, "int8")
    cache.append(_rows(200, 2, d, 23), _rows(200, 2, d, 24))
    q = _rows(6, 4, d, 25)
    want, _, _, tol, _ = attention(cache, q, [3, 3], sm_scale=0.11)
    fused = torch.zeros(6, 9, d, dtype=torch.bfloat16, device="cuda")
    fused[:, 2:6] = q
    out = torch.zeros(6, 4, 2 * d, dtype=torch.bfloat16, device="cuda")[..., d:]
    assert cache.attend(fused[:, 2:6], sm_scale=0.11, out=out) is out
    within(out, want, tol, "out")
    odd = torch.zeros(6, 4, d + 1, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(cache.attend(odd, sm_scale=0.11), out)


def test_attend_past_32_bits_of_bytes():
    """Sequences whose codes start past 4 GiB, at places past 2 GiB of their own head."""
    from semblo_amd.kv_cache8 import QuantizedKVCache
    cache = QuantizedKVCache(num_seqs=5, num_kv_heads=4, head_dim=256, capacity=16384 * 64, device="cuda")
    cache.tables.table.copy_(cache.tables.table.flip(-1))
    rows = [3, 100, 0, 64, 190]
    cache.append(_rows(sum(rows), 4, 256, 26), _rows(sum(rows), 4, 256, 27), offsets=_offsets(rows))
    q = _rows(10, 4, 256, 28)
    out = cache.attend(q, accumulate=True)
    want, _, added, tol, _ = attention(cache, q, [2] * 5)
    within(out, want, tol, "out")
    within(cache.weights, added, added * 2.0 ** -12 + 2.0 ** -23, "weights")


def test_places_outside_the_room_are_read_inside_it():
    """A damaged table gives wrong numbers, and no access outside the cache."""
    cache = _cache(1, 1, 128, 256, "e4m3")
    cache.append(_rows(200, 1, 128, 1), _rows(200, 1, 128, 2))
    cache.tables.table[0, 0, 1] = 2 ** 31 - 1
    cache.tables.table[0, 0, 2] = -7
    cache.attend(_rows(1, 1, 128, 3), accumulate=True)
    cache.append(_rows(1, 1, 128, 4), _rows(1, 1, 128, 5), start=torch.tensor([70], dtype=torch.int32, device="cuda"))
    cache.lengths.fill_(2 ** 31 - 1)
    cache.attend(_rows(70, 1, 128, 6), accumulate=True)
    cache.evict(2)
    torch.cuda.synchronize()


def test_attend_with_a_negative_scale_and_a_scale_of_zero():
    d = 128
    cache = _cache(1, 2, d, 256, "e4m3")
    cache.append(_rows(250, 2, d, 60), _rows(250, 2, d, 61))
    for n in (2, 70):
        q = _rows(n, 4, d, 62)
        for scale in (-0.09, 0.0):
            out, lse = cache.attend(q, sm_scale=scale, return_lse=True)
            want, want_lse, _, tol, ltol = attention(cache, q, [n], sm_scale=scale)
            within(out, want, tol, "out")
            within(lse, want_lse, ltol, "lse")


@pytest.mark.parametrize("fmt", FORMATS)
def test_attend_of_many_rows_before_a_block_that_is_not_finite(fmt):
    d = 128
    cache = _cache(1, 1, d, 512, fmt)
    k, v = _rows(400, 1, d, 63), _rows(400, 1, d, 64)
    v[350, 0, 3] = float("inf")
    cache.append(k, v)
    q = _rows(120, 2, d, 65)
    out, lse = cache.attend(q, return_lse=True)            # rows 0 .. 39 end before the block of rows 320 .. 383
    assert torch.isfinite(lse).all()
    assert torch.isfinite(out[:40]).all() and out[40:].isnan().all()
    cache.append(k[:0], v[:0], start=torch.tensor([320], dtype=torch.int32, device="cuda"))
    want, _, _, tol, _ = attention(cache, q[:40], [40])
    within(out[:40], want, tol, "rows before")


def test_offsets_that_do_not_ascend_stay_inside_the_tensors():
    cache = _cache(3, 2, 128, 2048, "e4m3")
    cache.append(_rows(3 * 1500, 2, 128, 66), _rows(3 * 1500, 2, 128, 67))
    q = _rows(90, 4, 128, 68)
    for bad in ([0, 80, 10, 90], [90, 40, 0, 90], [-5, 3, 1000, 90], [0, 2 ** 31 - 1, -2 ** 31, 7]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        for hint in (1, 90):
            cache.attend(q, offsets=offsets, max_rows=hint, accumulate=True)
            cache.append(q[:, :2], q[:, 2:], offsets=offsets, max_rows=hint)
    torch.cuda.synchronize()
    assert int(cache.lengths.max()) <= 2048


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("blocks", [1, 10, 11, 20, 21, 33])
def test_attend_whole_and_in_shares(blocks, d):
    """Rooms on both sides of where a tile's keys are shared out."""
    cache = _cache(2, 1, d, blocks * BLOCK, "int8")
    lengths = [blocks * BLOCK, blocks * BLOCK - 37]
    cache.append(_rows(sum(lengths), 1, d, 76), _rows(sum(lengths), 1, d, 77), offsets=_offsets(lengths))
    for n in (1, 5, 17):
        q = _rows(2 * n, 4, d, 78)
        cache.weights.zero_()
        out, lse = cache.attend(q, accumulate=True, return_lse=True)
        want, want_lse, added, tol, ltol = attention(cache, q, [n, n])
        within(out, want, tol, "out")
        within(lse, want_lse, ltol, "lse")
        # (sums of probabilities, each off by twice its row's bound, over fp32 sums of a block's 64 and a head's rows)
        within(cache.weights, added, added * (2 * float(ltol.max()) + 2.0 ** -18) + 1e-30, "weights")


def test_a_row_that_is_not_finite_leaves_the_others_alone():
    d = 128
    cache = _cache(1, 2, d, 512, "int8")
    cache.append(_rows(450, 2, d, 70), _rows(450, 2, d, 71))
    for n in (4, 9, 100):
        q = _rows(n, 4, d, 72)
        want, want_lse, _, tol, ltol = attention(cache, q, [n])
        q[1, 2, 5], q[2, 0, 7] = float("nan"), float("inf")
        out, lse = cache.attend(q, return_lse=True)
        others = torch.ones(n, 4, dtype=torch.bool)
        others[1, 2] = others[2, 0] = False
        assert out[1, 2].isnan().all()
        within(out.cpu()[others], want[others], tol[others], "out")
        within(lse.cpu()[others], want_lse[others], ltol[others], "lse")


def test_a_cache_keeps_its_tensors():
    cache = _cache(1, 1, 128, 128, "e4m3")
    k, v, q = _rows(100, 1, 128, 73), _rows(100, 1, 128, 74), _rows(1, 1, 128, 75)
    cache.append(k, v)
    want = cache.attend(q)
    cache.codes_k = cache.codes_v = cache.scales = cache.tail = cache.tables = None
    fill = [torch.full((1 << n,), 255, dtype=torch.uint8, device="cuda") for n in range(4, 20)]
    assert torch.equal(cache.attend(q), want)
    del fill


# -- eviction -------------------------------------------------------------------------------


@pytest.mark.parametrize("blocks,keep,sink,recent", [(1, 1, 0, 1), (5, 3, 1, 1), (5, 3, 0, 3), (64, 20, 4, 7), (65, 64, 0, 1),
                                                     (1500, 700, 3, 40), (16000, 2, 0, 2), (16000, 9000, 1, 1),
                                                     (9, 12, 0, 1), (1024, 1, 0, 1)])
def test_evict_matches_the_definition(blocks, keep, sink, recent):
    from semblo_amd.kv_cache8 import CacheTables
    gen = torch.Generator().manual_seed(blocks + keep)
    s, h, room = 3, 2, min(blocks + 5, 16384)
    tables = CacheTables.new(s, h, room, "cuda")
    tables.table.copy_(torch.rand(s, h, room, generator=gen).argsort(-1))
    w = torch.rand(s, h, room, generator=gen) ** 6
    w = torch.where(w < 0.01, 0.0, w)
    w[0, 1] = 0.25                                         # all alike: the first ones stay
    w[1, 0, ::3], w[1, 0, 1::3] = -1.0, float("inf")
    w[2, 1, ::2] = float("nan")
    w[2, 0] = torch.randint(0, 3, (room,), generator=gen).float() * 1e-40      # subnormal
    tables.weights.copy_(w)
    n = torch.tensor([blocks, max(0, blocks - 3), blocks])[:, None].expand(s, h)
    tables.lengths.copy_((n * BLOCK - torch.tensor([[0], [11], [63]])).clamp_min(0))
    tables.open_block.copy_(torch.tensor([[blocks - 1, -1], [max(0, blocks - 4), 0], [blocks // 2, blocks - 1]]))
    want = evicted(tables, keep, sink, recent)
    before = [getattr(tables, name).clone() for name in tables.__slots__]
    into = tables.empty_like()
    assert tables.evict(keep, sink=sink, recent=recent, into=into) is into
    for name, old in zip(tables.__slots__, before):
        assert torch.equal(getattr(tables, name).view(torch.int32), old.view(torch.int32)), f"{name} changed"
    for out in (into, tables.evict(keep, sink=sink, recent=recent)):
        assert out.table.tolist() == want[0] and out.lengths.tolist() == want[2] and out.open_block.tolist() == want[3]
        torch.testing.assert_close(out.weights.cpu(), torch.tensor(want[1]), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("fmt", FORMATS)
def test_the_cache_goes_on_after_an_eviction(fmt):
    """Weights from attention, the least attended blocks gone, new rows into the open block and beyond."""
    d, hkv, hq = 128, 2, 4
    cache = _cache(2, hkv, d, 640, fmt)
    lengths = [600, 333]
    cache.append(_rows(933, hkv, d, 30, 1.5), _rows(933, hkv, d, 31), offsets=_offsets(lengths))
    cache.attend(_rows(60, hq, d, 32, 1.5), accumulate=True)
    want = evicted(cache.tables, 5, 1, 2)
    kept = [[[held(cache, s, h)[t] for t in range(2)] for h in range(hkv)] for s in range(2)]
    blocks = [[[cache.tables.table[s, h].tolist().index(p) for p in want[0][s][h][:5]] for h in range(hkv)] for s in range(2)]
    cache.evict(5, sink=1, recent=2)
    assert cache.lengths.tolist() == want[2] == [[4 * 64 + 24] * 2, [4 * 64 + 13] * 2]
    for s in range(2):
        for h in range(hkv):
            for t in range(2):
                x = torch.cat([kept[s][h][t][b * 64:(b + 1) * 64] for b in blocks[s][h]])
                assert torch.equal(held(cache, s, h)[t], x)
    k, v = _rows(2 * 350, hkv, d, 33), _rows(2 * 350, hkv, d, 34)
    cache.append(k, v)                                     # into the places that went free
    q = _rows(2 * 9, hq, d, 35)
    out, lse = cache.attend(q, return_lse=True)
    want, want_lse, _, tol, ltol = attention(cache, q, [9, 9])
    within(out, want, tol, "out")
    within(lse, want_lse, ltol, "lse")
    # the open block's rows were requantised from bf16: 24 old ones and the new
    place = int(cache.tables.table[0, 0, 4])
    scale = float(cache.scales[0, 0, 0, place])
    x = held(cache, 0, 0)[0][4 * 64 + 24:4 * 64 + 64]
    rows = k[:40, 0].double().cpu()
    assert bool(((x - rows).abs() <= _half_step(rows, scale, fmt)).all())


# -- streams and graphs -----------------------------------------------------------------------


def _steps(cache, rows, q, k, v, out):
    cache.append(k, v)
    cache.attend(q, accumulate=True, out=out)
    cache.evict(4, sink=1, recent=1)
    out.copy_(cache.attend(q))


def test_a_captured_decode_replays_as_the_eager_one():
    d, hkv, hq, s = 128, 2, 8, 3
    caches = [_cache(s, hkv, d, 384, "e4m3", seed=4) for _ in range(2)]
    prompt = [300, 64, 129]
    for c in caches:
        c.append(_rows(sum(prompt), hkv, d, 40), _rows(sum(prompt), hkv, d, 41), offsets=_offsets(prompt))
    q, k, v = _rows(s, hq, d, 42), _rows(s, hkv, d, 43), _rows(s, hkv, d, 44)
    out = torch.empty(s, hq, d, dtype=torch.bfloat16, device="cuda")
    # warm up on a third cache
    warm = _cache(s, hkv, d, 384, "e4m3")
    _steps(warm, 1, q, k, v, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _steps(caches[0], 1, q, k, v, out)
    eager = torch.empty_like(out)
    for step in range(70):
        q.copy_(_rows(s, hq, d, 100 + step))
        k.copy_(_rows(s, hkv, d, 200 + step))
        v.copy_(_rows(s, hkv, d, 300 + step))
        graph.replay()
        _steps(caches[1], 1, q, k, v, eager)
        if step % 23 == 0:
            torch.cuda.synchronize()
        assert torch.equal(out, eager), f"step {step}"
        _same(_state(caches[0]), _state(caches[1]))


def test_a_captured_ragged_call_follows_its_offsets():
    """Prompts of several blocks and their attention captured together, replayed with other rows, counts and lengths."""
    d, hkv, hq, seqs, tokens = 128, 2, 4, 3, 300
    caches = [_cache(seqs, hkv, d, 1280, "e4m3", seed=6) for _ in range(2)]
    k, v, q = _rows(tokens, hkv, d, 1), _rows(tokens, hkv, d, 2), _rows(tokens, hq, d, 3)
    offsets, out = _offsets([100, 100, 100]), torch.zeros(tokens, hq, d, dtype=torch.bfloat16, device="cuda")
    eager = out.clone()

    def step(cache, to):
        cache.append(k, v, offsets=offsets)
        cache.attend(q, offsets=offsets, accumulate=True, out=to)
    step(_cache(seqs, hkv, d, 1280, "e4m3"), out)          # warm up on another cache
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0], out)
    for i, rows in enumerate(([100, 100, 100], [0, 299, 1], [7, 64, 200], [300, 0, 0], [1, 1, 1], [65, 0, 130])):
        offsets.copy_(_offsets(rows))
        for x, heads in ((k, hkv), (v, hkv), (q, hq)):
            x.copy_(_rows(tokens, heads, d, 10 * i + heads))
        graph.replay()
        step(caches[1], eager)
        if i % 2:
            torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i}"
        _same(_state(caches[0]), _state(caches[1]))


def test_two_captured_graphs_of_one_pool():
    d = 128
    caches = [_cache(1, 2, d, 8192, "int8", seed=i) for i in range(2)]
    for i, c in enumerate(caches):
        c.append(_rows(8000, 2, d, 50 + i), _rows(8000, 2, d, 60 + i))
    qs = [_rows(1, 8, d, 70 + i) for i in range(2)]
    want = [c.attend(q) for c, q in zip(caches, qs)]
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for c, q in zip(caches, qs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(c.attend(q))
        graphs.append(g)
    # one after the other, as graphs of one pool are replayed
    for _ in range(3):
        graphs[0].replay()
        first = outs[0].clone()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want[0]) and torch.equal(outs[1], want[1])


def test_calls_on_two_streams_at_once():
    d = 128
    caches = [_cache(1, 2, d, 8192, "e4m3", seed=i) for i in range(2)]
    k, v, q = _rows(8000, 2, d, 80), _rows(8000, 2, d, 81), _rows(1, 8, d, 82)
    want = []
    for c in caches:
        c.append(k, v)
        want.append(c.attend(q))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(caches[i].attend(q))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


# -- refusals that need the device ---------------------------------------------------------------


def test_wrong_tensors_are_refused():
    cache = _cache(2, 2, 128, 128, "e4m3")
    k, q = _rows(4, 2, 128, 1), _rows(4, 4, 128, 2)
    cpu = k.cpu()
    for call in (lambda: cache.append(cpu, k), lambda: cache.append(k, cpu), lambda: cache.attend(q.cpu()),
                 lambda: cache.append(k, k, offsets=_offsets([2, 2]).cpu()),
                 lambda: cache.append(k, k, start=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: cache.attend(q, out=q), lambda: cache.attend(q, out=torch.empty_like(q[:1]).expand(4, 4, 128)), lambda: cache.attend(q, offsets=_offsets([4])),
                 lambda: cache.attend(q, offsets=_offsets([2, 2]).long()), lambda: cache.append(k[:3], k[:3]),
                 lambda: cache.attend(q, out=torch.empty(4, 4, 129, dtype=q.dtype, device="cuda")[..., 1:])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        cache.attend(q.clone().requires_grad_())
    into = cache.tables.empty_like()
    into.table = cache.tables.table.view(-1).as_strided(cache.tables.table.shape, cache.tables.table.stride(), 0)
    cache.tables.evict(2, into=into)                       # the very same table is fine
    assert math.isclose(float(decode(torch.tensor([0x7E]), "e4m3")), 448.0)
