"""Cases of the rotary embedding and the 8-bit cache run against the emulated library (tests/emu/session.py): every access
under the address sanitizer, results against their definitions in 64 bits.  Each case raises, or the emulation aborts,
on a mismatch or a memory fault."""
from __future__ import annotations

import sys
from pathlib import Path

import torch

TESTS = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(TESTS))

from cache8_util import attention, evicted, within  # noqa: E402


def _rows(t, heads, d, seed):
    return torch.randn(t, heads, d, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _offsets(rows):
    return torch.tensor([0, *rows]).cumsum(0).int()


def _cache(seqs, heads, d, capacity, fmt):
    from semblo_amd.kv_cache8 import QuantizedKVCache
    cache = QuantizedKVCache(num_seqs=seqs, num_kv_heads=heads, head_dim=d, capacity=capacity, fmt=fmt, device="cpu")
    cache.codes_k.fill_(0x7F if fmt == "e4m3" else 0x80)       # leftovers: NaN codes and scales
    cache.codes_v.fill_(0xFF if fmt == "e4m3" else 0x80)
    cache.scales.fill_(float("nan"))
    cache.tail.fill_(float("nan"))
    order = torch.rand(cache.tables.table.shape, generator=torch.Generator().manual_seed(1)).argsort(-1)
    cache.tables.table.copy_(order)
    return cache


def rotary(d, rotated, heads, interleaved) -> None:
    """Rotated rows against the definition in 64 bits, by the bounds of the GPU's tests (the emulation's sine is the host's)."""
    from semblo_amd.rotary import RotaryEmbedding
    from test_gpu_rotary import _close, _want
    d, rotated, heads, interleaved = int(d), int(rotated), int(heads), interleaved == "True"
    rope = RotaryEmbedding(d, base=10000.0, rotary_dim=rotated, interleaved=interleaved)
    q, k = _rows(7, heads, d, 1), _rows(7, 1, d, 2)
    pos = torch.tensor([0, 1, 63, 1000, 131071, -5, 2 ** 40 + 1])
    for inverse in (False, True):
        for got, x in zip(rope(pos, q, k, inverse=inverse), (q, k)):
            _close(got, *_want(rope, pos, x, inverse))
            assert torch.equal(got[..., rotated:], x[..., rotated:])
    print("rotary ok")


def attend(seqs, lengths, rows, hq, hkv, d, fmt, capacity) -> None:
    seqs, hq, hkv, d, capacity = int(seqs), int(hq), int(hkv), int(d), int(capacity)
    lengths, rows = [[int(x) for x in s.split("/")] for s in (lengths, rows)]
    cache = _cache(seqs, hkv, d, capacity, fmt)
    k, v = _rows(sum(lengths), hkv, d, 2), _rows(sum(lengths), hkv, d, 3)
    cache.append(k, v, offsets=_offsets(lengths))
    assert cache.lengths[:, 0].tolist() == lengths
    q = _rows(sum(rows), hq, d, 4)
    out, lse = cache.attend(q, offsets=_offsets(rows), max_rows=max(rows), accumulate=True, return_lse=True)
    want, want_lse, added, tol, ltol = attention(cache, q, rows)
    within(out, want, tol, "out")
    seen = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse), seen)
    within(lse[seen], want_lse[seen], ltol[seen], "lse")
    # (a block's weight sums probabilities, each off by twice the lse's bound at most)
    within(cache.weights, added, added * (2 * float(ltol.max()) + 2.0 ** -18) + 1e-30, "weights")
    print("attend ok")


def offsets_that_do_not_ascend(d, fmt) -> None:
    d = int(d)
    cache = _cache(3, 1, d, 1280, fmt)
    cache.append(_rows(3 * 400, 1, d, 66), _rows(3 * 400, 1, d, 67))
    q = _rows(40, 2, d, 68)
    for bad in ([0, 30, 10, 40], [40, 20, 0, 40], [-5, 3, 1000, 40], [0, 2 ** 31 - 1, -2 ** 31, 7]):
        offsets = torch.tensor(bad, dtype=torch.int32)
        for hint in (1, 40):
            cache.attend(q[:, :2], offsets=offsets, max_rows=hint, accumulate=True)
            cache.append(q[:, :1], q[:, 1:2], offsets=offsets, max_rows=hint)
    assert int(cache.lengths.max()) <= 1280
    print("offsets ok")


def places_and_lengths_out_of_range(d, fmt) -> None:
    d = int(d)
    cache = _cache(2, 1, d, 1280, fmt)
    cache.append(_rows(2 * 1200, 1, d, 5), _rows(2 * 1200, 1, d, 6))
    cache.tables.table[0, 0, ::3] = 2 ** 31 - 1
    cache.tables.table[1, 0, ::2] = -2 ** 31
    cache.tables.lengths[0] = 2 ** 31 - 1
    cache.tables.open_block[1] = 2 ** 30
    for n in (1, 80):
        cache.attend(_rows(2 * n, 2, d, 7), accumulate=True)
    cache.append(_rows(2, 1, d, 8), _rows(2, 1, d, 9))
    cache.tables.lengths[1] = -2 ** 31
    cache.attend(_rows(2, 2, d, 7), accumulate=True)
    cache.append(_rows(140, 1, d, 8), _rows(140, 1, d, 9))
    cache.evict(5)
    print("places ok")


def evict(blocks, keep, sink, recent) -> None:
    from semblo_amd.kv_cache8 import CacheTables
    blocks, keep, sink, recent = int(blocks), int(keep), int(sink), int(recent)
    gen = torch.Generator().manual_seed(blocks)
    t = CacheTables.new(2, 1, blocks + 3, "cpu")
    t.table.copy_(torch.rand(t.table.shape, generator=gen).argsort(-1))
    t.weights.copy_(torch.randint(0, 40, t.weights.shape, generator=gen) / 8.0)
    t.weights[1, 0, ::5] = float("nan")
    t.lengths.copy_(torch.tensor([[blocks * 64], [blocks * 64 - 63]]))
    t.open_block.copy_(torch.tensor([[blocks - 1], [blocks // 2]]))
    want = evicted(t, keep, sink, recent)
    out = t.evict(keep, sink=sink, recent=recent, into=t.empty_like())
    assert out.table.tolist() == want[0] and out.lengths.tolist() == want[2] and out.open_block.tolist() == want[3]
    torch.testing.assert_close(out.weights, torch.tensor(want[1]), rtol=0, atol=0, equal_nan=True)
    print("evict ok")


if __name__ == "__main__":
    globals()[sys.argv[1]](*sys.argv[2:])
