"""What the rotary embedding and the 8-bit cache refuse, on the CPU: nothing here reaches a GPU."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch


def _lib():
    from semblo_amd import _lib as lib
    if not lib.LIB_PATH.exists():
        pytest.skip("libsbsa.so is not built here")
    return lib.load()


def _struct(**kw):
    from semblo_amd.kv_cache8 import _Cache8
    p = 4096                                   # stand-in for a device pointer, never followed
    fields = dict(codes_k=p, codes_v=p, scales=p, tail=p, table=p, weights=p, lengths=p, open_block=p, counters=p,
                  overflow=p, num_seqs=2, num_kv_heads=2, num_blocks=8, head_dim=128, format=0)
    return ctypes.byref(_Cache8(**(fields | kw)))


P = 4096
ARG, UNSUPPORTED, CAPACITY = 1, 2, 4


@pytest.mark.parametrize("change,code", [
    (dict(codes_k=None), ARG), (dict(codes_v=4100), ARG), (dict(tail=4104), ARG), (dict(lengths=None), ARG),
    (dict(counters=None), ARG), (dict(num_seqs=0), ARG), (dict(num_kv_heads=0), ARG), (dict(num_blocks=0), ARG),
    (dict(head_dim=64), UNSUPPORTED), (dict(format=2), UNSUPPORTED), (dict(num_blocks=16385), UNSUPPORTED)])
def test_a_wrong_cache_is_refused(change, code):
    lib = _lib()
    c = _struct(**change)
    assert lib.sbsa_cache8_append(c, P, 256, 128, P, 256, 128, 4, None, None, 0, None) == code
    assert lib.sbsa_cache8_attend(c, P, 512, 128, 4, 4, None, 0, 0.1, P, 512, 128, None, 0, P, 1 << 30, None) == code


def test_wrong_rows_are_refused():
    lib = _lib()
    c = _struct()
    assert lib.sbsa_cache8_append(None, P, 256, 128, P, 256, 128, 4, None, None, 0, None) == ARG
    for k, st, sh, n in ((None, 256, 128, 4), (4098, 256, 128, 4), (P, 257, 128, 4), (P, 256, 124, 4), (P, 256, 128, 3),
                         (P, 256, 128, -2)):
        assert lib.sbsa_cache8_append(c, k, st, sh, P, 256, 128, n, None, None, 0, None) == ARG
        assert lib.sbsa_cache8_append(c, P, 256, 128, k, st, sh, n, None, None, 0, None) == ARG
    assert lib.sbsa_cache8_append(c, P, 256, 128, P, 256, 128, (1 << 24) + 2, None, None, 0, None) == UNSUPPORTED
    assert lib.sbsa_cache8_append(c, None, 0, 0, None, 0, 0, 0, None, None, 0, None) == 0      # nothing to do


def test_wrong_queries_and_workspaces_are_refused():
    lib = _lib()
    c = _struct(num_blocks=8192)

    def attend(q=P, st=512, heads=4, n=4, out=P, work=P, size=1 << 30):
        return lib.sbsa_cache8_attend(c, q, st, 128, heads, n, None, 0, 0.1, out, 512, 128, None, 0, work, size, None)
    assert attend(q=None) == ARG and attend(out=4098) == ARG and attend(st=511) == ARG and attend(n=3) == ARG
    assert attend(heads=3) == ARG and attend(heads=0) == ARG and attend(n=-2) == ARG
    assert attend(heads=34) == UNSUPPORTED and attend(n=1 << 23) == UNSUPPORTED
    need = lib.sbsa_cache8_attend_workspace_bytes(c, 4, 4, 0, 0, 0)
    assert need > 0 and attend(size=need - 1) == CAPACITY
    assert attend(work=None) == ARG and attend(work=4104) == ARG
    assert attend(n=0, q=None, out=None, work=None, size=0) == 0
    assert lib.sbsa_cache8_attend_workspace_bytes(c, 4, 4, 0, 0, 1) > need
    for wrong in ((None, 4, 4), (c, 1, 4), (c, 64, 4), (c, 4, 0)):
        assert lib.sbsa_cache8_attend_workspace_bytes(*wrong, 0, 0, 0) == 0


def test_wrong_evictions_are_refused():
    lib = _lib()

    def evict(keep=4, sink=1, recent=1, s=1, h=1, n=8, table=P, out=P):
        return lib.sbsa_cache8_evict(table, P, P, P, out, P, P, P, s, h, n, keep, sink, recent, None)
    for kw in (dict(table=None), dict(out=None), dict(recent=0), dict(sink=-1), dict(keep=0), dict(sink=4), dict(s=0),
               dict(h=0), dict(n=0), dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1)):
        assert evict(**kw) == ARG, kw
    assert evict(n=16385) == UNSUPPORTED


def test_wrong_rotations_are_refused():
    lib = _lib()

    def rotate(q=P, heads=2, k=P, kheads=1, pos=P, bytes_=8, n=3, d=128, r=64, turns=P, gain=1.0):
        return lib.sbsa_rotary(q, 256, 128, P, 256, 128, heads, k, 128, 128, P, 128, 128, kheads, pos, bytes_, 0, 1, n, d,
                               r, 0, turns, None, gain, 0, None)
    for kw in (dict(q=None), dict(heads=0), dict(k=None), dict(kheads=-1), dict(pos=None), dict(bytes_=2), dict(n=-1),
               dict(r=63), dict(r=0), dict(r=130), dict(turns=None), dict(gain=0.0), dict(gain=math.nan)):
        assert rotate(**kw) == ARG, kw
    assert rotate(d=514) == UNSUPPORTED and rotate(n=1 << 24) == UNSUPPORTED
    assert rotate(n=0, q=None, pos=None) == 0


def test_tensors_on_the_cpu_are_refused():
    from semblo_amd.kv_cache8 import CacheTables, QuantizedKVCache
    from semblo_amd.rotary import RotaryEmbedding
    with pytest.raises(RuntimeError):
        QuantizedKVCache(num_seqs=1, num_kv_heads=1, head_dim=128, capacity=64, device="cpu")
    with pytest.raises(RuntimeError):
        CacheTables.new(1, 1, 4, "cpu").evict(2)
    with pytest.raises(RuntimeError):
        RotaryEmbedding(64)(torch.arange(2), torch.zeros(2, 1, 64, dtype=torch.bfloat16))


def test_wrong_tables_and_caches_are_refused():
    from semblo_amd.kv_cache8 import CacheTables, QuantizedKVCache
    t = CacheTables.new(2, 1, 4, "cpu")
    parts = [getattr(t, n) for n in t.__slots__]
    for i, bad in enumerate((t.table.long(), t.weights.double(), t.lengths[:1], t.open_block.t())):
        with pytest.raises(ValueError):
            CacheTables(*[bad if j == i else p for j, p in enumerate(parts)])
    for kw in (dict(keep=0), dict(keep=2, sink=2), dict(keep=2, recent=0), dict(keep=2, sink=-1),
               dict(keep=2, into=CacheTables.new(2, 1, 5, "cpu"))):
        with pytest.raises(ValueError):
            t.evict(**kw)
    into = CacheTables.new(2, 1, 4, "cpu")
    whole = torch.zeros(12, dtype=torch.int32)
    t.table, into.table = whole[:8].view(2, 1, 4), whole[4:].view(2, 1, 4)
    with pytest.raises(ValueError, match="overlaps"):
        t.evict(2, into=into)
    make = dict(num_seqs=1, num_kv_heads=1, head_dim=128, capacity=64, device="cpu")
    for kw in (dict(head_dim=64), dict(capacity=0), dict(capacity=16384 * 64 + 1), dict(fmt="e5m2"), dict(num_seqs=0)):
        with pytest.raises(ValueError):
            QuantizedKVCache(**(make | kw))


def test_wrong_embeddings_are_refused():
    from semblo_amd.rotary import RotaryEmbedding
    for kw in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=130), dict(base=1.0), dict(base=math.inf),
               dict(scaling=dict(kind="other")), dict(scaling=dict(kind="linear", factor=0.0)),
               dict(scaling=dict(kind="linear", factor=2.0, original_length=4)), dict(scaling=dict(kind="yarn", factor=2.0)),
               dict(scaling=dict(kind="banded", factor=2.0, original_length=64, low_factor=4.0, high_factor=1.0)),
               dict(sections=(32, 31)), dict(sections=(70, -6))):
        with pytest.raises(ValueError):
            RotaryEmbedding(128, **kw)
    with pytest.raises(ValueError):
        RotaryEmbedding(514)
    rope = RotaryEmbedding(64)
    grid = RotaryEmbedding(64, sections=(16, 8, 8))
    q, pos = torch.zeros(2, 1, 64, dtype=torch.bfloat16), torch.arange(2)
    for call in (lambda: rope(pos, q.float()), lambda: rope(pos, q[0]), lambda: rope(pos, q[..., :32]),
                 lambda: rope(pos.float(), q), lambda: rope(pos[:1], q), lambda: grid(pos, q), lambda: rope(pos, q, q[:1]),
                 lambda: rope(pos, q, out_k=q), lambda: rope(pos, q, out_q=q[:1]),
                 lambda: rope(pos, q, out_q=q.view(1, 2, 64).transpose(0, 1)[:, :, :].expand(2, 1, 64).flip(0)[..., ::1].float())):
        with pytest.raises(ValueError):
            call()
    buf = torch.zeros(3, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps"):
        rope(pos, buf[:2], out_q=buf[1:])
    with pytest.raises(RuntimeError, match="backward"):
        rope(pos, q.clone().requires_grad_())
    k = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    both = torch.zeros(2, 4 * 64, dtype=torch.bfloat16)         # a row's query head and three key heads
    own_q, own_k = both[:, :64].view(2, 1, 64), both[:, 64:].view(2, 3, 64)
    for call in (lambda: rope(pos, k[:, :1], k, out_q=k[:, :1]), lambda: rope(pos, own_q, own_k, out_k=both[:, :192].view(2, 3, 64)),
                 lambda: rope(pos, q, q, out_q=own_q, out_k=own_q), lambda: rope(pos, own_k, q, out_q=own_k, out_k=own_k[:, 2:])):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    with pytest.raises(ValueError, match="stride of 0"):
        rope(pos, q, out_q=q[:1].clone().expand(2, 1, 64))
    with pytest.raises(RuntimeError):                           # in place in one buffer: only the device is wrong here
        rope(pos, own_q, own_k, out_q=own_q, out_k=own_k)


def test_frequencies_and_axes():
    from semblo_amd.rotary import rotary_frequencies, section_axes
    freq, gain = rotary_frequencies(8, 10000.0)
    assert gain == 1.0 and freq == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    assert rotary_frequencies(8, 10000.0, dict(kind="linear", factor=4.0))[0] == pytest.approx([f / 4 for f in freq])
    ntk = rotary_frequencies(8, 10000.0, dict(kind="ntk", factor=4.0))[0]
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(freq[-1] / 4)       # the slowest over the factor
    yarn, gain = rotary_frequencies(128, 10000.0, dict(kind="yarn", factor=4.0, original_length=4096))
    plain = rotary_frequencies(128, 10000.0)[0]
    assert gain == pytest.approx(0.1 * math.log(4) + 1)
    for y, f in zip(yarn, plain):
        turns = 4096 * f / (2 * math.pi)
        assert f / 4 * (1 - 1e-12) <= y <= f * (1 + 1e-12)
        if turns > 40:
            assert y == f
        if turns < 0.8:
            assert y == pytest.approx(f / 4)
    band = rotary_frequencies(128, 10000.0, dict(kind="banded", factor=8.0, original_length=8192))[0]
    for y, f in zip(band, plain):
        turns = 8192 * f / (2 * math.pi)
        w = min(1.0, max(0.0, (turns - 1) / 3))
        assert y == pytest.approx(f * (w + (1 - w) / 8))
    assert section_axes((2, 1, 1), 4) == [0, 0, 1, 2]
    assert section_axes((11, 11, 10), 32, True) == [i % 3 if i < 31 else 1 for i in range(32)]
    assert section_axes((4, 2, 2), 8, True) == [0, 1, 2, 0, 1, 2, 0, 0]


def test_a_dense_layer_checks_its_settings():
    from semblo_amd.config import SembloRuntimeConfig
    from semblo_amd.dense_layer import DenseCacheAttention
    from semblo_amd.rotary import RotaryEmbedding
    cfg = SembloRuntimeConfig(num_q_heads=6, num_kv_heads=2, head_dim=128)
    with pytest.raises(ValueError):
        DenseCacheAttention(cfg, capacity=64, device="cpu")
    cfg = SembloRuntimeConfig(num_q_heads=4, num_kv_heads=2, head_dim=128)
    with pytest.raises(ValueError):
        DenseCacheAttention(cfg, capacity=64, device="cpu", rotary=RotaryEmbedding(64))
