"""The dense layer behind semblo::attention: rotary, append, attention and eviction as a request runs them,
and the sessions that rotate for the model."""
from __future__ import annotations

import pytest
import torch

from cache8_util import BLOCK, attention, evicted, held, within
from gpu_util import assert_close_bf16

pytestmark = pytest.mark.gpu


def _rows(t, heads, d, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(t, heads, d, generator=gen) * scale).bfloat16().cuda()


def _causal(q, k, v, scale):
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1).transpose(0, 1), v.repeat_interleave(g, 1).transpose(0, 1)
    s = q.transpose(0, 1) @ k.transpose(1, 2) * scale
    s.masked_fill_(torch.ones(s.shape[1:], dtype=torch.bool).triu(1), float("-inf"))
    return (torch.softmax(s, -1) @ v).transpose(0, 1)


def _layer(name, d, hq, hkv, **kw):
    from semblo_amd.config import SembloRuntimeConfig
    from semblo_amd.dense_layer import DenseCacheAttention
    return DenseCacheAttention(SembloRuntimeConfig(num_q_heads=hq, num_kv_heads=hkv, head_dim=d), device="cuda",
                               layer_name=name, **kw)


@pytest.mark.parametrize("fmt,d,rotated", [("e4m3", 256, 64), ("int8", 128, 128)])
def test_a_request_through_the_operator(fmt, d, rotated):
    from semblo_amd.attention_op import sparse_attention_op
    from semblo_amd.rotary import RotaryEmbedding
    hq, hkv, prompt = 8, 2, 300
    rotary = RotaryEmbedding(d, rotary_dim=rotated, base=1e6)
    layer = _layer("test.dense", d, hq, hkv, capacity=512, fmt=fmt, rotary=rotary, keep_blocks=4, sink_blocks=1,
                   recent_blocks=2)
    empty = torch.empty(0, device="cuda")
    for request in range(2):                                # the second starts anew
        q, k, v = (_rows(prompt, h, d, 10 * request + i) for i, h in enumerate((hq, hkv, hkv)))
        pos = torch.arange(prompt, device="cuda")
        out = torch.empty(prompt, hq * d, dtype=torch.bfloat16, device="cuda")
        sparse_attention_op(pos, empty, empty, None, v.view(prompt, -1), q, k, out, "test.dense")
        qr, kr = rotary(pos, q, k)
        assert_close_bf16(out.view(prompt, hq, d), _causal(qr, kr, v, d ** -0.5), "prompt")
        got_k, got_v = held(layer.cache, 0, 1)
        step = layer.cache.scales.cpu()[:, 0, 1][:, layer.cache.tables.table[0, 1].long().cpu()[:5]].double()
        for got, x, s in ((got_k, kr, step[0]), (got_v, v, step[1])):
            x = x[:, 1].double().cpu()
            s = s.repeat_interleave(BLOCK)[:prompt, None]
            half = torch.maximum(x.abs() * 2.0 ** -4, 2.0 ** -10 * s) if fmt == "e4m3" else 0.5 * s
            assert bool(((got - x).abs() <= half + x.abs() * 2.0 ** -24).all())
        # the last 64 rows weighed the prompt's blocks: each row and query head once
        assert abs(float(layer.cache.weights.sum()) - 64 * hq) < 64 * hq * 2.0 ** -16
    tokens, evictions = prompt, 0
    for step in range(230):
        q, k, v = (_rows(1, h, d, 1000 + 3 * step + i) for i, h in enumerate((hq, hkv, hkv)))
        pos = torch.tensor([prompt + step], device="cuda")
        out = torch.empty(1, hq * d, dtype=torch.bfloat16, device="cuda")
        if tokens == 512:                                   # full: four blocks stay
            before = evicted(layer.cache.tables, 4, 1, 2)
            tokens, evictions = 256, evictions + 1
        else:
            before = None
        sparse_attention_op(pos, empty, empty, None, v, q, k, out, "test.dense")
        tokens += 1
        assert layer.tokens == tokens
        if before is not None:
            assert layer.cache.tables.table.tolist() == before[0]
        if before is not None or step % 40 == 0:
            assert layer.cache.lengths.unique().tolist() == [tokens]
            want, _, _, tol, _ = attention(layer.cache, rotary(pos, q), [1])
            within(out.view(1, hq, d), want, tol, f"step {step}")
    assert evictions == 1


def test_extend_goes_on_with_several_tokens():
    d, hq, hkv = 128, 8, 1
    layer = _layer("test.dense.extend", d, hq, hkv, capacity=400)
    q, k, v = (_rows(380, h, d, i) for i, h in enumerate((hq, hkv, hkv)))
    out = torch.empty(380, hq * d, dtype=torch.bfloat16, device="cuda")
    layer.prefill(q[:200], k[:200], v[:200], out[:200])
    for a, b in ((200, 205), (205, 300), (300, 301), (301, 380)):
        layer.extend(q[a:b], k[a:b], v[a:b], out[a:b])
        want, _, _, tol, _ = attention(layer.cache, q[a:b], [b - a])
        within(out[a:b].view(b - a, hq, d), want, tol, f"rows {a} to {b}")
    # the 8-bit keys and values stand near those of the whole prompt in bf16: e4m3 is off by 2^-4 at most,
    # of a key (a score by its share of 2^-4 |q| |k|) and of a value; random signs leave far less
    exact = _causal(q, k, v, d ** -0.5)
    assert float((out.view(380, hq, d).double().cpu() - exact).norm() / exact.norm()) < 2.0 ** -4
    with pytest.raises(RuntimeError, match="room"):
        layer.extend(q[:70], k[:70], v[:70], out[:70])


def test_a_request_of_one_token_and_a_capture():
    d, hq, hkv = 128, 4, 2
    layer = _layer("test.dense.one", d, hq, hkv, capacity=128)
    from semblo_amd.attention_op import sparse_attention_op
    empty = torch.empty(0, device="cuda")
    for request in range(2):
        layer.reset()
        for step in range(3):
            q, k, v = (_rows(1, h, d, 9 * request + 3 * step + i) for i, h in enumerate((hq, hkv, hkv)))
            out = torch.empty(1, hq * d, dtype=torch.bfloat16, device="cuda")
            sparse_attention_op(empty, empty, q, k, v, q, k, out, "test.dense.one")
            assert layer.tokens == step + 1 and layer.cache.lengths.unique().tolist() == [step + 1]
        want, _, _, tol, _ = attention(layer.cache, q, [1])
        within(out.view(1, hq, d), want, tol, f"request {request}")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.cache.append(k, v)
        with pytest.raises(RuntimeError, match="counts its tokens"):
            layer.extend(q, k, v, out)
    assert layer.tokens == 3


def test_layers_of_both_kinds_share_the_operator():
    from semblo_amd.attention_op import registered_layer
    from semblo_amd.config import SembloRuntimeConfig
    from semblo_amd.model import SembloAttention
    dense = _layer("test.mixed.0", 128, 4, 2, capacity=64)
    sparse = SembloAttention(SembloRuntimeConfig(num_q_heads=4, num_kv_heads=2, head_dim=128), layer_name="test.mixed.1")
    assert registered_layer("test.mixed.0") is dense and registered_layer("test.mixed.1") is sparse


@pytest.mark.parametrize("grid", [False, True])
def test_sessions_rotate_for_the_model(grid):
    """Projections without rotated queries and keys, and a rotary embedding: the same rows as from a model that
    rotates them itself, bit for bit, in the layer-major and the token-order session."""
    from semblo_amd.config import SembloRuntimeConfig
    from semblo_amd.model import SembloAttention
    from semblo_amd.rotary import RotaryEmbedding
    length, hq, hkv, d = 2048, 8, 2, 128
    rotary = RotaryEmbedding(d, rotary_dim=64, sections=(12, 10, 10) if grid else None)
    q, k, v = (_rows(length, h, d, 5 + i) for i, h in enumerate((hq, hkv, hkv)))
    flat = torch.arange(length, device="cuda")
    positions = torch.stack([flat, flat, flat]) if grid else flat
    q_post, k_post = rotary(positions, q, k)
    results = []
    for name, late in (("own", False), ("layer", True)):
        def project(rope, hidden):
            at = hidden[:, 0].long()
            post = (None, None) if late else (q_post[at], k_post[at])
            return post[0], post[1], v[at], q[at], k[at], None
        for order in ("layer", "token"):
            layer = SembloAttention(SembloRuntimeConfig(num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                                        query_chunk_size=512), layer_name=f"test.rotates.{name}.{order}")
            layer.attach_projections(project, lambda attn, gate: attn, rotary=rotary if late else None)
            hidden = flat[:, None].float()
            out = torch.empty(length, hq * d, dtype=torch.bfloat16, device="cuda")
            spans = [(s, s + 512) for s in range(0, length, 512)]
            if order == "layer":
                session = layer.begin_streamed_prefill(positions)
                for s, e in spans:
                    session.keys(positions[..., s:e], hidden[s:e], s, e)
                session.ingest()
                for s, e in spans:
                    out[s:e] = session.queries(positions[..., s:e], flat[s:e], hidden[s:e], s)
            else:
                session = layer.begin_token_outer_prefill(positions, 512, fit_tokens=1024)
                for s, e in spans:
                    out[s:e] = session.slice(hidden[s:e], s, e)
            session.finish()
            results.append(out)
    assert torch.equal(results[0], results[2]) and torch.equal(results[1], results[3])
