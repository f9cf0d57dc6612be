"""Shared helpers of the rotary and 8-bit cache tests: the definitions in 64 bits on the CPU."""
from __future__ import annotations

import math

import torch

BLOCK = 64
CODE_MAX = {"e4m3": 448.0, "int8": 127.0}


def decode(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    """The numbers that codes stand for, from their bits."""
    c = codes.long()
    if fmt == "int8":
        return (c - 256 * (c >= 128)).double()
    sign, e, m = 1.0 - 2.0 * (c >> 7), (c >> 3) & 15, c & 7
    v = torch.where(e == 0, m / 512.0, (1 + m / 8.0) * torch.exp2((e - 7).double()))
    return sign * torch.where((e == 15) & (m == 7), float("nan"), v)


def held(cache, s: int, h: int):
    """Keys and values [length, D] that a cache holds for one (sequence, head), in 64 bits."""
    n = int(cache.lengths[s, h])
    blocks = -(-n // BLOCK)
    place = cache.tables.table[s, h, :blocks].long().cpu()
    k = decode(cache.codes_k[s, h].cpu()[place], cache.fmt) * cache.scales[0, s, h].cpu()[place].double()[:, None, None]
    v = decode(cache.codes_v[s, h].cpu()[place], cache.fmt) * cache.scales[1, s, h].cpu()[place].double()[:, None, None]
    return k.flatten(0, 1)[:n], v.transpose(1, 2).flatten(0, 1)[:n]


def attention(cache, q: torch.Tensor, rows: list[int], first: int = 0, sm_scale: float | None = None):
    """(out, lse, weights added, bound of out's error, bound of lse's) in 64 bits, of the rows first .. first + sum(rows).

    The bounds.  A probability is rounded once, to fp16 (2^-11 of it), and the result once, to bf16 (2^-8 of
    it).  The scores are fp32 sums of D products and one scaling: off by at most (D + 8) 2^-24 of the
    products' magnitudes, which is a relative error of the probability, doubled by the normalisation; the
    exponential and the sums over the keys add no more than 2^-19.
    Below fp16's normal numbers the rounding is absolute: with the largest scale of the sequence's values as unit and
    2^11 over it, a probability times its block's scale (over a sum of at least 1) is off by at most
    2^-25 / 2^11 of the unit, and never by more than itself."""
    q = q.double().cpu()
    t, hq, d = q.shape
    g = hq // cache.num_kv_heads
    scale = d ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(t, hq, d, dtype=torch.float64)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    added = torch.zeros(cache.tables.weights.shape, dtype=torch.float64)
    at = first
    for s, n in enumerate(rows):
        for h in range(cache.num_kv_heads):
            k, v = held(cache, s, h)
            if n == 0 or k.shape[0] == 0:
                continue
            scales = cache.scales[1, s, h].cpu()[cache.tables.table[s, h].long().cpu()].double()[:-(-k.shape[0] // BLOCK)]
            of_key = scales.repeat_interleave(BLOCK)[:k.shape[0], None]
            for i in range(n):
                see = k.shape[0] - n + i + 1
                if see <= 0:
                    continue
                x = q[at + i, h * g:(h + 1) * g]
                sc = x @ k[:see].T * scale
                p = torch.softmax(sc, -1)
                out[at + i, h * g:(h + 1) * g] = p @ v[:see]
                lse[at + i, h * g:(h + 1) * g] = torch.logsumexp(sc, -1)
                off = (d + 8) * 2.0 ** -24 * (x.abs() @ k[:see].abs().T * abs(scale)).amax(-1) + 2.0 ** -20
                tol[at + i, h * g:(h + 1) * g] = 2.0 ** -8 * (p @ v[:see]).abs() + \
                    (p @ v[:see].abs()) * (2.0 ** -11 + 2 * off + 2.0 ** -19)[:, None] + \
                    torch.minimum(p, 2.0 ** -36 * scales.max() / of_key[:see, 0]) @ v[:see].abs()
                ltol[at + i, h * g:(h + 1) * g] = off + 2.0 ** -22 * (1 + lse[at + i, h * g:(h + 1) * g].abs())
                whole = torch.nn.functional.pad(p.sum(0), (0, -see % BLOCK))
                added[s, h, :whole.numel() // BLOCK] += whole.view(-1, BLOCK).sum(1)
        at += n
    return out, lse, added, tol, ltol


def within(got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor, what: str) -> None:
    got = got.double().cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f"{what}: other values are finite"
    ok = torch.isfinite(want)
    over = ((got - want).abs() - tol)[ok]
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f"{what}: {int((over > 0).sum())} of {over.numel()} past the bound, by up to {float(over.max()):.3g}"


def evicted(tables, keep: int, sink: int, recent: int):
    """CacheTables.evict by its definition, list by list."""
    table, weights = tables.table.tolist(), tables.weights.tolist()
    lengths, open_block = tables.lengths.tolist(), tables.open_block.tolist()
    for s, heads in enumerate(table):
        for h, places in enumerate(heads):
            n = -(-lengths[s][h] // BLOCK)
            w = [x if x > 0 else 0.0 for x in weights[s][h]]
            stay = list(range(n))
            if n > keep:
                middle = sorted(range(sink, n - recent), key=lambda b: (-w[b], b))[:keep - sink - recent]
                stay = [*range(sink), *sorted(middle), *range(n - recent, n)]
            gone = [b for b in range(n) if b not in set(stay)]
            table[s][h] = [places[b] for b in [*stay, *gone, *range(n, len(places))]]
            weights[s][h] = [weights[s][h][b] for b in stay] + [0.0] * (len(places) - len(stay))
            lengths[s][h] -= BLOCK * len(gone)
            o = open_block[s][h]
            open_block[s][h] = stay.index(o) if o in stay else -1
    return table, weights, lengths, open_block
