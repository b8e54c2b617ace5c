"""Paged caches for the tests: pages in random order, and what they stand for as dense sequences (CPU, fp64)."""

from __future__ import annotations

import math

import torch

from thundersync_amd.paged import CODES, PagedCache, stored_row


def random_cache(g, lengths, *, page, heads, dim, dtype, bits, device, stale=math.nan, spare=3):
    """(cache, table, per sequence keys and values [L, heads, dim]): codes of random scales, `stale` in every place that
    holds no token."""
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + spare, max(max(need, default=0), 1)
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lengths), width), pages - 1, dtype=torch.int32)
    row, at, dense = stored_row(dim), 0, []
    raw = {name: torch.full((pages, heads, page, row), stale) for name in ("key", "value")}
    scales = {name: 2.0 ** torch.randint(-9, -5, (pages, heads, page // 16), generator=g) for name in ("key", "value")}
    for s, n in enumerate(lengths):
        table[s, :need[s]] = order[at:at + need[s]].to(torch.int32)
        at += need[s]
        kv = []
        for name in ("key", "value"):
            x = torch.randn(n, heads, dim, generator=g)
            pos = torch.arange(n)
            ids = table[s].long()[pos // page]
            if bits == 8:
                scale = scales[name][ids, :, pos % page // 16][..., None]
                x = (x / scale).clamp(-448, 448).to(CODES).float()
                kv.append((x * scale).double())
            else:
                x = x.to(dtype).float()
                kv.append(x.double())
            raw[name][ids, :, pos % page, :dim] = x
            raw[name][ids, :, pos % page, dim:] = 0.0
        dense.append(kv)
    if bits == 8:
        pages_of = [raw[name].to(CODES).to(device) for name in ("key", "value")]
        args = [scales[name].float().to(device) for name in ("key", "value")]
    else:
        pages_of, args = [raw[name].to(dtype).to(device) for name in ("key", "value")], [None, None]
    return PagedCache(*pages_of, *args, dtype=dtype, head_dim=dim), table.to(device), dense


def int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def offsets_of(counts, device):
    return int32([sum(counts[:i]) for i in range(len(counts) + 1)], device)


def excess(got, want, bound) -> float:
    """How far the furthest value is past its bound (0 or less: none is); values that are not finite have to be the same."""
    got, want = got.double().cpu(), want.double()
    if not got.numel():
        return 0.0
    fine = want.isfinite()
    if not torch.equal(got[~fine].nan_to_num(nan=1.5), want[~fine].nan_to_num(nan=1.5)):
        return math.inf
    over = ((got - want).abs() - bound)[fine]
    return math.inf if bool(over.isnan().any()) else over.max().item() if over.numel() else 0.0
