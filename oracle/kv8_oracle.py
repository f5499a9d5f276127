"""The 8-bit K/V cache and the block-sparse attention, restated in 64 bits from their
definitions (test infrastructure).  Where a definition fixes an fp32 rounding (a scale, a
code, a score) the rounding is applied; everything else stays in float64."""

from __future__ import annotations

import torch

BLOCK = 16
TINY = 2.0 ** -100
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def r32(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.float32).to(torch.float64)


def _grid(y: torch.Tensor, dtype) -> torch.Tensor:
    """y rounded to the nearest code (ties to even)."""
    if dtype is torch.int8:
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def codes_of(rows: torch.Tensor, qmax: float, dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) of blocks rows [..., values]."""
    a = rows.abs().amax(-1)
    live = a >= TINY
    inv = torch.where(live, r32(qmax / a.clamp_min(TINY)), 0.0)
    return _grid(r32(rows * inv[..., None]), dtype), torch.where(live, r32(a / qmax), 0.0)


def blocked(x: torch.Tensor) -> torch.Tensor:
    """[H, n, D] -> [H, blocks, 16 * D], zeros past n."""
    H, n, D = x.shape
    nb = -(-n // BLOCK)
    y = torch.zeros((H, nb * BLOCK, D), dtype=torch.float64, device=x.device)
    y[:, :n] = x.double()
    return y.view(H, nb, BLOCK * D)


def quantize(x: torch.Tensor, dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """codes [H, blocks * 16, D] (float64) and scales [H, blocks] of rows x [H, n, D]."""
    H, n, D = x.shape
    c, s = codes_of(blocked(x), QMAX[dtype], dtype)
    return c.view(H, -1, D), s


def values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    H, rows, D = codes.shape
    return (codes.double().view(H, rows // BLOCK, -1) * scale.double()[..., None]).view(H, rows, D)


def digest(k: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """codes [H, blocks, 2, D] and scales [H, blocks]."""
    H, n, D = k.shape
    nb = -(-n // BLOCK)
    f = torch.cat([k.double(), k[:, -1:].double().expand(-1, nb * BLOCK - n, -1)], 1).view(H, nb, BLOCK, D)
    mm = torch.stack([f.amax(2), f.amin(2)], 2)
    c, s = codes_of(mm.view(H, nb, 2 * D), 127.0, torch.int8)
    return c.view(H, nb, 2, D), s


def select(q, dcodes, dscale, positions, top, sink=1, recent=1) -> torch.Tensor:
    """The ascending block lists [m, H, top] (-1 past a row's last visible block)."""
    m, Hq, D = q.shape
    H, nb_all = dscale.shape
    G = Hq // H
    out = torch.full((m, H, top), -1, dtype=torch.int64)
    pos = positions.tolist()
    for i in range(m):
        nb = (pos[i] + BLOCK) // BLOCK if pos[i] >= 0 else 0
        for h in range(H):
            x = q[i, h * G:(h + 1) * G].double()
            a = x.abs().amax(-1)
            a = torch.where(a >= TINY, a, 0.0)
            c, _ = codes_of(x, 127.0, torch.int8)
            mx, mn = dcodes[h, :nb, 0].double(), dcodes[h, :nb, 1].double()
            bound = torch.maximum(c[:, None] * mx, c[:, None] * mn).sum(-1)
            score = r32(r32(bound * a[:, None]).amax(0) * dscale[h, :nb].double()) if nb else torch.zeros(0)
            b = torch.arange(nb, device=score.device)
            forced = (b < sink) | (b >= nb - recent)
            score = torch.where(forced, torch.inf, score)
            order = torch.sort(score, descending=True, stable=True).indices[:top].sort().values
            out[i, h, :order.numel()] = order.cpu()
    return out


def attend(q, k, v, positions, blocks=None, scale=None):
    """(out [m, Hq, D], mass [m, Hq, D]) in float64: softmax(q k^T scale) v over the visible keys
    (of the listed blocks), zeros for a row that sees none; mass is the same sum over |v|."""
    m, Hq, D = q.shape
    H, n, _ = k.shape
    G = Hq // H
    out = torch.zeros((m, Hq, D), dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    scale = D ** -0.5 if scale is None else scale
    key = torch.arange(n, device=q.device)
    for h in range(H):
        see = key[None] <= positions.to(q.device).long()[:, None]
        if blocks is not None:
            nb = -(-n // BLOCK)
            bm = torch.zeros((m, nb + 1), dtype=torch.bool, device=q.device)
            lst = blocks[:, h].to(q.device).long()
            bm.scatter_(1, torch.where((lst < 0) | (lst >= nb), nb, lst), True)
            see = see & bm[:, :nb].repeat_interleave(BLOCK, 1)[:, :n]
        kk, vv = k[h].double(), v[h].double()
        kk, vv = torch.nan_to_num(kk, 0.0, 0.0, 0.0), torch.nan_to_num(vv, 0.0, 0.0, 0.0)
        any_ = see.any(1, keepdim=True)
        for g in range(G):
            s = (q[:, h * G + g].double() @ kk.T) * scale
            s = s.masked_fill(~see, -torch.inf)
            s = torch.where(any_, s, 0.0)
            p = torch.softmax(s, -1) * any_
            out[:, h * G + g] = p @ vv
            mass[:, h * G + g] = p @ vv.abs()
    return out, mass
