"""Plain 64-bit forms of the 8-bit block-scaled operators and of the grouped router, with the error bounds their tests use."""
from __future__ import annotations

import math

import numpy as np
import torch

B = 128
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # half a step, relative: finfo(t).eps / 2


def up(n):
    return -(-n // B)


def nearest_e4m3(v):
    """fp64 → the nearest e4m3 value, ties to the even code; |v| ≤ 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


def border(v, eps):
    """Step of the code where v (fp64) is within eps·|v| of the border between two codes, 0 elsewhere."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    f = v.abs() / step
    return torch.where(((f - torch.floor(f)) - 0.5).abs() <= eps * (f + 1.0), step, 0.0)


def codes_to_f64(q):
    return q.view(torch.float8_e4m3fn).to(torch.float64)


def quant_rows(v):
    """v fp64 [M, K] → (code values fp64 [M, K], stored scales fp64 [ceil(K/128), M])."""
    M, K = v.shape
    p = torch.nn.functional.pad(v, (0, up(K) * B - K)).view(M, up(K), B)
    amax = p.abs().amax(2)
    q = torch.where(amax[:, :, None] > 0, nearest_e4m3(p * 448.0 / torch.where(amax > 0, amax, 1.0)[:, :, None]), 0.0)
    return q.view(M, -1)[:, :K], (amax / 448.0).float().double().T.contiguous()


def quant_blocks(w):
    """w fp32 or bf16 [N, K] → (code values, scales [ceil(N/128), ceil(K/128)]); v · 448 and its quotient by amax are fp32."""
    N, K = w.shape
    p = torch.nn.functional.pad(w.float(), (0, up(K) * B - K, 0, up(N) * B - N)).view(up(N), B, up(K), B)
    amax = p.abs().amax((1, 3))
    q = nearest_e4m3((p * 448.0 / torch.where(amax > 0, amax, 1.0)[:, None, :, None]).double())
    return q.view(up(N) * B, -1)[:N, :K].contiguous(), (amax.double() / 448.0).float().double()


def spread(s, N, K):
    return s.double().repeat_interleave(B, 0)[:N].repeat_interleave(B, 1)[:, :K]


def gemm(xq, xs, wq, ws):
    """(y, Σ|terms|) of code values xq [M, K], scales xs [KB, M], wq [N, K], ws: fp64."""
    x = xq * xs.T.repeat_interleave(B, 1)[:, :xq.shape[1]]
    w = wq * spread(ws, *wq.shape)
    return x @ w.T, x.abs() @ w.abs().T


def sum_bound(K):
    """Of an fp32 sum of K exact products in any order, cut instead of rounded, relative to Σ|terms|: a step (2^-23) an addition, of which a value
    meets 128 in its block and one a block after it; three roundings of the scales' products."""
    return (128 + up(K) + 4) * 2.0 ** -23


def moe(ids, w, recs, x, limit=0.0, shared=None, gate=None):
    """Routed experts: recs[e] = ((q1, s1), (q3, s3), (q2, s2)) of code values and scales (None: not here).  Returns (out fp64, bound of an fp32
    result's error): the sums' bounds are carried through silu(g)·u; where a value of y is that near to the border of two codes it may take the other;
    d is rounded to bf16.  Third: the root of Σ_k (w·d)², what roundings that do not know of each other are relative to."""
    M, H = x.shape
    K = ids.shape[1]
    out = torch.zeros(M, H, dtype=torch.float64, device=x.device)
    tol, mag = torch.zeros_like(out), torch.zeros_like(out)
    xq, xs = quant_rows(x.double())
    for e, rec in enumerate(recs):
        m, k = (ids == e).nonzero(as_tuple=True)
        if rec is None or m.numel() == 0:
            continue
        (q1, s1), (q3, s3), (q2, s2) = rec
        I = q1.shape[0]
        g, ga = gemm(xq[m], xs[:, m], q1, s1)
        u, ua = gemm(xq[m], xs[:, m], q3, s3)
        dg, du = ga * sum_bound(H), ua * sum_bound(H)
        if limit > 0:
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        y = g * torch.sigmoid(g) * u
        # |silu'| ≤ 1.1, |silu(g)| ≤ |g|; the exponential, the division and the products of silu cost some 16 fp32 roundings together
        dy = 1.1 * dg * (u.abs() + du) + g.abs() * du + 2.0 ** -20 * y.abs()
        p = y.view(-1, I // B, B)
        amax = p.abs().amax(2, keepdim=True)
        damax = dy.view_as(p).amax(2, keepdim=True)
        safe = torch.where(amax > 0, amax, 1.0)
        v = p * 448.0 / safe
        eps = (dy.view_as(p) / p.abs().clamp_min(1e-300) + damax / safe + 2.0 ** -22).clamp_max(1.0)   # relative change of a quotient
        yq = nearest_e4m3(v.clamp(-448, 448))
        flip = torch.maximum(border(v, eps), torch.where(eps >= 0.5, v.abs() + 2.0 ** -9, 0.0))        # other code: at most a step away
        sc = (amax / 448.0).float().double()
        yv, yt = (yq * sc).view(-1, I), ((flip + yq.abs() * (damax / safe + 2.0 ** -23)) * sc).view(-1, I)
        W2 = q2 * spread(s2, H, I)
        d, da = yv @ W2.T, yv.abs() @ W2.abs().T
        dd = yt @ W2.abs().T + sum_bound(I) * da
        dd = dd + HALF[torch.bfloat16] * (d.abs() + dd)
        wk = w[m, k].double()[:, None]
        out.index_add_(0, m, wk * d)
        mag.index_add_(0, m, (wk * d) ** 2)
        tol.index_add_(0, m, wk.abs() * dd + 2.0 ** -23 * K * wk.abs() * d.abs())
    if shared is not None:
        sh = shared.double() * (1.0 if gate is None else torch.sigmoid(gate.double())[:, None])
        out, tol = out + sh, tol + 2.0 ** -20 * sh.abs()
    return out, tol, mag.sqrt()


def route(logits, bias, k, n_group, topk_group, group_top, score, renorm, scale):
    """The grouped router in 64 bits on numpy arrays: (ids, w)."""
    l = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    M, E = l.shape
    with np.errstate(over="ignore", invalid="ignore"):
        if score == "sigmoid":
            s = 1.0 / (1.0 + np.exp(-l))
        else:
            mx = l.max(1, keepdims=True)
            p = np.exp(l - np.where(np.isinf(mx), 0.0, mx))
            t = p.sum(1, keepdims=True)
            s = np.where(t > 0, p / np.where(t > 0, t, 1.0), 0.0)
    c = s + (0.0 if bias is None else bias.astype(np.float64))
    size = E // n_group
    top = np.sort(c.reshape(M, n_group, size), axis=2)[:, :, ::-1][:, :, : min(group_top, size)].sum(2)
    ids = np.zeros((M, k), np.int32)
    for m in range(M):
        groups = sorted(range(n_group), key=lambda g: (-top[m, g], g))[:topk_group] if topk_group < n_group else range(n_group)
        on = sorted(e for g in groups for e in range(g * size, (g + 1) * size))
        ids[m] = sorted(on, key=lambda e: (-c[m, e], e))[:k]
    w = np.take_along_axis(s, ids, 1)
    if renorm:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return ids, w * scale


def route_bound(logits, score):
    """Relative error of an fp32 weight: exp, 1 + e, a division, a sum of 16, a division, a product: under 32 half steps; the softmax's argument l - max is off by
    half a step of its own size, and its sum of up to 1024 terms, of which a lane adds 32 and a tree the rest, by 37."""
    if score == "sigmoid":
        return 32 * 2.0 ** -24
    f = np.where(np.isfinite(logits), logits, 0.0)
    return (80 + 4 * math.ceil(float(np.max(f.max(1) - f.min(1))))) * 2.0 ** -24
