"""The 8-bit cache and what reads it from their definitions in 64 bits, on the CPU: what the tests of the operators compare with."""
import numpy as np
import torch


def quantised(x, fmt):
    """fp32 rows [..., n] -> (codes as numbers fp64 [..., n], scales fp32 [...])."""
    x = np.asarray(x, dtype=np.float32).astype(np.float64)
    ok = np.isfinite(x).all(-1)
    x = np.where(ok[..., None], x, 0.0)
    a = np.abs(x).max(-1)
    if fmt == "int8":
        s = (a * np.float64(np.float32(1 / 127))).astype(np.float32)       # a product of two fp32 numbers is whole in 64 bits
    else:
        m, e = np.frexp(a)
        k = np.maximum(e - 9 + (m > 0.875), -126)
        s = np.where(a > 0, np.ldexp(1.0, k), 0.0).astype(np.float32)
    t = np.where(s > 0, s, 1.0).astype(np.float64)[..., None]
    y = np.where(s[..., None] > 0, x / t, 0.0)
    if fmt == "int8":
        c = np.clip(np.rint(y), -127, 127)
    else:
        step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 1e-300))), -6) - 3)
        c = np.rint(y / step) * step
    return np.where(ok[..., None], c, 0.0), np.where(ok, s, np.float32("nan")).astype(np.float32)


def fill(cache, gen):
    """Every row of a CompactKVCache random, as after long use; returns nothing."""
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if cache.fmt == "int8":
            codes.copy_(torch.randint(-127, 128, codes.shape, generator=gen, dtype=torch.int8))
        else:
            codes.copy_((torch.randn(codes.shape, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn))
        scales.copy_(torch.exp(0.5 * torch.randn(scales.shape, generator=gen)) / (80 if codes is cache.k else 40))


def held(cache, layer):
    """(keys, values) of a layer in 64 bits: [pages, G, page_size, n]."""
    f = lambda c, s: c[layer].float().cpu().double() * s[layer].cpu().double()[..., None]  # noqa: E731
    return f(cache.k, cache.k_scale), f(cache.v, cache.v_scale)


def visible(positions, spots, window, first):
    see = spots[None, :] <= positions[:, None]
    if window:
        see &= (positions[:, None] - spots[None, :] < window) | (spots[None, :] < first)
    return see


def attention(q, cache, layer, seqs, scale, window=None, first=0, sinks=None):
    """seqs: [(tokens, start, pages, parents or None)].  q [T, H, d] -> (out [T, H, dv], weighted |v| like it, the largest sum of |scale q k| of a row [T, H, 1], the largest
    weight times scale of a value row times the sum of all codes' magnitudes [T, H, dv])."""
    k, v = held(cache, layer)
    vs = cache.v_scale[layer].cpu().double()
    codes = cache.v[layer].float().cpu().double().abs()
    q, G = q.double().cpu(), cache.num_kv_heads
    T, H = q.shape[:2]
    R, at = H // G, 0
    out, mag, small = (torch.zeros(T, H, cache.vdim, dtype=torch.float64) for _ in range(3))
    top = torch.zeros(T, H, 1, dtype=torch.float64)
    for n, start, pages, parents in seqs:
        kk, vv, cc = (x[pages].transpose(0, 1).reshape(G, -1, x.shape[-1])[:, :start + n] for x in (k, v, codes))
        ss = vs[pages].transpose(0, 1).reshape(G, -1)[:, :start + n].nan_to_num(0.0)
        spots = np.arange(start + n)
        if parents is None:
            pos = spots[start:]
            see = visible(pos, spots, window, first)
        else:
            depth, mine = [], np.zeros((n, n), dtype=bool)
            for i, p in enumerate(parents):
                depth.append(depth[p] + 1 if p >= 0 else 0)
                if p >= 0:
                    mine[i] = mine[p]
                mine[i, i] = True
            pos = start + np.array(depth, dtype=np.int64)
            spots[start:] = pos
            see = visible(pos, spots, window, first)
            see[:, start:] &= mine
        see = torch.from_numpy(see)
        for h in range(H):
            x = q[at:at + n, h] @ kk[h // R].T * scale
            size = (q[at:at + n, h].abs() @ kk[h // R].abs().T * abs(scale)).masked_fill(~see, 0.0)
            x = x.masked_fill(~see, float("-inf"))
            m = x.amax(1, keepdim=True)
            m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
            w = torch.exp(x - m)
            total = w.sum(1, keepdim=True)
            if sinks is not None:
                total = total + torch.exp(sinks[h].double().cpu() - m)
            total = torch.where(total == 0, torch.ones_like(total), total)
            w = torch.where(see, w / total, torch.zeros_like(w))
            shown = [j for j in range(w.shape[1]) if bool(see[:, j].any())]
            wj, vj = w[:, shown], vv[h // R][shown]
            prod = torch.where(see[:, shown, None], wj[:, :, None] * vj[None], torch.zeros((), dtype=torch.float64)) if not bool(torch.isfinite(vj).all()) else None
            out[at:at + n, h] = prod.sum(1) if prod is not None else wj @ vj
            mag[at:at + n, h] = prod.abs().sum(1) if prod is not None else wj @ vj.abs()
            small[at:at + n, h] = (w * ss[h // R]).amax(1, keepdim=True) * (see.double() @ cc[h // R]) if w.shape[1] else 0.0
            top[at:at + n, h] = size.amax(1, keepdim=True) if size.shape[1] else 0.0
        at += n
    return out, mag, top, small


def off_by(q_dtype, out_dtype, keys, d, want, mag, top, small, decoded=False):
    """How far a result may be from `want`: one rounding of the result; weights that are rounded to 11 bits (22 for fp32 results) beside their fp32 sums; and the scores'
    error, which a weight and the sum that divides it both see.  Queries: bf16 numbers are held whole (22 bits of the largest), fp32 ones to 11 bits (22 for fp32 results).
    A sum of n fp32 terms is off by at most n 2^-23 of the terms' magnitudes (the tensor cores may cut instead of round).
    A weight times its value row's scale is held in fp16 over a reference R, and the largest such product so far is at least 2^6 R: it was when R was set, and both shrink by
    the same factor when the maximum grows.  fp16's least step is 2^-24, so each product is off by at most half of that times R, 2^-31 of the largest product, whatever its own
    size, and the result by that times the sum of the codes' magnitudes: `small`."""
    # decoded (bf16 results of sequences with more than 16 rows per kv head): keys and values reach the tensor cores as fp16(code * fp16(scale / unit)), two roundings of
    # 2^-11 on each number of a score's sum and of the result's, where scales are no further apart than 2^21
    wide = out_dtype == torch.float32
    decode = 2.0 ** -10 * 1.001 if decoded and not wide else 0.0
    part = 2.0 ** -21 if wide else 2.0 ** -11
    score = top * (decode + (2.0 ** -21 if wide or q_dtype == torch.bfloat16 else 2.0 ** -11) + (d + 4) * 2.0 ** -23)
    return want.abs() * torch.finfo(out_dtype).eps / 2 + mag * (2 * torch.expm1(score) + part + decode + (keys / 16 + 8) * 2.0 ** -23 + 2.0 ** -20) + small * 2.0 ** -31 + 1e-30
