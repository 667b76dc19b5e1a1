"""The 8-bit floating-point operators in 64 bits, for tests: quantisation from its definition, products of the numbers that codes and scales stand for, and how far a
result may be off."""
import torch

B = 128
F8 = torch.float8_e4m3fn
# A block's 128 products of two e4m3 numbers (8 bits of significand) are exact.  The tensor cores add 32 of them and a running sum at a time, aligned to the largest: 33 terms
# that lose less than 2^-23 of it each, four times a block.  Then one rounding of the scales' product, one of the sum and its product, per block.
SUM = 4 * 33 * 2.0 ** -23


def blocks(n):
    return (n + B - 1) // B


def scale_of(a):
    """2^k, the least k >= -126 with a <= 448 2^k, for a > 0; 0 for a = 0 (a in fp64)."""
    k = torch.ceil(torch.log2(torch.where(a > 0, a, torch.ones_like(a)) / 448))
    k = torch.where(torch.exp2(k - 1) * 448 >= a, k - 1, torch.where(torch.exp2(k) * 448 < a, k + 1, k)).clamp(min=-126)
    return torch.where(a > 0, torch.exp2(k), torch.zeros_like(a))


def step_of(y):
    """The distance of e4m3 numbers around y."""
    return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)


def nearest(y):
    return torch.round(y / step_of(y)) * step_of(y)


def spread_rows(s, K):
    return s.repeat_interleave(B, -1)[..., :K]


def spread_blocks(s, N, K):
    return s.repeat_interleave(B, -2)[..., :N, :].repeat_interleave(B, -1)[..., :K]


def quantize_rows(x):
    """(numbers of the codes, scales) of fp64 rows."""
    M, K = x.shape
    p = torch.nn.functional.pad(x, (0, -K % B)).view(M, blocks(K), B)
    ok = torch.isfinite(p).all(-1)
    s = scale_of(torch.where(ok[..., None], p, torch.zeros_like(p)).abs().amax(-1))
    c = nearest(p / torch.where(s > 0, s, torch.ones_like(s))[..., None])
    c = torch.where(ok[..., None], c, torch.zeros_like(c)).view(M, blocks(K) * B)[:, :K]
    return c, torch.where(ok, s, torch.full_like(s, float("nan")))


def quantize_blocks(w):
    N, K = w.shape
    p = torch.nn.functional.pad(w, (0, -K % B, 0, -N % B)).view(blocks(N), B, blocks(K), B).transpose(1, 2)
    ok = torch.isfinite(p).all(-1).all(-1)
    s = scale_of(torch.where(ok[..., None, None], p, torch.zeros_like(p)).abs().amax((-1, -2)))
    c = nearest(p / torch.where(s > 0, s, torch.ones_like(s))[..., None, None])
    c = torch.where(ok[..., None, None], c, torch.zeros_like(c)).transpose(1, 2).reshape(blocks(N) * B, -1)[:N, :K]
    return c, torch.where(ok, s, torch.full_like(s, float("nan")))


def rows_back(c, s):
    return c.double() * spread_rows(s.double(), c.shape[1])


def matrix_back(c, s):
    return c.double() * spread_blocks(s.double(), c.shape[-2], c.shape[-1])


def product(x, w):
    """(x w^T, how far fp32 sums of it may be off)."""
    return x @ w.transpose(-1, -2), (SUM + (2 * blocks(x.shape[-1]) + 2) * 2.0 ** -24) * (x.abs() @ w.abs().transpose(-1, -2))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def experts(h, ids, weights, w1, s1, w2, s2, out_dtype):
    """(out, how far it may be off) in 64 bits.  The activation between the products is quantised: where its fp32 error reaches the border between two codes, the code
    next to the right one is allowed for."""
    T, W = h.shape
    E, F = w1.shape[0], w1.shape[1] // 2
    x = rows_back(*quantize_rows(h.double()))
    out, off = (torch.zeros(T, W, dtype=torch.float64, device=h.device) for _ in range(2))
    size = torch.zeros_like(out)
    for e in range(E):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        z, dz = product(x[t], matrix_back(w1[e], s1[e]))
        g, u, dg, du = z[:, :F], z[:, F:], dz[:, :F], dz[:, F:]
        sil = g * torch.sigmoid(g)
        a = sil * u
        # silu's slope is at most 1.1; fp32 exp, quotient and product: eight roundings
        da = 1.1 * dg * (u.abs() + du) + (sil.abs() + 1.1 * dg) * du + 8 * 2.0 ** -24 * a.abs()
        c, s = quantize_rows(a)
        one = spread_rows(torch.where(s > 0, s, torch.ones_like(s)), F)
        y, dy = a / one, da / one
        step = step_of(y)
        border = ((y / step - torch.floor(y / step)) - 0.5).abs() * step          # from the middle between two codes
        near = border <= dy
        # a block whose largest magnitude may pass 448 scales: its smallest numbers may lie on a grid of twice the step
        most = torch.nn.functional.pad(a, (0, 0)).abs().view(-1, F // B, B).amax(-1)
        dmost = da.view(-1, F // B, B).amax(-1)
        moved = spread_rows(((most - dmost).clamp(min=0) <= 448 * s / 2) | (most + dmost > 448 * s), F)
        wrong = torch.where(near, step * one, torch.zeros_like(a)) + torch.where(moved, 2.0 ** -8 * one, torch.zeros_like(a))
        down = matrix_back(w2[e], s2[e])
        r, dr = product(c * one * (s.repeat_interleave(B, 1)[:, :F] > 0), down)
        dr = dr + wrong @ down.abs().T
        if out_dtype == torch.bfloat16:
            dr = dr + half_step(torch.bfloat16) * (r.abs() + dr)
        k = weights[t, j].double()[:, None]
        out.index_add_(0, t, k * r)
        off.index_add_(0, t, k.abs() * dr)
        size.index_add_(0, t, k.abs() * (r.abs() + dr))
    off = off + (ids.shape[1] + 1) * 2.0 ** -24 * size
    return out, off + half_step(out_dtype) * (out.abs() + off)
