"""Error bounds of the decode over the 8-bit cache, head by head and column by column.

u = 2^-24.  Of one token's weight (natural logarithm, relative):
  scores   fp32 sums of D exact products on the tensor pipe, 2 u a product (it may truncate): 2 D u size, size =
           max_t scale sum|q k|; up to 16 u size for the products with the scales, log2 e and the subtractions of the
           references, 4 u max|ev| for x + ev; Q in f16: 2^-25 of its row's power of two a lost bit below 2^-14.
  ex2      2^-22, and 2^-22 each for up to 16 corrections of a running reference.
The f16 weight 2^(x + ev - M): 2^-11 of itself; below f16's normals half a step 2^-25, in units where the largest of
the rows that are not all zeros is at least 1: 2^-25 W sum_t|code_td|, W = max p_t 2^ev_t over those rows.
Sums: a warp adds 16 tokens of 64 a step on the tensor pipe, 17 terms of 2 u: 34 u n / 64; merges and joins of the
segments 2 u each, fewer than 400 u.  Join: __expf and __logf 2^-20.  Output: 2^-8 of the value (bf16).
"""
import numpy as np

from oracle import cache_oracle as co

U = 2.0 ** -24


def gather(codes, sc, bt, b, n, w):
    """(codes, values, exponents) of the n tokens of sequence b, K (w = 0) or V (1)."""
    ps = codes.shape[2]
    t = np.arange(n)
    pg, sl = bt[b, t // ps], t % ps
    c, s = codes[w][pg, sl], sc[pg, :, w, sl]
    return c, co.cache_values(c, s), s.astype(np.float64) - 127


def expected(q, k, v, v_codes, ev, scale):
    """(O, LSE, bound of O, bound of LSE) of one sequence; q [Hq, D], k and v [L, Hkv, D] fp64."""
    Hq, D = q.shape
    n, Hkv, _ = k.shape
    G = Hq // Hkv
    wo, wl, mean_abs, size = co.decode(q, k, v, scale)
    if n == 0:
        return wo, wl, np.zeros_like(wo), np.zeros_like(wl)
    x = np.einsum("hd,lhd->hl", q, np.repeat(k, G, 1)) * scale
    p = np.exp(x - wl[:, None])                                           # [Hq, L]
    some = np.any((v_codes & 127) != 0, -1)                               # [L, Hkv] rows that are not all zeros
    held = np.repeat(np.where(some, 2.0 ** ev, 0.0), G, 1).T              # [Hq, L]
    W = (p * held).max(-1)
    code_sum = np.repeat(np.abs(co.e4m3_values()[v_codes]).sum(0), G, 0)  # [Hq, D]
    top = np.frexp(np.abs(q).max(-1))[1]
    lost = np.where(np.any((q != 0) & (np.abs(q) < 2.0 ** (top - 1 - 14.0)[:, None]), -1), 1.0, 0.0)
    dq = lost * scale * 2.0 ** (top - 1) * 2.0 ** -25 * np.repeat(np.abs(k).sum(-1).max(0), G)
    d = (2 * D + 16) * U * size + 4 * U * np.abs(ev).max() + dq + 17 * 2.0 ** -22
    sums = (0.6 * n + 400) * U + 2.0 ** -20
    tol_o = 2.0 ** -8 * np.abs(wo) + (mean_abs * (2.0 ** -11 + 2 * d + 2 * sums)[:, None] + 2.0 ** -25 * W[:, None] * code_sum) * (1 + 2.0 ** -7)
    return wo, wl, tol_o, d + sums + 4 * U * np.abs(wl) + 2.0 ** -20


def check(o, lse, q, codes, sc, bt, lens, scale=None):
    D = q.shape[2]
    scale = scale if scale is not None else 1 / np.sqrt(D)
    o, lse = o.float().cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    for b, n in enumerate(lens):
        _, k, _ = gather(codes, sc, bt, b, n, 0)
        vc, v, ev = gather(codes, sc, bt, b, n, 1)
        wo, wl, tol_o, tol_l = expected(q[b].double().numpy(), k, v, vc, ev, scale)
        if n == 0:
            assert np.all(o[b] == 0) and np.all(np.isneginf(lse[b])), b
            continue
        assert np.all(np.abs(lse[b] - wl) <= tol_l), (b, np.abs(lse[b] - wl).max(), tol_l.min())
        bad = ~(np.abs(o[b] - wo) <= tol_o)
        assert not bad.any(), (b, int(bad.sum()), float((np.abs(o[b] - wo) / tol_o).max()))


def marked(codes, sc, bt, lens):
    """Turns the cache's sequences into flat weights (keys 2^-6 of what they are) over values of one sign that tell
    where they are: of every 16 runs of 128 tokens, column d is 32 times larger in run d mod 16."""
    ps, D = codes.shape[2], codes.shape[4]
    for b, n in enumerate(lens):
        t = np.arange(n)
        pg, sl = bt[b, t // ps], t % ps
        sc[pg, :, 0, sl] -= 6
        here = ((t // 128) % 16)[:, None] == (np.arange(D) % 16)[None]
        codes[1][pg, sl] = (codes[1][pg, sl] & 7) | np.where(here, 0x60, 0x38)[:, None]    # 32 to 60, 1 to 1.875
        sc[pg, :, 1, sl] = 123
