"""Plain 64-bit statements of the low-bit operators, for their tests.

The 4-bit pool is read through index tables of its documented byte layout (one entry per
slot and dim), so nothing here shares a line with the kernels or the Python wrappers.
"""

import numpy as np
import torch

BLOCK = 2304


def layout():
    """Byte and shift of every (slot, dim) code and byte of every (slot, group) scale, K and V."""
    slot, dim = np.meshgrid(np.arange(16), np.arange(128), indexing="ij")
    k = (64 * slot + 4 * (4 * (dim % 32 // 8) + dim // 32) + dim % 8 // 2, 4 * (dim % 2))
    t, h, e = slot // 4, slot // 2 % 2, slot % 2
    v = (1024 + 512 * h + 64 * (dim % 32 // 4) + 16 * t + 4 * (dim // 32) + 2 * e + dim % 4 // 2, 4 * (dim % 2))
    s4, g4 = np.meshgrid(np.arange(16), np.arange(4), indexing="ij")
    ks = 2048 + 8 * s4 + 2 * g4
    vs = 2176 + 32 * (s4 // 4) + 16 * (s4 // 2 % 2) + 4 * g4 + 2 * (s4 % 2)
    return (k, ks), (v, vs)


def decode(pool):
    """(codes, scales) of K and of V: int [pages, heads, page, 128], float64 [pages, heads, page, 4]."""
    p = pool.cpu().numpy()
    n, h, per, _ = p.shape
    out = []
    for (byte, shift), sc in layout():
        codes = ((p[..., byte] >> shift) & 15).astype(np.int64).reshape(n, h, per * 16, 128)
        scales = np.stack([p[..., sc], p[..., sc + 1]], -1).copy().view(np.float16)[..., 0]
        out.append((torch.from_numpy(codes), torch.from_numpy(scales.astype(np.float64)).reshape(n, h, per * 16, 4)))
    return out


def values(pool):
    """K and V of every slot in float64 [pages, heads, page, 128]."""
    return [(c - 8).double() * s.repeat_interleave(32, -1) for c, s in decode(pool)]


def group_scales(x):
    """f16(min(max|x| / 7, 65504)) of rows [..., 128], float64 [..., 4]."""
    m = x.reshape(*x.shape[:-1], 4, 32).abs().amax(-1) / 7
    return m.clamp(max=65504.0).to(torch.float16).double()


def encode(k, v, pages):
    """A pool of ``pages`` pages (uint8) holding float64 rows k, v [pages, heads, page, 128]."""
    n, h, page, _ = k.shape
    p = np.zeros((n, h, page // 16, BLOCK), np.uint8)
    for ((byte, shift), sc), x in zip(layout(), (k, v)):
        s = group_scales(x)
        r = s.repeat_interleave(32, -1)
        c = (torch.where(r > 0, torch.round(x / torch.where(r > 0, r, torch.ones_like(r))), torch.zeros_like(x)).clamp(-7, 7) + 8)
        c = c.to(torch.uint8).numpy().reshape(n, h, page // 16, 16, 128)
        for half in (0, 4):
            at = shift == half
            p[..., byte[at]] |= c[..., at] << half
        b = s.numpy().astype(np.float16).reshape(n, h, page // 16, 16, 4, 1).view(np.uint8)
        p[..., sc] = b[..., 0]
        p[..., sc + 1] = b[..., 1]
    return torch.from_numpy(p)


def finish(x, norm, eps, positions, inv_freq):
    """RMSNorm (norm [128] or None) and rotation of rows [rows, heads, 128] in float64."""
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * norm.double().cpu()
    if inv_freq is not None:
        ang = positions.cpu().double()[:, None, None] * inv_freq.cpu().double()
        a, b = x[..., :64], x[..., 64:]
        x = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    return x


def attend(pool, table, lens, q, slot_pos, scale):
    """(out, each slot's largest probability, bound on the error) in float64.

    The bound counts the kernel's roundings: the output to bf16 (2^-8 relative), the softmax
    weight and its product with V's scale to f16 (2^-11 each, so 2^-10 of sum p |v|), fp32 sums
    (n / 128 + 16 additions, a block of 16 slots each, 8 warps, and the joins, cut at 2^-23 of
    sum p |v|), and the fp32 logits: 32 products of |q| and codes up to 7 a group and four
    groups, 2^-21 of their absolute sum for the rounding chain, which is an absolute error dl
    of a logit and a relative one 2 dl of every probability.  A weight is carried
    in f16 as at least 2^(e - 5) p s, p <= 1 the largest, e = min(15, 28 - X) and X at most the
    or of the V scales' exponent fields (5 bits are kept for the maximum to grow); below f16's normals it is rounded at 2^-25, before (then times s) and
    after the product, so each slot may add (1 + s) * 7 * 2^-(20 + e) (a code is at most 7, the
    weights' sum at least 1)."""
    kv = values(pool)
    (_, sk), (_, sv) = decode(pool)
    B, hq, _ = q.shape
    hkv, page = pool.shape[1], pool.shape[2] * 16
    grp = hq // hkv
    qd = q.cpu().double().reshape(B, hkv, grp, 128)
    out = torch.zeros(B, hkv, grp, 128, dtype=torch.float64)
    bound = torch.zeros_like(out)
    S = table.shape[1] * page
    score = torch.zeros(B, S, dtype=torch.float64)
    drel = torch.zeros(B, dtype=torch.float64)
    tb, ln = table.cpu().long(), lens.cpu().tolist()
    for b in range(B):
        at = torch.arange(ln[b])
        if slot_pos is not None:
            at = at[slot_pos[b, :ln[b]].cpu() >= 0]
        pg = tb[b][at // page]
        ok = (pg >= 0) & (pg < pool.shape[0])
        at, pg = at[ok], pg[ok]
        if not len(at):
            continue
        k, v = (x[pg, :, at % page] for x in kv)          # [n, hkv, 128]
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", qd[b], k) * scale, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, v)
        mass = torch.einsum("hgn,nhd->hgd", p, v.abs())
        big = 7 * torch.einsum("hgjd,nhj->hgn", qd[b].abs().reshape(hkv, grp, 4, 32), sk[pg, :, at % page])
        dl = 2.0 ** -21 * abs(scale) * big.amax()
        drel[b] = 2 * dl + 2.0 ** -20
        field = int(np.bitwise_or.reduce(sv[pg, :, at % page].numpy().astype(np.float16).view(np.uint16).ravel())) >> 10 & 31
        floor = (1 + sv[pg, :, at % page].max()) * 2.0 ** -(20 + min(15, 28 - field))
        bound[b] = (2.0 ** -8 * out[b].abs() + len(at) * 7 * floor +
                    (2.0 ** -10 + (len(at) / 128 + 16) * 2.0 ** -23 + 2 * drel[b]) * mass)
        score[b, at] = p.amax((0, 1))
    return out.reshape(B, hq, 128), score, bound.reshape(B, hq, 128), drel
