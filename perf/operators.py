"""Cases for the low-bit serving operators: appending keys and values, rotated on the way,
to a paged cache held in 4 bits; single-token attention over that cache; and the matrix
product in 8-bit integers with a scale for each token and each output channel.

``run`` computes a case either in its plain form (elementary torch operations in 32 bits)
or, where ``own`` is true, through the framework's public calls.

The 4-bit cache.  A pool is a uint8 tensor [pages][kv heads][page_size / 16][2304]; a
2304-byte block holds 16 slots of one kv head.  A row of 128 values is four groups of 32;
a group has the scale f16(min(max|x| / 7, 65504)) and each value the code
8 + clip(rint(x / scale), -7, 7).  Bytes of a block:
    0    K codes: slot s at 64 s; dim 32 j + 8 t + n is nibble n of the 32-bit word 4 t + j
    1024 V codes: slot s = 4 t + 2 h + e; dim 32 i + 4 g + n is nibble n of the 16-bit word
         at 512 h + 64 g + 16 t + 4 i + 2 e
    2048 K scales: f16, slot s, group j at 8 s + 2 j
    2176 V scales: f16, slot s = 4 t + 2 h + e, group i at 32 t + 16 h + 4 i + 2 e
"""

import math

import numpy as np
import torch

own = False

BLOCK, ROWS, DIM = 2304, 16, 128
DEV = "cuda"


# ---------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step's rows of a small batch: the launch latency counts
        {"name": "append_decode_8", "op": "append", "seqs": 8, "rows": 8, "heads": 28, "kv_heads": 4, "page": 16,
         "bias": True, "norm": False, "far": 40000},
        # one decode step's rows of a large batch, with q/k norms
        {"name": "append_decode_256", "op": "append", "seqs": 256, "rows": 256, "heads": 32, "kv_heads": 8, "page": 64,
         "bias": False, "norm": True, "far": 131072},
        # the prompts of five sequences of different lengths, appended in one call
        {"name": "append_prompts_16411", "op": "append", "seqs": 5, "rows": 16411, "heads": 28, "kv_heads": 4,
         "page": 64, "bias": True, "norm": False, "far": 32768},
        # one short sequence: the smallest attention call
        {"name": "attend_1x256", "op": "attend", "batch": 1, "heads": 16, "kv_heads": 2, "slots": 256, "page": 16,
         "lens": "full", "masked": True, "score": True},
        # sixteen capped sequences with freed slots and the eviction score
        {"name": "attend_16x1032", "op": "attend", "batch": 16, "heads": 28, "kv_heads": 4, "slots": 1032, "page": 16,
         "lens": "full", "masked": True, "score": True},
        # a large batch of capped sequences: streaming the cache is all there is
        {"name": "attend_64x4104", "op": "attend", "batch": 64, "heads": 32, "kv_heads": 8, "slots": 4104, "page": 64,
         "lens": "full", "masked": True, "score": True},
        # sequences of very different lengths (an empty one among them), no eviction
        {"name": "attend_ragged_12", "op": "attend", "batch": 12, "heads": 28, "kv_heads": 4, "slots": 32701,
         "page": 128, "lens": "ragged", "masked": False, "score": False},
        # one long sequence
        {"name": "attend_1x131071", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "slots": 131071, "page": 64,
         "lens": "full", "masked": False, "score": False},
        # one token through a q/k/v projection
        {"name": "int8_1x6144x2560", "op": "int8", "tokens": 1, "out": 6144, "in": 2560, "bias": False, "f32": False},
        # sixteen tokens through a gate/up projection: streaming the weight
        {"name": "int8_16x37888x3584", "op": "int8", "tokens": 16, "out": 37888, "in": 3584, "bias": False,
         "f32": False},
        # a ragged chunk of a few hundred tokens, partial sums kept in 32 bits
        {"name": "int8_333x2560x9728", "op": "int8", "tokens": 333, "out": 2560, "in": 9728, "bias": True, "f32": True},
        # the rows of a prompt through a gate/up projection
        {"name": "int8_8192x37888x3584", "op": "int8", "tokens": 8192, "out": 37888, "in": 3584, "bias": False,
         "f32": False},
    ]


HEADS = [(28, 4), (16, 2), (32, 8), (8, 2), (7, 1), (8, 8), (24, 4), (8, 1)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "int8", "int8"])
    heads, kv = rng.choice(HEADS)
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "append":
        rows = _log(rng, 1, 16000)
        return {"op": op, "seqs": max(1, min(rows, _log(rng, 1, 256))), "rows": rows, "heads": heads, "kv_heads": kv,
                "page": page, "bias": rng.random() < 0.5, "norm": rng.random() < 0.5, "far": _log(rng, 100, 400000)}
    if op == "attend":
        batch = _log(rng, 1, 200)
        slots = _log(rng, 1, max(2, min(131072, 2000000 // (batch * kv))))
        lens = rng.choice(["full", "ragged"])
        masked = rng.random() < 0.5
        return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv, "slots": slots, "page": page, "lens": lens,
                "masked": masked, "score": masked and rng.random() < 0.6}
    tokens = rng.choice([1, _log(rng, 2, 32), _log(rng, 33, 512), _log(rng, 513, 8000)])
    n, k = _log(rng, 100, 38000), _log(rng, 64, 19000)
    if tokens > 512:
        n = max(100, min(n, int(1.0e12 / (tokens * k))))
    return {"op": op, "tokens": tokens, "out": n, "in": k, "bias": rng.random() < 0.5, "f32": rng.random() < 0.3}


# ------------------------------------------------------------------ the cache's encoding
def _over(x, n):
    """x / n, correctly rounded (a division by a Python number multiplies by its rounded reciprocal)."""
    return x / torch.full_like(x, n)


def _scales(x):
    """f16 group scales of rows x [..., 128] (32-bit), shape [..., 4]."""
    return _over(x.reshape(*x.shape[:-1], 4, 32).abs().amax(-1), 7).clamp(max=65504.0).to(torch.float16)


def _codes(x, scale):
    """Codes 1..15 of rows x [..., 128] under their f16 scales [..., 4]."""
    s = scale.to(x.dtype).unsqueeze(-1)
    g = x.reshape(*x.shape[:-1], 4, 32)
    q = torch.where(s > 0, torch.round(g / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(g))
    return (q.clamp(-7, 7) + 8).to(torch.uint8).reshape(x.shape)


def _nibbles(c):
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _row_bytes(k, v):
    """The 144 bytes of each K, V row pair [..., 128] (32-bit): K codes, V codes, K scales,
    V scales, in the order of _bytes_of_slot."""
    lead = k.shape[:-1]
    ks, vs = _scales(k), _scales(v)
    kc = _codes(k, ks).reshape(*lead, 4, 4, 8).transpose(-3, -2).reshape(*lead, DIM)    # j t n -> t j n
    vc = _codes(v, vs).reshape(*lead, 4, 8, 4).transpose(-3, -2).reshape(*lead, DIM)    # i g n -> g i n
    return torch.cat([_nibbles(kc), _nibbles(vc), ks.view(torch.uint8), vs.view(torch.uint8)], -1)


def _row_values(b):
    """K and V rows [..., 128] in 32 bits of their bytes [..., 144]."""
    lead = b.shape[:-1]
    c = torch.stack([b[..., :128] & 15, b[..., :128] >> 4], -1).reshape(*lead, 2, DIM).to(torch.float32) - 8
    sc = b[..., 128:].contiguous().view(torch.float16).to(torch.float32).reshape(*lead, 2, 4, 1)
    k = c[..., 0, :].reshape(*lead, 4, 4, 8).transpose(-3, -2).reshape(*lead, 4, 32) * sc[..., 0, :, :]
    v = c[..., 1, :].reshape(*lead, 8, 4, 4).transpose(-3, -2).reshape(*lead, 4, 32) * sc[..., 1, :, :]
    return k.reshape(*lead, DIM), v.reshape(*lead, DIM)


def _bytes_of_slot(r):
    """The 144 bytes of slot r [rows] within a block, as [rows, 144] offsets."""
    r = r[:, None]
    t, h, e = r // 4, r // 2 % 2, r % 2
    i64 = torch.arange(64, device=r.device)
    w, lo = i64 // 2, i64 % 2  # 16-bit word 4 g + i of V and its byte
    i8 = torch.arange(8, device=r.device)
    return torch.cat([64 * r + i64, 1024 + 512 * h + 64 * (w // 4) + 16 * t + 4 * (w % 4) + 2 * e + lo,
                      2048 + 8 * r + i8, 2176 + 32 * t + 16 * h + 4 * (i8 // 2) + 2 * e + i8 % 2], 1)


def _blocks(k, v):
    """Pool blocks [..., n, 2304] of K and V rows [..., 16 n, 128] in 32 bits."""
    lead, n = k.shape[:-2], k.shape[-2] // ROWS
    where = torch.argsort(_bytes_of_slot(torch.arange(ROWS, device=k.device)).reshape(-1))
    return _row_bytes(k, v).reshape(*lead, n, BLOCK)[..., where]


# --------------------------------------------------------------------------- the inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _tables(g, seqs, per_seq, page, spare):
    """Page tables over a pool whose pages come in no order; entries past a sequence's
    pages are -1.  Returns the table and the number of pages."""
    need = (per_seq + page - 1) // page
    ends = torch.cumsum(need, 0)
    total = int(ends[-1]) + spare
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    width = max(1, int(need.max()))
    j = torch.arange(width, device=DEV)
    idx = (ends - need)[:, None] + j
    inside = j < need[:, None]
    return torch.where(inside, perm[idx.clamp(max=total - 1)], torch.full_like(idx, -1, dtype=torch.int32)), total


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "append":
        return _prepare_append(case, g)
    if case["op"] == "attend":
        return _prepare_attend(case, g)
    return _prepare_int8(case, g)


def _prepare_append(c, g):
    rows, seqs, hq, hkv = c["rows"], c["seqs"], c["heads"], c["kv_heads"]
    # rows of each sequence: uneven, every sequence at least one
    cuts = torch.sort(torch.randperm(max(1, rows - 1), generator=g, device=DEV)[: seqs - 1] + 1)[0]
    edge = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), cuts,
                      torch.full((1,), rows, dtype=torch.long, device=DEV)])
    count = edge[1:] - edge[:-1]
    seq = torch.repeat_interleave(torch.arange(count.numel(), device=DEV), count)
    have = torch.randint(0, 300, (count.numel(),), generator=g, device=DEV)  # slots in use before
    slots = have[seq] + torch.arange(rows, device=DEV) - edge[seq]
    start = torch.randint(0, max(1, c["far"]), (count.numel(),), generator=g, device=DEV)
    table, pages = _tables(g, count.numel(), have + count, c["page"], 3)
    qkv = _randn(g, rows, (hq + 2 * hkv) * DIM)
    # keys have a few large channels
    loud = 1 + 5 * (torch.rand(hkv * DIM, generator=g, device=DEV) < 0.03).to(torch.float32)
    qkv[:, hq * DIM:(hq + hkv) * DIM] *= loud
    s = {"case": c, "qkv": qkv.to(torch.bfloat16), "seq": seq.to(torch.int32), "slots": slots.to(torch.int32),
         "positions": (start[seq] + torch.arange(rows, device=DEV) - edge[seq]).to(torch.int32), "table": table,
         "pool": torch.zeros(pages, hkv, c["page"] // ROWS, BLOCK, dtype=torch.uint8, device=DEV),
         "inv_freq": torch.pow(torch.full((64,), 1e6, device=DEV), -torch.arange(64, device=DEV) / 64.0),
         "bias": (0.5 * _randn(g, (hq + 2 * hkv) * DIM)).to(torch.bfloat16) if c["bias"] else None,
         "q_norm": (1 + 0.1 * _randn(g, DIM)).to(torch.bfloat16) if c["norm"] else None,
         "k_norm": (1 + 0.1 * _randn(g, DIM)).to(torch.bfloat16) if c["norm"] else None}
    return s


def _prepare_attend(c, g):
    B, hq, hkv, S, page = c["batch"], c["heads"], c["kv_heads"], c["slots"], c["page"]
    if c["lens"] == "ragged":  # lengths over the whole range, with an empty one in a batch
        u = torch.rand(B, generator=g, device=DEV)
        lens = torch.exp(u * math.log(S + 1)).to(torch.int64).clamp(1, S)
        lens[0] = S
        if B > 2:
            lens[B // 2] = 0
    else:
        lens = torch.full((B,), S, dtype=torch.int64, device=DEV)
    table, pages = _tables(g, B, lens.clamp(min=1), page, 2)
    pool = torch.empty(pages, hkv, page // ROWS, BLOCK, dtype=torch.uint8, device=DEV)
    loud = 1 + 3 * (torch.rand(hkv, 1, DIM, generator=g, device=DEV) < 0.03).to(torch.float32)
    step = max(1, (1 << 20) // (hkv * page))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        pool[p:p + n] = _blocks(_randn(g, n, hkv, page, DIM) * loud, _randn(g, n, hkv, page, DIM))
    s = {"case": c, "pool": pool, "table": table, "lens": lens.to(torch.int32),
         "q": (1.5 * _randn(g, B, hq, DIM)).to(torch.bfloat16), "slot_pos": None, "score": None}
    if c["masked"]:  # a twentieth of the slots are free
        pos = torch.arange(S, device=DEV, dtype=torch.int32).repeat(B, 1)
        free = torch.rand(B, S, generator=g, device=DEV) < 0.05
        free[:, S // 2] = False
        s["slot_pos"] = torch.where(free, torch.full_like(pos, -1), pos)
    if c["score"]:
        s["score"] = torch.zeros(B, S, dtype=torch.float32, device=DEV)
    return s


def _prepare_int8(c, g):
    m, n, k = c["tokens"], c["out"], c["in"]
    x = _randn(g, m, k)
    x[:, torch.rand(k, generator=g, device=DEV) < 0.01] *= 8  # a few loud channels
    w = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=DEV)  # rows on 16-byte boundaries
    ws = torch.empty(n, dtype=torch.float32, device=DEV)
    for i in range(0, n, 4096):
        f = 0.02 * _randn(g, min(4096, n - i), k)
        ws[i:i + 4096] = f.abs().amax(1) / 127
        w[i:i + 4096, :k] = torch.round(f / ws[i:i + 4096, None]).clamp(-127, 127).to(torch.int8)
    return {"case": c, "x": x.to(torch.bfloat16), "w": w[:, :k], "w_scale": ws,
            "bias": (0.1 * _randn(g, n)).to(torch.bfloat16) if c["bias"] else None}


# ------------------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if own:
        from kvcacheboundaryprotection_b200 import lowbit

        if c["op"] == "append":
            q = lowbit.kv4_append(state["pool"], state["table"], state["qkv"], state["slots"], n_heads=c["heads"],
                                  seq=state["seq"], positions=state["positions"], inv_freq=state["inv_freq"],
                                  bias=state["bias"], q_norm=state["q_norm"], k_norm=state["k_norm"], eps=1e-6)
            k, v = lowbit.kv4_gather(state["pool"], state["table"], state["slots"], seq=state["seq"])
            return {"q": q, "k": k, "v": v}
        if c["op"] == "attend":
            out = lowbit.kv4_attend(state["pool"], state["table"], state["lens"], state["q"],
                                    slot_pos=state["slot_pos"], step_score=state["score"])
            return {"out": out} if state["score"] is None else {"out": out, "score": state["score"]}
        return lowbit.int8_linear(state["x"], state["w"], state["w_scale"], state["bias"],
                                  out_dtype=torch.float32 if c["f32"] else torch.bfloat16)
    if c["op"] == "append":
        return _plain_append(state)
    if c["op"] == "attend":
        return _plain_attend(state)
    return _plain_int8(state)


def _plain_append(s):
    """Bias, norm and rotation in 32 bits (the angles in 64: positions reach far), K and V
    into their blocks of the pool, and the rows read back as the values they stand for."""
    c = s["case"]
    hq, hkv, page = c["heads"], c["kv_heads"], c["page"]
    x = s["qkv"].to(torch.float32)
    if s["bias"] is not None:
        x = x + s["bias"].to(torch.float32)
    x = x.reshape(c["rows"], hq + 2 * hkv, DIM)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    if s["q_norm"] is not None:
        w = torch.cat([s["q_norm"].to(torch.float32).expand(hq, DIM), s["k_norm"].to(torch.float32).expand(hkv, DIM)])
        qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + 1e-6) * w
    ang = s["positions"].to(torch.float64)[:, None, None] * s["inv_freq"].to(torch.float64)
    co, si = torch.cos(ang).to(torch.float32), torch.sin(ang).to(torch.float32)
    a, b = qk[..., :64], qk[..., 64:]
    qk = torch.cat([a * co - b * si, b * co + a * si], -1)
    k = qk[:, hq:]
    slots = s["slots"].long()
    at = s["table"][s["seq"].long(), slots // page].long()
    row = slots % page
    blk, r = row // ROWS, row % ROWS
    byte = _bytes_of_slot(r)[:, None, :]
    here = (at[:, None, None], torch.arange(hkv, device=DEV)[None, :, None], blk[:, None, None], byte)
    s["pool"][here] = _row_bytes(k, v)
    k, v = _row_values(s["pool"][here])
    return {"q": qk[:, :hq].to(torch.bfloat16), "k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16)}


def _plain_attend(s):
    """softmax(q . k / sqrt(128)) v over each sequence's slots in 32 bits, and each slot's
    largest probability over the heads."""
    c = s["case"]
    B, hq, hkv, S, page = c["batch"], c["heads"], c["kv_heads"], c["slots"], c["page"]
    blocks = s["pool"][s["table"].clamp(min=0).long()]                     # [B, pages, hkv, page / 16, 2304]
    rows = blocks[..., _bytes_of_slot(torch.arange(ROWS, device=DEV)).reshape(-1)]
    k, v = _row_values(rows.transpose(1, 2).reshape(B, hkv, -1, BLOCK // ROWS)[:, :, :S])
    live = torch.arange(k.shape[2], device=DEV) < s["lens"][:, None]
    if s["slot_pos"] is not None:
        live = live & (s["slot_pos"] >= 0)
    live = live[:, None, None, :]
    q = s["q"].to(torch.float32).reshape(B, hkv, hq // hkv, DIM)
    l = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(DIM))
    l = torch.where(live, l, torch.full_like(l, -math.inf))
    top = l.amax(-1, keepdim=True)
    e = torch.where(live, torch.exp(l - torch.where(top > -math.inf, top, torch.zeros_like(top))), torch.zeros_like(l))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    out = {"out": torch.matmul(p, v).reshape(B, hq, DIM).to(torch.bfloat16)}
    if s["score"] is not None:
        out["score"] = torch.maximum(s["score"], p.amax((1, 2)))
    return out


def _plain_int8(s):
    """x rounded to 8 bits a token, the product of the whole numbers, the two scales."""
    c = s["case"]
    x = s["x"].to(torch.float32)
    top = x.abs().amax(1, keepdim=True)
    xs = _over(top, 127)
    # 127 x is exact, so half-way values (x = top / 2) are half-way in any precision
    xq = torch.round(127 * x / torch.where(top > 0, top, torch.ones_like(top))).clamp(-127, 127)
    y = torch.matmul(xq, s["w"].to(torch.float32).t()) * xs * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].to(torch.float32)
    return y if c["f32"] else y.to(torch.bfloat16)


# -------------------------------------------------------------------------- the work done
def _total_slots(c):
    """Slots that a pass reads: of a ragged batch the lengths' mean (they are drawn)."""
    if c["lens"] == "full":
        return c["batch"] * c["slots"]
    S, n = c["slots"], max(0, c["batch"] - (2 if c["batch"] > 2 else 1))
    return S + n * max(1.0, S / math.log(S + 1))


def work(case):
    c = case
    if c["op"] == "append":
        r, hq, hkv = c["rows"], c["heads"], c["kv_heads"]
        # qkv read, q written, K and V written in 4 bits, read back and written as bf16
        return {"bytes": r * 256 * (hq + 2 * hkv) + r * 256 * hq + 2 * r * hkv * 144 + r * hkv * 512 + 12 * r,
                "flops": 10 * r * 128 * (hq + 2 * hkv)}
    if c["op"] == "attend":
        n = _total_slots(c)
        extra = (4 * n if c["masked"] else 0) + (8 * n if c["score"] else 0)
        return {"bytes": n * c["kv_heads"] * 144 + extra + 4 * n / c["page"] + 512 * c["batch"] * c["heads"],
                "flops": 4 * n * c["heads"] * 128}
    m, n, k = c["tokens"], c["out"], c["in"]
    return {"bytes": n * k + 4 * n + 2 * m * k + (4 if c["f32"] else 2) * m * n + (2 * n if c["bias"] else 0),
            "flops": 2 * m * n * k}


# ---------------------------------------------------------------------- 64-bit definition
def _layout():
    """For K and V: byte and shift of (slot, dim), byte of (slot, group)'s scale."""
    slot, dim = np.meshgrid(np.arange(16), np.arange(128), indexing="ij")
    j, t, n = dim // 32, dim % 32 // 8, dim % 8
    k_byte, k_shift = 64 * slot + 4 * (4 * t + j) + n // 2, 4 * (n % 2)
    i, g, m = dim // 32, dim % 32 // 4, dim % 4
    st, sh, se = slot // 4, slot // 2 % 2, slot % 2
    v_byte, v_shift = 1024 + 512 * sh + 64 * g + 16 * st + 4 * i + 2 * se + m // 2, 4 * (m % 2)
    return (k_byte, k_shift, 1024 + 4 * slot + j), (v_byte, v_shift, 1024 + 64 + 16 * st + 8 * sh + 2 * i + se)


def _rows64(pool, page, slot):
    """K, V rows [n, hkv, 128] in 64 bits of the slots ``slot`` [n] of pages ``page`` [n]."""
    halves = pool.reshape(-1).view(torch.float16)
    hkv, per = pool.shape[1], pool.shape[2]
    base = ((page.long()[:, None] * hkv + torch.arange(hkv, device=pool.device)) * per + (slot // 16)[:, None]) * BLOCK
    out = []
    for byte, shift, scale in _layout():
        byte, shift, scale = (torch.from_numpy(a).to(pool.device) for a in (byte, shift, scale))
        r = slot % 16
        code = (pool.reshape(-1)[base[..., None] + byte[r][:, None]].long() >> shift[r][:, None]) & 15
        out.append((code - 8).double() * halves[base[..., None] // 2 + scale[r][:, None]].double())
    return out


def _quantised64(x):
    g = x.reshape(*x.shape[:-1], 4, 32)
    s = torch.minimum(g.abs().amax(-1, keepdim=True) / 7, torch.tensor(65504.0, dtype=torch.float64, device=x.device))
    s = s.to(torch.float16).double()
    return torch.where(s > 0, torch.round(g / s).clamp(-7, 7) * s, 0.0).reshape(x.shape)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "append":
        hq, hkv = c["heads"], c["kv_heads"]
        x = s["qkv"].double().reshape(c["rows"], -1, DIM)
        if s["bias"] is not None:
            x = x + s["bias"].double().reshape(-1, DIM)
        q, k, v = x.split([hq, hkv, hkv], 1)
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV),
                           s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]

        def finish(y, w):
            if w is not None:
                y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.double()
            z = torch.complex(y[..., :64].contiguous(), y[..., 64:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        return {"q": finish(q, s["q_norm"]), "k": _quantised64(finish(k, s["k_norm"])), "v": _quantised64(v)}
    if c["op"] == "attend":
        B, hq, hkv, page = c["batch"], c["heads"], c["kv_heads"], c["page"]
        out = torch.zeros(B, hq, DIM, dtype=torch.float64, device=DEV)
        score = None if s["score"] is None else s["score"].double()
        for b, n in enumerate(s["lens"].tolist()):
            at = torch.arange(n, device=DEV)
            if s["slot_pos"] is not None:
                at = at[s["slot_pos"][b, :n] >= 0]
            if not at.numel():
                continue
            k, v = _rows64(s["pool"], s["table"][b][at // page], at % page)
            q = s["q"][b].double().reshape(hkv, hq // hkv, DIM)
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(DIM), -1)
            out[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(hq, DIM)
            if score is not None:
                score[b, at] = torch.maximum(score[b, at], p.amax((0, 1)))
        return {"out": out} if score is None else {"out": out, "score": score}
    x = s["x"].double()
    most = x.abs().amax(1, keepdim=True)
    top, xq = most / 127, torch.where(most > 0, torch.round(x * 127 / most), 0.0)
    y = torch.empty(c["tokens"], c["out"], dtype=torch.float64, device=DEV)
    for i in range(0, c["out"], 8192):
        y[:, i:i + 8192] = (xq @ s["w"][i:i + 8192].double().t()) * top * s["w_scale"][i:i + 8192].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    return y
