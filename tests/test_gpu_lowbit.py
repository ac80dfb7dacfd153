"""The low-bit serving operators (include/kvbp.h, lowbit.py) against plain 64-bit statements
of the same formulas (tests/lowbit_ref.py), at the sizes and masks where they can go wrong.

Tolerances count roundings (they are derived beside each check); codes are held to the
definition: a stored value is the nearest multiple of its scale."""

import math

import numpy as np
import pytest
import torch

import lowbit_ref as ref
from kvcacheboundaryprotection_b200 import build, capi, lowbit

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _lib():
    build.build()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _table(g, need, n_pages, width):
    """Each sequence's pages (need[b] of them) drawn without repetition; -1 elsewhere."""
    perm = torch.randperm(n_pages, generator=g).tolist()
    t = torch.full((len(need), width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for j in range(n):
            t[b, j] = perm.pop()
    return t


# ------------------------------------------------------------------------------- append
def _append_case(rows, seqs, hq, hkv, page, bias, norm, rope, seed, far=300000):
    g = _gen(seed)
    seq = torch.sort(torch.randint(0, seqs, (rows,), generator=g))[0]
    slots = torch.zeros(rows, dtype=torch.int64)
    start = torch.randint(0, 40, (seqs,), generator=g)
    for b in range(seqs):
        at = (seq == b).nonzero().flatten()
        slots[at] = start[b] + torch.randperm(len(at), generator=g)
    width = int(slots.max()) // page + 2
    need = [int(slots[seq == b].max()) // page + 1 if (seq == b).any() else 0 for b in range(seqs)]
    n_pages = sum(need) + 2
    c = {
        "table": _table(g, need, n_pages, width), "seq": seq.to(torch.int32), "slots": slots.to(torch.int32),
        "qkv": torch.randn(rows, (hq + 2 * hkv) * 128, generator=g).to(BF),
        "positions": torch.randint(0, far, (rows,), generator=g, dtype=torch.int32) if rope else None,
        "inv_freq": (1e6 ** (-torch.arange(64) / 64.0)).float() if rope else None,
        "bias": torch.randn((hq + 2 * hkv) * 128, generator=g).to(BF) if bias else None,
        "q_norm": (1 + 0.2 * torch.randn(128, generator=g)).to(BF) if norm else None,
        "k_norm": (1 + 0.2 * torch.randn(128, generator=g)).to(BF) if norm else None,
        "pool": torch.randint(0, 256, (n_pages, hkv, page // 16, ref.BLOCK), generator=g, dtype=torch.uint8),
    }
    return c


def _on_gpu(c):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}


def _check_append(c, hq, hkv, q, pool_after, eps, stored):
    rows = c["qkv"].shape[0]
    x = c["qkv"].double()
    if c["bias"] is not None:
        x = x + c["bias"].double()
    x = x.reshape(rows, hq + 2 * hkv, 128)
    want_q = ref.finish(x[:, :hq], c["q_norm"], eps, c["positions"], c["inv_freq"])
    want_k = ref.finish(x[:, hq:hq + hkv], c["k_norm"], eps, c["positions"], c["inv_freq"])
    want_v = x[:, hq + hkv:]
    # fp32 work: a dozen roundings (2^-24 each) of values no larger than the row's largest,
    # then q's one rounding to bf16 (2^-8)
    top = want_q.abs().amax(-1, keepdim=True) if hq else None
    if hq:
        assert ((q.cpu().double() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -20 * top).all()
    page = c["pool"].shape[2] * 16
    pg = c["table"].long()[c["seq"].long(), c["slots"].long().clamp(min=0) // page]
    at = c["slots"].long().clamp(min=0) % page
    for (codes, scales), want in zip(ref.decode(pool_after), (want_k, want_v)):
        got_c, got_s = codes[pg, :, at][stored], scales[pg, :, at][stored]
        w = want[stored]
        s = (w.reshape(*w.shape[:-1], 4, 32).abs().amax(-1) / 7).clamp(max=65504.0)
        # f16's rounding (2^-11; 2^-25 absolute where subnormal) of an fp32 value
        assert ((got_s - s).abs() <= (2.0 ** -11 + 2.0 ** -20) * s + 2.0 ** -25).all()
        r = got_s.repeat_interleave(32, -1)
        assert (got_c >= 1).all() and (got_c <= 15).all()
        # nearest code of the stored scale: half a step, and the fp32 work's error; the ends may
        # miss by the scale's own rounding (7 * 2^-11 of a step), below half a step
        off = ((got_c - 8).double() * r - w).abs()
        assert (off <= r * 0.5 + 2.0 ** -20 * w.abs().amax(-1, keepdim=True) + (r == 0) * w.abs()).all()
    return pg, at


@pytest.mark.parametrize(
    "rows,seqs,hq,hkv,page,bias,norm,rope",
    [(1, 1, 4, 1, 16, False, False, False), (3, 2, 7, 1, 32, True, False, True), (5, 5, 8, 8, 16, False, True, True),
     (64, 3, 28, 4, 48, True, True, True), (33, 33, 32, 8, 64, False, True, True), (130, 1, 1, 1, 128, True, False, True),
     (17, 2, 0, 2, 16, False, False, False), (9, 4, 3, 3, 16, True, False, False)],
)
def test_append_stores_the_nearest_codes_and_touches_nothing_else(rows, seqs, hq, hkv, page, bias, norm, rope):
    c = _append_case(rows, seqs, hq, hkv, page, bias, norm, rope, 100 + rows)
    d = _on_gpu(c)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = lowbit.kv4_append(d["pool"], d["table"], d["qkv"], d["slots"], n_heads=hq, seq=d["seq"],
                          positions=d["positions"], inv_freq=d["inv_freq"], bias=d["bias"], q_norm=d["q_norm"],
                          k_norm=d["k_norm"], eps=1e-6, dev_err=err)
    assert int(err) == 0 and q.shape == (rows, hq, 128)
    after = d["pool"].cpu()
    pg, at = _check_append(c, hq, hkv, q, after, 1e-6, torch.ones(rows, dtype=torch.bool))
    # every byte of the other slots is as it was
    page_of = torch.zeros(c["pool"].shape[0], page, dtype=torch.bool)
    page_of[pg, at] = True
    for (old_c, old_s), (new_c, new_s) in zip(ref.decode(c["pool"]), ref.decode(after)):
        keep = ~page_of[:, None, :, None]
        assert torch.equal(old_c[keep.expand_as(old_c)], new_c[keep.expand_as(new_c)])
        a, b = old_s[keep.expand_as(old_s)], new_s[keep.expand_as(new_s)]
        assert torch.equal(torch.nan_to_num(a, nan=-1e9), torch.nan_to_num(b, nan=-1e9))
    # read-back: exactly bf16((code - 8) * scale)
    k, v = lowbit.kv4_gather(d["pool"], d["table"], d["slots"], seq=d["seq"], dev_err=err)
    k2, v2 = lowbit.kv4_gather(d["pool"], d["table"], d["slots"], seq=d["seq"], heads_first=True, dev_err=err)
    assert int(err) == 0
    for got, got2, want in zip((k, v), (k2, v2), ref.values(after)):
        assert torch.equal(got.cpu(), want[pg, :, at].float().to(BF))
        assert torch.equal(got2.transpose(0, 1), got)


def test_append_rows_per_sequence_skips_and_strided_rows():
    """Without seq the rows divide over the sequences; negative slots store nothing but give
    their q; qkv rows may be strided."""
    g = _gen(5)
    hq, hkv, page = 4, 2, 16
    wide = torch.randn(6, (hq + 2 * hkv) * 128 + 64, generator=g).to(BF)
    slots = torch.tensor([0, -1, 20, 3, -5, 17], dtype=torch.int32)
    table = torch.tensor([[4, 0], [2, 3]], dtype=torch.int32)
    pool = torch.zeros(6, hkv, 1, ref.BLOCK, dtype=torch.uint8)
    c = {"qkv": wide[:, :(hq + 2 * hkv) * 128].contiguous(), "bias": None, "q_norm": None, "k_norm": None,
         "positions": None, "inv_freq": None, "table": table, "seq": torch.tensor([0, 0, 0, 1, 1, 1], dtype=torch.int32),
         "slots": slots, "pool": pool}
    dp, err = pool.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    q = lowbit.kv4_append(dp, table.cuda(), wide.cuda()[:, :(hq + 2 * hkv) * 128], slots.cuda(), n_heads=hq, dev_err=err)
    assert int(err) == 0
    _check_append(c, hq, hkv, q, dp.cpu(), 1e-6, slots >= 0)
    k, v = lowbit.kv4_gather(dp, table.cuda(), slots.cuda())
    assert (k[[1, 4]] == 0).all() and (v[[1, 4]] == 0).all() and (k[0] != 0).any()


def test_append_rows_at_any_offset():
    """qkv, bias and norms off 16-byte boundaries give the bits of aligned ones; eight rows per
    CTA (many rows) those of one row per CTA."""
    g = _gen(6)
    hq, hkv, n = 3, 2, 2100
    cols = (hq + 2 * hkv) * 128
    wide = torch.randn(n, cols + 9, generator=g).to(BF).cuda()
    extra = torch.randn(cols + 300, generator=g).to(BF).cuda()
    freq = (1e4 ** (-torch.arange(64) / 64.0)).float().cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda") * 191
    seq = torch.zeros(n, dtype=torch.int32, device="cuda")
    slots = torch.randperm(n, generator=g).to(torch.int32).cuda()
    table = torch.randperm(140, generator=g).to(torch.int32)[None].cuda()
    got = []
    for off in (0, 1):
        pool = lowbit.kv4_pool(140, hkv, 16)
        qkv = wide[:, 1:1 + cols] if off else wide[:, 1:1 + cols].contiguous()
        bias, qn, kn = (extra[i + 1:i + 1 + m] for i, m in ((0, cols), (7, 128), (100, 128)))
        if not off:
            bias, qn, kn = bias.clone(), qn.clone(), kn.clone()
        kw = dict(n_heads=hq, inv_freq=freq, bias=bias, q_norm=qn, k_norm=kn)
        q = lowbit.kv4_append(pool, table, qkv, slots, seq=seq, positions=pos, **kw)
        got.append((q, pool))
        few = lowbit.kv4_pool(140, hkv, 16)
        for lo, hi in ((0, 900), (900, n)):
            part = lowbit.kv4_append(few, table, qkv[lo:hi], slots[lo:hi], seq=seq[lo:hi], positions=pos[lo:hi], **kw)
            assert torch.equal(part, q[lo:hi])
        assert torch.equal(few, pool)
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_append_the_same_row_twice_and_two_calls_on_two_streams():
    g = _gen(8)
    qkv = torch.randn(2, 6 * 128, generator=g).to(BF).cuda()
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    want = lowbit.kv4_pool(2, 2, 16)
    for b in range(2):
        lowbit.kv4_append(want, table[b:b + 1], qkv[b:b + 1], torch.tensor([5], dtype=torch.int32, device="cuda"), n_heads=2)
    twice = lowbit.kv4_pool(2, 2, 16)  # equal rows for one slot: that row
    seq = torch.tensor([0, 0, 1, 1], dtype=torch.int32, device="cuda")
    lowbit.kv4_append(twice, table, qkv.repeat_interleave(2, 0), torch.full((4,), 5, dtype=torch.int32, device="cuda"),
                      n_heads=2, seq=seq)
    assert torch.equal(twice, want)
    both = lowbit.kv4_pool(2, 2, 16)
    slot = torch.tensor([5], dtype=torch.int32, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for b in range(2):
        with torch.cuda.stream(streams[b]):
            lowbit.kv4_append(both, table[b:b + 1], qkv[b:b + 1], slot, n_heads=2)
    torch.cuda.synchronize()
    assert torch.equal(both, want)


def test_append_extreme_values():
    """Zero rows, values below and beyond the scale's range, infinities and NaN."""
    hq, hkv = 1, 1
    x = torch.zeros(7, 3 * 128)
    x[1, 128:256] = 1e-9           # below the smallest f16 scale: reads back as 0
    x[2, 128:256] = 3e6            # beyond 7 * 65504: saturates there
    x[3, 128 + 5] = math.inf
    x[3, 128 + 6] = -2.0
    x[4, 128 + 40] = math.nan      # group 1 of K only
    x[4, 128:160] = 3.5
    x[5, 256:] = -1e-6             # subnormal f16 scale
    x[6, 128:256] = torch.linspace(-7, 7, 128)
    d = x.to(BF).cuda()
    pool = torch.zeros(1, hkv, 1, ref.BLOCK, dtype=torch.uint8, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    slots = torch.arange(7, dtype=torch.int32, device="cuda")
    lowbit.kv4_append(pool, table, d, slots, n_heads=hq)
    k, v = (t[0, 0].float() for t in (ref.values(pool)))
    assert (k[0] == 0).all() and (v[0] == 0).all() and (k[1] == 0).all()
    assert (k[2] == 7 * 65504).all()
    assert k[3, 5] == 7 * 65504 and (k[3, 32:] == 0).all() and k[3, 6] == 0
    assert torch.isnan(k[4, 32:64]).all() and (k[4, :32] == 7 * float(torch.tensor(0.5).half())).all()
    assert (k[4, 64:] == 0).all() and (v[4] == 0).all()
    assert ((v[5] + 1e-6).abs() <= 7 * 2.0 ** -25 + 1e-8).all()
    assert ((k[6] - d[6, 128:256].float().cpu()).abs() <= 0.5 * (1 + 2.0 ** -11)).all()


def test_append_and_gather_out_of_range_slots_and_pages_are_skipped():
    hq, hkv, page = 2, 2, 16
    pool = torch.zeros(3, hkv, 1, ref.BLOCK, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[0, -1], [7, 2]], dtype=torch.int32, device="cuda")
    d = torch.ones(5, (hq + 2 * hkv) * 128, dtype=BF, device="cuda")
    seq = torch.tensor([0, 0, 1, 9, -1], dtype=torch.int32, device="cuda")
    slots = torch.tensor([16, 40, 3, 0, 0], dtype=torch.int32, device="cuda")  # no page, no entry, bad page, bad seqs
    for r in range(5):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        lowbit.kv4_append(pool, table, d[r:r + 1], slots[r:r + 1], n_heads=hq, seq=seq[r:r + 1].contiguous(), dev_err=err)
        assert int(err) == 4 and not pool.any(), r
        err.zero_()
        k, v = lowbit.kv4_gather(pool, table, slots[r:r + 1], seq=seq[r:r + 1].contiguous(), dev_err=err)
        assert int(err) == 4 and not k.any() and not v.any(), r
    lowbit.kv4_append(pool, table, d, slots, n_heads=hq, seq=seq)  # without a word to report to


# ------------------------------------------------------------------------------- attend
def _attend_case(lens, hq, hkv, page, masked, seed, loud=1.0, width=None, wide=False):
    """``wide``: a page table for more than 2048 slots, which the streaming kernel takes whatever
    the lengths; without it short sequences take the one-launch kernel."""
    g = _gen(seed)
    B = len(lens)
    need = [(n + page - 1) // page for n in lens]
    w = max(1, max(need)) + 1 if width is None else width
    w = max(w, 2100 // page + 2) if wide else w
    n_pages = sum(need) + 2
    k = torch.randn(n_pages, hkv, page, 128, generator=g).double()
    k[..., ::17] *= 6
    v = torch.randn(n_pages, hkv, page, 128, generator=g).double() * loud
    c = {"pool": ref.encode(k, v, n_pages), "table": _table(g, need, n_pages, w),
         "lens": torch.tensor(lens, dtype=torch.int32), "q": (2 * torch.randn(B, hq, 128, generator=g)).to(BF),
         "slot_pos": None}
    if masked:
        S = w * page - 3 if w * page - 3 >= max(lens) else w * page
        pos = torch.arange(S, dtype=torch.int32).repeat(B, 1)
        pos[torch.rand(B, S, generator=g) < 0.3] = -1
        c["slot_pos"] = pos
    return c


def _poison(c):
    """NaN scales and random codes in every slot no sequence may read: free ones, those past
    lens, and pages no table names."""
    page = c["pool"].shape[2] * 16
    live = torch.zeros(c["pool"].shape[0], page, dtype=torch.bool)
    for b, n in enumerate(c["lens"].tolist()):
        for s in range(n):
            if c["slot_pos"] is None or c["slot_pos"][b, s] >= 0:
                live[c["table"][b, s // page], s % page] = True
    p = c["pool"].numpy().copy()
    for (byte, shift), sc in ref.layout():
        for n, s in np.argwhere(~live.numpy()):
            p[n, :, s // 16, sc[s % 16]] = 0xFF
            p[n, :, s // 16, sc[s % 16] + 1] = 0x7F
    c["pool"] = torch.from_numpy(p)


def _check_attend(c, score=None, scale=None, dev_err_want=0):
    d = _on_gpu(c)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    s0 = None if score is None else score.clone()
    sc = None if score is None else score.cuda()
    out = lowbit.kv4_attend(d["pool"], d["table"], d["lens"], d["q"], slot_pos=d["slot_pos"], step_score=sc,
                            scale=scale, dev_err=err)
    torch.cuda.synchronize()
    assert int(err) == dev_err_want, capi.decode_dev_errors(int(err))
    want, p, bound, drel = ref.attend(c["pool"], c["table"], c["lens"], c["q"], c["slot_pos"],
                                      1 / math.sqrt(128) if scale is None else scale)
    off = (out.cpu().double() - want).abs()
    assert (off <= bound).all(), (off - bound).max()
    if sc is not None:
        p = p[:, :s0.shape[1]]
        w = torch.maximum(s0.double(), p)
        # fp32 probabilities: the logits' error (drel) and a few roundings
        assert ((sc.cpu().double() - w).abs() <= (drel[:, None] + 2.0 ** -20) * w + 2.0 ** -60).all()
    return out


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (6, 2), (4, 1), (28, 4), (8, 1), (32, 8), (5, 5)])
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("wide", [False, True])
def test_attend_lengths_around_every_edge(hq, hkv, page, wide):
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 100, 257, 0, 48, 7]
    _check_attend(_attend_case(lens, hq, hkv, page, False, hq * 100 + page, wide=wide))


@pytest.mark.parametrize("B,n", [(1, 2000), (3, 700), (20, 513), (150, 60), (300, 33), (2500, 5)])
def test_attend_short_forms_from_one_to_sixteen_warps_a_head(B, n):
    g = _gen(B)
    lens = torch.randint(0, n + 1, (B,), generator=g)
    lens[0] = n
    for masked in (False, True):
        c = _attend_case(lens.tolist(), 4, 1, 16, masked, B + n)
        if masked:
            c["slot_pos"][:, 0] = 1
            _check_attend(c, torch.rand(c["slot_pos"].shape, generator=g) * (torch.rand(c["slot_pos"].shape, generator=g) < 0.3))
        else:
            _check_attend(c)


@pytest.mark.parametrize("hq,hkv,page,lens", [(28, 4, 16, [1000, 1, 300]), (7, 1, 64, [2500]), (16, 2, 128, [700] * 9),
                                              (32, 8, 16, [64] * 40), (8, 8, 32, [0, 5, 4000])])
@pytest.mark.parametrize("wide", [False, True])
def test_attend_masked_with_score_and_poisoned_free_slots(hq, hkv, page, lens, wide):
    c = _attend_case(lens, hq, hkv, page, True, 7 + hq, wide=wide)
    for b, n in enumerate(lens):
        if n:
            c["slot_pos"][b, n // 2] = 5  # no sequence without a live slot here
    _poison(c)
    B, S = c["slot_pos"].shape
    score = torch.rand(B, S, generator=_gen(3)) * (torch.rand(B, S, generator=_gen(4)) < 0.5)
    _check_attend(c, score)
    _check_attend(c)
    c["slot_pos"] = None  # a score without a mask needs clean slots
    c["pool"] = _attend_case(lens, hq, hkv, page, False, 7 + hq, wide=wide)["pool"]
    _check_attend(c, torch.zeros(B, S))


@pytest.mark.parametrize("wide", [False, True])
def test_attend_sequences_without_a_live_slot_give_zeros(wide):
    c = _attend_case([40, 40, 0, 700], 8, 2, 16, True, 11, wide=wide)
    c["slot_pos"][0] = -1
    c["slot_pos"][3, :700] = -1
    _poison(c)
    score = torch.full(c["slot_pos"].shape, 0.25)
    out = _check_attend(c, score, dev_err_want=16)
    assert (out[[0, 2, 3]] == 0).all() and (out[1] != 0).any()


@pytest.mark.parametrize("wide", [False, True])
def test_attend_one_live_slot_returns_its_value(wide):
    c = _attend_case([300, 300], 4, 1, 16, True, 12, wide=wide)
    c["slot_pos"][:] = -1
    c["slot_pos"][0, 299] = 9
    c["slot_pos"][1, 0] = 0
    _poison(c)
    _check_attend(c, torch.zeros(c["slot_pos"].shape))


@pytest.mark.parametrize("loud", [1e-7, 1e-4, 3e4, 2e5])
@pytest.mark.parametrize("wide", [False, True])
def test_attend_value_magnitudes(loud, wide):
    """V scales from f16's subnormals to its top: the weights keep their precision."""
    _check_attend(_attend_case([600, 33], 4, 1, 32, False, 13, loud=loud, wide=wide))


def test_attend_mixed_magnitudes_rescale_the_running_sums():
    """V scales that grow along the sequence, and logits that do: every stage rescales."""
    c = _attend_case([3000], 8, 1, 64, False, 14)
    g = _gen(2)
    n = c["pool"].shape[0]
    k, v = torch.randn(n, 1, 64, 128, generator=g).double(), torch.randn(n, 1, 64, 128, generator=g).double()
    for j, p in enumerate(c["table"][0].tolist()):
        if p >= 0:
            v[p] *= 10.0 ** (j / 8 - 3)
            k[p] *= 0.2 + j / 20
    c["pool"] = ref.encode(k, v, n)
    _check_attend(c, torch.zeros(1, 3000))


@pytest.mark.parametrize("wide", [False, True])
def test_attend_nan_in_a_live_slot_reaches_only_its_sequence(wide):
    c = _attend_case([200, 200], 4, 2, 16, False, 15, wide=wide)
    p = c["pool"].numpy().copy()
    (_, ks), _ = ref.layout()
    p[c["table"][0, 3], 0, 0, ks[5, 2] + 1] = 0x7F  # slot 53 of head 0: a NaN K scale
    p[c["table"][0, 3], 0, 0, ks[5, 2]] = 0xFF
    out = lowbit.kv4_attend(torch.from_numpy(p).cuda(), c["table"].cuda(), c["lens"].cuda(), c["q"].cuda()).cpu()
    clean = lowbit.kv4_attend(c["pool"].cuda(), c["table"].cuda(), c["lens"].cuda(), c["q"].cuda()).cpu()
    assert torch.isnan(out[0, :2]).all()
    assert torch.equal(out[0, 2:], clean[0, 2:]) and torch.equal(out[1], clean[1])


@pytest.mark.parametrize("width", [7, 200])
def test_attend_bad_pages_and_lengths(width):
    c = _attend_case([100, 64], 4, 2, 16, False, 16, width=width)
    c["table"][0, 2] = 9999
    c["table"][1, 0] = -1
    _check_attend(c, dev_err_want=4)
    c = _attend_case([100, 64], 4, 2, 16, False, 17, width=width)
    d = _on_gpu(c)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    c["table"][0, :] = c["table"][0, :].clamp(min=0)
    long = torch.tensor([10 ** 6, -3], dtype=torch.int32, device="cuda")
    out = lowbit.kv4_attend(d["pool"], c["table"].cuda(), long, d["q"], dev_err=err)
    assert int(err) == 4
    c["lens"] = torch.tensor([16 * width, 0], dtype=torch.int32)  # as many slots as the table has
    want, _, bound, _ = ref.attend(c["pool"], c["table"], c["lens"], c["q"], None, 1 / math.sqrt(128))
    assert ((out.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("wide", [False, True])
def test_attend_scale_and_unusual_queries(wide):
    c = _attend_case([130, 20], 4, 2, 16, False, 18, wide=wide)
    c["q"][0, 0] = 0
    c["q"][0, 1] *= 1e-30
    c["q"][1, 2] = (c["q"][1, 2].float() * 1e-3).to(BF)
    _check_attend(c, scale=0.5)
    _check_attend(c, scale=-0.02)
    c["q"][1, 3, 4] = math.inf
    d = _on_gpu(c)
    out = lowbit.kv4_attend(d["pool"], d["table"], d["lens"], d["q"])
    assert torch.isnan(out[1, 3]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[1, :3]).all()


def test_attend_many_sequences_and_one_long():
    """More sequences than one launch takes, and one whose parts every CTA shares."""
    lens = [(37 * b) % 90 for b in range(1100)]
    _check_attend(_attend_case(lens, 2, 1, 16, False, 19, wide=True))
    _check_attend(_attend_case([3, 0, 5] * 30, 8, 8, 16, False, 23, wide=True))
    c = _attend_case([30011], 4, 1, 64, True, 20)
    _check_attend(c, torch.zeros(c["slot_pos"].shape))


def test_attend_offsets_past_32_bits():
    """Pages whose bytes lie beyond 2^31 and 2^32 of the pool."""
    hkv, page = 8, 128
    n_pages = (1 << 32) // (hkv * page // 16 * ref.BLOCK) + 40
    small = _attend_case([page * 3 + 5, 9], 16, hkv, page, False, 21, width=4)
    pool = torch.zeros(n_pages, hkv, page // 16, ref.BLOCK, dtype=torch.uint8, device="cuda")
    high = [n_pages - 1 - 3 * j for j in range(small["pool"].shape[0])]
    pool[torch.tensor(high, device="cuda")] = small["pool"].cuda()
    table = torch.where(small["table"] >= 0, torch.tensor(high, dtype=torch.int32)[small["table"].long()], -1).to(torch.int32)
    out = lowbit.kv4_attend(pool, table.cuda(), small["lens"].cuda(), small["q"].cuda())
    want, _, bound, _ = ref.attend(small["pool"], small["table"], small["lens"], small["q"], None, 1 / math.sqrt(128))
    assert ((out.cpu().double() - want).abs() <= bound).all()
    d = torch.randn(1, (16 + 2 * hkv) * 128, generator=_gen(1)).to(BF).cuda()
    slots = torch.tensor([page + 3], dtype=torch.int32, device="cuda")
    lowbit.kv4_append(pool, table[:1].cuda(), d, slots, n_heads=16)
    k, v = lowbit.kv4_gather(pool, table[:1].cuda(), slots)
    pg = pool[int(table[0, 1])][None].cpu()
    wk, wv = (x[0, :, 3].float().to(BF) for x in ref.values(pg))
    assert torch.equal(k[0].cpu(), wk) and torch.equal(v[0].cpu(), wv) and k.any()


@pytest.mark.parametrize("wide", [False, True])
def test_attend_only_empty_sequences(wide):
    c = _attend_case([0, 0, 0], 8, 2, 16, True, 24, wide=wide)
    score = torch.rand(c["slot_pos"].shape, generator=_gen(9))
    assert not _check_attend(c, score).any()


@pytest.mark.parametrize("wide", [False, True])
def test_attend_sequences_that_share_pages(wide):
    """A common prefix kept once: the tables of two sequences name the same pages."""
    c = _attend_case([100, 70, 33], 8, 2, 16, False, 25, wide=wide)
    c["table"][1, :4] = c["table"][0, :4]
    c["table"][2, :2] = c["table"][0, :2]
    _check_attend(c)


def test_attend_is_deterministic():
    c = _on_gpu(_attend_case([900, 3, 2000, 0, 77], 28, 4, 16, True, 22))
    s = [torch.zeros(c["slot_pos"].shape, device="cuda") for _ in range(3)]
    o = [lowbit.kv4_attend(c["pool"], c["table"], c["lens"], c["q"], slot_pos=c["slot_pos"], step_score=x) for x in s]
    assert all(torch.equal(o[0], x) for x in o) and all(torch.equal(s[0], x) for x in s)


# --------------------------------------------------------------------------------- int8
def _int8_case(M, N, K, seed, bias):
    g = _gen(seed)
    x = torch.randn(M, K, generator=g)
    x[:, ::97] *= 9
    w = 0.05 * torch.randn(N, K, generator=g)
    return x.to(BF), w.to(BF), (0.3 * torch.randn(N, generator=g)).to(BF) if bias else None


def _codes64(x):
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    return torch.where(top > 0, torch.round(x * 127 / top), torch.zeros_like(x)), (top / 127)[:, 0]


@pytest.mark.parametrize("rows,K", [(1, 1), (3, 7), (5, 128), (2, 3000), (7, 16385), (4, 20000), (300, 896)])
def test_quantize_rows(rows, K):
    x, _, _ = _int8_case(rows, 1, K, rows + K, False)
    x[0] = 0
    q, s = lowbit.int8_quantize_rows(x.cuda())
    want_q, want_s = _codes64(x)
    assert q.shape == (rows, K) and (q.stride(0) % 16 == 0 or rows == 1)
    assert torch.equal(q.cpu().double(), want_q)  # 127 x is exact: no value sits near a border by rounding
    assert ((s.cpu().double() - want_s).abs() <= 2.0 ** -24 * want_s).all()


def test_quantize_rows_strided_and_misaligned_input():
    x = torch.randn(9, 300, generator=_gen(1)).to(BF)
    for view in (x[:, 1:200], x[::2, 3:], x[:, :296]):
        q, s = lowbit.int8_quantize_rows(view.cuda() if view.is_contiguous() else x.cuda().as_strided(
            view.shape, view.stride(), view.storage_offset()))
        assert torch.equal(q.cpu().double(), _codes64(view)[0])


SIZES = [(1, 1, 1), (1, 129, 33), (1, 1000, 4001), (1, 260, 30720), (1, 129, 30721), (1, 38000, 3590), (2, 1000, 4001), (5, 300, 1000), (2, 100, 128), (16, 256, 512), (17, 300, 1000), (32, 640, 2048), (33, 129, 255),
         (64, 384, 384), (65, 1000, 900), (127, 129, 4097), (128, 128, 128), (130, 513, 640), (257, 700, 96),
         (300, 2560, 1024), (513, 257, 1281), (1000, 1153, 777), (4, 4608, 3584), (1, 20000, 256), (4500, 1153, 300), (300, 20000, 640), (700, 25700, 200)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dt", [BF, torch.float32])
def test_int8_linear(M, N, K, dt):
    bias = (M + N) % 2 == 0
    x, w, b = _int8_case(M, N, K, M + N + K, bias)
    wq, ws = lowbit.int8_quantize_rows(w.cuda())
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = lowbit.int8_linear(x.cuda(), wq, ws, None if b is None else b.cuda(), out_dtype=dt, dev_err=err)
    assert int(err) == 0 and y.dtype is dt and y.shape == (M, N)
    xq, xs = _codes64(x)
    wc, wsc = _codes64(w)
    want = (xq @ wc.t()) * xs[:, None] * wsc[None]
    # exact integer sums; scales (2^-24 each), their conversion and two products: six roundings
    tol = 6 * 2.0 ** -24 * want.abs()
    if b is not None:
        want = want + b.double()
        tol = tol + 2.0 ** -24 * want.abs()
    if dt is BF:
        tol = tol + 2.0 ** -8 * want.abs()
    assert ((y.cpu().double() - want).abs() <= tol * (1 + 2.0 ** -8) + 2.0 ** -140).all()


def test_int8_linear_rows_that_are_zero_or_not_finite():
    for rows, zero, nan, inf in ((40, 3, 7, 21), (4, 0, 1, 3)):
        x, w, b = _int8_case(rows, 200, 300, 5, True)
        x[zero] = 0
        x[nan, 11] = math.nan
        x[inf, 0] = -math.inf
        wq, ws = lowbit.int8_quantize_rows(w.cuda())
        y = lowbit.int8_linear(x.cuda(), wq, ws, b.cuda()).cpu()
        assert torch.equal(y[zero], b) and torch.isnan(y[nan]).all() and torch.isnan(y[inf]).all()
        rest = [r for r in range(rows) if r not in (nan, inf)]
        assert torch.isfinite(y[rest]).all()
        for r in range(4):  # a single row takes its own kernel
            alone = lowbit.int8_linear(x[r:r + 1].cuda(), wq, ws, b.cuda()).cpu()
            assert torch.equal(torch.nan_to_num(alone[0], nan=-1e4), torch.nan_to_num(y[r], nan=-1e4))


@pytest.mark.parametrize("M", [1, 4, 6])
def test_int8_linear_strided_and_misaligned_rows(M):
    """The one-token kernel and the two-kernel path take rows at any stride and offset."""
    x, w, b = _int8_case(2 * M, 300, 520, 8, True)
    wq, ws = lowbit.int8_quantize_rows(w.cuda())
    for rows, first, K in ((2, 0, 520), (1, 3, 501), (2, 1, 517), (1, 8, 512)):
        view = x.cuda()[::rows][:M, first:first + K]
        wv = lowbit.int8_quantize_rows(w[:, :K].contiguous().cuda())
        y = lowbit.int8_linear(view, *wv, b.cuda())
        assert torch.equal(y, lowbit.int8_linear(view.contiguous(), *wv, b.cuda()))
        q, s = lowbit.int8_quantize_rows(view)  # the same codes: exact sums, one rounding
        want = (q.double() @ wv[0].double().t()) * s.double()[:, None] * wv[1].double() + b.cuda().double()
        assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() * (1 + 2.0 ** -8) + 8 * 2.0 ** -24 * (want - b.cuda().double()).abs()).all()


def test_int8_linear_extreme_codes_do_not_overflow():
    K = 131071
    x = torch.full((2, K), -3.0, dtype=BF, device="cuda")
    w = torch.full((130, 131072), -128, dtype=torch.int8, device="cuda")[:, :K]
    ws = torch.ones(130, device="cuda")
    y = lowbit.int8_linear(x, w, ws, out_dtype=torch.float32)
    want = 127 * 128 * K * (3.0 / 127)
    assert ((y.double() - want).abs() <= 6 * 2.0 ** -24 * want).all()


def test_int8_linear_out_buffer_and_empty_batch():
    x, w, _ = _int8_case(0, 64, 128, 5, False)
    wq, ws = lowbit.int8_quantize_rows(w.cuda())
    assert lowbit.int8_linear(x.cuda(), wq, ws).shape == (0, 64)
    x, _, _ = _int8_case(3, 64, 128, 5, False)
    out = torch.empty(3, 64, dtype=BF, device="cuda")
    assert lowbit.int8_linear(x.cuda(), wq, ws, out=out) is out
    assert torch.equal(out, lowbit.int8_linear(x.cuda(), wq, ws))


@pytest.mark.parametrize("M,N,K", [(1, 260, 300), (7, 130, 640), (40, 300, 2048), (130, 1000, 1500), (2000, 5000, 200)])
@pytest.mark.parametrize("f32", [0, 1])
def test_product_entry_with_row_strides_leaves_the_gaps_alone(M, N, K, f32):
    """kvbp_int8_gemm from stored codes: the bits of int8_linear, into a wider output."""
    x, w, b = _int8_case(M, N, K, M + N, True)
    wq, ws = lowbit.int8_quantize_rows(w.cuda())
    xq, xs = lowbit.int8_quantize_rows(x.cuda())
    dt = torch.float32 if f32 else BF
    want = lowbit.int8_linear(x.cuda(), wq, ws, b.cuda(), out_dtype=dt)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for pad in (3, 8):
        out = torch.full((M, N + pad), 7.0, dtype=dt, device="cuda")
        bias = b.cuda()
        capi.check(capi.lib().kvbp_int8_gemm(torch.cuda.current_stream().cuda_stream, f32, M, N, K, wq.data_ptr(),
                                             max(wq.stride(0), (K + 15) // 16 * 16), ws.data_ptr(), xq.data_ptr(),
                                             max(xq.stride(0), (K + 15) // 16 * 16), xs.data_ptr(), bias.data_ptr(),
                                             out.data_ptr(), N + pad, err.data_ptr()), "int8_gemm")
        assert torch.equal(out[:, :N], want) and (out[:, N:] == 7).all() and int(err) == 0


@pytest.mark.parametrize("M,N,K", [(1, 512, 1024), (20, 512, 1024), (700, 14000, 256)])
def test_int8_linear_as_a_graph_and_on_two_streams_at_once(M, N, K):
    x, w, b = _int8_case(M, N, K, 3, True)
    wq, ws = lowbit.int8_quantize_rows(w.cuda())
    b = b.cuda()
    xs = [(x * f).to(BF).cuda() for f in (1.0, -2.5)]
    want = [lowbit.int8_linear(v, wq, ws, b) for v in xs]
    cur = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lowbit.int8_linear(cur, wq, ws, b)
    for v, y in zip(xs * 2, want * 2):
        cur.copy_(v)
        graph.replay()
        assert torch.equal(out, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(lowbit.int8_linear(xs[i], wq, ws, b))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_weight_quantised_right_before_its_product():
    """The product may fetch weights ahead of the token codes, but not ahead of the kernel that
    writes them: quantise and multiply back to back, many times, with changing weights."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for M in (1, 16):
        x = torch.randn(M, 2048, generator=g, device="cuda").to(BF)
        ws = [torch.randn(4096, 2048, generator=g, device="cuda").to(BF) for _ in range(2)]
        buf = torch.empty(4096, 2048, dtype=torch.int8, device="cuda")
        sc = torch.empty(4096, device="cuda")
        want = [lowbit.int8_linear(x, *lowbit.int8_quantize_rows(w)) for w in ws]
        torch.cuda.synchronize()
        L, got = capi.lib(), []
        for i in range(40):
            st = torch.cuda.current_stream().cuda_stream
            capi.check(L.kvbp_int8_quant_rows(st, 4096, 2048, ws[i % 2].data_ptr(), 2048, buf.data_ptr(), 2048,
                                              sc.data_ptr()), "quant")
            got.append(lowbit.int8_linear(x, buf, sc))
        assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))


# ------------------------------------------------------------------------------ together
def test_refusals_on_the_gpu():
    pool = lowbit.kv4_pool(2, 1, 16)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 9, 128, dtype=BF, device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        lowbit.kv4_attend(pool, table, lens, q)                    # a group of 9
    with pytest.raises(ValueError):
        lowbit.kv4_attend(pool, table, lens.cpu(), q[:, :4].contiguous())  # another device
    with pytest.raises(ValueError):
        lowbit.kv4_append(pool, table.long(), q.view(1, -1), lens, n_heads=7)
    x = torch.zeros(2, 17, dtype=BF, device="cuda")
    w, s = lowbit.int8_quantize_rows(torch.ones(32, 32, dtype=BF, device="cuda"))
    y = torch.ones(1, 32, dtype=BF, device="cuda")
    with pytest.raises(capi.KVBPError, match="overlap"):  # CTAs would read what others wrote
        lowbit.int8_linear(y, w, s, out=y)
    with pytest.raises(capi.KVBPError, match="overlap"):
        p = torch.zeros(1, 4, 128, dtype=BF, device="cuda")
        lowbit.kv4_attend(pool, table, lens, p, out=p)
    with pytest.raises(ValueError):  # weight rows off their 16-byte boundaries
        lowbit.int8_linear(x, torch.zeros(4, 17, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"))


def _layer(cache, table, lens, h, W, pos, hq):
    """q/k/v projection -> append -> attention -> o projection of one low-bit layer."""
    qkv = lowbit.int8_linear(h, *W["qkv"], W["b"])
    q = lowbit.kv4_append(cache, table, qkv, lens, n_heads=hq, positions=pos, inv_freq=W["inv_freq"])
    att = lowbit.kv4_attend(cache, table, lens + 1, q)
    return lowbit.int8_linear(att.view(att.shape[0], -1), *W["o"])


def _layer_setup(B, hidden, hq, hkv, page, width, seed):
    g = _gen(seed)
    W = {"qkv": lowbit.int8_quantize_rows((0.05 * torch.randn((hq + 2 * hkv) * 128, hidden, generator=g)).to(BF).cuda()),
         "o": lowbit.int8_quantize_rows((0.05 * torch.randn(hidden, hq * 128, generator=g)).to(BF).cuda()),
         "b": torch.randn((hq + 2 * hkv) * 128, generator=g).to(BF).cuda(),
         "inv_freq": (1e6 ** (-torch.arange(64) / 64.0)).float().cuda()}
    cache = lowbit.kv4_pool(B * width, hkv, page)
    table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width).cuda()
    return W, cache, table, g


def test_layer_steps_together_eager_and_as_a_graph():
    """Forty decode steps of one layer: each step's attention sees the rows the steps before
    appended; a captured step replayed gives the eager bits."""
    B, hidden, hq, hkv, page, width = 5, 512, 8, 2, 16, 4
    W, cache, table, g = _layer_setup(B, hidden, hq, hkv, page, width, 31)
    lens = torch.tensor([0, 3, 15, 16, 20], dtype=torch.int32, device="cuda")
    hs = (torch.randn(40, B, hidden, generator=g)).to(BF).cuda()
    eager, start = [], lens.clone()
    for t in range(40):
        n = start + t
        out = _layer(cache, table, n, hs[t], W, n, hq)
        eager.append(out)
        if t in (0, 17, 39):  # against the 64-bit statement of attention over the pool as it is
            qkv = lowbit.int8_linear(hs[t], *W["qkv"], W["b"])
            x = qkv.cpu().double().view(B, -1, 128)
            q = ref.finish(x[:, :hq], None, 0, n.cpu(), W["inv_freq"]).to(BF)
            att = lowbit.kv4_attend(cache, table, n + 1, q.cuda())
            want, _, bound, _ = ref.attend(cache.cpu(), table.cpu(), (n + 1).cpu(), q, None, 1 / math.sqrt(128))
            assert ((att.cpu().double() - want).abs() <= bound).all()
    cache2 = lowbit.kv4_pool(B * width, hkv, page)
    h, n = hs[0].clone(), start.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _layer(lowbit.kv4_pool(B * width, hkv, page), table, n, h, W, n, hq)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _layer(cache2, table, n, h, W, n, hq)
        n += 1
    for t in range(40):
        h.copy_(hs[t])
        graph.replay()
        assert torch.equal(out, eager[t]), t
    assert torch.equal(cache, cache2)


def test_two_graphs_on_two_streams_do_not_share_a_workspace():
    cases = [_on_gpu(_attend_case([4000, 100], 8, 2, 16, True, 40 + i)) for i in range(2)]
    want = [lowbit.kv4_attend(c["pool"], c["table"], c["lens"], c["q"], slot_pos=c["slot_pos"]) for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(lowbit.kv4_attend(c["pool"], c["table"], c["lens"], c["q"], slot_pos=c["slot_pos"]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(50):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_follow_the_current_stream():
    c = _on_gpu(_attend_case([500], 4, 1, 16, False, 50))
    want = lowbit.kv4_attend(c["pool"], c["table"], c["lens"], c["q"])
    s = torch.cuda.Stream()
    q = torch.zeros_like(c["q"])
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        q.copy_(c["q"])
        out = lowbit.kv4_attend(c["pool"], c["table"], c["lens"], q)
    s.synchronize()
    assert torch.equal(out, want)
