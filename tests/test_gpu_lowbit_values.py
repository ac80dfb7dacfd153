"""The low-bit serving operators over the whole range of their values: attention where some
groups of V are far louder than others or one slot outweighs the rest, stored codes beside NaN.

Bounds count roundings of the formulas, group by group, and are small against the values
themselves (asserted), whatever exponents a kernel chooses."""

import math

import pytest
import torch

import lowbit_ref as ref
from kvcacheboundaryprotection_b200 import build, capi, lowbit

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _lib():
    build.build()


# ------------------------------------------------------------------------------- attend
def _bound(pool, table, lens, q, slot_pos, scale):
    """(out, each slot's largest probability, bound on out's error, that of a probability) in
    float64.

    The output is rounded to bf16 (2^-8).  A slot's weight, and that times V's scale, are rounded
    to f16 (2^-11 each).  Where these are below f16's normals they are rounded to a fixed step
    instead: with weights held at 2^10 or more for the largest p of the slots and scales at 2^-5
    or more for the largest scale S of a group (its exponent's field 10 to 15 after a power of two of the group's
    own), the steps' halves, 2^-25, are 2^-30 S p_max at most, or 2^-49 p_max where S itself is
    subnormal (a scale moved up by 2^14 only), times a code of at most 7, and once more 2^-35 of p_max s for the
    weight alone.  Moving a scale down may round it too, by 2^-25 where S is moved below 1, so
    2^-24 S of a weight's code.  fp32 sums: n / 128 + 16 additions, cut at 2^-23 of sum p |v|.
    Logits: 2^-21 of the sum of their products' absolute values, an absolute error dl that is a
    relative one of 2 dl in every probability."""
    kv = ref.values(pool)
    (_, sk), (_, sv) = ref.decode(pool)
    B, hq, _ = q.shape
    hkv, page = pool.shape[1], pool.shape[2] * 16
    qd = q.cpu().double().reshape(B, hkv, hq // hkv, 128)
    out = torch.zeros_like(qd)
    bound, mass = torch.zeros_like(qd), torch.zeros_like(qd)
    score = torch.zeros(B, table.shape[1] * page, dtype=torch.float64)
    drel = torch.zeros(B, dtype=torch.float64)
    tb = table.cpu().long()
    for b, n in enumerate(lens.cpu().tolist()):
        at = torch.arange(n)
        if slot_pos is not None:
            at = at[slot_pos[b, :n].cpu() >= 0]
        if not len(at):
            continue
        pg = tb[b][at // page]
        k, v = (x[pg, :, at % page] for x in kv)
        s = sv[pg, :, at % page]                                       # [n, hkv, 4]
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", qd[b], k) * scale, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, v)
        mass[b] = torch.einsum("hgn,nhd->hgd", p, v.abs())
        big = 7 * torch.einsum("hgjd,nhj->hgn", qd[b].abs().reshape(hkv, -1, 4, 32), sk[pg, :, at % page])
        drel[b] = 2 * 2.0 ** -21 * abs(scale) * big.amax() + 2.0 ** -20
        top = p.amax(-1)[..., None]                                    # [hkv, heads of it, 1]
        most = s.amax(0).repeat_interleave(32, -1)[:, None]            # [hkv, 1, 128]
        step = 7 * (len(at) * top * ((2.0 ** -30 + 2.0 ** -35) * most + 2.0 ** -49) + 2.0 ** -24 * most)
        bound[b] = (2.0 ** -8 * out[b].abs() + step +
                    (2.0 ** -10 + 2.0 ** -21 + (len(at) / 128 + 16) * 2.0 ** -23 + 2 * drel[b]) * mass[b])
        score[b, at] = p.amax((0, 1))
        # all of it is small against the largest outputs of its own group of dims
        assert (bound[b] <= 2.0 ** -6 * mass[b].reshape(hkv, -1, 4, 32).amax(-1).repeat_interleave(32, -1)).all()
    return out.reshape(B, hq, 128), score, bound.reshape(B, hq, 128), drel, mass.reshape(B, hq, 128)


def _check(c, scored=False):
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    S = c["table"].shape[1] * c["pool"].shape[2] * 16
    got = torch.zeros(c["q"].shape[0], S, device="cuda") if scored else None
    out = lowbit.kv4_attend(d["pool"], d["table"], d["lens"], d["q"], step_score=got, dev_err=err)
    assert int(err) == 0, capi.decode_dev_errors(int(err))
    want, score, bound, drel, mass = _bound(c["pool"], c["table"], c["lens"], c["q"], None, 1 / math.sqrt(128))
    off = (out.cpu().double() - want).abs()
    assert (off <= bound).all(), ((off / bound).max(), off.max())
    if scored:
        assert ((got.cpu().double() - score).abs() <= (drel[:, None] + 2.0 ** -20) * score + 2.0 ** -60).all()
    return out, want, mass


# half-width of V's values, of each group of 32 dims
LOUD = {"one channel": (20.0, 0.3, 0.3, 0.3), "around 14": (5.0, 7.0, 0.4, 0.4), "far apart": (1e5, 0.3, 1e-3, 30.0),
        "all loud": (1e5, 9e4, 1.2e5, 1e5), "all quiet": (1e-3, 2e-3, 1e-4, 1e-3), "ordinary": (1.0, 1.0, 1.0, 1.0)}


def _pool(g, n, page, hkv, amps, gap, q0, one_channel):
    """n slots (whole pages) of hkv heads; a slot in the middle with almost no value whose logit
    lies ``gap`` nats above the others' (they are within a nat of each other)."""
    pages = (n + page - 1) // page
    k = 0.2 * torch.randn(pages * page, hkv, 128, generator=g).double()
    v = torch.randn(pages * page, hkv, 128, generator=g).double()
    amp = torch.tensor(amps, dtype=torch.float64).repeat_interleave(32)
    if one_channel:  # a single value of group 0 is loud, always to the same side
        amp[:32] = 0.3
    v *= amp
    if one_channel:
        v[..., 5] = amps[0] + 0.1 * v[..., 5]
    if gap:
        at = n // 2
        k[at] = q0 * (gap * math.sqrt(128) / q0.square().sum(-1, keepdim=True))
        v[at] *= 1e-4
    shape = (pages, page, hkv, 128)
    return ref.encode(k.view(shape).transpose(1, 2), v.view(shape).transpose(1, 2), pages)


def _case(n, hq, hkv, page, amps, gap, seed, width=None, seqs=1, one_channel=False):
    """``seqs`` sequences over the same pages (a page may be shared by readers), each its queries."""
    g = torch.Generator().manual_seed(seed)
    q0 = 2 * torch.randn(hkv, 128, generator=g).double()
    q = q0.repeat_interleave(hq // hkv, 0) + 0.1 * torch.randn(seqs, hq, 128, generator=g).double()
    pool = _pool(g, n, page, hkv, amps, gap, q0, one_channel)
    pages = pool.shape[0]
    table = torch.full((seqs, pages if width is None else max(pages, width)), -1, dtype=torch.int32)
    table[:, :pages] = torch.arange(pages - 1, -1, -1)
    pool = pool.flip(0).contiguous()
    return {"pool": pool, "table": table, "lens": torch.full((seqs,), n, dtype=torch.int32), "q": q.to(BF)}


@pytest.mark.parametrize("amps", LOUD)
@pytest.mark.parametrize("gap", [0.0, 9.0, 12.0])
@pytest.mark.parametrize("n,hq,hkv,page,width", [(512, 4, 1, 16, None), (1999, 7, 1, 64, None), (130, 4, 2, 16, 140),
                                                 (3001, 8, 2, 64, None), (20011, 4, 1, 64, None)])
def test_attend_loud_and_quiet_groups_of_values(amps, gap, n, hq, hkv, page, width):
    """Each group of 32 dims keeps its precision, whatever the other groups hold and however far
    one slot's weight lies above the rest: short and streaming forms."""
    c = _case(n, hq, hkv, page, LOUD[amps], gap, n + len(amps), width, one_channel=amps == "one channel")
    _check(c, scored=True)


@pytest.mark.parametrize("gap", [0.0, 9.0, 12.0])
def test_attend_loud_values_one_warp_a_head(gap):
    """Many sequences: one warp has all of a head's slots."""
    out, want, mass = _check(_case(512, 2, 1, 16, LOUD["around 14"], gap, 3, seqs=1200))
    # and without a lean to either side (the numerator and the sum of weights agree): bf16's
    # roundings of 128 dims, each off by 2^-9.3 on average squared, add up to 2^-12.8 of the whole
    lean = ((out.cpu().double() - want) * want.sign()).sum() / want.abs().sum()
    assert abs(lean) <= 2.0 ** -10


@pytest.mark.parametrize("width", [None, 200])
def test_attend_one_slot_with_far_scales_returns_its_row(width):
    """One live slot: its row comes back, each group within f16's and bf16's roundings."""
    amp = torch.tensor([3.8e-4, 2.86, 60000.0, 6e-6], dtype=torch.float64).repeat_interleave(32) * 7
    v = (amp * torch.linspace(-1, 1, 32).double().repeat(4)).view(1, 1, 1, 128).expand(1, 1, 16, 128)
    pool = ref.encode(torch.zeros_like(v), v, 1)
    table = torch.zeros(1, 1 if width is None else width, dtype=torch.int32)
    c = {"pool": pool, "table": table, "lens": torch.tensor([1], dtype=torch.int32), "q": torch.ones(1, 3, 128, dtype=BF)}
    out, want, _ = _check(c)
    row = ref.values(pool)[1][0, 0, 0]
    assert ((out.cpu().double()[0] - row).abs() <= (2.0 ** -8 + 2.0 ** -10) * row.abs()).all()


@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("n,width", [(1900, None), (6000, None), (500, 200)])
def test_attend_values_that_grow_or_fall_along_the_sequence(up, n, width):
    """V from 1e-3 to 1e5, group by group at other places, and logits that grow: the running sums
    are rescaled again and again."""
    g = torch.Generator().manual_seed(n)
    c = _case(n, 8, 1, 16, LOUD["ordinary"], 0.0, n, width)
    pages = (n + 15) // 16
    v = torch.randn(pages, 1, 16, 128, generator=g).double()
    k = torch.randn(pages, 1, 16, 128, generator=g).double() * (torch.arange(pages) / pages).view(-1, 1, 1, 1)
    for j in range(4):
        v[..., 32 * j:32 * j + 32] *= 10.0 ** (8 * torch.arange(pages) / pages - 3 - j).view(-1, 1, 1, 1)
    if not up:
        k, v = k.flip(0), v.flip(0)
    c["pool"] = ref.encode(k, v, pages).flip(0).contiguous()
    _check(c, scored=True)


@pytest.mark.parametrize("width", [None, 200])
def test_attend_nan_in_one_group_of_values_leaves_the_others(width):
    c = _case(300, 4, 1, 16, LOUD["around 14"], 9.0, 8, width)
    clean = lowbit.kv4_attend(c["pool"].cuda(), c["table"].cuda(), c["lens"].cuda(), c["q"].cuda()).cpu()
    p = c["pool"].numpy().copy()
    _, (_, vs) = ref.layout()
    p[c["table"][0, 5], 0, 0, vs[3, 1]:vs[3, 1] + 2] = (0xFF, 0x7F)  # slot 83, group 1: a NaN scale
    out = lowbit.kv4_attend(torch.from_numpy(p).cuda(), c["table"].cuda(), c["lens"].cuda(), c["q"].cuda()).cpu()
    assert torch.isnan(out[..., 32:64]).all()
    keep = torch.ones(128, dtype=torch.bool)
    keep[32:64] = False
    assert torch.equal(out[..., keep], clean[..., keep])


@pytest.mark.parametrize("width", [None, 200])
@pytest.mark.parametrize("e", range(20, 33))
def test_attend_logits_beyond_float32s_whole_numbers(e, width):
    """Equal logits of 2^e: the mean of the slots that have them, where their neighbours in
    float32 lie 2^(e - 23) apart."""
    n, page, hkv, hq = 150, 16, 1, 5
    g = torch.Generator().manual_seed(e)
    v = torch.randn(10, hkv, page, 128, generator=g).double()
    for mantissa in (1.0, 1.37, 1.9):
        k = torch.full((10, hkv, page, 128), 7.0, dtype=torch.float64)
        k[:, :, 1::2] = -7.0
        k[:4] *= 0.5  # the largest logit comes after some stages
        q = torch.full((1, hq, 128), 2.0 ** (e - 10), dtype=torch.float64).to(BF)
        c = {"pool": ref.encode(k, v, 10), "table": torch.arange(10, dtype=torch.int32)[None], "q": q,
             "lens": torch.tensor([n], dtype=torch.int32)}
        if width:
            c["table"] = torch.nn.functional.pad(c["table"], (0, width - 10), value=-1)
        d = {a: b.cuda() for a, b in c.items()}
        scale = mantissa * 2.0 ** 10 / (7 * 128) / math.log2(math.e)  # q . k scale log2(e) = mantissa 2^e
        out = lowbit.kv4_attend(d["pool"], d["table"], d["lens"], d["q"], scale=scale).cpu().double()[0]
        rows = ref.values(c["pool"])[1][:, 0].reshape(-1, 128)[64:n:2]
        want, mass = rows.mean(0), rows.abs().mean(0)
        # bf16's rounding of the output, f16's of the weights and their products with the scales
        assert ((out - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -10 + 2.0 ** -16) * mass).all(), (e, mantissa)


# ------------------------------------------------------------------------------- append
def test_append_groups_without_a_scale_get_code_eight():
    """Groups whose scale is NaN or rounds to 0 hold code 8 throughout, infinities and ordinary
    values beside the NaN among them; their neighbours hold their own codes."""
    x = torch.zeros(6, 3 * 128)
    x[:, 128:] = torch.linspace(-7, 7, 32).repeat(8)
    for row, (at, value) in enumerate([(128 + 40, math.nan), (256 + 99, math.nan), (128 + 5, -math.nan)]):
        x[row, at] = value
    x[1, 256 + 98], x[1, 256 + 97] = math.inf, -math.inf
    x[3, 128:160] = 1e-9
    x[3, 384 - 32:] = -1e-30
    x[4, 256 + 33] = math.inf
    pool = torch.full((1, 1, 1, ref.BLOCK), 0xA5, dtype=torch.uint8, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    d = x.to(BF)
    lowbit.kv4_append(pool, table, d.cuda(), torch.arange(6, dtype=torch.int32, device="cuda"), n_heads=1)
    for part, ((codes, scales), first) in enumerate(zip(ref.decode(pool), (128, 256))):
        c, s = codes[0, 0, :6].reshape(6, 4, 32), scales[0, 0, :6]
        v = d[:, first:first + 128].double().reshape(6, 4, 32)
        empty = s.isnan() | (s == 0)
        want_empty = torch.zeros(6, 4, dtype=torch.bool)
        for row, group in {0: [(0, 1), (2, 0), (3, 0)], 1: [(1, 3), (3, 3)]}[part]:
            want_empty[row, group] = True
        assert torch.equal(empty, want_empty) and (c[empty] == 8).all()
        plain = torch.round(v / s[..., None]).clamp(-7, 7) + 8
        assert torch.equal(c[~empty].double(), plain[~empty])


# --------------------------------------------------------------------------------- int8
TOPS = [9.2e-41, 1e-38, 1.3e-37, 3.5e-37, 4e-37, 1e-30, 1.0, 2.6e36, 2.8e36, 1e37, 1e38, 3.3e38]


def _rows(K, seed):
    """A bf16 row of each largest value in TOPS, half-way values (top / 2 and so on) among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(len(TOPS), K, generator=g).double() * 2 - 1
    x[:, :: 7] = 0.5
    x[:, 3 % K] = -1.0
    x = (x * torch.tensor(TOPS, dtype=torch.float64)[:, None]).to(BF)
    assert torch.isfinite(x).all()
    return x


def _codes64(x):
    """Codes and scales of the definition; bf16 values and 127 times them are exact in float64."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    return torch.round(127 * x / top), (top / 127)[:, 0]


@pytest.mark.parametrize("K", [5, 300, 1000, 1003, 2500, 4096, 4099, 9000, 9007, 17000, 17001])
@pytest.mark.parametrize("first", [0, 1])
def test_quantize_rows_at_the_ends_of_the_range(K, first):
    """Vector loads, tails, misaligned rows, short and long rows."""
    x = _rows(K, K)
    wide = torch.zeros(len(TOPS), K + 16, dtype=BF)
    wide[:, first:first + K] = x
    q, s = lowbit.int8_quantize_rows(wide.cuda()[:, first:first + K])
    want_q, want_s = _codes64(x)
    assert torch.equal(q.cpu().double(), want_q)
    # the quotient's rounding: 2^-24, or half of the smallest subnormal
    assert ((s.cpu().double() - want_s).abs() <= 2.0 ** -24 * want_s + 2.0 ** -150).all()


@pytest.mark.parametrize("K", [300, 1003, 2048])
def test_int8_linear_codes_at_the_ends_of_the_range(K):
    """An identity weight gives the codes back, in the one-token kernel and the others."""
    x = _rows(K, K + 1).cuda()
    w = torch.zeros(K, (K + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :K]
    w.fill_diagonal_(1)
    want, scale = _codes64(x.cpu())
    sw = torch.ones(K, device="cuda")
    for y in (lowbit.int8_linear(x, w, sw, out_dtype=torch.float32),
              torch.cat([lowbit.int8_linear(x[r:r + 1], w, sw, out_dtype=torch.float32) for r in range(len(TOPS))])):
        v = want * scale[:, None]
        assert ((y.cpu().double() - v).abs() <= 2.0 ** -23 * v.abs() + 2.0 ** -149 * want.abs()).all()


@pytest.mark.parametrize("M", [1, 12, 40, 100, 300, 5000])
@pytest.mark.parametrize("dt", [BF, torch.float32])
def test_int8_linear_outputs_at_the_ends_of_the_range(M, dt):
    """Finite outputs of tokens near bf16's largest value, and of its smallest: sum * x_scale alone
    would overflow.  One token, split tiles of every width, and the persistent form (5000)."""
    K, N = 640, 1100
    g = torch.Generator().manual_seed(M)
    tops = torch.tensor([3e38, 1.0, 2e37, 1e-30, 1e36, 1e-36, 3e22])[torch.arange(M) % 7].double()
    x = ((torch.rand(M, K, generator=g).double() * 2 - 1) * tops[:, None]).to(BF)
    w = (1e-3 * torch.randn(N, K, generator=g)).to(BF)
    wq, ws = lowbit.int8_quantize_rows(w.cuda())
    y = lowbit.int8_linear(x.cuda(), wq, ws, out_dtype=dt).cpu().double()
    xq, xs = _codes64(x)
    want = (xq @ wq.cpu().double().t()) * xs[:, None] * ws.cpu().double()
    assert (want.abs().amax(1) / tops).amin() > 1e-4 and want.abs().max() < 3e38
    # the token's scale, the sum's conversion, two products, and bf16's rounding
    tol = (5 * 2.0 ** -24 + (2.0 ** -8 if dt is BF else 0)) * want.abs()
    assert ((y - want).abs() <= tol * (1 + 2.0 ** -8) + 2.0 ** -132).all()
