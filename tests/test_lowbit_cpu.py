"""Refusals and host arithmetic of the low-bit operators, without a GPU: the C entry points
check every argument before their first CUDA call, the Python ones before they launch."""

import pytest
import torch

from kvcacheboundaryprotection_b200 import build, capi, lowbit

import lowbit_ref as ref

BF = torch.bfloat16
A = 1 << 20  # an aligned address that is never read


@pytest.fixture(scope="module")
def L():
    build.build()
    return capi.lib()


def _append(L, **kw):
    a = dict(rows=2, per=1, seq=A, B=2, Hq=4, Hkv=2, D=128, page=16, pages=4, width=2, qkv=A, ldq=1024, bias=None,
             qn=None, kn=None, eps=1e-6, freq=None, pos=None, slots=A, table=A, q=A + 65536, pool=A, err=None)
    a.update(kw)
    return L.kvbp_kv4_append(None, *a.values())


def _gather(L, **kw):
    a = dict(rows=2, per=1, seq=A, B=2, Hkv=2, D=128, page=16, pages=4, width=2, slots=A, table=A, pool=A, k=A, v=A,
             rs=256, hs=128, err=None)
    a.update(kw)
    return L.kvbp_kv4_gather(None, *a.values())


def _attn(L, **kw):
    a = dict(B=2, Hq=4, Hkv=2, D=128, page=16, pages=4, width=2, q=A, pool=A, table=A, lens=A, pos=None, S=0, scale=0.1,
             out=A + 65536, score=None, ws=A, wsb=1 << 30, err=None)
    a.update(kw)
    return L.kvbp_kv4_attn(None, *a.values())


@pytest.mark.parametrize("call", [_append, _gather, _attn])
@pytest.mark.parametrize(
    "bad,status",
    [(dict(pool=None), 1), (dict(table=None), 1), (dict(D=64), 2), (dict(page=24), 1), (dict(page=0), 1),
     (dict(B=0), 1), (dict(Hkv=0), 1), (dict(pages=0), 1), (dict(width=0), 1), (dict(pool=A + 8), 1),
     (dict(page=65536, width=65536), 1)],
)
def test_pool_refusals(L, call, bad, status):
    assert call(L, **bad) == status and L.kvbp_last_error().startswith(b"kv4_")


@pytest.mark.parametrize(
    "bad", [dict(rows=0), dict(rows=-1), dict(qkv=None), dict(slots=None), dict(q=None), dict(freq=A), dict(ldq=1000),
            dict(seq=None, per=0), dict(Hq=-1), dict(q=A + 65544), dict(q=A), dict(q=A + 2048)])
def test_append_refusals(L, bad):
    assert _append(L, **bad) == 1


@pytest.mark.parametrize("bad", [dict(rows=0), dict(slots=None), dict(k=None), dict(v=None), dict(rs=100), dict(hs=132),
                                 dict(k=A + 8), dict(seq=None, per=0)])
def test_gather_refusals(L, bad):
    assert _gather(L, **bad) == 1


@pytest.mark.parametrize(
    "bad,status",
    [(dict(q=None), 1), (dict(lens=None), 1), (dict(out=None), 1), (dict(ws=None, width=1000), 1), (dict(wsb=100, width=1000), 1), (dict(Hq=5), 1), (dict(Hq=0), 1),
     (dict(Hq=18), 2), (dict(Hq=8192, Hkv=1024), 2), (dict(pos=A), 1), (dict(score=A), 1), (dict(S=-1), 1),
     (dict(q=A + 8), 1), (dict(out=A + 65544), 1), (dict(out=A), 1), (dict(ws=A + 4, width=1000), 1)],
)
def test_attention_refusals(L, bad, status):
    assert _attn(L, **bad) == status


def test_attention_workspace(L):
    assert L.kvbp_kv4_attn_workspace(2, 4, 2, 2048, 1) == 0  # short sequences: one launch, none needed
    plain = L.kvbp_kv4_attn_workspace(2, 4, 2, 2049, 0)
    assert plain > 0 and plain == L.kvbp_kv4_attn_workspace(100, 32, 8, 100000, 0)  # no score: whatever the size
    scored = L.kvbp_kv4_attn_workspace(2, 4, 2, 2050, 1)
    assert scored - plain == 2 * 2 * 64 + 2 * 2 * 2064 * 2 * 4  # (ref, sum) and the logits of 2064 slots, 2 heads each
    assert L.kvbp_kv4_attn_workspace(0, 4, 2, 100, 1) == 0


def _gemm(L, **kw):
    a = dict(f32=0, M=2, N=64, K=32, w=A, ldw=32, ws=A, xq=A, ldq=32, xs=A, bias=None, out=A + 65536, ldo=64, err=None)
    a.update(kw)
    return L.kvbp_int8_gemm(None, *a.values())


@pytest.mark.parametrize(
    "bad,status",
    [(dict(w=None), 1), (dict(ws=None), 1), (dict(xq=None), 1), (dict(xs=None), 1), (dict(out=None), 1), (dict(M=0), 1),
     (dict(N=0), 1), (dict(K=0), 1), (dict(K=33), 1), (dict(ldw=40, K=32), 1), (dict(ldq=40), 1), (dict(ldo=60), 1),
     (dict(w=A + 8), 1), (dict(xq=A + 8), 1), (dict(out=A + 65537), 1), (dict(f32=1, out=A + 65538), 1),
     (dict(K=131072, ldw=131072, ldq=131072), 2), (dict(M=0x7fffffff), 2), (dict(N=65536 * 128, ldo=65536 * 128), 2),
     (dict(out=A), 1), (dict(w=A + 65536 + 64, out=A + 65536), 1)],
)
def test_product_refusals(L, bad, status):
    assert _gemm(L, **bad) == status


def test_linear_and_quantisation_refusals(L):
    assert L.kvbp_int8_quant_rows(None, 0, 8, A, 8, A, 16, A) == 1
    assert L.kvbp_int8_quant_rows(None, 2, 8, A, 7, A, 16, A) == 1
    assert L.kvbp_int8_quant_rows(None, 2, 8, A, 8, A, 8, A) == 1   # q rows off 16-byte boundaries
    assert L.kvbp_int8_quant_rows(None, 2, 8, A, 8, A + 4, 16, A) == 1
    assert L.kvbp_int8_quant_rows(None, 2, 8, None, 8, A, 16, A) == 1
    need = L.kvbp_int8_linear_workspace(5, 100)
    assert need == 5 * 112 + 20 and L.kvbp_int8_linear_workspace(1, 100) == 0
    lin = lambda ws, n, M=5, x=A, out=A + 65536: L.kvbp_int8_linear(  # noqa: E731
        None, 0, M, 64, 100, A, 112, A, x, 100, None, out, 64, ws, n, None)
    assert lin(None, need) == 1 and lin(A, need - 1) == 1 and lin(A + 8, need) == 1
    assert lin(None, 0, M=1, x=None) == 1
    for M in (1, 5):
        assert lin(A + 131072, need, M=M, x=A + 65536) == 1 and b"overlap x" in L.kvbp_last_error()
        assert lin(A + 131072, need, M=M, out=A + 64) == 1 and b"overlap w" in L.kvbp_last_error()


# ---------------------------------------------------------------- the Python entry points
def _kv(hq=4, hkv=2):
    pool = torch.zeros(4, hkv, 1, 2304, dtype=torch.uint8)
    table = torch.zeros(2, 2, dtype=torch.int32)
    qkv = torch.zeros(2, (hq + 2 * hkv) * 128, dtype=BF)
    slots = torch.zeros(2, dtype=torch.int32)
    return pool, table, qkv, slots


def test_python_refuses_cpu_tensors_last():
    """A call whose arguments all fit gets as far as the device check."""
    pool, table, qkv, slots = _kv()
    build.build()
    for call in (lambda: lowbit.kv4_append(pool, table, qkv, slots, n_heads=4),
                 lambda: lowbit.kv4_gather(pool, table, slots),
                 lambda: lowbit.kv4_attend(pool, table, slots, torch.zeros(2, 4, 128, dtype=BF)),
                 lambda: lowbit.int8_quantize_rows(torch.zeros(2, 8, dtype=BF)),
                 lambda: lowbit.int8_linear(torch.zeros(2, 16, dtype=BF), torch.zeros(3, 16, dtype=torch.int8), torch.ones(3))):
        with pytest.raises(ValueError, match="CUDA devices only"):
            call()


def test_python_append_refusals():
    pool, table, qkv, slots = _kv()
    f = torch.zeros(64)
    with pytest.raises(ValueError, match="columns"):
        lowbit.kv4_append(pool, table, qkv, slots, n_heads=5)
    with pytest.raises(ValueError, match="go together"):
        lowbit.kv4_append(pool, table, qkv, slots, n_heads=4, inv_freq=f)
    with pytest.raises(ValueError, match="inv_freq"):
        lowbit.kv4_append(pool, table, qkv, slots, n_heads=4, inv_freq=f[:63], positions=slots)
    with pytest.raises(ValueError, match="slots"):
        lowbit.kv4_append(pool, table, qkv, slots.long(), n_heads=4)
    with pytest.raises(ValueError, match="slots"):
        lowbit.kv4_append(pool, table, qkv, slots[:1], n_heads=4)
    with pytest.raises(ValueError, match="pool"):
        lowbit.kv4_append(pool[..., :2303], table, qkv, slots, n_heads=4)
    with pytest.raises(ValueError, match="page_table"):
        lowbit.kv4_append(pool, table.t(), qkv, slots, n_heads=4)
    with pytest.raises(ValueError, match="page_table"):
        lowbit.kv4_append(pool, table[0], qkv, slots, n_heads=4)
    with pytest.raises(ValueError, match="bfloat16"):
        lowbit.kv4_append(pool, table, qkv.float(), slots, n_heads=4)
    with pytest.raises(ValueError, match="contiguous"):
        lowbit.kv4_append(pool, table, qkv.t().contiguous().t(), slots, n_heads=4)
    with pytest.raises(ValueError, match="pass seq"):
        lowbit.kv4_append(pool, table, qkv[:1], slots[:1], n_heads=4)
    with pytest.raises(ValueError, match="bias"):
        lowbit.kv4_append(pool, table, qkv, slots, n_heads=4, bias=qkv[0, :-1].contiguous())
    with pytest.raises(ValueError, match="k_norm"):
        lowbit.kv4_append(pool, table, qkv, slots, n_heads=4, k_norm=torch.ones(128))
    with pytest.raises(ValueError, match="q_out"):
        lowbit.kv4_append(pool, table, qkv, slots, n_heads=4, q_out=torch.zeros(2, 3, 128, dtype=BF))
    with pytest.raises(ValueError, match="empty"):
        lowbit.kv4_append(pool, torch.zeros(2, 0, dtype=torch.int32), qkv, slots, n_heads=4)


def test_python_attend_and_pool_refusals():
    pool, table, _, lens = _kv()
    q = torch.zeros(2, 4, 128, dtype=BF)
    with pytest.raises(ValueError, match="whole groups"):
        lowbit.kv4_attend(pool, table, lens, torch.zeros(2, 3, 128, dtype=BF))
    with pytest.raises(ValueError, match="whole groups"):
        lowbit.kv4_attend(pool, table, lens, torch.zeros(2, 18, 128, dtype=BF))
    with pytest.raises(ValueError, match="q must"):
        lowbit.kv4_attend(pool, table, lens, q[:, :, :64])
    with pytest.raises(ValueError, match="lens"):
        lowbit.kv4_attend(pool, table, lens[:1], q)
    with pytest.raises(ValueError, match="slot_pos"):
        lowbit.kv4_attend(pool, table, lens, q, slot_pos=torch.zeros(2, 8))
    with pytest.raises(ValueError, match="step_score"):
        lowbit.kv4_attend(pool, table, lens, q, slot_pos=torch.zeros(2, 8, dtype=torch.int32), step_score=torch.zeros(2, 9))
    with pytest.raises(ValueError, match="out"):
        lowbit.kv4_attend(pool, table, lens, q, out=torch.zeros(2, 4, 128))
    with pytest.raises(ValueError, match="dev_err"):
        lowbit.kv4_attend(pool, table, lens, q, dev_err=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="multiple of 16"):
        lowbit.kv4_pool(4, 2, 24, device="cpu")
    with pytest.raises(ValueError):
        lowbit.kv4_pool(0, 2, 16, device="cpu")
    assert lowbit.kv4_pool(3, 2, 48, device="cpu").shape == (3, 2, 3, 2304)
    with pytest.raises(ValueError, match="slots"):
        lowbit.kv4_gather(pool, table, torch.zeros(2, 1, dtype=torch.int32))


def test_python_linear_refusals():
    x, w, s = torch.zeros(2, 16, dtype=BF), torch.zeros(3, 16, dtype=torch.int8), torch.ones(3)
    for bad in (dict(x=x.float()), dict(x=x[0]), dict(w=w.float()), dict(w=torch.zeros(3, 32, dtype=torch.int8)),
                dict(w=torch.zeros(3, 17, dtype=torch.int8)[:, :16]), dict(s=s[:2]), dict(s=s.double()),
                dict(x=x.t().contiguous().t()), dict(x=x[:1].expand(2, 16))):
        a = dict(x=x, w=w, s=s)
        a.update(bad)
        with pytest.raises(ValueError, match=r"must|columns|rows"):
            lowbit.int8_linear(a["x"], a["w"], a["s"])
    with pytest.raises(ValueError, match="out_dtype"):
        lowbit.int8_linear(x, w, s, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="bias"):
        lowbit.int8_linear(x, w, s, torch.zeros(3))
    with pytest.raises(ValueError, match="at least one"):
        lowbit.int8_linear(x[:, :0], w[:, :0], s)
    assert lowbit.kv4_append(*_kv()[:2], torch.zeros(0, 1024, dtype=BF), torch.zeros(0, dtype=torch.int32), n_heads=4).shape == (0, 4, 128)


def test_reference_encoding_round_trips():
    """The tests' own encoder and decoder agree, and a value is within half its scale."""
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, 3, 32, 128, generator=g).double() for _ in range(2))
    pool = ref.encode(k, v, 2)
    for x, got, (codes, scales) in zip((k, v), ref.values(pool), ref.decode(pool)):
        s = scales.repeat_interleave(32, -1)
        assert torch.equal(scales, ref.group_scales(x)) and codes.min() >= 1 and codes.max() <= 15
        assert ((got - x).abs() <= 0.5 * s).all()


def test_python_refuses_sizes_past_32_bits():
    """Sizes that the library's 32-bit arguments cannot hold are refused, not cut (tensors without
    memory: nothing is read)."""
    big = (1 << 32) + 3  # would pass as 3
    i32, meta = torch.int32, "meta"
    pool = torch.empty(4, 2, 1, 2304, dtype=torch.uint8, device=meta)
    table = torch.empty(2, 2, dtype=i32, device=meta)
    two = torch.empty(2, dtype=i32, device=meta)
    q = torch.empty(2, 4, 128, dtype=BF, device=meta)
    rows = torch.empty(big, 1, dtype=BF, device=meta)
    w, s = torch.empty(3, 16, dtype=torch.int8, device=meta), torch.empty(3, device=meta)
    calls = [
        lambda: lowbit.kv4_attend(pool, table, two, q, slot_pos=torch.empty(2, big, dtype=i32, device=meta)),
        lambda: lowbit.kv4_attend(pool, table, two, q, step_score=torch.empty(2, big, device=meta)),
        lambda: lowbit.kv4_attend(pool, torch.empty(2, big, dtype=i32, device=meta), two, q),
        lambda: lowbit.kv4_attend(pool, torch.empty(2, 1 << 28, dtype=i32, device=meta), two, q),  # 2^32 slots
        lambda: lowbit.kv4_gather(pool, table, torch.empty(2 * big, dtype=i32, device=meta)),
        lambda: lowbit.kv4_append(pool, table, torch.empty(2, big, dtype=BF, device=meta)[:, :1024], two, n_heads=4),
        lambda: lowbit.kv4_append(pool, table, torch.empty(big, 1024, dtype=BF, device=meta), two, n_heads=4),
        lambda: lowbit.int8_quantize_rows(rows),
        lambda: lowbit.int8_linear(rows, w[:, :1], s),
        lambda: lowbit.int8_linear(torch.empty(2, 16, dtype=BF, device=meta), torch.empty(big, 16, dtype=torch.int8, device=meta), s),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="32-bit"):
            call()
            pytest.fail(f"call {i}")
