"""Refusals of the speculative decoding operators, without a GPU: the C entry points check every
argument before their first CUDA call, the Python ones before they launch."""

import ctypes as C
import dataclasses
import types

import pytest
import torch

from kvcacheboundaryprotection_b200 import build, capi, speculative as sp

import spec_ref as ref

BF = torch.bfloat16
_FIELDS = [f.name for f in dataclasses.fields(sp.SlotState) if f.name != "engine"]
A = 1 << 30  # an aligned address that is never read


@pytest.fixture(scope="module")
def L():
    build.build()
    return capi.lib()


def _attn(L, **kw):
    a = dict(B=2, T=5, Hq=4, Hkv=2, D=128, S=64, q=A, k=2 * A, v=3 * A, kd=4 * A, vd=5 * A, parents=6 * A, pos=7 * A,
             lens=8 * A, scale=0.1, out=9 * A, score=10 * A, ws=11 * A, wsb=1 << 30, err=None)
    a.update(kw)
    return L.kvbp_tree_attn(None, *a.values())


@pytest.mark.parametrize(
    "bad,status",
    [(dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(kd=None), 1), (dict(vd=None), 1),
     (dict(parents=None), 1), (dict(out=None), 1), (dict(D=64), 2), (dict(B=0), 1), (dict(B=65536), 1), (dict(T=0), 2),
     (dict(T=129), 2), (dict(Hkv=0), 1), (dict(Hkv=3), 1), (dict(Hq=0), 1), (dict(S=-1), 1), (dict(Hq=258, Hkv=2), 2),
     (dict(q=A + 8), 1), (dict(k=2 * A + 2), 1), (dict(vd=5 * A + 4), 1), (dict(out=9 * A + 8), 1), (dict(ws=11 * A + 4), 1),
     (dict(ws=None), 1), (dict(wsb=1000), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1),
     (dict(out=A), 1), (dict(out=A + 4096), 1), (dict(score=2 * A), 1), (dict(ws=3 * A), 1), (dict(score=9 * A + 64), 1),
     (dict(ws=9 * A), 1), (dict(out=6 * A), 1), (dict(S=0x7fffffff), 1), (dict(B=65535, Hkv=8, Hq=8, S=1 << 22), 1)],
)
def test_attention_refusals(L, bad, status):
    assert _attn(L, **bad) == status and L.kvbp_last_error().startswith(b"tree_attn")


def test_attention_workspace(L):
    one = L.kvbp_tree_attn_workspace(1, 8, 8, 2, 256, 0)
    assert one > 0 and one % 256 == 0
    assert L.kvbp_tree_attn_workspace(1, 128, 8, 1, 256, 1) > one  # two row tiles a unit
    for bad in ((0, 8, 8, 2), (1, 0, 8, 2), (1, 129, 8, 2), (1, 8, 8, 3), (1, 8, 0, 2), (1, 8, 258, 2)):
        assert L.kvbp_tree_attn_workspace(*bad, 256, 0) == 0


def _verify(L, **kw):
    a = dict(B=2, T=5, V=100, f32=0, target=A, ldt=100, temp=None, tokens=A, parents=A, draft=A, ldd=100, u=A, s=A, path=A,
             n=A, token=A, ws=None, wsb=0, err=None)
    a.update(kw)
    return L.kvbp_tree_verify(None, *a.values())


@pytest.mark.parametrize(
    "bad,status",
    [(dict(target=None), 1), (dict(tokens=None), 1), (dict(parents=None), 1), (dict(u=None), 1), (dict(s=None), 1),
     (dict(path=None), 1), (dict(n=None), 1), (dict(token=None), 1), (dict(B=0), 1), (dict(V=0), 1), (dict(T=0), 2),
     (dict(T=129), 2), (dict(ldt=99), 1), (dict(ldd=99), 1), (dict(target=A + 1), 1), (dict(f32=1, target=A + 2), 1),
     (dict(draft=A + 2), 1)],
)
def test_verification_refusals(L, bad, status):
    assert _verify(L, **bad) == status and L.kvbp_last_error().startswith(b"tree_verify")


def _state(at, **kw):
    s = capi.State(2, 64, 8, *[at + i * (1 << 20) for i in range(9)])
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _commit(L, **kw):
    a = dict(st_in=_state(A), st_out=_state(2 * A), cfg=capi.EvictCfg(32, 8, 0, 1, 4, 4, 1), T=5, path=3 * A, n=4 * A,
             score=5 * A, layers=2, Hkv=2, D=128, kd=6 * A, vd=7 * A, k=8 * A, v=9 * A, step=10 * A, pos=11 * A, cnt=12 * A,
             step_o=13 * A, pos_o=14 * A, cnt_o=15 * A, log=16 * A, cap=100, write=17 * A, err=None)
    a.update(kw)
    for k in ("st_in", "st_out", "cfg"):
        a[k] = C.byref(a[k]) if a[k] is not None else None
    return L.kvbp_tree_commit(None, *a.values())


@pytest.mark.parametrize(
    "bad,status",
    [(dict(st_in=None), 1), (dict(st_out=None), 1), (dict(path=None), 1), (dict(n=None), 1), (dict(step=None), 1),
     (dict(pos_o=None), 1), (dict(cnt=None), 1), (dict(log=None), 1), (dict(write=None), 1), (dict(T=0), 2), (dict(T=129), 2),
     (dict(D=64), 2), (dict(Hkv=0), 1), (dict(layers=-1), 1), (dict(kd=None), 1), (dict(v=None), 1), (dict(k=8 * A + 8), 1),
     (dict(kd=8 * A), 1), (dict(v=8 * A), 1), (dict(st_out=_state(2 * A, S=65)), 1), (dict(st_out=_state(A + 4)), 1),
     (dict(st_out=_state(A, attn=A)), 1), (dict(st_in=_state(A, slot_pos=None)), 1), (dict(cap=-1), 1),
     (dict(cfg=capi.EvictCfg(0, 8, 0, 1, 4, 4, 1)), 1), (dict(cfg=capi.EvictCfg(32, 0, 0, 1, 4, 4, 1)), 1),
     (dict(cfg=capi.EvictCfg(32, 8, 99, 1, 4, 4, 1)), 1), (dict(cfg=capi.EvictCfg(32, 8, 8, 1, 4, 4, 1)), 2),
     (dict(cfg=capi.EvictCfg(32, 8, 0, 1, -1, 4, 1)), 1), (dict(write=10 * A), 1), (dict(step_o=11 * A), 1),
     (dict(step_o=13 * A, pos_o=13 * A), 1), (dict(log=5 * A + 64), 1),
     (dict(st_in=_state(A, S=20000), st_out=_state(2 * A, S=20000)), 2)],
)
def test_commit_refusals(L, bad, status):
    assert _commit(L, **bad) == status and L.kvbp_last_error().startswith(b"tree_commit")


def test_pending_update_refusals(L):
    st = _state(A)
    for a in ((None, A, 2 * A, 3 * A), (C.byref(st), None, 2 * A, 3 * A), (C.byref(st), A, None, 3 * A),
              (C.byref(st), A, 2 * A, None), (C.byref(_state(A, slot_pos=None)), A, 2 * A, 3 * A)):
        assert L.kvbp_score_update_pending(None, *a, None) == 1 and L.kvbp_last_error().startswith(b"score_update")


def _tensors(B=2, T=4, hq=4, hkv=2, S=20):
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)  # noqa: E731
    return dict(q=z(B, T, hq, 128), k_cache=z(B, hkv, S, 128), v_cache=z(B, hkv, S, 128), k_draft=z(B, hkv, T, 128),
                v_draft=z(B, hkv, T, 128), parents=z(B, T, dt=torch.int32))


@pytest.mark.parametrize(
    "name,value",
    [("q", torch.zeros(2, 4, 3, 128, dtype=BF)), ("q", torch.zeros(2, 4, 4, 64, dtype=BF)), ("q", torch.zeros(2, 4, 4, 128)),
     ("q", torch.zeros(2, 4, 512, dtype=BF)), ("q", torch.zeros(2, 4, 128, 4, dtype=BF).transpose(2, 3)),
     ("k_cache", torch.zeros(2, 2, 21, 128, dtype=BF)), ("v_cache", torch.zeros(2, 2, 20, 128)),
     ("k_draft", torch.zeros(2, 2, 5, 128, dtype=BF)), ("parents", torch.zeros(2, 4, dtype=torch.int64)),
     ("parents", torch.zeros(2, 5, dtype=torch.int32)), ("slot_pos", torch.zeros(2, 21, dtype=torch.int32)),
     ("lens", torch.zeros(3, dtype=torch.int32)), ("node_score", torch.zeros(2, 4, 20)), ("out", torch.zeros(2, 4, 4, 128)),
     ("dev_err", torch.zeros(2, dtype=torch.int32)), ("none", None)],
)
def test_python_attention_refusals(name, value):
    """What does not fit is a ValueError; so are tensors that fit but lie on the CPU ("none")."""
    t = _tensors()
    if name != "none":
        t[name] = value
    kw = {k: t.pop(k) for k in list(t) if k in ("slot_pos", "lens", "node_score", "out", "dev_err")}
    with pytest.raises(ValueError):
        sp.tree_attend(*t.values(), **kw)


def test_python_attention_of_nothing_and_too_many_nodes():
    assert sp.tree_attend(*_tensors(B=0).values()).shape == (0, 4, 4, 128)
    for T in (0, 129):
        with pytest.raises(ValueError, match="nodes"):
            sp.tree_attend(*_tensors(T=T).values())


@pytest.mark.parametrize(
    "name,value",
    [("target", torch.zeros(2, 4, 50, dtype=torch.float16)), ("target", torch.zeros(2, 200)), ("target", torch.zeros(2, 4, 0)),
     ("target", torch.zeros(2, 4, 100)[..., ::2]), ("target", torch.zeros(2, 8, 50)[:, ::2][:, :, :50].transpose(0, 1)),
     ("target", torch.zeros(2, 6, 50)[:, :4]), ("tokens", torch.zeros(2, 4)), ("parents", torch.zeros(2, 3, dtype=torch.int32)),
     ("accept_u", torch.zeros(2, 4, dtype=torch.float64)), ("sample_u", torch.zeros(2, 1)),
     ("temperature", torch.zeros(1)), ("draft_probs", torch.zeros(2, 4, 50, dtype=BF)), ("draft_probs", torch.zeros(2, 4, 51)),
     ("none", None)],
)
def test_python_verification_refusals(name, value):
    t = dict(target=torch.zeros(2, 4, 50), tokens=torch.zeros(2, 4, dtype=torch.int32),
             parents=torch.zeros(2, 4, dtype=torch.int32), accept_u=torch.zeros(2, 4), sample_u=torch.zeros(2))
    if name != "none":
        t[name] = value
    kw = {k: t.pop(k) for k in list(t) if k in ("temperature", "draft_probs")}
    with pytest.raises(ValueError):
        sp.verify_tree(*t.values(), **kw)


def _slot_state(B=2, S=20, W=4, cap=30):
    i, f = torch.int32, torch.float32
    z = lambda *s, dt=i: torch.zeros(*s, dtype=dt)  # noqa: E731
    return sp.SlotState(z(B, S), z(B, S), z(B, S), z(B, S), z(B, S, dt=f), z(B, S, dt=f), z(B, S, dt=torch.float64),
                        z(B, S, dt=f), z(B, W), z(B), z(B), z(B, cap), z(B))


def test_engines_with_per_head_retention_are_refused():
    names = dict(attn="attn_s", prefill="prefill_s")
    eng = types.SimpleNamespace(per_head=False, **{names.get(k, k): getattr(_slot_state(), k) for k in _FIELDS})
    state = sp.SlotState.of(eng)
    assert state.engine is eng and state.like().engine is None and state.attn is eng.attn_s
    eng.per_head = True
    with pytest.raises(ValueError, match="per-KV-head"):
        sp.SlotState.of(eng)


def test_python_commit_refusals():
    def call(state=None, path=(2, 4), n=(2,), kd=(3, 2, 2, 4, 128), k=(3, 2, 2, 20, 128), **kw):
        return sp.commit_tree(state or _slot_state(), torch.zeros(path, dtype=torch.int32), torch.zeros(n, dtype=torch.int32),
                              torch.zeros(kd, dtype=BF), torch.zeros(kd, dtype=BF), torch.zeros(k, dtype=BF),
                              torch.zeros(k, dtype=BF), **kw)

    cases = [dict(), dict(path=(2,)), dict(path=(3, 4)), dict(n=(3,)), dict(kd=(2, 2, 4, 128)), dict(kd=(3, 2, 2, 5, 128)),
             dict(k=(3, 2, 2, 21, 128)), dict(k=(2, 2, 2, 20, 128)), dict(node_score=torch.zeros(2, 4, 20)),
             dict(out=_slot_state(S=21)), dict(out=_slot_state(W=5)), dict(path=(2, 129), kd=(3, 2, 2, 129, 128)),
             dict(state=_slot_state(cap=0)), dict(evict=sp.EvictionSpec(policy="no_such_policy")),
             dict(evict=sp.EvictionSpec(regime="never"))]
    for kw in cases:
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError):
        sp.SlotState(*[torch.zeros(2, 3)] * 13)._struct()


def test_reference_statements():
    """The plain statements that the GPU tests compare with, on cases done by hand."""
    assert ref.sees([-1, 0, 0, 2, 5, -2, 5]) == [[0], [0, 1], [0, 2], [0, 2, 3], None, None, None]
    import numpy as np

    t = np.log(np.array([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]))
    assert ref.verify(t, [0, 0], [-1, 0], [0, 0.4], 0.15) == ([0, 1], 1)  # 0.4 < 0.5; 0.15 of [.1, .1, .8]
    assert ref.verify(t, [0, 0], [-1, 0], [0, 0.6], 0.59) == ([0], 1)  # rejected: [0, .3, .2], 0.295 < 0.3
    q = np.array([[0.8, 0.1, 0.1]] * 2)
    assert ref.verify(t, [0, 0], [-1, 0], [0, 0.7], 0.5, draft=q) == ([0], 1)  # 0.56 >= 0.5; residual [0, .2, .1]
    assert ref.verify(t, [0, 1], [-1, 0], [0, 0.99], 0.95, draft=q)[0] == [0, 1]  # q below p: always
