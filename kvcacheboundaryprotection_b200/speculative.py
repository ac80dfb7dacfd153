"""Speculative decoding over the capped slot cache: a draft proposes a tree of tokens per
sequence, the target forwards them together, and the accepted path enters the cache.
``include/kvbp.h`` states the arithmetic.

* ``tree_attend`` is one layer's attention of the tree's nodes over the slots and their
  ancestors, with the eviction score of every (node, key);
* ``verify_tree`` walks the tree against the target's logits with given random numbers and
  returns the accepted path and one more token;
* ``commit_tree`` appends the path to the slots (metadata, score updates, cadence eviction) and
  copies its K and V rows from the drafts into the caches of every layer.

A tree is ``parents`` [B, T] int32 (T <= 128): node 0 is the root (-1), a node's parent comes
before it, a parent below -1 marks an unused node.

Every call enqueues on the current stream of its tensors' device, allocates what it returns
(and its workspace) from torch's caching allocator, and can be captured in a CUDA graph.
Arguments that do not fit raise ``ValueError``, those that the library itself refuses
``capi.KVBPError``; problems found on the device set bits of ``dev_err``, an int32 tensor of one
element, when one is given.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field, fields
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import capi
from .capi import lib
from .engine import EvictionSpec
from .lowbit import _BF16, _F32, _I32, _SCALE, HEAD_DIM, _fits, _launch, _need, _ptr

MAX_NODES = 128


@lru_cache(maxsize=1024)
def _attn_workspace(B: int, T: int, hq: int, hkv: int, S: int, score: bool) -> int:
    return lib().kvbp_tree_attn_workspace(B, T, hq, hkv, S, score)


@lru_cache(maxsize=1024)
def _verify_workspace(B: int, T: int, vocab: int) -> int:
    return lib().kvbp_tree_verify_workspace(B, T, vocab)


def _nodes(T: int) -> None:
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {T}")


def tree_attend(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_draft: torch.Tensor,
                v_draft: torch.Tensor, parents: torch.Tensor, *, slot_pos: Optional[torch.Tensor] = None,
                lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                node_score: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                dev_err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of every node of the tree: q [B, T, heads, 128] bf16 over the live slots of
    k_cache / v_cache [B, kv_heads, S, 128] (s < lens[b] where ``lens`` [B] is given, slot_pos[b, s]
    >= 0 where ``slot_pos`` [B, S] is) and the node's ancestors and itself among k_draft / v_draft
    [B, kv_heads, T, 128].  ``node_score`` [B, T, S + T] float32 is max-accumulated with every
    (node, key)'s largest probability over the heads.  ``scale`` defaults to 1 / sqrt(128).
    Returns out [B, T, heads, 128] bf16, zeros for unused nodes."""
    dev = q.device
    if q.dim() != 4 or k_cache.dim() != 4:
        raise ValueError("q must be [B, T, heads, 128] and k_cache [B, kv heads, S, 128]")
    B, T, hq, _ = q.shape
    hkv, S = k_cache.shape[1], k_cache.shape[2]
    _need(q, "q", _BF16, dev, (B, T, hq, HEAD_DIM))
    _need(k_cache, "k_cache", _BF16, dev, (B, hkv, S, HEAD_DIM))
    _need(v_cache, "v_cache", _BF16, dev, (B, hkv, S, HEAD_DIM))
    _need(k_draft, "k_draft", _BF16, dev, (B, hkv, T, HEAD_DIM))
    _need(v_draft, "v_draft", _BF16, dev, (B, hkv, T, HEAD_DIM))
    _need(parents, "parents", _I32, dev, (B, T))
    if hkv == 0 or hq == 0 or hq % hkv or hq // hkv > 128:
        raise ValueError(f"{hq} query heads over {hkv} kv heads: whole groups of at most 128 are supported")
    if slot_pos is not None:
        _need(slot_pos, "slot_pos", _I32, dev, (B, S))
    if lens is not None:
        _need(lens, "lens", _I32, dev, (B,))
    if node_score is not None:
        _need(node_score, "node_score", _F32, dev, (B, T, S + T))
    if out is None:
        out = torch.empty_like(q)
    else:
        _need(out, "out", _BF16, dev, (B, T, hq, HEAD_DIM))
    if dev_err is not None:
        _need(dev_err, "dev_err", _I32, dev, (1,))
    if B == 0:
        return out
    _nodes(T)
    _fits(S + T, B * hq)
    ws_bytes = _attn_workspace(B, T, hq, hkv, S, node_score is not None)
    ws = q.new_empty((ws_bytes + 1) // 2) if ws_bytes else None
    _launch(
        lib().kvbp_tree_attn, "tree_attn", dev, B, T, hq, hkv, HEAD_DIM, S, q.data_ptr(),
        k_cache.data_ptr() if S else None, v_cache.data_ptr() if S else None, k_draft.data_ptr(), v_draft.data_ptr(),
        parents.data_ptr(), _ptr(slot_pos) if S else None, _ptr(lens), _SCALE if scale is None else scale,
        out.data_ptr(), _ptr(node_score), _ptr(ws), ws_bytes, _ptr(dev_err),
    )
    return out


def _rows3(x: torch.Tensor, name: str, B: int, T: int, V: int) -> int:
    """Row stride of [B, T, V] rows that lie evenly apart."""
    if x.shape != (B, T, V):
        raise ValueError(f"{name} must have shape {(B, T, V)}, got {tuple(x.shape)}")
    sb, st, sv = x.stride()
    ld = st if T > 1 else sb if B > 1 else V
    if (V > 1 and sv != 1) or ld < V or (B > 1 and T > 1 and sb != T * st):
        raise ValueError(f"{name}'s rows must be dense and evenly apart")
    return ld


def verify_tree(target: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, accept_u: torch.Tensor,
                sample_u: torch.Tensor, *, temperature: Optional[torch.Tensor] = None,
                draft_probs: Optional[torch.Tensor] = None, dev_err: Optional[torch.Tensor] = None,
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accept a path of the drafted tree: ``target`` [B, T, vocab] bf16 or float32 are the target's
    logits at every node (rows may be padded), ``tokens`` [B, T] int32 the nodes' tokens, ``accept_u``
    [B, T] and ``sample_u`` [B] float32 uniform numbers in [0, 1), ``temperature`` [B] float32 (0:
    greedy; None: 1).  ``draft_probs`` [B, T, vocab] float32 are the distributions that each node's
    children were drawn from; None for a draft that is not random (its most likely tokens).

    Returns path [B, T] int32 (accepted nodes, the root first, then -1), n_path [B] (their number)
    and next_token [B] (drawn from what the target has left at the last accepted node).  The tokens
    follow the target's distribution if the random numbers are uniform and independent of the draft, and
    siblings were drawn independently, with replacement, from ``draft_probs`` (draws without replacement,
    as of a sampled top-k, do not keep it) or, without ``draft_probs``, were chosen in any way."""
    dev = target.device
    if target.dim() != 3 or target.dtype not in (_BF16, _F32):
        raise ValueError("target must be [B, T, vocab] of bfloat16 or float32")
    B, T, V = target.shape
    _need(tokens, "tokens", _I32, dev, (B, T))
    _need(parents, "parents", _I32, dev, (B, T))
    _need(accept_u, "accept_u", _F32, dev, (B, T))
    _need(sample_u, "sample_u", _F32, dev, (B,))
    if temperature is not None:
        _need(temperature, "temperature", _F32, dev, (B,))
    if draft_probs is not None and (draft_probs.dtype is not _F32 or draft_probs.device != dev or draft_probs.dim() != 3):
        raise ValueError(f"draft_probs must be [B, T, vocab] of float32 on {dev}")
    if dev_err is not None:
        _need(dev_err, "dev_err", _I32, dev, (1,))
    path = torch.empty(B, T, dtype=_I32, device=dev)
    n_path = torch.empty(B, dtype=_I32, device=dev)
    token = torch.empty(B, dtype=_I32, device=dev)
    if B == 0:
        return path, n_path, token
    _nodes(T)
    if V == 0:
        raise ValueError("the vocabulary must not be empty")
    _fits(V, B)
    ldt = _rows3(target, "target", B, T, V)
    ldd = _rows3(draft_probs, "draft_probs", B, T, V) if draft_probs is not None else 0
    ws_bytes = _verify_workspace(B, T, V)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _launch(
        lib().kvbp_tree_verify, "tree_verify", dev, B, T, V, target.dtype is _F32, target.data_ptr(), ldt,
        _ptr(temperature), tokens.data_ptr(), parents.data_ptr(), _ptr(draft_probs), ldd, accept_u.data_ptr(),
        sample_u.data_ptr(), path.data_ptr(), n_path.data_ptr(), token.data_ptr(), _ptr(ws), ws_bytes, _ptr(dev_err),
    )
    return path, n_path, token


@dataclass(frozen=True)
class SlotState:
    """The eviction state of B sequences (``kvbp_state`` and the counters beside it): [B, S] arrays of
    the slots, the bitmap of retained positions ``posmap`` [B, W], the eviction log [B, evcap]."""

    slot_pos: torch.Tensor
    insert_step: torch.Tensor
    last_access: torch.Tensor
    access_count: torch.Tensor
    attn: torch.Tensor
    max_attn: torch.Tensor
    cumul: torch.Tensor
    prefill: torch.Tensor
    posmap: torch.Tensor
    seq_step: torch.Tensor
    next_pos: torch.Tensor
    evlog: torch.Tensor
    evcount: torch.Tensor
    engine: Optional[object] = field(default=None, repr=False, compare=False)  # whose arrays they are (``of``)

    @classmethod
    def of(cls, engine) -> "SlotState":
        """The state of a ``CappedKVEngine`` (its own arrays).  A commit evicts after the whole path, so build
        the engine with ``extra_slots`` >= the longest path - 1.  What a commit finds on the device (no free
        slot among it) goes to the engine's error word unless another is given: ``engine.check_device_errors()``.
        Each commit first applies the scores that the engine's last step has left pending.
        The engine's ``token_log`` and ``retained_log`` hold its own steps only.

        Engines with per-head retention are refused: these operators know no head masks and signals.  The ranks
        of a tensor-parallel engine have the scores of their own heads: reduce ``node_score`` to its maximum over
        the ranks before the commit, or their states part."""
        if engine.per_head:
            raise ValueError("engines with per-KV-head retention have no slot state that commits could change")
        return cls(engine.slot_pos, engine.insert_step, engine.last_access, engine.access_count, engine.attn_s,
                   engine.max_attn, engine.cumul, engine.prefill_s, engine.posmap, engine.seq_step, engine.next_pos,
                   engine.evlog, engine.evcount, engine)

    def like(self) -> "SlotState":
        """Another state of the same sizes, with the same eviction log."""
        return SlotState(*[self.evlog if f.name == "evlog" else torch.empty_like(getattr(self, f.name))
                           for f in fields(self) if f.name != "engine"])

    def _struct(self) -> tuple:
        """(kvbp_state, its device, log size) after the checks."""
        dev = self.slot_pos.device
        if self.slot_pos.dim() != 2 or self.posmap.dim() != 2 or self.evlog.dim() != 2:
            raise ValueError("slot_pos, posmap and evlog must be matrices")
        (B, S), W, cap = self.slot_pos.shape, self.posmap.shape[1], self.evlog.shape[1]
        for name in ("slot_pos", "insert_step", "last_access", "access_count"):
            _need(getattr(self, name), name, _I32, dev, (B, S))
        for name in ("attn", "max_attn", "prefill"):
            _need(getattr(self, name), name, _F32, dev, (B, S))
        _need(self.cumul, "cumul", torch.float64, dev, (B, S))
        _need(self.posmap, "posmap", _I32, dev, (B, W))
        _need(self.evlog, "evlog", _I32, dev, (B, cap))
        for name in ("seq_step", "next_pos", "evcount"):
            _need(getattr(self, name), name, _I32, dev, (B,))
        _fits(S, W)
        arrays = (self.slot_pos, self.insert_step, self.last_access, self.access_count, self.attn, self.max_attn,
                  self.cumul, self.prefill, self.posmap)
        return capi.State(B, S, W, *[t.data_ptr() for t in arrays]), dev, cap


def _evict_cfg(spec: Optional[EvictionSpec]):
    if spec is None:
        return None
    if spec.regime not in ("decode", "prefill"):
        raise ValueError("the eviction regime must be 'decode' or 'prefill'")
    n_prefix, n_suffix = spec.sizes()
    return capi.EvictCfg(spec.capacity, spec.evict_every, capi.policy_id(spec.policy), int(spec.protect), n_prefix,
                         n_suffix, int(spec.regime == "decode"))


def commit_tree(state: SlotState, path: torch.Tensor, n_path: torch.Tensor, k_draft: torch.Tensor,
                v_draft: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                node_score: Optional[torch.Tensor] = None, evict: Optional[EvictionSpec] = None,
                out: Optional[SlotState] = None, dev_err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Append the accepted path to the slots: for i < n_path[b], node path[b, i] takes the lowest
    free slot as the next position, with the metadata and (where ``node_score`` [B, T, S + T] is
    given) the score update of its own step; then, where the step counter passed a multiple of
    ``evict.evict_every``, one eviction down to the capacity.  K and V rows of what stays are copied
    from k_draft / v_draft [layers, B, kv_heads, T, 128] into k_cache / v_cache [layers, B, kv_heads,
    S, 128].  ``state`` is updated in place, or, with ``out`` (of the same sizes), left as it is and the
    new state written there, so that a step can be taken back (the eviction log is appended to in
    place when both share it).

    Returns write_slot [B, T] int32: each path entry's slot, -1 where there is none."""
    st_in, dev, cap = state._struct()
    B, S = st_in.B, st_in.S
    engine = state.engine
    new = state if out is None else out
    st_out, dev_out, cap_out = (st_in, dev, cap) if out is None else out._struct()
    if (st_out.B, st_out.S, st_out.W, dev_out) != (B, S, st_in.W, dev):
        raise ValueError("out must be a state of the same sizes on the same device")
    T = path.shape[-1] if path.dim() else 0
    _need(path, "path", _I32, dev, (B, T))
    _need(n_path, "n_path", _I32, dev, (B,))
    if k_draft.dim() != 5:
        raise ValueError("k_draft must be [layers, B, kv heads, T, 128]")
    L, _, hkv = k_draft.shape[:3]
    for name, t, rows in (("k_draft", k_draft, T), ("v_draft", v_draft, T), ("k_cache", k_cache, S),
                          ("v_cache", v_cache, S)):
        _need(t, name, _BF16, dev, (L, B, hkv, rows, HEAD_DIM))
    if node_score is not None:
        _need(node_score, "node_score", _F32, dev, (B, T, S + T))
    if dev_err is None and engine is not None:
        dev_err = engine.dev_err
    if dev_err is not None:
        _need(dev_err, "dev_err", _I32, dev, (1,))
    cfg = _evict_cfg(evict)
    write_slot = torch.empty(B, T, dtype=_I32, device=dev)
    if B == 0:
        return write_slot
    _nodes(T)
    if S == 0 or st_in.W == 0 or cap_out == 0:
        raise ValueError("the state must not be empty")
    _fits(L * hkv * 8)
    if L * hkv == 0:
        L = 0
    if engine is not None:  # the old state's last step is part of it
        with torch.cuda.device(dev):
            engine.apply_pending_scores()
    _launch(
        lib().kvbp_tree_commit, "tree_commit", dev, C.byref(st_in), C.byref(st_out),
        None if cfg is None else C.byref(cfg), T, path.data_ptr(), n_path.data_ptr(), _ptr(node_score), L, hkv, HEAD_DIM,
        k_draft.data_ptr() if L else None, v_draft.data_ptr() if L else None, k_cache.data_ptr() if L else None,
        v_cache.data_ptr() if L else None, state.seq_step.data_ptr(), state.next_pos.data_ptr(),
        state.evcount.data_ptr(), new.seq_step.data_ptr(), new.next_pos.data_ptr(), new.evcount.data_ptr(),
        new.evlog.data_ptr(), cap_out, write_slot.data_ptr(), _ptr(dev_err),
    )
    return write_slot
