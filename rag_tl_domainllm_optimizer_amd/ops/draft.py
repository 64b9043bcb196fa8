"""Checking drafted tokens: a forward over a tree of guesses per row instead of one token (no grad).

A step of it: :func:`draft_tree` makes the plan of the batch's trees (node 0 of a row is its last token, every other node continues an earlier
one); the model runs all nodes as rows, at the positions ``tree.pos``, its layers attending with :func:`tree_attention` over the cache and the
node's own ancestors (``CausalLM.verify``); what the model would write after each node is sampled from the logits; :func:`tree_accept` follows it
through the tree and appends the keys and values of the nodes on that path to the cache of every layer. Nodes that were not
accepted never touch the cache. All of it stays on the device and can be captured in a graph."""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import List, Optional

import torch

from . import reference as ref
from ._ext import native, on_gpu
from .attention import FP8_KV_D, kv_dequantize, kv_quantize_rows

MAX_NODES = 64  # a node's ancestors are the bits of one word


@dataclass
class DraftTree:
    """Trees of a batch, [rows, nodes] each: parent int32 (as given), see int64 (bit j: the node itself or its ancestor j; 0: not
    a node), pos int32. ``heads``: of rows that :func:`tree_attention` read with it, by key heads, head size and columns, the query heads (None: not
    always as many)."""

    parent: torch.Tensor
    see: torch.Tensor
    pos: torch.Tensor
    heads: dict = field(default_factory=dict)

    @property
    def shape(self):
        return self.see.shape


def _ints(t, name, shape, like):
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or t.device != like.device:
        raise ValueError(f"{name}: int32 {tuple(shape)} on {like.device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.contiguous()


def _scales(k_cache, v_cache, k_scale, v_scale) -> bool:
    """whether the caches are fp8, with the scales that go with them"""
    fp8 = k_scale is not None
    if fp8 != (v_scale is not None) or fp8 != (k_cache.dtype == torch.uint8) or v_cache.dtype != k_cache.dtype:
        raise ValueError("an fp8 cache (uint8) has scales of its keys and values, another one has none")
    if fp8 and (k_cache.shape[-1] != FP8_KV_D or any(s.dtype != torch.float32 or s.shape[:-1] != k_cache.shape[:-2] or s.shape[-1] < k_cache.shape[-2]
                                                     for s in (k_scale, v_scale))):
        raise ValueError(f"an fp8 cache has heads of {FP8_KV_D} and fp32 scales of every slot")
    return fp8


def _nodes(tree):
    if tree.see.dim() != 2 or not 1 <= tree.see.shape[1] <= MAX_NODES:
        raise ValueError(f"a tree [rows, 1 .. {MAX_NODES} nodes] expected, got {tuple(tree.shape)}")


def _rows_of(Hkv, D, cols):
    return -1 if Hkv >> 16 or D >> 17 or cols >> 30 else (Hkv << 17 | D) << 30 | cols


def draft_tree(parent: torch.Tensor, nodes: Optional[torch.Tensor] = None, pos0: Optional[torch.Tensor] = None) -> DraftTree:
    """The plan of drafted trees: ``parent`` int32 [rows, nodes <= 64] holds an earlier node of the row for each (anything else: none, a tree of its
    own), ``nodes`` int32 [rows] how many of a row's are nodes (0: the row idles; default all), ``pos0`` int32 [rows] the position
    of node 0 (default 0)."""
    if on_gpu(parent):
        return DraftTree(*native().draft_tree(parent, nodes, pos0))
    if parent.dim() != 2 or not 1 <= parent.shape[1] <= MAX_NODES:
        raise ValueError(f"parent: [rows, 1 .. {MAX_NODES} nodes] expected, got {tuple(parent.shape)}")
    parent = _ints(parent, "parent", parent.shape, parent)
    nodes = None if nodes is None else _ints(nodes, "nodes", parent.shape[:1], parent)
    pos0 = None if pos0 is None else _ints(pos0, "pos0", parent.shape[:1], parent)
    return DraftTree(parent, *ref.draft_tree(parent, nodes, pos0))


def tree_attention(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_len: torch.Tensor, tree: DraftTree, Hq: int,
                   kv_start: Optional[torch.Tensor] = None, window: int = 0, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None, as_stored: bool = False) -> torch.Tensor:
    """Attention of drafted tokens -> [rows * nodes, Hq * D]. ``qkv`` [rows * nodes, >= (Hq + 2 Hkv) * D] holds the nodes' rotated rows [q | k | v];
    node i sees the slots [kv_start, kv_len) of its row in the caches [rows, Hkv, Smax, D] and its ancestors' and its own
    key; with ``window`` only those less than ``window`` positions before it (a node's, in masks of the caller's own too, is how many nodes it
    sees). Nothing is appended to the caches; rows that are not
    nodes come out as zeros. ``out`` may be columns of wider rows, but shares nothing with ``qkv``. What a node does not see, of other
    nodes or outside its window, does not reach it, NaN and infinities among it. uint8 caches hold e4m3 (heads of 128), as
    ``kv_quantize_rows`` and decoding write them, with their slots' scales in ``k_scale``, ``v_scale`` [rows, Hkv, >= Smax].
    Over these, nodes count with the keys and values of ``qkv`` as a prompt's tokens do, before they are rounded; with ``as_stored`` they count as
    :func:`tree_accept` will store them, which is what decoding token by token sees."""
    if on_gpu(qkv):
        return native().tree_attention(qkv, k_cache, v_cache, kv_len, kv_start, tree.see, out, Hq, window, scale, k_scale, v_scale, as_stored, tree.heads)
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"caches [rows, heads, slots, dim] expected, got {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    _nodes(tree)
    B, Hkv, Smax, D = k_cache.shape
    N = tree.shape[1]
    if tree.shape[0] != B or qkv.dim() != 2 or qkv.shape[0] != B * N:
        raise ValueError(f"qkv: {B} rows of {N} nodes expected, got {tuple(qkv.shape)} for a tree {tuple(tree.shape)}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv or qkv.shape[1] < (Hq + 2 * Hkv) * D:
        raise ValueError(f"{Hq} heads over {Hkv} of {D} do not fit {qkv.shape[1]} columns")
    fp8 = _scales(k_cache, v_cache, k_scale, v_scale)
    if qkv.dtype != (torch.bfloat16 if fp8 else k_cache.dtype) and not (fp8 and qkv.dtype == torch.float32):
        raise ValueError(f"caches of {k_cache.dtype} under queries of {qkv.dtype}")
    key = _rows_of(Hkv, D, qkv.shape[1])
    if key < 0:
        raise ValueError(f"{Hkv} key heads of {D} in {qkv.shape[1]} columns")
    if as_stored and not fp8:
        raise ValueError("only an fp8 cache stores nodes otherwise than they are")
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    if window < 0 or not 0 < scale < math.inf:
        raise ValueError(f"window {window}, scale {scale}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (qkv, k_cache, v_cache)):
        raise ValueError("tree_attention has no gradient")
    if out is not None and (out.dtype != qkv.dtype or tuple(out.shape) != (B * N, Hq * D)):
        raise ValueError(f"out: {qkv.dtype} {(B * N, Hq * D)} expected, got {out.dtype} {tuple(out.shape)}")
    kv_len = _ints(kv_len, "kv_len", (B,), qkv)
    kv_start = None if kv_start is None else _ints(kv_start, "kv_start", (B,), qkv)
    if fp8:
        k_cache, v_cache = (kv_dequantize(c, sc[..., :Smax], k) for c, sc, k in ((k_cache, k_scale, True), (v_cache, v_scale, False)))
    kind = qkv.dtype
    if as_stored:
        q, *kv = qkv[:, :(Hq + 2 * Hkv) * D].float().split([Hq * D, Hkv * D, Hkv * D], 1)
        qkv = torch.cat([q] + [kv_dequantize(*kv_quantize_rows(x.reshape(B * N, Hkv, D), k), k).view(B * N, Hkv * D) for x, k in zip(kv, (True, False))], 1)
    o = ref.tree_attention(qkv, k_cache, v_cache, kv_len, tree.see, Hq, kv_start, window, scale).to(kind)
    if tree.heads.setdefault(key, Hq) != Hq:
        tree.heads[key] = None
    return o if out is None else out.copy_(o)


def tree_accept(tree: DraftTree, tokens: torch.Tensor, choice: torch.Tensor, drafts: List[torch.Tensor], k_cache: torch.Tensor,
                v_cache: torch.Tensor, kv_len: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                Hq: Optional[int] = None):
    """The path that the model agrees with -> (its length int32 [rows], its nodes int32 [rows, nodes] (-1 behind them), the token after it int64
    [rows]). ``tokens`` / ``choice`` int64 [rows, nodes]: the drafted tokens, and what the model writes after each; the path starts at node 0 and goes
    on with the child whose token is the choice (the first of equal ones). Keys and values of its nodes go from ``drafts``
    (per layer the rows that :func:`tree_attention` read) to the slots from ``kv_len`` of the caches [layers, rows, Hkv, Smax, D]; ``kv_len``
    itself is the caller's to advance by the length. An idle row has length 0 and token -1. A path ends
    with the cache: its last node is the one that took the last slot, the token the choice after that; a row without a slot idles.
    ``Hq``: query heads in front of the keys in ``drafts``, by default as :func:`tree_attention` read rows of this width with this tree; others
    hold nothing behind [q | k | v]. ``k_scale`` / ``v_scale`` [layers, rows, Hkv, >= Smax]: the caches are fp8, and rows are rounded into them as ``kv_store_fp8`` does."""
    if Hq is not None and Hq < 1:
        raise ValueError(f"{Hq} query heads")
    if on_gpu(k_cache):
        return native().tree_accept(tree.parent, tree.see, tokens, choice, drafts, k_cache, v_cache, kv_len, k_scale, v_scale, Hq or 0, tree.heads)
    if k_cache.dim() != 5 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError(f"caches [layers, rows, heads, slots, dim] expected, got {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    _nodes(tree)
    L, B, Hkv, Smax, D = k_cache.shape
    if tree.shape[0] != B or tuple(tokens.shape) != tuple(tree.shape) or tuple(choice.shape) != tuple(tree.shape):
        raise ValueError(f"tree {tuple(tree.shape)}, tokens {tuple(tokens.shape)} and choice {tuple(choice.shape)} of {B} rows do not go together")
    if tokens.dtype != torch.int64 or choice.dtype != torch.int64:
        raise ValueError("tokens and choice: int64 expected")
    if D < 1 or Hkv < 1:
        raise ValueError("caches of no heads")
    for a, b in ((k_cache, v_cache), (k_scale, v_scale)):
        if a is not None and b is not None and a.numel() and (a.data_ptr() == b.data_ptr() or any(
                st == 0 and n > 1 for t in (a, b) for st, n in zip(t.stride(), t.shape))):
            raise ValueError("layers, or keys and values, of one memory")
    fp8 = _scales(k_cache, v_cache, k_scale, v_scale)
    if len(drafts) != L or any(x.dim() != 2 or x.shape != drafts[0].shape or (x.dtype != k_cache.dtype and not fp8) or x.shape[0] != B * tree.shape[1]
                               for x in drafts):
        raise ValueError(f"drafts: rows [q | k | v] of {B * tree.shape[1]} nodes in {k_cache.dtype} for each of {L} layers expected")
    cols = drafts[0].shape[1]
    heads = tree.heads.get(_rows_of(Hkv, D, cols), 0) if Hq is None else Hq
    if heads is None:
        raise ValueError("rows of this width were read with different heads: Hq says which these have")
    Hq = heads or cols // D - 2 * Hkv
    if Hq < 1 or Hq % Hkv or cols < (Hq + 2 * Hkv) * D or (not heads and cols % D):
        raise ValueError(f"{Hq} heads over {Hkv} of {D} do not fit drafts of {cols} columns")
    drafts = [x[:, :(Hq + 2 * Hkv) * D] for x in drafts]
    kv_len = _ints(kv_len, "kv_len", (B,), k_cache)
    store = (lambda x, k: kv_quantize_rows(x, k)) if fp8 else None
    return ref.tree_accept(tree.parent, tree.see, tokens, choice, drafts, k_cache, v_cache, kv_len, store, k_scale, v_scale)
