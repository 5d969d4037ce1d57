"""Trees of drafted tokens around the paged decode: the torch-facing entry points.

* ``tree_plan(parents, cache_seqlens, block_table, tree_lens)`` -> ``TreePlan(mask, positions, slots, prefix_lens)``:
  what each drafted token sees, its position and its cache row, from the nodes' parents.
* ``tree_accept(plan, tokens, targets)`` -> ``Accepted(path, counts, next_tokens, keep_lens)``: the drafted path that
  the model's own choices agree with.
* ``kv_keep_path(kv_cache, slots, path)``: that path's rows together at the front of the tree, in place.

A step that verifies trees is ``reserve_pages`` -> ``tree_plan`` (with ``tree_lens`` the nodes reserved times the
reservation's ``granted``) -> ``kv_append_slots`` (the plan's slots and positions) -> ``get_mla_metadata`` over the plan's ``prefix_lens`` -> ``flash_mla_with_kvcache(..., tree=plan)`` -> ``tree_accept`` ->
``kv_keep_path`` (each layer's cache) -> ``release_pages`` (to ``keep_lens``).  Calls are queued on torch's current stream
of the tensors' device, synchronise nothing, and can be captured in a HIP graph.  The reference decodes one token or a
causal run of them and has no counterpart of these.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import MlaTreePlanArgs
from .api import TreePlan, _launch, new_tensor
from .serving import _cache_struct, _require

_PLAN = struct.Struct("=4Q4i4Q")
assert _PLAN.size == ctypes.sizeof(MlaTreePlanArgs)

_INT32 = (torch.int32,)
_INTS = (torch.int32, torch.int64)


class Accepted(NamedTuple):
    """What :func:`tree_accept` gives: ``path [B, s_q]`` the kept nodes in order (-1 behind the last), ``counts [B]`` how
    many they are, ``keep_lens [B]`` the sequences' lengths with them alone, all int32, and ``next_tokens [B]`` the
    model's token after the last one, in the tokens' dtype (-1 where none is kept)."""
    path: torch.Tensor
    counts: torch.Tensor
    next_tokens: torch.Tensor
    keep_lens: torch.Tensor


def _grid(t: torch.Tensor, name: str, dtype: torch.dtype, shape, index: int) -> None:
    """A contiguous ``shape`` tensor of ``dtype`` on GPU ``index``; what it is not, said in full only where it is not."""
    if t.get_device() == index and t.dtype is dtype and t.shape == shape and t.is_contiguous():
        return
    _require(t, name)
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the other tensors on cuda:{index}")
    raise ValueError(f"{name} must be a contiguous {str(dtype).replace('torch.', '')} tensor {list(shape)}")


def _first_grid(t: torch.Tensor, name: str, dtypes) -> int:
    """Checks the ``[B, s_q]`` tensor that gives a call its shape; its GPU's index."""
    index = t.get_device()
    if index < 0:
        _require(t, name)
    if t.dtype not in dtypes or t.dim() != 2 or not t.is_contiguous():
        kinds = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        raise ValueError(f"{name} must be a contiguous {kinds} tensor [B, s_q]")
    if not 1 <= t.shape[1] <= _lib.MLA_TREE_MAX_NODES:
        raise ValueError(f"s_q must be in [1, {_lib.MLA_TREE_MAX_NODES}]")
    return index


def tree_plan(parents: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
              tree_lens: Optional[torch.Tensor] = None) -> TreePlan:
    """Plan of a step in which the last ``tree_lens[b]`` tokens of ``cache_seqlens[b]`` are a tree of drafted ones.

    ``parents [B, s_q]`` (int32, s_q <= 64): node i's parent, a lower node, or -1 for a root, which follows the prefix.
    Any other value drops the node, and with it what hangs below it: no node sees it and it sees none, itself neither;
    so do nodes past ``tree_lens`` (int32 ``[B]``, by default all are s_q long).  ``tree_lens`` is what the step's
    ``reserve_pages`` added to ``cache_seqlens``: 0 for a request that it did not grant, whose last tokens would be taken
    for the tree otherwise, overwritten by the append and released.  A dropped node is known by its mask, 0, and its
    position, -1: the decode still gives it a row, the attention of the prefix alone (lse -inf only where that is empty),
    and within the tree's length it still has its row in the cache.  A sequence shorter than its tree has none of it."""
    index = _first_grid(parents, "parents", _INT32)
    device = parents.device
    B, s_q = shape = parents.shape
    _grid(cache_seqlens, "cache_seqlens", torch.int32, (B,), index)
    if tree_lens is not None:
        _grid(tree_lens, "tree_lens", torch.int32, (B,), index)
    if block_table.get_device() != index:
        _require(block_table, "block_table", device)
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError("block_table must be a [B, P] int32 tensor with unit column stride")
    (_, P), (stride, unit) = block_table.shape, block_table.stride()
    if P < 1 or (P > 1 and unit != 1) or (B > 1 and stride < P) or (B > 1 and stride >= 2 ** 31):
        raise ValueError("block_table must have columns of unit stride, and rows below 2^31 apart that do not overlap")
    mask = new_tensor(shape, torch.int64, device)
    positions, slots, prefix = torch.empty_like(parents), torch.empty_like(parents), torch.empty_like(cache_seqlens)
    a = MlaTreePlanArgs.from_buffer_copy(_PLAN.pack(
        parents.data_ptr(), cache_seqlens.data_ptr(), tree_lens.data_ptr() if tree_lens is not None else 0,
        block_table.data_ptr(), stride if B > 1 else P, P, B, s_q, mask.data_ptr(), positions.data_ptr(),
        slots.data_ptr(), prefix.data_ptr()))
    _launch("mla_tree_plan", _lib.load().mla_tree_plan, device, ctypes.byref(a))
    return TreePlan(mask, positions, slots, prefix)


def tree_accept(plan: TreePlan, tokens: torch.Tensor, targets: torch.Tensor) -> Accepted:
    """The path that the model agrees with, of each sequence's tree.

    ``tokens [B, s_q]`` are the drafted tokens, ``targets [B, s_q]`` what the model chose after each node (both int32
    or both int64).  Node 0 is the token that the step before decided (its ``next_tokens``): it is kept.  From there the
    path goes on, while there is one, to the child whose token is the target of the node before; of several with that
    token to the lowest.  Where node 0 is no root nothing is kept."""
    index = _first_grid(tokens, "tokens", _INTS)
    device, dtype, shape = tokens.device, tokens.dtype, tokens.shape
    B, s_q = shape
    mask, _, _, prefix = plan
    _grid(targets, "targets", dtype, shape, index)
    _grid(mask, "plan.mask", torch.int64, shape, index)
    _grid(prefix, "plan.prefix_lens", torch.int32, (B,), index)
    path, after = new_tensor(shape, torch.int32, device), new_tensor((B,), dtype, device)
    counts, keep = torch.empty_like(prefix), torch.empty_like(prefix)
    _launch("mla_tree_accept", _lib.load().mla_tree_accept, device, mask.data_ptr(), prefix.data_ptr(), tokens.data_ptr(),
            targets.data_ptr(), int(dtype is torch.int64), B, s_q, path.data_ptr(), counts.data_ptr(), after.data_ptr(),
            keep.data_ptr())
    return Accepted(path, counts, after, keep)


def kv_keep_path(kv_cache, slots: torch.Tensor, path: torch.Tensor) -> None:
    """Move the tokens of ``path [B, s_q]`` (int32, from :func:`tree_accept`) together: cache row ``slots[b, k]`` takes
    the token of row ``slots[b, path[b, k]]``, as if all were read before any is written; in place, bit for bit, in
    every cache format.  ``slots`` is the plan's.  Entries below their own place k and slots outside the cache name
    nothing; a row that slots name twice holds one of its values afterwards.  A drafted token's position is its depth's, so what is moved needs no new rotation."""
    c, _, device = _cache_struct(kv_cache, None)
    if path.get_device() != device.index:
        _require(path, "path", device)
    _first_grid(path, "path", _INT32)
    _grid(slots, "slots", torch.int32, path.shape, device.index)
    _launch("mla_kv_keep_path", _lib.load().mla_kv_keep_path, device, ctypes.byref(c), slots.data_ptr(), path.data_ptr(),
            *path.shape)
