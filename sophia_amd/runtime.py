"""Continuous-batching runtime around the hybrid decoder.

``SlotAllocator`` hands out and takes back the cache slots that
``Transformer.forward_step`` indexes (every KDA recurrent state, conv history
and MLA latent cache has one row per slot), growing the model's caches when
all slots are taken and zeroing a slot's KDA caches when it is handed out.

``RuntimeCacheState`` and ``forward_cached_decode`` are the functional cached
decode of the reference (ml/modeling/cache_decode.py:12-143): a step takes the
tokens and the cache state the previous step returned, loads that state,
advances it and returns the logits with the new state.  The reference runs
tokens after the first step one position at a time (its model takes T > 1
only at start_pos 0, runtime_host.py:146-170); here every step is one
``forward_step``, whatever its number of tokens.

``pack_trees`` and ``verify_trees`` are greedy decoding with drafted tokens: a
server proposes a tree of continuations for each running sequence, one step runs
all of them, and the longest part that the model itself says is kept.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops
from .decoder import DraftTrees, Transformer
from .state import RuntimeCacheSnapshot


class SlotAllocator:
    """Cache slots of ``model`` for continuous batching (host bookkeeping).

    ``allocate(n)`` returns n free slots (int32, on the model's device),
    lowest numbers first, with their KDA caches zeroed; when fewer than n are
    free the model's caches grow (``Transformer.ensure_batch_capacity``, at
    least doubling).  ``release(slots)`` returns them.  Slot numbers stay
    valid for as long as they are held."""

    def __init__(self, model: Transformer) -> None:
        self.model = model
        self._capacity = int(model.runtime_batch_capacity())
        self._free = list(range(self._capacity - 1, -1, -1))
        self._held: set[int] = set()

    @property
    def capacity(self) -> int:
        return self._capacity

    @property
    def in_use(self) -> int:
        return len(self._held)

    def held(self) -> list[int]:
        return sorted(self._held)

    def allocate(self, n: int) -> torch.Tensor:
        n = int(n)
        if n < 0:
            raise ValueError(f"cannot allocate {n} slots")
        if n > len(self._free):
            grown = max(2 * self._capacity, len(self._held) + n)
            self.model.ensure_batch_capacity(grown)
            self._free = list(range(grown - 1, self._capacity - 1, -1)) + self._free
            self._capacity = grown
        taken = [self._free.pop() for _ in range(n)]
        self._held.update(taken)
        dev = self.model.tok_embeddings.weight.device
        slots = torch.tensor(taken, dtype=torch.int32, device=dev)
        if n:
            self.model.reset_slots(slots)
        return slots

    def release(self, slots) -> None:
        values = [int(s) for s in (slots.tolist() if isinstance(slots, torch.Tensor) else slots)]
        if len(set(values)) != len(values):
            raise ValueError(f"slots released twice in one call: {sorted(values)}")
        for s in values:
            if s not in self._held:
                raise ValueError(f"slot {s} is not held")
        for s in values:
            self._held.remove(s)
            self._free.append(s)
        self._free.sort(reverse=True)


@dataclass
class RuntimeCacheState:
    """A decode's cache between steps (cache_decode.py:12-16)."""

    cache: RuntimeCacheSnapshot
    batch_size: int
    cache_pos: int

    def clone(self) -> "RuntimeCacheState":
        return RuntimeCacheState(cache=self.cache.clone(), batch_size=int(self.batch_size),
                                 cache_pos=int(self.cache_pos))


def forward_cached_decode(*, model: Transformer, input_ids: torch.Tensor,
                          cache_state: RuntimeCacheState | None, start_pos: int | None,
                          logits_to_keep: int | None) -> tuple[torch.Tensor, RuntimeCacheState]:
    """One cached decode step (cache_decode.py:79-143): ``input_ids`` [B, T]
    continue the sequences held by ``cache_state`` (None: a fresh prefill,
    which needs start_pos 0 or None).  Returns (logits [B, T', vocab] -- the
    last ``logits_to_keep`` positions, all of them when it is None or 0 --,
    the new state, dumped to the host).  The same errors as the reference
    for inconsistent positions and batch sizes (ValueError)."""
    if logits_to_keep is not None and int(logits_to_keep) < 0:
        raise ValueError(f"logits_to_keep must be >= 0 when provided, got {logits_to_keep}")
    if input_ids.dim() != 2 or int(input_ids.size(1)) <= 0:
        raise ValueError("input_ids must be [B, T] with T >= 1")
    bsz, seqlen = int(input_ids.size(0)), int(input_ids.size(1))
    # Every check runs before the caches are touched or anything is launched.
    cache_pos = 0 if cache_state is None else int(cache_state.cache_pos)
    if cache_pos + seqlen > int(model.args.max_seq_len):
        raise ValueError("sequence exceeds max_seq_len")
    if cache_state is None:
        if start_pos is not None and int(start_pos) != 0:
            raise ValueError("cache_state is required when start_pos > 0 for cached decode")
        model.ensure_batch_capacity(bsz)
        model.reset_runtime_cache()
    else:
        if cache_pos < 0:
            raise ValueError(f"cache cache_pos must be >= 0, got {cache_pos}")
        if start_pos is not None and int(start_pos) != cache_pos:
            raise ValueError(f"start_pos ({start_pos}) must match cache cache_pos ({cache_pos})")
        cache_state = cache_state.clone()
        batch = int(cache_state.batch_size or bsz)
        if batch <= 0:
            raise ValueError(f"cache batch_size must be > 0, got {batch}")
        if batch != bsz:
            raise ValueError(f"cache batch_size does not match input_ids: {batch} != {bsz}")
        model.cache_load(cache_state.cache)
    dev = model.tok_embeddings.weight.device
    slots = torch.arange(bsz, dtype=torch.int32, device=dev)
    keep = 0 if logits_to_keep is None else int(logits_to_keep)
    ids = input_ids.to(dev)
    if seqlen == 1 and cache_pos > 0:
        logits = model.forward_step(decode_ids=ids[:, 0], decode_slots=slots,
                                    decode_pos=torch.full((bsz,), cache_pos, dtype=torch.long, device=dev),
                                    max_decode_len=cache_pos + 1).unsqueeze(1)
    else:
        logits = model.forward_step(prefill_ids=ids.reshape(-1), prefill_lens=[seqlen] * bsz,
                                    prefill_pos=[cache_pos] * bsz, prefill_slots=slots,
                                    all_logits=keep != 1)
        logits = logits.view(bsz, seqlen if keep != 1 else 1, -1)
    if keep > 0:
        logits = logits[:, -keep:, :]
    next_pos = cache_pos + seqlen
    return logits, RuntimeCacheState(cache=model.cache_dump(device="cpu", cache_pos=next_pos, batch_size=bsz),
                                     batch_size=bsz, cache_pos=next_pos)


def pack_trees(model: Transformer, trees, slots, cached) -> DraftTrees:
    """``DraftTrees`` on the model's device from host lists: ``trees[s]`` =
    (tokens, parents) of sequence s, node 0 its last known token (parent -1),
    each other node after its parent (an index into the tree); ``slots[s]`` its
    cache slot and ``cached[s]`` the tokens in it, to which the deepest path is
    added within max_seq_len."""
    dev = model.tok_embeddings.weight.device
    slots, cached = ([int(v) for v in (t.tolist() if isinstance(t, torch.Tensor) else t)] for t in (slots, cached))
    if not len(trees) == len(slots) == len(cached):
        raise ValueError("slots and cached need one entry per tree")
    if len(set(slots)) != len(slots):
        raise ValueError(f"two trees share a cache slot: {sorted(slots)}")
    capacity = model.runtime_batch_capacity()
    if any(not 0 <= s < capacity for s in slots):
        raise ValueError(f"cache slots must be in [0, {capacity})")
    tokens, parents, offsets = [], [], [0]
    for (toks, pars), length in zip(trees, cached):
        if len(toks) != len(pars) or not 1 <= len(toks) <= ops.TREE_NODES:
            raise ValueError(f"a tree has 1..{ops.TREE_NODES} nodes, each with a token and a parent")
        if int(pars[0]) != -1 or any(not 0 <= int(p) < i for i, p in enumerate(pars) if i):
            raise ValueError("node 0 is the root (parent -1), and every other node comes after its parent")
        if any(not 0 <= int(t) < int(model.args.vocab_size) for t in toks):
            raise ValueError("a token is outside the vocabulary")
        depth = [length + 1]
        for p in pars[1:]:
            depth.append(depth[int(p)] + 1)
        if length < 0 or max(depth) > int(model.args.max_seq_len):
            raise ValueError("cached token counts must be >= 0" if length < 0 else "sequence exceeds max_seq_len")
        tokens += [int(t) for t in toks]
        parents += [int(p) for p in pars]
        offsets.append(len(tokens))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    i64 = lambda v: torch.tensor(v, dtype=torch.int64, device=dev)  # noqa: E731
    return DraftTrees(i64(tokens), i32(offsets), i32(parents), i32(slots), i64(cached),
                      max((len(t) for t, _ in trees), default=0), max(cached, default=0))


@dataclass
class Verified:
    """The outcome of ``verify_trees``, on the device: ``path`` int32 [N,
    max_nodes] (the kept nodes, -1 behind them), ``n_path`` int32 [N],
    ``next_token`` int64 [N] (the token after the path: the next tree's node 0;
    -1: there is none, as the last node's logits are all masked or NaN, and the
    sequence ends), ``cached`` int64 [N] (tokens in the caches now), ``logits``
    [rows, vocab] of every node, adjusted."""

    path: torch.Tensor
    n_path: torch.Tensor
    next_token: torch.Tensor
    cached: torch.Tensor
    logits: torch.Tensor


def verify_trees(model: Transformer, trees: DraftTrees, **controls) -> Verified:
    """One step of greedy decoding with drafted tokens: the nodes of all trees
    through the model, their logits adjusted (``controls``: the penalties, biases
    and masks of ``ops.adjust_logits``, per sequence; allowed_rows per node;
    ``history`` holds the tokens in the caches, history_len == cached: node 0 is a
    node of every path already, and counts as generated), the drafted tokens
    walked as far as they are the model's own choices, and the caches advanced
    along that path.  A sequence gains n_path tokens in its caches, at least one,
    and knows the next: what steps over trees of one node give.  Decode steps
    (``forward_step``) round elsewhere (``Transformer.forward_tree``), so where two
    logits are closer than that, they may choose the other.  Nothing is read back
    on the host, so the step is capturable."""
    draft = model.forward_tree(trees)
    logits = draft.logits
    if controls:
        logits = ops.adjust_logits(logits, cu_nodes=trees.cu_nodes, parents=trees.parents, tokens=trees.token_ids,
                                   max_nodes=trees.max_nodes, out=logits, **controls)
    path, n_path, next_token, _ = ops.tree_accept(logits, trees.token_ids, trees.cu_nodes, trees.parents,
                                                  max_nodes=trees.max_nodes, strict=True)
    model.commit_tree(draft, path, n_path)
    return Verified(path, n_path, next_token, trees.cached + n_path, logits)


__all__ = ["RuntimeCacheState", "SlotAllocator", "Verified", "forward_cached_decode", "pack_trees", "verify_trees"]
