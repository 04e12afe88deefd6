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

``PagedLatents`` keeps the MLA layers' latents in pages that sequences can share,
and ``beam_search`` follows the best continuations of prompts in them.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops
from .decoder import DraftTrees, PagePools, SophiaMLA, Transformer
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
    model._refuse_paged(lambda: range(bsz), "forward_cached_decode")
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
    cache slot, which has no latents in pages (RuntimeError), and ``cached[s]`` the
    tokens in it, to which the deepest path is added within max_seq_len."""
    dev = model.tok_embeddings.weight.device
    slots, cached = ([int(v) for v in (t.tolist() if isinstance(t, torch.Tensor) else t)] for t in (slots, cached))
    if not len(trees) == len(slots) == len(cached):
        raise ValueError("slots and cached need one entry per tree")
    if len(set(slots)) != len(slots):
        raise ValueError(f"two trees share a cache slot: {sorted(slots)}")
    capacity = model.runtime_batch_capacity()
    if any(not 0 <= s < capacity for s in slots):
        raise ValueError(f"cache slots must be in [0, {capacity})")
    model._refuse_paged(lambda: slots, "pack_trees")
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


class PagedLatents:
    """The latents of ``model``'s MLA layers in pages (host bookkeeping, and on the
    device a pool [n_pages, page_size, kv_rank] per layer and one table).

    A slot holds pages for its tokens, in order; a page may be held by several
    slots.  ``reserve(slot, length)`` gives a slot pages of its own up to ``length``
    tokens, ``share(src, dst, length)`` makes a slot go on from the first ``length``
    tokens of another, ``release(slots)`` gives their pages back (a page is free
    when its last holder is gone), ``compact()`` moves the held pages to the lowest
    places of the pools.  ``Transformer.forward_step(pages=)`` writes and reads the
    pages, ``Transformer.fork_slots(pages=)`` moves them between slots on the device:
    the slots of such a fork may hold each other's pages afterwards, so they are
    released together, and other slots do not ``share`` theirs.  Pages that several
    slots have are read alone: no slot that has them writes below the tokens that are
    shared, neither in a step nor by a fork into it.  What works on the slots'
    own caches refuses a slot that holds pages: drafted steps, cached decoding,
    ``cache_dump`` and ``cache_load`` with latents.

    ``dtype``: of the pages, that of the model's activations (default: of its
    embedding).  ``max_len``: tokens of a slot at most (default: max_seq_len)."""

    def __init__(self, model: Transformer, n_pages: int, *, page_size: int = 64, max_len: int | None = None,
                 dtype: torch.dtype | None = None) -> None:
        n_pages, page_size = int(n_pages), int(page_size)
        if n_pages < 1 or not 1 <= page_size <= 65536 or page_size & (page_size - 1):
            raise ValueError(f"n_pages must be >= 1 and page_size a power of two up to 65536, got {n_pages} and {page_size}")
        args = model.args
        rank, q_rank = int(args.mla_kv_rank), int(args.mla_q_rank)
        if rank not in (32, 64, 128, 256) or q_rank % 8 or q_rank + rank > 512:
            raise ValueError("paged latents need mla_kv_rank 32, 64, 128 or 256 and mla_q_rank a multiple of 8, together at most 512")
        weight = model.tok_embeddings.weight
        self.device, self.page_size, self.n_pages = weight.device, page_size, n_pages
        longest = int(args.max_seq_len) if max_len is None else int(max_len)
        if longest < 1:
            raise ValueError(f"max_len must be >= 1, got {longest}")
        self._width = -(-longest // page_size)
        self.max_len = self._width * page_size
        dt = weight.dtype if dtype is None else dtype
        self.pools = {m: torch.zeros(n_pages, page_size, rank, dtype=dt, device=self.device)
                      for m in model.modules() if isinstance(m, SophiaMLA)}
        self.table = torch.full((int(model.runtime_batch_capacity()), self._width), -1, dtype=torch.int32, device=self.device)
        self._free = list(range(n_pages - 1, -1, -1))
        self._holders = [0] * n_pages
        self._held: dict[int, dict[int, int]] = {}     # of a slot: place in its row -> page
        if getattr(model, "_page_pools", None) is None:      # (a model pickled as a whole before there were any)
            model._page_pools = PagePools()
        model._page_pools.add(self)

    @property
    def slots(self) -> list[int]:
        """The slots that hold pages: whose latents are here."""
        return sorted(self._held)

    @property
    def pages_free(self) -> int:
        return len(self._free)

    def held(self, slot: int) -> list[int]:
        """The pages of a slot, in the order of its tokens."""
        return [p for _, p in sorted(self._held.get(int(slot), {}).items())]

    def ensure_slots(self, n: int) -> None:
        """Rows of the table for slots 0 .. n - 1 (the old ones stay valid, the table is a new
        tensor: a step captured before has the old one, as after growth of the caches)."""
        if int(n) > int(self.table.size(0)):
            grown = self.table.new_full((int(n), self._width), -1)
            grown[: self.table.size(0)].copy_(self.table)
            self.table = grown

    def _places(self, length: int) -> int:
        length = int(length)
        if not 0 <= length <= self.max_len:
            raise ValueError(f"a slot holds at most {self.max_len} tokens, got {length}")
        return -(-length // self.page_size)

    def _set(self, slot: int, places: dict[int, int]) -> None:
        if places:
            at = torch.tensor(list(places), dtype=torch.int64).to(self.device)
            self.table[slot, at] = torch.tensor(list(places.values()), dtype=torch.int32).to(self.device)
            self._held.setdefault(slot, {}).update(places)

    def reserve(self, slot: int, length: int, *, first: int = 0) -> None:
        """Pages of its own for the tokens first .. length - 1 of ``slot``, where it
        has none (all or nothing: RuntimeError where fewer are free).  ``first``: the
        tokens before are to come from other slots (``fork_slots``)."""
        slot = int(slot)
        if slot < 0:
            raise ValueError(f"slots are >= 0, got {slot}")
        end, begin = self._places(length), min(int(first), int(length)) // self.page_size
        if int(first) < 0:
            raise ValueError(f"first must be >= 0, got {first}")
        missing = [j for j in range(begin, end) if j not in self._held.get(slot, {})]
        if len(missing) > len(self._free):
            raise RuntimeError(f"{len(missing)} pages needed, {len(self._free)} free")
        self.ensure_slots(slot + 1)
        places = {}
        for j in missing:
            places[j] = self._free.pop()
            self._holders[places[j]] = 1
        self._set(slot, places)

    def share(self, src: int, dst: int, length: int) -> None:
        """Slot ``dst``, which holds no pages, goes on from the first ``length`` tokens of
        ``src``: it holds the pages that these fill too, and a copy of the one that they fill
        in part.  (The latents alone: KDA states are moved by ``fork_slots``, or are those of
        a prompt's ``cache_dump(latents=False)`` at that length.)  ``src`` has the pages that it was given:
        ValueError where a fork on the device has put others in their places."""
        src, dst, places = int(src), int(dst), self._places(length)
        if src < 0 or dst < 0:
            raise ValueError(f"slots are >= 0, got {src} and {dst}")
        if self._held.get(dst):
            raise ValueError(f"slot {dst} holds pages")
        have = self._held.get(src, {})
        if any(j not in have for j in range(places)):
            raise ValueError(f"slot {src} holds fewer than {length} tokens")
        if places and self.table[src, :places].tolist() != [have[j] for j in range(places)]:
            raise ValueError(f"slot {src} has pages of other slots, from a fork")
        full = int(length) // self.page_size
        if places > full and not self._free:
            raise RuntimeError("1 page needed, 0 free")
        self.ensure_slots(dst + 1)
        new = {j: have[j] for j in range(full)}
        for p in new.values():
            self._holders[p] += 1
        if places > full:
            new[full] = self._free.pop()
            self._holders[new[full]] = 1
            self._copy([have[full]], [new[full]])
        self._set(dst, new)

    def release(self, slots) -> None:
        """Gives back what ``slots`` hold (each of them once)."""
        values = [int(s) for s in (slots.tolist() if isinstance(slots, torch.Tensor) else slots)]
        if len(set(values)) != len(values):
            raise ValueError(f"slots released twice in one call: {sorted(values)}")
        values = [s for s in values if s in self._held]
        for s in values:
            for p in self._held.pop(s).values():
                self._holders[p] -= 1
                if self._holders[p] == 0:
                    self._free.append(p)
        self._free.sort(reverse=True)
        if values:
            self.table.index_fill_(0, torch.tensor(values, dtype=torch.int64).to(self.device), -1)

    def compact(self) -> int:
        """Moves pages so that the held ones are the first of the pools, and names them anew
        in all rows; returns how many are held.  Page ids read before are void."""
        count = self.n_pages - len(self._free)
        src = [p for p in range(count, self.n_pages) if self._holders[p]]
        dst = [p for p in range(count) if not self._holders[p]]
        if not src:
            return count
        self._copy(src, dst)
        names = torch.arange(self.n_pages, dtype=torch.int32)
        names[torch.tensor(src)] = torch.tensor(dst, dtype=torch.int32)
        moved = dict(zip(src, dst))
        names = names.to(self.device)
        self.table.copy_(torch.where(self.table >= 0, names[self.table.clamp(min=0).long()], self.table))
        for places in self._held.values():
            for j, p in places.items():
                places[j] = moved.get(p, p)
        for s, d in moved.items():
            self._holders[d], self._holders[s] = self._holders[s], 0
        self._free = list(range(self.n_pages - 1, count - 1, -1))
        return count

    def _copy(self, src: list[int], dst: list[int]) -> None:
        for i in range(0, len(src), ops.MOVES):      # (none of the places is a source)
            pair = [torch.tensor(t[i:i + ops.MOVES], dtype=torch.int32).to(self.device) for t in (src, dst)]
            pools = list(self.pools.values())
            for j in range(0, len(pools), ops.POOLS):
                ops.page_copy(*pair, pools[j:j + ops.POOLS])


@dataclass
class Beams:
    """The outcome of ``beam_search``, on the device, the best beam first: ``tokens``
    int64 [N, beams, max_new] (``pad_token`` behind an end, -1 in beams that there
    are not), ``scores`` fp32 [N, beams] (log probabilities; -inf: no such beam),
    ``ended`` bool [N, beams] (by an end token)."""

    tokens: torch.Tensor
    scores: torch.Tensor
    ended: torch.Tensor


@torch.no_grad()
def beam_search(model: Transformer, slots: SlotAllocator, pages: PagedLatents, prompts, *, beams: int, max_new: int,
                end_token: int | None = None, pad_token: int = 0, adjust=None) -> Beams:
    """The ``beams`` most probable continuations of each prompt that are found by going on
    from the ``beams`` best at every token (``max_new`` of them, or up to ``end_token``).

    ``prompts``: token lists (or 1-d tensors) of any lengths.  All beams of a prompt share
    its pages; each has pages of its own for what it generates.  ``pad_token``, any number, fills
    the output behind an end.  ``adjust(logits, tokens)``, if given, returns the logits [rows, vocab]
    to choose by, for the tokens [rows, t] generated so far, pads behind ends among them
    (``ops.adjust_logits``).  The slots and pages that it takes are given back.  After the
    prompts nothing is read back on the host."""
    prompts = [[int(t) for t in (p.tolist() if isinstance(p, torch.Tensor) else p)] for p in prompts]
    B, N, max_new = int(beams), len(prompts), int(max_new)
    if N == 0 or any(not p for p in prompts):
        raise ValueError("prompts must hold a token each at least")
    if any(not 0 <= t < int(model.args.vocab_size) for p in prompts for t in p):
        raise ValueError("a token is outside the vocabulary")
    if not 1 <= B <= ops.BEAMS or max_new < 1 or N * B > ops.MOVES:
        raise ValueError(f"beams must be in [1, {ops.BEAMS}], max_new >= 1 and the beams of all prompts at most {ops.MOVES}")
    lens = [len(p) for p in prompts]
    longest = max(lens) + max_new - 1           # (the last token is chosen, and goes into no cache)
    if longest > min(int(model.args.max_seq_len), pages.max_len):
        raise ValueError("sequence exceeds max_seq_len")
    dev = pages.device
    taken = slots.allocate(N * B)
    mine = [int(s) for s in taken.tolist()]
    try:
        for i, s in enumerate(mine):
            n = lens[i // B]
            pages.reserve(s, n + max_new - 1, first=0 if i % B == 0 else n)
        own = taken.view(N, B)
        at = torch.tensor(lens, dtype=torch.int64).to(dev).repeat_interleave(B)       # tokens in the caches of each beam
        ids = torch.tensor([t for p in prompts for t in p], dtype=torch.int64).to(dev)
        logits = model.forward_step(prefill_ids=ids, prefill_lens=lens, prefill_pos=[0] * N, prefill_slots=own[:, 0].contiguous(),
                                    pages=pages)
        history = torch.empty((N, 1, 0), dtype=torch.int64, device=dev)
        scores, ended, width = torch.zeros(N, dtype=torch.float32, device=dev), None, 1
        for t in range(max_new):
            if adjust is not None:
                shape = logits.shape
                logits = adjust(logits, history.reshape(N * width, t))
                if logits.shape != shape:
                    raise ValueError(f"adjust must return logits {list(shape)}, got {list(logits.shape)}")
            scores, parent, token = ops.beam_select(logits, scores.reshape(-1), width, keep=B, ended=ended, pad_token=pad_token)
            kept = parent.long().clamp(min=0)
            history = torch.cat([torch.gather(history, 1, kept[:, :, None].expand(N, B, t)), token[:, :, None]], 2)
            was = torch.zeros((N, B), dtype=torch.bool, device=dev) if ended is None else torch.gather(ended.view(N, width), 1, kept)
            done = was if end_token is None else was | (token == int(end_token))
            history[:, :, t] = torch.where(was, int(pad_token), history[:, :, t])
            ended, width = done.reshape(-1).contiguous(), B
            if t + 1 == max_new:
                break
            src = torch.where(parent >= 0, torch.gather(own, 1, kept), -1).reshape(-1).contiguous()
            model.fork_slots(src, taken, at, pages=pages)
            # (ended beams and places without a beam have a token of the vocabulary run, whose logits nobody reads)
            ids = torch.where(done, 0, token.clamp(min=0)).reshape(-1)
            logits = model.forward_step(decode_ids=ids, decode_slots=taken, decode_pos=at, max_decode_len=longest, pages=pages)
            at = at + 1
        tokens = torch.where(torch.isinf(scores)[:, :, None], -1, history)
        return Beams(tokens, scores, ended.view(N, B) & ~torch.isinf(scores))
    finally:
        pages.release(mine)
        slots.release(mine)


__all__ = ["Beams", "PagedLatents", "RuntimeCacheState", "SlotAllocator", "Verified", "beam_search", "forward_cached_decode",
           "pack_trees", "verify_trees"]
