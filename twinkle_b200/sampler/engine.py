"""Native generation engine: paged KV cache + continuous batched decode on the owned decoder.

Fills the role vLLM plays for the reference (``src/twinkle/sampler/vllm_sampler/vllm_engine.py:47-863``):
per-token logprobs of the *processed* distribution (after temperature / top-k / top-p), prompt logprobs
and their top-k for distillation, ``max_tokens = 0`` scoring, stop tokens / strings, per-request LoRA (a
batch may mix adapters — the segmented LoRA kernel serves them in one launch), routed-expert capture for
MoE router replay, weight updates from tensors (no reload).

Prefill runs the training forward kernels (varlen flash attention) with a sink that writes K/V into the
paged cache; decode runs one token per live sequence through ``ops.paged_attention_decode``.
"""
from __future__ import annotations

import math
import os
from dataclasses import dataclass, field
from typing import Any, Callable, Dict, Iterator, List, Optional, Sequence, Tuple

import torch

from .. import ops
from ..data_format import SampledSequence, SampleResponse, SamplingParams
from ..models.config import DecoderConfig
from ..models.decoder import DecoderModel, PackedBatch
from ..models.layers import LoraBatch, lora_batch
from ..models.parallel_layer import CacheView


class PagedKVCache:
    """Per layer K and V pools ``[num_blocks, block_size, Hkv, width]`` (key and value rows have the layer's own widths; latent
    attention keeps one row that serves as both, layers that keep nothing per token have no pool) + a free list.  Layers with a
    short convolution in front of attention also have a history pool ``[num_slots, taps − 1, channels]``, recurrent layers an
    fp32 state pool ``[num_slots, heads, dim, vdim]``; a sequence owns one slot of all of them.  Block 0 and slot 0 are never
    handed out so that the all-zero rows that fill up a captured batch are harmless."""

    def __init__(self, cfg: DecoderConfig, num_blocks: int, block_size: int, device, dtype, num_slots: int = 0):
        self.cfg, self.block_size, self.num_blocks, self.device, self.dtype = cfg, block_size, num_blocks, device, dtype
        self.num_slots = num_slots if any(cfg.conv_layout()) or any(cfg.state_layout()) else 0
        self.build()

    def build(self) -> None:
        """(Re)create empty pools and free lists."""
        mk = lambda *shape: torch.zeros(shape, device=self.device, dtype=self.dtype)  # noqa: E731
        layout = self.cfg.kv_layout()
        self.k = [mk(self.num_blocks, self.block_size, h, d) if h * d else None for h, d, _ in layout]
        self.v = [mk(self.num_blocks, self.block_size, h, e) if h * e else None for h, _, e in layout]
        none = [None] * len(layout)
        self.conv = [mk(self.num_slots, *c) if c else None for c in self.cfg.conv_layout() or none]
        self.state = [torch.zeros(self.num_slots, *c, device=self.device) if c else None for c in self.cfg.state_layout() or none]
        self.free: List[int] = list(range(self.num_blocks - 1, 0, -1))
        self.sharers: Dict[int, int] = {}          # blocks with several owners → owners beyond the first
        self.free_slots: List[int] = list(range(self.num_slots - 1, 0, -1))

    def drop(self) -> None:
        """Give the pools' memory back (``build`` makes new ones)."""
        self.k = self.v = self.conv = self.state = None

    @staticmethod
    def block_bytes(cfg: DecoderConfig, block_size: int, elem: int) -> int:
        return elem * block_size * sum(h * (d + e) for h, d, e in cfg.kv_layout())

    @staticmethod
    def slot_bytes(cfg: DecoderConfig, elem: int) -> int:
        return elem * sum(math.prod(c) for c in cfg.conv_layout() if c) + 4 * sum(math.prod(c) for c in cfg.state_layout() if c)

    def allocate_slot(self) -> int:
        if not self.num_slots:
            return 0
        if not self.free_slots:
            raise RuntimeError(f'per-sequence state exhausted: {self.num_slots - 1} sequences are live')
        return self.free_slots.pop()

    def release_slot(self, slot: int) -> None:
        if slot:
            self.free_slots.append(slot)

    def allocate(self, n: int) -> List[int]:
        if n > len(self.free):
            raise RuntimeError(f'KV cache exhausted: need {n} blocks, {len(self.free)} free')
        return [self.free.pop() for _ in range(n)]

    def release(self, blocks: Sequence[int]) -> None:
        """Give an owner's blocks back; one with other owners stays theirs."""
        if self.sharers:
            mine, blocks = blocks, []
            for b in mine:
                left = self.sharers.get(b, 0)
                if left > 1:
                    self.sharers[b] = left - 1
                elif left:
                    del self.sharers[b]
                else:
                    blocks.append(b)
        self.free.extend(reversed(list(blocks)))

    def fork(self, blocks: Sequence[int], n_tokens: int, n_blocks: Sequence[int]) -> Tuple[List[List[int]], List[Tuple[int, int, int]]]:
        """Block lists of ``n_blocks[i]`` blocks each for continuations of a sequence whose first ``n_tokens`` tokens lie in ``blocks``: they
        share its full blocks and own the rest.  Beside them the copies ``(from, to, tokens)`` that put the tokens of the last, partly filled block where each
        continues it (``copy``)."""
        full, rest = divmod(n_tokens, self.block_size)
        own = self.allocate(sum(max(n, full + (rest > 0)) - full for n in n_blocks))
        lists, copies, at = [], [], 0
        for n in n_blocks:
            mine = own[at:at + max(n, full + (rest > 0)) - full]
            at += len(mine)
            lists.append(list(blocks[:full]) + mine)
            if rest:
                copies.append((blocks[full], mine[0], rest))
        for b in blocks[:full]:
            self.sharers[b] = self.sharers.get(b, 0) + len(n_blocks)
        return lists, copies

    def copy(self, copies: Sequence[Tuple[int, int, int]], slots: Sequence[Tuple[int, int]] = ()) -> None:
        """Tokens of blocks ``(from, to, tokens)`` in all layers' pools, and rows ``(from, to)`` of the history and state pools."""
        if copies:
            ops.cache_copy(self.k + self.v, *zip(*copies))
        if slots and self.num_slots:
            ops.cache_copy(self.conv + self.state, *zip(*slots))

    def compact(self, lists: Sequence[List[int]], num_blocks: Optional[int] = None) -> None:
        """Move the blocks of all live sequences, whose lists are given and renumbered in place, to the front of the pools; with ``num_blocks`` the pools are
        then replaced by ones of that many blocks."""
        live = {b for blocks in lists for b in blocks}
        if len(live) + len(self.free) != self.num_blocks - 1 or live & set(self.free):
            raise RuntimeError(f'{self.num_blocks - 1 - len(self.free)} blocks are in use, the lists name {len(live)}')
        if num_blocks is not None and num_blocks <= len(live):
            raise RuntimeError(f'{len(live)} live blocks do not fit a cache of {num_blocks}')
        holes = [b for b in range(1, len(live) + 1) if b not in live]
        place = dict(zip(sorted((b for b in live if b > len(live)), reverse=True), holes))
        self.copy([(b, to, self.block_size) for b, to in place.items()])
        for blocks in lists:
            blocks[:] = [place.get(b, b) for b in blocks]
        self.sharers = {place.get(b, b): n for b, n in self.sharers.items()}
        if num_blocks is not None and num_blocks != self.num_blocks:
            kept = len(live) + 1
            for pools in (self.k, self.v):
                for i, old in enumerate(pools):
                    if old is not None:
                        pools[i] = torch.zeros((num_blocks, ) + old.shape[1:], device=old.device, dtype=old.dtype)
                        pools[i][:kept] = old[:kept]
            self.num_blocks = num_blocks
        self.free = list(range(self.num_blocks - 1, len(live), -1))

    def blocks_for(self, n_tokens: int) -> int:
        return (n_tokens + self.block_size - 1) // self.block_size


@dataclass
class _Seq:
    request: int
    prompt: List[int]
    params: SamplingParams
    slot: int = -1          # LoRA slot (−1 = base)
    lora_rank: int = 0
    lora_scale: float = 0.0
    lora_target: Any = None
    blocks: List[int] = field(default_factory=list)
    state_slot: int = 0     # row of the convolution-history and state pools
    tokens: List[int] = field(default_factory=list)
    logprobs: List[float] = field(default_factory=list)
    topk: List[List[Tuple[int, float]]] = field(default_factory=list)
    done: bool = False
    stop_reason: str = 'length'
    generator: Optional[torch.Generator] = None
    routed: Optional[List[torch.Tensor]] = None
    text_tail: str = ''
    vision: Optional[Dict[str, Any]] = None   # pixel_values, image_grid_thw, mrope_position_ids [3, L] of a prompt with images
    rope_delta: int = 0                        # rotary position − token index for the tokens after the prompt (images compress positions)
    linear: Dict[int, Tuple[torch.Tensor, torch.Tensor]] = field(default_factory=dict)  # layer → (conv rows, recurrent state) of linear-attention layers
    origin: Optional['_Seq'] = field(default=None, compare=False, repr=False)    # the sequence whose prompt this one shares (itself: others share its own)

    @property
    def length(self) -> int:
        return len(self.prompt) + len(self.tokens)


class NativeEngine:

    def __init__(self, model: DecoderModel, cfg: DecoderConfig, device=None, num_blocks: Optional[int] = None, block_size: int = 16,
                 max_batch: int = 256, gpu_memory_utilization: float = 0.85, decode: Optional[Callable[[List[int]], str]] = None, share_prompts: bool = False):
        """``share_prompts``: sequences with the same prompt (the samples of a request, repeated prompts) run through it once, share its full cache
        blocks and read them once per step.  Results then differ by the rounding of other tile shapes and orders of sums."""
        self.model, self.cfg, self.share_prompts = model, cfg, share_prompts
        # Shared pages are read once per step where that is expected to take this much less time than reading them per sequence (``ops.shared_times``); 0: wherever there are any
        self.share_from = 1.0
        self._share_captured = True            # until such a step could not be captured
        self._plan: Tuple[Any, Optional[ops.SharedPrefix]] = (None, None)      # of the last step with shared prompts
        self.device = device or next(model.parameters()).device
        if share_prompts and self.device.type == 'cuda' and not hasattr(ops.ext(), 'cache_copy'):
            raise RuntimeError("share_prompts: this process runs on a serving subset without the part 'sharing' (ops.build.prefer_serving)")
        self.dtype = next(model.parameters()).dtype
        if num_blocks is None:
            elem = 2 if self.dtype != torch.float32 else 4
            per_block = PagedKVCache.block_bytes(cfg, block_size, elem)
            if self.device.type == 'cuda' and per_block:
                free, _ = torch.cuda.mem_get_info(self.device)
                free = free * gpu_memory_utilization * 0.9 - (max_batch + 1) * PagedKVCache.slot_bytes(cfg, elem)
                num_blocks = max(int(free // per_block), 64)
            else:
                num_blocks = 1024
        self.cache = PagedKVCache(cfg, num_blocks, block_size, self.device, self.dtype, num_slots=max_batch + 1)
        self.max_batch = max_batch
        self.decode_text = decode
        self.capture_routing = False
        self.use_cuda_graphs = bool(int(os.environ.get('TWINKLE_SAMPLER_CUDA_GRAPHS', '1')))
        self._graphs: Dict[Tuple[int, int], Dict[str, Any]] = {}

    # --------------------------------------------------------------- LoRA
    def _lora_for(self, seqs: Sequence[_Seq], lens: Sequence[int]) -> Optional[LoraBatch]:
        if all(s.slot < 0 for s in seqs):
            return None
        segs, lo = [], 0
        for s, n in zip(seqs, lens):
            segs.append((lo, lo + n, s.slot, s.lora_rank, s.lora_scale))
            lo += n
        return LoraBatch(segs, self.device, [s.lora_target for s in seqs])

    # -------------------------------------------------- what a sequence holds
    def admit(self, seqs: Sequence[_Seq]) -> None:
        """Blocks for the prompt, the tokens it may generate and one more, and a slot for convolution history and state."""
        for s in seqs:
            s.blocks = self.cache.allocate(self.cache.blocks_for(len(s.prompt) + (s.params.max_tokens or 0) + 1))
            s.state_slot = self.cache.allocate_slot()

    def fork(self, origin: _Seq, seqs: Sequence[_Seq]) -> None:
        """Let ``seqs`` continue the prompt of ``origin``, which has run: its full blocks are shared, the rest and the state are copied (a state that has gone beyond the prompt cannot be)."""
        who = lambda s: (s.prompt, s.slot, s.lora_rank, s.lora_scale, s.lora_target)  # noqa: E731
        if not origin.blocks or len({id(s) for s in seqs}) < len(seqs) or any(who(s) != who(origin) or s.blocks or s.tokens for s in seqs):
            raise ValueError('fork: a sequence that has run, and others that have not, each once, with its prompt and adapter')
        if origin.tokens and (origin.state_slot or origin.linear):
            raise ValueError(f'fork: the state of the sequence has seen {len(origin.tokens)} tokens behind its prompt')
        if self.cache.num_slots and len(seqs) > len(self.cache.free_slots):
            raise RuntimeError(f'per-sequence state exhausted: {len(seqs)} forks, {len(self.cache.free_slots)} slots')
        self._fork(origin, seqs)

    def _fork(self, origin: _Seq, seqs: Sequence[_Seq]) -> None:
        lists, copies = self.cache.fork(origin.blocks, len(origin.prompt), [self.cache.blocks_for(len(s.prompt) + (s.params.max_tokens or 0) + 1) for s in seqs])
        slots = []
        for s, blocks in zip(seqs, lists):
            s.blocks, s.state_slot, s.origin = blocks, self.cache.allocate_slot(), origin
            s.linear, s.rope_delta, s.routed = dict(origin.linear), origin.rope_delta, None if origin.routed is None else [r[:len(origin.prompt)] for r in origin.routed]
            if s.state_slot:
                slots.append((origin.state_slot, s.state_slot))
        origin.origin = origin
        self.cache.copy(copies, slots)

    def compact(self, seqs: Sequence[_Seq], num_blocks: Optional[int] = None) -> None:
        """Bring the blocks of all live sequences together at the front of the cache; with ``num_blocks`` the cache is given that size."""
        self.cache.compact([s.blocks for s in seqs], num_blocks)
        if num_blocks is not None:
            self._graphs.clear()          # captured steps hold the addresses of the pools

    def _shared(self, seqs: Sequence[_Seq], rows: int, captured: bool = False) -> Optional[ops.SharedPrefix]:
        """The plan of a step whose sequences share prompts (None: nothing to share), filled up to ``rows`` sequences; ``captured``: with room for others in a
        captured step."""
        if not self.share_prompts or self.cfg.layer_specs is not None or not any(s.origin is not None for s in seqs):
            return None
        sizes, blocks, last = [], [], None
        for s in seqs:
            if s.origin is not None and s.origin is last:
                sizes[-1] += 1
            else:
                sizes.append(1)
                blocks.append(len(s.prompt) // self.cache.block_size if s.origin is not None else 0)
            last = s.origin
        blocks = [b if n > 1 else 0 for n, b in zip(sizes, blocks)]
        heads, kv_heads = self._heads()
        if not any(blocks):
            return None
        # which way is faster changes with the answers' lengths, but slowly; and with the room that they have
        widest, longest = max(len(s.blocks) for s in seqs), max(s.length for s in seqs)
        key = (tuple(sizes), tuple(blocks), rows, captured, self.share_from, widest, longest >> 8)
        if self._plan[0] != key:
            bs, plan = self.cache.block_size, None
            own = [s.length - b * bs for s, b in zip(seqs, (b for n, b in zip(sizes, blocks) for _ in range(n)))]
            if not self.share_from or self._pays(sizes, blocks, own, bs << max(widest - 1, 0).bit_length(), captured):
                sizes, blocks = sizes + [1] * (rows - len(seqs)), blocks + [0] * (rows - len(seqs))
                most = max(len(s.blocks) - b for s, b in zip(seqs, (b for n, b in zip(sizes, blocks) for _ in range(n)))) * bs
                plan = ops.shared_prefix(sizes, blocks, bs, heads, kv_heads, self.device, own=most)
                if captured:      # room in steps, so that the plans of a shrinking batch take the same graphs; a call's workspace goes by it
                    room = min(ops.prefix_items(rows, kv_heads, self.device, heads // kv_heads), max(16, 1 << (plan.items - 1).bit_length()))
                    plan = ops.shared_prefix(sizes, blocks, bs, heads, kv_heads, self.device, room, most)
            self._plan = key, plan
        return self._plan[1]

    def _pays(self, sizes: Sequence[int], blocks: Sequence[int], own: Sequence[int], room: int, captured: bool) -> bool:
        """Whether a step of these groups is expected to be faster with shared pages read once; never where the kernel does not take the cache.  An eager step, whose time is mostly the
        host's, has to save the 9 us that the call takes longer there (20 against 11)."""
        (heads, kv_heads), (_, width, value) = self._heads(), self.cfg.kv_layout()[0]
        if self.dtype != torch.bfloat16 or width not in (64, 128) or value != width or self.cache.block_size % 8:
            return False
        together, apart = ops.shared_times(sizes, blocks, own, self.cache.block_size, heads, kv_heads, width, room, self.device)
        return apart > self.share_from * together + (0.0 if captured else 9.0)

    def _heads(self) -> Tuple[int, int]:
        return self.cfg.num_attention_heads, self.cfg.kv_layout()[0][0]

    def grow(self, seqs: Sequence[_Seq]) -> None:
        """Extend the block list of sequences whose next token crosses a block boundary."""
        for s in seqs:
            need = self.cache.blocks_for(s.length + 1) - len(s.blocks)
            if need > 0:
                s.blocks += self.cache.allocate(need)

    def release(self, seqs: Sequence[_Seq]) -> None:
        for s in seqs:
            self.cache.release(s.blocks)
            self.cache.release_slot(s.state_slot)
            s.blocks, s.state_slot, s.linear, s.origin = [], 0, {}, None

    def _prompt_rows(self, seqs: Sequence[_Seq], lens: Sequence[int]) -> torch.Tensor:
        """Rows of the cache pools for packed prompts ``[ΣL]``, listed on the host and copied once."""
        bs = self.cache.block_size
        if self.device.type == 'cuda':
            return ops.ext().prompt_rows([s.blocks for s in seqs], lens, bs, True).to(self.device, non_blocking=True)
        return torch.tensor([s.blocks[p // bs] * bs + p % bs for s, n in zip(seqs, lens) for p in range(n)], dtype=torch.int64, device=self.device)

    def _prompt_view(self, seqs: Sequence[_Seq], lens: Sequence[int]) -> CacheView:
        """Cache places of packed prompts: one row per token, built on the host and copied once."""
        bs = self.cache.block_size
        rows, slots, left = [], [], []
        for s, n in zip(seqs, lens):
            rows += [s.blocks[p // bs] * bs + p % bs for p in range(n)]
            slots += [s.state_slot] * n
            left += range(n - 1, -1, -1)
        mk = lambda x, dt: torch.tensor(x, dtype=dt).to(self.device, non_blocking=True)  # noqa: E731
        return CacheView(self.cache, mk(rows, torch.int64), mk(slots, torch.int32), mk(left, torch.int32))

    # ------------------------------------------------------------- prefill
    @torch.no_grad()
    def prefill(self, seqs: List[_Seq]) -> torch.Tensor:
        """Runs all prompts as one packed row; fills the KV cache; returns the final-norm hidden state of
        every prompt token ``[ΣL, H]`` (the caller picks last tokens / scores prompts)."""
        lens = [len(s.prompt) for s in seqs]
        ids = torch.tensor([t for s in seqs for t in s.prompt], dtype=torch.long, device=self.device)
        pos = torch.cat([torch.arange(n, device=self.device) for n in lens])
        bounds = [0]
        for n in lens:
            bounds.append(bounds[-1] + n)
        cu = torch.tensor(bounds, dtype=torch.int32, device=self.device)
        self.admit(seqs)
        rows: List[torch.Tensor] = []       # places of all tokens, when a layer wants them

        def sink(layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
            if not rows:
                rows.append(self._prompt_rows(seqs, lens))
            ops.cache_write(self.cache.k[layer], self.cache.v[layer], rows[0], k, v)

        def linear_state(layer: int, conv: torch.Tensor, state: torch.Tensor) -> None:  # hybrid stacks: what decode continues from
            for i, s in enumerate(seqs):
                s.linear[layer] = (conv[i], state[i])

        sink.linear_state = linear_state
        batch = PackedBatch(ids, pos, cu, max(lens))
        if self.cfg.layer_specs is not None:
            batch.cache = self._prompt_view(seqs, lens)
        if any(s.vision for s in seqs):  # prompts with images: patches, grids and (time, height, width) positions beside the row
            p3, pix, grids = [], [], []
            for s, n in zip(seqs, lens):
                if s.vision:
                    m = torch.as_tensor(s.vision['mrope_position_ids']).long()
                    pix.append(torch.as_tensor(s.vision['pixel_values']))
                    grids.append(torch.as_tensor(s.vision['image_grid_thw']).long().view(-1, 3))
                    s.rope_delta = int(m.max()) + 1 - n
                else:
                    m = torch.arange(n).expand(3, -1)
                p3.append(m)
            batch.position_ids = torch.cat(p3, 1).to(self.device)
            batch.pixel_values = torch.cat(pix, 0).to(self.device, self.dtype)
            batch.image_grid_thw = torch.cat(grids, 0).to(self.device)
        self.model.set_record_routing(self.capture_routing)
        with lora_batch(self._lora_for(seqs, lens)):
            hidden = self.model(batch, kv_sink=sink)
        if self.capture_routing:
            routed = self.model.collect_routed_experts()
            if routed is not None:
                for s, a, b in zip(seqs, bounds[:-1], bounds[1:]):
                    s.routed = [r[a:b].cpu() for r in routed]
        return hidden

    # --------------------------------------------------------------- decode
    def _decode_body(self, tokens, positions, table, seq_lens, lora: Optional[LoraBatch], seqs: Optional[List[_Seq]] = None,
                     rope_positions: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None, prefix: Optional[ops.SharedPrefix] = None) -> torch.Tensor:
        """One decode token per row from device tensors only (what a CUDA graph captures). Linear-attention layers of
        hybrid stacks keep their state on the sequences (``seqs``) and always run eagerly."""
        cfg, B = self.cfg, tokens.shape[0]
        if cfg.layer_specs is not None:      # one forward serves prompts and steps: the view tells the layers which it is
            bs = self.cache.block_size
            rows = table.gather(1, (positions // bs).unsqueeze(1)).squeeze(1).long() * bs + positions % bs
            batch = PackedBatch(tokens, positions, None, 1, cache=CacheView(self.cache, rows, slots, torch.zeros_like(slots), table, seq_lens))
            with lora_batch(lora):
                return self.model.logits(self.model(batch)).float()
        # ``positions`` index the KV cache; the rotary position differs from it after a prompt with images
        cos, sin = ops.rope_tables(positions if rope_positions is None else rope_positions, cfg.rotary_dim, cfg.rope_theta, cfg.rope_scaling)
        local = None
        if cfg.rope_local_theta:       # sliding-window layers of Gemma-3 rotate with a base of their own
            local = ops.rope_tables(positions if rope_positions is None else rope_positions, cfg.rotary_dim, cfg.rope_local_theta, None)
        x = self.model.embed_ids(tokens)
        bs = self.cache.block_size
        rows = table.gather(1, (positions // bs).unsqueeze(1)).squeeze(1).long() * bs + positions % bs
        with lora_batch(lora):
            for li, layer in enumerate(self.model.layers):
                at = layer.self_attn
                h = layer.pre(x)
                if getattr(layer, 'is_linear', False):
                    conv = torch.stack([s.linear[li][0] for s in seqs])
                    st = torch.stack([s.linear[li][1] for s in seqs])
                    y, conv, st = at.step(h, conv, st)
                    for i, s in enumerate(seqs):
                        s.linear[li] = (conv[i], st[i])
                    n, x = layer.after_attention(x, y)
                    x = x + layer.feed_forward(n)
                    continue
                q, k, v, gate = at.heads_from(h, *(local if (local is not None and getattr(at, 'local_rope', False)) else (cos, sin)))
                ops.cache_write(self.cache.k[li], self.cache.v[li], rows, *at.cache_entry(k, v))
                extras = {n: getattr(at, n, None) for n in ('window', 'softcap', 'sinks')}
                if prefix is not None and q.shape[1] == prefix.heads and self.cache.k[li].shape[2] == prefix.kv_heads and not extras['window'] and not extras['softcap'] and extras['sinks'] is None:
                    o = ops.paged_attention_shared(q, self.cache.k[li], self.cache.v[li], table, seq_lens, prefix, at.scale)
                else:
                    o = ops.paged_attention_decode(q, self.cache.k[li], self.cache.v[li], table, seq_lens, at.scale, **extras)
                n, x = layer.after_attention(x, at.project_out(o, gate))
                x = x + layer.feed_forward(n)
            x = self.model.norm(x)
        return self.model.logits(x).float()

    def _graph_for(self, B: int, max_blocks: int, prefix: Optional[ops.SharedPrefix] = None):
        """A captured decode step for batch bucket ``B`` and block-table width ``max_blocks`` (both powers of two); with ``prefix`` one that reads shared prompts by a plan in static
        memory, for plans of the same room that the kernels are laid out for alike.
        Inputs live in static tensors that ``decode_step`` fills before every replay; rows beyond the live batch have
        length 0 and write their K/V into block 0, which no sequence owns."""
        shared = () if prefix is None else (prefix.items, *ops.ext().paged_shared_split(B, prefix.heads, prefix.kv_heads, prefix.pieces, prefix.own))
        key = (B, max_blocks, shared)
        ent = self._graphs.get(key)
        if ent is not None:
            return ent
        dev = self.device
        ints = torch.zeros(B * (max_blocks + 2), dtype=torch.int32, device=dev)       # filled by one copy per step
        st = {'tokens': torch.zeros(B, dtype=torch.long, device=dev), 'ints': ints, 'table': ints[:B * max_blocks].view(B, max_blocks),
              'seq_lens': ints[B * max_blocks:B * (max_blocks + 1)], 'slots': ints[B * (max_blocks + 1):], 'prefix': None, 'holds': None}
        if prefix is not None:
            st['prefix'], st['holds'] = prefix._replace(plan=prefix.plan.clone()), prefix.plan

        def body():
            # the token of a step is the last of its sequence; rows that fill up the batch have length 0 and position 0
            return self._decode_body(st['tokens'], (st['seq_lens'] - 1).clamp_min(0).long(), st['table'], st['seq_lens'], None, slots=st['slots'], prefix=st['prefix'])

        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):  # warm-up outside the capture: one-time kernel attribute set-up, allocator warm-up
            for _ in range(2):
                body()
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st['logits'] = body()
        st['graph'] = graph
        self._graphs[key] = st
        return st

    def _captured(self, B: int, max_blocks: int, prefix: Optional[ops.SharedPrefix]):
        """``_graph_for``, or None with a warning: capture is an optimisation, the eager path is always valid."""
        try:
            return self._graph_for(B, max_blocks, prefix)
        except Exception as e:
            import logging
            logging.getLogger('twinkle_b200').warning(f'CUDA-graph capture of the decode step failed ({type(e).__name__}: {e}); running {"eagerly" if prefix is None else "without shared reading"}')
            return None

    @torch.no_grad()
    def decode_step(self, seqs: List[_Seq], last_tokens: torch.Tensor) -> torch.Tensor:
        """One token for every sequence; returns logits ``[B, V]`` (fp32).  On a GPU the per-token work of a whole
        layer stack is a few dozen short kernels, so the step is replayed from a CUDA graph (one per batch-size
        bucket) unless adapters or routing capture need the eager path."""
        B = len(seqs)
        max_blocks = max(len(s.blocks) for s in seqs)
        lora = self._lora_for(seqs, [1] * B)
        use_graph = (self.use_cuda_graphs and self.device.type == 'cuda' and lora is None and not self.capture_routing and not self.cfg.is_moe
                     and not any(getattr(l, 'is_linear', False) for l in self.model.layers) and not any(s.rope_delta for s in seqs)
                     # windows, score caps and latent attention decode through the PyTorch form, which reads lengths on the host
                     and not self.cfg.sliding_window and not self.cfg.attn_logit_softcapping and not self.cfg.is_mla and not self.cfg.attn_sinks)
        if use_graph:
            Bb = 1 << max(B - 1, 0).bit_length()
            Mb = 1 << max(max_blocks - 1, 0).bit_length()
            prefix = self._shared(seqs, Bb, captured=True) if self._share_captured else None
            st = self._captured(Bb, Mb, prefix)
            if st is None and prefix is not None:       # pages are then read per sequence
                self._share_captured, prefix = False, None
                st = self._captured(Bb, Mb, None)
            if st is None:
                self.use_cuda_graphs = False
            if st is not None:
                # a fresh pinned tensor each time: the allocator hands it out again only when the copy is done
                ints = torch.empty(Bb * (Mb + 2), dtype=torch.int32, pin_memory=True)
                ops.ext().pack_step(ints, Bb, Mb, [s.blocks for s in seqs], [s.length for s in seqs], [s.state_slot for s in seqs])
                st['ints'].copy_(ints, non_blocking=True)
                if prefix is not None and st['holds'] is not prefix.plan:
                    st['prefix'].plan.copy_(prefix.plan)
                    st['holds'] = prefix.plan
                if B < Bb:
                    st['tokens'].zero_()
                st['tokens'][:B].copy_(last_tokens)
                st['graph'].replay()
                return st['logits'][:B]
        positions = torch.tensor([s.length - 1 for s in seqs], device=self.device)
        table = torch.zeros(B, max_blocks, dtype=torch.int32, device=self.device)
        for i, s in enumerate(seqs):
            table[i, :len(s.blocks)] = torch.tensor(s.blocks, dtype=torch.int32)
        seq_lens = torch.tensor([s.length for s in seqs], dtype=torch.int32, device=self.device)
        self.model.set_record_routing(self.capture_routing)
        deltas = [s.rope_delta for s in seqs]
        rope_pos = positions + torch.tensor(deltas, device=self.device) if any(deltas) else None
        slots = torch.tensor([s.state_slot for s in seqs], dtype=torch.int32, device=self.device)
        logits = self._decode_body(last_tokens, positions, table, seq_lens, lora, seqs, rope_pos, slots, self._shared(seqs, B))
        if self.capture_routing:
            routed = self.model.collect_routed_experts()  # per layer [B, k]: the experts of the token just fed
            if routed is not None:
                for i, s in enumerate(seqs):
                    rows = [r[i:i + 1].cpu() for r in routed]
                    s.routed = rows if s.routed is None else [torch.cat([a, b], 0) for a, b in zip(s.routed, rows)]
        return logits

    # ------------------------------------------------------------- sampling
    def _sample(self, seqs: List[_Seq], logits: torch.Tensor) -> Tuple[List[int], List[float], List[Optional[List[Tuple[int, float]]]]]:
        toks, lps, tops = [], [], []
        groups: Dict[Tuple, List[int]] = {}
        for i, s in enumerate(seqs):
            p = s.params
            groups.setdefault((p.temperature, p.top_k, p.top_p, p.repetition_penalty != 1.0 or s.generator is not None, i if (
                p.repetition_penalty != 1.0 or s.generator is not None) else -1), []).append(i)
        out_tok = [0] * len(seqs)
        out_lp = [0.0] * len(seqs)
        out_top: List[Optional[List[Tuple[int, float]]]] = [None] * len(seqs)
        for (temp, tk, tp, _special, _), idxs in groups.items():
            lg = logits[idxs]
            for j, i in enumerate(idxs):
                rp = seqs[i].params.repetition_penalty
                if rp != 1.0:
                    seen = torch.tensor(sorted(set(seqs[i].prompt + seqs[i].tokens)), device=lg.device)
                    vals = lg[j, seen]
                    lg[j, seen] = torch.where(vals > 0, vals / rp, vals * rp)
            gen = seqs[idxs[0]].generator if len(idxs) == 1 else None
            tok, lp = ops.ref.sample_tokens(lg, temp, tk, tp, gen) if not lg.is_cuda else ops.sample_tokens(lg, temp, tk, tp, gen)
            for j, i in enumerate(idxs):
                out_tok[i], out_lp[i] = int(tok[j]), float(lp[j])
                k = seqs[i].params.logprobs
                if k and k > 1:
                    proc = torch.log_softmax(lg[j] / max(temp, 1e-6), -1) if temp > 0 else torch.log_softmax(lg[j], -1)
                    v, ix = proc.topk(min(k, proc.numel()))
                    out_top[i] = [(int(a), float(b)) for a, b in zip(ix, v)]
        return out_tok, out_lp, out_top

    def _check_stop(self, s: _Seq, tok: int, eos: Optional[int]) -> None:
        p = s.params
        if (eos is not None and tok == eos) or tok in p.stop_token_ids():
            s.done, s.stop_reason = True, 'stop'
            return
        strs = p.stop_strings()
        if strs and self.decode_text is not None:
            s.text_tail = (s.text_tail + self.decode_text([tok]))[-256:]
            if any(x in s.text_tail for x in strs):
                s.done, s.stop_reason = True, 'stop'
                return
        if p.max_tokens is not None and len(s.tokens) >= p.max_tokens:
            s.done, s.stop_reason = True, 'length'

    # ----------------------------------------------------------------- API
    @torch.no_grad()
    def generate(self, prompts: List[List[int]], params: List[SamplingParams], lora: Optional[List[Optional[Dict[str, Any]]]] = None,
                 eos_token_id: Optional[int] = None, on_token: Optional[Callable[[int, int, float], None]] = None,
                 vision: Optional[List[Optional[Dict[str, Any]]]] = None) -> List[SampleResponse]:
        """``prompts[i]`` is sampled ``params[i].num_samples`` times.  ``lora[i]`` = ``{slot, rank, scale, target}`` or None."""
        responses = [SampleResponse() for _ in prompts]
        seqs: List[_Seq] = []
        for i, (pr, sp) in enumerate(zip(prompts, params)):
            lo = (lora[i] if lora else None) or {}
            for n in range(sp.num_samples):
                g = None
                if sp.seed is not None:
                    g = torch.Generator(device=self.device).manual_seed(sp.seed + n)
                seqs.append(_Seq(i, list(pr), sp, lo.get('slot', -1), lo.get('rank', 0), lo.get('scale', 0.0), lo.get('target'), generator=g,
                                 vision=vision[i] if vision else None))
        for lo_i in range(0, len(seqs), self.max_batch):
            self._run_group(seqs[lo_i:lo_i + self.max_batch], responses, eos_token_id, on_token)
        return responses

    def _start(self, seqs: List[_Seq]) -> Tuple[List[_Seq], torch.Tensor, List[int]]:
        """Run the prompts; ``(sequences, hidden states, first row of every sequence in them)``.  With shared prompts each different one runs
        once, and its sequences come one after the other."""
        firsts, order = list(range(len(seqs))), list(range(len(seqs)))
        if self.share_prompts:
            seen: Dict[Any, int] = {}
            for i, s in enumerate(seqs):
                if s.vision is None:
                    firsts[i] = seen.setdefault((tuple(s.prompt), s.slot, s.lora_rank, s.lora_scale, id(s.lora_target)), i)
            order.sort(key=lambda i: (firsts[i], i))
        run = [i for i in order if firsts[i] == i]
        hidden = self.prefill([seqs[i] for i in run])
        row, at = {}, 0
        for i in run:
            row[i] = at
            at += len(seqs[i].prompt)
        for i in run:
            others = [seqs[j] for j in order if firsts[j] == i and j != i and not seqs[j].params.scoring_only]
            if others:
                self._fork(seqs[i], others)
        return [seqs[i] for i in order], hidden, [row[firsts[i]] for i in order]

    def _run_group(self, seqs: List[_Seq], responses, eos, on_token) -> None:
        seqs, hidden, begins = self._start(seqs)
        lens = [len(s.prompt) for s in seqs]
        ends = torch.tensor([a + n - 1 for a, n in zip(begins, lens)], device=self.device)
        # prompt scoring (teacher logprobs for distillation / max_tokens == 0)
        need_prompt = [s.params.prompt_logprobs is not None for s in seqs]
        if any(need_prompt):
            for s, off, n, need in zip(seqs, begins, lens, need_prompt):
                if need and responses[s.request].prompt_logprobs is None:
                    h = hidden[off:off + n]
                    ids = torch.tensor(s.prompt[1:] + [0], device=self.device)
                    temp = s.params.temperature if s.params.temperature > 0 else 1.0
                    lp, _ = ops.fused_linear_logprob(h, self.model.head_weight(), ids, temp)
                    responses[s.request].prompt_logprobs = [None] + [float(x) for x in lp[:-1]]
                    k = s.params.prompt_logprobs
                    if k and k > 0:
                        lg = torch.log_softmax(self.model.logits(h[:-1]).float() / temp, -1)
                        v, ix = lg.topk(min(k, lg.shape[-1]), -1)
                        responses[s.request].topk_prompt_logprobs = [None] + [[(int(a), float(b)) for a, b in zip(r_i, r_v)]
                                                                             for r_i, r_v in zip(ix.tolist(), v.tolist())]
        live = [s for s in seqs if not s.params.scoring_only]
        for s in seqs:
            if s.params.scoring_only:
                s.done = True
        if live:
            idx = [i for i, s in enumerate(seqs) if not s.params.scoring_only]
            logits = self.model.logits(hidden[ends[idx]]).float()
            while live:
                toks, lps, tops = self._sample(live, logits)
                for s, t, lp, tp in zip(live, toks, lps, tops):
                    s.tokens.append(t)
                    s.logprobs.append(lp)
                    if tp is not None:
                        s.topk.append(tp)
                    if on_token is not None:
                        on_token(s.request, t, lp)
                    self._check_stop(s, t, eos)
                nxt = [s for s in live if not s.done]
                if not nxt:
                    break
                last = torch.tensor([s.tokens[-1] for s in nxt], device=self.device)
                self.grow(nxt)
                logits = self.decode_step(nxt, last)
                live = nxt
        self.release(seqs)
        if self.device.type == 'cuda':       # before any result leaves: a key that was not stored, a kernel that gave up waiting
            torch.cuda.current_stream(self.device).synchronize()
            with torch.cuda.device(self.device):
                code = ops.ext().read_and_clear_error()
            if code:
                raise RuntimeError(f'a kernel reported error {code} during generation (a block outside the cache, or a bounded wait that expired)')
        for s in seqs:
            if not s.params.scoring_only:
                responses[s.request].sequences.append(SampledSequence(stop_reason=s.stop_reason, tokens=s.tokens, logprobs=s.logprobs,
                                                                      topk_logprobs=s.topk or None, routed_experts=s.routed))

    def reset_prefix_cache(self) -> None:
        """No cross-request prefix reuse is kept, so there is nothing stale to drop after a weight update."""
        return None
