"""Llama-3-70B-architecture decode stack under Helix context parallelism.

One decode step of the attention block of every layer on one CP rank::

    split-KV paged attention over the LOCAL KV shard   ->  (o [B, Hq, D], lse [B, Hq])
    Helix exchange + LSE combine (head scatter)        ->  x [B, Hq/N, D]
    o_proj with this rank's K-slice of W_o             ->  y [B, hidden]   (partial sum over ranks)

The KV cache of every sequence is split evenly over the ``cp_size`` ranks; each rank holds all KV
heads of its shard.  Weights are random-init (N(0, 0.02)), KV ~ N(0, 1): there is no checkpoint
loading here, the stack exists to drive and measure the kernels on the shapes of a real model.

With ``draft_tokens`` the stack also verifies drafted tokens (:meth:`HelixDecodeStack.verify_step`): the step's new tokens of all sequences
get their pages and slots on the device, their K and V go into this rank's part of the cache, every token attends to the cache and
to its ancestors in the tree, and :meth:`HelixDecodeStack.commit` keeps those that were accepted.
The reference leaves all of this to vLLM (``benchmark/sbatch/run_gb200_aiperf_v3.sbatch:284-305``).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional

import torch
import torch.distributed as dist

from .. import api
from ..ops import attention, oproj as oproj_mod, paged
from ..ops._ext import ext
from ..utils import env
from ..utils.tracing import nvtx_range


@dataclass
class LlamaDecodeConfig:
    n_layers: int = 80
    n_q_heads: int = 64
    n_kv_heads: int = 8
    head_dim: int = 128
    hidden: int = 8192
    page_size: int = 16
    dtype: torch.dtype = torch.bfloat16

    @staticmethod
    def llama3_70b(**kw) -> "LlamaDecodeConfig":
        return LlamaDecodeConfig(**kw)

    @staticmethod
    def tiny(**kw) -> "LlamaDecodeConfig":
        base = dict(n_layers=2, n_q_heads=16, n_kv_heads=2, head_dim=128, hidden=256)
        base.update(kw)
        return LlamaDecodeConfig(**base)


class HelixDecodeStack:
    """KV cache shard, o_proj slices and workspace of one CP rank, plus the decode step."""

    def __init__(self, cfg: LlamaDecodeConfig, *, batch: int, local_ctx: int, cp_size: int = 1, cp_rank: int = 0,
                 group: Optional[dist.ProcessGroup] = None, device="cuda", seed: int = 0,
                 workspace: Optional[torch.Tensor] = None, kv_std: float = 1.0,
                 fuse_oproj: Optional[bool] = False, draft_tokens: int = 0, w_bits: int = 16):
        """``draft_tokens``: most tokens of one sequence that :meth:`verify_step` and :meth:`commit` will ever add (pages are set aside
        for them); ``w_bits=4`` keeps the o_proj weights in 4 bits with a scale per 128 columns."""
        assert cfg.n_q_heads % cp_size == 0, "query heads must divide evenly over the CP ranks"
        self.cfg, self.batch, self.local_ctx = cfg, batch, local_ctx
        self.cp_size, self.cp_rank, self.group = cp_size, cp_rank, group
        self.device = torch.device(device)
        self.heads_local = cfg.n_q_heads // cp_size
        # exchange + combine + o_proj as one kernel: True / False, or None = whenever the shape fits that kernel
        # (a request that does not fit runs the two-kernel chain, and is counted as such)
        fits = cp_size > 1 and self.device.type == "cuda" and api.alltoall_combine_oproj_fits(
            batch, self.heads_local, cfg.head_dim, cfg.hidden, cp_size)
        self.fuse_oproj = (bool(fits) if fuse_oproj is None else bool(fuse_oproj and fits)) and w_bits == 16
        self.k_local = self.heads_local * cfg.head_dim
        self.scale = 1.0 / math.sqrt(cfg.head_dim)
        gen = torch.Generator(device=self.device)
        gen.manual_seed(seed * 1000 + cp_rank)
        pages_per_seq = (local_ctx + cfg.page_size - 1) // cfg.page_size
        if w_bits not in (4, 16):
            raise ValueError("w_bits must be 4 or 16")
        self.w_bits = w_bits
        self.draft_tokens = draft_tokens
        self.plan: Optional[paged.TablePlan] = None
        spare = batch * ((draft_tokens + cfg.page_size - 1) // cfg.page_size + 1) if draft_tokens else 0
        self.n_pages = batch * pages_per_seq + spare
        # pages of a sequence are scattered over the pool, as a paged allocator would leave them
        perm = torch.randperm(self.n_pages, generator=torch.Generator().manual_seed(seed)).int()
        owned = perm[:batch * pages_per_seq].view(batch, pages_per_seq)
        self.block_table = torch.nn.functional.pad(owned, (0, spare // batch if spare else 0)).to(self.device)
        self.seq_lens = torch.full((batch,), local_ctx, dtype=torch.int32, device=self.device)
        # state of ops.paged.extend_tables: the pages each sequence holds, the free ones, committed tokens over all ranks
        self.held = torch.full((batch,), pages_per_seq, dtype=torch.int32, device=self.device)
        self.free_pages = perm[batch * pages_per_seq:].to(self.device)
        self.free_used = torch.zeros(1, dtype=torch.int32, device=self.device)
        # pages and mask bits that were not to be had, over all calls so far (see check_room)
        self.lost = torch.zeros(1, dtype=torch.int64, device=self.device)
        self.ctx_lens = torch.full((batch,), local_ctx * cp_size, dtype=torch.int32, device=self.device)
        shape = (self.n_pages, cfg.n_kv_heads, cfg.page_size, cfg.head_dim)
        self.k_cache: List[torch.Tensor] = []
        self.v_cache: List[torch.Tensor] = []
        self.w_o: List[torch.Tensor] = []
        self.prepack_oproj = env.oproj_prepack()
        self._w_o_packed = [None] * cfg.n_layers
        for _ in range(cfg.n_layers):
            k = torch.empty(shape, dtype=cfg.dtype, device=self.device).normal_(0, kv_std, generator=gen)
            v = torch.empty(shape, dtype=cfg.dtype, device=self.device).normal_(0, kv_std, generator=gen)
            w = torch.empty(cfg.hidden, self.k_local, dtype=cfg.dtype, device=self.device).normal_(0, 0.02, generator=gen)
            self.k_cache.append(k)
            self.v_cache.append(v)
            self.w_o.append(w)
        if workspace is not None:
            self.workspace = workspace
        elif cp_size > 1:
            self.workspace = api.allocate_workspace(cp_size, cp_rank, device=device if self.device.type == "cpu" else "cuda",
                                                    mnnvl=True, cpu_group=group)
            api.init_workspace(self.workspace, cp_rank, cp_size)
            dist.barrier(group=group)
        else:
            self.workspace = None
        self._graph = None
        self._static_q = None
        self._static_y = None

    # ---- one layer / one step --------------------------------------------------------------------
    @property
    def max_local(self) -> int:
        """Most tokens that a sequence can have on this rank."""
        return self.block_table.shape[1] * self.cfg.page_size if self.draft_tokens else self.local_ctx

    def layer(self, l: int, q: torch.Tensor) -> torch.Tensor:
        with nvtx_range(f"layer{l}.attention"):
            o, lse = attention.gqa_decode(q, self.k_cache[l], self.v_cache[l], self.block_table, self.seq_lens,
                                          scale=self.scale, max_seq_len=self.max_local, kv_stable=True)
        if self.cp_size > 1 and self.fuse_oproj:
            # exchange + combine + o_proj in one launch: W_o streams while the exchange is in flight
            return api.alltoall_combine_oproj(o, lse, self._oproj_weight(l), self.workspace, self.cp_rank, self.cp_size)
        if self.cp_size > 1:
            x = api.alltoall_combine(o, lse, self.workspace, self.cp_rank, self.cp_size)
        else:
            x = o
        return oproj_mod.oproj(x.reshape(self.batch, self.k_local), self._oproj_weight(l))

    def _oproj_weight(self, l: int):
        """The layer's o_proj weight in the layout the GEMM streams fastest: packed once, on first use
        (one contiguous bulk copy per pipeline stage instead of strided tensor copies); the plain matrix
        stays in ``w_o`` for the one-kernel path and for oracles.  ``prepack_oproj=False`` keeps the plain one."""
        if self.w_bits == 4:
            if self._w_o_packed[l] is None:
                self._w_o_packed[l] = oproj_mod.quantize_weight_int4(self.w_o[l], 128)
            return self._w_o_packed[l]
        if not self.prepack_oproj or not self.w_o[l].is_cuda or self.w_o[l].shape[0] % 128 or self.w_o[l].shape[1] % 64:
            return self.w_o[l]
        if self._w_o_packed[l] is None:
            self._w_o_packed[l] = oproj_mod.prepack_weight(self.w_o[l])
        return self._w_o_packed[l]

    def decode_step(self, q_all: torch.Tensor) -> torch.Tensor:
        """``q_all [L, B, Hq, D]`` on the device -> ``y [L, B, hidden]`` (this rank's partial sums)."""
        ys = [self.layer(l, q_all[l]) for l in range(self.cfg.n_layers)]
        return torch.stack(ys)

    def _run_layers(self, q_all: torch.Tensor, l0: int, l1: int) -> torch.Tensor:
        y = None
        for l in range(l0, l1):
            y = self.layer(l, q_all[l])
        return y

    def _step_last(self, q_all: torch.Tensor) -> torch.Tensor:
        return self._run_layers(q_all, 0, self.cfg.n_layers)

    # ---- drafted tokens ---------------------------------------------------------------------------
    def _extend(self, q_start: torch.Tensor, rows: int, parents, mask_words: int) -> paged.TablePlan:
        plan = paged.extend_tables(self.block_table, self.held, self.free_pages, self.free_used, self.ctx_lens, q_start, rows=rows,
                                   page_size=self.cfg.page_size, parents=parents, mask_words=mask_words, cp_size=self.cp_size,
                                   cp_rank=self.cp_rank)
        self.lost += plan.missing
        if mask_words and rows > 64 * mask_words * self.cp_size:         # one sequence may have more tokens here than a mask has bits
            self.lost += (plan.draft_lens - 64 * mask_words).clamp(min=0).sum()
        return plan

    def check_room(self) -> None:
        """Raise if a :meth:`verify_step` or :meth:`commit` so far had tokens for which there was no page or no mask bit (waits for the
        device).  From such a call on the outputs are wrong: tokens that are stored nowhere are counted, or do not see themselves."""
        lost = int(self.lost)
        if lost:
            raise RuntimeError(f"this stack has outgrown draft_tokens={self.draft_tokens}: {lost} pages or mask bits were missing")

    def verify_step(self, q_all: torch.Tensor, k_all: torch.Tensor, v_all: torch.Tensor, q_start: torch.Tensor,
                    parents: Optional[torch.Tensor] = None, *, max_new: int = 0) -> torch.Tensor:
        """One pass over drafted tokens: ``q_all [L, rows, Hq, D]``, ``k_all`` / ``v_all [L, rows, Hkv, D]``, rows ``q_start[b]`` to
        ``q_start[b + 1]`` are sequence ``b``'s, ``parents [rows]`` their tree (``None``: chains), at most 256 of a sequence on a
        rank; see :func:`ops.paged.extend_tables`.  ``max_new``: most tokens of one sequence in this step (0: unknown, up to
        ``draft_tokens``); masks are made for so many, and the attention is divided by it.
        Returns ``y [L, rows, hidden]`` (this rank's partial sums).  Committed lengths stay as they are: the next call overwrites
        the drafted tokens, unless :meth:`commit` keeps some.  No host synchronisation, so the step can be captured.  ``plan`` holds
        the step's places; :meth:`check_room` says whether all tokens of all steps had one."""
        if not self.draft_tokens:
            raise RuntimeError("this stack was made without draft_tokens")
        if not 0 <= max_new <= min(self.draft_tokens, 256 * self.cp_size):
            raise ValueError(f"max_new must be at most draft_tokens ({self.draft_tokens}) and 256 on a rank")
        rows = q_all.shape[1]
        longest = max_new or max(min(self.draft_tokens, rows), 1)
        words = min((longest + 64 * self.cp_size - 1) // (64 * self.cp_size), 4)       # a rank holds every cp_size-th token
        plan = self.plan = self._extend(q_start, rows, parents, words)
        ys = []
        for l in range(self.cfg.n_layers):
            paged.append_kv(k_all[l], v_all[l], self.k_cache[l], self.v_cache[l], plan.slots)
            with nvtx_range(f"layer{l}.tree_attention"):
                o, lse = attention.tree_decode(q_all[l], self.k_cache[l], self.v_cache[l], self.block_table, plan.seq_lens, q_start,
                                               plan.draft_lens, plan.mask, scale=self.scale, max_seq_len=self.max_local, max_q_len=longest)
            x = api.alltoall_combine(o, lse, self.workspace, self.cp_rank, self.cp_size) if self.cp_size > 1 else o
            ys.append(oproj_mod.oproj(x.reshape(rows, self.k_local), self._oproj_weight(l)))
        return torch.stack(ys)

    def commit(self, k_all: torch.Tensor, v_all: torch.Tensor, accepted: torch.Tensor, q_start: torch.Tensor) -> None:
        """Keep drafted tokens: ``accepted`` are their rows in ``k_all`` / ``v_all``, in the order of their positions, and ``q_start [B + 1]``
        says which of them belong to which sequence.  A path through a tree becomes a run of tokens behind the committed ones.
        Tokens without a page (:meth:`check_room`) count as committed all the same: lengths are those of all ranks."""
        if not self.draft_tokens:
            raise RuntimeError("this stack was made without draft_tokens")
        plan = self.plan = self._extend(q_start, accepted.numel(), None, 0)
        for l in range(self.cfg.n_layers):
            paged.append_kv(k_all[l][accepted], v_all[l][accepted], self.k_cache[l], self.v_cache[l], plan.slots)
        self.ctx_lens += q_start.diff()
        self.seq_lens.copy_(plan.seq_lens)

    # ---- end-to-end call: pinned host input -> host output ---------------------------------------
    def capture(self, q_example: torch.Tensor, head_layers: Optional[int] = None) -> None:
        """Capture the step in CUDA graphs (call after at least one eager warm-up step).

        Two graphs: the first ``head_layers`` layers and the rest.  ``decode_step_host`` copies the
        queries of the head layers, starts the head graph, and lets the (much larger) copy of the
        remaining layers' queries run on a second stream underneath it; the tail graph waits for that
        copy.  With one graph the whole host-to-device copy sat in front of the first kernel."""
        L = self.cfg.n_layers
        if head_layers is None:
            head_layers = min(8, L // 2)
        self._head_layers = head_layers if 0 < head_layers < L else 0
        self._static_q = torch.empty_like(q_example, device=self.device)
        self._static_q.copy_(q_example)
        self._copy_stream = torch.cuda.Stream(device=self.device)
        self._copy_done = torch.cuda.Event()
        s = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(s):
            self._step_last(self._static_q)
            self._graphs = []
            bounds = [(0, self._head_layers), (self._head_layers, L)] if self._head_layers else [(0, L)]
            for l0, l1 in bounds:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    self._static_y = self._run_layers(self._static_q, l0, l1)
                self._graphs.append(g)
        torch.cuda.current_stream(self.device).wait_stream(s)
        self._graph = self._graphs[-1]

    def _replay(self) -> None:
        for g in self._graphs:
            g.replay()

    def decode_step_device(self, q_dev: torch.Tensor) -> torch.Tensor:
        """Step on device-resident ``q``; returns the last layer's ``y`` (``[B, hidden]``)."""
        if self._graph is not None:
            self._static_q.copy_(q_dev, non_blocking=True)
            self._replay()
            return self._static_y
        return self._step_last(q_dev)

    def decode_step_host(self, q_pinned: torch.Tensor, out_pinned: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Public end-to-end step: copies ``q`` from pinned host memory, runs every layer, copies
        the result (``[B, hidden]``) back to the host and waits for it."""
        main = torch.cuda.current_stream(self.device)
        if self._graph is not None:
            k = self._head_layers
            if k:
                # the previous step ended with a synchronize, so nothing still reads _static_q
                self._static_q[:k].copy_(q_pinned[:k], non_blocking=True)
                self._copy_stream.wait_stream(main)
                with torch.cuda.stream(self._copy_stream):
                    self._static_q[k:].copy_(q_pinned[k:], non_blocking=True)
                    self._copy_done.record(self._copy_stream)
                self._graphs[0].replay()
                main.wait_event(self._copy_done)
                self._graphs[1].replay()
            else:
                self._static_q.copy_(q_pinned, non_blocking=True)
                self._replay()
            y = self._static_y
        else:
            q_dev = torch.empty_like(q_pinned, device=self.device)
            q_dev.copy_(q_pinned, non_blocking=True)
            y = self._step_last(q_dev)
        if out_pinned is None:
            out_pinned = torch.empty(y.shape, dtype=y.dtype, pin_memory=True)
        out_pinned.copy_(y, non_blocking=True)
        main.synchronize()
        return out_pinned

    # ---- accounting ------------------------------------------------------------------------------
    def kernels_per_step(self) -> int:
        """Kernels of this library that one step launches (a split attention or o_proj call is two); counted for a GPU of 148
        SMs where the stack is not on one."""
        sms = torch.cuda.get_device_properties(self.device).multi_processor_count if self.device.type == "cuda" else 148
        attn = ext().gqa_launches(self.batch, self.cfg.n_kv_heads, self.max_local, sms)
        if self.cp_size > 1 and self.fuse_oproj:
            return self.cfg.n_layers * (attn + 1)
        if self.w_bits == 4:
            return self.cfg.n_layers * (attn + (1 if self.cp_size > 1 else 0) + -(-self.batch // 128))
        packed = self.prepack_oproj and self.cfg.hidden % 128 == 0 and self.k_local % 64 == 0
        own = packed or not oproj_mod.library_gemm_pays(self.batch, self.k_local)
        proj = ext().oproj_launches(self.batch, self.cfg.hidden, self.k_local, packed, sms) if own else 0
        return self.cfg.n_layers * (attn + (1 if self.cp_size > 1 else 0) + proj)

    def h2d_bytes_per_step(self) -> int:
        c = self.cfg
        return c.n_layers * self.batch * c.n_q_heads * c.head_dim * 2

    def d2h_bytes_per_step(self) -> int:
        return self.batch * self.cfg.hidden * 2
